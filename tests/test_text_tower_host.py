"""CPU: frequencies and 4-bit weights made on the host, and what the text tower's ops refuse (on a
context without a device, so that nothing can be launched)."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NONE, LINEAR, THETA, PARTS = range(4)


def frequencies(dim, theta, scaling=NONE, factor=1.0, trained=0):
    f, m = np.zeros(dim // 2, np.float32), C.c_float()
    ok = abi.load().qw_rotary_frequencies_host(dim, theta, scaling, factor, trained, abi._ptr(f), C.byref(m))
    return ok, f, m.value


def test_frequencies():
    i = np.arange(64)
    plain = 1e6 ** (-i / 64)
    ok, f, m = frequencies(128, 1e6)
    assert ok and m == 1.0
    np.testing.assert_allclose(f, plain, rtol=2 ** -24)
    ok, f, m = frequencies(128, 1e6, LINEAR, 4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=2 ** -24)
    ok, f, m = frequencies(128, 1e6, THETA, 4.0)
    assert f[0] == 1.0 and m == 1.0
    np.testing.assert_allclose(f[-1], plain[-1] / 4, rtol=1e-6)
    ok, f, m = frequencies(128, 1e6, PARTS, 4.0, 8192)
    turns = 8192 * plain / (2 * math.pi)
    np.testing.assert_allclose(f[turns > 32], plain[turns > 32], rtol=2 ** -24)
    np.testing.assert_allclose(f[turns < 1], plain[turns < 1] / 4, rtol=2 ** -24)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((f < plain) & (f > plain / 4))[between].all()
    np.testing.assert_allclose(m, 0.1 * math.log(4) + 1, rtol=1e-6)


@pytest.mark.parametrize("args", [(0, 1e4), (7, 1e4), (8, 0.0), (8, -1.0), (8, math.inf), (8, math.nan),
                                  (8, 1e4, LINEAR, 0.5), (8, 1e4, LINEAR, math.nan), (8, 1e4, 4, 2.0),
                                  (8, 1e4, PARTS, 2.0, 0), (2, 1e4, THETA, 2.0)])
def test_frequencies_refused(args):
    assert not frequencies(*args)[0]


@pytest.mark.parametrize("outputs,inputs,group", [(1, 32, 32), (3, 192, 64), (5, 256, 128), (2, 512, 256)])
def test_quantized_weights(outputs, inputs, group):
    rng = np.random.default_rng(outputs)
    w = R.random_bf16(rng, outputs, inputs)
    w[0, :group] = 0  # a group of zeros
    packed = np.zeros((outputs, inputs // 8), np.uint32)
    scales = np.zeros((outputs, inputs // group), np.uint16)
    assert abi.load().qw_w4_quantize_host(abi._ptr(w), outputs, inputs, group, abi._ptr(packed), abi._ptr(scales))
    s = np.repeat(R.wide(scales), group, 1)
    q = R.unpack(packed).astype(np.float64) - 8
    x = R.wide(w)
    most = np.abs(x).reshape(outputs, -1, group).max(-1)
    np.testing.assert_allclose(R.wide(scales), most / 7, rtol=R.HALF_STEP)
    want = np.clip(np.rint(np.divide(x, s, out=np.zeros_like(x), where=s > 0)), -8, 7)
    assert (q == want).all()
    # half a step of the grid, and what the scale's rounding takes from the largest
    assert (np.abs(s * q - x) <= 0.5 * s + np.abs(x) * R.HALF_STEP * 1.01).all()


def test_quantize_refused():
    w, p, s = np.zeros(256, np.uint16), np.zeros(64, np.uint32), np.zeros(64, np.uint16)
    fn = abi.load().qw_w4_quantize_host
    for outputs, inputs, group in ((0, 32, 32), (1, 0, 32), (1, 32, 0), (1, 48, 48), (1, 96, 64), (1, 192, 192)):
        assert not fn(abi._ptr(w), outputs, inputs, group, abi._ptr(p), abi._ptr(s))
    for bits in (0x7f80, 0xff80, 0x7fc0):
        w[5] = bits
        assert not fn(abi._ptr(w), 1, 32, 32, abi._ptr(p), abi._ptr(s))


# ---- refusals ------------------------------------------------------------------


class Fake:
    def __init__(self, folder):
        out = os.path.join(folder, "libfake_context.so")
        cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
        subprocess.check_call(["gcc", "-std=c11", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                               "-I" + os.path.join(ROOT, "qwen_metal_b200", "csrc"), "-I" + cuda + "/include",
                               os.path.join(ROOT, "tests", "fake_context.c"), "-o", out])
        self.own, self.lib = C.CDLL(out), abi.load()
        self.own.fake_context.restype = self.own.fake_tensor.restype = C.c_void_p
        self.own.fake_open.argtypes = [C.c_void_p, C.c_int]
        self.own.fake_tensor.argtypes = [C.c_void_p, C.c_int, C.c_size_t]
        # (a device that no machine has: a call that passes its checks ends there)
        self.gpu, self.other = self.own.fake_context(4096, 1), self.own.fake_context(4097, 1)

    def bf16(self, n, gpu=None):
        return self.own.fake_tensor(gpu or self.gpu, abi.BF16, n)

    def u32(self, n):
        return self.own.fake_tensor(self.gpu, abi.U32, n)

    def f32(self, n):
        return self.own.fake_tensor(self.gpu, abi.F32, n)

    def says(self, name, args, open_chain=True):
        """What a call with these named arguments answers."""
        self.own.fake_open(self.gpu, int(open_chain))
        assert getattr(self.lib, name)(self.gpu, *args.values()) == 0
        return self.lib.h3_gpu_error(self.gpu).decode()


PASSED = "unknown CUDA error"  # no message: the checks had nothing to say


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return Fake(str(tmp_path_factory.mktemp("fake")))


def rotary_args(f, tokens=5, heads=4, kv=2, dim=64, rotary=64):
    return dict(qo=f.bf16(tokens * heads * dim), ko=f.bf16(tokens * kv * dim),
                q=f.bf16(tokens * heads * dim), k=f.bf16(tokens * kv * dim), positions=f.u32(tokens),
                frequencies=f.f32(rotary // 2), tokens=tokens, heads=heads, kv_heads=kv, head_dim=dim,
                rotary_dim=rotary, layout=0, magnitude=1.0)


def test_rotary_refusals(fake):
    base, name = rotary_args(fake), "qw_gpu_rotary_bf16"
    assert fake.says(name, base) == PASSED
    assert fake.says(name, dict(base, qo=base["q"], ko=base["k"])) == PASSED
    assert fake.says(name, dict(base, ko=None, k=None)) == PASSED
    assert "h3_gpu_begin" in fake.says(name, base, open_chain=False)
    short = dict(qo=fake.bf16(5 * 4 * 64 - 1), q=None, ko=None, k=fake.bf16(1), positions=fake.u32(4),
                 frequencies=fake.f32(31))
    for key, bad in short.items():
        assert "absent or too small" in fake.says(name, {**base, key: bad}), key
    assert "not BF16" in fake.says(name, dict(base, q=fake.f32(5 * 4 * 64)))
    assert "not U32" in fake.says(name, dict(base, positions=fake.f32(5)))
    assert "not F32" in fake.says(name, dict(base, frequencies=fake.bf16(32)))
    assert "another device" in fake.says(name, dict(base, q=fake.bf16(5 * 4 * 64, fake.other)))
    for change in (dict(tokens=0), dict(heads=0), dict(head_dim=63), dict(rotary_dim=66), dict(rotary_dim=0),
                   dict(rotary_dim=31), dict(head_dim=0), dict(head_dim=514, rotary_dim=64, heads=0, kv_heads=0),
                   dict(layout=2), dict(magnitude=math.inf), dict(magnitude=math.nan), dict(kv_heads=0)):
        assert fake.says(name, {**base, **change}) not in (PASSED, ""), change
    for a, b in (("qo", "ko"), ("qo", "k"), ("ko", "q")):
        big = fake.bf16(5 * 4 * 64)
        assert "also an input" in fake.says(name, {**base, a: big, b: big})
    assert "large" in fake.says(name, dict(base, tokens=2 ** 32 - 1, heads=2 ** 32 - 1))


def cache_args(f, batch=3, width=4, page=16, pages=7, kv=2, dim=128):
    return dict(table=f.u32(batch * width), start=f.u32(batch + 1), length=f.u32(batch)), \
        dict(kp=f.bf16(pages * page * kv * dim), vp=f.bf16(pages * page * kv * dim))


def append_args(f):
    batch, pools = cache_args(f)
    return dict(qo=f.bf16(5 * 4 * 128), **pools, q=f.bf16(5 * 4 * 128), k=f.bf16(5 * 2 * 128),
                v=f.bf16(5 * 2 * 128), positions=None, frequencies=f.f32(64), **batch, batch=3, tokens=5,
                table_width=4, page_rows=16, heads=4, kv_heads=2, head_dim=128, rotary_dim=128, layout=1,
                magnitude=1.0)


def attend_args(f):
    batch, pools = cache_args(f)
    return dict(o=f.bf16(5 * 4 * 128), q=f.bf16(5 * 4 * 128), **pools, **batch, batch=3, tokens=5, max_new=2,
                table_width=4, page_rows=16, heads=4, kv_heads=2, head_dim=128, scale=0.1)


@pytest.mark.parametrize("name,make", [("qw_gpu_rotary_append_bf16", append_args),
                                       ("qw_gpu_paged_attention_bf16", attend_args)])
def test_cache_refusals(fake, name, make):
    base = make(fake)
    assert fake.says(name, base) == PASSED
    assert "h3_gpu_begin" in fake.says(name, base, open_chain=False)
    for change in (dict(page_rows=8), dict(page_rows=24), dict(page_rows=8192), dict(page_rows=0), dict(batch=0),
                   dict(table_width=0), dict(table_width=2 ** 31, page_rows=4096), dict(tokens=0), dict(heads=0),
                   dict(kv_heads=0)):
        assert fake.says(name, {**base, **change}) not in (PASSED, ""), change
    for key, bad in dict(table=fake.u32(11), start=fake.u32(3), length=fake.u32(2), kp=fake.bf16(16 * 2 * 128 - 1),
                         vp=None, q=fake.bf16(5 * 4 * 128 - 1)).items():
        assert "absent or too small" in fake.says(name, {**base, key: bad}), key
    assert "not U32" in fake.says(name, dict(base, table=fake.f32(12)))
    assert "another device" in fake.says(name, dict(base, kp=fake.bf16(7 * 16 * 2 * 128, fake.other)))
    assert "also an input" in fake.says(name, dict(base, vp=base["kp"]))


def test_append_refusals(fake):
    base, name = append_args(fake), "qw_gpu_rotary_append_bf16"
    assert fake.says(name, dict(base, qo=base["q"])) == PASSED
    assert fake.says(name, dict(base, positions=fake.u32(5))) == PASSED
    assert "absent or too small" in fake.says(name, dict(base, positions=fake.u32(4)))
    for a, b in (("kp", "k"), ("vp", "v"), ("kp", "q"), ("qo", "kp"), ("qo", "v")):
        big = fake.bf16(7 * 16 * 2 * 128)
        assert "also an input" in fake.says(name, {**base, a: big, b: big}), (a, b)
    assert fake.says(name, dict(base, rotary_dim=130)) not in (PASSED, "")
    assert fake.says(name, dict(base, layout=7)) not in (PASSED, "")


def test_attention_refusals(fake):
    base, name = attend_args(fake), "qw_gpu_paged_attention_bf16"
    for change in (dict(head_dim=64), dict(heads=3), dict(max_new=0), dict(scale=0.0), dict(scale=-1.0),
                   dict(scale=math.inf), dict(scale=math.nan), dict(tokens=2 ** 31, heads=4)):
        assert fake.says(name, {**base, **change}) not in (PASSED, ""), change
    for other in ("q", "kp", "vp"):
        big = fake.bf16(7 * 16 * 2 * 128)
        assert "also an input" in fake.says(name, {**base, "o": big, other: big}), other


def test_linear_refusals(fake):
    name = "qw_gpu_linear_w4_bf16"
    base = dict(y=fake.bf16(3 * 10), x=fake.bf16(3 * 256), w=fake.u32(10 * 32), s=fake.bf16(10 * 2), z=None, b=None,
                rows=3, input_dim=256, output_dim=10, group=128)
    assert fake.says(name, base) == PASSED
    assert fake.says(name, dict(base, z=fake.bf16(20), b=fake.bf16(10))) == PASSED
    assert "h3_gpu_begin" in fake.says(name, base, open_chain=False)
    for change in (dict(rows=0), dict(input_dim=0), dict(output_dim=0), dict(group=0), dict(group=16), dict(group=96),
                   dict(group=192), dict(input_dim=224), dict(rows=2 ** 19 + 1), dict(output_dim=2 ** 30 + 1)):
        assert "unsupported" in fake.says(name, {**base, **change}), change
    for key, bad in dict(y=fake.bf16(29), x=fake.bf16(3 * 256 - 1), w=fake.u32(319), s=fake.bf16(19),
                         z=fake.bf16(19), b=fake.bf16(9)).items():
        assert "absent or too small" in fake.says(name, {**base, key: bad}), key
    assert "not U32" in fake.says(name, dict(base, w=fake.bf16(320)))
    assert "another device" in fake.says(name, dict(base, x=fake.bf16(3 * 256, fake.other)))
    assert "also an input" in fake.says(name, dict(base, y=base["x"]))
