"""What a text tower that is served token by token asks of the library, as cases that can
be timed: rotary positions, their form that fills a paged K/V cache, attention of new
tokens over that cache, and linear layers with 4-bit weights.

  rotary  q and k of grouped heads rotated by their tokens' positions.
  append  a layer's new tokens: q rotated, k rotated and v copied into the cache's pages.
  attend  a layer's new tokens attend over the cache: one token of each sequence (a step
          of generation), a chunk of one long prompt, or both in one batch.
  linear  y = x W^T + bias with 4-bit weights, a scale (and a zero point) per group.

layers: how many layers' calls a chain holds, each with a cache or weights of its own, as a
host program enqueues them.  Head counts are the text tower's (32 on 8) and others the
library's benchmarks have; lengths run from one token to the longest contexts.
"""
import functools
import math

import numpy as np
import torch

own = False

GOLDEN = 0.6180339887498949


def listed():
    return [
        # The prompt of one image through the text tower: the smallest call.
        _rotary("rotary-412", tokens=412, first=0),
        # A long document's chunk, half of every head rotated, neighbouring pairs, stretched
        # positions far out.
        _rotary("rotary-part-16384", tokens=16384, first=100000, rotary_dim=64, half=False,
                scaling="parts"),
        # One generated token of each of 64 sequences, four layers to a chain.
        _append("append-64", batch=64, new=1, context=2048, page_rows=16, layers=4),
        # A prompt's first chunk into an empty cache, with rows behind it that are padding.
        _append("append-4096", batch=1, new=4096, context=4096, page_rows=64, tail=37),
        # One token of one sequence: launch latency.
        _attend("attend-1-of-2000", batch=1, context=2000, page_rows=16),
        # A step of 64 sequences of unequal lengths.
        _attend("attend-64-of-4096", batch=64, context=4096, page_rows=16, layers=2),
        # One sequence with a very long context: all SMs on one row.
        _attend("attend-1-of-131072", batch=1, context=131072, page_rows=64, layers=2),
        # A chunk of a long prompt over what the earlier chunks left.
        _attend("attend-chunk-2048", batch=1, new=2048, context=16384, page_rows=64),
        # Twenty sequences that generate and four prompts that begin, in one batch.
        _attend("attend-mixed", batch=24, short=20, new=300, context=4100, page_rows=16, tail=11),
        # The q, k, v projection of one token, eight layers to a chain.
        _linear("linear-1", rows=1, inputs=4096, outputs=6144, layers=8),
        # A step of 13 sequences through a wide layer, zero points, small groups.
        _linear("linear-13-zeros", rows=13, inputs=4096, outputs=12288, group=32, zeros=True, layers=2),
        # A prompt's rows, bias.
        _linear("linear-412", rows=412, inputs=4096, outputs=4096, bias=True),
    ]


def _case(name, op, **given):
    case = dict(given, op=op)
    if name:
        case["name"] = name
    return case


def _rotary(name, tokens, first, heads=32, kv_heads=8, head_dim=128, rotary_dim=128, half=True,
            scaling="none"):
    return _case(name, "rotary", tokens=tokens, first=first, heads=heads, kv_heads=kv_heads,
                 head_dim=head_dim, rotary_dim=rotary_dim, half=half, scaling=scaling)


def _append(name, batch, new, context, page_rows, heads=32, kv_heads=8, rotary_dim=128, half=True,
            scaling="none", layers=1, tail=0, short=0):
    return _case(name, "append", batch=batch, short=short, new=new, context=context,
                 page_rows=page_rows, heads=heads, kv_heads=kv_heads, head_dim=128,
                 rotary_dim=rotary_dim, half=half, scaling=scaling, layers=layers, tail=tail)


def _attend(name, batch, context, page_rows, new=1, short=0, heads=32, kv_heads=8, layers=1, tail=0):
    return _case(name, "attend", batch=batch, short=short, new=new, context=context,
                 page_rows=page_rows, heads=heads, kv_heads=kv_heads, layers=layers, tail=tail)


def _linear(name, rows, inputs, outputs, group=128, zeros=False, bias=False, layers=1):
    return _case(name, "linear", rows=rows, inputs=inputs, outputs=outputs, group=group, zeros=zeros,
                 bias=bias, layers=layers)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _spread(rng, lo, hi):
    """A whole number, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "linear", "linear"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (24, 24), (16, 8), (28, 4), (8, 1)])
    half, scaling = rng.random() < 0.6, rng.choice(["none", "linear", "parts"])
    page_rows = rng.choice([16, 32, 64, 128, 256])
    layers, tail = rng.choice([1, 2, 4]), rng.choice([0, 0, rng.randint(1, 60)])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
        return _rotary("", _spread(rng, 1, 16384), rng.choice([0, rng.randint(1, 1 << 20)]), heads,
                       kv_heads, head_dim, rotary_dim, half, scaling)
    if op == "linear":
        group = rng.choice([32, 64, 128])
        inputs = group * max(1, _spread(rng, 512, 12288) // group)
        return _linear("", _spread(rng, 1, 512), inputs, _spread(rng, 100, 12288), group,
                       rng.random() < 0.5, rng.random() < 0.3, layers)
    kind = rng.choice(["step", "step", "chunk", "mixed"])
    batch = {"step": _spread(rng, 1, 128), "chunk": rng.choice([1, 1, 2, 3]), "mixed": rng.randint(3, 24)}[kind]
    new = 1 if kind == "step" else _spread(rng, 2, 4096 if kind == "chunk" else 512)
    short = rng.randint(1, batch - 1) if kind == "mixed" else 0
    context = new + _spread(rng, 1, 131072 if kind == "step" and batch < 9 else 16384)
    if op == "append":
        context = min(context, 8192)
        return _append("", batch, min(new, context), context, page_rows, heads, kv_heads,
                       rng.choice([128, 128, 64, 32]), half, scaling, layers, tail, short)
    return _attend("", batch, context, page_rows, new, short, heads, kv_heads,
                   1 if kind == "chunk" else min(layers, 2), tail)


# ---- what a pass cannot do without ------------------------------------------


def _lengths(c):
    """New tokens and cache lengths (the new tokens among them) of a batch's sequences: the
    first `short` have one new token, the others up to `new`; unequal unless there is one."""
    b = np.arange(c["batch"])
    part = np.where(b > 0, 1.0 - 0.75 * ((b * GOLDEN) % 1.0), 1.0)
    new = np.where(b < c["short"], 1, np.maximum(1, (c["new"] * part[::-1]).astype(np.int64)))
    old = np.maximum(0, ((c["context"] - c["new"]) * part).astype(np.int64))
    return new, old + new


def work(case):
    """Bytes and operations of one pass: every input and output once; of a cache the rows
    that are seen or written; 2 operations per multiply-add of visible scores, of P V and of
    products, 6 per rotated pair."""
    c = case
    if c["op"] == "linear":
        weights = c["inputs"] * c["outputs"] // 2
        groups = c["outputs"] * (c["inputs"] // c["group"]) * 2 * (2 if c["zeros"] else 1)
        ends = 2 * c["rows"] * (c["inputs"] + c["outputs"]) + (2 * c["outputs"] if c["bias"] else 0)
        return {"bytes": float(c["layers"] * (weights + groups + ends)),
                "flops": 2.0 * c["layers"] * c["rows"] * c["inputs"] * c["outputs"]}
    if c["op"] == "rotary":
        each = c["tokens"] * (c["heads"] + c["kv_heads"])
        return {"bytes": float(each * c["head_dim"] * 4 + c["tokens"] * 4),
                "flops": 3.0 * each * c["rotary_dim"]}
    new, length = _lengths(c)
    n = int(new.sum())
    if c["op"] == "append":
        moved = n * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"] * 4
        return {"bytes": float(c["layers"] * moved),
                "flops": 3.0 * c["layers"] * n * (c["heads"] + c["kv_heads"]) * c["rotary_dim"]}
    visible = float((new * (length - new) + new * (new + 1) // 2).sum())
    moved = n * c["heads"] * 512 + int(length.sum()) * c["kv_heads"] * 512
    return {"bytes": float(c["layers"] * moved), "flops": 512.0 * c["layers"] * c["heads"] * visible}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


# ---- inputs -------------------------------------------------------------------


class _State:
    pass


def _frequencies(c):
    """Frequencies of the rotated pairs and the factor on cosine and sine: none; linear
    (positions over 8); by parts (fast pairs as they are, slow ones over 8, a ramp between
    32 and 1 turns within 8192 positions)."""
    pairs = c["rotary_dim"] // 2
    f = 1e6 ** (-np.arange(pairs) / pairs)
    if c["scaling"] == "linear":
        return (f / 8).astype(np.float32), 1.0
    if c["scaling"] == "parts":
        turns = 8192 * f / (2 * np.pi)
        keep = np.clip((turns - 1) / (32 - 1), 0, 1)
        return (f * keep + f / 8 * (1 - keep)).astype(np.float32), 0.1 * math.log(8) + 1.0
    return f.astype(np.float32), 1.0


def prepare(case, seed):
    c, s = case, _State()
    s.case = c
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        return t.normal_(mean, std, generator=gen)

    if c["op"] == "linear":
        _prepare_linear(s, c, gen, normal)
    elif c["op"] == "rotary":
        s.frequencies, s.magnitude = _frequencies(c)
        s.frequencies = torch.from_numpy(s.frequencies).cuda()
        at = torch.arange(c["tokens"], device="cuda", dtype=torch.int64)
        # (prompts packed one behind the other: positions start anew)
        s.positions = (at % max(1, c["tokens"] * 5 // 8) + c["first"]).to(torch.int32)
        s.q = normal(c["tokens"], c["heads"], c["head_dim"])
        s.k = normal(c["tokens"], c["kv_heads"], c["head_dim"])
    else:
        _prepare_cache(s, c, gen, normal)
    torch.cuda.synchronize()
    if own:
        _bind(s, c)
    return s


def _prepare_linear(s, c, gen, normal):
    """Weights as a checkpoint has them: eight 4-bit columns to a word, the lowest bits
    first; values near 0 are the most frequent."""
    layers, outs, ins = c["layers"], c["outputs"], c["inputs"]
    shape = (layers, outs, ins // 8)
    s.weight = torch.zeros(shape, dtype=torch.int32, device="cuda")
    for i in range(8):
        q = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(8, 2.7, generator=gen)
        s.weight |= q.round_().clamp_(0, 15).to(torch.int32) << (4 * i)
    groups = (layers, outs, ins // c["group"])
    s.scales = (normal(*groups).abs() * 0.25 + 0.75) * (0.4 / math.sqrt(ins))
    s.zeros = normal(*groups, std=0.7, mean=7.8) if c["zeros"] else None
    s.bias = normal(layers, outs, std=0.1) if c["bias"] else None
    s.x = normal(layers, c["rows"], ins)


def _prepare_cache(s, c, gen, normal):
    new, length = _lengths(c)
    rows = c["page_rows"]
    pages = -(-length // rows)
    width, count = int(pages.max()) + 1, int(pages.sum()) + 3
    order = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((c["batch"], width), dtype=torch.int32, device="cuda")
    first = np.concatenate([[0], np.cumsum(pages)])
    for b in range(c["batch"]):
        table[b, :pages[b]] = order[first[b]:first[b + 1]]
    s.page_table, s.width = table, width
    s.total = int(new.sum())
    s.tokens = s.total + c["tail"]
    s.most_new = int(new.max())
    s.token_start = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    s.cache_len = torch.from_numpy(length.astype(np.int32)).cuda()
    layers, kv, dim = c["layers"], c["kv_heads"], 128
    s.key_pages = normal(layers, count, rows, kv, dim)
    s.value_pages = normal(layers, count, rows, kv, dim)
    s.q = normal(layers, s.tokens, c["heads"], dim)
    s.out = torch.zeros_like(s.q)
    if c["op"] == "append":
        s.frequencies, s.magnitude = _frequencies(c)
        s.frequencies = torch.from_numpy(s.frequencies).cuda()
        s.k = normal(layers, s.tokens, kv, dim)
        s.v = normal(layers, s.tokens, kv, dim)


# ---- a pass ----------------------------------------------------------------------


def run(s):
    if own:
        return _chain(s)
    return {"linear": _plain_linear, "rotary": _plain_rotary, "append": _plain_append,
            "attend": _plain_attend}[s.case["op"]](s)


def _rotated(x, positions, frequencies, magnitude, half):
    """x [..., tokens, heads, dim]; angles in 64 bits, the rotation in 32."""
    pairs = frequencies.numel()
    angle = positions.double()[:, None] * frequencies.double()
    cos = (angle.cos() * magnitude).float()[:, None, :]
    sin = (angle.sin() * magnitude).float()[:, None, :]
    x = x.float()
    part, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if half:
        a, b = part[..., :pairs], part[..., pairs:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(torch.bfloat16)


def _plain_rotary(s):
    half = s.case["half"]
    return {"q": _rotated(s.q, s.positions, s.frequencies, s.magnitude, half),
            "k": _rotated(s.k, s.positions, s.frequencies, s.magnitude, half)}


def _plain_append(s):
    n, half, rows = s.total, s.case["half"], s.case["page_rows"]
    token = torch.arange(n, device="cuda", dtype=torch.int32)
    sequence = torch.searchsorted(s.token_start[1:], token, right=True)
    row = s.cache_len[sequence] - s.token_start[sequence + 1] + token
    at = s.page_table[sequence, (row // rows).long()].long() * rows + row % rows
    out = s.out
    out[:, :n] = _rotated(s.q[:, :n], row, s.frequencies, s.magnitude, half)
    s.key_pages.flatten(1, 2)[:, at] = _rotated(s.k[:, :n], row, s.frequencies, s.magnitude, half)
    s.value_pages.flatten(1, 2)[:, at] = s.v[:, :n]
    return {"q": list(out.unbind(0)), "keys": list(s.key_pages.unbind(0)),
            "values": list(s.value_pages.unbind(0))}


def _plain_attend(s):
    c = s.case
    layers, batch, kv, rows = c["layers"], c["batch"], c["kv_heads"], c["page_rows"]
    share = c["heads"] // kv
    new, length = s.token_start[1:] - s.token_start[:-1], s.cache_len
    most = (s.width - 1) * rows
    key = torch.arange(most, device="cuda")
    at = s.page_table[:, :s.width - 1].long()[:, key // rows] * rows + key % rows
    i = torch.arange(s.most_new, device="cuda")
    token = (s.token_start[:-1, None] + i).clamp_(max=s.tokens - 1)
    q = s.q[:, token].float().view(layers, batch, s.most_new, kv, share, 128)
    q = q.permute(0, 1, 3, 2, 4, 5).reshape(layers, batch, kv, s.most_new * share, 128)
    keys = s.key_pages.flatten(1, 2)[:, at].float().permute(0, 1, 3, 4, 2)
    scores = torch.matmul(q, keys).mul_(128 ** -0.5).view(layers, batch, kv, s.most_new, share, most)
    seen = key < (length - new)[:, None, None] + i[:, None] + 1
    scores.masked_fill_(~seen[None, :, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    values = s.value_pages.flatten(1, 2)[:, at].float().permute(0, 1, 3, 2, 4)
    o = torch.matmul(scores.flatten(3, 4), values).view(layers, batch, kv, s.most_new, share, 128)
    o = (o / total).permute(0, 1, 3, 2, 4, 5).reshape(layers, batch, s.most_new, c["heads"], 128)
    out, real = s.out, i < new[:, None]
    out[:, token[real]] = o[:, real].to(torch.bfloat16)
    return list(out.unbind(0))


def _unpacked(weight):
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    return ((weight[..., None] >> shift) & 15).flatten(-2)


def _plain_linear(s):
    group = s.case["group"]
    q = _unpacked(s.weight).float().unflatten(-1, (-1, group))
    q = q - (8.0 if s.zeros is None else s.zeros.float()[..., None])
    w = (q * s.scales.float()[..., None]).flatten(-2)
    y = torch.matmul(s.x.float(), w.transpose(-1, -2))
    if s.bias is not None:
        y = y + s.bias.float()[:, None, :]
    return list(y.to(torch.bfloat16).unbind(0))


# ---- the library's calls -----------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _gpu():
    """The program's one context."""
    from qwen_metal_b200 import abi
    return abi.Gpu()


class _Tensor:
    """A tensor of the library with the values of a torch tensor, freed with its last user
    (a view of it included)."""

    def __init__(self, t):
        gpu, n = _gpu(), t.numel()
        if t.dtype == torch.int32:
            self.handle = gpu.u32(t.cpu().numpy())
        elif t.dtype == torch.float32:
            self.handle = gpu.f32(t.cpu().numpy())
        else:
            self.handle = gpu.new_bf16(n)
            self.__cuda_array_interface__ = {
                "shape": (n,), "typestr": "<i2", "version": 3, "strides": None,
                "data": (gpu.lib.qw_gpu_tensor_device_ptr(self.handle), False)}
            torch.cuda.synchronize()  # the library clears a new tensor on its own stream
            self.view(*t.shape).copy_(t)

    def __del__(self):
        gpu = _gpu()
        if gpu.handle:
            gpu.free(self.handle)

    def view(self, *shape):
        return torch.as_tensor(self, device="cuda").view(torch.bfloat16).view(*shape)


def _call(s, name, *arguments):
    """Bind one call of the C ABI, its arguments converted once as a C host has them."""
    fn = getattr(_gpu().lib, name)
    bound = [_gpu().handle] + [a.handle if isinstance(a, _Tensor) else a for a in arguments]
    bound = [a if a is None or isinstance(a, kind) else kind(a) for kind, a in zip(fn.argtypes, bound)]
    s.calls.append(functools.partial(fn, *bound))
    s.kept.extend(a for a in arguments if isinstance(a, _Tensor))


def _bind(s, c):
    """The library's tensors of a state, which take the place of torch's, and its calls."""
    s.calls, s.kept = [], []
    if c["op"] == "linear":
        outs = []
        for n in range(c["layers"]):
            y = _Tensor(torch.zeros((c["rows"], c["outputs"]), dtype=torch.bfloat16, device="cuda"))
            _call(s, "qw_gpu_linear_w4_bf16", y, _Tensor(s.x[n]), _Tensor(s.weight[n]),
                  _Tensor(s.scales[n]), None if s.zeros is None else _Tensor(s.zeros[n]),
                  None if s.bias is None else _Tensor(s.bias[n]), c["rows"], c["inputs"],
                  c["outputs"], c["group"])
            outs.append(y.view(c["rows"], c["outputs"]))
        s.outputs = outs
        s.x = s.weight = s.scales = s.zeros = s.bias = None
    elif c["op"] == "rotary":
        q, k = _Tensor(torch.zeros_like(s.q)), _Tensor(torch.zeros_like(s.k))
        _call(s, "qw_gpu_rotary_bf16", q, k, _Tensor(s.q), _Tensor(s.k), _Tensor(s.positions),
              _Tensor(s.frequencies), c["tokens"], c["heads"], c["kv_heads"], c["head_dim"],
              c["rotary_dim"], int(c["half"]), s.magnitude)
        s.outputs = {"q": q.view(*s.q.shape), "k": k.view(*s.k.shape)}
        s.q = s.k = None
    else:
        _bind_cache(s, c)
    torch.cuda.synchronize()


def _bind_cache(s, c):
    table, start, length = _Tensor(s.page_table), _Tensor(s.token_start), _Tensor(s.cache_len)
    append = c["op"] == "append"
    frequencies = _Tensor(s.frequencies) if append else None
    outs, keys, values = [], [], []
    for n in range(c["layers"]):
        out, q = _Tensor(s.out[n]), _Tensor(s.q[n])
        kp, vp = _Tensor(s.key_pages[n]), _Tensor(s.value_pages[n])
        if append:
            _call(s, "qw_gpu_rotary_append_bf16", out, kp, vp, q, _Tensor(s.k[n]), _Tensor(s.v[n]),
                  None, frequencies, table, start, length, c["batch"], s.tokens, s.width,
                  c["page_rows"], c["heads"], c["kv_heads"], 128, c["rotary_dim"], int(c["half"]),
                  s.magnitude)
            keys.append(kp.view(*s.key_pages[n].shape))
            values.append(vp.view(*s.value_pages[n].shape))
        else:
            _call(s, "qw_gpu_paged_attention_bf16", out, q, kp, vp, table, start, length, c["batch"],
                  s.tokens, s.most_new, s.width, c["page_rows"], c["heads"], c["kv_heads"], 128,
                  128 ** -0.5)
        outs.append(out.view(*s.out[n].shape))
    s.outputs = {"q": outs, "keys": keys, "values": values} if append else outs
    s.q = s.out = s.key_pages = s.value_pages = s.k = s.v = None


def _chain(s):
    gpu = _gpu()
    gpu.begin()
    if not all([call() for call in s.calls]):
        raise RuntimeError(gpu.error())
    gpu.submit()
    return s.outputs


# ---- the definitions in 64 bits ------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "linear":
        return [_exact_linear(s, c, n) for n in range(c["layers"])]
    if c["op"] == "rotary":
        return {"q": _exact_turn(s.q, s.positions, s), "k": _exact_turn(s.k, s.positions, s)}
    start, length = s.token_start.tolist(), s.cache_len.tolist()
    outs, keys, values = [], [], []
    for n in range(c["layers"]):
        out = torch.zeros(s.q[n].shape, dtype=torch.float64, device="cuda")
        kp, vp = s.key_pages[n].double(), s.value_pages[n].double()
        for b in range(c["batch"]):
            lo, hi = start[b], start[b + 1]
            rows = torch.arange(length[b], device="cuda")
            page = s.page_table[b].long()[torch.div(rows, c["page_rows"], rounding_mode="floor")]
            if c["op"] == "append":
                new = rows[length[b] - (hi - lo):]
                out[lo:hi] = _exact_turn(s.q[n, lo:hi], new, s)
                kp[page[new], new % c["page_rows"]] = _exact_turn(s.k[n, lo:hi], new, s)
                vp[page[new], new % c["page_rows"]] = s.v[n, lo:hi].double()
            else:
                k, v = kp[page, rows % c["page_rows"]], vp[page, rows % c["page_rows"]]
                out[lo:hi] = _exact_softmax(s.q[n, lo:hi].double(), k, v, c)
        outs.append(out)
        keys.append(kp)
        values.append(vp)
    return {"q": outs, "keys": keys, "values": values} if c["op"] == "append" else outs


def _exact_linear(s, c, n):
    w = torch.empty((c["outputs"], c["inputs"]), dtype=torch.float64, device="cuda")
    for i in range(8):
        w[:, i::8] = torch.bitwise_and(torch.div(
            s.weight[n].long() & 0xffffffff, 16 ** i, rounding_mode="floor"), 15).double()
    for g in range(c["inputs"] // c["group"]):
        columns = w[:, g * c["group"]:(g + 1) * c["group"]]
        columns -= 8 if s.zeros is None else s.zeros[n, :, g:g + 1].double()
        columns *= s.scales[n, :, g:g + 1].double()
    y = s.x[n].double() @ w.t()
    return y if s.bias is None else y + s.bias[n].double()


def _exact_turn(x, positions, s):
    """The rotation as a product of complex numbers."""
    pairs = s.frequencies.numel()
    turn = torch.polar(torch.full((1, pairs), float(s.magnitude), dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * s.frequencies.double()[None])
    out = x.double()
    first = slice(0, pairs) if s.case["half"] else slice(0, 2 * pairs, 2)
    second = slice(pairs, 2 * pairs) if s.case["half"] else slice(1, 2 * pairs, 2)
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn[:, None]
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_softmax(q, k, v, c):
    """Token i of n sees the keys up to its own, some tokens and one head at a time."""
    n, total, share = q.shape[0], k.shape[0], c["heads"] // c["kv_heads"]
    out = torch.empty_like(q)
    step = max(1, (1 << 27) // total)
    for h in range(c["heads"]):
        for at in range(0, n, step):
            score = q[at:at + step, h] @ k[:, h // share].t() / math.sqrt(128.0)
            own_row = torch.arange(total - n + at, total - n + at + score.shape[0], device="cuda")
            score[torch.arange(total, device="cuda")[None] > own_row[:, None]] = -math.inf
            out[at:at + step, h] = torch.softmax(score, -1) @ v[:, h // share]
    return out
