"""Plain 64-bit forms of the text tower's ops (rotary positions, the paged cache, attention over
it, 4-bit linear layers), and how far a bf16 result may be from them."""
import numpy as np

from qwen_metal_b200 import abi

HALF_STEP = 2.0 ** -8  # of bf16, relative


def random_bf16(rng, *shape, std=1.0):
    return abi.f32_to_bf16((rng.standard_normal(shape) * std).astype(np.float32))


def wide(bits):
    return abi.bf16_to_f32(bits).astype(np.float64)


def rotate(x, positions, frequencies, magnitude, halves):
    """x [tokens, heads, dim] float64 -> the rotated x and the sum of magnitudes each element is made of."""
    pairs = len(frequencies)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    cos, sin = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    first = np.arange(pairs) if halves else 2 * np.arange(pairs)
    second = first + pairs if halves else first + 1
    out, size = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * abs(magnitude)
    return out, size


def check_rotated(got_bits, exact, size):
    # One rounding to bf16; cosine and sine are within 2^-21 of a turn's (the reduced angle is rounded
    # to 24 bits, sincospi is good to 2 units in the last place), product and sum round three times.
    err = np.abs(wide(got_bits) - exact)
    bound = HALF_STEP * np.abs(exact) + 2.0 ** -20 * size
    assert (err <= bound).all(), float((err - bound).max())


class Cache:
    """A paged cache with sequences of `new` new tokens and `length` rows each."""

    def __init__(self, rng, new, length, page_rows, kv_heads, dim=128, tail=0, spare=2, stale=None):
        self.new, self.length = np.asarray(new), np.asarray(length)
        self.batch, self.page_rows, self.kv_heads, self.dim = len(new), page_rows, kv_heads, dim
        pages = -(-self.length // page_rows)
        self.width = max(1, int(pages.max()) + 1)
        self.pages = int(pages.sum()) + spare
        order = rng.permutation(self.pages)
        # (entries past a sequence's last page are not read: they name no page at all)
        self.table = np.full((self.batch, self.width), 0xffffffff, np.uint32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.uint32)
        self.tokens = max(1, int(self.start[-1]) + tail)
        shape = (self.pages, page_rows, kv_heads, dim)
        self.k, self.v = random_bf16(rng, *shape), random_bf16(rng, *shape)
        if stale is not None:  # what rows outside the sequences hold
            used = np.zeros((self.pages, page_rows), bool)
            for b in range(self.batch):
                used[self.rows(b)] = True
            self.k[~used], self.v[~used] = stale, stale

    def rows(self, b, count=None):
        r = np.arange(self.length[b] if count is None else count)
        return self.table[b, r // self.page_rows].astype(np.int64), r % self.page_rows

    def upload(self, gpu):
        return (gpu.bf16(self.k), gpu.bf16(self.v), gpu.u32(self.table), gpu.u32(self.start),
                gpu.u32(self.length))


def attention(cache, q, scale):
    """[tokens, heads, 128] float64 results, the sums of p |v|, and which rows are a sequence's."""
    heads = q.shape[1]
    share = heads // cache.kv_heads
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    real = np.zeros(q.shape[0], bool)
    k, v = wide(cache.k), wide(cache.v)
    for b in range(cache.batch):
        lo, hi = int(cache.start[b]), int(cache.start[b + 1])
        real[lo:hi] = True
        keys, values = k[cache.rows(b)], v[cache.rows(b)]
        for i in range(hi - lo):
            seen = max(0, int(cache.length[b]) - (hi - lo) + i + 1)
            if not seen:
                continue
            for h in range(heads):
                s = keys[:seen, h // share] @ wide(q[lo + i, h]) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[lo + i, h] = p @ values[:seen, h // share]
                size[lo + i, h] = p @ np.abs(values[:seen, h // share])
    return out, size, real


def check_attention(got_bits, exact, size):
    # The result's rounding to bf16, and each weight's on its way into the product with V; scores
    # (fp32 sums of 128 products of magnitude up to some tens) and exponentials add less than 2^-12.
    err = np.abs(wide(got_bits) - exact)
    bound = HALF_STEP * np.abs(exact) + (HALF_STEP + 2.0 ** -12) * size
    assert np.isfinite(wide(got_bits)).all()
    assert (err <= bound).all(), float((err - bound).max())


def unpack(words):
    """[n, k / 8] words -> [n, k] whole numbers 0 .. 15."""
    return ((words[..., None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).reshape(words.shape[0], -1)


def linear_w4(x_bits, words, scales, zeros, bias, group):
    """y in float64, the sum of magnitudes it is made of, and those that roundings of weights go by."""
    q = unpack(words).astype(np.float64)
    z = np.full(scales.shape, 8.0) if zeros is None else wide(zeros)
    s, z = np.repeat(wide(scales), group, 1), np.repeat(z, group, 1)
    x = wide(x_bits)
    y = x @ (s * (q - z)).T
    size = np.abs(x) @ (np.abs(s) * (np.abs(q - 8) + np.abs(z - 8))).T
    # with many rows a weight is rounded to bf16, and q - z before it where z is not whole
    rounded = np.abs(x) @ (np.abs(s * (q - z)) * np.where(z == np.rint(z), 1.0, 2.0)).T
    if bias is not None:
        y, size = y + wide(bias), size + np.abs(wide(bias))
    return y, size, rounded


def check_linear(got_bits, y, size, rounded):
    # One rounding to bf16; sums of a group's 128 products (at most 4096 in one group) and of the groups
    # in fp32, each addition within 2^-23 of its operands: well below 2^-14 of the magnitudes for groups
    # of up to 128 columns.  With more than 16 rows the weights are rounded to bf16, half a step each.
    err = np.abs(wide(got_bits) - y)
    bound = HALF_STEP * np.abs(y) + 2.0 ** -14 * size
    if got_bits.shape[0] > 16:
        bound = bound + HALF_STEP * rounded
    assert (err <= bound).all(), float((err - bound).max())
