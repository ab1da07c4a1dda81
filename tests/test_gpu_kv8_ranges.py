"""The 8-bit cache's attention over long rows and uneven weights, against 64 bits.

What ``test_gpu_kv8.py`` says of the errors holds; here the sums and the floor of small weights are counted as the
kernels make them, so that a bound is a small part of the result also where one key has most of a long row's mass:

* sums: 128 products of a tile in one accumulator, then a multiply-add with a power (2^x itself is off by 2^-22) per
  tile and per part that is joined, each off by 2^-23 at most (a sum that is cut off rather than rounded):
  ``(128 + 3 tiles + 256) 2^-23`` of sum_j w_j |v_j|, for the row sum the same;
* one-token kernel: a weight (times the scale of V) is two e4m3 numbers hi + lo / 32, taken times 128 against the largest
  of its tile of 128 keys, or 2^-12 of the row's largest: off by 2^-8 of itself or by 2^-10 / 32 of 128, 2^-22 of that;
* prefill kernel: a weight (times the scale of V) is an fp16 number, 2^-11, or 2^-25 where the weights of 64 keys sum to
  2^7 at least (one of them 2^7 when the reference is taken, all of them after it was raised): 2^-32 of the row's sum;
* fp32 kernel: nothing of the kind, bf16 inputs or not.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8 as oracle
from qwenquest_b200.kv8 import KV8Cache
from tests.test_gpu_kv8 import GEOMETRIES, _Batch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TILE = 128


def _dev(x, dtype=torch.int64):
    return torch.tensor(np.asarray(x), dtype=dtype, device=DEV)


def _check(got, q, k, v, v_scale, scaling, form):
    """One query ``q`` [heads, dim] against ``k``, ``v`` float64 [n, kv, dim]; ``form``: decode, extend or fp32."""
    heads, dim = q.shape
    n, kv, _ = k.shape
    tiles = -(-n // TILE)
    q64 = q.double().numpy()
    got = got.double().cpu().numpy().reshape(heads, dim)
    step = torch.finfo(q.dtype).eps / 2
    for h in range(heads):
        kh, vh, s = k[:, h // (heads // kv)], v[:, h // (heads // kv)], v_scale[:, h // (heads // kv)].astype(np.float64)
        x = kh @ q64[h] * scaling
        w = np.exp(x - x.max())
        w /= w.sum()
        out, size = w @ vh, w @ np.abs(vh)
        spread = (np.abs(kh) @ np.abs(q64[h])).max() * scaling
        rel = 2 * (dim + 8) * 2.0 ** -24 * spread + 2 * 2.0 ** -22 + 2 * (TILE + 3 * tiles + 256) * 2.0 ** -23
        err = rel * size
        codes = np.abs(vh) / s[:, None]
        if form == "decode":
            pad = tiles * TILE - n
            top = np.maximum(np.pad(w * s, (0, pad)).reshape(tiles, TILE).max(1), 2.0 ** -12 * (w * s).max())
            err = err + 2.0 ** -8 * size + 2.0 ** -22 * top @ np.pad(codes, ((0, pad), (0, 0))).reshape(tiles, TILE, dim).sum(1)
        elif form == "extend":
            err = err + 2.0 ** -11 * size + 2.0 ** -32 * (w * s).sum() * codes.sum(0)
        tol = step * np.abs(out) + (1 + step) * err + 1e-37
        off = np.abs(got[h] - out)
        assert (off <= tol).all(), (h, float((off / np.abs(out)).max()), float((off / tol).max()), float((tol / np.abs(out)).max()))


class _Sinks:
    """One request of ``n`` tokens over scattered blocks: keys of even scores but for a few positions that hold most of
    a head's mass, 50 to 99.9 % of it, with small values; the other values are between 0.5 and 1.5, so that what the
    tail loses is the result's."""

    MASSES = (0.5, 0.9, 0.95, 0.98, 0.99, 0.995, 0.998, 0.999)

    def __init__(self, n, sinks, seed, dim=128, block=64, spread=0.3, dtype=torch.bfloat16):
        rng = np.random.default_rng(seed)
        pages = -(-n // block)
        shape = (pages + 1, 1, block, dim)
        heads = len(self.MASSES)
        scale = np.float32(2.0 ** -7)
        self.order = rng.permutation(pages + 1)[:pages]
        pos = np.arange(n)
        self.slots = self.order[pos // block] * block + pos % block
        at = (self.slots // block, 0, self.slots % block)
        k = np.zeros(shape, dtype=np.uint8)
        v = np.zeros(shape, dtype=np.uint8)
        kx = rng.standard_normal((n, dim)) * 60
        kx[:, 0] = 0
        kx[sinks] = 0
        kx[sinks, 0] = 448
        vx = (0.5 + rng.random((n, dim))) * 128
        vx[sinks] = 2.0 ** -3 * rng.random((len(sinks), dim))
        k[at] = oracle.to_e4m3(kx)
        v[at] = oracle.to_e4m3(vx)
        self.scaling = dim ** -0.5
        q = rng.standard_normal((heads, dim)) * spread
        for h, m in enumerate(self.MASSES):  # the sinks' score against the mean weight of the tail, e^0.06 or so
            q[h, 0] = np.log(n * m / (1 - m) / len(sinks)) / (self.scaling * 448 * scale)
        self.q = torch.from_numpy(q[None]).to(dtype)
        scales = np.full(shape[:2], scale, dtype=np.float32)
        self.cache = KV8Cache.from_tensors(
            [torch.from_numpy(k).to(DEV).view(torch.float8_e4m3fn)], [torch.from_numpy(v).to(DEV).view(torch.float8_e4m3fn)],
            [torch.from_numpy(scales).to(DEV)], [torch.from_numpy(scales).to(DEV)])
        self.n, self.block = n, block
        self.k, self.v = oracle.rows(k, scales, self.slots), oracle.rows(v, scales, self.slots)
        self.v_scale = np.full((n, 1), scale, dtype=np.float32)
        self.table = _dev(self.order[None], torch.int32)

    def check(self, got, form, seen=None, q=None):
        seen = np.arange(self.n) if seen is None else seen
        _check(got, self.q[0] if q is None else q, self.k[seen], self.v[seen], self.v_scale[seen], self.scaling, form)


@pytest.mark.parametrize(("n", "sinks"), [
    (32768, [0]), (131072, [0]), (131071, [70000]), (131072, [0, 1, 131071]), (8192, [0]), (2049, [2048]), (300, [5])])
def test_decode_behind_a_key_with_most_of_the_mass(n, sinks):
    """A lone request (a cluster, or all shares), and as many as fill the GPU, a whole one to each CTA."""
    s = _Sinks(n, sinks, seed=n + len(sinks))
    lone = s.cache.decode_attention(0, s.q.to(DEV), s.table, [0], [n], s.scaling)
    many = 300
    full = s.cache.decode_attention(0, s.q.to(DEV).expand(many, -1, -1), s.table, [0] * many, [n] * many, s.scaling)
    s.cache.synchronize()
    s.check(lone[0], "decode")
    s.check(full[0], "decode")
    s.check(full[many // 2 + 1], "decode")
    s.check(full[many - 1], "decode")


@pytest.mark.parametrize(("n", "top"), [(32768, 32768), (40000, 4096)])
def test_selected_rows_behind_a_key_with_most_of_the_mass(n, top):
    """All rows in another order, and a selection of pages, with the heavy key among them."""
    s = _Sinks(n, [0], seed=n + top)
    rng = np.random.default_rng(top)
    pages = np.concatenate([[0], 1 + rng.permutation(n // s.block - 1)])[:top // s.block]
    pos = (pages[:, None] * s.block + np.arange(s.block)).ravel()
    rows = _dev(s.slots[pos], torch.int32)
    lone = s.cache.sparse_decode_attention(0, s.q.to(DEV), rows[None], [top], s.scaling)
    many = 300
    full = s.cache.sparse_decode_attention(0, s.q.to(DEV).expand(many, -1, -1), rows.expand(many, -1).contiguous(),
                                           [top] * many, s.scaling)
    s.cache.synchronize()
    for got in (lone[0], full[0], full[many - 1]):
        s.check(got, "decode", seen=pos)


@pytest.mark.parametrize(("n", "new", "sinks"), [
    (8192, 5000, [0]), (32768, 5000, [0]), (131072, 5000, [0]), (131072, 40, [0]), (32768, 5000, [20000]),
    (8192, 8192, [0, 130])])
def test_extend_behind_a_key_with_most_of_the_mass(n, new, sinks):
    """Enough query rows that a thread block takes all keys of its own, and so few that they are cut."""
    s = _Sinks(n, sinks, seed=n + new)
    q = s.q.expand(new, -1, -1).contiguous()
    out = s.cache.extend_attention(0, q.to(DEV), s.table, [0], [n], [n - new], [0], s.scaling)
    s.cache.synchronize()
    for t in (0, 31, new // 2, new - 1):
        s.check(out[t], "extend", seen=np.arange(n - new + t + 1))


@pytest.mark.parametrize(("heads", "kv"), [(8, 1), (32, 4), (16, 1)])
def test_a_lone_request_of_131072_keys(heads, kv):
    """A pair cut over all shares and joined from their records; keys and values of either sign, uneven scores."""
    n, dim, block = 131072 + 77, 128, 64
    rng = np.random.default_rng(heads)
    pages = -(-n // block)
    codes = [oracle.to_e4m3(rng.standard_normal((pages, kv, block, dim)) * 90 + 60) for _ in range(2)]
    scales = [np.ldexp(1.0, rng.integers(-9, -5, (pages, kv))).astype(np.float32) for _ in range(2)]
    order = rng.permutation(pages)
    slots = order[np.arange(n) // block] * block + np.arange(n) % block
    cache = KV8Cache.from_tensors(*([torch.from_numpy(c).to(DEV).view(torch.float8_e4m3fn)] for c in codes),
                                  *([torch.from_numpy(x).to(DEV)] for x in scales))
    q = torch.from_numpy(rng.standard_normal((1, heads, dim))).to(torch.bfloat16)
    out = cache.decode_attention(0, q.to(DEV), _dev(order[None], torch.int32), [0], [n], dim ** -0.5)
    rows = cache.sparse_decode_attention(0, q.to(DEV), _dev(slots, torch.int32)[None], [n], dim ** -0.5)
    cache.synchronize()
    k, v = (oracle.rows(c, x, slots) for c, x in zip(codes, scales))
    for got in (out, rows):
        _check(got[0], q[0], k, v, scales[1][slots // block], dim ** -0.5, "decode")


@pytest.mark.parametrize(("kv", "heads", "dim", "block", "dtype"), GEOMETRIES)
@pytest.mark.parametrize("seq", [[1, 63, 129, 700], [2600, 30]])
def test_each_kernel_within_its_own_bound(kv, heads, dim, block, dtype, seq):
    """Ordinary values, values of one sign (what is lost shows) and scales far apart, against the bound of the kernel
    that runs: bf16 with head_dim 128 on the tensor cores, up to 16 heads to a KV head for one token; the rest in fp32."""
    tc = dtype == torch.bfloat16 and dim == 128
    one = "decode" if tc and heads // kv <= 16 else "fp32"
    for kind in ("both signs", "one sign", "scales"):
        def scales(rng, shape):
            return (np.exp2(rng.integers(-20, 6, shape)) * (1 + rng.random(shape))).astype(np.float32)

        b = _Batch(seq, kv, dim, block, seed=sum(seq) + dim + heads, heads=heads, dtype=dtype,
                   scales=scales if kind == "scales" else None)
        if kind == "scales":
            b.ks[0] = np.where(np.isnan(b.ks[0]), b.ks[0], np.float32(2.0 ** -8))
            b.cache.k_scale[0].copy_(torch.from_numpy(b.ks[0]))
        if kind == "one sign":
            b.v[0] &= 0x7F
            b.cache.v[0].view(torch.uint8).copy_(torch.from_numpy(b.v[0]))
        q = b.queries(len(seq))
        args = b.table_dev, _dev(b.reqs), _dev(seq)
        out = b.cache.decode_attention(0, q.to(DEV), *args, b.scaling)
        rows = np.full((len(seq), max(seq)), -1, dtype=np.int64)
        for i, s in enumerate(seq):
            rows[i, :s] = b.slots(i, b.rng.permutation(s))
        picked = b.cache.sparse_decode_attention(0, q.to(DEV), _dev(rows, torch.int32), _dev(seq, torch.int32), b.scaling)
        new = [min(s, n) for s, n in zip(seq, (40, 30, 129, 300))]
        offsets = np.concatenate([[0], np.cumsum(new)])
        many = b.queries(int(offsets[-1]))
        ext = b.cache.extend_attention(0, many.to(DEV), *args, _dev(np.subtract(seq, new)), _dev(offsets), b.scaling)
        b.cache.synchronize()
        for i, s in enumerate(seq):
            at = b.slots(i, np.arange(s))
            k, v = (oracle.rows(c, x, at) for c, x in ((b.k[0], b.ks[0]), (b.v[0], b.vs[0])))
            v_scale = b.vs[0][at // block]
            _check(out[i], q[i], k, v, v_scale, b.scaling, one)
            order = np.argsort(at)[np.searchsorted(np.sort(at), rows[i, :s])]
            _check(picked[i], q[i], k[order], v[order], v_scale[order], b.scaling, one)
            for t in {0, new[i] // 2, new[i] - 1}:
                n = s - new[i] + t + 1
                row = offsets[i] + t
                _check(ext[row], many[row], k[:n], v[:n], v_scale[:n], b.scaling, "extend" if tc else "fp32")


@pytest.mark.parametrize("zeros", [1 << 12, 1 << 21])
def test_keys_of_zero_values_before_the_first_others(zeros):
    """Blocks of zeros have the smallest scale, 2^-126, and so the largest share of a row's sum for the reference that
    they set: the sum stays finite over 2^21 of them, and the keys behind them get their part of the mass."""
    kv, heads, dim, block, real, new = 1, 8, 128, 64, 128, 4800
    n = zeros + new
    cache = KV8Cache(1, 2 + new // block, kv, dim, DEV, block_size=block)
    x = torch.zeros(block + new, kv, dim, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(x)
    v[block:block + real] = 1.0  # the first of the new tokens
    cache.append(0, x, v, torch.arange(block + new, device=DEV))
    assert cache.v_scale[0][0].item() == 2.0 ** -126
    table = torch.cat([torch.zeros(zeros // block, dtype=torch.int32, device=DEV),
                       torch.arange(1, 1 + new // block, dtype=torch.int32, device=DEV)])[None]
    q = torch.ones(new, heads, dim, device=DEV, dtype=torch.bfloat16)  # all scores are 0: even weights
    ext = cache.extend_attention(0, q, table, [0], [n], [zeros], [0], 0.1)
    many = 300
    lens = [zeros + real + 5] * many
    full = cache.decode_attention(0, q[:many], table, [0] * many, lens, 0.1)
    lone = cache.decode_attention(0, q[:1], table, [0], lens[:1], 0.1)
    cache.synchronize()
    seen = torch.arange(1, new + 1, device=DEV, dtype=torch.float64)
    for got, want in ((ext, seen.clamp(max=real) / (zeros + seen)), (full, torch.full((many,), real / lens[0], device=DEV)),
                      (lone, torch.full((1,), real / lens[0], device=DEV))):
        want = want[:, None].double()
        off = float(((got.double() - want).abs() / want).max())
        assert off <= 2.0 ** -8 + 2.0 ** -9
