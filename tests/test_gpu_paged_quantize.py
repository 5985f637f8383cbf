"""The quantized append byte for byte against tqkv_affine_quantize: long ragged
prompts (eight tokens a workgroup from 2,048 on) and values on which quantizers
differ."""
import numpy as np
import pytest

import oracle_lib as O
from inputs import grid_bf16, kv_bf16
from paged_ref import AFFINE, Paged

pytestmark = pytest.mark.gpu

LAYOUTS = [(4, 4, 64), (8, 8, 32), (4, 8, 128), (8, 4, 32)]


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


def quantized(T, x, gs, bits):
    """What the library's quantizer makes of rows x [n, D]."""
    n, D = x.shape
    dx = T.DeviceArray.of(x)
    out = [T.DeviceArray((n, D * bits // 32), np.uint32)] + [T.DeviceArray((n, D // gs), np.uint16) for _ in range(2)]
    T.affine_quantize(dx.ptr, 1, n, D, gs, bits, *[t.ptr for t in out])
    T.hip().sync()
    return [t.numpy() for t in out]


def append(T, p, x, counts, gap=0):
    """x [gap + tokens + behind, 2 Hkv, D]; every byte of the pool compared."""
    Hkv, D, R = p.Hkv, p.D, p.R
    starts = np.cumsum([gap, *counts]).astype(np.int32)
    total = int(starts[-1]) - gap
    want = [[t.copy() for t in side] for side in p.sides]
    b = np.repeat(np.arange(p.B), counts)
    row = np.concatenate([np.arange(n - c, n) for n, c in zip(p.lens, counts)]).astype(np.int64)
    page = p.table[b, row // R]
    for i, (side, bits) in enumerate(zip(want, (p.bk, p.bv))):
        y = np.ascontiguousarray(x[gap:gap + total, i * Hkv:(i + 1) * Hkv]).reshape(-1, D)
        for t, src in zip(side, quantized(T, y, p.gs, bits)):
            t[page, :, row % R] = src.reshape(total, Hkv, -1)
    d = p.device(T)
    dx, ds = T.DeviceArray.of(x), T.DeviceArray.of(starts)
    T.paged_append(d.view(), dx.ptr, dx.ptr + 2 * Hkv * D, ds.ptr, len(x), 2 * Hkv * D, D)
    T.hip().sync()
    for got, w in zip(d.host(), want):
        for t, u in zip(got, w):
            assert np.array_equal(t, u), np.argwhere(t != u)[:5]
    if p.weights is not None:
        w = p.weights.copy()
        w[b, :, row] = 0
        assert np.array_equal(d.weights.numpy(), w)


def ragged(total, batch, seed):
    """Counts of `batch` sequences, some empty, that add up to total."""
    cuts = np.sort(np.random.default_rng(seed).integers(0, total + 1, batch - 1))
    cuts[:2] = 0
    counts = np.diff([0, *cuts, total])
    counts[batch // 2 - 1], counts[batch // 2] = 0, counts[batch // 2] + counts[batch // 2 - 1]
    return [int(c) for c in counts]


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("tokens,Hkv", [(2047, 3), (2048, 1), (2049, 3), (2055, 2)])
def test_prompts_of_many_tokens(T, bk, bv, gs, D, tokens, Hkv):
    if gs > D:
        pytest.skip("a group is at most a row")
    counts = ragged(tokens - 5, 9, tokens)  # five tokens lie outside the sequences
    lens = [c + 7 * (i % 3) for i, c in enumerate(counts)]
    p = Paged(lens, Hkv, D, 16, AFFINE, bk, bv, gs, spare=1, seed=D, track=Hkv == 3)
    if p.weights is not None:
        p.weights += 1.5
    print("[quantize] prompts", bk, bv, gs, D, tokens, Hkv, flush=True)
    append(T, p, kv_bf16((tokens, 2 * Hkv, D), tokens, frac=0.02, mult=4.0), counts, gap=2)


def awkward(n, heads, D, gs, seed):
    """Rows on which quantizers differ, ordinary ones between them in every
    wavefront: ties, zeros, constant groups, the least step, the type's ends,
    infinities and NaN."""
    rng = np.random.default_rng(seed)
    x = grid_bf16((n, heads, D), seed)
    f = O.bf16_to_f32(x)
    bits = x.copy()
    for i in range(n):
        for h in range(heads):
            g = slice(int(rng.integers(0, D // gs)) * gs, None)
            g = slice(g.start, g.start + gs)
            kind = int(rng.integers(0, 14))
            if kind == 0:
                f[i, h, g] = 0.0
            elif kind == 1:
                f[i, h, g] = -0.0
            elif kind == 2:
                f[i, h, g] = rng.choice([1.0, -3.5, 1e-30, -2e38])
            elif kind == 3:
                f[i, h, g] *= np.float32(1e-7)
            elif kind == 4:
                f[i, h, g] *= np.float32(1e38)
            elif kind == 5:
                f[i, h, g] *= np.float32(1e-38)
            elif kind == 6:  # multiples of a step: codes at and next to halves
                f[i, h, g] = rng.integers(-15, 31, gs) * np.float32(0.5)
            elif kind == 7:
                f[i, h, g] = rng.integers(0, 511, gs) * np.float32(0.5)
            elif kind == 8:
                f[i, h, g.start] = rng.choice([np.inf, -np.inf])
            elif kind == 9:
                f[i, h, g.start + 1], f[i, h, g.start + 5] = np.inf, -np.inf
            elif kind == 10:
                f[i, h, g.start + int(rng.integers(0, gs))] = np.nan
            elif kind == 11:
                f[i, h, g] = np.nan
    with np.errstate(over="ignore"):
        return np.where(f == O.bf16_to_f32(x), bits, O.bf16_from_f32(f))


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("tokens", [61, 2051])
def test_values_on_which_quantizers_differ(T, bk, bv, gs, D, tokens):
    if gs > D:
        pytest.skip("a group is at most a row")
    counts = ragged(tokens, 5, tokens)
    p = Paged(counts, 2, D, 32, AFFINE, bk, bv, gs, seed=D)
    print("[quantize] awkward", bk, bv, gs, D, tokens, flush=True)
    append(T, p, awkward(tokens, 4, D, gs, tokens + D + bk), counts)


@pytest.mark.parametrize("bits", [4, 8])
def test_every_bf16_beside_every_scale(T, bits):
    """All finite bf16 values, in groups that share a magnitude, so that each
    value meets many steps, those above 2^100 among them."""
    every = np.arange(0x10000, dtype=np.uint32).astype(np.uint16)
    every = every[(every & 0x7F80) != 0x7F80]
    rng = np.random.default_rng(bits)
    rows = []
    for spread in (1, 2, 5, 20):  # exponents of a group within `spread`
        mag = (every & 0x7FFF).astype(np.int64)
        order = np.argsort(mag + rng.integers(0, spread * 128, mag.size))
        rows.append(every[order])
    x = np.concatenate(rows)
    x = x[:x.size // 512 * 512].reshape(-1, 2, 256)
    x = np.concatenate([x, x[::-1]])
    p = Paged([len(x)], 1, 256, 64, AFFINE, bits, bits, 32, seed=3)
    print("[quantize] every value", bits, len(x), flush=True)
    append(T, p, np.ascontiguousarray(x), [len(x)])
