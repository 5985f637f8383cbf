"""Paged decode attention over affine values of very different magnitudes:
every channel of the output is as near the 64-bit one as its own terms allow
(paged_bounds.py), whatever lies in other rows, groups and channels."""
import numpy as np
import pytest

import oracle_lib as O
import paged_bounds as PB
from inputs import kv_bf16
from paged_ref import AFFINE, Paged

pytestmark = pytest.mark.gpu

LAYOUTS = [(4, 4, 64), (8, 8, 32), (4, 8, 128), (8, 4, 32)]
DIMS = [64, 128, 256, 512]


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


def pool(D, bk, bv, gs, lens=(700, 33), Hkv=1, R=16, seed=3, track=False):
    if gs > D:
        pytest.skip("a group is at most a row")
    return Paged(list(lens), Hkv, D, R, AFFINE, bk, bv, gs, seed=seed, track=track).fill(seed + D)


def at(p, b, rows):
    """Index of a pool buffer: the rows of sequence b, all KV heads."""
    rows = np.asarray(rows)  # advanced indices at the two ends: [rows, KV heads, .]
    return p.table[b, rows // p.R], slice(None), rows % p.R


def times(p, b, rows, groups, power):
    """The values of `groups` of sequence b's rows times 2^power."""
    for t in p.sides[1][1:]:
        x = O.bf16_to_f32(t[at(p, b, rows)])
        x[..., groups] *= np.float32(2.0 ** power)
        t[at(p, b, rows)] = O.bf16_from_f32(x)


def attend(T, p, tag, scale=None, H=4, seed=5):
    scale = p.D ** -0.5 if scale is None else scale
    q = kv_bf16((p.B, H, p.D), seed)
    out, tol, gain, gtol = PB.attend(p, q, scale)
    d = p.device(T)
    print("[spread]", tag, flush=True)
    got = O.bf16_to_f32(d.attend(q, scale))
    PB.check(got, out, tol, tag)
    if p.weights is not None:
        PB.check(d.weights.numpy(), p.weights + gain, gtol + 2.0 ** -23 * (p.weights + gain), tag + " weights")
    return got


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("power", [7, 12, 17, 24, 30, 60, 110])
def test_one_group_of_one_row(T, D, bk, bv, gs, power):
    p = pool(D, bk, bv, gs)
    times(p, 0, [350], [0], power)
    times(p, 1, [2], [-1], power)
    attend(T, p, f"one group {D} {bk} {bv} {gs} 2^{power}")


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("power", [-60, -30, -17, 12, 30])
def test_one_group_of_every_row(T, D, bk, bv, gs, power):
    p = pool(D, bk, bv, gs, track=True)
    for b, n in enumerate(p.lens):
        times(p, b, range(n), [D // gs // 2], power)
    attend(T, p, f"group {D} {bk} {bv} {gs} 2^{power}")


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", DIMS)
def test_a_power_for_every_group_of_every_row(T, D, bk, bv, gs):
    p = pool(D, bk, bv, gs, lens=(700, 33, 1, 200))
    for t in range(1, 3):
        power = np.random.default_rng(D).integers(-20, 21, p.sides[1][t].shape)
        p.sides[1][t][...] = O.bf16_from_f32(O.bf16_to_f32(p.sides[1][t]) * (2.0 ** power).astype(np.float32))
    attend(T, p, f"every group {D} {bk} {bv} {gs}")


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("rise", [-0.2, 0.2])
def test_magnitudes_that_rise_or_fall_along_the_rows(T, D, rise):
    p = pool(D, 4, 8, 64)
    for i in range(700):
        times(p, 0, [i], slice(None), round(rise * (i - 350)))
    attend(T, p, f"rise {D} {rise}")


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("power", [18, 30])
def test_a_large_row_of_little_weight(T, D, power):
    """Of about 2^-25 of the largest weight."""
    p = pool(D, 8, 8, 32, lens=(700,))
    q = O.bf16_to_f32(kv_bf16((1, 1, D), 5)).astype(np.float64)[0, 0]
    s = p.rows(0, 0, 700)[1] @ q * 0.5 * 1.4427
    row = int(np.abs(s - s.max() + 25).argmin())
    times(p, 0, [row], slice(None), power)
    attend(T, p, f"light row {D} 2^{power} of weight 2^{s[row] - s.max():.1f}", scale=0.5, H=1)


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("where", ["first", "middle", "all"])
def test_rows_of_zeros(T, D, bk, bv, gs, where):
    """As they are appended: steps of 1e-7 and no bias."""
    p = pool(D, bk, bv, gs)
    zero = p.stored(np.zeros((1, D), np.uint16), bv)
    for b, n in enumerate(p.lens):
        rows = {"first": range(n // 2), "middle": range(n // 3, n // 2, 3), "all": range(n)}[where]
        for t, z in zip(p.sides[1], zero):
            t[at(p, b, rows)] = z[0]
    got = attend(T, p, f"zeros {D} {bk} {bv} {gs} {where}")
    assert where != "all" or np.all(got == 0)


@pytest.mark.parametrize("bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("part", [1, 2])
@pytest.mark.parametrize("bits", [0x7F80, 0xFF80, 0x7FC0])
def test_infinite_scales_and_biases(T, D, bk, bv, gs, part, bits):
    """Infinite (or NaN) channels stay in their group."""
    p = pool(D, bk, bv, gs)
    t = p.sides[1][part]
    page, _, row = at(p, 0, 350)
    t[page, :, row, 0] = bits
    page, _, row = at(p, 1, 1)
    t[page, :, row, -1] = bits
    got = attend(T, p, f"infinite {D} {bk} {bv} {gs} {part} {bits:x}")
    assert np.all(np.isfinite(got[0, :, gs:])) and not np.any(np.isfinite(got[0, :, :gs]))


@pytest.mark.parametrize("D", DIMS)
def test_a_row_whose_range_passes_f32(T, D):
    """Finite bf16 rows from one end of the type to the other: the append stores
    an infinite scale. Groups of other rows' size are not touched by it."""
    p = pool(D, 4, 4, 32)
    x = O.bf16_to_f32(kv_bf16((1, D), 9))
    x[0, 0], x[0, 1] = 3.3e38, -3.3e38
    for t, z in zip(p.sides[1], p.stored(O.bf16_from_f32(x), 4)):
        t[at(p, 0, [100])] = z[0]
    got = attend(T, p, f"range {D}")
    assert np.all(np.isfinite(got[0, :, 32:]))


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("power", [-70, 115])
def test_all_values_of_one_magnitude(T, D, power):
    p = pool(D, 4, 4, 64)
    for b, n in enumerate(p.lens):
        times(p, b, range(n), slice(None), power)
    attend(T, p, f"magnitude {D} 2^{power}")


@pytest.mark.parametrize("D", DIMS)
def test_spread_values_over_the_whole_card(T, D):
    """Many parts, joined; partial steps; invalid pages between."""
    p = pool(D, 4, 4, 64, lens=(9001, 77), Hkv=2, R=64, track=True)
    p.table[0, 30] = -1
    rng = np.random.default_rng(D)
    for i in rng.integers(0, 9001, 200):
        times(p, 0, [i], [int(rng.integers(0, D // 64))], int(rng.integers(-30, 40)))
    attend(T, p, f"card {D}")


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("window", [70, 333])
def test_spread_values_in_windows_of_two_sets_of_heads(T, D, window):
    """20 query heads a KV head; the large group inside the window, and before
    it, where it does not count."""
    p = pool(D, 8, 8, 32, lens=(700, 33, 0, 340), track=True)
    times(p, 0, [690], [1], 25)
    times(p, 0, [100], [0], 60)
    times(p, 3, [339], [-1], 40)
    q = kv_bf16((p.B, 20, D), 6)
    out, tol, gain, gtol = PB.attend(p, q, 0.1, window)
    d = p.device(T)
    print("[spread] windows", D, window, flush=True)
    PB.check(O.bf16_to_f32(d.attend(q, 0.1, window)), out, tol, "windows")
    PB.check(d.weights.numpy(), gain, gtol + 2.0 ** -23 * gain, "windows weights")


@pytest.mark.parametrize("D", DIMS)
def test_spread_values_in_some_of_many_short_sequences(T, D):
    """Several sequences a workgroup, some of its wavefronts in a second pass
    while others go on; the same every time."""
    rng = np.random.default_rng(D)
    p = pool(D, 4, 4, 64, lens=tuple(int(n) for n in rng.integers(0, 90, 500)), Hkv=2)
    for b in range(0, 500, 2):
        if p.lens[b]:
            times(p, b, [int(rng.integers(0, p.lens[b]))], [int(rng.integers(0, D // 64))], int(rng.integers(10, 50)))
    q = kv_bf16((p.B, 4, D), 7)
    out, tol, _, _ = PB.attend(p, q, D ** -0.5)
    d = p.device(T)
    print("[spread] short", D, flush=True)
    first = d.attend(q, D ** -0.5)
    PB.check(O.bf16_to_f32(first), out, tol, "short")
    for _ in range(5):
        assert np.array_equal(d.attend(q, D ** -0.5), first)
