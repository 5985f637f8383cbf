"""Paged decode attention within the bounds of paged_bounds.py, which are tight
enough to tell a wrong answer from a rounded one: every layout, windows, long
and many sequences, infinite values and extreme queries."""
import numpy as np
import pytest

import oracle_lib as O
import paged_bounds as PB
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged

pytestmark = pytest.mark.gpu

LAYOUTS = [(BF16, 16, 16, 64), (AFFINE, 4, 4, 64), (AFFINE, 8, 8, 32), (AFFINE, 8, 4, 64),
           (AFFINE, 4, 8, 32), (AFFINE, 4, 4, 128)]


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


def attend(T, p, H, tag, window=-1, max_rows=None, scale=None, q=None):
    scale = p.D ** -0.5 if scale is None else scale
    q = kv_bf16((p.B, H, p.D), 11 * H + p.D) if q is None else q
    out, tol, gain, gtol = PB.attend(p, q, scale, window, max_rows)
    d = p.device(T)
    print("[numerics]", tag, flush=True)
    got = O.bf16_to_f32(d.attend(q, scale, window, max_rows))
    PB.check(got, out, tol, tag)
    if p.weights is not None:
        w = d.weights.numpy()
        PB.check(w, p.weights + gain, gtol + 2.0 ** -23 * (p.weights + gain), tag + " weights")
        assert np.array_equal(w[gain == 0], p.weights[gain == 0])
    return got


@pytest.mark.parametrize("kind,bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("R,H,Hkv", [(16, 6, 2), (64, 16, 1)])
def test_every_layout(T, kind, bk, bv, gs, D, R, H, Hkv):
    if gs > D:
        pytest.skip("a group is at most a row")
    p = Paged([1, 0, 300, 16, 33, 128], Hkv, D, R, kind, bk, bv, gs, spare=1, seed=D, track=True).fill(D + R)
    p.weights += p.rng.random(p.weights.shape, np.float32)
    attend(T, p, H, f"layout {kind} {bk} {bv} {gs} {D}")


@pytest.mark.parametrize("kind,bk,bv,gs", [(BF16, 16, 16, 64), (AFFINE, 4, 4, 64), (AFFINE, 8, 8, 32)])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("window", [1, 15, 16, 33, 65, 200, 1203, 5000])
def test_windows(T, kind, bk, bv, gs, D, window):
    """What lies before the window is NaN here."""
    p = Paged([300, 5, 0, 1203], 2, D, 64, kind, bk, bv, gs, seed=window, track=window in (33, 1203)).fill(window)
    for b, n in enumerate(p.lens):
        for row in range(0, max(0, int(n) - window)):
            for side in p.sides:
                side[-1][p.table[b, row // 64], :, row % 64] = 0x7FC0
    attend(T, p, 4, f"window {window} {kind} {D}", window=window)


@pytest.mark.parametrize("kind,D,n,G", [(BF16, 64, 33001, 3), (BF16, 256, 20011, 2), (AFFINE, 128, 70007, 1),
                                        (AFFINE, 512, 12345, 17)])
def test_one_sequence_over_the_whole_card(T, kind, D, n, G):
    attend(T, Paged([n], 1, D, 256, kind, seed=n, track=G != 2).fill(n), G, f"long {kind} {D}")


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_sharp_softmax(T, kind, D):
    p = Paged([500, 129], 2, D, 64, kind, seed=12, track=True).fill(12)
    for scale in (0.5, -0.3, 0.0):
        attend(T, p, 4, f"sharp {kind} {D} {scale}", scale=scale)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n", [1, 40, 9000])
def test_infinite_values_of_bf16_rows(T, D, n):
    """A channel with an infinite value is infinite, of that sign; with both
    signs, or a NaN, it is NaN; the other channels are as they would be."""
    p = Paged([n, 33], 2, D, 16, BF16, seed=n).fill(n)
    v = p.sides[1][0]
    for row, ch, bits in [(0, 0, 0x7F80), (n // 2, 3, 0xFF80), (n - 1, D - 1, 0x7FC0), (0, 9, 0x7F80),
                          (n - 1, 9, 0xFF80), (n // 3, 20, 0x7F80), (n // 2, 20, 0x7F80)]:
        v[p.table[0, row // 16], 1, row % 16, ch] = bits
    got = attend(T, p, 4, f"infinite values {D} {n}", scale=0.1 * D ** -0.5)
    assert got[0, 2, 0] == np.inf and got[0, 3, 3] == -np.inf and np.isnan(got[0, 2, D - 1])
    assert np.all(np.isfinite(got[0, :2])) and np.count_nonzero(~np.isfinite(got)) == 2 * 5


@pytest.mark.parametrize("kind,bk,bv,gs", LAYOUTS[:3])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("power", [90, 120, 122])
def test_queries_near_the_largest_of_the_type(T, kind, bk, bv, gs, D, power):
    """Scores of up to 2^126: the row of the largest one has all the weight."""
    n = 200
    p = Paged([n], 1, D, 32, kind, bk, bv, gs, seed=D, track=True).fill(D)
    q = O.bf16_to_f32(kv_bf16((1, 4, D), 17)) * np.float32(2.0 ** power)
    _, k, v, _ = p.rows(0, 0, n)
    s = k @ q[0].T.astype(np.float64) * D ** -0.5
    first, second = np.sort(s, 0)[-1], np.sort(s, 0)[-2]
    x = np.abs(q[0].T.astype(np.float64))
    ck, zk, _ = PB.parts_of(p, p.sides[0], p.bk, 0, 0, n)
    sure = first - second > 4 * (D + 64) * 2.0 ** -24 * ((ck + zk) @ x).max(0) * D ** -0.5
    assert np.count_nonzero(sure) >= 3 and np.abs(s).max() < 2.0 ** 126
    d = p.device(T)
    print("[numerics] large queries", kind, D, power, flush=True)
    got = O.bf16_to_f32(d.attend(O.bf16_from_f32(q), D ** -0.5))
    for h in np.nonzero(sure)[0]:
        want = v[s[:, h].argmax()]
        assert np.all(np.abs(got[0, h] - want) <= (2.0 ** -8 + 2.0 ** -9) * np.abs(want) + 2.0 ** -20)
    assert np.all(np.isfinite(d.weights.numpy())) and abs(d.weights.numpy().sum() - 4) < 1e-3
