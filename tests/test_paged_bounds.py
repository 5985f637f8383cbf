"""The paged attention's error bounds (paged_bounds.py) reject answers that a
plausible mistake gives, and accept what the formats' roundings give."""
import numpy as np
import pytest

import oracle_lib as O
import paged_bounds as PB
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged, values_of

LAYOUTS = [(BF16, 16, 16, 64), (AFFINE, 4, 4, 64), (AFFINE, 8, 8, 32), (AFFINE, 8, 4, 64),
           (AFFINE, 4, 8, 32), (AFFINE, 4, 4, 128)]


def half_rounded(x, bits):
    return (x.astype(np.float16).astype(np.float64) if bits != 16 else
            O.bf16_to_f32(O.bf16_from_f32(x.astype(np.float32))).astype(np.float64))


@pytest.mark.parametrize("kind,bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_wrong_answers_lie_outside_the_bounds(kind, bk, bv, gs, D):
    if gs > D:
        pytest.skip("a group is at most a row")
    n, scale = 300, D ** -0.5
    p = Paged([n], 1, D, 16, kind, bk, bv, gs, seed=D).fill(D)
    q = kv_bf16((1, 4, D), 11 * 4 + D)
    out, tol, gain, gtol = PB.attend(p, q, scale)
    _, k, v, _ = p.rows(0, 0, n)
    qf = O.bf16_to_f32(q).astype(np.float64)[0]

    def answer(k, v, uniform=False):
        s = qf @ k.T * scale
        w = np.exp(s - s.max(1, keepdims=True)) if not uniform else np.ones_like(s)
        w /= w.sum(1, keepdims=True)
        return w @ v, w.sum(0)

    def outside(o, g, share, gshare):
        assert np.mean(PB.errors(o, out[0], tol[0]) > 1) >= share
        assert np.mean(PB.errors(g, gain[0, 0, :n], gtol[0, 0, :n]) > 1) >= gshare

    # What f32 (and f16 values, rounded to bf16 at the end) makes of it lies inside.
    o, g = answer(k.astype(np.float32), half_rounded(v, bv).astype(np.float32))
    assert PB.errors(O.bf16_to_f32(O.bf16_from_f32(o.astype(np.float32))), out[0], tol[0]).max() <= 1
    assert PB.errors(g, gain[0, 0, :n], gtol[0, 0, :n]).max() <= 1
    outside(0 * out[0], 0 * g, 0.9, 1.0)
    outside(*answer(k, v, uniform=True), 0.9, 0.9)
    w = answer(k, v)[1]
    swapped = k.copy()  # the heaviest row's key and the lightest's
    swapped[[w.argmax(), w.argmin()]] = k[[w.argmin(), w.argmax()]]
    o, g = answer(swapped, v)
    assert np.mean(PB.errors(o, out[0], tol[0]) > 1) >= 0.25
    assert PB.errors(g, gain[0, 0, :n], gtol[0, 0, :n])[[w.argmax(), w.argmin()]].min() > 1
    if kind == AFFINE:  # one group's biases left out, of the keys and of the values
        flat = [[t.copy() for t in side] for side in p.sides]
        for side in flat:
            side[2][..., 0] = 0
        rows = np.arange(n)
        at = (p.table[0, rows // 16], 0, rows % 16)
        k0 = values_of([t[at] for t in flat[0]], bk, gs)
        v0 = values_of([t[at] for t in flat[1]], bv, gs)
        outside(*answer(k0, v), 0.5, 0.9)
        o, _ = answer(k, v0)  # (biases of both signs nearly cancel for a head now and then)
        assert np.mean(PB.errors(o, out[0], tol[0])[:, :gs] > 1) >= 0.7


def test_infinities_and_nan_are_compared():
    want = np.array([np.inf, -np.inf, np.nan, 1.0, 1.0])
    tol = np.full(5, 0.1)
    assert PB.errors(want, want, tol).max() == 0
    for i, bad in enumerate([np.nan, np.inf, 1.0, np.nan, np.inf]):
        got = want.copy()
        got[i] = bad
        assert PB.errors(got, want, tol)[i] > 1
