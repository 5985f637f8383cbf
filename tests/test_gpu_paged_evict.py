"""Eviction followed by attention over the new pages, with rows whose old page
is invalid among those that are kept."""
import numpy as np
import pytest

import oracle_lib as O
import paged_bounds as PB
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged
from test_gpu_paged import evict

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("hole", [False, True])
def test_attention_after_an_eviction(T, kind, hole):
    """A row without a page takes a place in the new pages all the same. What is
    attended to there is what the new page held: zeros, in pages that the caller
    cleared."""
    p = Paged([200, 150, 40], 2, 64, 16, kind, spare=20, seed=43, track=True).fill(43)
    p.weights[...] = p.rng.random(p.weights.shape)
    for side in p.sides:
        for t in side:
            t[p.spare] = 0
    if hole:
        p.table[0, 3] = -1
        p.table[1, 8:] = p.pages + 5  # the last rows, which always stay
    kept = [[p.choose(b, h, 60, 2, 30) for h in range(2)] for b in range(3)]
    dst, lens, weights, pool = evict(T, p, 60, 2, 30, 7)
    new = Paged([60, 60, 40], 2, 64, 16, kind, stride=dst.shape[1], track=True)
    new.pages, new.table, new.lens, new.sides, new.weights = p.pages, dst, lens, pool, weights
    for b in range(3):  # the rows behind the last are not looked at
        assert all(len(rows) == lens[b] for rows in kept[b])
    q = kv_bf16((3, 4, 64), 8)
    out, tol, gain, gtol = PB.attend(new, q, 0.125)
    print("[evict] attend", kind, hole, flush=True)
    d = new.device(T)
    PB.check(O.bf16_to_f32(d.attend(q, 0.125)), out, tol, "after eviction")
    got = d.weights.numpy()
    PB.check(got, new.weights + gain, gtol + 2.0 ** -23 * (np.abs(new.weights) + gain), "weights")
    if hole:  # those rows' weight went to zeros: each has that of a score of 0
        for h in range(2):
            gone = np.nonzero(kept[1][h] // 16 >= 8)[0]
            assert gone.size >= 22 and np.ptp(gain[1, h, gone]) < 1e-12
