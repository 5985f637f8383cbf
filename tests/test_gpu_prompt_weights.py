"""Small softmax weights over affine pages: one key far above all others, which
hold the values."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from paged_ref import AFFINE, Paged, values_of
from test_gpu_prompt import T, run_paged, say, starts_of  # noqa: F401 (T: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[3], [140]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [500, 5000])
def test_weights_far_below_the_largest(T, counts, D, bits, n):
    """The first key's value is zero and its weight nearly one; the others', 15 to
    19 nats below, are all of the output. A weight may be off by 2^-11 of itself
    or 2^-32 of the largest: not by the 2^-25 that f16 alone would leave."""
    rng = np.random.default_rng(D + n)
    starts = starts_of(counts)
    q = np.zeros((counts[0], 2, D), np.float32)
    q[..., 0] = 8.0
    q = O.bf16_from_f32(q)
    p = Paged([n], 1, D, 16, AFFINE, bits, bits, 32, seed=5)
    for row in range(n):
        k, v = np.zeros((1, D), np.float32), rng.standard_normal((1, D)).astype(np.float32) + 2.0
        if row == 0:
            k[:, 0], v = 1.0, 0.0 * v
        p.write(0, row, O.bf16_from_f32(k), O.bf16_from_f32(v))
    for below in (15.0, 17.0, 17.4, 19.0):
        say("small weights", counts, D, bits, n, below)
        scale = below / 8.0
        got = O.bf16_to_f32(run_paged(T, p, q, starts, scale))
        want, tol = R.paged(p, q, starts, scale)
        # That tolerance has 2^-25 of |v - out| a key, summed: 2^-32 in its place,
        # and the largest weight in it, which 2^-25 bounds from below, is one.
        for i in range(counts[0]):
            see = n - counts[0] + i + 1
            rows = np.arange(see)
            at = (p.table[0, rows // 16], 0, rows % 16)
            v = values_of([t[at] for t in p.sides[1]], bits, 32)
            for h in range(2):
                tol[i, h] -= (2.0 ** -25 - 2.0 ** -32) * np.abs(v - want[i, h]).sum(0)
        assert tol.min() > 0.0
        R.check(got, want, tol, f"small weights {below}")
        assert np.median(tol / np.maximum(np.abs(want), 1e-30)) < 0.1  # a tolerance that says something
