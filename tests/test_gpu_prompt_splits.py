"""Prompt attention with divided keys: partial results of every kernel, the rows
that the join does again, and windows of any width."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged
from test_gpu_prompt import T, run_packed, run_paged, say, starts_of  # noqa: F401 (T: the fixture)

pytestmark = pytest.mark.gpu


def some(a, b, seed, most=40):
    """Tokens of [a, b): both ends, and a few of the rest."""
    rng = np.random.default_rng(seed)
    t = np.arange(a, b)
    return t if len(t) <= most else np.unique(np.r_[t[:3], t[-3:], rng.choice(t, most - 6)])


@pytest.mark.parametrize("D,G,counts", [(64, 1, [9000]), (128, 1, [8700, 300]), (128, 2, [9001]), (256, 1, [4500]), (512, 1, [4600, 1])])
@pytest.mark.parametrize("causal,window", [(True, -1), (True, 5000), (True, 700), (False, -1)])
def test_packed_with_divided_keys(T, D, G, counts, causal, window):
    say("packed splits", D, G, counts, causal, window)
    n = sum(counts)
    starts = starts_of(counts)
    assert T.packed_attend_workspace_size(len(counts), G, 1, D, n) > 0
    x = kv_bf16((n, G + 2, D), D + n, frac=0.02, mult=4.0)
    got = O.bf16_to_f32(run_packed(T, x, G, 1, starts, D ** -0.5, causal, window))
    f = O.bf16_to_f32(x).astype(np.float64)
    for a, b in zip(starts[:-1], starts[1:]):
        at = some(a, b, D)
        want, tol = R.attend(f[at, :G], f[a:b, G], f[a:b, G + 1], at - a, D ** -0.5, causal, window)
        R.check(got[at], want, tol, "packed splits")


@pytest.mark.parametrize("D,n", [(64, 9000), (128, 9000), (256, 4500), (512, 4500)])
@pytest.mark.parametrize("what", ["v inf", "v nan", "k nan"])
def test_packed_splits_that_are_not_finite(T, D, n, what):
    """Token n - 200 holds infinities or NaN: queries before it are as without it,
    those behind it meet it in one partial result of several."""
    say("packed splits", D, n, what)
    starts = starts_of([n])
    assert T.packed_attend_workspace_size(1, 1, 1, D, n) > 0
    x = kv_bf16((n, 3, D), D)
    f = O.bf16_to_f32(x).astype(np.float64)
    bad, at = (0x7F80 if "inf" in what else 0x7FC0), n - 200
    reached = np.array([5, D - 1])
    if what[0] == "v":
        x[at, 2, reached] = bad
    else:
        x[at, 1] = bad
    got = O.bf16_to_f32(run_packed(T, x, 1, 1, starts, D ** -0.5))
    t = np.r_[some(0, at, D), np.arange(at - 5, at)]
    want, tol = R.attend(f[t, :1], f[:, 1], f[:, 2], t, D ** -0.5)
    R.check(got[t], want, tol, "before")
    t = some(at, n, D)
    if what[0] == "v":
        assert np.all(got[t][..., reached] == np.inf if "inf" in what else np.isnan(got[t][..., reached]))
        want, tol = R.attend(f[t, :1], f[:, 1], f[:, 2], t, D ** -0.5)
        rest = np.setdiff1d(np.arange(D), reached)
        R.check(got[t][..., rest], want[..., rest], tol[..., rest], "beside")
    else:
        assert np.all(np.isnan(got[t]))


def divided(T, p, counts, rows):
    """The call's keys are divided: beyond the dequantized rows of many queries'
    affine pages there is room for two partial results and more."""
    need = T.paged_prefill_workspace_size(p.device(T).view(), 1, sum(counts), rows)
    slab = 4 * p.B * p.Hkv * rows * p.D if p.kind == AFFINE and counts == COUNTS[1] else 0
    return need >= slab + sum(counts) * 2 * (p.D + 2) * 4


# Few queries divide keys from 1,024 on; 40 and 70 rows of a head the blocks of a
# prompt.
COUNTS = [[4, 3], [40, 30]]


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("what", ["v", "k"])
def test_pages_with_divided_keys_that_are_not_finite(T, kind, counts, D, what):
    say("paged splits", kind, counts, D, what)
    lens = [6000, 2500]
    p = Paged(lens, 1, D, 16, kind, 8, 8, 32, seed=5).fill(4)
    starts = starts_of(counts)
    q = kv_bf16((sum(counts), 1, D), 3)
    want, tol = R.paged(p, q, starts, D ** -0.5)
    side = p.sides[1 if what == "v" else 0]
    n, m = lens[0], counts[0]
    for row in (n - 2, n - 1):  # seen by the first sequence's last two queries (the last)
        at = (p.table[0, row // 16], 0, row % 16)
        if kind == BF16:
            side[0][at][3] = 0x7F80 if what == "v" else 0x7FC0
            reached = np.array([3])
        else:
            side[1][at][0] = 0x7FC0
            reached = np.arange(32)
    assert divided(T, p, counts, p.stride * p.R)
    got = O.bf16_to_f32(run_paged(T, p, q, starts, D ** -0.5))
    clean = np.r_[0:m - 2, m:sum(counts)]
    R.check(got[clean], want[clean], tol[clean], "before")
    hit = got[m - 2:m]
    if what == "v":
        assert not np.any(np.isfinite(hit[..., reached]))
        rest = np.setdiff1d(np.arange(D), reached)
        R.check(hit[..., rest], want[m - 2:m][..., rest], tol[m - 2:m][..., rest], "beside")
    else:
        assert np.all(np.isnan(hit))


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("side", [0, 1])
def test_affine_rows_far_apart_with_divided_keys(T, counts, D, side):
    """A sequence's last key (value) is 2^60 times as large as the others: its
    other queries are as with an ordinary one there."""
    say("far splits", counts, D, side)
    lens = [6000, 2500]
    pools = [Paged(lens, 1, D, 16, AFFINE, 8, 8, 32, seed=5).fill(4) for _ in range(2)]
    for b, n in enumerate(lens):
        x = [O.bf16_to_f32(kv_bf16((1, D), 10 * n + i)) for i in range(2)]
        x[side] = x[side] * np.float32(2.0 ** 60)
        pools[1].write(b, n - 1, *[O.bf16_from_f32(y) for y in x])
    starts = starts_of(counts)
    q = kv_bf16((sum(counts), 1, D), 3)
    want, tol = R.paged(pools[0], q, starts, D ** -0.5)
    assert divided(T, pools[1], counts, pools[1].stride * 16)
    got = O.bf16_to_f32(run_paged(T, pools[1], q, starts, D ** -0.5))
    before = np.ones(sum(counts), bool)
    before[starts[1:] - 1] = False
    if side == 1:  # values are bf16 in such a head: half a step of each
        want, tol = R.paged(pools[1], q, starts, D ** -0.5)
    R.check(got[before], want[before], tol[before], "far splits")
