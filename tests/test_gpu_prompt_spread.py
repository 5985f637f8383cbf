"""Affine rows whose groups differ in magnitude: queries keep the bits of what
they see, whatever the rows and groups beside it hold. Over the pages, for few
queries a sequence and for many, against 64 bits."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, Paged, codes_of, values_of
from test_gpu_prompt import T, run_paged, say, starts_of  # noqa: F401 (T: the fixture)

pytestmark = pytest.mark.gpu

FEW, MANY = [3, 3], [150, 90]
LENS = [150, 90]


def bf16(x):
    return O.bf16_from_f32(np.asarray(x, np.float32))


def stored(p, i, n, side):
    """(values, what their groups' scales and biases allow at most) of a
    sequence's rows, f64 [n, D]."""
    r = np.arange(n)
    at = (p.table[i, r // 16], 0, r % 16)
    t, bits = [x[at] for x in p.sides[side]], (p.bk, p.bv)[side]
    s, z = (np.repeat(O.bf16_to_f32(x).astype(np.float64), p.gs, axis=-1) for x in t[1:])
    return values_of(t, bits, p.gs), np.maximum(np.abs(z), np.abs(s * (2 ** bits - 1) + z))


def value_pool(D, bits, gs, far, shape, few):
    """Values of size 1 in the rows that some queries see alone, 2^far times as
    large from there on; `shape`: around zero, far from zero (a range of 2^-5 of
    the bias), or codes over a bias of zero."""
    p = Paged(LENS, 1, D, 16, AFFINE, 4, bits, gs, seed=5)
    rng = np.random.default_rng(D + bits)
    for b, n in enumerate(LENS):
        small = n - 2 if few else n // 2
        for row in range(n):
            k, v = rng.standard_normal((2, 1, D))
            if shape == "bias":
                v = 1.0 + v * 2.0 ** -7
            p.write(b, row, bf16(k), bf16(v * (1.0 if row <= small else 2.0 ** far)))
            at = (p.table[b, row // 16], 0, row % 16)
            if shape == "codes" and row <= small:
                p.sides[1][0][at] = rng.integers(0, 1 << 32, D * bits // 32, dtype=np.uint32)
                p.sides[1][1][at] = bf16(rng.uniform(0.5, 1.0, D // gs) / (2 ** bits - 1))
                p.sides[1][2][at] = 0
    return p


@pytest.mark.parametrize("counts", [FEW, MANY])
@pytest.mark.parametrize("D,gs", [(64, 32), (128, 64), (256, 128), (512, 32)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", ["zero", "bias", "codes"])
def test_values_of_small_groups_keep_their_bits(T, counts, D, gs, bits, shape):
    """Beside ones 2^18 to 2^28 times larger elsewhere; a window of one key gives the
    stored value itself. Where groups' largest values lie less than 2^28 apart, a
    value may be off by half of f16's step, 2^-11 of itself or 2^-25 in units in
    which the head's largest is 2^14 or more, so the group's 2^-14 or more:
    2^-11 of its group's largest; and by half of 2^-25 if it is rounded before it
    is brought to these units (what is below 2^-14 there, by 2^-11 of itself).
    The units leave the largest below 2^15, so that this may hold up to 2^29
    apart; where it does not a value is bf16 (half a step, 2^-8 of it)."""
    q = kv_bf16((sum(counts), 2, D), D)
    starts = starts_of(counts)
    for far in (18, 22, 24, 25, 26, 28):
        p = value_pool(D, bits, gs, far, shape, counts == FEW)
        for window in (1, 24):
            say("small values", counts, D, gs, bits, shape, far, window)
            got = O.bf16_to_f32(run_paged(T, p, q, starts, D ** -0.5, window))
            for i, n in enumerate(LENS):
                a, e = int(starts[i]), int(starts[i + 1])
                (k, _), (v, most) = stored(p, i, n, 0), stored(p, i, n, 1)
                near = most.max() < 2.0 ** 28 * most[most > 0].min()
                f = O.bf16_to_f32(q[a:e]).astype(np.float64)
                at = np.arange(n - (e - a), n)
                # (Half a step is 2^-11: of a value, and of a weight; keys alike.)
                want, tol = R.attend(f, k, v, at, D ** -0.5, True, window, None, 2.0 ** -11 + 2.0 ** -24,
                                     2.0 ** -24 if near else 2.0 ** -8, 2.0 ** -11 if near else 2.0 ** -8)
                assert 0.0 < np.abs(want[0]).max() < 8.0  # no share of the large ones
                some, _ = R.attend(f, k, 1.5 * 2.0 ** -11 * most, at, D ** -0.5, True, window)
                tol += 1.01 * some
                if near:  # in place of the head's largest's share of it
                    tol -= 2.0 ** -39 * np.abs(v).max()
                assert tol.min() > 0.0
                R.check(got[a:e], want, tol, f"small values {far} {window}")


@pytest.mark.parametrize("counts", [FEW, MANY])
@pytest.mark.parametrize("D,gs", [(64, 32), (128, 64), (256, 128), (512, 32)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("far", [16, 20, 24, 32, 60])
def test_keys_of_small_groups_keep_their_bits(T, counts, D, gs, bits, far):
    """Every seventh key's first group is 2^far times larger than all others, and
    the queries' channels there are zero: the scores are those of the other
    groups. Where f16's steps could move them by 2^-10 they are f32's, with
    nothing lost to the large ones."""
    say("small keys", counts, D, gs, bits, far)
    p = Paged(LENS, 1, D, 16, AFFINE, bits, 8, gs, seed=5)
    rng = np.random.default_rng(D + bits)
    for b, n in enumerate(LENS):
        for row in range(n):
            k, v = rng.standard_normal((2, 1, D))
            if row % 7 == 3:
                k[:, :gs] *= 2.0 ** far
            p.write(b, row, bf16(k), bf16(v))
    x = rng.standard_normal((sum(counts), 2, D))
    x[..., :gs] = 0.0
    q = bf16(x)
    starts = starts_of(counts)
    scale = 2.0 * D ** -0.5  # scores of a few units
    got = O.bf16_to_f32(run_paged(T, p, q, starts, scale))
    want, tol = R.paged(p, q, starts, scale)
    # f16's steps in a score: D channels below 2^15 times half of 2^-24, in units
    # in which the largest channels of the query and of the key are below 2^15.
    # Where that is 2^-10 or more, it is f32 that the tolerance counts.
    step = D * 2.0 ** 15 * 2.0 ** -25 * scale * np.log2(np.e) / 2.0 ** 30
    qf = np.abs(O.bf16_to_f32(q)).max(-1)
    for i, n in enumerate(LENS):
        a, e = int(starts[i]), int(starts[i + 1])
        k, v = (stored(p, i, n, side)[0] for side in range(2))
        if step * qf[a:e].min() * np.abs(k).max() < 2.0 ** -10:
            continue
        f = O.bf16_to_f32(q[a:e]).astype(np.float64)
        want[a:e], tol[a:e] = R.attend(f, k, v, np.arange(n - (e - a), n), scale, off_v=2.0 ** -11 + 2.0 ** -24, off_w=2.0 ** -11)
    assert far < 32 or tol.max() < 0.2
    R.check(got, want, tol, f"small keys {far}")


@pytest.mark.parametrize("counts", [[3, 2], MANY])
@pytest.mark.parametrize("D,gs", [(64, 32), (128, 64), (256, 128), (512, 32)])
@pytest.mark.parametrize("bits", [4, 8])
def test_groups_of_zeros_cost_the_others_nothing(T, counts, D, gs, bits):
    """The quantizer stores a group of zeros as a scale of -1e-7 (its least) with
    codes and bias of zero: beside values of 20,000 the results are those, bit
    for bit, of a scale of zero, of which nothing could be lost."""
    say("zeros", counts, D, gs, bits)
    p = Paged(LENS, 1, D, 16, AFFINE, 4, bits, gs, seed=5)
    rng = np.random.default_rng(D + bits)
    for b, n in enumerate(LENS):
        for row in range(n):
            k, v = rng.standard_normal((2, 1, D))
            v *= 20000.0
            if row % 5 == 2:
                v[:, :gs] = 0.0
            if row % 11 == 4:
                v[:] = 0.0
            p.write(b, row, bf16(k), bf16(v))
    q = kv_bf16((sum(counts), 2, D), D)
    starts = starts_of(counts)
    want, tol = R.paged(p, q, starts, D ** -0.5)
    first = run_paged(T, p, q, starts, D ** -0.5)
    R.check(O.bf16_to_f32(first), want, tol, "zeros")
    _, scales, biases = p.sides[1]
    none = (biases == 0) & (np.abs(O.bf16_to_f32(scales)) < 1e-6)
    assert none.sum() >= 40 and not codes_of(p.sides[1][0], bits).reshape(*none.shape, gs)[none].any()
    scales[none] = 0
    assert np.array_equal(run_paged(T, p, q, starts, D ** -0.5), first)
