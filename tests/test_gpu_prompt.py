"""Attention of packed sequences on the GPU, over their own tokens and over the
paged cache, against 64 bits; and the paged cache's calls as a server makes
them, one after the other."""
import ctypes

import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, GUARD, Paged
from paged_ref import check as check_decode
from test_gpu_capture import captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


def say(*a):
    print("[prompt]", *a, flush=True)


def poisoned(T, need):
    """A workspace: whatever it holds before the call is no answer."""
    return T.DeviceArray((max(need, 16),), np.uint8, np.full((max(need, 16),), 0xFF, np.uint8))


def run_packed(T, x, H, Hkv, starts, scale, causal=True, window=-1, pad=0, workspace=True, stream=None):
    """x bf16 [tokens, H + 2 Hkv, D], a fused projection; starts may leave tokens out at both ends."""
    n, _, D = x.shape
    width = x.shape[1] * D + pad
    buf = np.full((n, width), GUARD, np.uint16)
    buf[:, :x.shape[1] * D] = x.reshape(n, -1)
    dbuf, ds = T.DeviceArray.of(buf), T.DeviceArray.of(np.asarray(starts, np.int32))
    out = T.DeviceArray((n, H, D), np.uint16, np.full((n, H, D), GUARD, np.uint16))
    B = len(starts) - 1
    need = T.packed_attend_workspace_size(B, H, Hkv, D, n)
    ws = poisoned(T, need) if workspace else None
    k = dbuf.ptr + 2 * H * D
    T.packed_attend(dbuf.ptr, width, k, k + 2 * Hkv * D, width, D, B, H, Hkv, D, ds.ptr, n, scale, out.ptr, causal, window,
                    ws.ptr if ws else None, need if ws else 0, stream)
    T.hip().sync()
    return out.numpy()


def run_paged(T, p, q, starts, scale, window=-1, max_rows=None, pad=0, workspace=True, d=None):
    n, H, D = q.shape
    d = d or p.device(T)
    kv = d.view()
    buf = np.full((n, H * D + pad), GUARD, np.uint16)
    buf[:, :H * D] = q.reshape(n, -1)
    dq, ds = T.DeviceArray.of(buf), T.DeviceArray.of(np.asarray(starts, np.int32))
    out = T.DeviceArray((n, H, D), np.uint16, np.full((n, H, D), GUARD, np.uint16))
    most = max_rows or p.stride * p.R
    need = T.paged_prefill_workspace_size(kv, H, n, most)
    ws = poisoned(T, need) if workspace else None
    T.paged_prefill_attend(kv, dq.ptr, H * D + pad, H, ds.ptr, n, scale, most, out.ptr, window, ws.ptr if ws else None,
                           need if ws else 0)
    T.hip().sync()
    return out.numpy()


def starts_of(counts, gap=0):
    return np.concatenate([[gap], gap + np.cumsum(counts)]).astype(np.int32)


def close(got, want, tol, starts, tag):
    a, b = int(starts[0]), int(starts[-1])
    assert np.all(got[:a] == GUARD) and np.all(got[b:] == GUARD), "rows outside the sequences"
    R.check(O.bf16_to_f32(got[a:b]), want[a:b], tol[a:b], tag)


# ------------------------------------------------------------------- packed
PACKED = [
    # D, Hkv, G, counts, causal, window
    (128, 1, 1, [1], True, -1),
    (128, 2, 4, [1, 0, 2, 63, 64, 65, 7], True, -1),
    (128, 1, 3, [130, 257, 16], True, -1),
    (128, 1, 8, [333], False, -1),
    (128, 2, 5, [200, 31], True, 1),
    (128, 1, 2, [500, 3], True, 100),
    (128, 1, 32, [40, 9], True, -1),
    (128, 1, 1, [1500], True, -1),
    (64, 3, 1, [90, 0, 0, 128, 1], True, -1),
    (64, 1, 7, [150, 66], False, -1),
    (64, 2, 2, [700], True, 64),
    (256, 1, 2, [100, 65, 1], True, -1),
    (256, 2, 1, [300], True, 17),
    (256, 1, 4, [77], False, -1),
    (512, 1, 4, [70, 1, 33], True, -1),
    (512, 2, 16, [40], True, 9),
    (512, 1, 1, [260], False, -1),
]


@pytest.mark.parametrize("D,Hkv,G,counts,causal,window", PACKED)
@pytest.mark.parametrize("loose", [False, True])
def test_packed(T, D, Hkv, G, counts, causal, window, loose):
    """loose: tokens before and behind the sequences, padded rows, no workspace."""
    say("packed", D, Hkv, G, counts, causal, window, loose)
    gap = 5 * loose
    starts = starts_of(counts, gap)
    n, H = int(starts[-1]) + 3 * loose, G * Hkv
    x = kv_bf16((n, H + 2 * Hkv, D), D + sum(counts), frac=0.02, mult=4.0)
    got = run_packed(T, x, H, Hkv, starts, D ** -0.5, causal, window, 8 * loose, not loose)
    want, tol = R.packed(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], starts, D ** -0.5, causal, window)
    close(got, want, tol, starts, "packed")


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_packed_scales(T, D, scale):
    say("scale", D, scale)
    x = kv_bf16((150, 4, D), D)
    starts = starts_of([100, 50])
    want, tol = R.packed(x[:, :2], x[:, 2:3], x[:, 3:], starts, scale)
    close(run_packed(T, x, 2, 1, starts, scale), want, tol, starts, "scale")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_packed_many_sequences(T, D):
    rng = np.random.default_rng(D)
    counts = rng.integers(0, 9, 1024)
    say("many", D, counts.sum())
    starts = starts_of(counts, 2)
    x = kv_bf16((int(starts[-1]) + 1, 4, D), D)
    want, tol = R.packed(x[:, :2], x[:, 2:3], x[:, 3:], starts, D ** -0.5)
    close(run_packed(T, x, 2, 1, starts, D ** -0.5), want, tol, starts, "many")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_scores_that_leave_one_key_and_that_grow(T, D):
    """Scores that rise with the key (the running maximum moves in every tile)
    and large ones that one key takes whole."""
    say("rising", D)
    n = 400
    x = kv_bf16((n, 3, D), D)
    q, k = O.bf16_to_f32(x[:, 0]).copy(), O.bf16_to_f32(x[:, 1]).copy()
    q[:, 0], k[:, 0] = 8.0, np.arange(n) * 0.5
    x[:, 0], x[:, 1] = O.bf16_from_f32(q), O.bf16_from_f32(k)
    starts = starts_of([n])
    for scale in (0.05, 1.0):
        want, tol = R.packed(x[:, :1], x[:, 1:2], x[:, 2:], starts, scale)
        close(run_packed(T, x, 1, 1, starts, scale), want, tol, starts, "rising")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("size", [1e36, 1e-36])
def test_values_keep_their_range(T, D, size):
    say("range", D, size)
    x = kv_bf16((90, 3, D), D)
    x[:, 2] = O.bf16_from_f32(O.bf16_to_f32(x[:, 2]) * np.float32(size))
    x[:, 2, :4] = kv_bf16((90, 4), 1)  # channels of ordinary size beside them
    starts = starts_of([90])
    want, tol = R.packed(x[:, :1], x[:, 1:2], x[:, 2:], starts, D ** -0.5)
    close(run_packed(T, x, 1, 1, starts, D ** -0.5), want, tol, starts, "range")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("what", ["v inf", "v nan", "k nan", "k inf"])
def test_what_later_keys_hold_reaches_no_earlier_query(T, D, what):
    """Token 70 of 200 holds infinities or NaN: queries before it, and those of
    another sequence, are as without it; those that see it are not finite there."""
    say("later", D, what)
    x = kv_bf16((260, 4, D), D)
    starts = starts_of([200, 60])
    want, tol = R.packed(x[:, :2], x[:, 2:3], x[:, 3:], starts, D ** -0.5)
    bad = 0x7F80 if "inf" in what else 0x7FC0
    if what[0] == "v":
        x[70, 3, 5], x[70, 3, D - 1] = bad, bad
    else:
        x[70, 2] = bad
    got = O.bf16_to_f32(run_packed(T, x, 2, 1, starts, D ** -0.5))
    rows = np.r_[0:70, 200:260]
    R.check(got[rows], want[rows], tol[rows], what)
    after = got[70:200]
    if what == "v inf":
        assert np.all(after[:, :, [5, D - 1]] == np.inf)
    elif what[0] == "v":
        assert np.all(np.isnan(after[:, :, [5, D - 1]]))
    if what[0] == "v":
        rest = np.delete(np.arange(D), [5, D - 1])
        R.check(after[:, :, rest], want[70:200][:, :, rest], tol[70:200][:, :, rest], what)
    elif what == "k nan":
        assert np.all(np.isnan(after))


# -------------------------------------------------------------------- paged
PAGED = [
    # kind, bk, bv, gs, D, R, Hkv, G, lens, counts, window
    (BF16, 16, 16, 64, 128, 16, 2, 4, [5, 40, 0, 133], [5, 17, 0, 1], -1),
    (BF16, 16, 16, 64, 128, 64, 1, 1, [1000], [300], -1),
    (BF16, 16, 16, 64, 128, 16, 1, 4, [777, 90, 4000], [6, 6, 6], -1),
    (BF16, 16, 16, 64, 128, 256, 1, 7, [300, 65], [64, 65], 40),
    (BF16, 16, 16, 64, 64, 32, 2, 2, [513, 64, 1], [129, 64, 1], -1),
    (BF16, 16, 16, 64, 64, 16, 1, 16, [2000], [3], 900),
    (BF16, 16, 16, 64, 256, 128, 1, 2, [260, 31], [70, 31], -1),
    (BF16, 16, 16, 64, 256, 16, 1, 1, [1500, 3], [2, 3], 64),
    (BF16, 16, 16, 64, 512, 32, 1, 16, [150, 64], [20, 1], -1),
    (BF16, 16, 16, 64, 512, 64, 2, 1, [700], [100], 33),
    (AFFINE, 4, 4, 64, 128, 16, 2, 4, [5, 40, 0, 133], [5, 17, 0, 1], -1),
    (AFFINE, 4, 4, 64, 128, 64, 1, 2, [1900], [260], -1),
    (AFFINE, 8, 4, 32, 128, 32, 1, 1, [444, 3], [5, 2], 70),
    (AFFINE, 8, 8, 32, 64, 16, 1, 3, [222, 100], [222, 4], -1),
    (AFFINE, 4, 8, 64, 64, 256, 1, 1, [3000], [2], -1),
    (AFFINE, 8, 8, 32, 256, 64, 1, 2, [400, 64], [90, 8], 128),
    (AFFINE, 4, 4, 128, 256, 16, 1, 4, [130], [130], -1),
    (AFFINE, 4, 8, 128, 512, 128, 1, 4, [200, 70], [30, 3], -1),
    (AFFINE, 8, 8, 64, 512, 16, 1, 8, [90], [90], 20),
]


@pytest.mark.parametrize("kind,bk,bv,gs,D,R_,Hkv,G,lens,counts,window", PAGED)
@pytest.mark.parametrize("loose", [False, True])
def test_paged(T, kind, bk, bv, gs, D, R_, Hkv, G, lens, counts, window, loose):
    say("paged", kind, bk, bv, gs, D, R_, Hkv, G, lens, counts, window, loose)
    p = Paged(lens, Hkv, D, R_, kind, bk, bv, gs, spare=2, seed=D + R_).fill(D + sum(lens))
    starts = starts_of(counts, 3 * loose)
    q = kv_bf16((int(starts[-1]) + 2 * loose, G * Hkv, D), 7 * D)
    got = run_paged(T, p, q, starts, D ** -0.5, window, None, 8 * loose, not loose)
    want, tol = R.paged(p, q, starts, D ** -0.5, window)
    close(got, want, tol, starts, "paged")


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_paged_edges(T, kind, D):
    """More queries than rows (the first see none), lengths out of range, a
    bound below the length, pages that are none, among them whole sequences'."""
    say("edges", kind, D)
    gs = 32
    p = Paged([100, 3, -2, 1 << 30, 70, 64], 1, D, 16, kind, 4, 8, gs, stride=12, spare=1, seed=4).fill(3)
    p.table[0, 2], p.table[0, 5] = -1, p.pages
    p.table[4] = 2 ** 31 - 1
    counts = [20, 9, 4, 30, 5, 64]
    starts = starts_of(counts, 1)
    q = kv_bf16((int(starts[-1]) + 1, 2, D), D)
    for most in (None, 50):
        want, tol = R.paged(p, q, starts, D ** -0.5, max_rows=most)
        close(run_paged(T, p, q, starts, D ** -0.5, max_rows=most), want, tol, starts, "edges")
        assert np.all(want[starts[1]:starts[1] + 6] == 0.0)


@pytest.mark.parametrize("kind,bk,bv", [(BF16, 16, 16), (AFFINE, 4, 8), (AFFINE, 8, 4)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_few_rows_edges(T, kind, bk, bv, D):
    """The same with few queries a sequence, which another kernel takes; one of
    the sequences has many all the same."""
    say("few edges", kind, bk, bv, D)
    p = Paged([100, 3, -2, 1 << 30, 70, 64, 9, 190], 1, D, 16, kind, bk, bv, 32, stride=12, spare=1, seed=4).fill(3)
    p.table[0, 2], p.table[0, 5] = -1, p.pages
    p.table[4] = 2 ** 31 - 1
    counts = [2, 5, 1, 3, 1, 1, 0, 25]
    starts = starts_of(counts, 1)
    q = kv_bf16((int(starts[-1]) + 1, 2, D), D)
    for most, window in ((None, -1), (50, -1), (None, 7)):
        want, tol = R.paged(p, q, starts, D ** -0.5, window, max_rows=most)
        close(run_paged(T, p, q, starts, D ** -0.5, window, max_rows=most), want, tol, starts, "few edges")
        assert np.all(want[starts[1]:starts[1] + 2] == 0.0)


@pytest.mark.parametrize("counts", [[2, 3], [150, 90]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_affine_scales(T, D, counts, scale):
    say("affine scales", D, counts, scale)
    p = Paged([200, 90], 1, D, 16, AFFINE, 8, 8, 64, seed=5).fill(3)
    q = kv_bf16((sum(counts), 2, D), D)
    want, tol = R.paged(p, q, starts_of(counts), scale)
    close(run_paged(T, p, q, starts_of(counts), scale), want, tol, starts_of(counts), "affine scales")


@pytest.mark.parametrize("counts", [[2, 3], [150, 90]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("kq,ks,vs", [(1e18, 1e-18, 1e36), (1e-18, 1e18, 1e-34), (1e-3, 1.0, 1e5)])
def test_affine_ranges(T, D, counts, kq, ks, vs):
    """Keys and values of any magnitude, the queries to match; a few keys much
    smaller than the others."""
    say("affine ranges", D, counts, kq, ks, vs)
    p = Paged([200, 90], 1, D, 16, AFFINE, 4, 8, 32, seed=5)
    rng = np.random.default_rng(D)
    for b in range(2):
        for row in range(int(p.lens[b])):
            small = 2.0 ** -6 if row % 7 == 3 else 1.0
            k, v = (O.bf16_from_f32((rng.standard_normal((1, D)) * m).astype(np.float32)) for m in (ks * small, vs))
            p.write(b, row, k, v)
    q = O.bf16_from_f32((rng.standard_normal((sum(counts), 2, D)) * kq).astype(np.float32))
    scale = D ** -0.5 / float(np.float32(kq * ks))
    want, tol = R.paged(p, q, starts_of(counts), scale)
    close(run_paged(T, p, q, starts_of(counts), scale), want, tol, starts_of(counts), "affine ranges")


@pytest.mark.parametrize("counts", [[3, 3], [150, 90]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_affine_values_far_apart(T, D, counts):
    """The last rows' values are 2^60 times larger than the others': queries
    that see the small ones alone keep them."""
    say("far apart", D, counts)
    p = Paged([150, 90], 1, D, 16, AFFINE, 8, 8, 32, seed=5)
    rng = np.random.default_rng(D)
    small = [147 if counts[0] == 3 else 60, 87 if counts[0] == 3 else 40]
    for b in range(2):
        for row in range(int(p.lens[b])):
            k, v = (O.bf16_from_f32((rng.standard_normal((1, D)) * m).astype(np.float32)) for m in (1.0, 1.0 if row <= small[b] else 2.0 ** 60))
            p.write(b, row, k, v)
    q = kv_bf16((sum(counts), 2, D), D)
    starts = starts_of(counts)
    want, tol = R.paged(p, q, starts, D ** -0.5)
    assert 0 < np.abs(want[0]).max() < 8.0 and tol[0].max() < 1.0  # no share of the large ones
    close(run_paged(T, p, q, starts, D ** -0.5), want, tol, starts, "far apart")


@pytest.mark.parametrize("counts", [[3, 3], [150, 90]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("large", [2.0 ** 60, np.inf])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 18])
def test_affine_keys_far_apart(T, D, counts, large, size):
    """The last row's key is far larger than the others', or infinite: queries
    before it are as with an ordinary one there, bounds included."""
    say("keys far apart", D, counts, large, size)
    pools = []
    for top in (1.0, large):
        p = Paged([150, 90], 1, D, 16, AFFINE, 8, 8, 32, seed=5)
        rng = np.random.default_rng(D)
        for b in range(2):
            n = int(p.lens[b])
            for row in range(n):
                k, v = (rng.standard_normal((1, D)).astype(np.float32) for _ in range(2))
                last = row == n - 1
                k *= 2.0 ** 60 if last and top != 1.0 else size
                p.write(b, row, O.bf16_from_f32(k), O.bf16_from_f32(v))
            if top == np.inf:
                p.sides[0][1][p.table[b, (n - 1) // 16], 0, (n - 1) % 16] = 0x7F80  # its scales
        pools.append(p)
    q = O.bf16_from_f32(np.random.default_rng(D + 1).standard_normal((sum(counts), 2, D)).astype(np.float32) / np.float32(size))
    starts = starts_of(counts)
    want, tol = R.paged(pools[0], q, starts, D ** -0.5)
    got = O.bf16_to_f32(run_paged(T, pools[1], q, starts, D ** -0.5)[:sum(counts)])
    before = np.ones(sum(counts), bool)
    before[starts[1:] - 1] = False
    R.check(got[before], want[before], tol[before], "keys far apart")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("few", [False, True])
def test_values_next_to_the_largest(T, D, few):
    """Sums of values that pass f32 where their mean does not."""
    say("largest", D, few)
    p = Paged([70], 1, D, 16, BF16, seed=5).fill(2)
    top = O.bf16_from_f32(np.array([3.3e38], np.float32))[0]
    p.sides[1][0][..., 7] = np.where(p.sides[1][0][..., 7] == GUARD, GUARD, top)
    counts = [3] if few else [70]
    q = kv_bf16((counts[0], 2, D), D)
    starts = starts_of(counts)
    want, tol = R.paged(p, q, starts, D ** -0.5)
    assert want[..., 7].min() > 3.2e38
    # The result may round up to the type's infinity: half a step below it does not.
    close(run_paged(T, p, q, starts, D ** -0.5), want, tol, starts, "largest")


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("counts", [[6], [90]])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("what", ["v", "k"])
def test_pages_with_infinities_and_nan(T, kind, D, counts, what):
    """A later row's value (or key) is not finite: earlier queries are as
    without it, and channels (queries) that it reaches are not finite."""
    say("not finite", kind, D, counts, what)
    n = 200
    p = Paged([n], 1, D, 16, kind, 8, 8, 32, seed=5).fill(4)
    starts = starts_of(counts)
    q = kv_bf16((counts[0], 2, D), 3)
    want, tol = R.paged(p, q, starts, D ** -0.5)
    at = (p.table[0, (n - 4) // 16], 0, (n - 4) % 16)  # seen by the last four queries
    side = p.sides[1 if what == "v" else 0]
    if kind == BF16:
        side[0][at][3] = 0x7F80 if what == "v" else 0x7FC0
        reached = [3]
    else:
        side[1][at][0] = 0x7FC0  # a group's scale
        reached = list(range(32))
    got = O.bf16_to_f32(run_paged(T, p, q, starts, D ** -0.5))
    m = counts[0] - 4
    R.check(got[:m], want[:m], tol[:m], "before")
    if what == "v":
        assert not np.any(np.isfinite(got[m:][..., reached]))
        rest = np.setdiff1d(np.arange(D), reached)
        R.check(got[m:][..., rest], want[m:][..., rest], tol[m:][..., rest], "beside")
    else:
        assert np.all(np.isnan(got[m:]))


@pytest.mark.parametrize("kind,D,R_", [(BF16, 128, 16), (AFFINE, 128, 64), (BF16, 64, 128), (BF16, 256, 32), (AFFINE, 512, 16)])
@pytest.mark.parametrize("counts", [[1, 1], [5, 2], [40, 7]])
def test_paged_long(T, kind, D, R_, counts):
    """Few queries over many rows: the keys are divided."""
    say("long", kind, D, R_, counts)
    p = Paged([9001, 2500], 1, D, R_, kind, 4, 4, 32, seed=6).fill(1)
    starts = starts_of(counts)
    q = kv_bf16((sum(counts), 4, D), D)
    for window in (-1, 3000):
        want, tol = R.paged(p, q, starts, D ** -0.5, window)
        close(run_paged(T, p, q, starts, D ** -0.5, window), want, tol, starts, "long")


def test_one_query_is_the_decode_attention(T):
    """A count of one a sequence: both calls agree with 64 bits."""
    p = Paged([900, 17, 300], 2, 128, 16, BF16, seed=6).fill(1)
    q = kv_bf16((3, 8, 128), 5)
    d = p.device(T)
    got = run_paged(T, p, q, starts_of([1, 1, 1]), 128 ** -0.5, d=d)
    out, tol, _, _ = p.attend(q, 128 ** -0.5)
    check_decode(O.bf16_to_f32(d.attend(q, 128 ** -0.5)), out, tol, "decode")
    want, tol = R.paged(p, q, starts_of([1, 1, 1]), 128 ** -0.5)
    R.check(O.bf16_to_f32(got), want, tol, "prefill")


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_same_bits_every_run_and_shared_pages(T, kind):
    p = Paged([640, 640, 80], 2, 128, 16, kind, 4, 4, 64, seed=6).fill(1)
    p.table[1, :20] = p.table[0, :20]  # a common prompt
    q = kv_bf16((30, 8, 128), 5)
    starts = starts_of([10, 10, 10])
    d = p.device(T)
    first = run_paged(T, p, q, starts, 128 ** -0.5, d=d)
    want, tol = R.paged(p, q, starts, 128 ** -0.5)
    close(first, want, tol, starts, "shared pages")
    for i in range(3):
        assert np.array_equal(run_paged(T, p, q, starts, 128 ** -0.5, d=d, workspace=i == 1), first)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_captured_prefill_follows_starts_and_lengths(T, kind):
    D, H, n, B = 128, 4, 96, 3
    p = Paged([700, 64, 300], 1, D, 16, kind, 4, 4, 64, stride=50, seed=2).fill(1)
    d = p.device(T)
    dq, ds = T.DeviceArray((n, H, D), np.uint16), T.DeviceArray((B + 1,), np.int32)
    out = T.DeviceArray((n, H, D), np.uint16)
    need = T.paged_prefill_workspace_size(d.view(), H, n, 800)
    ws = poisoned(T, need)
    q = kv_bf16((n, H, D), 8)
    T.hip().copy_in(dq.ptr, q)

    def call(stream):
        T.paged_prefill_attend(d.view(), dq.ptr, H * D, H, ds.ptr, n, D ** -0.5, 800, out.ptr, -1, ws.ptr, need, stream)

    with captured(T, call) as launch:
        for lens, counts in [([700, 64, 300], [6, 64, 1]), ([650, 10, 0], [90, 3, 0]), ([1, 1, 1], [1, 1, 1]), ([700, 64, 300], [6, 64, 1])]:
            p.lens = np.array(lens, np.int32)
            starts = starts_of(counts)
            T.hip().copy_in(d.lens.ptr, p.lens)
            T.hip().copy_in(ds.ptr, starts)
            T.hip().copy_in(out.ptr, np.full((n, H, D), GUARD, np.uint16))
            launch()
            got = out.numpy()
            want, tol = R.paged(p, q, starts, D ** -0.5)
            close(got, want, tol, starts, "captured")
            assert np.array_equal(run_paged(T, p, q, starts, D ** -0.5, max_rows=800, d=d), got)


def test_captured_without_a_workspace_size_to_grow(T):
    """No workspace under a capture: the library's scratch that is there, grown before."""
    x = kv_bf16((70, 4, 128), 2)
    starts = starts_of([50, 20])
    want = run_packed(T, x, 2, 1, starts, 0.1, workspace=False)
    dbuf, ds = T.DeviceArray.of(x), T.DeviceArray.of(starts)
    out = T.DeviceArray((70, 2, 128), np.uint16)
    k = dbuf.ptr + 2 * 2 * 128

    def call(stream):
        T.packed_attend(dbuf.ptr, 512, k, k + 256, 512, 128, 2, 2, 1, 128, ds.ptr, 70, 0.1, out.ptr, True, -1, None, 0, stream)

    with captured(T, call) as launch:
        for i in range(3):
            T.hip().copy_in(out.ptr, np.full((70, 2, 128), GUARD, np.uint16))
            launch()
            assert np.array_equal(out.numpy(), want)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("counts", [[3, 2], [150, 90]])
def test_pages_past_32_bits(T, kind, counts):
    """The same pages behind the first 2^32 bytes (and 2^31 elements) of a pool:
    what the append writes there and the attention reads are the near ones' bits."""
    say("far pages", kind, counts)
    D, R_, Hkv, H = 512, 256, 4, 4
    p = Paged([300, 200], Hkv, D, R_, kind, 8, 8, 64, seed=5).fill(2)
    near = p.device(T)
    page = p.sides[0][0][0].nbytes
    far = (1 << 32) // page + 3  # bf16: 2^31 elements too
    sides, big = [], []
    for side in p.sides:
        for x in side:
            big.append(T.DeviceArray(((far + p.pages) * x[0].nbytes,), np.uint8))
            T.hip().copy_in(big[-1].ptr + far * x[0].nbytes, x)
            sides.append(big[-1].ptr)
    table = T.DeviceArray.of(np.where(p.table >= 0, p.table + far, -1).astype(np.int32))
    view = near.view(num_pages=far + p.pages, slots=sides, table=table.ptr)
    n, width = sum(counts), (H + 2 * Hkv) * D
    x = kv_bf16((n, width), 7)
    dx, ds = T.DeviceArray.of(x), T.DeviceArray.of(starts_of(counts))
    turns, m = T.rope_turns(128)
    dt = T.DeviceArray.of(np.array(turns, np.uint64))
    k = dx.ptr + 2 * H * D
    slots = np.array([[p.table[b, row // R_], row % R_, row, b] for b, c in enumerate(counts)
                      for row in range(int(p.lens[b]) - c, int(p.lens[b]))], np.int32)
    outs = []
    for kv, first in ((near.view(), 0), (view, far)):
        s = slots.copy()
        s[:, 0] += first
        dsl, q, out = T.DeviceArray.of(s), T.DeviceArray((n, H, D), np.uint16), T.DeviceArray((n, H, D), np.uint16)
        T.paged_append_rope(kv, T.rope(128, 0, m, dt.ptr), dx.ptr, H, width, q.ptr, H * D, k, k + 2 * Hkv * D, width, D, dsl.ptr, n)
        T.paged_prefill_attend(kv, q.ptr, H * D, H, ds.ptr, n, D ** -0.5, 512, out.ptr)
        T.hip().sync()
        outs.append(out.numpy())
    assert np.array_equal(*outs)
    for t, b, x in zip([t for side in near.sides for t in side], big, [x for side in p.sides for x in side]):
        assert np.array_equal(t.numpy(), T.hip().download(b.ptr + far * x[0].nbytes, x.shape, x.dtype))


def test_two_streams_at_once(T):
    """Calls on two streams with workspaces of their own, queued together."""
    D, H = 128, 8
    pools = [Paged([1500, 700], 2, D, 16, AFFINE, 4, 8, 64, seed=s).fill(s) for s in (1, 2)]
    counts = [600, 700]
    q = kv_bf16((sum(counts), H, D), 3)
    starts = starts_of(counts)
    alone = [run_paged(T, p, q, starts, D ** -0.5) for p in pools]
    dq, ds = T.DeviceArray.of(q), T.DeviceArray.of(starts)
    on = [p.device(T) for p in pools]
    most = pools[0].stride * 16
    need = T.paged_prefill_workspace_size(on[0].view(), H, sum(counts), most)
    ws = [poisoned(T, need) for _ in on]
    outs = [T.DeviceArray((sum(counts), H, D), np.uint16) for _ in on]
    T.hip().sync()
    streams = [T.hip().stream() for _ in on]
    for _ in range(3):
        for d, w, out, s in zip(on, ws, outs, streams):
            T.paged_prefill_attend(d.view(), dq.ptr, H * D, H, ds.ptr, sum(counts), D ** -0.5, most, out.ptr, -1, w.ptr, need, s)
    T.hip().sync()
    for s in streams:
        T.hip().h.hipStreamDestroy(ctypes.c_void_p(s))
    for out, want in zip(outs, alone):
        assert np.array_equal(out.numpy(), want)


# ------------------------------------------------------------ as a server does
@pytest.mark.parametrize("kind,D,rd,interleaved", [(BF16, 128, 128, False), (AFFINE, 128, 64, True), (BF16, 64, 22, False),
                                                   (AFFINE, 256, 256, False), (AFFINE, 512, 128, True)])
def test_prompts_steps_and_endings(T, kind, D, rd, interleaved):
    """Pages reserved, queries and keys rotated into them, prompts attended in
    chunks, single tokens decoded, a rejected draft taken back, sequences ended
    and others admitted: every call's result against 64 bits."""
    say("server", kind, D, rd)
    B, Hkv, G, R_, width, pages = 4, 1, 2, 16, 12, 30
    H = Hkv * G
    p = Paged([0] * B, Hkv, D, R_, kind, 4, 8, 32, stride=width, spare=pages - 1, seed=1)
    assert p.pages == pages - 1
    t = R.Tables([0] * B, R_, width, p.pages, seed=3)
    p.table, p.lens = t.table, t.lens
    d = p.device(T)
    free, count = T.DeviceArray.of(t.free), T.DeviceArray.of(np.array([t.count], np.int32))
    tables = T.page_tables(B, R_, p.pages, d.table.ptr, width, d.lens.ptr, free.ptr, count.ptr)
    turns, m = T.rope_turns(rd, 10000.0, T.ROPE_LINEAR, 2.0)
    dturns = T.DeviceArray.of(np.array(turns, np.uint64))
    rope = T.rope(rd, interleaved, m, dturns.ptr)
    theta, _ = R.thetas(rd, 10000.0, 1, 2.0)
    scale = D ** -0.5
    rounds = [([70, 0, 20, 33], None), ([30, 5, 1, 1], None), ([1, 1, 1, 1], None), ([4, 1, 0, 1], None),
              ([0, 0, 0, 0], [101, 1 << 30, 1 << 30, 0]), ([1, 1, 1, 90], None), ([1, 1, 1, 1], None)]
    for i, (counts, keep) in enumerate(rounds):
        if keep is not None:
            dk = T.DeviceArray.of(np.array(keep, np.int32))
            T.paged_release(tables, dk.ptr)
            T.hip().sync()
            t.release(keep)
            assert np.array_equal(d.table.numpy(), t.table) and np.array_equal(d.lens.numpy(), t.lens)
        n = sum(counts)
        if n == 0:
            continue
        dc = T.DeviceArray.of(np.array(counts, np.int32))
        starts, granted, slots = T.DeviceArray((B + 1,), np.int32), T.DeviceArray((B,), np.int32), T.DeviceArray((n, 4), np.int32)
        T.paged_reserve(tables, dc.ptr, n, starts.ptr, granted.ptr, slots.ptr)
        hs, hg, hslots = t.reserve(counts, n)
        assert np.array_equal(granted.numpy(), hg) and np.all(hg >= 0)
        x = kv_bf16((n, H + 2 * Hkv, D), 100 + i)
        dx = T.DeviceArray.of(x)
        q = T.DeviceArray((n, H, D), np.uint16)
        step = (H + 2 * Hkv) * D
        k = dx.ptr + 2 * H * D
        T.paged_append_rope(d.view(), rope, dx.ptr, H, step, q.ptr, H * D, k, k + 2 * Hkv * D, step, D, slots.ptr, n)
        out = T.DeviceArray((n, H, D), np.uint16)
        T.paged_prefill_attend(d.view(), q.ptr, H * D, H, starts.ptr, n, scale, width * R_, out.ptr)
        T.hip().sync()
        assert np.array_equal(slots.numpy(), hslots)
        assert np.array_equal(d.table.numpy(), t.table) and np.array_equal(d.lens.numpy(), t.lens)
        # The rotation, then from what the pool holds now.
        want, tol = R.rotated(x[:, :H], hslots[:, 2], theta, m, interleaved)
        R.check(O.bf16_to_f32(q.numpy()), want, tol, "queries")
        p.sides = d.host()
        want, tol = R.paged(p, q.numpy(), hs, scale)
        R.check(O.bf16_to_f32(out.numpy()), want, tol, "prefill")
        if all(c == 1 for c in counts):
            got = d.attend(q.numpy(), scale)
            want, tol, _, _ = p.attend(q.numpy(), scale)
            check_decode(O.bf16_to_f32(got), want, tol, "decode")
        if kind == BF16:
            for j, (page, row, position, b) in enumerate(hslots):
                assert np.array_equal(p.sides[1][0][page, :, row], x[j, H + Hkv:])
