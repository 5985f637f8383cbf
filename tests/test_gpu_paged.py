"""The paged cache on the GPU through the C ABI, against a 64-bit restatement of
its definitions (paged_ref.py): append, decode attention with and without
gathered weights, eviction, and the three in a loop."""
import ctypes

import numpy as np
import pytest

import oracle_lib as O
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged, check
from test_gpu_capture import captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


def say(*a):
    print("[paged]", *a, flush=True)


# ------------------------------------------------------------------- append
def append(T, p, counts, seed, heads_before=0, pad=0, gap=0):
    """lens already count the new rows: host and device appended, compared
    byte for byte, rows behind and pages beside included."""
    total = sum(counts)
    heads = heads_before + 2 * p.Hkv
    width = heads * p.D + pad
    buf = kv_bf16((gap + total + 3, width), seed, frac=0.02, mult=4.0)
    starts = np.cumsum([gap, *counts]).astype(np.int32)
    d = p.device(T)
    dbuf, dstarts = T.DeviceArray.of(buf), T.DeviceArray.of(starts)
    at = dbuf.ptr + 2 * heads_before * p.D
    T.paged_append(d.view(), at, at + 2 * p.Hkv * p.D, dstarts.ptr, gap + total + 3, width, p.D)
    T.hip().sync()
    for b, count in enumerate(counts):
        for j in range(count):
            x = buf[starts[b] + j, heads_before * p.D:heads * p.D].reshape(2, p.Hkv, p.D)
            p.write(b, int(p.lens[b]) - count + j, x[0], x[1])
    for got, want in zip(d.host(), p.sides):
        for g, w in zip(got, want):
            assert np.array_equal(g, w)
    if p.weights is not None:
        assert np.array_equal(d.weights.numpy(), p.weights)


APPENDS = [
    # kind, bits k/v, gs, D, R, Hkv, lens after, counts
    (BF16, 16, 16, 64, 128, 16, 3, [5, 40, 0, 33], [5, 17, 0, 33]),
    (BF16, 16, 16, 64, 64, 32, 1, [1], [1]),
    (BF16, 16, 16, 64, 256, 64, 8, [100, 64, 65], [36, 64, 1]),
    (BF16, 16, 16, 64, 512, 256, 2, [300, 7], [299, 0]),
    (AFFINE, 4, 4, 64, 128, 16, 3, [5, 40, 0, 33], [5, 17, 0, 33]),
    (AFFINE, 8, 8, 32, 64, 32, 1, [1, 31], [1, 30]),
    (AFFINE, 8, 4, 32, 256, 64, 5, [100, 64, 65], [36, 64, 1]),
    (AFFINE, 4, 8, 128, 512, 128, 2, [300, 7], [299, 0]),
    (AFFINE, 4, 4, 32, 512, 16, 1, [19], [19]),
    (AFFINE, 8, 8, 128, 128, 16, 7, [2, 3, 4], [1, 1, 1]),
]


@pytest.mark.parametrize("kind,bk,bv,gs,D,R,Hkv,lens,counts", APPENDS)
@pytest.mark.parametrize("strided", [False, True])
def test_append_writes_the_rows_and_nothing_else(T, kind, bk, bv, gs, D, R, Hkv, lens, counts,
                                                 strided):
    say("append", kind, bk, bv, gs, D, R, Hkv, lens, counts, strided)
    p = Paged(lens, Hkv, D, R, kind, bk, bv, gs, spare=2, seed=D + R, track=strided)
    if p.weights is not None:
        p.weights += 1.5
    append(T, p, counts, 3 * D + R, heads_before=2 * strided, pad=8 * strided, gap=2 * strided)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_append_skips_what_has_no_place(T, kind):
    """Rows below 0, past the table, on pages outside the pool."""
    p = Paged([40, 70, 50, 9], 2, 128, 16, kind, stride=4, spare=3, seed=5, track=True)
    p.weights += 2.0
    p.table[0, 1] = -1
    p.table[1, 3] = p.pages
    p.table[2, 0] = 0x7FFFFFFF
    p.table[2, 2] = -0x80000000
    say("append without a place", kind)
    append(T, p, [40, 20, 50, 12], 77)  # sequence 1 runs past 64 rows; 3 starts at row -3


def test_append_one_token_a_sequence_without_starts(T):
    for kind in (BF16, AFFINE):
        p = Paged([1, 17, 33], 4, 128, 16, kind, seed=9)
        say("append step", kind)
        x = kv_bf16((3, 8, 128), 4)
        d, dx = p.device(T), T.DeviceArray.of(x)
        T.paged_append(d.view(), dx.ptr, dx.ptr + 4 * 128 * 2, None, 3, 8 * 128, 128)
        T.hip().sync()
        for b in range(3):
            p.write(b, int(p.lens[b]) - 1, x[b, :4], x[b, 4:])
        for got, want in zip(d.host(), p.sides):
            for g, w in zip(got, want):
                assert np.array_equal(g, w)


# ------------------------------------------------------------------- attend
def attend(T, p, H, tag, window=-1, max_rows=None, scale=None, qmult=1.0):
    scale = p.D ** -0.5 if scale is None else scale
    q = O.bf16_from_f32(qmult * O.bf16_to_f32(kv_bf16((p.B, H, p.D), 11 * H + p.D)))
    out, tol, gain, gtol = p.attend(q, scale, window, max_rows)
    d = p.device(T)
    got = d.attend(q, scale, window, max_rows)
    check(O.bf16_to_f32(got), out, tol, tag)
    if p.weights is not None:
        w = d.weights.numpy()
        check(w, p.weights.astype(np.float64) + gain, gtol + 2.0 ** -23 * (p.weights + gain), tag + " weights")
        untouched = gain == 0
        assert np.array_equal(w[untouched], p.weights[untouched])
    return q, got, d


LAYOUTS = [
    # kind, bits k/v, gs
    (BF16, 16, 16, 64), (AFFINE, 4, 4, 64), (AFFINE, 8, 8, 32), (AFFINE, 8, 4, 64),
    (AFFINE, 4, 8, 32), (AFFINE, 4, 4, 128),
]


@pytest.mark.parametrize("kind,bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("R,H,Hkv", [(16, 6, 2), (64, 16, 1)])
def test_attend_matches_64_bits(T, kind, bk, bv, gs, D, R, H, Hkv):
    if gs > D:
        pytest.skip("a group is at most a row")
    say("attend", kind, bk, bv, gs, D, R, H, Hkv)
    p = Paged([1, 0, 300, 16, 33, 128], Hkv, D, R, kind, bk, bv, gs, spare=1, seed=D, track=R == 16)
    if p.weights is not None:
        p.weights += p.rng.random(p.weights.shape, np.float32)
    attend(T, p.fill(D + R), H, f"attend D={D}")


@pytest.mark.parametrize("G", [1, 2, 5, 15, 16, 17, 20, 32])
@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_group_sizes(T, G, kind):
    say("attend G", G, kind)
    p = Paged([77, 300], 2, 128, 32, kind, seed=G, track=G in (5, 17))
    attend(T, p.fill(G), 2 * G, f"G={G}")


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1000, 5003])
@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_lengths_of_one_sequence(T, n, kind):
    say("attend n", n, kind)
    p = Paged([n], 1, 128, 16, kind, seed=n, track=n % 2 == 1)
    attend(T, p.fill(n), 4, f"n={n}")


@pytest.mark.parametrize("kind,D,n,G", [(BF16, 64, 33001, 3), (BF16, 512, 20011, 2), (AFFINE, 128, 70007, 1),
                                        (AFFINE, 512, 12345, 17)])
def test_attend_one_sequence_over_the_whole_card(T, kind, D, n, G):
    """A KV head's rows in more parts than a wavefront has lanes."""
    say("attend long", kind, D, n, G)
    p = Paged([n], 1, D, 256, kind, seed=n, track=G != 2)
    attend(T, p.fill(n), G, f"n={n}")


def test_attend_more_pages_than_a_block_of_the_table(T):
    """Many KV heads, so that a part of the sequence has hundreds of pages,
    some of them invalid."""
    say("attend pages")
    p = Paged([17600, 300], 64, 64, 16, BF16, seed=14)
    p.table[0, 270] = p.table[0, 511] = p.table[0, 800] = -1
    attend(T, p.fill(15), 64, "pages")


@pytest.mark.parametrize("window", [1, 15, 32, 33, 200, 299, 300, 5000])
@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_windows(T, window, kind):
    say("attend window", window, kind)
    p = Paged([300, 5, 0, 1203], 2, 64, 16, kind, seed=window, track=window in (33, 200))
    attend(T, p.fill(window), 4, f"window={window}", window=window)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_leaves_out_invalid_pages(T, kind):
    """Pages outside the pool hold no rows; a sequence of nothing else gets
    zeros, and its weights stay."""
    say("attend invalid pages", kind)
    p = Paged([100, 100, 40, 64], 2, 128, 16, kind, seed=3, track=True)
    p.weights += 0.25
    p.table[0, 2] = -7
    p.table[0, 6] = p.pages
    p.table[1, 0] = 0x7FFFFFFF
    p.table[2, :] = -1
    p.fill(8)
    _, got, _ = attend(T, p, 8, "invalid pages")
    assert np.all(got[2] == 0)


@pytest.mark.parametrize("D", [128, 512])
@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_a_page_named_twice(T, kind, D):
    """Its rows count twice, each place with weights of its own."""
    say("attend page twice", kind, D)
    p = Paged([100, 50], 2, D, 16, kind, seed=5, track=True).fill(5)
    p.table[0, 4] = p.table[0, 1]
    p.table[1, :3] = p.table[0, 1]
    attend(T, p, 8, "page twice", max_rows=93)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_lengths_outside_the_table(T, kind):
    say("attend lens", kind)
    p = Paged([64, 64, 64], 2, 128, 16, kind, seed=4, track=True).fill(4)
    p.lens[:] = [-5, 1000, 0x7FFFFFFF]
    attend(T, p, 4, "lens")
    attend(T, p, 4, "max_rows", max_rows=39)


def test_attend_garbage_behind_the_rows_is_not_read(T):
    """NaN and infinity behind the last row and before the window."""
    for kind in (BF16, AFFINE):
        p = Paged([37, 20], 2, 128, 32, kind, seed=6).fill(6)
        say("garbage", kind)
        for side in p.sides:
            for t in side:
                if t.dtype == np.uint16:
                    behind = t[p.table[0, 1], :, 5:]
                    behind[...] = np.where(np.arange(behind.shape[-1]) % 2, 0x7F80, 0xFFFF)
        p.sides[1][-1][p.table[0, 0], :, :4] = 0x7F80
        p.sides[0][-1][p.table[0, 0], :, :4] = 0x7FC0
        q = kv_bf16((2, 4, 128), 1)
        d = p.device(T)
        clean = Paged([37, 20], 2, 128, 32, kind, seed=6).fill(6)
        out, tol, _, _ = clean.attend(q, 0.1, 33)
        check(O.bf16_to_f32(d.attend(q, 0.1, 33)), out, tol, "garbage")


@pytest.mark.parametrize("kind", [BF16, AFFINE])
def test_attend_sharp_and_extreme_scores(T, kind):
    say("extreme scores", kind)
    p = Paged([500, 129], 2, 128, 64, kind, seed=12, track=True).fill(12)
    attend(T, p, 4, "sharp", qmult=16.0)
    attend(T, p, 4, "flat", scale=0.0)
    attend(T, p, 4, "negative", scale=-0.3)


def test_attend_type_extremes_in_bf16_rows(T):
    """A key that gives -inf has no weight; all keys -inf give zeros; values of
    the type's largest magnitude come back."""
    p = Paged([40, 40, 40], 1, 64, 16, BF16, seed=13)
    p.fill(13)
    one = O.bf16_from_f32(np.ones(64, np.float32))
    q = np.broadcast_to(one, (3, 2, 64)).copy()
    page = p.table[0, 1]
    p.sides[0][0][page, 0, 3, 0] = 0xFF80  # -inf in row 19 of sequence 0
    p.sides[0][0][p.table[1], :, :, 5] = 0xFF80
    p.sides[0][0][p.table[2]] = 0
    p.sides[1][0][p.table[2]] = 0x7F7F
    say("extremes")
    got = O.bf16_to_f32(p.device(T).attend(q, 0.125))
    assert np.all(got[1] == 0)
    assert np.all(np.abs(got[2] / O.bf16_to_f32(np.uint16(0x7F7F)) - 1) <= 2.0 ** -8)
    keep = np.r_[0:19, 20:40]
    ok, k, v, _ = p.rows(0, 0, 40)
    s = k[keep].sum(1) * 0.125
    w = np.exp(s - s.max())
    want = (w / w.sum()) @ v[keep]
    assert np.all(np.abs(got[0] - want) <= 2.0 ** -7 * (w / w.sum() @ np.abs(v[keep])))


@pytest.mark.parametrize("D", [128, 512])
@pytest.mark.parametrize("power", [-75, -14, 14, 60, 118])
def test_attend_values_of_any_magnitude(T, D, power):
    """Affine values times powers of two, one sequence's pages larger than the
    others' by 2^20 half way: the f16 unit follows them."""
    say("magnitude", D, power)
    p = Paged([700, 33], 1, D, 16, AFFINE, 4, 8, 64, seed=power % 97).fill(3)
    late = p.table[0, 20:44]
    for t in p.sides[1][1:]:
        x = O.bf16_to_f32(t) * np.float32(2.0 ** min(power, 100)) * np.float32(2.0 ** max(power - 100, 0))
        x[late] *= np.float32(2.0 ** (-20 if power > 100 else 20))
        t[...] = O.bf16_from_f32(x)
    q = kv_bf16((2, 4, D), 8)
    out, tol, _, _ = p.attend(q, 0.05)
    check(O.bf16_to_f32(p.device(T).attend(q, 0.05)), out, tol, f"2^{power}")


@pytest.mark.parametrize("power", [-60, 40])
def test_attend_queries_of_any_magnitude(T, power):
    """Queries times a power of two, the scale times its inverse."""
    for kind in (BF16, AFFINE):
        p = Paged([300, 40], 2, 128, 32, kind, seed=19).fill(19)
        q = kv_bf16((2, 4, 128), 8)
        d = p.device(T)
        big = O.bf16_from_f32(O.bf16_to_f32(q) * np.float32(2.0 ** power))
        say("queries", kind, power)
        assert np.array_equal(d.attend(q, 0.09), d.attend(big, float(np.float32(0.09) * 2.0 ** -power)))


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("power", [-126, -100, 0])
def test_attend_scales_and_queries_that_vanish(T, kind, power):
    """Scores of nothing, and of a factor below f32's smallest, beside rows
    that are masked: every row of the window has the same weight."""
    p = Paged([17, 50, 3], 2, 128, 16, kind, 8, 4, 32, seed=21, spare=1).fill(22)
    q = kv_bf16((3, 4, 128), 23)
    q[0] = 0
    q[1] = O.bf16_from_f32(O.bf16_to_f32(q[1]) * np.float32(2.0 ** power))
    for scale in (2.0 ** -60, 0.0):
        out, tol, _, _ = p.attend(q, scale, 33)
        check(O.bf16_to_f32(p.device(T).attend(q, scale, 33)), out, tol, f"2^{power} x {scale}")


def test_attend_shared_pages(T):
    """A prompt's pages shared by every sequence, their weights apart."""
    for kind in (BF16, AFFINE):
        p = Paged([90, 75, 64], 2, 128, 16, kind, seed=15, track=True)
        p.table[1:, :4] = p.table[0, :4]
        say("shared", kind)
        attend(T, p.fill(15), 8, "shared pages")


@pytest.mark.parametrize("B", [1, 3, 257, 1024])
def test_attend_batches(T, B):
    say("batch", B)
    rng = np.random.default_rng(B)
    p = Paged(list(rng.integers(0, 70 if B > 3 else 3000, B)), 1, 64, 16, BF16, seed=B, track=B == 3)
    attend(T, p.fill(B), 2, f"B={B}")


def test_attend_strided_queries_and_library_scratch(T):
    p = Paged([200, 31, 1], 2, 128, 16, AFFINE, seed=21).fill(21)
    H, D = 8, 128
    q = kv_bf16((3, H + 4, D), 5)
    d = p.device(T)
    say("strided q")
    want = d.attend(np.ascontiguousarray(q[:, 2:2 + H]), 0.09)
    dq = T.DeviceArray.of(q)
    out = T.DeviceArray((3, H, D), np.uint16)
    T.paged_decode_attend(d.view(), dq.ptr + 2 * 2 * D, (H + 4) * D, H, 0.09, p.stride * p.R, out.ptr)
    T.hip().sync()
    assert np.array_equal(out.numpy(), want)


def test_attend_is_the_same_every_time(T):
    p = Paged([4000, 17, 900], 4, 128, 64, BF16, seed=22, track=True).fill(22)
    q = kv_bf16((3, 16, 128), 6)
    say("repeat")
    runs = []
    for _ in range(3):
        d = p.device(T)
        runs.append((d.attend(q, 0.09), d.weights.numpy()))
    for a, w in runs[1:]:
        assert np.array_equal(a, runs[0][0]) and np.array_equal(w, runs[0][1])


def test_offsets_past_32_bits(T):
    """Pages whose byte offsets pass 2^32, written and read (the pool itself is
    not filled)."""
    Hkv, D, R, pages = 8, 128, 64, 40000  # 5.2 GB of keys
    say("large pool")
    k, v = (T.DeviceArray((pages, Hkv, R, D), np.uint16) for _ in range(2))
    table = np.array([[39999, 33001, 5], [32768, 39998, 0]], np.int32)
    lens = np.array([130, 100], np.int32)
    counts = [130, 100]
    x = kv_bf16((230, 2 * Hkv, D), 31)
    dx, dt, dl = T.DeviceArray.of(x), T.DeviceArray.of(table), T.DeviceArray.of(lens)
    starts = T.DeviceArray.of(np.array([0, 130, 230], np.int32))
    kv = T.paged_kv(T.CACHE_BF16, 2, Hkv, D, R, pages, [k.ptr, v.ptr], dt.ptr, 3, dl.ptr)
    T.paged_append(kv, dx.ptr, dx.ptr + Hkv * D * 2, starts.ptr, 230, 2 * Hkv * D, D)
    q = kv_bf16((2, 16, D), 32)
    dq, out = T.DeviceArray.of(q), T.DeviceArray((2, 16, D), np.uint16)
    T.paged_decode_attend(kv, dq.ptr, 16 * D, 16, 0.09, 192, out.ptr)
    T.hip().sync()
    p = Paged(lens, Hkv, D, R)
    for b, at in enumerate((0, 130)):
        for j in range(counts[b]):
            p.write(b, j, x[at + j, :Hkv], x[at + j, Hkv:])
    want, tol, _, _ = p.attend(q, 0.09)
    check(O.bf16_to_f32(out.numpy()), want, tol, "large pool")


# -------------------------------------------------------------------- evict
def evict(T, p, budget, sinks, recent, seed, alias=False, kept_out=True, move_weights=True):
    """Moves to the spare pages; compares every byte. Returns the new state."""
    B, Hkv, R = p.B, p.Hkv, p.R
    width = -(-budget // R) + 1
    need = [-(-min(max(int(n), 0), p.stride * R, budget) // R) for n in p.lens]
    assert sum(need) <= len(p.spare), (sum(need), len(p.spare))
    dst = np.full((B, width), -1, np.int32)
    order = np.random.default_rng(seed).permutation(p.spare)
    at = 0
    for b, c in enumerate(need):
        dst[b, :c] = order[at:at + c]
        at += c
    d = p.device(T)
    ddst = T.DeviceArray.of(dst)
    dlens = d.lens if alias else T.DeviceArray.of(np.full(B, 77, np.int32))
    start = np.full((B, Hkv, width * R), 3.25, np.float32)
    dw = T.DeviceArray.of(start)
    dk = T.DeviceArray.of(np.full((B, Hkv, budget), 99, np.int32))
    T.paged_evict(d.view(), budget, sinks, recent, ddst.ptr, width, dlens.ptr,
                  dw.ptr if move_weights else None, dk.ptr if kept_out else None)
    T.hip().sync()
    want_kept = np.full((B, Hkv, budget), -1, np.int32)
    want_w = start.copy()
    want = [[t.copy() for t in side] for side in p.sides]
    lens = np.array([min(max(int(n), 0), p.stride * R, budget) for n in p.lens], np.int32)
    for b in range(B):
        for h in range(Hkv):
            rows = p.choose(b, h, budget, sinks, recent)
            want_kept[b, h, :len(rows)] = rows
            want_w[b, h, :len(rows)] = p.weights[b, h, rows]
            to = np.arange(len(rows))
            ps, pd = p.table[b, rows // R], dst[b, to // R]
            ok = (ps >= 0) & (ps < p.pages) & (pd >= 0) & (pd < p.pages)
            for side, new in zip(p.sides, want):
                for t, u in zip(side, new):
                    u[pd[ok], h, to[ok] % R] = t[ps[ok], h, rows[ok] % R]
    if kept_out:
        assert np.array_equal(dk.numpy(), want_kept)
    assert np.array_equal(dlens.numpy(), lens)
    got_w = dw.numpy()
    assert np.array_equal(got_w.view(np.uint32), (want_w if move_weights else start).view(np.uint32))
    for got, w in zip(d.host(), want):
        for g, x in zip(got, w):
            assert np.array_equal(g, x)
    return dst, lens, want_w, want


EVICTS = [
    # lens, budget, sinks, recent
    ([100, 33, 0, 64], 40, 4, 8), ([500], 100, 0, 0), ([257, 1], 256, 0, 256), ([300], 5, 5, 0),
    ([300], 7, 3, 4), ([5000, 4097], 1000, 4, 128), ([20, 30], 64, 1, 1), ([10000], 9999, 2, 3),
    ([70], 1, 0, 0), ([70], 1, 0, 1),
]


@pytest.mark.parametrize("lens,budget,sinks,recent", EVICTS)
@pytest.mark.parametrize("kind,R", [(BF16, 16), (AFFINE, 32), (AFFINE, 128)])
def test_evict_keeps_the_heaviest(T, lens, budget, sinks, recent, kind, R):
    say("evict", lens, budget, sinks, recent, kind, R)
    p = Paged(lens, 2, 64 if R < 128 else 128, R, kind, 4, 8 if R == 32 else 4, 32, spare=3 + sum(-(-min(n, budget) // R) for n in lens),
              seed=budget, track=True).fill(budget)
    w = p.rng.random(p.weights.shape) ** 6
    p.weights[...] = np.where(p.rng.random(p.weights.shape) < 0.3, 0.0, w)
    evict(T, p, budget, sinks, recent, budget, alias=R == 32, kept_out=R != 128 or budget < 500,
          move_weights=budget != 1000)


@pytest.mark.parametrize("which", ["equal", "two", "specials", "close", "negative"])
def test_evict_orders_weights(T, which):
    """Ties go to the lower row; NaN ranks with -inf, -0 with 0."""
    say("evict weights", which)
    p = Paged([9000, 300], 2, 64, 16, BF16, spare=300, seed=41, track=True)
    n = p.weights.size
    r = p.rng
    if which == "equal":
        p.weights[...] = 0.5
    elif which == "two":
        p.weights[...] = np.where(r.random(p.weights.shape) < 0.2, 1.0, np.nextafter(np.float32(1), 2))
    elif which == "specials":
        pick = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -np.nan], np.float32)
        p.weights[...] = pick[r.integers(0, len(pick), p.weights.shape)]
    elif which == "close":
        p.weights[...] = (np.float32(1).view(np.uint32) + r.integers(0, 4000, n).astype(np.uint32)).view(
            np.float32).reshape(p.weights.shape)
    else:
        p.weights[...] = r.standard_normal(p.weights.shape)
    for budget in (1234, 250):
        evict(T, p, budget, 3, 100, budget)


@pytest.mark.parametrize("kind,bk,bv,gs", LAYOUTS)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_evict_moves_every_row_format(T, kind, bk, bv, gs, D):
    if gs > D:
        pytest.skip("a group is at most a row")
    say("evict format", kind, bk, bv, gs, D)
    p = Paged([333, 7, 150], 3, D, 16, kind, bk, bv, gs, spare=24, seed=D + gs, track=True).fill(D)
    p.weights[...] = p.rng.random(p.weights.shape)
    evict(T, p, 131, 3, 20, D)


@pytest.mark.parametrize("budget", [5000, 40001])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long_sequences(T, budget, ties):
    """More rows than the selection holds in registers."""
    say("evict long", budget, ties)
    p = Paged([70001, 33000, 32769], 1, 64, 256, AFFINE, spare=500, seed=45, track=True)
    w = p.rng.random(p.weights.shape)
    p.weights[...] = np.floor(8 * w) if ties else w
    evict(T, p, budget, 4, 1000, budget)


def test_evict_with_invalid_pages_and_lengths(T):
    p = Paged([200, 150, 64], 2, 64, 16, AFFINE, spare=20, seed=43, track=True).fill(43)
    p.weights[...] = p.rng.random(p.weights.shape)
    p.table[0, 3] = -1
    p.table[1, 0] = p.pages + 5
    p.lens[2] = -3
    say("evict invalid")
    evict(T, p, 50, 2, 10, 1, alias=True)
    p.lens[2] = 100000
    evict(T, p, 60, 0, 0, 2)


# ------------------------------------------------------------------- in use
@pytest.mark.parametrize("kind,D,H,Hkv,R", [(BF16, 128, 8, 2, 16), (AFFINE, 128, 8, 2, 32),
                                            (AFFINE, 64, 4, 4, 16)])
def test_prompt_steps_and_evictions(T, kind, D, H, Hkv, R):
    """Prompts appended, then steps that append, attend and gather, with an
    eviction of the batch each time a sequence passes its budget."""
    budget, sinks, recent = 96, 4, 24
    p = Paged([0, 0, 0], Hkv, D, R, kind, stride=10, seed=51, spare=400, track=True)
    say("in use", kind, D)
    free = list(p.spare)

    def grow():
        for b in range(p.B):
            for i in range(-(-int(p.lens[b]) // R)):
                if p.table[b, i] < 0:
                    p.table[b, i] = free.pop()

    prompt = [90, 33, 61]
    p.lens[:] = prompt
    grow()
    append(T, p, prompt, 60)
    for step in range(12):
        p.lens += 1
        grow()
        append(T, p, [1, 1, 1], 100 + step)
        q = kv_bf16((3, H, D), 200 + step)
        out, tol, gain, gtol = p.attend(q, D ** -0.5)
        d = p.device(T)
        check(O.bf16_to_f32(d.attend(q, D ** -0.5)), out, tol, f"step {step}")
        w = d.weights.numpy()
        check(w, p.weights + gain, gtol + 2.0 ** -23 * (p.weights + gain), f"step {step} weights")
        p.weights = w
        if p.lens.max() > budget + 3:
            p.spare = np.array(free, np.int32)
            dst, lens, neww, pool = evict(T, p, budget, sinks, recent, step, alias=step % 2 == 0)
            p.sides, p.lens = pool, lens
            p.table[...] = -1
            p.table[:, :min(dst.shape[1], p.stride)] = dst[:, :p.stride]
            p.weights[...] = 0.0
            k = min(neww.shape[2], p.weights.shape[2])
            p.weights[:, :, :k] = neww[:, :, :k]
            free = [f for f in free if f not in set(dst[dst >= 0].tolist())]


def test_captured_steps_follow_the_device_lengths(T):
    """Append and attention captured once, replayed as the sequences grow,
    eager work between; every replay equals the eager calls."""
    D, H, Hkv, R, B = 128, 8, 2, 16, 3
    p = Paged([20, 47, 3], Hkv, D, R, AFFINE, stride=8, seed=61, spare=24, track=True).fill(61)
    p.table[...] = np.random.default_rng(2).permutation(p.pages)[:24].reshape(3, 8)
    p.fill(62)
    d, e = p.device(T), p.device(T)
    q = T.DeviceArray((B, H, D), np.uint16)
    x = T.DeviceArray((B, 2 * Hkv, D), np.uint16)
    outs = [T.DeviceArray((B, H, D), np.uint16) for _ in range(2)]
    need = T.paged_decode_workspace_size(d.view(), H, 128)
    ws = [T.DeviceArray((need,), np.uint8) for _ in range(2)]
    say("capture")

    def step(pool, i, stream):
        T.paged_append(pool.view(), x.ptr, x.ptr + 2 * Hkv * D, None, B, 2 * Hkv * D, D, stream)
        T.paged_decode_attend(pool.view(), q.ptr, H * D, H, 0.09, 128, outs[i].ptr, -1, ws[i].ptr,
                              need, stream)

    with captured(T, lambda s: step(d, 0, s)) as launch:
        for i in range(5):
            p.lens += 1
            for pool in (d, e):
                T.hip().copy_in(pool.lens.ptr, p.lens)
            T.hip().copy_in(q.ptr, kv_bf16((B, H, D), 300 + i))
            T.hip().copy_in(x.ptr, kv_bf16((B, 2 * Hkv, D), 400 + i))
            launch()
            step(e, 1, None)
            T.hip().sync()
            assert np.array_equal(outs[0].numpy(), outs[1].numpy()), f"replay {i}"
            assert np.array_equal(d.weights.numpy(), e.weights.numpy()), f"replay {i}"
    for a, b in zip(d.host(), e.host()):
        for t, u in zip(a, b):
            assert np.array_equal(t, u)


def test_captured_eviction(T):
    p = Paged([400, 90], 2, 64, 16, BF16, spare=40, seed=71, track=True).fill(71)
    d = p.device(T)
    width, budget = 8, 120
    dst = p.spare[:16].reshape(2, 8)
    ddst, dl = T.DeviceArray.of(dst), T.DeviceArray((2,), np.int32)
    dw, dk = T.DeviceArray((2, 2, 128), np.float32), T.DeviceArray((2, 2, budget), np.int32)
    say("captured eviction")

    def call(stream):
        T.paged_evict(d.view(), budget, 4, 16, ddst.ptr, width, dl.ptr, dw.ptr, dk.ptr, None, 0, stream)

    with captured(T, call) as launch:
        for i in range(3):
            p.weights[...] = np.random.default_rng(i).random(p.weights.shape)
            T.hip().copy_in(d.weights.ptr, p.weights)
            launch()
            want = np.full((2, 2, budget), -1, np.int32)
            for b in range(2):
                for h in range(2):
                    rows = p.choose(b, h, budget, 4, 16)
                    want[b, h, :len(rows)] = rows
            assert np.array_equal(dk.numpy(), want), f"replay {i}"
            assert np.array_equal(dl.numpy(), [120, 90])


def test_two_streams_at_once(T):
    """Two pools' calls on two streams, a workspace each."""
    hip = T.hip()
    pools = [Paged([3000, 100], 2, 128, 16, k, seed=80 + k).fill(80 + k) for k in (BF16, AFFINE)]
    q = kv_bf16((2, 8, 128), 9)
    want = [p.device(T).attend(q, 0.09) for p in pools]
    say("two streams")
    ds = [p.device(T) for p in pools]
    dq = T.DeviceArray.of(q)
    outs = [T.DeviceArray((2, 8, 128), np.uint16) for _ in pools]
    streams = [hip.stream() for _ in pools]
    most = pools[0].stride * 16
    need = T.paged_decode_workspace_size(ds[0].view(), 8, most)
    ws = [T.DeviceArray((need,), np.uint8) for _ in pools]
    hip.sync()
    for _ in range(20):
        for i, d in enumerate(ds):
            T.paged_decode_attend(d.view(), dq.ptr, 8 * 128, 8, 0.09, most, outs[i].ptr, -1, ws[i].ptr,
                                  need, streams[i])
    hip.sync()
    for out, w in zip(outs, want):
        assert np.array_equal(out.numpy(), w)
    for s in streams:
        hip.h.hipStreamDestroy(ctypes.c_void_p(s))
