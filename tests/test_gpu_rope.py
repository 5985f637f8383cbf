"""Rotary positions on the GPU against 64 bits: both layouts, parts of a head,
every scaling, far positions, strides, in place; and the append that rotates,
bit for bit the rotation and the append apart."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged
from test_gpu_capture import captured

pytestmark = pytest.mark.gpu
GUARD = 0x7FC1


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


class Turns:
    """A rope on the device, and its angles in 64 bits."""

    def __init__(self, T, rd, interleaved, **scaling):
        turns, m = T.rope_turns(rd, **scaling)
        self.d = T.DeviceArray.of(np.array(turns, np.uint64))
        self.rope = T.rope(rd, interleaved, m, self.d.ptr)
        self.theta, self.m = R.thetas(rd, scaling.pop("base", 10000.0), **scaling)
        assert abs(self.m - m) <= 2.0 ** -23 * self.m
        self.m = float(m)
        self.interleaved = interleaved


def apply(T, r, x, positions, inplace=False, beside=0, pad=0, stride=1):
    """x bf16 [tokens, heads, D] in a buffer with `beside` heads behind them and
    `pad` elements a token; (out rows, whole out buffer)."""
    n, H, D = x.shape
    width = (H + beside) * D + pad
    buf = np.full((n, width), GUARD, np.uint16)
    buf[:, :H * D] = x.reshape(n, -1)
    dx = T.DeviceArray.of(buf)
    pos = np.full((n, stride), -77, np.int32)
    pos[:, 0] = positions
    dp = T.DeviceArray.of(pos)
    out = dx if inplace else T.DeviceArray(buf.shape, np.uint16, np.full(buf.shape, GUARD, np.uint16))
    T.rope_apply(r.rope, dp.ptr, stride, n, dx.ptr, H, D, width, D, out.ptr, width, D)
    T.hip().sync()
    got = out.numpy()
    assert np.all(got[:, H * D:] == GUARD)
    return got[:, :H * D].reshape(n, H, D)


CASES = [
    # D, rd, heads, tokens
    (128, 128, 40, 5), (128, 128, 1, 1), (64, 64, 3, 33), (256, 64, 7, 9), (512, 512, 2, 3), (512, 384, 16, 2),
    (128, 44, 5, 6), (64, 2, 2, 4), (128, 126, 3, 3), (96, 80, 4, 7), (8, 6, 9, 11), (1024, 1024, 2, 2), (24, 24, 1, 100),
    (16, 16, 1024, 2), (1024, 1022, 1024, 2), (1024, 1022, 700, 3),
]


@pytest.mark.parametrize("D,rd,heads,tokens", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_rope(T, D, rd, heads, tokens, interleaved, inplace):
    print("[rope]", D, rd, heads, tokens, interleaved, inplace, flush=True)
    r = Turns(T, rd, interleaved)
    x = kv_bf16((tokens, heads, D), D + rd)
    rng = np.random.default_rng(rd)
    positions = rng.integers(0, 5000, tokens)
    positions[0] = 0
    got = apply(T, r, x, positions, inplace, beside=2, pad=8 * (D % 16 == 0), stride=3)
    want, tol = R.rotated(x, positions, r.theta, r.m, interleaved)
    assert np.array_equal(got[..., rd:], x[..., rd:])
    R.check(O.bf16_to_f32(got)[..., :rd], want[..., :rd], tol[..., :rd], "rope")
    if positions[0] == 0:
        assert np.array_equal(got[0], x[0])  # position 0 turns nothing


@pytest.mark.parametrize("scaling", [
    dict(scaling=1, factor=8.0), dict(scaling=2, factor=4.0), dict(scaling=3, factor=8.0, original=8192.0, low=1.0, high=4.0),
    dict(scaling=4, factor=16.0, original=4096.0, low=1.0, high=32.0), dict(scaling=4, factor=3.0, original=10.0, low=1.0, high=2.0),
    dict(scaling=3, factor=0.5, original=100.0, low=0.1, high=9.0), dict(base=1.5), dict(base=1e9)])
@pytest.mark.parametrize("rd", [2, 64, 128])
def test_scalings(T, scaling, rd):
    print("[rope scaling]", scaling, rd, flush=True)
    r = Turns(T, rd, False, **scaling)
    x = kv_bf16((40, 2, 128), 3)
    positions = np.concatenate([np.arange(20), np.random.default_rng(1).integers(0, 200000, 20)])
    want, tol = R.rotated(x, positions, r.theta, r.m, False)
    R.check(O.bf16_to_f32(apply(T, r, x, positions)), want, tol, "scaling")


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(T, interleaved):
    """Positions up to 2^31 - 1; the tolerance counts the 64-bit angles' own error."""
    r = Turns(T, 64, interleaved)
    positions = np.array([2 ** 20, 2 ** 24 + 1, 2 ** 27 - 1, 10 ** 9 + 7, 2 ** 31 - 1])
    x = kv_bf16((5, 3, 64), 9)
    # The reference's theta is off by 2^-52 of itself or so: exact turns instead.
    from fractions import Fraction
    turns = T.rope_turns(64)[0]
    angle = np.array([[float(Fraction(int(p) * t % 2 ** 64, 2 ** 64)) for t in turns] for p in positions]) * 2 * np.pi
    y = O.bf16_to_f32(x).astype(np.float64)
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :32], y[..., 32:])
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    u, v = a * c - b * s, a * s + b * c
    got = O.bf16_to_f32(apply(T, r, x, positions)).astype(np.float64)
    gu, gv = (got[..., 0::2], got[..., 1::2]) if interleaved else (got[..., :32], got[..., 32:])
    each = (np.abs(a) + np.abs(b)) * (2 * np.pi * 2.0 ** -24 + 2.0 ** -21)
    R.check(gu, u, 2.0 ** -8 * np.abs(u) + each, "far, first")
    R.check(gv, v, 2.0 ** -8 * np.abs(v) + each, "far, second")


def test_turns_against_64_bits(T):
    for rd in (2, 64, 130, 1024):
        for kw in (dict(), dict(scaling=1, factor=7.0), dict(scaling=2, factor=5.0), dict(scaling=3, factor=8.0, original=8192.0),
                   dict(scaling=4, factor=8.0, original=2048.0, high=32.0)):
            turns, m = T.rope_turns(rd, 500000.0, **kw)
            theta, mag = R.thetas(rd, 500000.0, **kw)
            got = np.array([t / 2.0 ** 64 * 2 * np.pi for t in turns])
            # The power's own error in 64 bits, and half a unit of the turns: 2^-65 of a turn.
            assert np.all(np.abs(got - theta) <= 2.0 ** -46 * theta + 2 * np.pi * 2.0 ** -65), (rd, kw)
            assert abs(m - mag) <= 2.0 ** -23 * mag


def test_tokens_of_negative_position_stay(T):
    r = Turns(T, 128, False)
    x = kv_bf16((6, 4, 128), 5)
    positions = np.array([3, -1, 7, -2 ** 31, 0, -1])
    got = apply(T, r, x, positions)
    assert np.all(got[positions < 0] == GUARD)
    alone = apply(T, r, x[positions >= 0], positions[positions >= 0])
    assert np.array_equal(got[positions >= 0], alone)


def test_many_tokens_and_extremes(T):
    r = Turns(T, 64, True)
    x = kv_bf16((5001, 3, 64), 5)
    x[17, 0, :4] = O.bf16_from_f32(np.array([np.inf, 1.0, np.nan, 2.0], np.float32))
    x[18, 1, :2] = O.bf16_from_f32(np.array([3e38, 1e-39], np.float32))
    positions = np.arange(5001)
    got = O.bf16_to_f32(apply(T, r, x, positions))
    assert np.all(~np.isfinite(got[17, 0, :2])) and np.all(np.isnan(got[17, 0, 2:4]))
    want, tol = R.rotated(x, positions, r.theta, r.m, True)
    keep = np.ones(5001, bool)
    keep[17] = False
    tol[18, 1, :2] += 2.0 ** -9 * 3e38  # next to the largest value
    R.check(got[keep], want[keep], tol[keep], "many")


# ------------------------------------------------------------------- append
APPENDS = [
    # kind, bk, bv, gs, D, R, Hkv, G, rd, lens, counts
    (BF16, 16, 16, 64, 128, 16, 3, 4, 128, [5, 40, 0, 33], [5, 17, 0, 33]),
    (BF16, 16, 16, 64, 64, 32, 1, 1, 22, [1], [1]),
    (BF16, 16, 16, 64, 256, 64, 8, 2, 64, [100, 64, 65], [36, 64, 1]),
    (BF16, 16, 16, 64, 512, 256, 2, 0, 512, [300, 7], [299, 0]),
    (AFFINE, 4, 4, 64, 128, 16, 3, 4, 128, [5, 40, 0, 33], [5, 17, 0, 33]),
    (AFFINE, 8, 8, 32, 64, 32, 1, 5, 30, [1, 31], [1, 30]),
    (AFFINE, 8, 4, 32, 256, 64, 5, 1, 64, [100, 64, 65], [36, 64, 1]),
    (AFFINE, 4, 8, 128, 512, 128, 2, 0, 96, [300, 7], [299, 0]),
    # A token's work in more than 2^16 pieces, of one token a workgroup and of two.
    (BF16, 16, 16, 64, 512, 16, 1, 1020, 510, [3], [3]),
    (AFFINE, 4, 4, 64, 128, 16, 1, 1020, 126, [520], [520]),
]


def slots_of(p, counts):
    s = []
    for b, c in enumerate(counts):
        for row in range(int(p.lens[b]) - c, int(p.lens[b])):
            s.append([p.table[b, row // p.R], row % p.R, row, b])
    return np.array(s, np.int32).reshape(-1, 4)


class Entered:
    """The same tokens through rotation and append apart, and at once."""

    def __init__(self, T, p, counts, G, r, seed, slots=None, positions=None, pad=0):
        n, H = sum(counts), G * p.Hkv
        width = (H + 2 * p.Hkv) * p.D + pad
        self.n, self.H, self.D, self.width = n, H, p.D, width
        self.buf = kv_bf16((n, width), seed, frac=0.02, mult=4.0)
        self.slots = slots_of(p, counts) if slots is None else slots
        self.positions = positions
        self.T, self.p, self.r = T, p, r
        self.counts = counts

    def together(self, stream=None, inplace=False):
        T, p = self.T, self.p
        d, dbuf, ds = p.device(T), T.DeviceArray.of(self.buf), T.DeviceArray.of(self.slots)
        q = dbuf if inplace else T.DeviceArray((self.n, self.H, p.D), np.uint16, np.full((self.n, self.H, p.D), GUARD, np.uint16))
        k = dbuf.ptr + 2 * self.H * p.D
        dp = None if self.positions is None else T.DeviceArray.of(np.asarray(self.positions, np.int32))
        T.paged_append_rope(d.view(), self.r.rope, dbuf.ptr if self.H else None, self.H, self.width, q.ptr if self.H else None,
                            self.width if inplace else self.H * p.D, k, k + 2 * p.Hkv * p.D, self.width, p.D, ds.ptr, self.n,
                            None if dp is None else dp.ptr, 1, stream)
        T.hip().sync()
        got = q.numpy()
        return d, got[:, :self.H * p.D].reshape(self.n, self.H, p.D) if inplace else got

    def apart(self):
        T, p = self.T, self.p
        d, dbuf = p.device(T), T.DeviceArray.of(self.buf)
        dp = T.DeviceArray.of(np.asarray(self.slots[:, 2] if self.positions is None else self.positions, np.int32))
        starts = T.DeviceArray.of(np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32))
        T.rope_apply(self.r.rope, dp.ptr, 1, self.n, dbuf.ptr, self.H + p.Hkv, p.D, self.width, p.D, dbuf.ptr, self.width, p.D)
        k = dbuf.ptr + 2 * self.H * p.D
        T.paged_append(d.view(), k, k + 2 * p.Hkv * p.D, starts.ptr, self.n, self.width, p.D)
        T.hip().sync()
        return d, dbuf.numpy()[:, :self.H * p.D].reshape(self.n, self.H, p.D)


def same(a, b):
    for x, y in zip(a.host(), b.host()):
        for s, t in zip(x, y):
            assert np.array_equal(s, t)
    if a.weights is not None:
        assert np.array_equal(a.weights.numpy(), b.weights.numpy())


@pytest.mark.parametrize("kind,bk,bv,gs,D,R_,Hkv,G,rd,lens,counts", APPENDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_append_rope_is_rope_and_append(T, kind, bk, bv, gs, D, R_, Hkv, G, rd, lens, counts, interleaved, inplace):
    print("[enter]", kind, bk, bv, gs, D, R_, Hkv, G, rd, lens, counts, interleaved, inplace, flush=True)
    p = Paged(lens, Hkv, D, R_, kind, bk, bv, gs, spare=2, seed=D + R_, track=inplace)
    if p.weights is not None:
        p.weights += 1.5
    r = Turns(T, rd, interleaved, scaling=4, factor=4.0, original=64.0, high=32.0)
    e = Entered(T, p, counts, G, r, D + rd, positions=np.random.default_rng(1).integers(0, 9999, sum(counts)) if inplace else None,
                pad=8 * inplace)
    (a, qa), (b, qb) = e.together(inplace=inplace), e.apart()
    assert np.array_equal(qa, qb)
    same(a, b)


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("tokens", [9, 3000])
def test_append_rope_leaves_out_what_has_no_place(T, kind, tokens):
    """Padding, pages and rows out of range, sequences out of range."""
    Hkv, D, R_ = 2, 64, 16
    p = Paged([tokens + 40, 20], Hkv, D, R_, kind, 4, 8, 32, spare=1, seed=3, track=True)
    p.weights += 2.0
    r = Turns(T, 64, False)
    slots = slots_of(p, [tokens, 0])
    bad = [[-1, 0, -1, -1], [-1, 3, 40, 0], [p.pages, 0, 41, 0], [2 ** 31 - 1, 0, 42, 0], [0, R_, 43, 0], [0, -1, 44, 0]]
    slots[:6] = bad
    slots[6, 3], slots[7, 3], slots[8, 2] = 2, -1, 2 ** 30  # the row is written, no weight is cleared
    e = Entered(T, p, [tokens, 0], 2, r, 5, slots=slots)
    d, q = e.together()
    assert np.all(q[0] == GUARD) and not np.any(q[1:] == GUARD)
    # The rows that have a place, one by one.
    good = Entered(T, p, [tokens - 6, 0], 2, r, 5, slots=slots[6:])
    good.buf = e.buf[6:]
    dg, qg = good.together()
    assert np.array_equal(q[6:], qg)
    same(d, dg)
    w = d.weights.numpy()
    assert int((w == 0.0).sum()) == Hkv * (tokens - 9) and np.all((w == 0.0) | (w == 2.0))


def test_captured_append_rope(T):
    """A step captured with room for more tokens than it has, replayed over new
    slots and tokens."""
    Hkv, D, R_, H, n = 2, 128, 16, 4, 6
    p = Paged([50, 60, 70], Hkv, D, R_, BF16, seed=3)
    r = Turns(T, 128, False)
    d = p.device(T)
    width = (H + 2 * Hkv) * D
    buf, slots = T.DeviceArray((n, width), np.uint16), T.DeviceArray((n, 4), np.int32)
    q = T.DeviceArray((n, H, D), np.uint16)
    k = buf.ptr + 2 * H * D

    def call(stream):
        T.paged_append_rope(d.view(), r.rope, buf.ptr, H, width, q.ptr, H * D, k, k + 2 * Hkv * D, width, D, slots.ptr, n, None, 1, stream)

    with captured(T, call) as launch:
        for i in range(4):
            x = kv_bf16((n, width), 50 + i)
            m = 3 + i % 3
            s = np.full((n, 4), -1, np.int32)
            for j in range(m):
                b, row = j % 3, 10 + 7 * i + j
                s[j] = [p.table[b, row // R_], row % R_, row, b]
            T.hip().copy_in(buf.ptr, x)
            T.hip().copy_in(slots.ptr, s)
            before = d.host()
            launch()
            got = d.host()
            rows = x.reshape(n, H + 2 * Hkv, D)
            turned = apply(T, r, rows[:m, :H + Hkv], s[:m, 2])
            assert np.array_equal(q.numpy()[:m], turned[:, :H])
            for j in range(m):
                before[0][0][s[j, 0], :, s[j, 1]] = turned[j, H:]
                before[1][0][s[j, 0], :, s[j, 1]] = rows[j, H + Hkv:]
            for side in (0, 1):
                assert np.array_equal(got[side][0], before[side][0])
