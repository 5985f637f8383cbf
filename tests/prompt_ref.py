"""Page tables, rotary positions and the attention of packed sequences on the
host, from their definitions, in whole numbers and 64 bits. Nothing here calls
the library under test."""
import math

import numpy as np

import oracle_lib as O
from paged_ref import codes_of, values_of


# ------------------------------------------------------------------- tables
class Tables:
    """A table, lengths and a stack of free pages."""

    def __init__(self, lens, R, width, pages, seed=0):
        rng = np.random.default_rng(seed)
        self.R, self.width, self.pages, self.B = R, width, pages, len(lens)
        self.table = np.full((self.B, width), -1, np.int32)
        self.lens = np.asarray(lens, np.int32)
        order, at = rng.permutation(pages).astype(np.int32), 0
        for b, n in enumerate(lens):
            p = min(-(-max(int(n), 0) // R), width)
            self.table[b, :p] = order[at:at + p]
            at += p
        self.free = np.full(pages, -7, np.int32)
        self.count = pages - at
        self.free[:self.count] = order[at:]

    def held(self, b):
        return min(max(int(self.lens[b]), 0), self.width * self.R)

    def reserve(self, counts, tokens):
        """(starts, granted, slots) and the new state."""
        height = min(max(self.count, 0), self.pages)
        pages = places = 0
        granted, takes = [], []
        for b, want in enumerate(counts):
            want, n = max(int(want), 0), self.held(b)
            need = -(-(n + want) // self.R) - -(-n // self.R)
            fits = n + want <= self.width * self.R
            if fits:
                pages, places = pages + need, places + want
            ok = fits and (need == 0 or pages <= height) and (want == 0 or places <= tokens)
            granted.append(want if ok else -1)
            takes.append(need if ok else 0)
        top = at = height - sum(takes)
        starts, slots = [0], []
        for b, got in enumerate(granted):
            n, got = self.held(b), max(got, 0)
            first = -(-n // self.R)
            self.table[b, first:first + takes[b]] = self.free[at:at + takes[b]]
            at += takes[b]
            for row in range(n, n + got):
                page = int(self.table[b, row // self.R])
                slots.append([page if 0 <= page < self.pages else -1, row % self.R, row, b])
            self.lens[b] = n + got
            starts.append(starts[-1] + got)
        self.count = top
        slots += [[-1, 0, -1, -1]] * (tokens - len(slots))
        return (np.array(starts, np.int32), np.array(granted, np.int32),
                np.array(slots, np.int32).reshape(-1, 4))

    def release(self, keep, shared=None):
        self.count = min(max(self.count, 0), self.pages)
        for b in range(self.B):
            n = self.held(b)
            k = min(max(int(keep[b]), 0), n)
            first = max(-(-k // self.R), int(shared[b]) if shared is not None else 0)
            for j in range(first, -(-n // self.R)):
                page = int(self.table[b, j])
                if 0 <= page < self.pages and self.count < self.pages:
                    self.free[self.count] = page
                    self.count += 1
                self.table[b, j] = -1
            self.lens[b] = k


# --------------------------------------------------------------------- rope
def thetas(rd, base, scaling=0, factor=1.0, original=1.0, low=1.0, high=4.0):
    """(radians a position of each pair, magnitude), in 64 bits."""
    if scaling == 2 and rd > 2:
        base = base * factor ** (rd / (rd - 2))
    theta = np.array([base ** (-2.0 * i / rd) for i in range(rd // 2)])
    if scaling == 1:
        return theta / factor, 1.0
    if scaling == 3:
        stays = np.clip((original * theta / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        return stays * theta + (1.0 - stays) * theta / factor, 1.0
    if scaling == 4:
        def channel(turns):
            return rd * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
        first, last = max(math.floor(channel(high)), 0), min(math.ceil(channel(low)), rd - 1)
        go = np.clip((np.arange(rd // 2) - first) / max(last - first, 0.001), 0.0, 1.0)
        return (1.0 - go) * theta + go * theta / factor, 0.1 * math.log(factor) + 1.0
    return theta, 1.0


def rotated(x, positions, theta, magnitude, interleaved):
    """(rows f64, tolerance) of bf16 rows x [tokens, heads, D]. Tolerance:
    half a bf16 step of the result (2^-8 of it, or of the least normal value),
    and the f32 roundings of a pair: the fraction of a turn (2^-33 of one and
    f32's half step, together below 2^-24 turns, 2 pi of them in radians), cosine and sine (two steps
    each allowed, 2^-22), their product with the magnitude, two products and a
    sum (2^-24 each)."""
    rd = 2 * len(theta)
    y = O.bf16_to_f32(x).astype(np.float64)
    a = (y[..., 0:rd:2] if interleaved else y[..., :rd // 2]).copy()
    b = (y[..., 1:rd:2] if interleaved else y[..., rd // 2:rd]).copy()
    # The angle modulo a turn first: position * theta carries few bits below a radian.
    angle = np.asarray(positions, np.float64)[:, None] * theta[None]
    c, s = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    u, v = a * c - b * s, a * s + b * c
    tol = np.zeros_like(y)
    # 64-bit angles here: half a step of position * theta, 2^-53 of it.
    each = 2 * np.pi * 2.0 ** -24 + 2.0 ** -21 + np.abs(angle)[:, None] * 2.0 ** -52
    size = (np.abs(a) + np.abs(b)) * abs(magnitude) * each
    lo, hi = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    y[..., lo], y[..., hi] = u, v
    tol[..., lo] = tol[..., hi] = size
    tol[..., :rd] += 2.0 ** -8 * (np.abs(y[..., :rd]) + 2.0 ** -126)
    return y, tol


# ---------------------------------------------------------------- attention
def halves(side, bits, gs):
    """Whether V's groups allow largest values within 2^26 of each other (the
    library takes f16 within 2^28)."""
    s, z = (O.bf16_to_f32(t).astype(np.float64) for t in side[1:])
    top = np.maximum(np.abs(z), np.abs(s * (2 ** bits - 1) + z))
    return top.max(initial=0.0) <= 2.0 ** 26 * top[top > 0].min(initial=np.inf)


def attend(q, k, v, at, scale, causal=True, window=-1, ok=None, off=0.0, off_v=0.0, off_w=2.0 ** -8):
    """One sequence and one KV head: q f64 [m, G, D] at positions `at`, k and v
    f64 [n, D], ok: keys that can be seen at all, off, off_v, off_w: how far a
    key's or value's channel or a weight may be rounded, relative to it. (out,
    tolerance) f64.

    Tolerance: half a bf16 step of the output (2^-8 of it); the weights'
    rounding, which the sum of the rounded weights takes out of what they share:
    off_w sum w |v - out| (and where it is f16's, 2^-25 each of the largest for
    subnormal ones); the values', off_v sum w |v|; and the f32 arithmetic: a
    score's sum (2^-24 of the products' magnitudes an addition) and exp2's
    argument and result move a weight by their size, twice for the sum's; the
    running sums of weights and outputs 2^-24 an addition."""
    m, G, D = q.shape
    n = len(k)
    out, tol = np.zeros((m, G, D)), np.zeros((m, G, D))
    ok = np.ones(n, bool) if ok is None else ok
    t = np.arange(n)
    for i in range(m):
        see = ok.copy()
        if causal:
            see &= t <= at[i]
            if window > 0:
                see &= t > at[i] - window
        if not see.any():
            continue
        ks, vs = k[see], v[see]
        s = (q[i] @ ks.T) * scale
        w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        out[i] = w @ vs
        sums = ((D + 16) * 2.0 ** -24 + off) * (np.abs(q[i]) @ np.abs(ks).T).max(-1) * abs(scale)
        if off:  # f16's subnormals: 2^-25 where the largest is 2^14 or more
            sums = sums + 2.0 ** -39 * np.abs(k).max() * np.abs(q[i]).sum(-1) * abs(scale)
        d = 2 * (sums + 2.0 ** -22 * (np.abs(s).max(-1) + 4)) + see.sum() * 2.0 ** -24
        for g in range(G):
            spread = w[g] @ np.abs(vs - out[i, g])
            tol[i, g] = 2.0 ** -8 * np.abs(out[i, g]) + 1.02 * off_w * spread + 1.01 * (d[g] + off_v) * (w[g] @ np.abs(vs)) + 1e-30
            if off_w < 2.0 ** -8:  # f16's subnormals: of weights, and of values whose largest is 2^14 or more
                tol[i, g] += 2.0 ** -25 * np.abs(vs - out[i, g]).sum(0) + 2.0 ** -39 * np.abs(v).max()
    return out, tol


def packed(q, k, v, starts, scale, causal=True, window=-1):
    """bf16 q [T, H, D], k, v [T, Hkv, D]: (out, tolerance) f64 [T, H, D]."""
    T, H, D = q.shape
    Hkv = k.shape[1]
    G = H // Hkv
    qf, kf, vf = (O.bf16_to_f32(x).astype(np.float64) for x in (q, k, v))
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    for a, b in zip(starts[:-1], starts[1:]):
        for h in range(Hkv):
            o, t = attend(qf[a:b, h * G:(h + 1) * G], kf[a:b, h], vf[a:b, h], np.arange(b - a), scale, causal, window)
            out[a:b, h * G:(h + 1) * G], tol[a:b, h * G:(h + 1) * G] = o, t
    return out, tol


def paged(p, q, starts, scale, window=-1, max_rows=None):
    """A paged_ref.Paged pool p, bf16 q [T, H, D]: (out, tolerance) f64."""
    T, H, D = q.shape
    G = H // p.Hkv
    qf = O.bf16_to_f32(q).astype(np.float64)
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    for i in range(p.B):
        a, b = int(starts[i]), int(starts[i + 1])
        n = min(max(int(p.lens[i]), 0), p.stride * p.R, max_rows or 1 << 60)
        if a == b or n == 0:
            continue
        r = np.arange(n)
        page = p.table[i, r // p.R]
        ok = (page >= 0) & (page < p.pages)
        for h in range(p.Hkv):
            at = (np.where(ok, page, 0), h, r % p.R)
            # Affine keys: scale * code + bias (an f32 fused multiply-add, 2^-24) as f16, 2^-11.
            k = values_of([t[at] for t in p.sides[0]], p.bk, p.gs)
            k[~ok] = 0.0
            v = values_of([t[at] for t in p.sides[1]], p.bv, p.gs)
            v[~ok] = 0.0
            # Affine values and the weights with them: f16 (2^-11), or bf16 (2^-8).
            h16 = p.bv != 16 and halves([t[at][ok] for t in p.sides[1]], p.bv, p.gs)
            o, t = attend(qf[a:b, h * G:(h + 1) * G], k, v, np.arange(n - (b - a), n), scale, True, window, ok,
                          0.0 if p.bk == 16 else 2.0 ** -11 + 2.0 ** -24, 0.0 if p.bv == 16 else 2.0 ** -11 + 2.0 ** -24 if h16 else 2.0 ** -8,
                          2.0 ** -11 if h16 else 2.0 ** -8)
            out[a:b, h * G:(h + 1) * G], tol[a:b, h * G:(h + 1) * G] = o, t
    return out, tol


def check(got, want, tol, tag):
    got = np.asarray(got, np.float64)
    err = np.abs(got - want)
    worst = float(np.max(err / np.maximum(tol, 1e-300))) if err.size else 0.0
    print(f"[{tag}] worst error {worst:.3f} of its tolerance, max {err.max() if err.size else 0:.3e}", flush=True)
    assert np.all(np.isfinite(got)), f"{tag}: non-finite"
    assert worst <= 1.0, tag
