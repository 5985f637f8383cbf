"""A paged cache on the host, in 64 bits: the pool's rows, the append, the
attention with its gathered weights, and the eviction, from their definitions.
Shared by the paged cache's GPU tests; nothing here calls the library under
test but to upload (`Paged.device`)."""
import numpy as np

import oracle_lib as O

BF16, AFFINE = 0, 1
GUARD = 0x7FC0  # bf16 NaN: what the pool holds where nothing was written


def codes_of(packed, bits):
    shifts = np.arange(0, 32, bits, dtype=np.uint32)
    c = (packed[..., None] >> shifts) & np.uint32(2 ** bits - 1)
    return c.reshape(*packed.shape[:-1], -1).astype(np.float64)


def values_of(side, bits, gs):
    """f64 values of stored rows: (rows bf16,) or (packed, scales, biases)."""
    if bits == 16:
        return O.bf16_to_f32(side[0]).astype(np.float64)
    s, b = (np.repeat(O.bf16_to_f32(t).astype(np.float64), gs, axis=-1) for t in side[1:])
    return codes_of(side[0], bits) * s + b


class Paged:
    """A pool and its sequences on the host. lens: rows held; the table gives
    every sequence pages of its own in a shuffled order (spare pages last)."""

    def __init__(self, lens, Hkv, D, R, kind=BF16, bk=4, bv=4, gs=64, stride=None, spare=0, seed=0,
                 track=False):
        self.rng = np.random.default_rng(seed)
        self.kind, self.Hkv, self.D, self.R, self.gs = kind, Hkv, D, R, gs
        self.bk, self.bv = (bk, bv) if kind == AFFINE else (16, 16)
        self.B = len(lens)
        self.lens = np.asarray(lens, np.int32)
        need = [max(0, -(-int(n) // R)) for n in lens]
        self.stride = stride or max(1, max(need))
        need = [min(p, self.stride) for p in need]
        self.table = np.full((self.B, self.stride), -1, np.int32)
        used = sum(need)
        self.pages = max(1, used + spare)
        order = self.rng.permutation(used).astype(np.int32)
        at = 0
        for b, p in enumerate(need):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.spare = np.arange(used, used + spare, dtype=np.int32)
        self.sides = [self.empty(self.bk), self.empty(self.bv)]
        self.weights = np.zeros((self.B, Hkv, self.stride * R), np.float32) if track else None

    def empty(self, bits):
        lead = (self.pages, self.Hkv, self.R)
        if bits == 16:
            return [np.full((*lead, self.D), GUARD, np.uint16)]
        return [np.full((*lead, self.D * bits // 32), 0xFFFFFFFF, np.uint32)] + \
            [np.full((*lead, self.D // self.gs), GUARD, np.uint16) for _ in range(2)]

    def stored(self, x, bits):
        """What rows x (bf16 [..., D]) are stored as."""
        return [x] if bits == 16 else list(O.affine_quantize(np.ascontiguousarray(x), self.gs, bits))

    def write(self, b, row, k, v):
        """Row `row` of sequence b, all heads: k, v bf16 [Hkv, D]."""
        if not 0 <= row < self.stride * self.R:
            return
        page = self.table[b, row // self.R]
        if not 0 <= page < self.pages:
            return
        for side, x, bits in zip(self.sides, (k, v), (self.bk, self.bv)):
            for dst, src in zip(side, self.stored(x, bits)):
                dst[page, :, row % self.R] = src
        if self.weights is not None:
            self.weights[b, :, row] = 0.0

    def fill(self, seed, mult=4.0):
        """Rows [0, lens) of every sequence, N(0, 1) with a few large channels."""
        rng = np.random.default_rng(seed)
        for bits, side in zip((self.bk, self.bv), self.sides):
            for b in range(self.B):
                n = min(max(int(self.lens[b]), 0), self.stride * self.R)
                x = rng.standard_normal((n, self.Hkv, self.D)).astype(np.float32)
                x[..., rng.permutation(self.D)[:2]] *= np.float32(mult)
                src = self.stored(O.bf16_from_f32(x), bits)
                for row in range(n):
                    page = self.table[b, row // self.R]
                    if 0 <= page < self.pages:
                        for dst, s in zip(side, src):
                            dst[page, :, row % self.R] = s[row]
        return self

    def rows(self, b, h, n):
        """(valid [n], keys [n, D], values [n, D], scores' magnitude [n, D]) in f64."""
        r = np.arange(n)
        page = self.table[b, r // self.R]
        ok = (page >= 0) & (page < self.pages)
        at = (np.where(ok, page, 0), h, r % self.R)
        k = values_of([t[at] for t in self.sides[0]], self.bk, self.gs)
        v = values_of([t[at] for t in self.sides[1]], self.bv, self.gs)
        big = np.abs(k)
        if self.bk != 16:  # the codes enter the products with up to 128 added
            s, z = (np.repeat(np.abs(O.bf16_to_f32(t[at]).astype(np.float64)), self.gs, axis=-1)
                    for t in self.sides[0][1:])
            big = s * (codes_of(self.sides[0][0][at], self.bk) + 256.0) + z
        return ok, k, v, big

    def attend(self, q, scale, window=-1, max_rows=None):
        """q bf16 [B, H, D]: (output f64, its tolerance, weights to add f64,
        theirs). The tolerances count roundings: half a bf16 step of the
        output (2^-8 of it); each weight's, 2^-16 as a bf16 pair (2^-8 of what
        the first part's 2^-8 left), 2^-11 as the f16 that affine rows take,
        and there each value's as f16 too (half a step of 10 stored bits,
        2^-11: 2^-11 + 2^-11 = 2^-10 of a term), with
        what f16 loses of small weights (2^-32 of the largest) and small
        values (2^-30 of the largest); the f32 score sums (a step 2^-24 an
        addition of the products' magnitudes) and exp2's argument and result,
        which move a weight by their size."""
        H, D = q.shape[1], self.D
        G = H // self.Hkv
        qf = O.bf16_to_f32(q).astype(np.float64)
        out = np.zeros((self.B, H, D))
        tol = np.zeros_like(out)
        gain = np.zeros((self.B, self.Hkv, self.stride * self.R))
        gtol = np.zeros_like(gain)
        for b in range(self.B):
            n = min(max(int(self.lens[b]), 0), self.stride * self.R, max_rows or 1 << 60)
            lo = max(0, n - window) if window > 0 else 0
            for h in range(self.Hkv):
                if n == 0:
                    continue
                ok, k, v, big = self.rows(b, h, n)
                ok[:lo] = False
                if not ok.any():
                    continue
                k, v, big, r = k[ok], v[ok], big[ok], np.nonzero(ok)[0]
                for e in range(h * G, (h + 1) * G):
                    s = k @ qf[b, e] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    sums = (D + 16) * 2.0 ** -24 * (big @ np.abs(qf[b, e])).max() * abs(scale)
                    d = 2 * (sums + 2.0 ** -22 * (np.abs(s).max() + 4))  # of a weight, and of their sum
                    out[b, e] = p @ v
                    each = (2.0 ** -10 if self.bv != 16 else 2.0 ** -16) + d + n * 2.0 ** -24
                    tol[b, e] = 2.0 ** -8 * np.abs(out[b, e]) + 1.01 * each * (p @ np.abs(v)) + 1e-30
                    if self.bv != 16:
                        tol[b, e] += (n * 2.0 ** -32 * p.max() + 2.0 ** -30) * np.abs(v).max()
                    gain[b, h, r] += p
                    gtol[b, h, r] += (d + n * 2.0 ** -24) * p + 1e-12
        return out, tol, gain, gtol

    def choose(self, b, h, budget, sinks, recent):
        """Kept rows of (b, h), ascending."""
        n = min(max(int(self.lens[b]), 0), self.stride * self.R)
        if n <= budget:
            return np.arange(n)
        w = self.weights[b, h, :n].astype(np.float64)
        w[np.isnan(w)] = -np.inf
        mid = np.arange(sinks, n - recent)
        best = mid[np.lexsort((mid, -w[mid]))][:budget - sinks - recent]
        return np.sort(np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)]))

    def device(self, T):
        return OnDevice(T, self)


class OnDevice:
    """The pool uploaded, and the library's view of it."""

    def __init__(self, T, p):
        self.T, self.p = T, p
        self.sides = [[T.DeviceArray.of(t) for t in side] for side in p.sides]
        self.table, self.lens = T.DeviceArray.of(p.table), T.DeviceArray.of(p.lens)
        self.weights = T.DeviceArray.of(p.weights) if p.weights is not None else None

    def view(self, **other):
        p = self.p
        c = dict(kind=p.kind, batch=p.B, kv_heads=p.Hkv, dim=p.D, page_rows=p.R, num_pages=p.pages,
                 slots=[t.ptr for side in self.sides for t in side], table=self.table.ptr,
                 table_stride=p.stride, lens=self.lens.ptr,
                 weights=self.weights.ptr if self.weights is not None else None, group_size=p.gs,
                 bits_k=p.bk, bits_v=p.bv)
        c.update(other)
        return self.T.paged_kv(**c)

    def host(self):
        return [[t.numpy() for t in side] for side in self.sides]

    def attend(self, q, scale, window=-1, max_rows=None, workspace=True, stream=None):
        """Output bf16 [B, H, D] of a call (and the device array it is in)."""
        T, p, H = self.T, self.p, q.shape[1]
        kv = self.view()
        most = max_rows or p.stride * p.R
        dq = T.DeviceArray.of(q)
        out = T.DeviceArray((p.B, H, p.D), np.uint16, np.full((p.B, H, p.D), 0x7FC1, np.uint16))
        need = T.paged_decode_workspace_size(kv, H, most)
        # Whatever a workspace holds before the call is no answer.
        ws = T.DeviceArray((need,), np.uint8, np.full((need,), 0xFF, np.uint8)) if workspace else None
        T.paged_decode_attend(kv, dq.ptr, H * p.D, H, scale, most, out.ptr, window,
                              ws.ptr if ws else None, need if ws else 0, stream)
        T.hip().sync()
        return out.numpy()


def check(got, want, tol, tag):
    err = np.abs(np.asarray(got, np.float64) - want)
    worst = float(np.max(err / np.maximum(tol, 1e-300))) if err.size else 0.0
    print(f"[{tag}] worst error {worst:.3f} of its tolerance, max {err.max():.3e}", flush=True)
    assert np.all(np.isfinite(np.asarray(got, np.float64))), f"{tag}: non-finite"
    assert worst <= 1.0, tag
