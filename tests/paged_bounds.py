"""Bounds of the paged decode attention's error, row by row and channel by
channel, beside its values in 64 bits (from paged_ref.py's pool). What a call
computes for one (sequence, head), and how far each step may be off:

  scores   s_t = scale q.k_t. The products of D terms in f32, in any order: at
           most D + 16 additions, each 2^-24 of the terms' magnitudes. An affine
           key's terms are s c q and z q: the codes enter as they are. Queries
           enter affine products as f16 in a unit of the head's largest: parts
           below 2^-27 of it lose at most 2^-34 of it. exp2's argument and
           result, the scale in log2 units and the join's powers: at most
           sixteen roundings of 2^-24 of the score, or of 1.
  weights  p_t = 2^(s_t - m) / l. l: f32 sums, at most n / 16 + 64 a lane and
           part. As operands: a bf16 pair (2^-16 of each), or, over affine rows
           whose values have magnitudes within 2^16 of each other, f16 (half a
           step of 10 stored bits, 2^-11, and 2^-32 of the largest weight).
  values   bf16 rows are exact. Affine rows' are f16 (2^-11 of each, and 2^-21 of
           the largest value that their group's scale and bias allow) or, where
           magnitudes differ more, bf16 pairs (2^-16).
  output   f32 sums over the rows, at most n / 4 + 64 additions of 2^-24 of the
           terms' magnitudes; half a bf16 step, 2^-8 of the result.
"""
import numpy as np

import oracle_lib as O
from paged_ref import codes_of


def parts_of(p, side, bits, b, h, n):
    """(codes' part, bias' part, bound) [n, D] in f64, magnitudes, of the rows of
    one side; bf16 rows: (|x|, 0, |x|)."""
    r = np.arange(n)
    page = p.table[b, r // p.R]
    page = np.where((page >= 0) & (page < p.pages), page, 0)
    at = (page, h, r % p.R)
    if bits == 16:
        x = np.abs(O.bf16_to_f32(side[0][at]).astype(np.float64))
        return x, np.zeros_like(x), x
    s, z = (np.repeat(np.abs(O.bf16_to_f32(t[at]).astype(np.float64)), p.gs, axis=-1) for t in side[1:])
    return s * codes_of(side[0][at], bits), z, s * (2.0 ** bits - 1) + z


def attend(p, q, scale, window=-1, max_rows=None):
    """q bf16 [B, H, D]: (output f64, its bound, weights to add f64, theirs)."""
    H, D = q.shape[1], p.D
    G = H // p.Hkv
    qf = O.bf16_to_f32(q).astype(np.float64)
    out = np.zeros((p.B, H, D))
    tol = np.zeros_like(out)
    gain = np.zeros((p.B, p.Hkv, p.stride * p.R))
    gtol = np.zeros_like(gain)
    step = 2.0 ** -24
    for b in range(p.B):
        n = min(max(int(p.lens[b]), 0), p.stride * p.R, max_rows or 1 << 60)
        lo = max(0, n - window) if window > 0 else 0
        for h in range(p.Hkv):
            if n == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                ok, k, v, _ = p.rows(b, h, n)
                ok[:lo] = False
                if not ok.any():
                    continue
                ck, zk, _ = (t[ok] for t in parts_of(p, p.sides[0], p.bk, b, h, n))
                most = parts_of(p, p.sides[1], p.bv, b, h, n)[2][ok]
                k, v, r = k[ok], v[ok], np.nonzero(ok)[0]
                av = np.abs(v)
                # Rows that f16 weights can multiply: their bounds lie within 2^16
                # of the least that is not 0.
                some = most[np.isfinite(most) & (most > 0)]
                near = most <= (some.min() if some.size else 0.0) * 2.0 ** 16
                for e in range(h * G, (h + 1) * G):
                    x = np.abs(qf[b, e])
                    s = k @ qf[b, e] * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    d = (D + 16) * step * ((ck + zk) @ x) * abs(scale)
                    if p.bk != 16:
                        d = d + 2.0 ** -34 * x.max() * ck.sum(1) * abs(scale)
                    d = d + 16 * step * (np.abs(s) + np.abs(s).max() + 1)
                    sums = (len(r) / 16 + 64) * step
                    o = w @ v
                    pv = w @ av
                    t = (w * d) @ av + (w @ d + sums) * np.abs(o) + (len(r) / 4 + 64) * step * pv
                    if p.bv == 16:
                        t += 2.0 ** -16 * pv
                    else:
                        t += (2.0 ** -11 + 2.0 ** -11) * pv + 2.0 ** -21 * (w @ most)
                        t += 2.0 ** -32 * w.max() * np.where(near, av, 0.0).sum(0)
                    out[b, e] = o
                    tol[b, e] = 1.01 * t + 2.0 ** -8 * np.abs(o) + 2.0 ** -133
                    gain[b, h, r] += w
                    gtol[b, h, r] += 1.01 * (d + w @ d + sums) * w + 2.0 ** -86
    return out, tol, gain, gtol


def errors(got, want, tol):
    """Error over bound; infinities and NaN count 0 where both have the same."""
    got = np.asarray(got, np.float64)
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        err = np.where(np.isfinite(want), np.abs(got - want) / tol, np.inf)
    return np.where(same, 0.0, np.where(np.isnan(err), np.inf, err))


def check(got, want, tol, tag):
    err = errors(got, want, tol)
    worst = float(err.max()) if err.size else 0.0
    print(f"[{tag}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{tag}: {np.count_nonzero(err > 1.0)} of {err.size} beyond their bounds"
