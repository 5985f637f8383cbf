"""Operators of the paged KV cache, measured: the append, the decode attention that reads the pages, the eviction.

A pool holds pages of `page` rows, [pages, KV heads, page, .] in every buffer (bf16 rows, or the affine triple of
packed codes, scales and biases); a sequence's rows are the pages that its row of the table names. `kind` of a case:

  append  new tokens' keys and values into the pages, from a (possibly strided) projection buffer
  attend  one new token's attention over the pages, `track` adding each row's attention weight to its running sum
  evict   keep the heaviest rows of every KV head (with the first and the last ones), moved to new pages

Where `own` is false, run() computes the plain form with elementary torch operations; where it is true, run() makes
the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_CHUNK = 1 << 25  # elements handled at a time while inputs are made


def _T():
    """The framework's binding, on the HIP runtime that torch has loaded (one runtime a process)."""
    path = os.path.join(_ROOT, "lumen-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tqkv
    if tqkv._hip is None:
        lib = os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")
        if os.path.exists(lib):
            tqkv.HIP_PATH = lib
    return tqkv


# ------------------------------------------------------------------ cases
def _append(**c):
    return dict(dict(kind="append", H=0, Hkv=8, D=128, page=64, bk=16, bv=16, gs=64, held=0, track=False), **c)


def _attend(**c):
    return dict(dict(kind="attend", H=32, Hkv=8, D=128, page=64, bk=16, bv=16, gs=64, ragged=True, window=-1, track=False), **c)


def _evict(**c):
    return dict(dict(kind="evict", Hkv=8, D=128, page=64, bk=16, bv=16, gs=64, ragged=True, sinks=4), **c)


def listed():
    return [
        # A serving batch's decode step: one token a sequence, read out of the fused QKV projection. Latency.
        _append(name="append_step", B=64, new=1, held=700, H=32, page=16, track=True),
        # Prompts of a prefill batch, ragged, into a bf16 pool out of the fused projection. HBM bandwidth.
        _append(name="append_prompts_bf16", B=12, new=4096, H=32),
        # The same into a 4-bit pool: quantized on the way.
        _append(name="append_prompts_4bit", B=6, new=4096, bk=4, bv=4),
        # A single user's decode step at a short context: the smallest call, latency.
        _attend(name="attend_single_short", B=1, n=777, ragged=False, page=16),
        # A single user far into a long document: the work of one sequence split over the whole card.
        _attend(name="attend_single_long", B=1, n=131071, ragged=False),
        # A ragged serving batch over a 4-bit pool, 17 to 16,000 rows a sequence.
        _attend(name="attend_ragged_4bit", B=32, n=16000, bk=4, bv=4),
        # Full-size contexts, head dim 256, two query heads a KV head, 4-bit: HBM bandwidth.
        _attend(name="attend_batch_32k", B=16, H=16, D=256, n=32768, ragged=False, bk=4, bv=4),
        # Full-attention layers of head dim 512 with 16 query heads a KV head, bf16.
        _attend(name="attend_wide_heads", B=4, H=32, Hkv=2, D=512, n=8179, ragged=False, page=32),
        # A sliding-window layer: 8-bit keys and values, groups of 32, the last 1,024 rows of long sequences.
        _attend(name="attend_window_8bit", B=8, H=16, D=256, n=20000, ragged=False, window=1024, bk=8, bv=8, gs=32),
        # A step whose attention weights steer the eviction: each row's weight added to its running sum.
        _attend(name="attend_tracked", B=16, n=8192, track=True),
        # One long sequence cut back to its budget.
        _evict(name="evict_single", B=1, n=16384, budget=2048, recent=128, ragged=False),
        # A batch over a 4-bit pool cut back to its budget.
        _evict(name="evict_batch_4bit", B=16, n=30000, budget=4096, recent=256, bk=4, bv=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "attend", "evict"))
    D = rng.choice((64, 128, 128, 256, 512))
    bk, bv = rng.choice(((16, 16), (16, 16), (4, 4), (8, 8), (8, 4)))
    gs = rng.choice((32, 64, 64, 128)) if D > 64 else rng.choice((32, 64))
    page = rng.choice((16, 16, 32, 64, 64, 128, 256))
    if kind == "append":
        c = _append(B=_log(rng, 1, 64), new=_log(rng, 1, 4096), Hkv=rng.choice((1, 2, 8, 16)), D=D, page=page, bk=bk, bv=bv, gs=gs,
                    held=rng.choice((0, rng.randint(1, 500))), track=rng.random() < 0.3)
        c["H"] = c["Hkv"] * rng.choice((0, 1, 4))
        while work(c)["bytes"] > 4e8:
            c["new"] = c["new"] // 2 + 1
        return c
    if kind == "attend":
        Hkv = rng.choice((1, 2, 4, 8))
        c = _attend(B=_log(rng, 1, 64), H=Hkv * rng.choice((1, 2, 3, 4, 5, 7, 8, 16) if Hkv < 8 else (1, 2, 4, 4, 6, 8)), Hkv=Hkv, D=D, n=_log(rng, 1, 131072), page=page,
                    bk=bk, bv=bv, gs=gs, ragged=rng.random() < 0.7, track=rng.random() < 0.25)
        c["window"] = rng.choice((-1, -1, -1, rng.randint(1, 4096)))
        while c["B"] * c["Hkv"] * c["n"] * _row_bytes(c) > 9e8:
            c["n"] = c["n"] // 2 + 1
        return c
    n = _log(rng, 64, 65536)
    c = _evict(B=_log(rng, 1, 32), Hkv=rng.choice((1, 2, 8)), D=D, n=n, page=page, bk=bk, bv=bv, gs=gs, ragged=rng.random() < 0.7, sinks=rng.choice((0, 1, 4, 7)))
    while c["B"] * c["Hkv"] * c["n"] * _row_bytes(c) > 5e8:
        c["n"] = c["n"] // 2 + 1
    c["budget"] = max(16, int(c["n"] * rng.uniform(0.05, 0.9)))
    c["recent"] = rng.randint(0, c["budget"] - c["sinks"])
    return c


# ------------------------------------------------------------------ sizes
def _side_bytes(c, bits):
    return 2 * c["D"] if bits == 16 else c["D"] * bits // 8 + 4 * (c["D"] // c["gs"])


def _row_bytes(c):
    """Bytes of one row, keys and values, of one KV head."""
    return _side_bytes(c, c["bk"]) + _side_bytes(c, c["bv"])


def _lens(c):
    """Rows that each sequence holds (for an append: after it), from the case alone."""
    r = random.Random(sum((i + 1) * ord(ch) for i, ch in enumerate(repr(sorted((k, v) for k, v in c.items() if k != "name")))))
    if c["kind"] == "append":
        return [c["held"] + n for n in _news(c)]
    if not c["ragged"]:
        return [c["n"]] * c["B"]
    got = [_log(r, min(17, c["n"]), c["n"]) for _ in range(c["B"])]
    if c["B"] >= 4 and c["n"] < 1000:
        got[r.randrange(c["B"])] = 0  # a batch slot that holds nothing yet
    return got


def _news(c):
    """New tokens of each sequence of an append."""
    r = random.Random(c["B"] * 7919 + c["new"])
    return [1 if c["new"] == 1 else r.randint(int(b == 0), c["new"]) for b in range(c["B"])]


def work(case):
    c = case
    lens = _lens(c)
    if c["kind"] == "append":
        t = sum(_news(c))
        return {"bytes": t * c["Hkv"] * (4 * c["D"] + _row_bytes(c) + (4 if c["track"] else 0)), "flops": 0}
    if c["kind"] == "attend":
        seen = sum(min(n, c["window"]) if c["window"] > 0 else n for n in lens)
        return {"bytes": seen * c["Hkv"] * (_row_bytes(c) + (8 if c["track"] else 0)) + 4 * c["B"] * c["H"] * c["D"], "flops": 4 * seen * c["H"] * c["D"]}
    moved = sum(min(n, c["budget"]) for n in lens)
    return {"bytes": c["Hkv"] * (4 * sum(lens) + moved * (2 * _row_bytes(c) + 8)), "flops": 0}


# ------------------------------------------------------------------ plain building blocks
def _away(x):
    """Rounds to whole numbers, halves away from zero."""
    t = torch.trunc(x)
    return t + torch.where((x - t).abs() >= 0.5, torch.sign(x), torch.zeros_like(x))


def _quantize(x, bits, gs):
    """(packed words as int32, scales, biases) of bf16 rows [..., D]: the cache's affine format, in 32 bits."""
    lead, D = x.shape[:-1], x.shape[-1]
    v = x.float().reshape(-1, D // gs, gs)
    bins = torch.tensor(float(2 ** bits - 1), device=x.device)  # a tensor: a divide by a plain number is a multiply
    lo, hi = v.amin(-1), v.amax(-1).clamp_min(0.0)
    scale = torch.clamp_min((hi - lo) / bins, 1e-7)
    side = lo.abs() > hi.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, lo, hi)
    q0 = _away(edge / scale)
    zero = q0 == 0
    scale = torch.where(zero, scale, edge / torch.where(zero, torch.ones_like(q0), q0))
    bias = torch.where(zero, torch.zeros_like(edge), edge)
    code = _away((v - bias[..., None]) / scale[..., None]).clamp(0.0, float(2 ** bits - 1))
    code = code.to(torch.int32).reshape(-1, D * bits // 32, 32 // bits)  # 4 and 8 bits: no code straddles a word
    words = torch.zeros(code.shape[:-1], dtype=torch.int32, device=x.device)
    for i in range(32 // bits):
        words |= code[..., i] << (i * bits)
    return (words.reshape(*lead, D * bits // 32), scale.to(torch.bfloat16).reshape(*lead, D // gs), bias.to(torch.bfloat16).reshape(*lead, D // gs))


def _values(t, bits, gs, dtype=torch.float32):
    """The values that stored rows stand for: bf16 rows, or scale * code + bias."""
    if bits == 16:
        return t[0].to(dtype)
    words, scales, biases = t
    lead, D = words.shape[:-1], words.shape[-1] * 32 // bits
    shift = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    code = ((words[..., None] >> shift) & (2 ** bits - 1)).to(dtype).reshape(*lead, D // gs, gs)
    return (code * scales.to(dtype)[..., None] + biases.to(dtype)[..., None]).reshape(*lead, D)


class _Rand:
    """Seeded draws on the device."""

    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda")
        salt = sum((i + 1) * ord(ch) for i, ch in enumerate(repr(sorted((k, v) for k, v in case.items() if k != "name")))) % 100003
        self.g.manual_seed(int(seed) * 100003 + salt)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def rows(self, *shape):
        """bf16 K or V rows: N(0, 1) with 2% of the channels four times larger."""
        big = self.uniform(shape[-1]) < 0.02
        return (self.normal(*shape) * torch.where(big, 4.0, 1.0)).to(torch.bfloat16)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _pool(c, r, pages):
    """Buffers of a pool, all rows filled: K's, then V's."""
    out = []
    for bits in (c["bk"], c["bv"]):
        lead = (pages, c["Hkv"], c["page"])
        if bits == 16:
            side = [torch.empty(*lead, c["D"], dtype=torch.bfloat16, device="cuda")]
        else:
            side = [torch.empty(*lead, c["D"] * bits // 32, dtype=torch.int32, device="cuda")]
            side += [torch.empty(*lead, c["D"] // c["gs"], dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        step = max(1, _CHUNK // (c["Hkv"] * c["page"] * c["D"]))
        for a in range(0, pages, step):
            x = r.rows(min(step, pages - a), c["Hkv"], c["page"], c["D"])
            for dst, src in zip(side, [x] if bits == 16 else _quantize(x, bits, c["gs"])):
                dst[a:a + step] = src
        out.append(side)
    return out


def _pages(c, n):
    return (n + c["page"] - 1) // c["page"]


def _handle(s, c, table, lens, weights=None):
    """The framework's view of the pool, as a program keeps it between calls."""
    T = _T()
    kind = T.CACHE_BF16 if c["bk"] == 16 else T.CACHE_AFFINE
    ptrs = [t.data_ptr() for side in s["pool"] for t in side]
    return T.paged_kv(kind, c["B"], c["Hkv"], c["D"], c["page"], s["pool"][0][0].shape[0], ptrs, table.data_ptr(), table.shape[1], lens.data_ptr(),
                      None if weights is None else weights.data_ptr(), c["gs"], c["bk"], c["bv"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = {k: v for k, v in case.items() if k != "name"}
    r = _Rand(c, seed)
    lens = _lens(c)
    width = max(1, max(_pages(c, n) for n in lens))
    held = [_pages(c, n) for n in lens]
    extra = [_pages(c, min(n, c["budget"])) for n in lens] if c["kind"] == "evict" else []
    total = sum(held)
    s = {"case": c, "lens": lens, "dlens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "pool": _pool(c, r, max(1, total + sum(extra)))}
    order = r.perm(total).to(torch.int32) if total else torch.zeros(0, dtype=torch.int32, device="cuda")
    s["table"] = torch.full((c["B"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, p in enumerate(held):
        s["table"][b, :p] = order[at:at + p]
        at += p
    rows = width * c["page"]
    if c["kind"] == "append":
        heads, news = c["H"] + 2 * c["Hkv"], _news(c)
        t = sum(news)
        s["qkv"] = r.rows(max(t, 1), heads, c["D"])  # K's heads behind the queries', V's behind K's
        s["tokens"] = t
        s["starts"] = torch.tensor([sum(news[:b]) for b in range(c["B"] + 1)], dtype=torch.int32, device="cuda")
        if c["track"]:
            s["weights"] = r.uniform(c["B"], c["Hkv"], rows)
    elif c["kind"] == "attend":
        s["q"] = r.normal(c["B"], c["H"], c["D"]).to(torch.bfloat16)
        if c["track"]:
            s["weights"] = 4.0 * r.uniform(c["B"], c["Hkv"], rows) ** 8
    else:
        # Running sums are heavy-tailed, and a fifth of the rows was never looked at.
        w = torch.exp(2.0 * r.normal(c["B"], c["Hkv"], rows))
        s["weights"] = torch.where(r.uniform(c["B"], c["Hkv"], rows) < 0.2, torch.zeros_like(w), w)
        width2 = max(1, _pages(c, c["budget"]))
        s["dst"] = torch.full((c["B"], width2), -1, dtype=torch.int32, device="cuda")
        order, at = (r.perm(sum(extra)) + total).to(torch.int32), 0
        for b, p in enumerate(extra):
            s["dst"][b, :p] = order[at:at + p]
            at += p
        s["first"] = total  # the new pages are the pool's last ones
    if own:
        T = _T()
        if c["kind"] == "attend" and c["track"]:
            s["now"] = torch.empty_like(s["weights"])
        s["kv"] = _handle(s, c, s["table"], s["dlens"], s.get("now", s.get("weights")))
        if c["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            s["ws"] = torch.empty(max(16, T.paged_decode_workspace_size(s["kv"], c["H"], rows)), dtype=torch.uint8, device="cuda")
        elif c["kind"] == "evict":
            s["ws"] = torch.empty(max(16, T.paged_evict_workspace_size(s["kv"], c["budget"])), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    return {"append": _run_append, "attend": _run_attend, "evict": _run_evict}[c["kind"]](s, c)


def _held_values(s, c, first=0):
    """What the pool's pages from `first` on stand for: bf16 pools themselves, quantized ones dequantized."""
    if c["bk"] == 16:
        return [side[0][first:] for side in s["pool"]]
    if not own:
        return [_values([t[first:] for t in side], bits, c["gs"]).to(torch.bfloat16) for side, bits in zip(s["pool"], (c["bk"], c["bv"]))]
    T, out = _T(), []
    for side, bits in zip(s["pool"], (c["bk"], c["bv"])):
        words, scales, biases = (t[first:] for t in side)
        x = torch.empty(*words.shape[:-1], c["D"], dtype=torch.bfloat16, device="cuda")
        T.affine_dequantize(words.data_ptr(), scales.data_ptr(), biases.data_ptr(), x.numel() // c["D"], c["D"], c["gs"], bits, x.data_ptr(), _stream())
        out.append(x)
    return out


def _run_append(s, c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    k, v = s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]
    if own:
        _T().paged_append(s["kv"], k.data_ptr(), v.data_ptr(), None if c["new"] == 1 else s["starts"].data_ptr(), s["tokens"], s["qkv"].stride(0), D, _stream())
    elif s["tokens"]:
        count = (s["starts"][1:] - s["starts"][:-1]).long()
        b = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), count, output_size=s["tokens"])
        row = torch.arange(s["tokens"], device="cuda") - s["starts"].long()[b] + (s["dlens"].long() - count)[b]
        page = s["table"].long()[b, row // c["page"]]
        for x, side, bits in ((k, s["pool"][0], c["bk"]), (v, s["pool"][1], c["bv"])):
            for dst, src in zip(side, [x] if bits == 16 else _quantize(x[:s["tokens"]], bits, c["gs"])):
                dst[page, :, row % c["page"]] = src[:s["tokens"]]
        if c["track"]:
            s["weights"][b, :, row] = 0.0
    out = {"pool": _held_values(s, c)}
    if c["track"]:
        out["weights"] = s["weights"]
    return out


def _sequence(s, c, b, i, dtype=torch.float32):
    """Values [Hkv, n, D] of sequence b's keys (i = 0) or values (i = 1)."""
    n = s["lens"][b]
    pages = s["table"][b, :_pages(c, n)].long()
    x = _values([t[pages] for t in s["pool"][i]], (c["bk"], c["bv"])[i], c["gs"], dtype)
    return x.permute(1, 0, 2, 3).reshape(c["Hkv"], -1, c["D"])[:, :n]


def _run_attend(s, c):
    scale = c["D"] ** -0.5
    if own:
        if c["track"]:
            s["now"].copy_(s["weights"])  # the sums so far: every pass starts from them
        _T().paged_decode_attend(s["kv"], s["q"].data_ptr(), c["H"] * c["D"], c["H"], scale, s["table"].shape[1] * c["page"], s["out"].data_ptr(),
                                 c["window"], s["ws"].data_ptr(), s["ws"].numel(), _stream())
        return {"out": s["out"], "weights": s["now"]} if c["track"] else {"out": s["out"]}
    out = torch.zeros_like(s["q"])
    now = s["weights"].clone() if c["track"] else None
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        lo = max(0, n - c["window"]) if c["window"] > 0 else 0
        k, v = (_sequence(s, c, b, i)[:, lo:] for i in (0, 1))
        q = s["q"][b].float().reshape(c["Hkv"], -1, c["D"])
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        x = torch.exp(x - x.amax(-1, keepdim=True))
        p = x / x.sum(-1, keepdim=True)
        out[b] = torch.matmul(p, v.contiguous()).reshape(c["H"], c["D"]).to(torch.bfloat16)
        if c["track"]:
            now[b, :, lo:n] += p.sum(1)
    return {"out": out, "weights": now} if c["track"] else {"out": out}


def _choose(w, n, c):
    """Rows kept of each KV head, ascending [Hkv, m]: the first, the last, the heaviest between (ties: the lower row)."""
    m = min(n, c["budget"])
    if n <= c["budget"]:
        return torch.arange(n, device=w.device).expand(c["Hkv"], n)
    key = w[:, :n].clone()
    key[:, :c["sinks"]] = math.inf
    key[:, n - c["recent"]:] = math.inf
    first = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :m]
    return torch.sort(first, dim=1)[0]


def _run_evict(s, c):
    B, Hkv, m = c["B"], c["Hkv"], c["budget"]
    kept = torch.full((B, Hkv, m), -1, dtype=torch.int32, device="cuda")
    lens = torch.empty(B, dtype=torch.int32, device="cuda")
    new = torch.zeros(B, Hkv, s["dst"].shape[1] * c["page"], device="cuda")
    if own:
        _T().paged_evict(s["kv"], m, c["sinks"], c["recent"], s["dst"].data_ptr(), s["dst"].shape[1], lens.data_ptr(), new.data_ptr(), kept.data_ptr(),
                         s["ws"].data_ptr(), s["ws"].numel(), _stream())
    else:
        lens.copy_(s["dlens"].clamp_max(m))
        for b, n in enumerate(s["lens"]):
            if n == 0:
                continue
            at = _choose(s["weights"][b], n, c)
            k = at.shape[1]
            kept[b, :, :k] = at.to(torch.int32)
            new[b, :, :k] = torch.gather(s["weights"][b], 1, at)
            head = torch.arange(Hkv, device="cuda")[:, None]
            to = torch.arange(k, device="cuda")[None]
            src, dst = s["table"][b].long()[at // c["page"]], s["dst"][b].long()[to // c["page"]]
            for side in s["pool"]:
                for t in side:
                    t[dst, head, to % c["page"]] = t[src, head, at % c["page"]]
    return {"kept": kept, "lens": lens, "weights": new, "pool": _held_values(s, c, s["first"])}


# ------------------------------------------------------------------ 64 bits
def _exact_code(x, bits, gs):
    """(codes, scales, biases) in 64 bits of a quantized row. The format fixes the quotients: the step, the end's place and
    each element's place are IEEE quotients and differences of 32-bit values, so these are taken in 32 bits here too."""
    g = x.float().unflatten(-1, (-1, gs))
    low, none = g.min(-1, keepdim=True)[0], torch.zeros((), device=x.device)
    high = torch.maximum(g.max(-1, keepdim=True)[0], none)
    step = torch.maximum((high - low) / torch.full_like(low, 2 ** bits - 1), torch.full_like(low, 1e-7))
    down = low.abs() > high.abs()
    step, end = torch.where(down, step, -step), torch.where(down, low, high)

    def whole(r):  # halves away from zero; the half is added in 64 bits, where it is exact
        return torch.floor(r.double().abs() + 0.5) * torch.sign(r).double()

    at = whole(end / step).float()
    step = torch.where(at == 0, step, end / torch.where(at == 0, torch.ones_like(at), at))
    base = torch.where(at == 0, none, end)
    return whole((g - base) / step).clamp(0, 2 ** bits - 1), step.to(torch.bfloat16).double(), base.to(torch.bfloat16).double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = s["case"]
    page, table = c["page"], s["table"].cpu()

    def stored(i, first=0):
        """The pool's keys or values in 64 bits."""
        bits, side = (c["bk"], c["bv"])[i], s["pool"][i]
        if bits == 16:
            return side[0][first:].double()
        words = side[0][first:]
        codes = torch.stack([(words >> o) & (2 ** bits - 1) for o in range(0, 32, bits)], -1).double().flatten(-2)
        return codes * side[1][first:].double().repeat_interleave(c["gs"], -1) + side[2][first:].double().repeat_interleave(c["gs"], -1)

    if c["kind"] == "append":
        pools, weights = [stored(0), stored(1)], s.get("weights")
        news, t = _news(c), 0
        for b, count in enumerate(news):
            x = s["qkv"][t:t + count, c["H"]:]
            t += count
            for i, bits in enumerate((c["bk"], c["bv"])):
                y = x[:, i * c["Hkv"]:(i + 1) * c["Hkv"]]
                if bits != 16:
                    code, step, base = _exact_code(y, bits, c["gs"])
                    y = (code * step + base).flatten(-2)
                done = 0
                while done < count:  # page by page
                    row = c["held"] + done
                    k = min(count - done, page - row % page)
                    pools[i][int(table[b, row // page]), :, row % page:row % page + k] = y[done:done + k].double().transpose(0, 1)
                    done += k
            if c["track"]:
                weights[b, :, c["held"]:c["held"] + count] = 0.0
        return {"pool": pools, "weights": weights.double()} if c["track"] else {"pool": pools}
    if c["kind"] == "attend":
        out = torch.zeros(c["B"], c["H"], c["D"], dtype=torch.float64, device="cuda")
        now = s["weights"].double() if c["track"] else None
        group = c["H"] // c["Hkv"]
        for b, n in enumerate(s["lens"]):
            if n == 0:
                continue
            begin = n - c["window"] if 0 < c["window"] < n else 0
            rows = torch.arange(begin, n, device="cuda")
            where = s["table"][b].long()[rows // page]
            for h in range(c["Hkv"]):
                k, v = ([t[where, h, rows % page] for t in side] for side in s["pool"])
                if c["bk"] == 16:
                    k, v = k[0].double(), v[0].double()
                else:
                    k, v = (torch.stack([(t[0] >> o) & (2 ** bits - 1) for o in range(0, 32, bits)], -1).double().flatten(-2)
                            * t[1].double().repeat_interleave(c["gs"], -1) + t[2].double().repeat_interleave(c["gs"], -1)
                            for t, bits in ((k, c["bk"]), (v, c["bv"])))
                for g in range(group):
                    e = h * group + g
                    x = torch.mv(k, s["q"][b, e].double()) / math.sqrt(c["D"])
                    p = torch.exp(x - x.max())
                    p = p / p.sum()
                    out[b, e] = torch.mv(v.t().contiguous(), p)
                    if c["track"]:
                        now[b, h, begin:n] += p
        return {"out": out, "weights": now} if c["track"] else {"out": out}
    m = c["budget"]
    kept = torch.full((c["B"], c["Hkv"], m), -1, dtype=torch.int64)
    lens = torch.tensor([min(n, m) for n in s["lens"]])
    new = torch.zeros(c["B"], c["Hkv"], s["dst"].shape[1] * page, dtype=torch.float64)
    every = s["weights"].cpu()
    dst = s["dst"].cpu()
    pools = [stored(0), stored(1)]
    for b, n in enumerate(s["lens"]):
        for h in range(c["Hkv"]):
            w = every[b, h, :n].double()
            rows = torch.arange(n)
            if n > m:  # the m-th largest of the rows between decides; its ties go to the lowest rows
                free = torch.zeros(n, dtype=torch.bool)
                free[c["sinks"]:n - c["recent"]] = True
                room = m - c["sinks"] - c["recent"]
                take = ~free
                if room:
                    cut = torch.topk(w[free], room)[0][-1]
                    take |= free & (w > cut)
                    ties = torch.nonzero(free & (w == cut))[:, 0]
                    take[ties[:m - int(take.sum())]] = True
                rows = torch.nonzero(take)[:, 0]
            k = len(rows)
            if k == 0:
                continue
            kept[b, h, :k] = rows
            new[b, h, :k] = w[rows]
            to = torch.arange(k)
            a = (table[b].long()[rows // page].cuda(), h, (rows % page).cuda())
            z = (dst[b].long()[to // page].cuda(), h, (to % page).cuda())
            for p in pools:
                p[z] = p[a]
    return {"kept": kept, "lens": lens, "weights": new, "pool": [p[s["first"]:] for p in pools]}
