"""Operators around the paged KV cache, measured: its page tables, rotary positions, and the attention of whole prompts.

`kind` of a case:

  tables  finished sequences give their pages back, then new tokens get pages, slots and positions
  rope    rotary positions applied to the heads of a (possibly fused) projection
  enter   queries rotated, keys rotated and written with the values into the slots of their pages (bf16 rows)
  packed  attention of sequences that lie one behind the other, keys and values read out of the fused projection
  paged   attention of each sequence's newest tokens over all of its rows in the pages (bf16 or affine rows)

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
def _tables(**c):
    return dict(dict(kind="tables", page=16, spare=1.0, done=0.0), **c)


def _rope(**c):
    return dict(dict(kind="rope", H=40, D=128, rd=128, pairs="halves", scaling="none", factor=1.0, far=8192, beside=8), **c)


def _enter(**c):
    return dict(dict(kind="enter", H=32, Hkv=8, D=128, rd=128, pairs="halves", scaling="none", factor=1.0, page=16), **c)


def _packed(**c):
    return dict(dict(kind="packed", H=32, Hkv=8, D=128, ragged=True, causal=True, window=-1), **c)


def _paged(**c):
    return dict(dict(kind="paged", H=32, Hkv=8, D=128, page=64, bk=16, bv=16, gs=64, ragged=True, window=-1), **c)


def listed():
    return [
        # A decode step of a full serving batch: one token a sequence, a page for the few that cross one, some slots finished. Latency.
        _tables(name="tables_step", B=256, held=6000, new=1, done=0.02),
        # Prompts admitted to a batch whose other sequences have finished: pages and slots of 40,000 tokens.
        _tables(name="tables_prompts", B=24, held=3000, new=4096, page=64, done=0.7),
        # A decode step's queries and keys out of the fused projection, far into a long context. Latency.
        _rope(name="rope_step", tokens=64, scaling="ramp", factor=16.0, far=131072),
        # Prompts' heads of 256 channels, a quarter of them rotated, neighbours as pairs, positions divided. HBM bandwidth.
        _rope(name="rope_prompts", tokens=20011, H=24, D=256, rd=64, pairs="neighbours", scaling="linear", factor=8.0, beside=0),
        # A decode step's queries rotated, keys rotated and appended with the values, one call. Latency.
        _enter(name="enter_step", B=64, new=1, held=2000, scaling="bands", factor=8.0),
        # The same for the prompts of a prefill batch. HBM bandwidth.
        _enter(name="enter_prompts", B=10, new=4096, held=0, page=64),
        # A single user's short prompt: the smallest attention, latency.
        _packed(name="packed_short", B=1, n=77, ragged=False),
        # A prefill batch of ragged prompts up to 8,192 tokens. Matrix products.
        _packed(name="packed_prompts", B=8, n=8192),
        # A prefill chunk of two long documents over a 4-bit pool. Matrix products.
        _paged(name="paged_chunk_4bit", B=2, n=30011, new=2048, bk=4, bv=4, ragged=False),
        # Drafted tokens of a serving batch checked against their bf16 pages: 6 tokens a sequence. HBM bandwidth.
        _paged(name="paged_drafts", B=32, n=24000, new=6, page=16),
        # A sliding-window layer's chunk: head dim 256, 8-bit keys and values in groups of 32, the last 1,024 rows.
        _paged(name="paged_window_8bit", B=6, H=16, D=256, n=5000, new=1500, bk=8, bv=8, gs=32, window=1024),
        # Full-attention layers of head dim 512, 16 query heads a KV head, bf16.
        _paged(name="paged_wide_heads", B=3, Hkv=2, D=512, n=4099, new=1023, page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _scaled(rng):
    s = rng.choice(("none", "none", "linear", "base", "bands", "ramp"))
    return dict(scaling=s, factor=1.0 if s == "none" else rng.choice((2.0, 3.5, 8.0, 32.0)))


def draw(rng):
    kind = rng.choice(("tables", "rope", "enter", "packed", "packed", "paged", "paged", "paged"))
    D = rng.choice((64, 128, 128, 256, 512))
    page = rng.choice((16, 16, 32, 64, 64, 128, 256))
    if kind == "tables":
        new = rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 2, 4096)))
        c = _tables(B=_log(rng, 1, 512), held=_log(rng, 1, 20000), new=new, page=page, spare=rng.choice((1.0, 1.0, 0.5)), done=rng.choice((0.0, 0.1, 0.6)))
        while c["B"] * c["new"] > 100000:
            c["new"] = c["new"] // 2 + 1
        while c["B"] * c["held"] // page > 400000:
            c["held"] //= 2
        return c
    if kind == "rope":
        c = _rope(tokens=_log(rng, 1, 20000), H=rng.randint(1, 64), D=D, rd=rng.choice((D, D, D // 2, D // 4, 2 * rng.randint(1, D // 2))),
                  pairs=rng.choice(("halves", "neighbours")), far=_log(rng, 100, 1 << 20), beside=rng.choice((0, 1, 8)), **_scaled(rng))
        while c["tokens"] * (c["H"] + c["beside"]) * D > 1.2e8:
            c["tokens"] = c["tokens"] // 2 + 1
        return c
    if kind == "enter":
        Hkv = rng.choice((1, 2, 4, 8, 16))
        c = _enter(B=_log(rng, 1, 64), new=rng.choice((1, _log(rng, 2, 4096))), held=rng.choice((0, _log(rng, 1, 20000))), H=Hkv * rng.choice((1, 2, 4, 5, 8)), Hkv=Hkv,
                   D=D, rd=rng.choice((D, D, D // 2, D // 4, 2 * rng.randint(1, D // 2))), pairs=rng.choice(("halves", "neighbours")), page=page, **_scaled(rng))
        while c["B"] * c["new"] * (c["H"] + 2 * Hkv) * D > 1.2e8:
            c["new"] = c["new"] // 2 + 1
        while c["B"] * c["held"] * Hkv * D > 4e8:
            c["held"] //= 2
        return c
    Hkv = rng.choice((1, 2, 4, 8))
    H = Hkv * rng.choice((1, 2, 3, 4, 5, 7, 8, 16) if Hkv < 8 else (1, 2, 4, 4, 6))
    window = rng.choice((-1, -1, -1, _log(rng, 1, 4096)))
    if kind == "packed":
        c = _packed(B=_log(rng, 1, 32), n=_log(rng, 1, 8192), H=H, Hkv=Hkv, D=D, ragged=rng.random() < 0.7, window=window, causal=window > 0 or rng.random() < 0.8)
        while work(c)["flops"] > 1.2e12 or c["B"] * c["n"] * (H + 2 * Hkv) * D > 4e8 or c["n"] * c["n"] * H > 4e9:
            c["n"] = c["n"] // 2 + 1
        return c
    bk, bv = rng.choice(((16, 16), (16, 16), (4, 4), (8, 8), (8, 4)))
    gs = rng.choice((32, 64, 64, 128)) if D > 64 else rng.choice((32, 64))
    c = _paged(B=_log(rng, 1, 32), H=H, Hkv=Hkv, D=D, n=_log(rng, 1, 40000), page=page, bk=bk, bv=bv, gs=gs, ragged=rng.random() < 0.7, window=window)
    c["new"] = min(c["n"], rng.choice((_log(rng, 1, 16), _log(rng, 1, 4096))))
    while c["B"] * c["Hkv"] * c["n"] * _row_bytes(c) > 6e8:
        c["n"] = c["n"] // 2 + 1
        c["new"] = min(c["n"], c["new"])
    while work(c)["flops"] > 1.2e12 or c["B"] * c["new"] * H * D > 2e8 or c["new"] * c["n"] * H > 4e9:
        c["new"] = c["new"] // 2 + 1
    return c


# ------------------------------------------------------------------ sizes
def _side_bytes(c, bits):
    return 2 * c["D"] if bits == 16 else c["D"] * bits // 8 + 4 * (c["D"] // c["gs"])


def _row_bytes(c):
    """Bytes of one row, keys and values, of one KV head."""
    return _side_bytes(c, c["bk"]) + _side_bytes(c, c["bv"])


def _rng(c):
    return random.Random(sum((i + 1) * ord(ch) for i, ch in enumerate(repr(sorted((k, v) for k, v in c.items() if k != "name")))))


def _news(c):
    """New tokens of each sequence, from the case alone."""
    r = _rng(c)
    if c["kind"] == "packed":
        got = [r.randint(1, c["n"]) if c["ragged"] else c["n"] for _ in range(c["B"])]
    elif c["kind"] == "paged":
        got = [r.randint(1, c["new"]) if c["ragged"] else c["new"] for _ in range(c["B"])]
    else:
        return [1 if c["new"] == 1 else r.randint(int(b == 0), c["new"]) for b in range(c["B"])]
    if c["ragged"] and c["B"] >= 4 and c["new" if c["kind"] == "paged" else "n"] < 1000:
        got[r.randrange(1, c["B"])] = 0  # a batch slot without new tokens
    return got


def _lens(c):
    """Rows that each sequence holds, the new ones among them (tables: before the call)."""
    r, news = _rng(dict(c, salt=1)), _news(c)
    if c["kind"] == "packed":
        return news
    if c["kind"] == "paged":
        return [max(n, _log(r, max(1, min(17, c["n"])), c["n"]) if c["ragged"] else c["n"]) for n in news]
    held = [r.randint(0, c["held"]) for _ in news]
    return held if c["kind"] == "tables" else [h + n for h, n in zip(held, news)]


def _keeps(c):
    """Rows that each sequence of a tables case keeps: finished ones none, one in a hundred rolls back a few."""
    r = _rng(dict(c, salt=2))
    return [0 if r.random() < c["done"] else max(0, n - r.randint(1, 40)) if r.random() < 0.01 else n for n in _lens(c)]


def _width(c):
    """Entries of a sequence's row of the table."""
    rows = c["held"] + c["new"] if c["kind"] == "tables" else max(_lens(c))
    return max(1, _pages(c, rows))


def _pages(c, n):
    return (n + c["page"] - 1) // c["page"]


def _visible(c):
    """(query, key) pairs that the mask leaves, and rows that some query sees, of one head over all sequences."""
    pairs = rows = 0
    for n, m in zip(_lens(c), _news(c)):
        if m == 0:
            continue
        if not c.get("causal", True):
            pairs, rows = pairs + m * n, rows + n
            continue
        w = c["window"] if c["window"] > 0 else n
        full = max(0, min(m, n - w))  # queries whose window is full: those at positions from w on
        at = n - m  # the first query's position
        short = m - full
        pairs += full * w + short * (at + 1) + short * (short - 1) // 2
        rows += min(n, w + m - 1)
    return pairs, rows


def work(case):
    c = case
    if c["kind"] == "tables":
        lens, keeps, news = _lens(c), _keeps(c), _news(c)
        back = sum(_pages(c, n) - _pages(c, k) for n, k in zip(lens, keeps))
        taken = sum(_pages(c, k + m) - _pages(c, k) for k, m in zip(keeps, news))
        return {"bytes": 12 * back + 8 * taken + 24 * c["B"] + 16 * sum(news), "flops": 0}
    if c["kind"] == "rope":
        return {"bytes": c["tokens"] * (4 * c["H"] * c["D"] + 4), "flops": 3 * c["tokens"] * c["H"] * c["rd"]}
    if c["kind"] == "enter":
        t = sum(_news(c))
        return {"bytes": t * (4 * (c["H"] + 2 * c["Hkv"]) * c["D"] + 16), "flops": 3 * t * (c["H"] + c["Hkv"]) * c["rd"]}
    pairs, rows = _visible(c)
    row = 4 * c["D"] if c["kind"] == "packed" else _row_bytes(c)
    return {"bytes": rows * c["Hkv"] * row + 4 * sum(_news(c)) * c["H"] * c["D"], "flops": 4 * pairs * c["H"] * c["D"]}


# ------------------------------------------------------------------ plain building blocks
def _away(x):
    """Rounds to whole numbers, halves away from zero."""
    t = torch.trunc(x)
    return t + torch.where((x - t).abs() >= 0.5, torch.sign(x), torch.zeros_like(x))


def _quantize(x, bits, gs):
    """(packed words as int32, scales, biases) of bf16 rows [..., D]: the cache's affine format."""
    lead, D = x.shape[:-1], x.shape[-1]
    v = x.float().reshape(-1, D // gs, gs)
    lo, hi = v.amin(-1), v.amax(-1).clamp_min(0.0)
    scale = torch.clamp_min((hi - lo) / float(2 ** bits - 1), 1e-7)
    scale = torch.where(lo.abs() > hi.abs(), scale, -scale)
    edge = torch.where(lo.abs() > hi.abs(), lo, hi)
    q0 = _away(edge / scale)
    scale = torch.where(q0 == 0, scale, edge / torch.where(q0 == 0, torch.ones_like(q0), q0))
    bias = torch.where(q0 == 0, torch.zeros_like(edge), edge)
    code = _away((v - bias[..., None]) / scale[..., None]).clamp(0.0, float(2 ** bits - 1))
    code = code.to(torch.int32).reshape(-1, D * bits // 32, 32 // bits)  # 4 and 8 bits: no code straddles a word
    words = (code << torch.arange(0, 32, bits, device=x.device, dtype=torch.int32)).sum(-1, dtype=torch.int64)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return (words.reshape(*lead, D * bits // 32), scale.to(torch.bfloat16).reshape(*lead, D // gs), bias.to(torch.bfloat16).reshape(*lead, D // gs))


def _values(t, bits, gs):
    """The values that stored rows stand for: bf16 rows, or scale * code + bias."""
    if bits == 16:
        return t[0].float()
    words, scales, biases = t
    lead, D = words.shape[:-1], words.shape[-1] * 32 // bits
    shift = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    code = ((words[..., None] >> shift) & (2 ** bits - 1)).float().reshape(*lead, D // gs, gs)
    return (code * scales.float()[..., None] + biases.float()[..., None]).reshape(*lead, D)


class _Rand:
    """Seeded draws on the device."""

    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 100003 + _rng(case).randrange(100003))

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def rows(self, *shape):
        """bf16 rows: N(0, 1) with 2% of the channels four times larger."""
        big = self.uniform(shape[-1]) < 0.02
        out = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        flat = out.view(-1, shape[-1])
        step = max(1, _CHUNK // shape[-1])
        for a in range(0, flat.shape[0], step):
            b = min(flat.shape[0], a + step)
            flat[a:b] = self.normal(b - a, shape[-1]) * torch.where(big, 4.0, 1.0)
        return out

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _pool(c, r, pages):
    """Buffers of a pool, all rows filled: K's, then V's."""
    out = []
    for bits in (c.get("bk", 16), c.get("bv", 16)):
        lead = (pages, c["Hkv"], c["page"])
        if bits == 16:
            out.append([r.rows(*lead, c["D"])])
            continue
        side = [torch.empty(*lead, c["D"] * bits // 32, dtype=torch.int32, device="cuda")]
        side += [torch.empty(*lead, c["D"] // c["gs"], dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        step = max(1, _CHUNK // (c["Hkv"] * c["page"] * c["D"]))
        for a in range(0, pages, step):
            for dst, src in zip(side, _quantize(r.rows(min(step, pages - a), c["Hkv"], c["page"], c["D"]), bits, c["gs"])):
                dst[a:a + step] = src
        out.append(side)
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(c, r, held, width):
    """A table of `held` pages a sequence in any order, and the pages in that order."""
    order = r.perm(sum(held))
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    table[col < _ints(held)[:, None]] = order
    return table


def _stream():
    return torch.cuda.current_stream().cuda_stream


_SCALING = {"none": 0, "linear": 1, "base": 2, "bands": 3, "ramp": 4}
_BASE = 500000.0


def _original(c):
    """The context that the scaled frequencies were trained for; a frequency's turns in it decide about its scaling."""
    return 8192.0


def _ends(c):
    """Turns in the original context below which a frequency is divided by the factor, and above which it stays."""
    return (1.0, 32.0) if c["scaling"] == "ramp" else (1.0, 4.0)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = {k: v for k, v in case.items() if k != "name"}
    r = _Rand(c, seed)
    s = {"case": c}
    if c["kind"] == "tables":
        lens, news = _lens(c), _news(c)
        held, width = [_pages(c, n) for n in lens], _width(c)
        want = sum(_pages(c, k + m) - _pages(c, k) for k, m in zip(_keeps(c), news))
        spare = int(want * c["spare"])  # with what comes back, more than enough or not quite
        total = sum(held) + spare
        # One buffer: table, lens, free pages, their number. A pass starts from the state before the call.
        free = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        table = _table(c, r, held, width)
        free[:spare] = r.perm(spare) + sum(held)
        s["before"] = torch.cat([table.flatten(), _ints(lens), free, _ints([spare])])
        s["now"] = torch.empty_like(s["before"])
        s["keep"], s["add"], s["pages"], s["tokens"] = _ints(_keeps(c)), _ints(news), total, sum(news)
        s["starts"] = torch.empty(c["B"] + 1, dtype=torch.int32, device="cuda")
        s["granted"] = torch.empty(c["B"], dtype=torch.int32, device="cuda")
        s["slots"] = torch.empty(max(1, s["tokens"]), 4, dtype=torch.int32, device="cuda")
    elif c["kind"] == "rope":
        s["x"] = r.rows(c["tokens"], c["H"] + c["beside"], c["D"])  # values' heads beside the others
        s["positions"] = (r.uniform(c["tokens"]) * c["far"]).to(torch.int32).clamp_max(c["far"] - 1)
        s["out"] = torch.empty(c["tokens"], c["H"], c["D"], dtype=torch.bfloat16, device="cuda")
    elif c["kind"] == "enter":
        lens, news = _lens(c), _news(c)
        t = sum(news)
        s["qkv"] = r.rows(max(t, 1), c["H"] + 2 * c["Hkv"], c["D"])
        s["tokens"] = t
        held = [_pages(c, n) for n in lens]
        s["table"] = _table(c, r, held, _width(c))
        s["lens"] = _ints(lens)
        s["pool"] = _pool(c, r, max(1, sum(held)))
        b = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), _ints(news).long())
        first = _ints(lens).long() - _ints(news).long()
        row = torch.arange(t, device="cuda") - (torch.cumsum(_ints(news).long(), 0) - _ints(news).long())[b] + first[b]
        s["slots"] = torch.stack([s["table"].long()[b, row // c["page"]], row % c["page"], row, b], 1).to(torch.int32).contiguous()
        s["q_out"] = torch.empty(max(t, 1), c["H"], c["D"], dtype=torch.bfloat16, device="cuda")
    elif c["kind"] == "packed":
        news = _news(c)
        t = sum(news)
        s["qkv"] = r.rows(max(t, 1), c["H"] + 2 * c["Hkv"], c["D"])
        s["tokens"], s["counts"] = t, news
        s["starts"] = _ints([sum(news[:b]) for b in range(c["B"] + 1)])
        s["out"] = torch.empty(max(t, 1), c["H"], c["D"], dtype=torch.bfloat16, device="cuda")
    else:
        lens, news = _lens(c), _news(c)
        t = sum(news)
        held = [_pages(c, n) for n in lens]
        s["tokens"], s["counts"], s["held"] = t, news, lens
        s["table"], s["lens"] = _table(c, r, held, _width(c)), _ints(lens)
        s["pool"] = _pool(c, r, max(1, sum(held)))
        s["q"] = r.normal(max(t, 1), c["H"], c["D"]).to(torch.bfloat16)
        s["starts"] = _ints([sum(news[:b]) for b in range(c["B"] + 1)])
        s["out"] = torch.empty_like(s["q"])
    if own:
        T = _T()
        if c["kind"] == "tables":
            n, now, rows = c["B"] * _width(c), s["now"].data_ptr(), c["B"]
            s["pt"] = T.page_tables(c["B"], c["page"], s["pages"], now, _width(c), now + 4 * n, now + 4 * (n + rows), now + 4 * (n + rows + s["pages"]))
        if c["kind"] in ("rope", "enter"):
            low, high = _ends(c)
            turns, magnitude = T.rope_turns(c["rd"], _BASE, _SCALING[c["scaling"]], c["factor"], _original(c), low, high)
            s["turns"] = torch.tensor([t - (t >> 63 << 64) for t in turns], dtype=torch.int64, device="cuda")
            s["rope"] = T.rope(c["rd"], c["pairs"] == "neighbours", magnitude, s["turns"].data_ptr())
        if c["kind"] in ("enter", "paged"):
            ptrs = [t.data_ptr() for side in s["pool"] for t in side]
            s["kv"] = T.paged_kv(T.CACHE_BF16 if c.get("bk", 16) == 16 else T.CACHE_AFFINE, c["B"], c["Hkv"], c["D"], c["page"], s["pool"][0][0].shape[0], ptrs,
                                 s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), None, c.get("gs", 64), c.get("bk", 16), c.get("bv", 16))
        if c["kind"] == "packed":
            s["ws"] = torch.empty(max(16, T.packed_attend_workspace_size(c["B"], c["H"], c["Hkv"], c["D"], s["tokens"])), dtype=torch.uint8, device="cuda")
        if c["kind"] == "paged":
            size = T.paged_prefill_workspace_size(s["kv"], c["H"], s["tokens"], s["table"].shape[1] * c["page"])
            s["ws"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    return {"tables": _run_tables, "rope": _run_rope, "enter": _run_enter, "packed": _run_packed, "paged": _run_paged}[c["kind"]](s, c)


def _run_tables(s, c):
    B, width, R, P, tokens = c["B"], _width(c), c["page"], s["pages"], s["tokens"]
    s["now"].copy_(s["before"])
    table, lens, free, count = torch.split(s["now"], [B * width, B, P, 1])
    table = table.view(B, width)
    out = {"table": table, "lens": lens, "free": free, "count": count, "starts": s["starts"], "granted": s["granted"], "slots": s["slots"]}
    if own:
        T, st = _T(), _stream()
        T.paged_release(s["pt"], s["keep"].data_ptr(), None, st)
        T.paged_reserve(s["pt"], s["add"].data_ptr(), tokens, s["starts"].data_ptr(), s["granted"].data_ptr(), s["slots"].data_ptr(), st)
        return out
    # Back: the pages behind the last row kept, in order, on top of the free ones.
    col = torch.arange(width, device="cuda")[None]
    n, keep = lens.long(), torch.minimum(s["keep"], lens).long()
    gone = (col >= ((keep + R - 1) // R)[:, None]) & (col < ((n + R - 1) // R)[:, None])
    at = torch.where(gone, count.long() + torch.cumsum(gone.flatten().long(), 0).view(B, width) - 1, torch.full_like(table, P).long())
    stack = torch.cat([free, free[:1]])  # the last place takes what is not written
    stack[at.flatten()] = table.flatten()
    free.copy_(stack[:P])
    count += gone.sum().to(torch.int32)
    table.masked_fill_(gone, -1)
    lens.copy_(keep)
    # Out: a sequence gets its tokens where the pages and places left by those before it are enough.
    n, a, avail = keep, s["add"].long(), count.long()
    held = (n + R - 1) // R
    need = (n + a + R - 1) // R - held
    fits = n + a <= width * R
    pages = torch.cumsum(torch.where(fits, need, torch.zeros_like(need)), 0)
    places = torch.cumsum(torch.where(fits, a, torch.zeros_like(a)), 0)
    ok = fits & ((need == 0) | (pages <= avail)) & ((a == 0) | (places <= tokens))
    got, take = torch.where(ok, a, torch.zeros_like(a)), torch.where(ok, need, torch.zeros_like(need))
    ends, base, total = torch.cumsum(got, 0), torch.cumsum(take, 0) - take, take.sum()
    new = (col >= held[:, None]) & (col < (held + take)[:, None])
    src = avail - total + base[:, None] + col - held[:, None]
    table.copy_(torch.where(new, free[src.clamp(0, P - 1)], table))
    count -= total.to(torch.int32)
    lens.copy_(n + got)
    s["starts"][:1] = 0
    s["starts"][1:] = ends
    s["granted"].copy_(torch.where(ok, a, torch.full_like(a, -1)))
    i = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(ends, i, right=True).clamp_max(B - 1)
    row = n[b] + i - (ends - got)[b]
    slot = torch.stack([table.long()[b, (row // R).clamp(0, width - 1)], row % R, row, b], 1)
    none = torch.tensor([-1, 0, -1, -1], device="cuda")
    s["slots"][:tokens] = torch.where((i < ends[-1])[:, None], slot, none).to(torch.int32)
    return out


def _theta(c, device="cuda"):
    """(radians a position of each pair, magnitude of the rotated channels), in 64 bits."""
    rd, f = c["rd"], c["factor"]
    i = torch.arange(rd // 2, dtype=torch.float64, device=device)
    base = _BASE * f ** (rd / (rd - 2)) if c["scaling"] == "base" and rd > 2 else _BASE
    theta = torch.exp(-2.0 * i / rd * math.log(base))
    low, high = _ends(c)
    if c["scaling"] == "linear":
        return theta / f, 1.0
    if c["scaling"] == "bands":
        keep = ((theta * _original(c) / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return theta * (keep + (1.0 - keep) / f), 1.0
    if c["scaling"] == "ramp":
        channel = lambda turns: rd * math.log(_original(c) / (2 * math.pi * turns)) / (2 * math.log(_BASE))  # noqa: E731
        first, last = max(math.floor(channel(high)), 0), min(math.ceil(channel(low)), rd - 1)
        go = ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return theta * (1.0 - go + go / f), 0.1 * math.log(f) + 1.0
    return theta, 1.0


def _rotated(x, positions, c):
    """Rows [tokens, heads, D] rotated, in 32 bits (the angles in 64), rounded once."""
    theta, m = _theta(c)
    angle = positions.double()[:, None] * theta[None]
    cos, sin = (torch.cos(angle) * m).float()[:, None], (torch.sin(angle) * m).float()[:, None]
    v, rd = x[..., :c["rd"]].float(), c["rd"]
    if c["pairs"] == "neighbours":
        u = v.reshape(*v.shape[:-1], rd // 2, 2)
        a, b = u[..., 0], u[..., 1]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(v.shape)
    else:
        a, b = v[..., :rd // 2], v[..., rd // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y.to(x.dtype), x[..., rd:]], -1)


def _run_rope(s, c):
    if own:
        H, D = c["H"], c["D"]
        _T().rope_apply(s["rope"], s["positions"].data_ptr(), 1, c["tokens"], s["x"].data_ptr(), H, D, s["x"].stride(0), D, s["out"].data_ptr(), H * D, D, _stream())
        return s["out"]
    s["out"].copy_(_rotated(s["x"][:, :c["H"]], s["positions"], c))
    return s["out"]


def _run_enter(s, c):
    H, Hkv, D, t = c["H"], c["Hkv"], c["D"], s["tokens"]
    q, k, v = s["qkv"][:, :H], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]
    if own:
        step = s["qkv"].stride(0)
        _T().paged_append_rope(s["kv"], s["rope"], q.data_ptr(), H, step, s["q_out"].data_ptr(), H * D, k.data_ptr(), v.data_ptr(), step, D, s["slots"].data_ptr(), t,
                               None, 1, _stream())
    elif t:
        page, row, position = s["slots"][:, 0].long(), s["slots"][:, 1].long(), s["slots"][:, 2]
        s["q_out"][:t] = _rotated(q[:t], position, c)
        s["pool"][0][0][page, :, row] = _rotated(k[:t], position, c)
        s["pool"][1][0][page, :, row] = v[:t]
    return {"q": s["q_out"][:t], "k": s["pool"][0][0], "v": s["pool"][1][0]}


def _attend(q, k, v, c):
    """Attention of the newest rows q [m, H, D] over k and v [Hkv, n, D] in 32 bits, rounded once."""
    m, n, Hkv = q.shape[0], k.shape[1], c["Hkv"]
    y = q.float().reshape(m, Hkv, -1, c["D"]).permute(1, 2, 0, 3).reshape(Hkv, -1, c["D"])
    x = torch.matmul(y, k.transpose(1, 2).contiguous()).view(Hkv, -1, m, n) * c["D"] ** -0.5
    if c.get("causal", True):
        at, key = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        hidden = key > at
        if c["window"] > 0:
            hidden |= key <= at - c["window"]
        x.masked_fill_(hidden, -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    return torch.matmul(x.view(Hkv, -1, n), v.contiguous()).view(Hkv, -1, m, c["D"]).permute(2, 0, 1, 3).reshape(m, c["H"], c["D"]).to(torch.bfloat16)


def _run_packed(s, c):
    H, Hkv, D, t = c["H"], c["Hkv"], c["D"], s["tokens"]
    q, k, v = s["qkv"][:, :H], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]
    if own:
        step = s["qkv"].stride(0)
        _T().packed_attend(q.data_ptr(), step, k.data_ptr(), v.data_ptr(), step, D, c["B"], H, Hkv, D, s["starts"].data_ptr(), t, D ** -0.5, s["out"].data_ptr(),
                           c["causal"], c["window"], s["ws"].data_ptr(), s["ws"].numel(), _stream())
        return s["out"][:t]
    a = 0
    for m in s["counts"]:
        if m:
            s["out"][a:a + m] = _attend(q[a:a + m], k[a:a + m].float().transpose(0, 1), v[a:a + m].float().transpose(0, 1), c)
        a += m
    return s["out"][:t]


def _run_paged(s, c):
    H, D, t = c["H"], c["D"], s["tokens"]
    if own:
        _T().paged_prefill_attend(s["kv"], s["q"].data_ptr(), H * D, H, s["starts"].data_ptr(), t, D ** -0.5, s["table"].shape[1] * c["page"], s["out"].data_ptr(),
                                  c["window"], s["ws"].data_ptr(), s["ws"].numel(), _stream())
        return s["out"][:t]
    a = 0
    for b, (n, m) in enumerate(zip(s["held"], s["counts"])):
        if m == 0:
            continue
        lo = max(0, n - m - c["window"] + 1) // c["page"] if c["window"] > 0 else 0  # pages that no query sees are left out
        pages = s["table"][b, lo:_pages(c, n)].long()
        k, v = (_values([x[pages] for x in side], bits, c["gs"]).permute(1, 0, 2, 3).reshape(c["Hkv"], -1, D)[:, :n - lo * c["page"]]
                for side, bits in zip(s["pool"], (c["bk"], c["bv"])))
        s["out"][a:a + m] = _attend(s["q"][a:a + m], k, v, c)
        a += m
    return s["out"][:t]


# ------------------------------------------------------------------ 64 bits
def _exact_turn(x, positions, c):
    """Rows rotated in 64 bits: the pairs as complex numbers, times e^(i angle)."""
    theta, m = _theta(c)
    w = torch.polar(torch.full((len(positions), c["rd"] // 2), m, dtype=torch.float64, device="cuda"), positions.double()[:, None] * theta)[:, None]
    d = x.double()
    half = c["rd"] // 2
    if c["pairs"] == "neighbours":
        z = torch.complex(d[..., 0:c["rd"]:2], d[..., 1:c["rd"]:2]) * w
        d[..., 0:c["rd"]:2], d[..., 1:c["rd"]:2] = z.real, z.imag
    else:
        z = torch.complex(d[..., :half], d[..., half:c["rd"]]) * w
        d[..., :half], d[..., half:c["rd"]] = z.real, z.imag
    return d


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = s["case"]
    if c["kind"] == "tables":
        return _exact_tables(s, c)
    if c["kind"] == "rope":
        return _exact_turn(s["x"][:, :c["H"]], s["positions"], c)
    H, Hkv, D, t = c["H"], c["Hkv"], c["D"], s["tokens"]
    if c["kind"] == "enter":
        k, v = (side[0].double() for side in s["pool"])
        page, row, position = (s["slots"][:, i].long() for i in range(3))
        if t:
            k[page, :, row] = _exact_turn(s["qkv"][:t, H:H + Hkv], position, c)
            v[page, :, row] = s["qkv"][:t, H + Hkv:].double()
        return {"q": _exact_turn(s["qkv"][:t, :H], position, c), "k": k, "v": v}
    out = torch.zeros(t, H, D, dtype=torch.float64, device="cuda")
    a = 0
    for b, m in enumerate(s["counts"]):
        n = m if c["kind"] == "packed" else s["held"][b]
        for h in range(Hkv if m else 0):
            if c["kind"] == "packed":
                k, v = s["qkv"][a:a + m, H + h].double(), s["qkv"][a:a + m, H + Hkv + h].double()
            else:
                rows = torch.arange(n, device="cuda")
                where = s["table"][b].long()[rows // c["page"]]
                k, v = (_exact_rows([x[where, h, rows % c["page"]] for x in side], bits, c["gs"]) for side, bits in zip(s["pool"], (c["bk"], c["bv"])))
            for g in range(H // Hkv):
                e = h * (H // Hkv) + g
                y = (s["qkv"] if c["kind"] == "packed" else s["q"])[a:a + m, e].double()
                for i in range(0, m, 2048):
                    x = y[i:i + 2048] @ k.t().contiguous() / math.sqrt(D)
                    if c.get("causal", True):
                        back = (torch.arange(i, i + len(x), device="cuda") + n - m)[:, None] - torch.arange(n, device="cuda")[None]  # how far behind its query a key lies
                        x[(back < 0) | (back >= (c["window"] if c["window"] > 0 else n))] = -math.inf
                    out[a + i:a + i + len(x), e] = torch.softmax(x, -1) @ v
        a += m
    return out


def _exact_rows(t, bits, gs):
    if bits == 16:
        return t[0].double()
    code = torch.stack([(t[0] >> o) & (2 ** bits - 1) for o in range(0, 32, bits)], -1).double().flatten(-2)
    return code * t[1].double().repeat_interleave(gs, -1) + t[2].double().repeat_interleave(gs, -1)


def _exact_tables(s, c):
    """The same by a walk over the sequences, in Python's integers."""
    B, width, R, P, tokens = c["B"], _width(c), c["page"], s["pages"], s["tokens"]
    flat = s["before"].cpu().tolist()
    table = [flat[b * width:(b + 1) * width] for b in range(B)]
    lens, free, count = flat[B * width:B * width + B], flat[B * width + B:-1], flat[-1]
    for b, keep in enumerate(s["keep"].tolist()):
        keep = min(keep, lens[b])
        for j in range(-(-keep // R), -(-lens[b] // R)):
            free[count], table[b][j] = table[b][j], -1
            count += 1
        lens[b] = keep
    pages = places = 0
    granted, takes = [], []
    for b, a in enumerate(s["add"].tolist()):
        need = -(-(lens[b] + a) // R) - -(-lens[b] // R)
        fits = lens[b] + a <= width * R
        pages, places = pages + need * fits, places + a * fits
        ok = fits and (need == 0 or pages <= count) and (a == 0 or places <= tokens)
        granted.append(a if ok else -1)
        takes.append(need if ok else 0)
    at = count - sum(takes)
    left = at
    slots, starts = [], [0]
    for b, a in enumerate(granted):
        first = -(-lens[b] // R)
        table[b][first:first + takes[b]] = free[at:at + takes[b]]
        at += takes[b]
        for row in range(lens[b], lens[b] + max(a, 0)):
            slots.append([table[b][row // R], row % R, row, b])
        lens[b] += max(a, 0)
        starts.append(len(slots))
    slots += [[-1, 0, -1, -1]] * (max(1, tokens) - len(slots))
    return {"table": torch.tensor(table), "lens": torch.tensor(lens), "free": torch.tensor(free), "count": torch.tensor([left]), "starts": torch.tensor(starts),
            "granted": torch.tensor(granted), "slots": torch.tensor(slots)}
