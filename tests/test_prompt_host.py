"""Page tables, rotary positions and prompt attention without a GPU: every
refusal comes before any launch, sizes are host arithmetic, the binding's
structs are the header's."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import prompt_ref as R
import tqkv as T
from test_paged_host import A, BAD_VIEWS, refused, view

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def tables(**other):
    c = dict(batch=4, page_rows=64, num_pages=10, table=A, table_stride=8, lens=A, free_pages=A, free_count=A)
    c.update(other)
    return T.page_tables(**c)


@pytest.mark.parametrize("other,status", [
    (dict(batch=0), T.EINVAL_SHAPE), (dict(batch=1025), T.EUNSUPPORTED), (dict(page_rows=24), T.EUNSUPPORTED),
    (dict(num_pages=0), T.EINVAL_SHAPE), (dict(num_pages=1 << 31), T.EINVAL_SHAPE), (dict(table_stride=0), T.EINVAL_SHAPE),
    (dict(table_stride=(1 << 24) + 1), T.EINVAL_SHAPE), (dict(table=None), T.EINVAL_ARG), (dict(lens=None), T.EINVAL_ARG),
    (dict(free_pages=None), T.EINVAL_ARG), (dict(free_count=None), T.EINVAL_ARG), (dict(table=A + 1), T.EINVAL_ARG),
    (dict(lens=A + 2), T.EINVAL_ARG), (dict(free_pages=A + 2), T.EINVAL_ARG), (dict(free_count=A + 3), T.EINVAL_ARG)])
def test_tables_that_no_call_takes(other, status):
    refused(status, T.paged_reserve, tables(**other), A, 4, A, A, A)
    refused(status, T.paged_release, tables(**other), A)


def test_table_refusals():
    ok = dict(tables=tables(), counts=A, tokens=4, starts=A, granted=A, slots=A)
    for other, status in [(dict(counts=None), T.EINVAL_ARG), (dict(starts=None), T.EINVAL_ARG), (dict(tokens=-1), T.EINVAL_SHAPE),
                          (dict(tokens=1 << 31), T.EINVAL_SHAPE), (dict(slots=A + 8), T.EINVAL_ARG), (dict(counts=A + 2), T.EINVAL_ARG),
                          (dict(starts=A + 1), T.EINVAL_ARG), (dict(granted=A + 2), T.EINVAL_ARG)]:
        refused(status, T.paged_reserve, **{**ok, **other})
    refused(T.EINVAL_ARG, T.paged_release, tables(), None)
    refused(T.EINVAL_ARG, T.paged_release, tables(), A + 2)
    refused(T.EINVAL_ARG, T.paged_release, tables(), A, A + 2)
    assert T.lib().tqkv_paged_reserve(None, A, 1, A, None, None, None) == T.EINVAL_ARG
    assert T.lib().tqkv_paged_release(None, A, None, None) == T.EINVAL_ARG


def test_turns_refusals_and_values():
    for args, status in [((3,), T.EINVAL_SHAPE), ((0,), T.EINVAL_SHAPE), ((-2,), T.EINVAL_SHAPE), ((1026,), T.EINVAL_SHAPE),
                         ((64, 1.0), T.EINVAL_ARG), ((64, float("nan")), T.EINVAL_ARG), ((64, float("inf")), T.EINVAL_ARG),
                         ((64, 1e4, 5), T.EUNSUPPORTED), ((64, 1e4, -1), T.EUNSUPPORTED), ((64, 1e4, 1, 0.0), T.EINVAL_ARG),
                         ((64, 1e4, 1, float("inf")), T.EINVAL_ARG), ((64, 1e4, 2, 1e-9), T.EINVAL_ARG),
                         ((64, 1e4, 3, 2.0, 0.0), T.EINVAL_ARG), ((64, 1e4, 3, 2.0, 10.0, 0.0), T.EINVAL_ARG),
                         ((64, 1e4, 4, 2.0, 10.0, 4.0, 4.0), T.EINVAL_ARG), ((64, 1e4, 4, 2.0, 10.0, 4.0, float("inf")), T.EINVAL_ARG)]:
        refused(status, T.rope_turns, *args)
    assert T.lib().tqkv_rope_turns(None, None, None) == T.EINVAL_ARG
    for rd in (2, 6, 64, 1024):
        for kw in (dict(), dict(scaling=1, factor=7.0), dict(scaling=2, factor=5.0), dict(scaling=3, factor=8.0, original=8192.0),
                   dict(scaling=4, factor=8.0, original=2048.0, high=32.0), dict(scaling=4, factor=0.5, original=1.0, high=32.0)):
            turns, m = T.rope_turns(rd, 500000.0, **kw)
            theta, mag = R.thetas(rd, 500000.0, **kw)
            got = np.array([t / 2.0 ** 64 * 2 * np.pi for t in turns])
            # The power's own error in 64 bits, and half a unit of the turns: 2^-65 of a turn.
            assert np.all(np.abs(got - theta) <= 2.0 ** -46 * theta + 2 * np.pi * 2.0 ** -65), (rd, kw)
            assert abs(m - mag) <= 2.0 ** -23 * abs(mag)
    # More than a turn a position: the whole turns fall away.
    assert abs(T.rope_turns(2, 10.0, 1, 0.1)[0][0] / 2.0 ** 64 - (10.0 / (2 * np.pi)) % 1.0) < 1e-15


def rope(**other):
    c = dict(rotary_dim=64, interleaved=0, magnitude=1.0, turns=A)
    c.update(other)
    return T.rope(**c)


BAD_ROPES = [(dict(rotary_dim=0), T.EINVAL_SHAPE), (dict(rotary_dim=63), T.EINVAL_SHAPE), (dict(rotary_dim=130), T.EINVAL_SHAPE),
             (dict(interleaved=2), T.EINVAL_ARG), (dict(turns=None), T.EINVAL_ARG), (dict(turns=A + 4), T.EINVAL_ARG)]


def test_rope_refusals():
    ok = dict(rope=rope(), positions=A, position_stride=1, tokens=4, x=A, heads=8, dim=128, x_token_stride=1024, x_head_stride=128,
              out=2 * A, out_token_stride=1024, out_head_stride=128)
    for other, status in [*[(dict(rope=rope(**r)), s) for r, s in BAD_ROPES], (dict(dim=100), T.EUNSUPPORTED), (dict(dim=1032), T.EUNSUPPORTED),
                          (dict(dim=0), T.EUNSUPPORTED), (dict(heads=0), T.EINVAL_SHAPE), (dict(heads=1025), T.EUNSUPPORTED),
                          (dict(tokens=-1), T.EINVAL_SHAPE), (dict(tokens=1 << 40), T.EINVAL_SHAPE), (dict(positions=None), T.EINVAL_ARG),
                          (dict(x=None), T.EINVAL_ARG), (dict(out=None), T.EINVAL_ARG), (dict(x=A + 8), T.EINVAL_ARG),
                          (dict(out=A + 8), T.EINVAL_ARG), (dict(positions=A + 2), T.EINVAL_ARG), (dict(x_token_stride=1020), T.EINVAL_ARG),
                          (dict(x_head_stride=4), T.EINVAL_ARG), (dict(out_token_stride=4), T.EINVAL_ARG), (dict(out_head_stride=12), T.EINVAL_ARG),
                          (dict(out=A, out_token_stride=2048), T.EINVAL_ARG)]:
        refused(status, T.rope_apply, **{**ok, **other})
    T.rope_apply(**{**ok, "tokens": 0, "x": None})
    bad = rope()
    bad.reserved = 1
    refused(T.EINVAL_ARG, T.rope_apply, **{**ok, "rope": bad})
    assert T.lib().tqkv_rope_apply(None, A, 1, 1, A, 1, 128, 128, 128, A, 128, 128, None) == T.EINVAL_ARG


def test_append_rope_refusals():
    ok = dict(kv=view(), rope=rope(), q=A, H=8, q_stride=1024, q_out=2 * A, q_out_stride=1024, k=A, v=A, token_stride=1024, head_stride=128,
              slots=A, tokens=4)
    for other, status in [*[(dict(kv=view(**v)), s) for v, s in BAD_VIEWS], *[(dict(rope=rope(**r)), s) for r, s in BAD_ROPES],
                          (dict(H=-1), T.EINVAL_SHAPE), (dict(H=1025), T.EUNSUPPORTED), (dict(q=None), T.EINVAL_ARG),
                          (dict(q_out=None), T.EINVAL_ARG), (dict(k=None), T.EINVAL_ARG), (dict(v=None), T.EINVAL_ARG),
                          (dict(slots=None), T.EINVAL_ARG), (dict(slots=A + 4), T.EINVAL_ARG), (dict(positions=A + 2), T.EINVAL_ARG),
                          (dict(q=A + 8), T.EINVAL_ARG), (dict(q_out=A + 2), T.EINVAL_ARG), (dict(q_stride=4), T.EINVAL_ARG),
                          (dict(q_out_stride=4), T.EINVAL_ARG), (dict(q_out=A, q_out_stride=2048), T.EINVAL_ARG), (dict(k=A + 8), T.EINVAL_ARG),
                          (dict(v=A + 8), T.EINVAL_ARG), (dict(token_stride=12), T.EINVAL_ARG), (dict(head_stride=4), T.EINVAL_ARG),
                          (dict(tokens=-1), T.EINVAL_SHAPE), (dict(tokens=1 << 40), T.EINVAL_SHAPE)]:
        refused(status, T.paged_append_rope, **{**ok, **other})
    T.paged_append_rope(**{**ok, "tokens": 0, "k": None})


def test_packed_refusals():
    ok = dict(q=A, q_stride=1024, k=A, v=A, token_stride=1024, head_stride=128, batch=2, H=8, H_kv=4, D=128, starts=A, tokens=64, scale=0.1,
              out=2 * A, workspace=A, workspace_bytes=1 << 40)
    for other, status in [(dict(q=None), T.EINVAL_ARG), (dict(k=None), T.EINVAL_ARG), (dict(v=None), T.EINVAL_ARG), (dict(out=None), T.EINVAL_ARG),
                          (dict(starts=None), T.EINVAL_ARG), (dict(q=A + 8), T.EINVAL_ARG), (dict(k=A + 2), T.EINVAL_ARG),
                          (dict(v=A + 8), T.EINVAL_ARG), (dict(out=A + 8), T.EINVAL_ARG), (dict(starts=A + 2), T.EINVAL_ARG),
                          (dict(q_stride=4), T.EINVAL_ARG), (dict(token_stride=4), T.EINVAL_ARG), (dict(head_stride=4), T.EINVAL_ARG),
                          (dict(batch=0), T.EINVAL_SHAPE), (dict(batch=1025), T.EUNSUPPORTED), (dict(D=96), T.EUNSUPPORTED),
                          (dict(D=0), T.EUNSUPPORTED), (dict(H=0), T.EINVAL_SHAPE), (dict(H=6), T.EINVAL_SHAPE), (dict(H_kv=0), T.EINVAL_SHAPE),
                          (dict(H=132), T.EUNSUPPORTED), (dict(tokens=-1), T.EINVAL_SHAPE), (dict(tokens=1 << 31), T.EINVAL_SHAPE),
                          (dict(token_stride=-1024), T.EUNSUPPORTED), (dict(token_stride=1 << 27), T.EUNSUPPORTED),
                          (dict(window=4, causal=False), T.EINVAL_ARG)]:
        refused(status, T.packed_attend, **{**ok, **other})
    T.packed_attend(**{**ok, "tokens": 0, "q": None})
    for args in [(0, 8, 4, 128, 64), (2, 7, 4, 128, 64), (2, 8, 4, 96, 64), (2, 8, 4, 128, -1), (2, 132, 4, 128, 64)]:
        assert T.packed_attend_workspace_size(*args) == 0


def test_paged_prefill_refusals():
    ok = dict(kv=view(), q=A, q_stride=1024, H=8, starts=A, tokens=64, scale=0.1, max_rows=512, out=2 * A, workspace=A, workspace_bytes=1 << 40)
    for other, status in [*[(dict(kv=view(**v)), s) for v, s in BAD_VIEWS], (dict(q=None), T.EINVAL_ARG), (dict(out=None), T.EINVAL_ARG),
                          (dict(starts=None), T.EINVAL_ARG), (dict(q=A + 8), T.EINVAL_ARG), (dict(out=A + 8), T.EINVAL_ARG),
                          (dict(starts=A + 2), T.EINVAL_ARG), (dict(q_stride=4), T.EINVAL_ARG), (dict(H=0), T.EINVAL_SHAPE),
                          (dict(H=6), T.EINVAL_SHAPE), (dict(H=132), T.EUNSUPPORTED), (dict(tokens=-1), T.EINVAL_SHAPE),
                          (dict(tokens=1 << 31), T.EINVAL_SHAPE), (dict(max_rows=0), T.EINVAL_SHAPE), (dict(max_rows=513), T.EINVAL_SHAPE)]:
        refused(status, T.paged_prefill_attend, **{**ok, **other})
    T.paged_prefill_attend(**{**ok, "tokens": 0, "q": None})
    assert T.paged_prefill_workspace_size(view(batch=0), 8, 64, 512) == 0
    assert T.paged_prefill_workspace_size(view(), 8, 64, 513) == 0
    assert T.paged_prefill_workspace_size(view(), 7, 64, 512) == 0


def test_workspaces_that_are_too_small():
    """A byte too few or off by 8: refused before any launch."""
    affine = view(kind=T.CACHE_AFFINE, batch=2)
    need = T.paged_prefill_workspace_size(affine, 8, 300, 512)
    assert need >= 4 * 2 * affine.kv_heads * 512 * affine.dim  # the dequantized rows
    ok = dict(kv=affine, q=A, q_stride=1024, H=8, starts=A, tokens=300, scale=0.1, max_rows=512, out=2 * A, workspace=A, workspace_bytes=need)
    for other in (dict(workspace_bytes=need - 1), dict(workspace_bytes=0), dict(workspace=A + 8)):
        refused(T.EINVAL_ARG, T.paged_prefill_attend, **{**ok, **other})
    # Splits alone: long rows of one sequence.
    long = view(kind=T.CACHE_BF16, batch=1, num_pages=4096, table_stride=4096)
    rows = 4096 * long.page_rows
    need = T.paged_prefill_workspace_size(long, 8, 2, rows)
    assert need > 0
    refused(T.EINVAL_ARG, T.paged_prefill_attend, **{**ok, "kv": long, "tokens": 2, "max_rows": rows, "workspace_bytes": need - 1})
    # (A split holds at least 16 keys a row of its block: 4,096 of 256 rows.)
    assert T.packed_attend_workspace_size(1, 8, 4, 128, 4096) == 0
    need = T.packed_attend_workspace_size(1, 1, 1, 128, 8192)
    assert need > 0
    refused(T.EINVAL_ARG, T.packed_attend, A, 128, A, A, 128, 128, 1, 1, 1, 128, A, 8192, 0.1, 2 * A, workspace=A, workspace_bytes=need - 1)


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"tqkv_page_tables": T.PageTables, "tqkv_rope_config": T.RopeConfig, "tqkv_rope": T.Rope}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "tqkv.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "abi.c", tmp_path / "abi"
    src.write_text("\n".join([*lines, "  return 0;\n}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = {tuple(s.split()[:-1]): int(s.split()[-1]) for s in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n") if s}
    for cname, py in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(py), cname
        for f, _ in py._fields_:
            assert got[(cname, f)] == getattr(py, f).offset, (cname, f)


def test_workspace_bounds():
    """What the header promises for all calls: partial results of a prompt's call
    are kept for fewer than 384 workgroups of 256 rows, of few rows' for 2,048 of
    32 and as many more as there are blocks."""
    rng = np.random.default_rng(1)
    tokens = np.unique(np.r_[1:300, np.geomspace(1, 2 ** 31 - 1, 400).astype(np.int64)])
    fell = False
    for D in (64, 128, 256, 512):
        for batch, H_kv, G in [(1, 1, 1), (1, 1, 32), (2, 8, 4), (7, 3, 5), (64, 8, 4), (1024, 16, 1), (1024, 1, 32)]:
            sizes = [T.packed_attend_workspace_size(batch, H_kv * G, H_kv, D, int(t)) for t in tokens]
            assert max(sizes) <= 4 * (D + 2) * 98304 + 256, (D, batch, H_kv, G)
            fell |= any(a > b for a, b in zip(sizes, sizes[1:]))
            for kind in (T.CACHE_BF16, T.CACHE_AFFINE):
                kv = view(kind=kind, batch=batch, kv_heads=H_kv, dim=D, num_pages=1 << 20, table_stride=1 << 14, bits_k=4, bits_v=8, group_size=32)
                cap = (1 << 14) * kv.page_rows
                for rows in (1, 900, int(rng.integers(1, cap)), cap):
                    sizes = [T.paged_prefill_workspace_size(kv, H_kv * G, int(t), rows) for t in tokens[::3]]
                    most = 4 * (D + 2) * (98304 + 32 * batch * H_kv) + 1024
                    if kind == T.CACHE_AFFINE:
                        most += 4 * batch * H_kv * rows * D + 520 * batch * H_kv
                    assert max(sizes) <= most, (D, batch, H_kv, G, kind, rows)
                    fell |= any(a > b for a, b in zip(sizes, sizes[1:]))
    assert fell  # why there is a bound to state


def test_out_is_not_q():
    refused(T.EINVAL_ARG, T.packed_attend, A, 1024, A, A, 1024, 128, 2, 8, 4, 128, A, 64, 0.1, A, workspace=A, workspace_bytes=1 << 40)
    refused(T.EINVAL_ARG, T.paged_prefill_attend, view(), A, 1024, 8, A, 64, 0.1, 512, A, workspace=A, workspace_bytes=1 << 40)
