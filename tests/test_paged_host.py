"""The paged cache's entry points without a GPU: every refusal comes before any
launch (nothing here reaches the HIP runtime), sizes are host arithmetic, and
the binding's struct is the header's."""
import ctypes
import os
import subprocess

import pytest

import tqkv as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # an aligned address that is never read


def view(**other):
    c = dict(kind=T.CACHE_AFFINE, batch=2, kv_heads=4, dim=128, page_rows=64, num_pages=10,
             slots=[A] * 6, table=A, table_stride=8, lens=A, weights=A, group_size=64, bits_k=4,
             bits_v=8)
    c.update(other)
    return T.paged_kv(**c)


BAD_VIEWS = [
    (dict(kind=T.CACHE_CODEBOOK), T.EUNSUPPORTED), (dict(kind=-1), T.EUNSUPPORTED),
    (dict(batch=0), T.EINVAL_SHAPE), (dict(batch=1025), T.EUNSUPPORTED),
    (dict(kv_heads=0), T.EINVAL_SHAPE), (dict(kv_heads=1025), T.EUNSUPPORTED),
    (dict(dim=96), T.EUNSUPPORTED), (dict(dim=1024), T.EUNSUPPORTED), (dict(dim=0), T.EUNSUPPORTED),
    (dict(page_rows=8), T.EUNSUPPORTED), (dict(page_rows=48), T.EUNSUPPORTED),
    (dict(page_rows=512), T.EUNSUPPORTED), (dict(num_pages=0), T.EINVAL_SHAPE),
    (dict(num_pages=1 << 31), T.EINVAL_SHAPE), (dict(table_stride=0), T.EINVAL_SHAPE),
    (dict(table_stride=(1 << 24) + 1), T.EINVAL_SHAPE), (dict(group_size=16), T.EUNSUPPORTED),
    (dict(dim=64, group_size=128), T.EUNSUPPORTED), (dict(bits_k=3), T.EUNSUPPORTED),
    (dict(bits_v=16), T.EUNSUPPORTED), (dict(table=None), T.EINVAL_ARG),
    (dict(lens=None), T.EINVAL_ARG), (dict(slots=[A] * 5 + [None]), T.EINVAL_ARG),
    (dict(slots=[A, A + 8] + [A] * 4), T.EINVAL_ARG), (dict(weights=A + 4), T.EINVAL_ARG),
    (dict(kind=T.CACHE_BF16, slots=[A, None] + [None] * 4), T.EINVAL_ARG),
]


def refused(status, call, *args, **kw):
    with pytest.raises(T.TqkvError) as e:
        call(*args, **kw)
    assert e.value.status == status, e.value


@pytest.mark.parametrize("other,status", BAD_VIEWS)
def test_views_that_no_entry_point_takes(other, status):
    kv = view(**other)
    refused(status, T.paged_append, kv, A, A, A, 4, 1024, 128)
    refused(status, T.paged_decode_attend, kv, A, 1024, 8, 0.1, 100, A)
    refused(status, T.paged_evict, kv, 64, 0, 0, A, 4, A)
    assert T.paged_decode_workspace_size(kv, 8, 100) == 0
    assert T.paged_evict_workspace_size(kv, 64) == 0


def test_no_view():
    assert T.lib().tqkv_paged_append(None, A, A, None, 1, 8, 8, None) == T.EINVAL_ARG
    assert T.lib().tqkv_paged_decode_attend(None, A, 8, 1, 1.0, -1, 1, A, None, 0, None) == T.EINVAL_ARG
    assert T.lib().tqkv_paged_evict(None, 1, 0, 0, A, 1, A, None, None, None, 0, None) == T.EINVAL_ARG
    assert T.lib().tqkv_paged_decode_workspace_size(None, 8, 100) == 0


def test_append_refusals():
    kv = view()
    ok = dict(kv=kv, k=A, v=A, starts=A, tokens=4, token_stride=1024, head_stride=128)
    for other, status in [(dict(k=None), T.EINVAL_ARG), (dict(v=None), T.EINVAL_ARG),
                          (dict(k=A + 8), T.EINVAL_ARG), (dict(v=A + 2), T.EINVAL_ARG),
                          (dict(starts=A + 1), T.EINVAL_ARG), (dict(tokens=-1), T.EINVAL_SHAPE),
                          (dict(tokens=1 << 40), T.EINVAL_SHAPE),
                          (dict(starts=None, tokens=3), T.EINVAL_SHAPE),
                          (dict(token_stride=1020), T.EINVAL_ARG), (dict(head_stride=4), T.EINVAL_ARG)]:
        refused(status, T.paged_append, **{**ok, **other})
    T.paged_append(**{**ok, "tokens": 0, "k": None, "v": None})  # nothing to do


def test_attend_refusals():
    kv = view()
    ok = dict(kv=kv, q=A, q_stride=1024, H=8, scale=0.1, max_rows=512, out=A, workspace=A,
              workspace_bytes=1 << 30)
    need = T.paged_decode_workspace_size(kv, 8, 512)
    for other, status in [(dict(q=None), T.EINVAL_ARG), (dict(out=None), T.EINVAL_ARG),
                          (dict(q=A + 8), T.EINVAL_ARG), (dict(out=A + 1), T.EINVAL_ARG),
                          (dict(q_stride=1022), T.EINVAL_ARG), (dict(H=0), T.EINVAL_SHAPE),
                          (dict(H=6), T.EINVAL_SHAPE), (dict(H=33 * 4), T.EUNSUPPORTED),
                          (dict(max_rows=0), T.EINVAL_SHAPE), (dict(max_rows=513), T.EINVAL_SHAPE),
                          (dict(workspace_bytes=need - 1), T.EINVAL_ARG),
                          (dict(workspace=A + 8), T.EINVAL_ARG)]:
        refused(status, T.paged_decode_attend, **{**ok, **other})
    huge = view(batch=1024, table_stride=1 << 24)
    refused(T.EUNSUPPORTED, T.paged_decode_attend, **{**ok, "kv": huge, "max_rows": 1 << 30})


def test_evict_refusals():
    ok = dict(kv=view(), budget=64, sinks=4, recent=8, dst_table=A, dst_stride=4, dst_lens=A,
              dst_weights=2 * A, kept=A)
    for other, status in [(dict(kv=view(weights=None)), T.EINVAL_ARG),
                          (dict(dst_table=None), T.EINVAL_ARG), (dict(dst_lens=None), T.EINVAL_ARG),
                          (dict(dst_weights=A), T.EINVAL_ARG), (dict(dst_table=A + 2), T.EINVAL_ARG),
                          (dict(dst_weights=A + 2), T.EINVAL_ARG), (dict(kept=A + 1), T.EINVAL_ARG),
                          (dict(dst_lens=A + 3), T.EINVAL_ARG), (dict(budget=0), T.EINVAL_SHAPE),
                          (dict(sinks=-1), T.EINVAL_SHAPE), (dict(recent=-1), T.EINVAL_SHAPE),
                          (dict(sinks=60, recent=5), T.EINVAL_SHAPE),
                          (dict(sinks=1 << 62, recent=1 << 62), T.EINVAL_SHAPE),
                          (dict(budget=257), T.EINVAL_SHAPE), (dict(dst_stride=0), T.EINVAL_SHAPE),
                          (dict(dst_stride=1 << 40), T.EINVAL_SHAPE),
                          (dict(kept=None, workspace=A, workspace_bytes=2 * 4 * 64 * 4 - 1), T.EINVAL_ARG)]:
        refused(status, T.paged_evict, **{**ok, **other})


def test_workspace_sizes():
    kv = view(weights=None)
    n = T.paged_decode_workspace_size(kv, 8, 512)
    tracked = T.paged_decode_workspace_size(view(), 8, 512)
    assert tracked - n == 2 * 8 * 512 * 4  # the scores
    assert T.paged_decode_workspace_size(view(), 8, 33) - T.paged_decode_workspace_size(kv, 8, 33) == 2 * 8 * 48 * 4
    assert n >= 2 * 8 * 130 * 4
    assert T.paged_decode_workspace_size(kv, 8, 513) == 0 and T.paged_decode_workspace_size(kv, 7, 512) == 0
    assert T.paged_evict_workspace_size(kv, 64) == 2 * 4 * 64 * 4
    assert T.paged_evict_workspace_size(kv, 0) == 0


def test_struct_layout_matches_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "tqkv.h"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(tqkv_paged_kv));']
    lines += [f'  printf("{f} %zu\\n", offsetof(tqkv_paged_kv, {f}));' for f, _ in T.PagedKv._fields_]
    src = tmp_path / "abi.c"
    src.write_text("\n".join(lines + ["  return 0;\n}"]))
    exe = tmp_path / "abi"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {line.split()[0]: int(line.split()[1]) for line in out if line}
    assert got["size"] == ctypes.sizeof(T.PagedKv)
    for f, _ in T.PagedKv._fields_:
        assert got[f] == getattr(T.PagedKv, f).offset, f
