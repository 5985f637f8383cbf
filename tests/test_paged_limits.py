"""Sizes and overlaps at which the paged cache's entry points draw their lines,
on the host (refusals come before any launch)."""
import pytest

import tqkv as T
from test_paged_host import A, refused, view


@pytest.mark.parametrize("weights", [None, A])
def test_no_workspace_for_calls_that_are_refused(weights):
    """Sizes that no window makes acceptable have no workspace."""
    many = view(batch=1024, table_stride=1 << 24, weights=weights)
    refused(T.EUNSUPPORTED, T.paged_decode_attend, many, A, 1024, 8, 0.1, 1 << 30, A)
    assert T.paged_decode_workspace_size(many, 8, 1 << 30) == 0
    wide = view(batch=1024, kv_heads=1024, dim=512, weights=weights)
    refused(T.EUNSUPPORTED, T.paged_decode_attend, wide, A, 1 << 24, 1 << 14, 0.1, 512, A)
    refused(T.EUNSUPPORTED, T.paged_decode_attend, wide, A, 1 << 24, 1 << 14, 0.1, 512, A, window=1)
    assert T.paged_decode_workspace_size(wide, 1 << 14, 512) == 0
    assert T.paged_decode_workspace_size(wide, 1 << 10, 512) > 0


def test_no_eviction_workspace_for_a_budget_that_is_refused():
    kv = view(table_stride=1 << 24)
    for budget, stride in (((1 << 29) + 1, 1 << 24), (0, 4)):
        refused(T.EINVAL_SHAPE, T.paged_evict, kv, budget, 0, 0, A, stride, A)
        assert T.paged_evict_workspace_size(kv, budget) == 0
    assert T.paged_evict_workspace_size(kv, 1 << 29) == 2 * 4 * 4 << 29


def test_eviction_refuses_overlapping_weights():
    """The rows' new weights may touch the old ones' end or begin, and no more."""
    kv = view(weights=16 * A)  # 2 x 4 x 512 weights: 16 KB
    ok = dict(kv=kv, budget=64, sinks=4, recent=8, dst_table=A, dst_stride=4, dst_lens=A, kept=None,
              workspace=A, workspace_bytes=0)  # too small a workspace: refused in any case
    new = 2 * 4 * 256 * 4
    for at in (16 * A, 16 * A + 4, 16 * A + (1 << 14) - 4, 16 * A - new + 4):
        with pytest.raises(T.TqkvError, match="overlaps") as e:
            T.paged_evict(**ok, dst_weights=at)
        assert e.value.status == T.EINVAL_ARG
    for at in (16 * A + (1 << 14), 16 * A - new, None):
        with pytest.raises(T.TqkvError, match="workspace"):
            T.paged_evict(**ok, dst_weights=at)
