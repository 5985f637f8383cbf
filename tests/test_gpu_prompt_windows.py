"""Windows next to the largest that the type holds, and more queries than rows:
the queries before a sequence's first row see none, the others all."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged
from test_gpu_prompt import T, say, starts_of  # noqa: F401 (T: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("counts", [[25, 9], [300, 200]])
@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 4, 2 ** 31 - 90, 2 ** 31 - 1, 2 ** 40])
def test_windows_next_to_the_largest(T, kind, D, counts, window):
    say("wide window", kind, D, counts, window)
    lens = [counts[0] - 5, counts[1] - 3]
    p = Paged(lens, 1, D, 16, kind, 4, 8, 32, stride=512, seed=5).fill(2)
    starts, n = starts_of(counts), sum(counts)
    q = kv_bf16((n, 1, D), 3)
    d = p.device(T)
    dq, ds = T.DeviceArray.of(q), T.DeviceArray.of(starts)
    out = T.DeviceArray((n, 1, D), np.uint16)
    rows = p.stride * p.R
    need = T.paged_prefill_workspace_size(d.view(), 1, n, rows)
    # Partial results that nothing wrote are numbers here, not NaN, which the join would notice.
    ws = T.DeviceArray((max(need, 16),), np.uint8, np.full((max(need, 16),), 0x3F, np.uint8))
    T.paged_prefill_attend(d.view(), dq.ptr, D, 1, ds.ptr, n, D ** -0.5, rows, out.ptr, window, ws.ptr, need)
    T.hip().sync()
    want, tol = R.paged(p, q, starts, D ** -0.5)
    got = O.bf16_to_f32(out.numpy())
    R.check(got, want, tol, "wide window")
    for i in range(2):
        assert np.all(got[starts[i]:starts[i + 1] - lens[i]] == 0.0)
