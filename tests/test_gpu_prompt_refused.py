"""A step whose batch holds a sequence that gets no pages: tokens laid out by
the slots of the reserve, not by what was asked."""
import numpy as np
import pytest

import oracle_lib as O
import prompt_ref as R
from inputs import kv_bf16
from paged_ref import AFFINE, BF16, Paged
from test_gpu_prompt import T, say  # noqa: F401 (T: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, AFFINE])
@pytest.mark.parametrize("counts,refused", [([20, 70, 9, 33], 1), ([1, 1, 1, 1], 2), ([40, 5, 200, 1], 2), ([300, 8, 8, 8], 0)])
def test_a_refused_sequence_and_those_behind_it(T, kind, counts, refused):
    say("refused", kind, counts, refused)
    B, Hkv, G, D, R_, width = 4, 1, 2, 128, 16, 12
    H = Hkv * G
    held = [16, 30, 32, 5]
    p = Paged(held, Hkv, D, R_, kind, 4, 8, 32, stride=width, spare=12, seed=1).fill(2)
    t = R.Tables([0] * B, R_, width, p.pages)
    t.table, t.lens = p.table, p.lens
    # A page short for it: the stack holds what the others need, and they are served in order.
    needs = [-(-(n + c) // R_) - -(-n // R_) for n, c in zip(held, counts)]
    if counts[refused] + held[refused] <= width * R_:
        t.count = sum(needs[:refused]) + max(needs[refused] - 1, 0)
        assert needs[refused] > 0
    else:
        t.count = sum(needs) - needs[refused]
    t.free = np.full(p.pages, -7, np.int32)
    t.free[:t.count] = p.spare[:t.count]
    # (Behind a sequence that asked for more than is left, those are served that need no page.)
    d = p.device(T)
    free, count = T.DeviceArray.of(t.free), T.DeviceArray.of(np.array([t.count], np.int32))
    tables = T.page_tables(B, R_, p.pages, d.table.ptr, width, d.lens.ptr, free.ptr, count.ptr)
    n = sum(counts)
    dc = T.DeviceArray.of(np.array(counts, np.int32))
    starts, granted, slots = T.DeviceArray((B + 1,), np.int32), T.DeviceArray((B,), np.int32), T.DeviceArray((n, 4), np.int32)
    T.paged_reserve(tables, dc.ptr, n, starts.ptr, granted.ptr, slots.ptr)
    T.hip().sync()
    hs, hg, hslots = t.reserve(counts, n)
    assert np.array_equal(granted.numpy(), hg) and hg[refused] == -1 and np.array_equal(slots.numpy(), hslots)
    assert np.array_equal(starts.numpy(), hs) and (hg >= 0).sum() >= 1
    # What each sequence asked to enter, and the same laid out by the slots: the
    # token at a slot's position of its sequence. Rows behind the last slot hold anything.
    asked = [kv_bf16((c, H + 2 * Hkv, D), 50 + b) for b, c in enumerate(counts)]
    x = kv_bf16((n, H + 2 * Hkv, D), 99)
    for i, (page, row, position, b) in enumerate(hslots):
        if b >= 0:
            x[i] = asked[b][position - held[b]]
    turns, m = T.rope_turns(D)
    dt = T.DeviceArray.of(np.array(turns, np.uint64))
    dx, q = T.DeviceArray.of(x), T.DeviceArray((n, H, D), np.uint16, np.full((n, H, D), 0x7FC1, np.uint16))
    out = T.DeviceArray((n, H, D), np.uint16, np.full((n, H, D), 0x7FC1, np.uint16))
    step = (H + 2 * Hkv) * D
    k = dx.ptr + 2 * H * D
    before = d.host()
    T.paged_append_rope(d.view(), T.rope(D, 0, m, dt.ptr), dx.ptr, H, step, q.ptr, H * D, k, k + 2 * Hkv * D, step, D, slots.ptr, n)
    T.paged_prefill_attend(d.view(), q.ptr, H * D, H, starts.ptr, n, D ** -0.5, width * R_, out.ptr)
    T.hip().sync()
    last = int(hs[-1])
    # The pool: every granted token's row where its sequence holds it, all else as it was.
    p.sides = d.host()
    theta, _ = R.thetas(D, 10000.0)
    written = np.zeros(before[0][0].shape[:3], bool)
    for i, (page, row, position, b) in enumerate(hslots[:last]):
        assert page == t.table[b, position // R_] and row == position % R_
        written[page, :, row] = True
        if kind == BF16:
            assert np.array_equal(p.sides[1][0][page, 0, row], asked[b][position - held[b], H + Hkv])
        else:
            for got, want in zip(p.sides[1], p.stored(asked[b][position - held[b]][H + Hkv:], 8)):
                assert np.array_equal(got[page, :, row], want)
    for side, was in zip(p.sides, before):
        for now, then in zip(side, was):
            assert np.array_equal(now[~written], then[~written])
    want, tol = R.rotated(x[:last, :H], hslots[:last, 2], theta, m, False)
    R.check(O.bf16_to_f32(q.numpy()[:last]), want, tol, "queries")
    want, tol = R.paged(p, q.numpy(), hs, D ** -0.5)
    R.check(O.bf16_to_f32(out.numpy()[:last]), want[:last], tol[:last], "prefill")
    assert np.all(out.numpy()[last:] == 0x7FC1)  # no sequence's
