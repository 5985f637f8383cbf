"""Page tables on the GPU against a walk over the sequences: reserve, release,
both in turn, captured, and what wrong tables leave alone."""
import numpy as np
import pytest

from prompt_ref import Tables
from test_gpu_capture import captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import tqkv
    assert tqkv.hip().device_count() > 0, "no GPU visible"
    return tqkv


class Device:
    def __init__(self, T, t, tokens=0):
        self.T, self.t = T, t
        self.table, self.lens, self.free = (T.DeviceArray.of(x) for x in (t.table, t.lens, t.free))
        self.count = T.DeviceArray.of(np.array([t.count], np.int32))
        self.starts = T.DeviceArray((t.B + 1,), np.int32, np.full(t.B + 1, -9, np.int32))
        self.granted = T.DeviceArray((t.B,), np.int32, np.full(t.B, -9, np.int32))
        self.slots = T.DeviceArray((tokens + 2, 4), np.int32, np.full((tokens + 2, 4), -9, np.int32))
        self.tokens = tokens

    def view(self, **other):
        t = self.t
        c = dict(batch=t.B, page_rows=t.R, num_pages=t.pages, table=self.table.ptr, table_stride=t.width,
                 lens=self.lens.ptr, free_pages=self.free.ptr, free_count=self.count.ptr)
        c.update(other)
        return self.T.page_tables(**c)

    def reserve(self, counts, stream=None):
        d = self.T.DeviceArray.of(np.asarray(counts, np.int32))
        self.T.paged_reserve(self.view(), d.ptr, self.tokens, self.starts.ptr, self.granted.ptr, self.slots.ptr, stream)
        self.T.hip().sync()

    def release(self, keep, shared=None, stream=None):
        d = self.T.DeviceArray.of(np.asarray(keep, np.int32))
        s = None if shared is None else self.T.DeviceArray.of(np.asarray(shared, np.int32))
        self.T.paged_release(self.view(), d.ptr, None if s is None else s.ptr, stream)
        self.T.hip().sync()

    def same(self, plan=None):
        t = self.t
        assert np.array_equal(self.lens.numpy(), t.lens)
        assert int(self.count.numpy()[0]) == t.count
        assert np.array_equal(self.table.numpy(), t.table)
        assert np.array_equal(self.free.numpy(), t.free)
        if plan is not None:
            starts, granted, slots = plan
            assert np.array_equal(self.starts.numpy(), starts)
            assert np.array_equal(self.granted.numpy(), granted)
            got = self.slots.numpy()
            assert np.array_equal(got[:self.tokens], slots)
            assert np.all(got[self.tokens:] == -9)  # behind the tokens nothing is written


CASES = [
    # lens, counts, tokens, R, width, spare pages
    ([0], [1], 1, 16, 1, 1),
    ([0], [0], 0, 16, 1, 1),
    ([15, 16, 17, 0], [1, 1, 1, 1], 4, 16, 3, 8),
    ([5, 0, 300, 64], [700, 33, 0, 1], 900, 64, 16, 20),       # fewer tokens than the bound
    ([5, 0, 300, 64], [700, 33, 0, 1], 734, 64, 16, 11),       # pages to the last one
    ([5, 0, 300, 64], [700, 33, 0, 1], 734, 64, 16, 10),       # one short: the first is refused
    ([5, 40, 9], [100, 8, 3], 111, 16, 4, 30),                 # past the table
    ([5, 40, 9], [20, 30, 3], 40, 16, 8, 30),                  # past the bound on tokens
    ([-4, 99999, 3], [10, 1, -5], 20, 32, 4, 9),               # lengths out of range, counts below 0
    ([7] * 1024, [1] * 1024, 1024, 16, 1, 0),                  # a whole batch without new pages
    ([16] * 1024, [1] * 1024, 1024, 16, 2, 1000),              # 24 of them refused
    ([3] * 700, [9] * 700, 6300, 16, 2, 900),
    ([100, 0, 31], [2000, 1500, 1], 3501, 256, 9, 20),         # the grid's tokens
    ([0, 0], [2 ** 31 - 1, 5], 10, 16, 4, 4),                  # a count that passes 32 bits with its length
]


@pytest.mark.parametrize("lens,counts,tokens,R,width,spare", CASES)
def test_reserve(T, lens, counts, tokens, R, width, spare):
    print("[reserve]", lens[:4], counts[:4], tokens, R, width, spare, flush=True)
    used = sum(min(-(-max(n, 0) // R), width) for n in lens)
    t = Tables(lens, R, width, used + spare, seed=len(lens))
    d = Device(T, t, tokens)
    d.reserve(counts)
    d.same(t.reserve(counts, tokens))


@pytest.mark.parametrize("lens,keep,shared,R,width", [
    ([33], [0], None, 16, 3), ([33], [33], None, 16, 3), ([33], [16], None, 16, 3), ([33], [17], None, 16, 3),
    ([100, 0, 64, 5], [-1, 5, 1000, 4], None, 16, 8), ([100, 80, 64], [0, 0, 40], [2, 9, 1], 16, 8),
    ([100, 80, 64], [0, 0, 40], [-3, 0, 4], 32, 8), ([5000] * 40, [0, 4999, 1200, 16] * 10, None, 16, 400),
    ([999] * 1024, [0, 500] * 512, None, 64, 16)])
def test_release(T, lens, keep, shared, R, width):
    print("[release]", lens[:4], keep[:4], shared, R, width, flush=True)
    t = Tables(lens, R, width, sum(-(-n // R) for n in lens) + 3, seed=R)
    d = Device(T, t)
    d.release(keep, shared)
    t.release(keep, shared)
    d.same()


def test_release_leaves_out_what_names_no_page(T):
    t = Tables([200, 90, 40], 16, 16, 30, seed=5)
    t.table[0, 2], t.table[0, 5], t.table[1, 0] = -1, 30, 2 ** 31 - 1
    d = Device(T, t)
    d.release([0, 0, 40])
    t.release([0, 0, 40])
    d.same()
    assert t.count == 30 - 13 - 6 - 3 + 13 - 2 + 6 - 1


def test_release_of_pages_named_twice_stays_in_the_stack(T):
    """More entries than pages: the stack takes what it holds."""
    t = Tables([64, 64], 16, 4, 8, seed=5)
    t.table[1] = t.table[0]
    t.count = 3
    d = Device(T, t)
    d.release([0, 0])
    t.release([0, 0])
    d.same()
    assert t.count == 8


@pytest.mark.parametrize("height", [-5, 10 ** 6])
def test_height_out_of_range(T, height):
    t = Tables([20, 5], 16, 8, 12, seed=2)
    t.free[:] = np.arange(12)
    t.count = height
    d = Device(T, t, 60)
    d.reserve([30, 12])
    d.same(t.reserve([30, 12], 60))


def test_reserve_then_release_leaves_the_stack_as_it_was(T):
    rng = np.random.default_rng(8)
    lens = rng.integers(0, 300, 90)
    t = Tables(lens, 16, 40, 2500, seed=3)
    before = (t.table.copy(), t.lens.copy(), t.free.copy(), t.count)
    d = Device(T, t, 90 * 200)
    counts = rng.integers(0, 200, 90)
    d.reserve(counts)
    plan = t.reserve(counts, 90 * 200)
    d.same(plan)
    assert np.all(plan[1] >= 0)
    d.release(before[1])
    for got, want in zip((d.table, d.lens, d.free, d.count), before):
        assert np.array_equal(got.numpy().reshape(-1), np.asarray(want).reshape(-1))


def test_a_serving_loop(T):
    """Admissions, steps, endings and refusals, 60 rounds."""
    rng = np.random.default_rng(4)
    t = Tables([0] * 33, 32, 20, 300, seed=1)
    d = Device(T, t, 1500)
    refused = 0
    for i in range(60):
        keep = np.where(rng.random(33) < 0.1, 0, t.lens)
        shared = rng.integers(0, 2, 33) if i % 7 == 3 else None
        d.release(keep, shared)
        t.release(keep, shared)
        counts = np.where(t.lens == 0, rng.integers(0, 400, 33), 1)
        d.reserve(counts)
        plan = t.reserve(counts, 1500)
        d.same(plan)
        refused += int((plan[1] < 0).sum())
    assert refused > 0


def test_without_slots_and_granted(T):
    t = Tables([20, 5], 16, 8, 12, seed=2)
    d = Device(T, t, 60)
    counts = T.DeviceArray.of(np.array([30, 12], np.int32))
    T.paged_reserve(d.view(), counts.ptr, 60, d.starts.ptr)
    T.hip().sync()
    starts, _, _ = t.reserve([30, 12], 60)
    d.same()
    assert np.array_equal(d.starts.numpy(), starts)
    assert np.all(d.granted.numpy() == -9) and np.all(d.slots.numpy() == -9)


@pytest.mark.parametrize("tokens", [40, 3000])
def test_captured_calls_follow_the_tables(T, tokens):
    t = Tables([3, 0, 70], 16, 300, 900, seed=9)
    d = Device(T, t, tokens)
    counts = T.DeviceArray.of(np.array([1, 7, 2], np.int32))
    keep = T.DeviceArray.of(np.array([2 ** 30] * 3, np.int32))

    def call(stream):
        T.paged_release(d.view(), keep.ptr, None, stream)
        T.paged_reserve(d.view(), counts.ptr, tokens, d.starts.ptr, d.granted.ptr, d.slots.ptr, stream)

    with captured(T, call) as launch:
        for i in range(4):
            c = np.array([1, 7 * i, tokens // 5 if i == 2 else 2], np.int32)
            k = np.array([2 ** 30, 0 if i == 3 else 5, 2 ** 30], np.int32)
            T.hip().copy_in(counts.ptr, c)
            T.hip().copy_in(keep.ptr, k)
            launch()
            t.release(k)
            d.same(t.reserve(c, tokens))
