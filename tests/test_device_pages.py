"""DevicePageTable: every value is a whole number, so every comparison is exact.

The model is a list-of-lists page table in Python with the documented order (the
o-th missing page, row by row, is the o-th from the top of the stack; a trim
puts pages back so that the last page of the last row ends lowest), and the
host-side PageTable, whose page order reserve must reproduce.
"""
import ctypes
import random

import numpy as np
import pytest
import torch

from specdec import _lib as L
from specdec.kvcache import PAGE, DevicePageTable, PageTable

gpu = pytest.mark.gpu
DEV = "cuda"


class Model:
    def __init__(self, B, W, n_pages):
        self.rows = [[] for _ in range(B)]
        self.shared = [0] * B
        self.W, self.n = W, n_pages
        self.stack = list(range(n_pages - 2, -1, -1))
        self.err = 0

    def reserve(self, lens, new, max_tokens):
        starts = [0]
        bad = 0
        for b, a in zip(lens, new):
            ok = b >= 0 and a >= 0 and b + a <= self.W * PAGE
            bad |= 0 if ok else 1
            starts.append(starts[-1] + (a if ok else 0))
        need = [-(-(b + a) // PAGE) for b, a in zip(lens, new)]
        short = [max(0, n - len(r)) for n, r in zip(need, self.rows)]
        if not bad and sum(short) > len(self.stack):
            bad = 4
        if not bad and starts[-1] > max_tokens:
            bad = 8
        slots = [-1] * max_tokens
        if bad:
            self.err |= bad
            return slots, starts
        for b, n in enumerate(short):
            self.rows[b] += [self.stack.pop() for _ in range(n)]
        at = 0
        for b, a in enumerate(new):
            for i in range(a):
                p = lens[b] + i
                slots[at] = self.rows[b][p // PAGE] * PAGE + p % PAGE
                at += 1
        return slots, starts

    def trim(self, lens):
        gone = []
        for b, n in enumerate(lens):
            keep = max(-(-max(n, 0) // PAGE), self.shared[b])
            gone += self.rows[b][keep:]
            self.rows[b] = self.rows[b][:keep]
        self.stack += gone[::-1]

    def same_as(self, t):
        bt = np.full((len(self.rows), self.W), -1)
        for b, r in enumerate(self.rows):
            bt[b, :len(r)] = r
        assert np.array_equal(t.block_table.cpu().numpy(), bt)
        assert t.owned.tolist() == [len(r) for r in self.rows]
        n = int(t.n_free)
        assert n == len(self.stack) and t.free[:n].tolist() == self.stack
        assert int(t.err) == self.err


def _lens(v):
    return torch.tensor(v, dtype=torch.long, device=DEV)


@gpu
@pytest.mark.parametrize("B,W,seed", [(1, 1, 0), (1, 40, 1), (7, 3, 2), (64, 66, 3), (1025, 5, 4),
                                      (2500, 9, 5)])
def test_random_runs_against_the_model(B, W, seed):
    rng = random.Random(seed)
    n_pages = B * W * 3 // 4 + 2
    t, m = DevicePageTable(B, W, n_pages, DEV), Model(B, W, n_pages)
    lens = [0] * B
    for step in range(12):
        if step % 3 == 0:                                   # ragged prompts or chunks
            new = [min(rng.choice([0, 1, PAGE, rng.randint(0, W * PAGE)]), W * PAGE - n)
                   for n in lens]
            room = sum(new) + rng.choice([0, 0, 5, 1000])
            got = t.reserve(_lens(lens), _lens(new), max_tokens=room)
        else:                                               # a round of k + 1 tokens
            k = rng.choice([1, 5, 17])
            if max(lens) + k > W * PAGE:
                k = 0
            new, room = [k] * B, B * k
            got = t.reserve(_lens(lens), k)
        before = m.err
        want = m.reserve(lens, new, room)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
        m.same_as(t)
        if m.err == before:
            lens = [n + a for n, a in zip(lens, new)]
        m.err = 0
        t.err.zero_()
        back = [n if rng.random() < 0.5 else rng.randint(0, n) for n in lens]
        if rng.random() < 0.3:
            back = [0] * B
        t.trim(_lens(back))
        m.trim(back)
        lens = back
        m.same_as(t)


@gpu
def test_reserve_hands_out_the_host_tables_pages():
    B, W, n = 33, 12, 300
    t, h = DevicePageTable(B, W, n, DEV), PageTable(B, W, n)
    rng = random.Random(7)
    lens = [0] * B
    for q in (5, 200, 1, 130, 17):
        t.reserve(_lens(lens), q)
        h.reserve(lens, q)
        assert np.array_equal(t.block_table.cpu().numpy(), h.bt)
        assert t.owned.tolist() == h.owned.tolist()
        assert t.free[:int(t.n_free)].tolist() == h.free
        lens = [n + rng.randint(0, q) for n in lens]


@gpu
def test_trim_undoes_reserve():
    t = DevicePageTable(40, 20, 700, DEV)
    t.reserve(_lens([0] * 40), _lens([50 * (i % 9) for i in range(40)]), max_tokens=40 * 400)
    base = _lens([50 * (i % 9) for i in range(40)])
    before = [x.clone() for x in (t.block_table, t.owned, t.free, t.n_free)]
    t.reserve(base, 1000)
    t.trim(base)
    assert all(torch.equal(a, b) for a, b in zip(before, (t.block_table, t.owned, t.free, t.n_free)))


@gpu
def test_shared_pages_stay():
    t, m = DevicePageTable(4, 8, 40, DEV), Model(4, 8, 40)
    lens = [3 * PAGE, 2 * PAGE + 1, 0, 5]
    t.reserve(_lens([0] * 4), _lens(lens), max_tokens=2000)
    m.reserve([0] * 4, lens, 2000)
    t.shared.copy_(torch.tensor([2, 1, 0, 4], dtype=torch.int32))
    m.shared = [2, 1, 0, 4]                                  # row 3 owns fewer than it shares
    t.trim(_lens([0, 0, 0, 0]))
    m.trim([0, 0, 0, 0])
    m.same_as(t)
    assert t.owned.tolist() == [2, 1, 0, 1]


@gpu
@pytest.mark.parametrize("lens,new,room,bit", [
    ([0, 0, 3 * PAGE], [1, 1, 1], 3, 1),                     # a row past its table
    ([0, -1, 0], [1, 1, 1], 3, 1),                           # a negative length
    ([0, 0, 0], [1, -2, 1], 3, 1),                           # a negative count
    ([0, 2 ** 62, 0], [1, 2 ** 62, 1], 3, 1),                # far out of range
    ([0, 0, 0], [3 * PAGE, 3 * PAGE, 3 * PAGE], 9 * PAGE, 4),   # eight pages wanted, seven free
    ([0, 0, 0], [4, 4, 4], 11, 8),                           # slots too small
])
def test_a_call_that_cannot_be_done_changes_nothing(lens, new, room, bit):
    t = DevicePageTable(3, 3, 8, DEV)
    before = [x.clone() for x in (t.block_table, t.owned, t.free, t.n_free)]
    slots, _ = t.reserve(_lens(lens), _lens(new), max_tokens=room)
    assert int(t.err) == bit and bool((slots == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, (t.block_table, t.owned, t.free, t.n_free)))
    with pytest.raises(RuntimeError):
        t.check_errors()
    t.check_errors()                                         # raised once
    t.reserve(_lens([0, 0, 0]), 1)
    t.check_errors()
    assert t.owned.tolist() == [1, 1, 1]


@gpu
def test_a_trim_of_more_pages_than_the_pool_has_changes_nothing():
    t = DevicePageTable(2, 3, 4, DEV)
    t.owned.fill_(3)                                         # a table that lies about its pages
    bt = t.block_table.clone()
    t.trim(_lens([0, 0]))
    assert int(t.err) == 1 and int(t.n_free) == 3 and torch.equal(t.block_table, bt)


@gpu
@pytest.mark.parametrize("field,value", [("n_free", 9), ("n_free", -1), ("owned", -1)])
def test_a_broken_table_hands_out_nothing(field, value):
    t = DevicePageTable(2, 3, 8, DEV)
    getattr(t, field).fill_(value)
    before = [x.clone() for x in (t.block_table, t.owned, t.free, t.n_free)]
    slots, _ = t.reserve(_lens([0, 0]), 5)
    assert int(t.err) == 1 and bool((slots == -1).all())
    if field == "n_free":
        t.trim(_lens([0, 0]))
    assert all(torch.equal(a, b) for a, b in zip(before, (t.block_table, t.owned, t.free, t.n_free)))


@gpu
@pytest.mark.parametrize("rows", [3, 100])                   # one launch, two launches
def test_a_floor_of_pages_takes_no_new_tokens(rows):
    t = DevicePageTable(rows, 3, 3 * rows + 1, DEV)
    lens, floor = [PAGE] * rows, torch.zeros(rows, dtype=torch.int32, device=DEV)
    t.reserve(_lens(lens), 0, slot_map=False)
    floor[rows - 1] = 2
    lens[rows - 1] = 2 * PAGE - 1
    before = [x.clone() for x in (t.block_table, t.owned, t.n_free)]
    slots, _ = t.reserve(_lens(lens), 2, floor=floor)
    assert int(t.err) == 16 and bool((slots == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, (t.block_table, t.owned, t.n_free)))
    with pytest.raises(RuntimeError, match="floor"):
        t.check_errors()
    new = [2] * (rows - 1) + [0]                             # nothing new in the row: no error
    t.reserve(_lens(lens), _lens(new), max_tokens=2 * rows, floor=floor)
    lens[rows - 1] = 2 * PAGE
    slots, _ = t.reserve(_lens(lens), 2, floor=floor)
    t.check_errors()
    assert bool((slots >= 0).all())
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens(lens), 2, floor=floor.long())
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens(lens), 2, floor=floor[:1])


@gpu
def test_captured_rounds_follow_the_device_lengths():
    """trim and reserve in a graph, replayed while the lengths move."""
    B, W, n = 16, 10, 200
    t, m = DevicePageTable(B, W, n, DEV), Model(B, W, n)
    lens = _lens([0] * B)
    t.reserve(lens, 1)                                       # load the kernels before the capture
    t.trim(lens)
    m.reserve([0] * B, [1] * B, B)
    m.trim([0] * B)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.trim(lens)
        slots, starts = t.reserve(lens, 9)
    rng = random.Random(3)
    cur = [0] * B
    for _ in range(10):
        lens.copy_(torch.tensor(cur))
        g.replay()
        m.trim(cur)
        want = m.reserve(cur, [9] * B, 9 * B)
        assert slots.tolist() == want[0] and starts.tolist() == want[1]
        m.same_as(t)
        cur = [c + rng.randint(0, 100) for c in cur]


@gpu
def test_nothing_to_reserve_and_more_room_than_tokens():
    t = DevicePageTable(3, 4, 20, DEV)
    slots, starts = t.reserve(_lens([0, 5, 7]), 0)
    assert slots.numel() == 0 and starts.tolist() == [0, 0, 0, 0]
    assert t.owned.tolist() == [0, 1, 1]                     # the lengths themselves need pages
    slots, starts = t.reserve(_lens([0, 5, 7]), _lens([0, 2, 0]), max_tokens=70000)
    assert slots[:2].tolist() == [5, 6] and bool((slots[2:] == -1).all())
    slots, _ = t.reserve(_lens([0, 5, 7]), 3, max_tokens=20)
    assert bool((slots[9:] == -1).all()) and bool((slots[:9] >= 0).all())


@gpu
def test_reserve_without_a_slot_map():
    a, b = DevicePageTable(5, 6, 40, DEV), DevicePageTable(5, 6, 40, DEV)
    new = _lens([0, 5, 600, 128, 1])
    slots, starts = a.reserve(_lens([0] * 5), new, slot_map=False)
    want, want_starts = b.reserve(_lens([0] * 5), new, max_tokens=800)
    assert slots is None and torch.equal(starts, want_starts)
    assert torch.equal(a.block_table, b.block_table) and torch.equal(a.n_free, b.n_free)
    assert int(a.err) == 0


@gpu
def test_refusals():
    t = DevicePageTable(3, 4, 20, DEV)
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens([0, 0]), 1)
    with pytest.raises(L.SpecdecError):
        t.reserve(torch.zeros(3, device=DEV), 1)
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens([0, 0, 0]), _lens([1, 1, 1]))        # no bound for the slots
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens([0, 0, 0]), -1)
    with pytest.raises(L.SpecdecError):
        t.reserve(_lens([0, 0, 0]), 1 << 64, slot_map=False)
    with pytest.raises(L.SpecdecError):
        t.reserve(torch.zeros(3, dtype=torch.long), 1)
    with pytest.raises(L.SpecdecError):
        DevicePageTable(3, 4, 1, DEV)
    s = (t.block_table, t.owned, t.shared, t.free, t.n_free, t.err)
    DevicePageTable.over(*s)
    with pytest.raises(L.SpecdecError):
        DevicePageTable.over(t.block_table.long(), *s[1:])
    with pytest.raises(L.SpecdecError):
        DevicePageTable.over(t.block_table, t.owned[:2], *s[2:])
    with pytest.raises(L.SpecdecError):
        DevicePageTable.over(t.block_table.t(), *s[1:])


def test_refusals_on_cpu():
    with pytest.raises(L.SpecdecError):
        DevicePageTable(3, 4, 20, "cpu")


def test_arguments_are_checked_before_any_launch():
    lib = L.lib()
    n, d = ctypes.c_void_p(0), ctypes.c_void_p(4096)

    def reserve(bt=d, stride=4, W=4, owned=d, pages=20, lens=d, each=1, B=3, slots=d, room=3, ws=d,
                nws=1 << 16):
        return lib.sd_pages_reserve(bt, stride, W, owned, d, pages, d, lens, n, each, n, B, slots,
                                    room, d, d, ws, nws, n)
    assert reserve(B=0) == 0
    assert reserve(B=-1) == -22 and reserve(bt=n) == -22 and reserve(lens=n) == -22
    assert reserve(W=0) == -22 and reserve(stride=3) == -22 and reserve(pages=0) == -22
    assert reserve(room=-1) == -22 and reserve(each=-1) == -22
    assert reserve(W=1 << 25, stride=1 << 25) == -95
    assert reserve(B=1 << 20, W=1 << 10, stride=1 << 10, nws=1 << 30) == -95
    assert reserve(ws=n) == -28 and reserve(nws=16) == -28
    assert lib.sd_pages_trim(d, 4, 4, d, n, d, 20, d, d, 3, d, n) == -22
    assert lib.sd_pages_trim(d, 4, 4, d, d, d, 20, d, d, 0, d, n) == 0


@gpu
@pytest.mark.parametrize("B", [65536, 65537, 70000])
@pytest.mark.parametrize("each", [1, 2, 5])
def test_more_rows_than_a_launch_cuts_into_runs(B, each):
    """Page b goes to row b: every slot is known."""
    want = torch.arange(B, device=DEV).view(-1, 1) * PAGE + torch.arange(each, device=DEV)
    zero = torch.zeros(B, dtype=torch.long, device=DEV)
    t = DevicePageTable(B, 1, B + 1, DEV)
    slots, starts = t.reserve(zero, each)
    assert torch.equal(slots.view(B, each), want)
    assert torch.equal(starts, torch.arange(B + 1, dtype=torch.int32, device=DEV) * each)
    assert torch.equal(t.block_table.view(-1), torch.arange(B, dtype=torch.int32, device=DEV))
    t.check_errors()
    t.trim(zero)
    assert int(t.n_free) == B
    slots, _ = t.reserve(zero, zero + each, max_tokens=B * each + 7)
    assert torch.equal(slots[:-7].view(B, each), want) and bool((slots[-7:] == -1).all())
    t.reserve(zero, each, slot_map=False)
    t.check_errors()


def test_tables_of_more_pages_than_are_counted_are_refused():
    lib = L.lib()
    n, d = ctypes.c_void_p(0), ctypes.c_void_p(4096)

    def trim(W, B):
        return lib.sd_pages_trim(d, W, W, d, d, d, 20, d, d, B, d, n)
    assert trim((1 << 24) - 1, 129) == -95 and trim(1 << 23, 1 << 20) == -95
    assert trim(1 << 24, 1) == -95
