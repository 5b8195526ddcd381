"""Moves of state slots (bm_hip_slots_copy_dev, bm_hip_slots_compact_dev),
byte for byte."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import at, gpu

pytestmark = pytest.mark.gpu


def note(msg):
    print("[case] " + msg, flush=True)


class Pool:
    """layers x slots of `size` bytes in a buffer with gaps, slot-major if
    `inside` (a slot's layers behind one another)."""

    def __init__(self, slots, layers, size, gap=0, shift=0, inside=False, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.slots, self.layers, self.size, self.shift = slots, layers, size, shift
        if inside:
            self.ls, self.ss = size + gap, layers * (size + gap) + gap
        else:
            self.ss, self.ls = size + gap, slots * (size + gap) + 3 * gap
        n = shift + max((layers - 1) * self.ls + (slots - 1) * self.ss + size, 1) + 16
        self.buf = torch.randint(0, 256, (n,), dtype=torch.uint8, generator=g).cuda()

    def descriptor(self):
        return bh.Slots(base=at(self.buf) + self.shift, n_slots=self.slots, n_layers=self.layers,
                        slot_bytes=self.size, slot_stride=self.ss, layer_stride=self.ls)

    def spans(self, slot):
        for l in range(self.layers):
            o = self.shift + l * self.ls + slot * self.ss
            yield slice(o, o + self.size)

    def moved(self, src, dst):
        """The buffer after the call: every pair reads the old one, the first
        pair of a dst counts."""
        old = self.buf.cpu().numpy()
        new, seen = old.copy(), set()
        for s, d in zip(src, dst):
            if not (-1 <= s < self.slots and 0 <= d < self.slots) or d in seen:
                continue
            seen.add(d)
            for a, b in zip(self.spans(max(s, 0)), self.spans(d)):
                new[b] = 0 if s < 0 else old[a]
        return new


def copy(hip, pools, src, dst, stream=None):
    ds = (bh.Slots * len(pools))(*[p.descriptor() for p in pools])
    s, d = gpu(np.array(src), torch.int32), gpu(np.array(dst), torch.int32)
    want = [p.moved(src, dst) for p in pools]
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_copy_dev(ds, len(pools), at(s), at(d), len(src), stream))
    torch.cuda.synchronize()
    for p, w in zip(pools, want):
        assert np.array_equal(p.buf.cpu().numpy(), w)


LISTS = [([0], [1]), ([3, 3, 3], [0, 1, 2]), ([0, 1, 2, 3], [1, 2, 3, 0]), ([0, 4], [4, 0]),
         ([-1, 2], [2, 5]), ([0, 1, 2], [5, 5, 5]), ([9, 1, 2], [5, 5, 5]), ([1, 2], [9, -1]),
         ([-2, 6, 1 << 30, 2], [0, 1, 2, 3]), ([2, 2], [2, 3]), ([-1], [0])]


@pytest.mark.parametrize("size,gap,shift", [(16, 0, 0), (4096, 16, 0), (100, 4, 4), (33, 7, 1),
                                            (1, 0, 3), (70000, 0, 16), (65552, 16, 0)])
@pytest.mark.parametrize("inside", [False, True])
def test_copy_lists(hip, size, gap, shift, inside):
    for src, dst in LISTS:
        note("copy size=%d %s -> %s" % (size, src, dst))
        copy(hip, [Pool(6, 3, size, gap, shift, inside, seed=size)], src, dst)


@pytest.mark.parametrize("n", [2, 17, 64, 65, 255, 256, 257, 1000, 1024])
def test_copy_many_pairs(hip, n):
    """Permutations, random parents and repeated destinations, over more than
    one pool at once."""
    r = np.random.default_rng(n)
    slots = n + 5
    for kind in ("permute", "parents", "anything"):
        if kind == "permute":
            dst = r.permutation(slots)[:n]
            src = r.permutation(dst)
        elif kind == "parents":
            dst = r.permutation(slots)[:n]
            src = r.choice(dst, n)
            src[::7] = -1
        else:
            src, dst = r.integers(-3, slots + 2, n), r.integers(-2, slots + 2, n)
        note("copy n=%d %s" % (n, kind))
        copy(hip, [Pool(slots, 2, 272, 0, 0, False, 1), Pool(slots, 1, 4 * 37, 4, 4, False, 2),
                   Pool(slots, 2, 9, 0, 0, True, 3)], [int(v) for v in src], [int(v) for v in dst])


def compacted(table, slots):
    live = sorted({s for s in table if 0 <= s < slots})
    n = len(live)
    free = [s for s in range(n) if s not in live]
    to = dict(zip([s for s in live if s >= n], free))
    return [to.get(s, s) for s in table], to, n


@pytest.mark.parametrize("slots,live", [(1, 1), (2, 1), (7, 0), (7, 7), (64, 20), (65, 33),
                                        (1000, 500), (1000, 999), (4097, 100), (65536, 300)])
@pytest.mark.parametrize("alias", [False, True])
def test_compact(hip, slots, live, alias):
    r = np.random.default_rng(slots + live)
    table = list(r.permutation(slots)[:live]) + [-1, slots, 1 << 30, -5]
    if live:
        table += [table[0], table[live - 1]]  # two sequences on one slot
    table = [int(v) for v in r.permutation(table)]
    size = 1040 if slots < 2000 else 16
    pools = [Pool(slots, 3, size, 0, 0, False, 5), Pool(slots, 1, 6, 1, 1, False, 6)]
    new, moves, n = compacted(table, slots)
    want = [p.moved(list(moves.keys()), list(moves.values())) for p in pools]
    ds = (bh.Slots * 2)(*[p.descriptor() for p in pools])
    t = gpu(np.array(table), torch.int32)
    out = t if alias else torch.full_like(t, 99)
    count = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    work = torch.full((hip.bm_hip_slots_compact_workspace_bytes(slots),), 0xFF, dtype=torch.uint8,
                      device="cuda")
    note("compact slots=%d live=%d" % (slots, live))
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_compact_dev(ds, 2, at(t), at(out), len(table), at(count), at(work),
                                          None))
    torch.cuda.synchronize()
    assert out.tolist() == new
    assert count.item() == n
    for p, w in zip(pools, want):
        assert np.array_equal(p.buf.cpu().numpy(), w)


def test_compact_of_an_empty_table(hip):
    p = Pool(5, 1, 64)
    before = p.buf.clone()
    count = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    work = torch.zeros(hip.bm_hip_slots_compact_workspace_bytes(5), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_compact_dev(C.byref(p.descriptor()), 1, None, None, 0, at(count),
                                          at(work), None))
    torch.cuda.synchronize()
    assert count.item() == 0 and torch.equal(before, p.buf)
    # without a place for the count
    t = torch.tensor([4], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_compact_dev(C.byref(p.descriptor()), 1, at(t), at(t), 1, None,
                                          at(work), None))
    torch.cuda.synchronize()
    assert t.tolist() == [0]


def test_copy_of_more_blocks_than_a_grid_row(hip):
    """1024 pairs leave a block four bytes of a slot: slots of 2^26 + 21 bytes
    need more blocks than a launch has along x.  Two slots change places."""
    n = (1 << 26) + 21
    buf = torch.randint(0, 256, (2, n), dtype=torch.uint8, device="cuda")
    want = buf.flip(0).clone()
    src, dst = gpu(np.array([0, 1] + [-1] * 1022), torch.int32), gpu(np.array([1, 0] + [-1] * 1022), torch.int32)
    d = bh.Slots(base=at(buf), n_slots=2, n_layers=1, slot_bytes=n, slot_stride=n, layer_stride=0)
    note("copy of 2 x %d bytes" % n)
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_copy_dev(C.byref(d), 1, at(src), at(dst), 1024, None))
    torch.cuda.synchronize()
    assert torch.equal(buf, want)
