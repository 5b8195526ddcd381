"""The batched recurrence's kernels that only large calls, many sequences or
unusual shapes reach, each by values: against the definition in 64 bits with the
bounds of tests/recurrence.py, slots byte for byte."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import ConvCase, SsmCase, at, check_rows, close, gpu
from test_gpu_recurrence import make
from test_gpu_slots import Pool, compacted, copy

pytestmark = pytest.mark.gpu
KINDS = ["conv", "scan1", "scan5", "scan24"]


def note(msg):
    print("[case] " + msg, flush=True)


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type_name,H,P,N,slot_pad", [
    ("f32", 16, 65, 12, 1), ("bf16", 16, 64, 32, 0), ("f16", 8, 64, 64, 3), ("bf16", 8, 64, 128, 0),
    ("f32", 8, 33, 256, 0), ("f16", 8, 130, 16, 1), ("f32", 4, 64, 100, 0), ("bf16", 5, 50, 200, 1)])
def test_token_states_past_the_caches(hip, type_name, H, P, N, slot_pad):
    """2^24 floats of states and more."""
    n = (1 << 24) // (H * P * N) + 1
    c = SsmCase(type_name, H, P, 1, N, [1] * n, step=True, seed=N, slot_pad=slot_pad)
    c.slots[3], c.slots[n // 2] = -1, c.slots[0]  # padding
    note("step %s H=%d P=%d N=%d, %d sequences" % (type_name, H, P, N, n))
    c.check(hip, "large states")


@pytest.mark.parametrize("type_name,channels,width,n", [
    ("f32", 1028, 4, 515), ("f32", 2048, 2, 514), ("f32", 4, 3, 1025), ("bf16", 2056, 4, 514),
    ("bf16", 4096, 3, 513), ("f16", 64, 4, 1027), ("f16", 2048, 2, 1026), ("bf16", 9, 4, 1025),
    ("f16", 520, 3, 1030)])
def test_conv_tokens_of_many_sequences(hip, type_name, channels, width, n):
    """Several sequences to a thread, with rows that 16-byte loads fit (and
    one that they do not), numbers of sequences that leave a part group."""
    c = ConvCase(type_name, channels, width, [1] * n, step=True, seed=n, act=width != 2,
                 bias=width != 3)
    c.slots[2], c.slots[n - 1], c.slots[n - 2] = -1, c.slots[1], 1 << 20  # padding
    note("conv_step %s channels=%d width=%d n=%d" % (type_name, channels, width, n))
    c.check(hip, "many")


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [2, 3, 4])
def test_conv_around_its_unit(hip, type_name, width):
    """Lengths around the 16 rows that a thread walks and the 8 that it loads
    together."""
    c = ConvCase(type_name, 72, width, [15, 16, 17, 7, 8, 9, 47, 48, 49, 0, 24, 25], seed=width,
                 front=1, tail=2)
    note("conv %s width=%d" % (type_name, width))
    c.check(hip, "unit")


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N", [5, 8])
def test_scan_of_many_heads_of_one_channel(hip, type_name, N):
    """70 heads in a block of 64 channels: more LDS than a kernel has unasked."""
    note("scan %s, 70 heads of one channel, N=%d" % (type_name, N))
    SsmCase(type_name, 70, 1, 1, N, [200, 3, 40], seed=N).check(hip, "heads of one")


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,P,G,N,lens", [
    (2, 32, 1, 16, [1500]), (2, 32, 1, 128, [700, 3, 1100]), (4, 64, 1, 40, [600, 150]),
    (6, 40, 3, 72, [700]), (3, 64, 3, 24, [400, 390]), (1, 96, 1, 200, [520]),
    (5, 64, 1, 9, [129, 257, 1])])
def test_scan_long_in_every_type(hip, type_name, H, P, G, N, lens):
    """Several units to a sequence, with one to eight tiles of a group."""
    note("scan %s H=%d P=%d G=%d N=%d lens=%s" % (type_name, H, P, G, N, lens))
    SsmCase(type_name, H, P, G, N, lens, seed=N).check(hip, "long")


# ---------------------------------------------------------------------------
# what the calls leave in the slots
# ---------------------------------------------------------------------------
def left_in_slots(c, kind, pool, stol):
    got = c.pool()
    for k in c.slots:
        if kind == "conv":
            assert np.array_equal(got[k], pool[k])
        else:
            close(got[k], pool[k], stol[k], "f32", "slot %d" % k)


@pytest.mark.parametrize("kind", KINDS)
def test_state_after_one_sequence_without_starts(hip, kind):
    c = make(kind, [150], seed=4)
    want = c.want()
    d = c.descriptor()
    d.seq_start = None
    w = c.workspace(hip, d) if kind != "conv" else None
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_conv_dev(C.byref(d), None) if kind == "conv" else
             hip.bm_hip_ssm_dev(C.byref(d), w, None))
    torch.cuda.synchronize()
    left_in_slots(c, kind, want[2], want[-1])


@pytest.mark.parametrize("kind", KINDS)
def test_state_after_parts_and_tokens(hip, kind):
    """A prompt in parts of several lengths, some by the single-token call:
    what its slot holds at the end is the whole's."""
    n = 175
    c = make(kind, [n], seed=6)
    want = c.want()
    d = c.descriptor()
    d.seq_start, d.n_seqs = None, 1
    fields = ["x", "y"] + ([] if kind == "conv" else ["z", "B", "C", "dt"])
    base = {f: getattr(d, f) for f in fields}
    f_prompt = hip.bm_hip_conv_dev if kind == "conv" else hip.bm_hip_ssm_dev
    f_step = hip.bm_hip_conv_step_dev if kind == "conv" else hip.bm_hip_ssm_step_dev
    d.n_tokens = n
    work = None if kind == "conv" else c.workspace(hip, d)  # the whole's, for all parts
    torch.cuda.synchronize()
    row = 0
    for take in (2, 1, 0, 40, 1, 130, 1):
        for f in fields:
            setattr(d, f, base[f] + row * getattr(d, f + "_stride") * 4)
        d.n_tokens = take
        rc = (f_step(C.byref(d), None) if take == 1 else f_prompt(C.byref(d), None)
              if kind == "conv" else f_prompt(C.byref(d), work, None))
        assert rc == 0, bh.last_error()
        row += take
    assert row == n
    torch.cuda.synchronize()
    left_in_slots(c, kind, want[2], want[-1])
    shape = (130,) if kind == "conv" else (c.H, c.P)
    check_rows(c.ybuf, c.y, want[0], want[1], "f32", shape, "parts")


# ---------------------------------------------------------------------------
# slots
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("slots,layers,size,gap", [
    (3, 1, (9 << 20) + 16 * 77, 0), (3, 24, (1 << 20) + 16, 32), (2, 1, (34 << 20) + 16 * 3, 0),
    (3, 2, (1 << 20) + 4 * 5, 4), (3, 1, (1 << 19) + 1, 0), (2, 1, (1 << 21) + 3, 1)])
def test_copy_of_few_pairs_of_large_slots(hip, slots, layers, size, gap):
    """One or two pairs with more columns to a block than it has threads."""
    for src, dst in (([0], [1]), ([0, 1], [1, 0]), ([-1, 0], [0, 1]), ([1, 1, 0], [0, 1, 1])):
        note("copy of %d x %d bytes, %s -> %s" % (layers, size, src, dst))
        copy(hip, [Pool(slots, layers, size, gap, 0, False, seed=layers)], src, dst)


@pytest.mark.parametrize("slots,live,layers,size", [(600, 300, 3, 5001), (2, 1, 1, 4 * (4096 * 1024 + 5)),
                                                    (64, 30, 24, 16 * 7000)])
def test_compact_of_more_moves_than_blocks(hip, slots, live, layers, size):
    """More than 4096 runs of 1024 words."""
    r = np.random.default_rng(slots)
    table = [int(v) for v in slots - 1 - r.permutation(slots - live)[:live]]  # most have to move
    p = Pool(slots, layers, size, 0, 0, False, 7)
    new, moves, n = compacted(table, slots)
    want = p.moved(list(moves.keys()), list(moves.values()))
    t = gpu(np.array(table), torch.int32)
    work = torch.full((hip.bm_hip_slots_compact_workspace_bytes(slots),), 0xFF, dtype=torch.uint8,
                      device="cuda")
    note("compact of %d slots of %d x %d bytes, %d moves" % (slots, layers, size, len(moves)))
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_compact_dev(C.byref(p.descriptor()), 1, at(t), at(t), len(table), None,
                                          at(work), None))
    torch.cuda.synchronize()
    assert t.tolist() == new
    assert np.array_equal(p.buf.cpu().numpy(), want)
