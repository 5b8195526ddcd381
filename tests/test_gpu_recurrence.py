"""The batched convolution and selective scan (bm_hip_conv_dev,
bm_hip_conv_step_dev, bm_hip_ssm_dev, bm_hip_ssm_step_dev) against the same
in 64 bits, with the bounds of tests/recurrence.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import (MARK, ConvCase, SsmCase, at, check_rows, close, conv_ref, f64, gpu, silu,
                        softplus)

pytestmark = pytest.mark.gpu
ALL = ["f32", "bf16", "f16"]


def note(msg):
    print("[case] " + msg, flush=True)


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type_name", ALL)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [1, 7, 64, 1030])
def test_conv_prompts(hip, type_name, width, channels):
    """Lengths around the unit of 32 rows and shorter than the window, rows
    before the first and behind the last sequence, odd strides."""
    for lens, pads in (([0, 1, 2, 3, 31, 32, 33, 64, 65, 5], dict(front=3, tail=2)),
                       ([100], dict(lead=3, row_pad=2)), ([1, 1, 1], dict(lead=8, slot_pad=5))):
        c = ConvCase(type_name, channels, width, lens, act=channels != 7, bias=width != 3,
                     seed=channels + width, **pads)
        note("conv %s width=%d channels=%d lens=%s" % (type_name, width, channels, lens))
        c.check(hip, "conv")


@pytest.mark.parametrize("type_name", ALL)
@pytest.mark.parametrize("channels", [1, 9, 512, 2056])
def test_conv_tokens(hip, type_name, channels):
    for n, width in ((1, 4), (5, 2), (70, 3)):
        note("conv_step %s channels=%d n=%d" % (type_name, channels, n))
        ConvCase(type_name, channels, width, [1] * n, step=True, seed=n, lead=channels % 3,
                 slot_pad=channels % 5).check(hip, "conv_step")


def test_conv_token_over_its_input(hip):
    c = ConvCase("f32", 300, 4, [1] * 6, step=True)
    rows, tols, pool = c.want()
    d = c.descriptor()
    d.y, d.y_stride = d.x, d.x_stride
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_conv_step_dev(C.byref(d), None))
    torch.cuda.synchronize()
    check_rows(c.buf, c.x, rows, tols, "f32", (300,), "in place")
    assert np.array_equal(c.pool(), pool)


# ---------------------------------------------------------------------------
# what both have in common: slots, padding, fresh sequences, bad row starts
# ---------------------------------------------------------------------------
def make(kind, lens, step=False, **k):
    if kind == "conv":
        return ConvCase("f32", 130, 4, lens, step=step, **k)
    H, P, G, N = {"scan1": (6, 10, 6, 1), "scan5": (4, 10, 2, 5), "scan24": (4, 40, 2, 24)}[kind]
    return SsmCase("f32", H, P, G, N, lens, step=step, **k)


KINDS = ["conv", "scan1", "scan5", "scan24"]


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_padding_and_repeated_slots(hip, kind, step):
    """Entries outside the pool and repeated ones: rows and slots untouched;
    the first that names a slot has it, also 64 and more entries earlier."""
    for slots in ([2, -1, 0, 9, 2, 1, 0, 1 << 30, -(1 << 31)], [-1] * 4, [3],
                  [5] + [-7] * 70 + [5, 4, 4]):
        lens = [1] * len(slots) if step else [3 + i % 5 for i in range(len(slots))]
        c = make(kind, lens, step, slots=slots, seed=len(slots), spare=9 - len(slots)
                 if len(slots) < 9 else 0)
        note("%s step=%s slots=%s" % (kind, step, slots[:10]))
        c.check(hip, "padding")


@pytest.mark.parametrize("kind", KINDS)
def test_slots_in_order_and_no_pool(hip, kind):
    make(kind, [4, 40, 0, 7], slots=None, spare=0).check(hip, "slot b")
    make(kind, [4, 40, 0, 7], slots=[1, 1, 2, 0], pool=False).check(hip, "no pool")
    make(kind, [1, 1, 1], True, slots=None, spare=1).check(hip, "step, slot b")
    make(kind, [1, 1, 1], True, pool=False).check(hip, "step, no pool")


@pytest.mark.parametrize("kind", KINDS)
def test_fresh(hip, kind):
    """Fresh sequences start from zeros, an empty one's slot becomes zero."""
    c = make(kind, [5, 0, 0, 2, 70], seed=3)
    c.fresh = [1, 1, 0, 0, 1]
    c.check(hip, "fresh")


@pytest.mark.parametrize("kind", KINDS)
def test_one_sequence_without_starts(hip, kind):
    c = make(kind, [150], seed=4)
    d = c.descriptor()
    rows, tols, pool = c.want()[:3]
    d.seq_start = None
    w = c.workspace(hip, d) if kind != "conv" else None
    torch.cuda.synchronize()
    if kind == "conv":
        bh.check(hip.bm_hip_conv_dev(C.byref(d), None))
    else:
        bh.check(hip.bm_hip_ssm_dev(C.byref(d), w, None))
    torch.cuda.synchronize()
    shape = (130,) if kind == "conv" else (c.H, c.P)
    check_rows(c.ybuf, c.y, rows, tols, "f32", shape, "one sequence")


@pytest.mark.parametrize("kind", KINDS)
def test_row_starts_out_of_range(hip, kind):
    """Starts below 0, above n_tokens and descending are clamped: nothing
    outside the rows is read or written, and no slot that is not named."""
    for starts in ([-5, 10, 20, 1 << 30], [0, 30, 10, 20], [1 << 30, 3, 3, -1]):
        c = make(kind, [10, 10, 10], seed=5)
        c.starts = starts
        rest = [k for k in range(c.n_slots) if k not in c.slots]
        before = c.pool_buf.clone()
        note("%s starts=%s" % (kind, starts))
        c.run(hip)
        assert torch.equal(before[rest], c.pool_buf[rest])
        if starts[0] == -5:  # still ascending: ordinary rows
            c = make(kind, [10, 10, 10], seed=5)
            c.starts = starts
            c.check(hip, "clamped")


@pytest.mark.parametrize("kind", KINDS)
def test_split_prompt_is_the_whole(hip, kind):
    """A prompt in one call, in two, and token by token: the same results
    within their bounds, the state carried by the slot."""
    n = 75
    whole, parts = make(kind, [n], seed=6), make(kind, [n], seed=6)
    rows, tols, pool = whole.want()[:3]
    whole.check(hip, "whole")
    d = parts.descriptor()
    d.seq_start, d.n_seqs = None, 1
    es = 4
    f_prompt = hip.bm_hip_conv_dev if kind == "conv" else hip.bm_hip_ssm_dev
    f_step = hip.bm_hip_conv_step_dev if kind == "conv" else hip.bm_hip_ssm_step_dev
    fields = ["x", "y"] if kind == "conv" else ["x", "y", "z", "B", "C", "dt"]
    base = {f: getattr(d, f) for f in fields}
    torch.cuda.synchronize()
    at_row, work = 0, []
    for take in (40, 1, 0, 30, 1, 1, 1, 1):
        for f in fields:
            stride = getattr(d, f + "_stride")
            setattr(d, f, base[f] + at_row * stride * es)
        d.n_tokens = take
        if take == 1:
            bh.check(f_step(C.byref(d), None))
        elif kind == "conv":
            bh.check(f_prompt(C.byref(d), None))
        else:
            work.append(parts.workspace(hip, d))
            torch.cuda.synchronize()
            bh.check(f_prompt(C.byref(d), work[-1], None))
        at_row += take
    assert at_row == n
    torch.cuda.synchronize()
    shape = (130,) if kind == "conv" else (parts.H, parts.P)
    check_rows(parts.ybuf, parts.y, rows, tols, "f32", shape, "parts")


# ---------------------------------------------------------------------------
# scan
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type_name", ALL)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8])
def test_scan_few_values(hip, type_name, N):
    for H, P, G in ((3, 64, 3), (8, 5, 2), (1, 1, 1), (2, 300, 1)):
        note("scan %s H=%d P=%d G=%d N=%d" % (type_name, H, P, G, N))
        SsmCase(type_name, H, P, G, N, [0, 1, 2, 31, 33, 64, 100, 17], seed=N, front=2, tail=1,
                lead=P % 4, gate=N != 3, skip=N != 4, bias=N != 5).check(hip, "scan")


@pytest.mark.parametrize("type_name", ALL)
@pytest.mark.parametrize("N", [9, 16, 20, 31, 32, 33, 64, 100, 128, 129, 256])
def test_scan_many_values(hip, type_name, N):
    for H, P, G in ((4, 64, 1), (6, 7, 3), (1, 33, 1), (2, 130, 2)):
        note("scan %s H=%d P=%d G=%d N=%d" % (type_name, H, P, G, N))
        SsmCase(type_name, H, P, G, N, [1, 0, 31, 32, 33, 65, 20], seed=N + P, front=1, tail=3,
                lead=N % 4, gate=N != 16, skip=N != 20, bias=N != 33).check(hip, "scan")


@pytest.mark.parametrize("type_name", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 6, 16, 128])
@pytest.mark.parametrize("lens", [[1500], [700, 3, 1100]])
def test_scan_long(hip, type_name, N, lens):
    """Sequences long enough to be worked on in parts."""
    note("scan %s N=%d lens=%s" % (type_name, N, lens))
    SsmCase(type_name, 2, 32, 2 if N == 1 else 1, N, lens, seed=N).check(hip, "long")


@pytest.mark.parametrize("N", [1, 24])
def test_scan_long_sequences_among_many_short_ones(hip, N):
    """More sequences than rows make units: the long ones' parts keep apart."""
    r = np.random.default_rng(12)
    lens = [int(v) for v in r.integers(0, 4, 150)]
    for at_ in (0, 40, 41, 120, 149):
        lens[at_] = int(r.integers(520, 700))
    SsmCase("f32", 2, 32, 2 if N == 1 else 1, N, lens, seed=N, front=1).check(hip, "many")


@pytest.mark.parametrize("N", [1, 24])
def test_scan_steps_given(hip, N):
    """Without softplus, and without bias: dt is the step itself."""
    for bias in (True, False):
        SsmCase("f32", 2, 20, 2, N, [50, 3], soft=False, bias=bias, rate=16.0).check(hip, "steps")


@pytest.mark.parametrize("N", [1, 24])
def test_scan_decays_that_vanish(hip, N):
    """Steps so large that a state is forgotten within a token, and so small
    that none is: softplus at both ends."""
    c = SsmCase("f32", 4, 12, 4, N, [90, 40], seed=8, bias=False)
    c.dt[:, 0] = 50.0
    c.dt[:, 1] = -60.0
    c.dt[::3, 2] = 25.0
    c.A[0] = -16.0
    c.check(hip, "decays")


def run_y(c, hip):
    c.run(hip)
    return f64(c.y).copy(), c.pool().copy()


@pytest.mark.parametrize("what", ["x", "B", "Cm", "dt", "z"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("N", [1, 5, 24, 128])
def test_scan_later_tokens_do_not_reach_earlier_ones(hip, N, what, value):
    """Infinities and NaN from one token on: earlier rows and other sequences
    are bit for bit what they were."""
    H, P = 2, 40
    G = H if N == 1 else 1
    lens = [37, 90, 20]
    clean = SsmCase("f32", H, P, G, N, lens, seed=9)
    y0, p0 = run_y(clean, hip)
    for row in (37 + 13, 37 + 50):
        c = SsmCase("f32", H, P, G, N, lens, seed=9)
        t = getattr(c, what)
        t[row] = value
        if what in ("dt", "z", "x"):
            t[row, -1] = 0.25
        note("scan N=%d %s=%r from row %d" % (N, what, value, row))
        y1, p1 = run_y(c, hip)
        keep = [r for r in range(sum(lens)) if r < row or r >= 37 + 90]
        assert np.array_equal(y0[keep], y1[keep])
        for b in (0, 2):
            assert np.array_equal(p0[c.slots[b]], p1[c.slots[b]])
        if what == "z":
            assert np.array_equal(p0, p1)
        if np.isnan(value):
            assert np.isnan(y1[row]).any()


@pytest.mark.parametrize("N", [1, 24])
def test_scan_infinite_values_come_through(hip, N):
    """A single infinite x makes its channel infinite or NaN from its row on,
    and leaves the others as they are."""
    c = SsmCase("f32", 1, 40, 1, N, [70], seed=10, gate=False, skip=False)
    rows, tols, pool, stol = c.want()
    c.x[20, 7] = float("inf")
    c.run(hip)
    y = f64(c.y)
    assert not np.isfinite(y[20:, 7]).any()
    for t in range(70):
        k = [p for p in range(40) if p != 7 or t < 20]
        close(y[t][k], rows[t].reshape(-1)[k], tols[t].reshape(-1)[k], "f32", "row %d" % t)


def test_scan_overflow_of_a_growing_state(hip):
    """A > 0: the state grows past fp32 and becomes infinite, not wrong."""
    for N in (1, 24):
        c = SsmCase("f32", 2, 8, 2, N, [200], seed=11, gate=False, skip=False, bias=False)
        c.A[:] = 3.0
        c.A[1] = -1.0
        c.dt[:] = 1.0
        c.run(hip)
        y, p = f64(c.y), c.pool()[c.slots[0]]
        assert not np.isfinite(y[-1, :8]).any() and np.isfinite(y[:, 8:]).all()
        assert not np.isfinite(p[0]).any() and np.isfinite(p[1]).all()


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type_name", ALL)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 7, 8, 16, 17, 32, 40, 64, 96, 128, 200, 256, 255])
def test_scan_tokens(hip, type_name, N):
    for H, P, G, n in ((3, 64, 3, 1), (8, 5, 2, 4), (2, 130, 1, 66)):
        for slot_pad in (0, 1):
            note("step %s H=%d P=%d G=%d N=%d n=%d" % (type_name, H, P, G, N, n))
            SsmCase(type_name, H, P, G, N, [1] * n, step=True, seed=N, lead=N % 3,
                    slot_pad=slot_pad, gate=N != 3, skip=N != 4, bias=N != 7).check(hip, "step")


def test_scan_token_over_its_input(hip):
    for what in ("x", "z"):
        c = SsmCase("f32", 3, 70, 1, 12, [1] * 5, step=True)
        rows, tols = c.want()[:2]
        d = c.descriptor()
        d.y, d.y_stride = getattr(d, what), d.x_stride
        torch.cuda.synchronize()
        rc = hip.bm_hip_ssm_step_dev(C.byref(d), None)
        if what == "z":
            assert rc == -2 and "overlaps z" in bh.last_error()
            continue
        torch.cuda.synchronize()
        for t in rows:
            close(f64(c.x)[t].reshape(3, 70), rows[t], tols[t], "f32", "in place")


def test_offsets_past_32_bits(hip):
    """The last slot of a pool of more than 2^32 floats, rows of a buffer of
    more than 2^32 values: prompts and single tokens."""
    H, P, N, far = 2, 16, 16, 3
    stride = (1 << 31) + 64
    pool = torch.empty(far * stride, dtype=torch.float32, device="cuda")
    xs, n = (1 << 24) - 16, 270
    rows = torch.empty(n * xs + 64, dtype=torch.float32, device="cuda")
    for step in (False, True):
        c = SsmCase("f32", H, P, 1, N, [1] * n if step else [n], step=step, slots=None, spare=0)
        c.slots = [-1] * (n - 1) + [2] if step else [2]
        c.n_slots = 3
        state = torch.randn(H * P * N, device="cuda")
        pool[2 * stride:2 * stride + H * P * N] = state
        c.pool_buf = torch.zeros((3, H * P * N), device="cuda")
        c.pool_buf[2] = state
        want, tols, new, stol = c.want()
        d = c.descriptor()
        d.state, d.state_stride = at(pool), stride
        wide = rows[:n * xs].view(n, xs)
        wide[:, :H * P] = c.x
        d.x, d.x_stride = at(rows), xs
        d.y, d.y_stride = at(rows) + 4 * H * P, xs
        w = None if step else c.workspace(hip, d)
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_ssm_step_dev(C.byref(d), None) if step
                 else hip.bm_hip_ssm_dev(C.byref(d), w, None))
        torch.cuda.synchronize()
        got = f64(wide[:, H * P:2 * H * P])
        for t in want:
            close(got[t].reshape(H, P), want[t], tols[t], "f32", "row %d" % t)
        close(f64(pool[2 * stride:2 * stride + H * P * N]).reshape(H, P, N), new[2], stol[2],
              "f32", "state")


def test_more_rows_than_a_grid_row_of_units(hip):
    """2^28 + 21 rows of one channel: more units than a launch has blocks of
    256 threads along x.  Two taps of 1 on integers: every sum is exact."""
    n = (1 << 28) + 21
    x = (torch.arange(n, device="cuda", dtype=torch.int32) % 101).to(torch.bfloat16)
    y = torch.full((n + 8,), -1.0, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(2, device="cuda")
    d = bh.Conv(type=bh.BF16, channels=1, width=2, silu=0, n_seqs=1, n_tokens=n, x=at(x),
                x_stride=1, w=at(w), y=at(y), y_stride=1)
    note("conv of %d rows" % n)
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_conv_dev(C.byref(d), None))
    torch.cuda.synchronize()
    assert y[0] == x[0] and torch.equal(y[1:n], x[1:] + x[:-1])
    assert (y[n:] == -1).all()


def test_join_of_more_blocks_than_a_grid_row(hip):
    """Many prompts, one of which is cut, with states of 512 blocks each: the
    join's grid is longer than a launch along x."""
    H, P, N, n = 64, 64, 128, 40000
    lens = [1] * (n - 1) + [3000]
    r = torch.Generator().manual_seed(3)
    T = sum(lens)
    x = torch.randn((T, H * P), generator=r).cuda().to(torch.bfloat16)
    BC = torch.randn((T, 2 * N), generator=r).cuda().to(torch.bfloat16)
    dt = torch.randn((T, H), generator=r).cuda().to(torch.bfloat16)
    A = -torch.rand(H, generator=r).cuda() - 0.1
    starts = gpu(np.concatenate([[0], np.cumsum(lens)]), torch.int32)

    def run(first, count, start, y):
        o = lambda t: at(t) + first * t.shape[1] * 2
        d = bh.Ssm(type=bh.BF16, n_heads=H, head_dim=P, n_groups=1, d_state=N, dt_softplus=1,
                   n_seqs=n if start is not None else 1, n_tokens=count, seq_start=at(start),
                   x=o(x), x_stride=H * P, B=o(BC), B_stride=2 * N, C=o(BC) + 2 * N,
                   C_stride=2 * N, dt=o(dt), dt_stride=H, A=at(A), y=at(y), y_stride=H * P)
        size = hip.bm_hip_ssm_workspace_bytes(C.byref(d))
        work = torch.empty(size + 256, dtype=torch.uint8, device="cuda")
        base = (work.data_ptr() + 255) // 256 * 256
        note("scan of %d rows, workspace %d MB" % (count, size >> 20))
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_ssm_dev(C.byref(d), C.c_void_p(base) if size else None, None))
        torch.cuda.synchronize()

    y = torch.zeros((T, H * P), dtype=torch.bfloat16, device="cuda")
    run(0, T, starts, y)
    # 3000 rows in units of 1344: three units to join
    # the cut prompt by itself: the same sums in another cut, each y within a
    # few roundings of the largest term; both are rounded to bf16
    alone = torch.zeros((3000, H * P), dtype=torch.bfloat16, device="cuda")
    run(n - 1, 3000, None, alone)
    a, b = y[n - 1:].float(), alone.float()
    scale = b.abs().amax(0, keepdim=True)
    assert ((a - b).abs() <= 2 * 2.0 ** -8 * b.abs() + 2.0 ** -8 * scale).all()
    # a prompt of one token: y = (C . B) softplus(dt) x, three factors in bf16
    k = 17
    want = ((BC[k, N:].double() @ BC[k, :N].double()) * torch.nn.functional.softplus(dt[k].double())
            ).repeat_interleave(P) * x[k].double()
    size = ((BC[k, N:].double().abs() @ BC[k, :N].double().abs())
            * torch.nn.functional.softplus(dt[k].double())).repeat_interleave(P) * x[k].double().abs()
    # the matrix operand M = C.B d has two bf16 pieces (2^-17 of it), sums of
    # 128 fp32 products (2^-17 of the absolute sum), one rounding to bf16
    assert ((y[k].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * size).all()


@pytest.mark.parametrize("kind", KINDS)
def test_repeated_slots_far_apart(hip, kind):
    """Repeats at every distance that the search for them treats apart: below
    64 entries, above, and past eight times 64."""
    n = 1300
    c = make(kind, [1] * n, step=True, seed=6)
    for first, again in ((0, 63), (1, 64), (2, 65), (70, 575), (71, 576), (64, 577), (130, 1299),
                         (1150, 1151), (640, 1200), (3, 1298)):
        c.slots[again] = c.slots[first]
    c.slots[5] = c.slots[900] = -1
    note("%s, %d slots with repeats" % (kind, n))
    c.check(hip, "repeats")
