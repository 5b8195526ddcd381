"""The gated delta rule against the rule in 64 bits, with the bounds of
tests/delta.py: prompts of ragged lengths, single tokens, drafted tokens."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from delta import EPS, DeltaCase, rule
from native import bh
from recurrence import MARK, at, check_rows, close, f64, gpu, sequences
from test_zz_no_alloc import _hip_runtime, _ok

pytestmark = pytest.mark.gpu


def note(msg):
    print("[case] " + msg, flush=True)


LENS = [70, 0, 1, 200, 33, 64, 32, 65, 128, 129]


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,P,G,N", [(4, 16, 2, 64), (3, 40, 3, 128), (2, 17, 1, 100), (1, 5, 1, 7),
                                     (4, 1, 4, 1), (2, 33, 2, 256), (2, 64, 1, 129), (2, 130, 2, 16),
                                     (1, 16, 1, 65), (2, 8, 2, 36), (1, 3, 1, 4), (1, 20, 1, 31)])
def test_prompts(hip, type_name, H, P, G, N):
    note("prompts %s %s" % (type_name, (H, P, G, N)))
    DeltaCase(type_name, H, P, G, N, LENS, seed=H + P + N).check(hip, "prompts")


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,P,G,N", [(4, 16, 2, 64), (3, 40, 3, 128), (2, 17, 1, 100), (1, 5, 1, 7),
                                     (4, 1, 4, 1), (2, 33, 2, 256), (2, 64, 1, 129), (2, 130, 2, 16),
                                     (2, 8, 2, 36), (1, 3, 1, 4), (1, 20, 1, 31), (2, 6, 1, 2)])
def test_single_tokens(hip, type_name, H, P, G, N):
    note("tokens %s %s" % (type_name, (H, P, G, N)))
    DeltaCase(type_name, H, P, G, N, [1] * 5, seed=H + P + N, step=True).check(hip, "tokens")


@pytest.mark.parametrize("lead,pad", [(1, 0), (0, 1), (3, 2), (2, 6), (8, 8), (4, 4)])
@pytest.mark.parametrize("type_name", ["f32", "bf16"])
def test_rows_on_any_alignment(hip, type_name, lead, pad):
    note("alignment %s %d %d" % (type_name, lead, pad))
    kw = dict(lead=lead, row_pad=pad, slot_pad=5, seed=lead + pad)
    DeltaCase(type_name, 2, 24, 1, 64, [100, 7], front=3, tail=2, **kw).check(hip, "prompts")
    DeltaCase(type_name, 2, 24, 1, 64, [1] * 3, step=True, **kw).check(hip, "tokens")


OPTIONS = [dict(gate=False), dict(decay=False), dict(bias=False), dict(soft=False),
           dict(beta="raw"), dict(beta=None), dict(norm=False), dict(pool=False), dict(frozen=True),
           dict(scale=-2.5), dict(eps=0.5), dict(rate=400.0),
           dict(norm=False, decay=False, beta=None, gate=False)]


@pytest.mark.parametrize("k", range(len(OPTIONS)))
@pytest.mark.parametrize("N", [12, 80])
def test_options(hip, k, N):
    note("options %s N=%d" % (OPTIONS[k], N))
    DeltaCase("f32", 4, 20, 2, N, [150, 9, 64], seed=k, **OPTIONS[k]).check(hip, "prompts")
    DeltaCase("bf16", 4, 20, 2, N, [150, 9, 64], seed=k, **OPTIONS[k]).check(hip, "prompts")
    DeltaCase("f16", 4, 20, 2, N, [1] * 4, seed=k, step=True, **OPTIONS[k]).check(hip, "tokens")


@pytest.mark.parametrize("step", [False, True])
def test_padding_and_fresh_sequences(hip, step):
    """Slots outside the pool and repeated ones are padding; fresh sequences
    start from zeros (single tokens do not read the flags)."""
    note("padding step=%s" % step)
    lens = [1] * 7 if step else [40, 70, 3, 0, 90, 35, 0]
    c = DeltaCase("f32", 2, 20, 1, 40, lens, slots=[3, -1, 5, 0, 3, 9, 99], spare=2, seed=4, step=step)
    c.fresh = [0, 0, 1, 0, 0, 0, 0]
    c.check(hip, "padding")
    if not step:
        c = DeltaCase("f32", 2, 20, 1, 40, lens, seed=5)
        c.fresh = [1, 0, 1, 1, 0, 1, 0]
        c.check(hip, "fresh")


def test_calls_without_rows(hip):
    """A fresh sequence's slot becomes zero, the others stay; frozen ones too."""
    for frozen in (False, True):
        note("no rows, frozen=%s" % frozen)
        c = DeltaCase("f32", 4, 40, 2, 24, [0] * 3, seed=1, frozen=frozen)
        c.fresh = [0, 1, 0]
        d = c.descriptor()
        for f in ("q", "k", "v", "dt", "beta", "z", "y"):
            setattr(d, f, None)
        want = c.pool_buf.clone()
        if not frozen:
            want[c.slots[1]] = 0.0
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_delta_dev(C.byref(d), None, None))
        torch.cuda.synchronize()
        assert torch.equal(c.pool_buf, want)


@pytest.mark.parametrize("longs", [[], [33], [200, 40, 64]])
def test_many_sequences_of_which_few_are_long(hip, longs):
    note("many sequences, long %s" % longs)
    r = np.random.default_rng(len(longs))
    lens = [int(v) for v in r.integers(0, 3, 150)]
    for i, n in enumerate(longs):
        lens[11 + 40 * i] = n
    DeltaCase("bf16", 2, 18, 1, 48, lens, front=5, tail=3, seed=3).check(hip, "many")


@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N", [40, 45, 100, 131, 252])
def test_many_short_sequences(hip, type_name, N, frozen):
    """More tiles of the states than the chip holds waves at once."""
    note("short sequences %s N=%d frozen=%s" % (type_name, N, frozen))
    DeltaCase(type_name, 40, 50, 8, N, [5, 1, 0, 8, 9, 17, 32, 3, 24], frozen=frozen,
              seed=N).check(hip, "short")


def test_a_sequence_alone_needs_no_starts(hip):
    for n in (1, 32, 33, 300):
        note("one sequence of %d" % n)
        c = DeltaCase("f32", 2, 20, 1, 40, [n], seed=n)
        rows, tols, pool, stol = c.want()
        d = c.descriptor()
        d.seq_start = None
        w = c.workspace(hip, d)
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_delta_dev(C.byref(d), w, None))
        torch.cuda.synchronize()
        check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "alone")
        k = c.slots[0]
        close(c.pool()[k], pool[k], stol[k], "f32", "state")


@pytest.mark.parametrize("type_name", ["f32", "bf16"])
def test_tokens_over_v(hip, type_name):
    note("y over v " + type_name)
    c = DeltaCase(type_name, 4, 24, 2, 40, [1] * 3, step=True, lead=1, row_pad=3, seed=8)
    rows, tols, _, _ = c.want()
    d = c.descriptor()
    d.y, d.y_stride = d.v, d.v_stride
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_delta_step_dev(C.byref(d), None))
    torch.cuda.synchronize()
    for t, want in rows.items():
        close(f64(c.v)[t].reshape(4, 24), want, tols[t], type_name, "row %d" % t)


def test_a_workspace_of_a_larger_call(hip):
    """Right in it, and nothing behind a call's own size is written."""
    big = DeltaCase("f32", 2, 40, 1, 72, [700, 90, 300], seed=1)
    n = hip.bm_hip_delta_workspace_bytes(C.byref(big.descriptor()))
    for lens in ([700, 90, 300], [65], [33] * 3, [1, 500]):
        note("shared workspace %s" % lens)
        c = DeltaCase("f32", 2, 40, 1, 72, lens, seed=2)
        rows, tols, pool, stol = c.want()
        d = c.descriptor()
        own = hip.bm_hip_delta_workspace_bytes(C.byref(d))
        assert own <= n
        work = torch.full((own + (1 << 20),), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_delta_dev(C.byref(d), at(work), None))
        torch.cuda.synchronize()
        assert (work[own:] == 0xFF).all()
        check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 40), "shared")


# ---------------------------------------------------------------------------
# sizes of values.  Each p has its own: the rule is linear in v and S, so
# powers of two come through whole.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("step", [False, True])
def test_values_of_any_size(hip, step):
    """v and S times powers of two from 2^-100 to 2^100, one per p: y and S
    come out times the same."""
    note("sizes step=%s" % step)
    lens = [1] * 3 if step else [130, 20, 70]
    make = lambda: DeltaCase("f32", 2, 24, 1, 64, lens, seed=6, step=step)
    c = make()
    p2 = torch.exp2(torch.linspace(-100, 100, 24, device="cuda").round()).repeat(2)
    c.v.mul_(p2)
    c.pool_buf.view(-1, 48, 64).mul_(p2[:, None])
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 24), "sizes")
    for k, want in stol.items():
        close(c.pool()[k], pool[k], want, "f32", "slot %d" % k)


@pytest.mark.parametrize("first", ["small", "large", "zero", "state"])
def test_sizes_that_change_within_a_sequence(hip, first):
    """Values 2^80 times smaller or larger from one chunk to another, or none
    at first: bounds go by the largest of each chunk."""
    note("changing sizes, %s first" % first)
    c = DeltaCase("f32", 2, 20, 1, 64, [260], seed=7, rate=0.5)
    f = torch.ones(260, device="cuda")
    if first == "small":
        f[:100] = 2.0 ** -80
    elif first == "large":
        f[100:] = 2.0 ** -80
    elif first == "zero":
        f[:150] = 0.0
        c.pool_buf.zero_()
    else:
        f[:] = 2.0 ** -60
    c.v.mul_(f[:, None])
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), first)
    k = c.slots[0]
    close(c.pool()[k], pool[k], stol[k], "f32", "state")


@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 16, 2.0 ** 20])
def test_rows_before_a_large_one_of_their_chunk(hip, size):
    """One v at the end of a chunk is `size` times the others.  The column's scale
    takes it to 2^10 .. 2^11, so that other operands are good to 2^-25 of that or
    size 2^-35.  As independent errors, w adds up 64 of them (8 times one) and y
    64 of w's: size 2^-29, besides the 2^-19 of fp32 sums and operands of 22 bits
    that kSpread allows."""
    note("rows before v = %g" % size)
    c = DeltaCase("f32", 2, 20, 1, 64, [128], seed=12, rate=0.5, gate=False)
    c.v[63, 7] = size
    c.v[127, 30] = -size
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "before")
    got = f64(c.y).reshape(128, 2, 20)
    for h, p, n in ((0, 7, 63), (1, 10, 127)):
        off = np.array([got[t, h, p] - rows[t][h, p] for t in range(n)])
        all_of_it = np.array([rows[t][h, p] for t in range(n)])
        rms = lambda v: np.sqrt((v * v).mean())
        assert rms(off) <= size * 2.0 ** -29 + rms(all_of_it) * 2.0 ** -19, (rms(off), rms(all_of_it))


@pytest.mark.parametrize("size", [-110, -60, -20, 0, 60])
@pytest.mark.parametrize("lens", [[130, 20], [64, 33, 5]])
def test_a_state_and_no_values(hip, lens, size):
    """v of zeros: all that is read is what the slots hold, however small."""
    note("no values, state 2^%d, %s" % (size, lens))
    c = DeltaCase("f32", 2, 20, 1, 64, lens, seed=11, rate=0.5)
    c.v.zero_()
    c.pool_buf.mul_(2.0 ** size)
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "no values")
    for k, want in stol.items():
        close(c.pool()[k], pool[k], want, "f32", "slot %d" % k)


@pytest.mark.parametrize("at_row", [0, 63, 64, 100, 129])
@pytest.mark.parametrize("what", ["v", "v max", "k", "q", "dt", "beta", "state"])
def test_infinities_and_nan_stay_where_they_belong(hip, what, at_row):
    """From its row on in its head or p; everything else as without it."""
    for value in ([3.0e38] if what == "v max" else [float("inf"), float("-inf"), float("nan")]):
        note("%s row %d %r" % (what, at_row, value))
        make = lambda: DeltaCase("f32", 2, 20, 2, 40, [130, 70], seed=9, bias=False, decay=True)
        c = make()
        rows, tols, pool, stol = c.want()
        h, p, n = 1, 7, 5
        if what.startswith("v"):
            c.v[at_row, h * 20 + p] = value
        elif what == "k":
            c.k[at_row, h * 40 + n] = value
        elif what == "q":
            c.q[at_row, h * 40 + n] = value
        elif what in ("dt", "beta"):
            value = float("nan")
            getattr(c, what)[at_row, h] = value
        else:
            c.pool_buf.view(-1, 2, 20, 40)[c.slots[0], h, p, n] = value
        if what == "v max":  # finite all the way in 64 bits; what passes fp32 is only not earlier
            rows, tols, pool, stol = c.want()
        c.run(hip)
        got, state = f64(c.y).reshape(-1, 2, 20), c.pool()[c.slots[0]]
        hit = np.zeros((200, 2, 20), bool)
        dead = np.zeros((2, 20), bool)
        if what in ("v", "state"):
            hit[(0 if what == "state" else at_row):130, h, p] = True
            dead[h, p] = True
        elif what == "q":
            hit[at_row, h] = True
        elif what != "v max":
            hit[at_row:130, h] = True
            dead[h] = True
        assert (~np.isfinite(got[hit])).all(), "%s: finite where it cannot be" % what
        assert (~np.isfinite(state[dead])).all()
        if what == "v max":
            hit[at_row:130, h, p] = True
            dead[h, p] = True
        for t in rows:
            keep = ~hit[t]
            close(got[t][keep], rows[t][keep], tols[t][keep], "f32", "%s row %d" % (what, t))
        close(state[~dead], pool[c.slots[0]][~dead], stol[c.slots[0]][~dead], "f32", "state")
        k = c.slots[1]
        close(c.pool()[k], pool[k], stol[k], "f32", "the other sequence's state")


@pytest.mark.parametrize("n", [20, 200])
def test_one_key_over_and_over(hip, n):
    """The same key in every row with b = 1: each row takes the row before's
    value back whole, and T is bidiagonal."""
    note("one key, %d rows" % n)
    c = DeltaCase("f32", 1, 20, 1, 64, [n], beta=None, decay=False, gate=False, seed=3)
    c.k.copy_(c.k[:1].expand_as(c.k))
    c.q.copy_(c.k)
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (1, 20), "one key")


def test_keys_of_zeros(hip):
    """Rows whose key is zero write nothing; a query of zeros reads nothing."""
    note("zero keys")
    for step, lens in ((False, [130, 5]), (True, [1, 1])):
        c = DeltaCase("bf16", 2, 20, 1, 40, lens, seed=3, step=step)
        c.k[::2] = 0.0
        c.q[::3] = 0.0
        c.check(hip, "zeros")


def test_drafts_are_scored_without_touching_the_state(hip):
    """Frozen sequences of a few rows: y as of a prompt, every slot as it was."""
    for lens in ([5] * 6, [1, 8, 40, 70]):
        note("drafts %s" % lens)
        c = DeltaCase("bf16", 4, 32, 2, 64, lens, frozen=True, seed=2)
        before = c.pool_buf.clone()
        c.check(hip, "drafts")
        assert torch.equal(before, c.pool_buf)


def test_slots_far_apart(hip):
    """Slots more than 2^32 bytes from each other."""
    note("far slots")
    for lens, step in (([70, 3], False), ([1, 1], True)):
        c = DeltaCase("f32", 1, 16, 1, 64, lens, slots=[2, 0], spare=1, seed=1, step=step)
        small = c.pool_buf
        stride = (1 << 30) + 64
        far = torch.empty(2 * stride + 1024, device="cuda")
        wide = torch.as_strided(far, (3, 1024), (stride, 1))
        wide.copy_(small)
        rows, tols, pool, stol = c.want()
        d = c.descriptor()
        d.state, d.state_stride = at(far), stride
        w = None if step else c.workspace(hip, d)
        torch.cuda.synchronize()
        bh.check(c.call(hip, d, w))
        torch.cuda.synchronize()
        check_rows(c.ybuf, c.y, rows, tols, "f32", (1, 16), "far")
        for k, tol in stol.items():
            close(f64(wide[k]).reshape(1, 16, 64), pool[k], tol, "f32", "slot %d" % k)
        assert torch.equal(wide[1], small[1])
        del far, wide


# ---------------------------------------------------------------------------
# as programs run it
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def rt():
    return _hip_runtime()


@pytest.fixture
def streams(rt):
    made = []
    for _ in range(2):
        s = C.c_void_p()
        _ok(rt.hipStreamCreateWithFlags(C.byref(s), 1), "hipStreamCreateWithFlags")
        made.append(s)
    yield made
    for s in made:
        rt.hipStreamDestroy(s)


@pytest.mark.parametrize("kind", ["prompts", "tokens", "drafts"])
def test_replays_equal_the_eager_calls(hip, rt, streams, kind):
    note("replays, " + kind)
    lens = {"prompts": [150, 3, 40], "tokens": [1] * 5, "drafts": [5, 2, 40]}[kind]
    c = DeltaCase("bf16", 4, 24, 2, 40, lens, step=kind == "tokens", frozen=kind == "drafts", seed=6)
    s = streams[0]
    d = c.descriptor()
    w = None if c.step else c.workspace(hip, d)
    start = c.pool_buf.clone()
    torch.cuda.synchronize()
    want = []
    for _ in range(4):
        assert c.call(hip, d, w, s.value) == 0, bh.last_error()
        _ok(rt.hipStreamSynchronize(s), "sync")
        want.append((c.y.clone(), c.pool_buf.clone()))
    c.pool_buf.copy_(start)
    torch.cuda.synchronize()
    graph, exe = C.c_void_p(), C.c_void_p()
    _ok(rt.hipStreamBeginCapture(s, 1), "hipStreamBeginCapture")
    rc = c.call(hip, d, w, s.value)
    _ok(rt.hipStreamEndCapture(s, C.byref(graph)), "hipStreamEndCapture")
    assert rc == 0, bh.last_error()
    _ok(rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0), "instantiate")
    try:
        for i in range(4):
            if c.work is not None:
                c.work.fill_(0xFF)
            c.y.fill_(3.0)
            torch.cuda.synchronize()
            _ok(rt.hipGraphLaunch(exe, s), "hipGraphLaunch")
            _ok(rt.hipStreamSynchronize(s), "sync")
            assert torch.equal(c.y, want[i][0]), "replay %d" % i
            assert torch.equal(c.pool_buf, want[i][1]), "replay %d: state" % i
            (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
    finally:
        rt.hipGraphExecDestroy(exe)
        rt.hipGraphDestroy(graph)


def test_two_calls_at_once(hip, rt, streams):
    """On two streams, with workspaces and slots of their own."""
    note("two streams")
    cs = [DeltaCase("bf16", 4, 40, 2, 64, [600, 30], seed=k) for k in range(2)]
    wants = [c.want() for c in cs]
    ds = [c.descriptor() for c in cs]
    ws = [c.workspace(hip, d) for c, d in zip(cs, ds)]
    torch.cuda.synchronize()
    for c, d, w, s in zip(cs, ds, ws, streams):
        assert c.call(hip, d, w, s.value) == 0, bh.last_error()
    torch.cuda.synchronize()
    for c, (rows, tols, pool, stol) in zip(cs, wants):
        check_rows(c.ybuf, c.y, rows, tols, "bf16", (4, 40), "two streams")
        for k, tol in stol.items():
            close(c.pool()[k], pool[k], tol, "f32", "slot %d" % k)


def test_the_same_twice_is_the_same(hip):
    note("repeatable")
    out = []
    for _ in range(2):
        c = DeltaCase("f32", 4, 40, 2, 72, [300, 20, 90], seed=5)
        c.run(hip)
        out.append((c.y.clone(), c.pool_buf.clone()))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_prompts_then_tokens(hip):
    """A prompt cut anywhere, its rest as single tokens: the states join."""
    note("prompt, then tokens")
    whole = DeltaCase("f32", 2, 24, 1, 40, [100], seed=11)
    rows, tols, pool, stol = whole.want()
    d = whole.descriptor()
    w = whole.workspace(hip, d)
    cut = 90
    d.n_tokens, d.seq_start = cut, None
    bh.check(hip.bm_hip_delta_dev(C.byref(d), w, None))
    d.n_seqs = 1
    size = whole.buf.element_size()
    for t in range(cut, 100):
        for f, stride in (("q", "q_stride"), ("k", "k_stride"), ("v", "v_stride"), ("dt", "dt_stride"),
                          ("beta", "beta_stride"), ("z", "z_stride"), ("y", "y_stride")):
            setattr(d, f, at(getattr(whole, f)) + t * getattr(d, stride) * size)
        bh.check(hip.bm_hip_delta_step_dev(C.byref(d), None))
    torch.cuda.synchronize()
    check_rows(whole.ybuf, whole.y, rows, tols, "f32", (2, 24), "joined")
    k = whole.slots[0]
    close(whole.pool()[k], pool[k], stol[k], "f32", "state")
