"""The batched recurrence as programs run it: captured and replayed, on other
streams than the library's, two calls at once, and all of it in a row between
two BitLinear products."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import ConvCase, SsmCase, at, check_rows, close, conv_ref, f64, gpu, half_step, ssm_ref
from test_zz_no_alloc import _hip_runtime, _ok

pytestmark = pytest.mark.gpu


def note(msg):
    print("[case] " + msg, flush=True)


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


def calls(hip, c, d, work):
    """The call of a case on a stream."""
    if isinstance(c, ConvCase):
        f = hip.bm_hip_conv_step_dev if c.step else hip.bm_hip_conv_dev
        return lambda s: f(C.byref(d), s)
    if c.step:
        return lambda s: hip.bm_hip_ssm_step_dev(C.byref(d), s)
    return lambda s: hip.bm_hip_ssm_dev(C.byref(d), work, s)


def cases():
    lens = [70, 0, 1, 200]
    return [("conv", ConvCase("f32", 130, 4, lens, seed=1)),
            ("conv_step", ConvCase("bf16", 64, 3, [1] * 5, step=True, seed=2)),
            ("scan, 1 value", SsmCase("f32", 6, 10, 6, 1, lens, seed=3)),
            ("scan, 24 values", SsmCase("f32", 4, 40, 2, 24, [300, 3, 150], seed=4)),
            ("scan, 128 values", SsmCase("bf16", 2, 64, 1, 128, [290], seed=5)),
            ("token, 24 values", SsmCase("f32", 4, 40, 2, 24, [1] * 7, step=True, seed=6))]


@pytest.mark.parametrize("k", range(6))
def test_replays_equal_the_eager_calls(hip, rt, streams, k):
    """Captured once, replayed with eager calls on other slots in between:
    each replay carries the state on as an eager call does, bit for bit, and
    reads the slots and row starts that are there then."""
    name, c = cases()[k]
    note(name)
    s = streams[0]
    d = c.descriptor()
    work = c.workspace(hip, d) if isinstance(c, SsmCase) and not c.step else None
    call = calls(hip, c, d, work)
    start = c.pool_buf.clone()
    torch.cuda.synchronize()
    want = []
    for _ in range(4):  # eager
        assert call(s.value) == 0, bh.last_error()
        _ok(rt.hipStreamSynchronize(s), "sync")
        want.append((c.y.clone(), c.pool_buf.clone()))
    c.pool_buf.copy_(start)
    torch.cuda.synchronize()
    graph, exe = C.c_void_p(), C.c_void_p()
    _ok(rt.hipStreamBeginCapture(s, 1), "hipStreamBeginCapture")
    rc = call(s.value)
    _ok(rt.hipStreamEndCapture(s, C.byref(graph)), "hipStreamEndCapture")
    assert rc == 0, bh.last_error()
    _ok(rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0), "instantiate")
    try:
        for i in range(3):
            if work is not None:
                c.work.fill_(0xFF)
            c.y.fill_(3.0)
            torch.cuda.synchronize()
            _ok(rt.hipGraphLaunch(exe, s), "hipGraphLaunch")
            _ok(rt.hipStreamSynchronize(s), "sync")
            rows = [r for r in range(c.x.shape[0])]
            assert torch.equal(c.y[rows], want[i][0][rows]), "replay %d" % i
            assert torch.equal(c.pool_buf, want[i][1]), "replay %d: state" % i
            # work of the program's own
            (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
        # another slot for the first sequence: the replay follows
        free = [v for v in range(c.n_slots) if v not in c.slots][0]
        c.pool_buf[free] = start[c.slots[0]]
        first = want[0][0][: c.starts[1]]
        old = c.pool_buf[c.slots[0]].clone()
        c.d_slots[0] = free
        torch.cuda.synchronize()
        _ok(rt.hipGraphLaunch(exe, s), "hipGraphLaunch")
        _ok(rt.hipStreamSynchronize(s), "sync")
        assert torch.equal(c.y[: c.starts[1]], first)
        assert torch.equal(c.pool_buf[c.slots[0]], old)
    finally:
        rt.hipGraphExecDestroy(exe)
        rt.hipGraphDestroy(graph)


def test_slot_moves_captured(hip, rt, streams):
    s = streams[0]
    pool = torch.randn((3, 8, 100), device="cuda")
    src = gpu(np.array([1, 2, 0, -1]), torch.int32)
    dst = gpu(np.array([0, 1, 2, 5]), torch.int32)
    table = gpu(np.array([7, -1, 2, 6, 7]), torch.int32)
    new, n = torch.zeros_like(table), torch.zeros(1, dtype=torch.int32, device="cuda")
    work = torch.zeros(hip.bm_hip_slots_compact_workspace_bytes(8), dtype=torch.uint8, device="cuda")
    d = bh.Slots(base=at(pool), n_slots=8, n_layers=3, slot_bytes=400, slot_stride=400,
                 layer_stride=3200)

    def both():
        return (hip.bm_hip_slots_copy_dev(C.byref(d), 1, at(src), at(dst), 4, s.value) or
                hip.bm_hip_slots_compact_dev(C.byref(d), 1, at(table), at(new), 5, at(n), at(work),
                                             s.value))

    def expected(p):
        q = p.clone()
        q[:, [0, 1, 2]] = p[:, [1, 2, 0]]
        q[:, 5] = 0.0
        r = q.clone()  # live 2, 6, 7: 6 -> 0, 7 -> 1
        r[:, 0], r[:, 1] = q[:, 6], q[:, 7]
        return r

    torch.cuda.synchronize()
    graph, exe = C.c_void_p(), C.c_void_p()
    _ok(rt.hipStreamBeginCapture(s, 1), "hipStreamBeginCapture")
    rc = both()
    _ok(rt.hipStreamEndCapture(s, C.byref(graph)), "hipStreamEndCapture")
    assert rc == 0, bh.last_error()
    _ok(rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0), "instantiate")
    try:
        for i in range(3):
            want = expected(pool)
            pool.add_(0.0)
            torch.cuda.synchronize()
            _ok(rt.hipGraphLaunch(exe, s), "hipGraphLaunch")
            _ok(rt.hipStreamSynchronize(s), "sync")
            assert torch.equal(pool, want), "replay %d" % i
            assert new.tolist() == [1, -1, 2, 0, 1] and n.item() == 3
            pool.copy_(torch.randn_like(pool))
    finally:
        rt.hipGraphExecDestroy(exe)
        rt.hipGraphDestroy(graph)


def test_two_streams_at_once(hip, rt, streams):
    """Calls on two streams with workspaces and pools of their own, in flight
    together, several times over."""
    for make in (lambda k: SsmCase("f32", 8, 64, 1, 24, [900, 40], seed=k),
                 lambda k: SsmCase("f32", 16, 64, 16, 1, [700, 300], seed=k),
                 lambda k: ConvCase("f32", 1000, 4, [500, 300], seed=k)):
        a, b = make(1), make(2)
        alone = []
        for c in (a, b):
            start = c.pool_buf.clone()
            c.run(hip)
            alone.append((c.y.clone(), c.pool_buf.clone(), start))
        ds = [c.descriptor() for c in (a, b)]
        ws = [c.workspace(hip, d) if isinstance(c, SsmCase) else None for c, d in zip((a, b), ds)]
        fs = [calls(hip, c, d, w) for c, d, w in zip((a, b), ds, ws)]
        for _ in range(5):
            for c, (_, _, start) in zip((a, b), alone):
                c.pool_buf.copy_(start)
                c.y.fill_(9.0)
            torch.cuda.synchronize()
            for f, s in zip(fs, streams):
                assert f(s.value) == 0, bh.last_error()
            for s in streams:
                _ok(rt.hipStreamSynchronize(s), "sync")
            for c, (y, pool, _) in zip((a, b), alone):
                assert torch.equal(c.y, y) and torch.equal(c.pool_buf, pool)


def test_calls_repeat_bit_for_bit(hip):
    """The same call on the same inputs: the same bits, whatever else ran."""
    for make in (lambda: SsmCase("f32", 8, 64, 1, 128, [700, 40, 333], seed=1),
                 lambda: SsmCase("f32", 64, 64, 64, 1, [1024], seed=2),
                 lambda: SsmCase("bf16", 8, 64, 1, 64, [1] * 40, step=True, seed=3)):
        got = []
        for _ in range(3):
            c = make()
            c.run(hip)
            got.append((c.y.clone(), c.pool_buf.clone()))
        for y, pool in got[1:]:
            assert torch.equal(y, got[0][0]) and torch.equal(pool, got[0][1])


def test_no_allocation(hip, rt):
    free0, free1, total = C.c_size_t(), C.c_size_t(), C.c_size_t()
    made = cases()
    fs = []
    for _, c in made:
        d = c.descriptor()
        w = c.workspace(hip, d) if isinstance(c, SsmCase) and not c.step else None
        fs.append((calls(hip, c, d, w), d))
    torch.cuda.synchronize()
    for f, _ in fs:
        assert f(None) == 0
    bh.check(hip.bm_hip_synchronize())
    _ok(rt.hipMemGetInfo(C.byref(free0), C.byref(total)), "hipMemGetInfo")
    for _ in range(3):
        for f, _ in fs:
            assert f(None) == 0
    bh.check(hip.bm_hip_synchronize())
    _ok(rt.hipMemGetInfo(C.byref(free1), C.byref(total)), "hipMemGetInfo")
    assert free0.value == free1.value


# ---------------------------------------------------------------------------
# a block of the model, for several sequences
# ---------------------------------------------------------------------------
def bitlinear(hip, x, gamma, packed, N, scale):
    M, K = x.shape
    out = torch.empty((M, N), device="cuda")
    xq = torch.empty((M, K), dtype=torch.int8, device="cuda")
    sx = torch.empty(M, device="cuda")
    act = torch.empty(hip.bm_hip_act_bytes(M, K), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_bitlinear_dev(at(x), M, K, at(gamma), at(packed), N, scale, 1, at(out),
                                      at(xq), K, at(sx), at(act), None))
    bh.check(hip.bm_hip_synchronize())
    return out


def test_a_block_between_its_products(hip):
    """in_proj, convolution of x, scan with z, B, C and dt out of in_proj's
    rows, out_proj: prompts of three sequences, one of them forked, then single
    tokens; the recurrence against the reference's own scalar step in the oracle
    (src/kernel.c:34-70), sequence by sequence and token by token."""
    r = np.random.default_rng(0)
    dm, nh, hd = 128, 4, 64
    di = nh * hd
    rows = 2 * di + 3 * nh
    w_in = gpu(bh.synth_ternary(3, 1, rows, dm, bh.SYNTH_P0_40))
    w_out = gpu(bh.synth_ternary(3, 2, dm, di, bh.SYNTH_P0_40))
    g_in, g_out = (gpu(1.0 + 0.1 * r.standard_normal(n), torch.float32) for n in (dm, di))
    cw = r.standard_normal((4, di)).astype(np.float32) * 0.5
    cb = r.standard_normal(di).astype(np.float32) * 0.1
    A = -np.exp(r.uniform(0, 2.5, nh)).astype(np.float32)
    dtb = r.uniform(-5, -2, nh).astype(np.float32)
    D = r.standard_normal(di).astype(np.float32)
    d_cw, d_cb, d_A, d_dtb, d_D = (gpu(a, torch.float32) for a in (cw, cb, A, dtb, D))
    n_slots = 6
    conv = torch.zeros((n_slots, 3, di), device="cuda")
    ssm = torch.zeros((n_slots, di), device="cuda")
    O = native.oracle()
    host = {k: dict(ring=np.zeros((3, di), np.float32), pos=0, st=np.zeros(di, np.float32))
            for k in range(n_slots)}

    def oracle_token(slot, proj):
        h = host[slot]
        p = h["pos"]
        y = np.empty(di, np.float32)
        proj = np.ascontiguousarray(proj)
        ring = [h["ring"][(p + i) % 3] for i in range(3)]
        O.orc_ssm_inner(bh.ptr(proj), di, nh, bh.ptr(dtb), bh.ptr(A), bh.ptr(cw), bh.ptr(cb),
                        bh.ptr(ring[0]), bh.ptr(ring[1]), bh.ptr(ring[2]), bh.ptr(h["st"]),
                        bh.ptr(D), bh.ptr(y), 0, di)
        h["pos"] = (p + 1) % 3
        return y

    def mixer(proj, lens, slots, step):
        """y of the block's rows; the slots move on."""
        T = proj.shape[0]
        xc, y = torch.empty((T, di), device="cuda"), torch.empty((T, di), device="cuda")
        start = gpu(np.concatenate([[0], np.cumsum(lens)]), torch.int32)
        sl = gpu(np.array(slots), torch.int32)
        col = lambda k: at(proj) + 4 * k
        c = bh.Conv(type=bh.F32, channels=di, width=4, silu=1, n_seqs=len(lens), n_tokens=T,
                    seq_start=at(start), slots=at(sl), x=col(di), x_stride=rows, w=at(d_cw),
                    bias=at(d_cb), state=at(conv), state_stride=3 * di, n_slots=n_slots, y=at(xc),
                    y_stride=di)
        s = bh.Ssm(type=bh.F32, n_heads=nh, head_dim=hd, n_groups=nh, d_state=1, dt_softplus=1,
                   n_seqs=len(lens), n_tokens=T, seq_start=at(start), slots=at(sl), x=at(xc),
                   x_stride=di, B=col(2 * di), B_stride=rows, C=col(2 * di + nh), C_stride=rows,
                   dt=col(2 * di + 2 * nh), dt_stride=rows, z=col(0), z_stride=rows, A=at(d_A),
                   dt_bias=at(d_dtb), D=at(d_D), state=at(ssm), state_stride=di, n_slots=n_slots,
                   y=at(y), y_stride=di)
        n = hip.bm_hip_ssm_workspace_bytes(C.byref(s))
        work = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        if step:
            bh.check(hip.bm_hip_conv_step_dev(C.byref(c), None))
            bh.check(hip.bm_hip_ssm_step_dev(C.byref(s), None))
        else:
            bh.check(hip.bm_hip_conv_dev(C.byref(c), None))
            bh.check(hip.bm_hip_ssm_dev(C.byref(s), at(work) if n else None, None))
        bh.check(hip.bm_hip_synchronize())
        return y

    def compare(y, proj, lens, slots):
        """Both sides round every operation to fp32: off by the bound that
        recurrence.py takes for one of them, twice; the magnitudes by the
        largest values of the run."""
        want, k = np.empty((proj.shape[0], di), np.float32), 0
        for n, slot in zip(lens, slots):
            for _ in range(n):
                want[k] = oracle_token(slot, f64(proj)[k].astype(np.float32))
                k += 1
        scale = np.abs(want).max()
        # up to 100 tokens of a state, 8 roundings each, and the functions'
        assert np.abs(f64(y) - want).max() <= 2 * (8 * 100 + 64) * 2.0 ** -24 * scale

    lens, slots = [37, 5, 61], [4, 0, 2]
    x = gpu(r.standard_normal((sum(lens), dm)), torch.float32)
    proj = bitlinear(hip, x, g_in, w_in, rows, 0.05)
    y = mixer(proj, lens, slots, False)
    compare(y, proj, lens, slots)
    out = bitlinear(hip, y, g_out, w_out, dm, 0.05)
    assert torch.isfinite(out).all()
    # sequence 2 goes on twice: its slot is forked
    pools = (bh.Slots * 2)(
        bh.Slots(base=at(conv), n_slots=n_slots, n_layers=1, slot_bytes=12 * di,
                 slot_stride=12 * di, layer_stride=0),
        bh.Slots(base=at(ssm), n_slots=n_slots, n_layers=1, slot_bytes=4 * di, slot_stride=4 * di,
                 layer_stride=0))
    src, dst = gpu(np.array([2]), torch.int32), gpu(np.array([5]), torch.int32)
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_copy_dev(pools, 2, at(src), at(dst), 1, None))
    bh.check(hip.bm_hip_synchronize())
    host[5] = {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in host[2].items()}
    slots = [4, 0, 2, 5]
    for _ in range(6):
        x = gpu(r.standard_normal((4, dm)), torch.float32)
        proj = bitlinear(hip, x, g_in, w_in, rows, 0.05)
        y = mixer(proj, [1] * 4, slots, True)
        compare(y, proj, [1] * 4, slots)
    # sequence 1 ends: the others' slots move together
    table = gpu(np.array([4, -1, 2, 5]), torch.int32)
    work = torch.empty(hip.bm_hip_slots_compact_workspace_bytes(n_slots), dtype=torch.uint8,
                       device="cuda")
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_slots_compact_dev(pools, 2, at(table), at(table), 4, None, at(work), None))
    bh.check(hip.bm_hip_synchronize())
    assert table.tolist() == [0, -1, 2, 1]
    host[0], host[1] = host[4], host[5]
    x = gpu(r.standard_normal((3, dm)), torch.float32)
    proj = bitlinear(hip, x, g_in, w_in, rows, 0.05)
    y = mixer(proj, [1] * 3, [0, 2, 1], True)
    compare(y, proj, [1] * 3, [0, 2, 1])
