"""The batched recurrence where a call is at the edge of what it is documented
to take: workspaces shared by calls of several sizes, kernels that only large
calls reach, values at the end of a type's range.  The oracle is the definition
in 64 bits with the bounds of tests/recurrence.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import TYPES, ConvCase, SsmCase, at, check_rows, close, f64, gpu, half_step

pytestmark = pytest.mark.gpu


def note(msg):
    print("[case] " + msg, flush=True)


@pytest.mark.parametrize("shape,rows,most", [((64, 64, 64, 1), 1024, 2049),
                                             ((2, 32, 1, 24), 4096, 4097)])
def test_a_workspace_serves_shorter_prompts(hip, shape, rows, most):
    """A workspace of the longest prompt's size, and a shorter one whose units
    are more: right, and nothing behind the workspace is written."""
    note("scan %s: %d rows in the workspace of %d" % (shape, rows, most))
    c = SsmCase("f32", *shape, [rows], seed=2)
    want, tols, pool, stol = c.want()
    d = c.descriptor()
    d.n_tokens = most
    n = hip.bm_hip_ssm_workspace_bytes(C.byref(d))
    d.n_tokens = rows
    assert hip.bm_hip_ssm_workspace_bytes(C.byref(d)) <= n
    work = torch.full((n + (1 << 20),), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_ssm_dev(C.byref(d), at(work), None))
    torch.cuda.synchronize()
    assert (work[n:] == 0xFF).all()
    check_rows(c.ybuf, c.y, want, tols, "f32", (c.H, c.P), "shorter")
    k = c.slots[0]
    close(c.pool()[k], pool[k], stol[k], "f32", "state")


@pytest.mark.parametrize("N", [0, 1, 24])
def test_calls_without_rows(hip, N):
    """Prompts without a row and tensors without an address: a fresh
    sequence's slot becomes zero, the others stay (N 0: the convolution)."""
    note("no rows, N=%d" % N)
    c = SsmCase("f32", 4, 40, 2, N, [0] * 3, seed=1) if N else ConvCase("f32", 130, 4, [0] * 3, seed=1)
    c.fresh = [0, 1, 0]
    d = c.descriptor()
    for f in ["x", "y"] + (["B", "C", "dt", "z"] if N else []):
        setattr(d, f, None)
    want = c.pool_buf.clone()
    want[c.slots[1]] = 0.0
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_ssm_dev(C.byref(d), None, None) if N else hip.bm_hip_conv_dev(C.byref(d), None))
    torch.cuda.synchronize()
    assert torch.equal(c.pool_buf, want)


@pytest.mark.parametrize("kind", ["conv", "conv_step", "scan1", "scan24", "step", "slots"])
def test_an_error_pending_is_not_the_calls(hip, kind):
    """A call does not fail for an error that the caller's own earlier HIP call
    left in the thread, and leaves it there."""
    rt = C.CDLL("libamdhip64.so")
    if kind == "slots":
        pool = torch.arange(8 * 16, dtype=torch.float32, device="cuda").view(8, 16)
        want = pool.clone()
        want[2] = pool[5]
        want[0], want[1] = want[2], want[7]
        d = bh.Slots(base=at(pool), n_slots=8, n_layers=1, slot_bytes=64, slot_stride=64)
        src, dst = gpu(np.array([5]), torch.int32), gpu(np.array([2]), torch.int32)
        table = gpu(np.array([2, 7]), torch.int32)
        work = torch.zeros(hip.bm_hip_slots_compact_workspace_bytes(8), dtype=torch.uint8,
                           device="cuda")
        f = lambda: (hip.bm_hip_slots_copy_dev(C.byref(d), 1, at(src), at(dst), 1, None) or
                     hip.bm_hip_slots_compact_dev(C.byref(d), 1, at(table), at(table), 2, None,
                                                  at(work), None))
    else:
        c = {"conv": lambda: ConvCase("f32", 64, 4, [40]),
             "conv_step": lambda: ConvCase("f32", 64, 4, [1] * 3, step=True),
             "scan1": lambda: SsmCase("f32", 2, 32, 2, 1, [300]),
             "scan24": lambda: SsmCase("f32", 2, 32, 2, 24, [300]),
             "step": lambda: SsmCase("f32", 2, 32, 2, 24, [1] * 3, step=True)}[kind]()
        rows, tols = c.want()[:2]
        d = c.descriptor()
        if kind.startswith("conv"):
            call = hip.bm_hip_conv_step_dev if c.step else hip.bm_hip_conv_dev
            f = lambda: call(C.byref(d), None)
        elif c.step:
            f = lambda: hip.bm_hip_ssm_step_dev(C.byref(d), None)
        else:
            w = c.workspace(hip, d)
            f = lambda: hip.bm_hip_ssm_dev(C.byref(d), w, None)
    torch.cuda.synchronize()
    note("%s with an error pending" % kind)
    refused = rt.hipMalloc(None, C.c_size_t(16))  # on the host: no pointer to fill
    assert refused != 0
    rc = f()
    assert rt.hipGetLastError() == refused
    assert rc == 0, bh.last_error()
    torch.cuda.synchronize()
    if kind == "slots":
        assert torch.equal(pool, want) and table.tolist() == [0, 1]
    else:
        shape = (64,) if kind.startswith("conv") else (c.H, c.P)
        check_rows(c.ybuf, c.y, rows, tols, "f32", shape, kind)


# ---------------------------------------------------------------------------
# a state that decays over thousands of tokens.  u = 2^-24.
# ---------------------------------------------------------------------------
def bare_state(H, N, T, rates, step):
    """States of 1 and no input, one channel per head: what is left after T
    tokens is the decays' product."""
    c = SsmCase("f32", H, 1, 1, N, [1] if step else [T], gate=False, skip=False, bias=False,
                soft=False, step=step, slots=None, spare=0)
    c.x.zero_()
    c.dt.fill_(1.0)
    c.A = gpu(-rates, torch.float32)
    c.pool_buf.fill_(1.0)
    return c


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("N", [1, 2, 4, 5, 24])
def test_one_decay(hip, N, step):
    """The decay of one token, rates from 2^-20 to 2^-5: rounded to nearest, off
    by u / 2 for values from 1/2 to 1; the sum p^2 / 2 + ... in front of it has
    three roundings of less than 2^-11, u / 100 at most with the series's rest.
    From 9 values on the scan's own operands have three bf16 pieces, off by u,
    and the hardware's exponential is good to u."""
    rates = np.exp2(np.linspace(-20, -5, 4096))
    c = bare_state(4096, N, 1, rates, step)
    note("one decay, N=%d step=%s" % (N, step))
    want = np.exp(f64(c.A))
    c.run(hip)
    err = (c.pool()[0].reshape(4096, N) - want[:, None]) * 2.0 ** 24
    lim = 0.51 if step or N <= 8 else 2.0
    assert np.abs(err).max() <= lim
    if step or N <= 8:
        # 4096 errors of at most 0.51 each about zero: their mean is off by
        # 0.04 once in exp(2 (0.04 4096)^2 / (4096 1.02^2)) > 10^5 such tests
        assert abs(err.mean()) <= 0.04


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("N", [1, 5])
def test_a_slow_state_keeps_its_value(hip, N, step):
    """T tokens of a rate of about 2^-10.  Every token rounds the state once,
    by u at most and to either side: T such errors sum up to more than 6 sqrt(T)
    u once in exp(6^2 / 2) / 2 > 10^7 states; a decay that is 0.12 u too
    small in every token would leave 0.12 T u, nearly twice as much.  The scan
    joins up to 64 units of equal decays, each rounded once: 64 u for these,
    64 u for the products, and the last unit's tokens: less than that."""
    T, H = 8192, 64
    rates = np.exp2(np.linspace(-10.5, -9.5, H))
    c = bare_state(H, N, T, rates, step)
    note("slow state, N=%d step=%s" % (N, step))
    want = np.exp(T * f64(c.A))
    if step:
        d = c.descriptor()
        torch.cuda.synchronize()
        for _ in range(T):
            bh.check(hip.bm_hip_ssm_step_dev(C.byref(d), None))
        torch.cuda.synchronize()
    else:
        c.run(hip)
    err = (c.pool()[0].reshape(H, N) / want[:, None] - 1.0) * 2.0 ** 24
    assert np.abs(err).max() <= 6 * T ** 0.5


@pytest.mark.parametrize("N", [1, 2, 3, 8])
def test_an_infinite_state_stays_infinite(hip, N):
    """An infinite state under finite inputs and decays, over units that end
    within a tile of rows, and by single tokens."""
    for lens, step in (([37, 16, 1], False), ([1] * 3, True)):
        c = SsmCase("f32", 2, 20, 1, N, lens, slots=None, spare=0, seed=N, step=step)
        c.A = gpu(np.array([-1e-6, -2.0]), torch.float32)
        c.pool_buf[1, :] = float("inf")
        note("infinite state, N=%d step=%s" % (N, step))
        c.run(hip)
        p = c.pool()
        assert np.isposinf(p[1]).all() and np.isfinite(p[[0, 2]]).all()


@pytest.mark.parametrize("N", [5, 24, 128])
@pytest.mark.parametrize("value", [3.4e38, float(np.finfo(np.float32).min), 1e38])
def test_the_largest_floats_do_not_reach_earlier_rows(hip, N, value):
    """A finite x at the end of fp32's range, past what a bf16 holds: earlier
    rows, other channels and other sequences are bit for bit what they were.
    Where it is within that range (1e38) or the state has up to 8 values, its
    own row is right, too."""
    H, P, lens, row, ch = 2, 40, [37, 90, 20], 37 + 50, 47
    def case():
        return SsmCase("f32", H, P, 1, N, lens, seed=9, gate=False, skip=False, soft=False)
    clean, c = case(), case()
    clean.run(hip)
    c.x[row, ch] = value
    note("x = %g, N=%d" % (value, N))
    with np.errstate(over="ignore"):
        rows, tols = c.want()[:2]
    c.run(hip)
    y0, y1 = f64(clean.y), f64(c.y)
    keep = [r for r in range(sum(lens)) if r < row or r >= 37 + 90]
    assert np.array_equal(y0[keep], y1[keep])
    rest = [k for k in range(H * P) if k != ch]
    assert np.array_equal(y0[row:37 + 90, rest], y1[row:37 + 90, rest])
    for b in (0, 2):
        assert np.array_equal(clean.pool()[c.slots[b]], c.pool()[c.slots[b]])
    if N <= 8 or abs(value) < 3.3e38:
        close(y1[row, ch], rows[row].reshape(-1)[ch], tols[row].reshape(-1)[ch], "f32", "its row")


def test_bf16_after_steps_that_forget_everything(hip):
    """Twenty steps whose decays vanish (exponents of -5120 powers of two in
    all), then twelve small ones: decays between the small ones are as good as
    without the sum before them.  u = 2^-24.  Of each term the bf16 operands
    have two pieces (2^-17 for both products), its sums and the exponential
    4 N + 200 roundings at most; the result is rounded once, by half of its own
    last place."""
    H, P, N, T = 2, 32, 32, 96
    c = SsmCase("bf16", H, P, 1, N, [T], seed=5, gate=False, skip=False, bias=False, soft=False)
    c.A = gpu(np.array([-1.0, -2.5]), torch.float32)
    r = np.random.default_rng(5)
    dt = np.exp(r.uniform(-6, -2, (T, H)))
    dt[np.arange(T) % 32 < 20] = 200.0
    c.dt.copy_(torch.as_tensor(dt))
    x, B, Cm = f64(c.x).reshape(T, H, P), f64(c.B), f64(c.Cm)
    dt, A, S = f64(c.dt), f64(c.A), c.pool()[c.slots[0]]
    M, want, mag = np.abs(S), np.empty((T, H, P)), np.empty((T, H, P))
    for t in range(T):
        a = np.exp(A * dt[t])[:, None, None]
        add = dt[t][:, None, None] * x[t][:, :, None] * B[t]
        S, M = a * S + add, a * M + np.abs(add)
        want[t], mag[t] = (S * Cm[t]).sum(-1), (M * np.abs(Cm[t])).sum(-1)
    note("bf16 after vanishing decays")
    c.run(hip)
    off = (2.0 ** -17 + (4 * N + 200) * 2.0 ** -24) * mag
    half = np.exp2(np.floor(np.log2(np.abs(want) + off)) - 8)
    assert (np.abs(f64(c.y).reshape(T, H, P) - want) <= off + half).all()


# ---------------------------------------------------------------------------
# growth: A d > 0.  The bounds of tests/recurrence.py take the exponents in.
# ---------------------------------------------------------------------------
GROWTH = [("f32", 1), ("f32", 5), ("f32", 9), ("f32", 24), ("bf16", 24), ("f16", 40), ("f32", 128),
          ("bf16", 128), ("f32", 200)]


def growing(type_name, N, T, rate, start, heads=2):
    """Head 0 grows by e^rate in each token, the last one decays."""
    c = SsmCase(type_name, heads, 40, 1, N, [T, 5], gate=False, skip=False, bias=False, soft=False,
                slots=None, spare=0, seed=N + T)
    c.A[:] = rate
    c.A[-1] = -0.5
    c.dt.fill_(1.0)
    c.pool_buf[0] = start
    return c


def check_growth(c, hip, what, rows_in_range=None, relative=0.0, lost=0.0):
    """c.check, where a result that rounds past the type's largest value, half
    a step above it, is infinite.  From row rows_in_range on the states of all
    heads but the last pass fp32's range and are not looked at.  relative and
    lost (of y): what the bounds of tests/recurrence.py do not have."""
    last = slice(c.H - 1, c.H)
    rows, tols, pool, stol = c.want()
    c.run(hip)
    got = f64(c.y).reshape(-1, c.H, c.P)
    top = torch.finfo(TYPES[c.type][1]).max * (1 + half_step(c.type) / 2)
    for t in rows:
        heads = slice(None) if rows_in_range is None or t < rows_in_range else last
        g, want = got[t][heads], rows[t][heads]
        tol = tols[t][heads] + relative * np.abs(want) + lost
        inf = np.isinf(g) & (np.abs(want) + tol >= top) & (g * want > 0)
        assert inf[np.abs(want) - tol > top].all(), "%s row %d" % (what, t)
        close(np.where(inf, 0.0, g), np.where(inf, 0.0, want), tol, c.type, "%s row %d" % (what, t))
    for k in stol:
        heads = slice(None) if rows_in_range is None or k == 0 else last
        close(c.pool()[k][heads], pool[k][heads], (stol[k] + relative * np.abs(pool[k]))[heads],
              "f32", "%s slot %d" % (what, k))


@pytest.mark.parametrize("type_name,N", GROWTH)
@pytest.mark.parametrize("T,rate", [(33, 3.0), (70, 3.0), (150, 1.0), (700, 0.5), (300, 30.0), (64, 80.0)])
def test_nothing_grows_into_nothing(hip, type_name, N, T, rate):
    """Growth past fp32 of a zero state under zero inputs: zero until the last
    token, whose own part is finite, in one unit and over several."""
    c = growing(type_name, N, T, rate, 0.0, heads=5)
    c.x[:T - 1] = 0.0
    note("zero state, %s N=%d, %d tokens of e^%g" % (type_name, N, T, rate))
    check_growth(c, hip, "nothing grows", T)


@pytest.mark.parametrize("type_name,N", GROWTH)
@pytest.mark.parametrize("T,rate,exponent", [(40, 3.0, -123), (180, 0.8, -123), (41, 2.0, -110),
                                             (36, 4.5, -145)])
def test_a_small_state_grows_past_any_decay(hip, type_name, N, T, rate, exponent):
    """A state of 2^exponent and no input: the decays over a unit, or over 32
    tokens, are past fp32, the states are not.  Below 2^-126 the two roundings
    of a token are 2^-150 each, whatever the state; those of token k grow with
    it, to 2^(-149 - exponent) e^(-rate k) of it: the sum over k below.  From 9
    values on each of a state's three bf16 pieces counts as zero below 2^-126,
    times a chunk's growth of up to 2^16 and C."""
    c = growing(type_name, N, T, rate, 2.0 ** exponent)
    c.x.zero_()
    if type_name != "f32":  # y itself would be rounded to nothing, or past fp16
        c.Cm.zero_()
    note("small state, %s N=%d, %d tokens of e^%g" % (type_name, N, T, rate))
    lost = 3 * 2.0 ** (16 - 126) * np.abs(f64(c.Cm)).max() * N if N > 8 else 0.0
    check_growth(c, hip, "small state", T, 2.0 ** (-149 - exponent) / (np.exp(rate) - 1), lost)
    assert np.isfinite(c.pool()[0]).all() and c.pool()[0, 0].min() > 1.0


@pytest.mark.parametrize("N", [1, 9, 128])
def test_a_chunk_with_some_growing_tokens(hip, N):
    """Steps of both signs: runs of growth that need a cut anywhere in a chunk,
    in one head of several that share B and C."""
    c = SsmCase("f32", 6, 40, 1, N, [300, 90, 33], gate=True, skip=True, bias=False, soft=False,
                seed=N)
    r = np.random.default_rng(N)
    dt = np.abs(r.standard_normal((423, 6))) * 0.5
    for at_ in (0, 7, 14, 21, 29, 37, 44, 60, 140, 147, 155, 290, 300, 307, 315, 380, 388, 395, 403):
        dt[at_:at_ + 3, 2] = -r.uniform(16, 20, 3)  # to e^60 at most
        dt[at_ + 3:at_ + 7, 2] = 30.0  # and forgotten
    c.dt.copy_(torch.as_tensor(dt))
    c.A[:] = -1.0
    note("steps of both signs, N=%d" % N)
    check_growth(c, hip, "both signs")


@pytest.mark.parametrize("type_name,N", [("f32", 1), ("f32", 24), ("bf16", 128), ("f32", 256)])
@pytest.mark.parametrize("head", [0, 3, 6])
def test_one_growing_head_under_softplus(hip, type_name, N, head):
    """Steps that softplus makes positive, one head of seven with A > 0: it
    alone grows, from nothing, past fp32 several times over."""
    T = 290
    c = SsmCase(type_name, 7, 40, 1, N, [T], bias=True, gate=True, skip=True, seed=N + head,
                slots=None, spare=0)
    c.A[head] = 3.0
    c.dt[:, head] = 2.0
    c.dt_bias[head] = 0.0
    c.pool_buf[0].view(7, 40, N)[head] = 0.0
    c.x[:T - 2].view(T - 2, -1)[:, 40 * head:40 * head + 40] = 0.0
    note("head %d grows, %s N=%d" % (head, type_name, N))
    check_growth(c, hip, "softplus")
