"""The gated delta rule where little is written: gates that are nearly or quite
shut, values that no gate lets through, keys of any length.  What a row writes,
b v |k|, and the state are then far from v, and both are held to the bounds of
tests/delta.py, which go by them alone."""
import numpy as np
import pytest
import torch

from delta import DeltaCase
from recurrence import check_rows, close, f64

pytestmark = pytest.mark.gpu

LENS = [130, 33, 20, 200]


def note(msg):
    print("[case] " + msg, flush=True)


def case(type_name="f32", lens=LENS, seed=0, step=False, **kw):
    """Few decays, so that a state holds what many rows have written."""
    kw = dict(dict(rate=0.5), **kw)
    return DeltaCase(type_name, 2, 20, 1, 64, [1] * 4 if step else lens, seed=seed, step=step, **kw)


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("start", ["zeros", "fresh", "carried"])
@pytest.mark.parametrize("logit", [-6, -9, -12, -20])
def test_gates_nearly_shut(hip, type_name, logit, start):
    note("b = sigmoid(N(%d, 1)) %s, %s" % (logit, type_name, start))
    c = case(type_name, seed=-logit)
    c.beta.add_(float(logit))
    if start == "zeros":
        c.pool_buf.zero_()
    elif start == "fresh":
        c.fresh = [1] * 4
    c.check(hip, "shut")


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("size", [-7, -10, -14, -20, -27, -40])
def test_small_b(hip, size, step):
    note("b near 2^%d step=%s" % (size, step))
    for zeros in (True, False):
        c = case(seed=-size, step=step, beta="raw", decay=zeros)
        c.beta.mul_(2.0 ** size)
        if zeros:
            c.pool_buf.zero_()
        c.check(hip, "small b")


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,P,G,N", [(2, 17, 1, 100), (1, 5, 1, 7), (4, 1, 4, 1), (2, 33, 2, 256),
                                     (2, 40, 1, 128), (1, 16, 1, 65)])
def test_gates_nearly_shut_of_any_size(hip, type_name, H, P, G, N):
    note("shut, %s %s" % (type_name, (H, P, G, N)))
    c = DeltaCase(type_name, H, P, G, N, [130, 33, 20, 200], seed=N, rate=0.5)
    c.beta.sub_(9.0)
    c.pool_buf.mul_(2.0 ** -12)
    c.check(hip, "shut")


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("size", [0, -7, -14, -20, -27, -60])
def test_no_gate_and_a_small_state(hip, size, step):
    """b = 0 beside ordinary v: all that is read is what the slots hold."""
    note("b = 0, state 2^%d step=%s" % (size, step))
    c = case(seed=1, step=step, beta="raw")
    c.beta.zero_()
    c.pool_buf.mul_(2.0 ** size)
    c.check(hip, "no gate")


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 40, 2.0 ** 60])
@pytest.mark.parametrize("type_name", ["f32", "bf16"])
def test_large_values_that_are_not_written(hip, type_name, size):
    """Rows of b = 0 with large v among ordinary ones."""
    note("unwritten v of %g %s" % (size, type_name))
    c = case(type_name, seed=2, beta="raw")
    for t in (0, 17, 63, 64, 90, 129, 140, 200, 382):
        c.beta[t] = 0.0
        c.v[t] *= size
    c.check(hip, "unwritten")


def test_gates_that_open_and_shut(hip):
    """2^30 more and less from one chunk to another, states that decay between."""
    note("open and shut")
    c = case(lens=[400, 90], seed=3, rate=4.0, beta="raw")
    f = torch.ones(490, device="cuda")
    f[:70] = f[200:330] = f[420:] = 2.0 ** -30
    c.beta.mul_(f[:, None])
    c.check(hip, "open and shut")


@pytest.mark.parametrize("size", [-20, -30, -60])
def test_small_values_after_none(hip, size):
    """A chunk in which nothing is written to a state of zeros comes first."""
    note("2^%d after nothing" % size)
    c = case(lens=[200, 40], seed=7)
    c.pool_buf.zero_()
    c.v[:100] = 0.0
    c.v[100:].mul_(2.0 ** size)
    c.check(hip, "after none")


def test_small_values_after_large_ones_that_are_gone(hip):
    """2^90 first, then 2^-70, with decays that leave nothing of a row two rows on."""
    note("2^-70 after 2^90")
    c = case(lens=[300], seed=8)
    c.A.fill_(-200.0)
    c.v[:100].mul_(2.0 ** 90)
    c.v[100:].mul_(2.0 ** -70)
    c.check(hip, "after large ones")


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("size", [-20, -8, 8, 20])
def test_keys_of_any_length(hip, size, step):
    """k and v times 2^size and b times 2^(-2 size): w comes out times 2^-size, and
    state and y as before."""
    note("keys of 2^%d step=%s" % (size, step))
    c = case(seed=4, step=step, norm=False, beta="raw")
    rows, tols, pool, stol = c.want()
    c.k.mul_(2.0 ** size)
    c.v.mul_(2.0 ** size)
    c.beta.mul_(4.0 ** -size)
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "keys")
    for k, tol in stol.items():
        close(c.pool()[k], pool[k], tol, "f32", "slot %d" % k)


def test_keys_of_many_lengths(hip):
    """The same with a size of its own for each row."""
    note("keys of many lengths")
    c = case(seed=5, norm=False, beta="raw")
    rows, tols, pool, stol = c.want()
    f = torch.exp2(torch.randint(-12, 13, (sum(LENS),), generator=torch.Generator().manual_seed(5))
                   .float()).cuda()[:, None]
    c.k.mul_(f)
    c.v.mul_(f)
    c.beta.div_(f * f)
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "keys")
    for k, tol in stol.items():
        close(c.pool()[k], pool[k], tol, "f32", "slot %d" % k)


@pytest.mark.parametrize("keys", ["any", "nearly equal"])
@pytest.mark.parametrize("step", [False, True])
def test_b_up_to_two(hip, keys, step):
    """A row of b = 2 turns its key's value round; no vector grows."""
    note("b in 1..2, keys %s step=%s" % (keys, step))
    c = case(seed=6, step=step, beta="raw")
    c.beta.add_(1.0)
    if keys != "any":
        c.k.mul_(2.0 ** -10).add_(c.k[:1].clone())
    rows, tols, pool, stol = c.want()
    c.run(hip)
    check_rows(c.ybuf, c.y, rows, tols, "f32", (2, 20), "b up to 2")
    for k, tol in stol.items():
        close(c.pool()[k], pool[k], tol, "f32", "slot %d" % k)


@pytest.mark.parametrize("lens,at_row", [([130], 70), ([130], 0), ([20], 7), ([1], 0)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_an_infinite_b(hip, value, lens, at_row):
    """The head is NaN from its row on, y and state, in prompts, short sequences
    and single tokens; the sigmoid of an infinite logit is 0 or 1."""
    note("b = %r, %s" % (value, lens))
    for step in ([True, False] if lens == [1] else [False]):
        c = DeltaCase("f32", 2, 20, 1, 64, lens, seed=9, step=step, beta="raw", gate=False)
        rows, tols, pool, stol = c.want()
        c.beta[at_row, 1] = value
        c.run(hip)
        got, state = f64(c.y).reshape(-1, 2, 20), c.pool()[c.slots[0]]
        assert np.isnan(got[at_row:, 1]).all() and np.isnan(state[1]).all()
        for t in rows:
            ok = slice(0, 1 if t >= at_row else 2)
            close(got[t][ok], rows[t][ok], tols[t][ok], "f32", "row %d" % t)
        close(state[0], pool[c.slots[0]][0], stol[c.slots[0]][0], "f32", "state")
        if value == value:
            c = DeltaCase("f32", 2, 20, 1, 64, lens, seed=9, step=step)
            c.beta[at_row, 1] = value
            c.check(hip, "logit")
