"""Arguments that the gated delta rule and the verification of drafts refuse,
before anything reaches the GPU, and the sizes of their workspaces.  The
pointers are addresses that are never read."""
import ctypes as C
import math

import pytest

import native
from native import bh

P = 1 << 40  # stands for a device address


def delta(**k):
    d = dict(type=bh.F32, n_heads=4, head_dim=16, n_groups=2, d_state=8, dt_softplus=1,
             beta_sigmoid=1, qk_norm=1, norm_eps=1e-6, scale=1.0, n_seqs=10, n_tokens=10,
             seq_start=P, slots=P, q=P, k=P, v=P, dt=P, beta=P, z=P, q_stride=16, k_stride=16,
             v_stride=64, dt_stride=4, beta_stride=4, z_stride=64, A=P, dt_bias=P, state=P,
             state_stride=512, n_slots=16, y=2 * P, y_stride=64)
    return bh.Delta(**dict(d, **k))


def verify(**k):
    d = dict(type=bh.F32, vocab=100, n_seqs=3, n_rows=9, row_start=P, target=P, target_stride=100,
             draft=P, draft_stride=100, temp=1.0, tokens=P, u=P, n_accepted=P, next_token=P,
             ratio=P, split_start=P)
    return bh.Verify(**dict(d, **k))


def refused(rc, word):
    assert rc == -2, rc
    assert word in bh.last_error(), bh.last_error()


W = C.c_void_p(P)


@pytest.mark.parametrize("word,change", [
    ("invalid", dict(type=3)), ("invalid", dict(type=-1)), ("invalid", dict(n_heads=0)),
    ("invalid", dict(n_groups=3)), ("invalid", dict(n_groups=0)), ("invalid", dict(d_state=0)),
    ("invalid", dict(d_state=257)), ("invalid", dict(head_dim=0)),
    ("invalid", dict(n_heads=65535, head_dim=64, n_groups=1)),
    ("n_seqs", dict(n_seqs=-1)), ("n_seqs", dict(n_seqs=(1 << 20) + 1, n_slots=1 << 21)),
    ("list", dict(n_seqs=(1 << 16) + 1, n_slots=1 << 17)),
    ("norm_eps", dict(norm_eps=0.0)), ("norm_eps", dict(norm_eps=-1e-6)),
    ("norm_eps", dict(norm_eps=math.nan)), ("norm_eps", dict(norm_eps=math.inf)),
    ("scale", dict(scale=math.nan)), ("scale", dict(scale=math.inf)),
    ("q needs", dict(q=None)), ("k needs", dict(k=None)), ("v needs", dict(v=None)),
    ("dt needs", dict(dt=None)), ("y needs", dict(y=None)), ("q needs", dict(q=P + 2)),
    ("k needs", dict(k_stride=15)), ("v needs", dict(v_stride=63)), ("v needs", dict(v_stride=1 << 24)),
    ("dt needs", dict(dt_stride=3)), ("beta needs", dict(beta_stride=3)),
    ("z needs", dict(z_stride=63)), ("y needs", dict(y_stride=63)),
    ("slots", dict(n_slots=0)), ("slots", dict(slots=None, n_slots=9)), ("slots", dict(state_stride=511)),
    ("addresses", dict(slots=P + 1)), ("addresses", dict(state=P + 2)),
    ("4 bytes", dict(A=P + 1)), ("4 bytes", dict(dt_bias=P + 2)),
    ("y overlaps q", dict(y=P + 8)), ("y overlaps v", dict(y=3 * P + 8, v=3 * P)),
    ("y overlaps z", dict(y=3 * P + 16, z=3 * P)), ("y overlaps beta", dict(y=3 * P, beta=3 * P)),
    ("y overlaps k", dict(y=3 * P, k=3 * P)), ("y overlaps dt", dict(y=3 * P, dt=3 * P))])
def test_delta_refuses(word, change):
    L = bh.lib()
    refused(L.bm_hip_delta_step_dev(C.byref(delta(**change)), None), word)
    refused(L.bm_hip_delta_dev(C.byref(delta(**change)), W, None), word)


@pytest.mark.parametrize("word,change", [
    ("seq_start", dict(seq_start=None)), ("n_tokens", dict(n_tokens=-1)),
    ("n_tokens", dict(n_tokens=1 << 30)), ("y overlaps v", dict(y=3 * P, v=3 * P)),
    ("y overlaps z", dict(y=3 * P, z=3 * P)), ("workspace", dict(n_tokens=33))])
def test_delta_prompts_refuse(word, change):
    refused(bh.lib().bm_hip_delta_dev(C.byref(delta(**change)), None, None), word)


def test_delta_workspace_is_on_256_bytes():
    refused(bh.lib().bm_hip_delta_dev(C.byref(delta(n_tokens=100)), C.c_void_p(P + 64), None), "workspace")


def test_steps_over_z_alone_are_refused():
    """y may be written over v, and over z where z is v."""
    L = bh.lib()
    refused(L.bm_hip_delta_step_dev(C.byref(delta(y=3 * P, z=3 * P)), None), "y overlaps z")
    for name in ("q", "k"):
        d = delta(y=3 * P, v=3 * P, head_dim=1, n_groups=4, d_state=1, q_stride=64, k_stride=64,
                  z=4 * P, **{name: 3 * P})
        refused(L.bm_hip_delta_step_dev(C.byref(d), None), "y overlaps " + name)
    if not L.bm_hip_available():  # past the checks: no GPU here
        assert L.bm_hip_delta_step_dev(C.byref(delta(y=3 * P, v=3 * P)), None) == -1
        assert L.bm_hip_delta_step_dev(C.byref(delta(y=3 * P, v=3 * P, z=3 * P)), None) == -1


def test_what_is_not_read_needs_no_address():
    L = bh.lib()
    if L.bm_hip_available():
        pytest.skip("would run with addresses that do not exist")
    for change in (dict(A=None, dt=None, dt_stride=0), dict(beta=None, beta_stride=0),
                   dict(z=None, z_stride=0), dict(qk_norm=0, norm_eps=0.0), dict(dt_bias=None),
                   dict(state=None, state_stride=0, n_slots=0)):
        assert L.bm_hip_delta_step_dev(C.byref(delta(**change)), None) == -1, bh.last_error()


def test_nothing_to_do():
    L = bh.lib()
    none = dict(q=None, k=None, v=None, dt=None, beta=None, z=None, y=None)
    assert L.bm_hip_delta_step_dev(C.byref(delta(n_seqs=0, **none)), None) == 0
    assert L.bm_hip_delta_dev(C.byref(delta(n_seqs=0, n_tokens=0, **none)), None, None) == 0
    assert L.bm_hip_verify_dev(C.byref(verify(n_seqs=0, n_rows=0, target=None, draft=None,
                                              tokens=None, u=None)), W, None) == 0
    refused(L.bm_hip_delta_dev(None, None, None), "descriptor")
    refused(L.bm_hip_delta_step_dev(None, None), "descriptor")
    refused(L.bm_hip_verify_dev(None, None, None), "descriptor")
    assert L.bm_hip_delta_workspace_bytes(None) == 0
    assert L.bm_hip_verify_workspace_bytes(None) == 0
    assert L.bm_hip_delta_workspace_bytes(C.byref(delta(n_tokens=-1))) == 0
    assert L.bm_hip_verify_workspace_bytes(C.byref(verify(vocab=0))) == 0


def delta_bytes(n_seqs, n_tokens, type_, heads, groups, state):
    d = bh.Delta(type=type_, n_heads=heads, head_dim=64, n_groups=groups, d_state=state,
                 n_seqs=n_seqs, n_tokens=n_tokens)
    return bh.lib().bm_hip_delta_workspace_bytes(C.byref(d))


@pytest.mark.parametrize("shape", [(bh.F32, 32, 16, 128), (bh.BF16, 1, 1, 1), (bh.F16, 6, 3, 256)])
def test_a_workspace_serves_fewer_rows_and_sequences(shape):
    rows = sorted(set(list(range(0, 700)) + list(range(700, 70000, 131)) + [1 << k for k in range(30)]))
    before = None
    for n in (1, 2, 3, 16, 64, 1000, 1 << 16, 1 << 20):
        sizes = [delta_bytes(n, t, *shape) for t in rows]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
        if before is not None:
            assert all(a <= b for a, b in zip(before, sizes))
        before = sizes
    # sequences that fit 32 rows need none, and a row of the others a bounded share
    assert before[rows.index(32)] == 0
    assert delta_bytes(1 << 20, 520, *shape) <= delta_bytes(1, 64 * (520 // 32 + 1), *shape)


@pytest.mark.parametrize("word,change", [
    ("invalid", dict(type=3)), ("invalid", dict(vocab=0)), ("invalid", dict(vocab=256001)),
    ("invalid", dict(n_seqs=-1)), ("invalid", dict(n_seqs=(1 << 20) + 1)),
    ("invalid", dict(n_rows=-1)), ("invalid", dict(n_rows=1 << 30)),
    ("row_start", dict(row_start=None)), ("target needs", dict(target=None)),
    ("target needs", dict(target=P + 2)), ("target needs", dict(target_stride=99)),
    ("target needs", dict(target_stride=1 << 24)), ("draft needs", dict(draft_stride=99)),
    ("draft needs", dict(draft=P + 1)), ("temp", dict(temp=-1.0)), ("temp", dict(temp=math.nan)),
    ("temp", dict(temp=math.inf)), ("required", dict(tokens=None)), ("required", dict(u=None)),
    ("required", dict(n_accepted=None)), ("required", dict(next_token=None)),
    ("required", dict(tokens=P + 2)), ("required", dict(ratio=P + 1)),
    ("required", dict(split_start=P + 2)), ("required", dict(row_start=P + 1))])
def test_verify_refuses(word, change):
    refused(bh.lib().bm_hip_verify_dev(C.byref(verify(**change)), W, None), word)


def test_verify_workspace():
    L = bh.lib()
    refused(L.bm_hip_verify_dev(C.byref(verify()), None, None), "workspace")
    refused(L.bm_hip_verify_dev(C.byref(verify()), C.c_void_p(P + 64), None), "workspace")
    size = lambda n, r, v: L.bm_hip_verify_workspace_bytes(C.byref(verify(n_seqs=n, n_rows=r, vocab=v)))
    for n in (1, 7, 100):
        for r in (0, 1, 8, 1000):
            for v in (1, 4096, 4097, 50257, 256000):
                assert size(n, r, v) <= min(size(n + 1, r, v), size(n, r + 1, v), size(n, r, min(v + 4096, 256000)))
    if not L.bm_hip_available():  # past the checks: no GPU here
        assert L.bm_hip_verify_dev(C.byref(verify(draft=None, ratio=None, split_start=None)), W, None) == -1
