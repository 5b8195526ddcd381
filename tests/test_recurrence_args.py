"""Arguments that the batched recurrence calls refuse, before anything reaches
the GPU: -2 with the reason, on the CPU as on the GPU.  The pointers are
addresses that are never read."""
import ctypes as C

import pytest

import native
from native import bh

P = 1 << 40  # stands for a device address


def conv(**k):
    d = dict(type=bh.F32, channels=64, width=4, silu=1, n_seqs=2, n_tokens=10, seq_start=P,
             slots=P, x=P, x_stride=64, w=P, bias=P, state=P, state_stride=192, n_slots=2,
             y=2 * P, y_stride=64)
    return bh.Conv(**dict(d, **k))


def ssm(**k):
    d = dict(type=bh.F32, n_heads=4, head_dim=16, n_groups=2, d_state=8, dt_softplus=1, n_seqs=2,
             n_tokens=10, seq_start=P, slots=P, x=P, B=P, C=P, dt=P, z=P, x_stride=64,
             B_stride=16, C_stride=16, dt_stride=4, z_stride=64, A=P, dt_bias=P, D=P, state=P,
             state_stride=512, n_slots=2, y=2 * P, y_stride=64)
    return bh.Ssm(**dict(d, **k))


def slots(**k):
    d = dict(base=P, n_slots=4, n_layers=2, slot_bytes=64, slot_stride=64, layer_stride=256)
    return bh.Slots(**dict(d, **k))


def refused(rc, word):
    assert rc == -2, rc
    assert word in bh.last_error(), bh.last_error()


SHARED = [("type", dict(type=3)), ("type", dict(type=-1)), ("n_seqs", dict(n_seqs=-1)),
          ("n_seqs", dict(n_seqs=(1 << 20) + 1, n_slots=1 << 21)),
          ("x needs", dict(x=None)), ("x needs", dict(x=P + 2)), ("y needs", dict(y=None)),
          ("y needs", dict(y_stride=63)), ("x needs", dict(x_stride=63)),
          ("x needs", dict(x_stride=1 << 24)), ("slots", dict(n_slots=0)),
          ("slots", dict(slots=None, n_slots=1)), ("addresses", dict(slots=P + 1)),
          ("addresses", dict(state=P + 2)), ("y overlaps x", dict(y=P + 8)),
          ("y overlaps x", dict(y=P + 4 * 64 * 3))]
PROMPTS = [("seq_start", dict(seq_start=None)), ("n_tokens", dict(n_tokens=-1)),
           ("n_tokens", dict(n_tokens=1 << 30)),
           ("y overlaps x", dict(y=P))]


@pytest.mark.parametrize("word,change", SHARED + PROMPTS + [
    ("width", dict(width=1)), ("width", dict(width=5)), ("channels", dict(channels=0)),
    ("invalid", dict(w=None)), ("slots", dict(state_stride=191))])
def test_conv_refuses(word, change):
    L = bh.lib()
    if (word, change) not in PROMPTS:
        refused(L.bm_hip_conv_step_dev(C.byref(conv(n_seqs=10, n_slots=16, **change) if "n_seqs" not in change and
                                               "n_slots" not in change else conv(**change)), None), word)
    refused(L.bm_hip_conv_dev(C.byref(conv(**change)), None), word)


@pytest.mark.parametrize("word,change", SHARED + PROMPTS + [
    ("invalid", dict(n_heads=0)), ("invalid", dict(n_groups=3)), ("invalid", dict(n_groups=0)),
    ("invalid", dict(d_state=0)), ("invalid", dict(d_state=257)), ("invalid", dict(head_dim=0)),
    ("B needs", dict(B=None)), ("C needs", dict(C_stride=15)), ("dt needs", dict(dt_stride=3)),
    ("dt needs", dict(dt=None)), ("z needs", dict(z_stride=60)), ("A is required", dict(A=None)),
    ("4 bytes", dict(D=P + 1)), ("slots", dict(state_stride=511)),
    ("x needs", dict(x=None, z=None)), ("y overlaps z", dict(y=3 * P + 16, z=3 * P)),
    ("y overlaps B", dict(y=3 * P + 16, B=3 * P))])
def test_ssm_refuses(word, change):
    L = bh.lib()
    w = C.c_void_p(P)
    if (word, change) not in PROMPTS:
        more = {} if "n_seqs" in change or "n_slots" in change else dict(n_seqs=10, n_slots=16)
        refused(L.bm_hip_ssm_step_dev(C.byref(ssm(**dict(more, **change))), None), word)
    refused(L.bm_hip_ssm_dev(C.byref(ssm(**change)), w, None), word)


def test_null_descriptors():
    L = bh.lib()
    refused(L.bm_hip_conv_dev(None, None), "descriptor")
    refused(L.bm_hip_conv_step_dev(None, None), "descriptor")
    refused(L.bm_hip_ssm_dev(None, None, None), "descriptor")
    refused(L.bm_hip_ssm_step_dev(None, None), "descriptor")
    assert L.bm_hip_ssm_workspace_bytes(None) == 0


def test_workspace_is_required():
    """Where the sizes ask for one: absent or misaligned is refused; its size
    does not go by the pointers."""
    L = bh.lib()
    d = ssm(n_heads=64, head_dim=64, n_groups=1, d_state=128, n_seqs=1, n_tokens=16384,
            x_stride=4096, z_stride=4096, y_stride=4096, B_stride=128, C_stride=128, dt_stride=64,
            state_stride=1 << 19, y=4 * P)
    n = L.bm_hip_ssm_workspace_bytes(C.byref(d))
    bare = bh.Ssm(type=d.type, n_heads=64, head_dim=64, n_groups=1, d_state=128, n_seqs=1,
                  n_tokens=16384)
    assert L.bm_hip_ssm_workspace_bytes(C.byref(bare)) == n
    # many short sequences: no more than the rows of long ones could need
    bare.n_seqs = 4096
    assert L.bm_hip_ssm_workspace_bytes(C.byref(bare)) < 8 * n + (1 << 30)
    if n:
        refused(L.bm_hip_ssm_dev(C.byref(d), None, None), "workspace")
        refused(L.bm_hip_ssm_dev(C.byref(d), C.c_void_p(P + 64), None), "workspace")


def test_nothing_to_do():
    """No sequences: done, without a GPU."""
    L = bh.lib()
    assert L.bm_hip_conv_dev(C.byref(conv(n_seqs=0)), None) == 0
    assert L.bm_hip_conv_step_dev(C.byref(conv(n_seqs=0)), None) == 0
    assert L.bm_hip_ssm_step_dev(C.byref(ssm(n_seqs=0)), None) == 0
    assert L.bm_hip_ssm_dev(C.byref(ssm(n_seqs=0, n_tokens=0)), C.c_void_p(P), None) == 0
    assert L.bm_hip_slots_copy_dev(C.byref(slots()), 1, None, None, 0, None) == 0


def test_y_beside_x_in_one_buffer_is_no_overlap():
    """Columns of one buffer: x at column 0, y at column 64 of 128; one column
    less is refused, whichever of the two comes first."""
    L = bh.lib()
    if L.bm_hip_available():
        pytest.skip("would run with addresses that do not exist")
    for first, second in (("x", "y"), ("y", "x")):
        d = {first: P, second: P + 4 * 64, "x_stride": 128, "y_stride": 128}
        rc = L.bm_hip_conv_dev(C.byref(conv(**d)), None)
        assert rc == -1, bh.last_error()  # past the checks: no GPU here
        d[second] = P + 4 * 63
        refused(L.bm_hip_conv_dev(C.byref(conv(**d)), None), "overlaps")


@pytest.mark.parametrize("change", [
    dict(base=None), dict(n_slots=0), dict(n_layers=0), dict(slot_bytes=0), dict(slot_stride=63),
    dict(layer_stride=200), dict(layer_stride=-256), dict(slot_bytes=1 << 41, slot_stride=1 << 41),
    dict(n_layers=65536)])
def test_pools_refused(change):
    L = bh.lib()
    p = C.c_void_p(P)
    refused(L.bm_hip_slots_copy_dev(C.byref(slots(**change)), 1, p, p, 2, None), "pool")
    refused(L.bm_hip_slots_compact_dev(C.byref(slots(**change)), 1, p, p, 2, None, p, None), "pool")


def test_slot_lists_refused():
    L = bh.lib()
    p, odd = C.c_void_p(P), C.c_void_p(P + 2)
    d = C.byref(slots())
    two = (bh.Slots * 2)(slots(), slots(n_slots=5))
    refused(L.bm_hip_slots_copy_dev(None, 1, p, p, 2, None), "pools")
    refused(L.bm_hip_slots_copy_dev(d, 0, p, p, 2, None), "pools")
    refused(L.bm_hip_slots_copy_dev(d, 9, p, p, 2, None), "pools")
    refused(L.bm_hip_slots_copy_dev(two, 2, p, p, 2, None), "pool 1")
    refused(L.bm_hip_slots_copy_dev(d, 1, p, p, -1, None), "lists")
    refused(L.bm_hip_slots_copy_dev(d, 1, p, p, 1025, None), "lists")
    refused(L.bm_hip_slots_copy_dev(d, 1, None, p, 2, None), "lists")
    refused(L.bm_hip_slots_copy_dev(d, 1, p, None, 2, None), "lists")
    refused(L.bm_hip_slots_copy_dev(d, 1, odd, p, 2, None), "lists")
    big = C.byref(slots(n_slots=65537, layer_stride=64 * 65537))
    refused(L.bm_hip_slots_compact_dev(big, 1, p, p, 2, None, p, None), "arguments")
    refused(L.bm_hip_slots_compact_dev(d, 1, p, p, -1, None, p, None), "arguments")
    refused(L.bm_hip_slots_compact_dev(d, 1, None, p, 2, None, p, None), "arguments")
    refused(L.bm_hip_slots_compact_dev(d, 1, p, None, 2, None, p, None), "arguments")
    refused(L.bm_hip_slots_compact_dev(d, 1, p, p, 2, None, None, None), "arguments")
    refused(L.bm_hip_slots_compact_dev(d, 1, p, p, 2, None, C.c_void_p(P + 8), None), "arguments")
    assert L.bm_hip_slots_compact_workspace_bytes(0) == 0
    assert L.bm_hip_slots_compact_workspace_bytes(65537) == 0
    assert L.bm_hip_slots_compact_workspace_bytes(65536) > 0


def test_new_table_overlapping_in_part_is_refused():
    L = bh.lib()
    p, d = C.c_void_p(P), C.byref(slots())
    for shift in (-4, 4, 12):
        refused(L.bm_hip_slots_compact_dev(d, 1, p, C.c_void_p(P + shift), 4, None, p, None),
                "overlaps")


@pytest.mark.parametrize("name", ["B", "C", "dt"])
def test_step_over_an_input_that_other_channels_read_is_refused(name):
    """y over x is allowed, but not where x is also B, C or dt."""
    L = bh.lib()
    p = C.c_void_p(P)
    apart = {k: C.c_void_p(3 * P) for k in ("B", "C", "dt", "z")}  # the others' rows
    d = ssm(n_heads=4, head_dim=1, n_groups=4, d_state=1, y=p, x_stride=64, y_stride=64,
            **dict(apart, **{"x": p, name: p, name + "_stride": 64}))
    refused(L.bm_hip_ssm_step_dev(C.byref(d), None), "overlaps " + name)


def test_long_slot_lists_are_refused():
    L = bh.lib()
    n = (1 << 16) + 1
    refused(L.bm_hip_conv_step_dev(C.byref(conv(n_seqs=n, n_slots=n)), None), "list")
    refused(L.bm_hip_ssm_step_dev(C.byref(ssm(n_seqs=n, n_slots=n)), None), "list")
    refused(L.bm_hip_conv_dev(C.byref(conv(n_seqs=n, n_slots=n)), None), "list")
    refused(L.bm_hip_ssm_dev(C.byref(ssm(n_seqs=n, n_slots=n)), C.c_void_p(P), None), "list")


def test_calls_without_rows_need_no_addresses():
    """An empty tensor's address may be null: no prompt rows, no sequences.
    Alignment and strides are still looked at."""
    L = bh.lib()
    none = dict(x=None, y=None)
    more = dict(none, B=None, C=None, dt=None, z=None)
    assert L.bm_hip_conv_step_dev(C.byref(conv(n_seqs=0, **none)), None) == 0
    assert L.bm_hip_ssm_step_dev(C.byref(ssm(n_seqs=0, **more)), None) == 0
    assert L.bm_hip_conv_dev(C.byref(conv(n_seqs=0, n_tokens=0, **none)), None) == 0
    assert L.bm_hip_ssm_dev(C.byref(ssm(n_seqs=0, n_tokens=0, **more)), None, None) == 0
    refused(L.bm_hip_conv_dev(C.byref(conv(n_tokens=0, x=None, y=P + 2)), None), "y needs")
    refused(L.bm_hip_ssm_dev(C.byref(ssm(n_tokens=0, **dict(more, B_stride=15))), None, None), "B needs")
    if not L.bm_hip_available():  # past the checks: no GPU here
        assert L.bm_hip_conv_dev(C.byref(conv(n_tokens=0, **none)), None) == -1
        assert L.bm_hip_ssm_dev(C.byref(ssm(n_tokens=0, **more)), None, None) == -1
