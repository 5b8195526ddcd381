"""The batched recurrence between two BitLinear products, as cases that can be
timed: the short causal convolution and the selective state space scan, each
for prompts of ragged lengths and for single tokens, and the moves of the
state slots that hold what they carry from call to call.

With own = False, run() computes an operator in its plain form, elementary
torch operations in 32 bits (sums of log decays in 64); with own = True it
makes the call that a user makes of the library.  exact() is the definition
in 64 bits, token by token.
"""
import ctypes
import math
import os
import random
import sys

import torch
import torch.nn.functional as F

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPE_IDS = {"f32": 0, "bf16": 1, "f16": 2}
CHUNK = 64  # tokens per chunk of the plain scan


def listed():
    return [
        # prompts of eight requests through the convolution of a 1B-shape
        # layer (d_inner 4096, four taps), joined in one call
        dict(name="conv_1b_prompts", kind="conv", type="f32", channels=4096, width=4, seqs=8,
             tokens=4096, silu=True, bias=True, spread=1),
        # many short requests, x, B and C convolved together, an odd number of
        # channels in rows that no vector load fits
        dict(name="conv_short_odd_bf16", kind="conv", type="bf16", channels=2307, width=4,
             seqs=61, tokens=1999, silu=True, bias=True, spread=2),
        # one request, one token: latency alone
        dict(name="conv_token_1", kind="conv_step", type="f32", channels=4096, width=4, seqs=1,
             silu=True, bias=True),
        # a full serving batch, one token each
        dict(name="conv_token_512", kind="conv_step", type="bf16", channels=4352, width=4,
             seqs=512, silu=True, bias=True),
        # the first token after one long prompt at the 1B shape of bench.py:
        # a state value per channel, B, C and dt per head
        dict(name="scan_1b_1024", kind="ssm", type="f32", heads=64, head_dim=64, groups=64,
             state=1, seqs=1, tokens=1024, gate=True, spread=0),
        # sixteen ragged requests at the 255M shape, one of them empty
        dict(name="scan_255m_ragged", kind="ssm", type="f32", heads=32, head_dim=64, groups=32,
             state=1, seqs=16, tokens=6001, gate=True, spread=3),
        # ragged requests, 64 state values per channel, two groups
        dict(name="scan_n64_ragged", kind="ssm", type="f32", heads=32, head_dim=64, groups=2,
             state=64, seqs=6, tokens=3001, gate=True, spread=4),
        # one long document, 128 state values per channel, one group
        dict(name="scan_n128_long_bf16", kind="ssm", type="bf16", heads=64, head_dim=64, groups=1,
             state=128, seqs=1, tokens=16384, gate=True, spread=0),
        # one request, one token at the 1B shape: latency alone
        dict(name="token_1b_1", kind="ssm_step", type="f32", heads=64, head_dim=64, groups=64,
             state=1, seqs=1, gate=True),
        # a serving batch with 128 state values per channel: the states' bytes
        dict(name="token_n128_128", kind="ssm_step", type="bf16", heads=64, head_dim=64, groups=1,
             state=128, seqs=128, gate=True),
        # the beams of a search take over their parents' states, 24 layers of
        # the 1B shape (state and three convolution rows per channel)
        dict(name="slots_beams", kind="slots", floats=16384, layers=24, slots=256, pairs=64),
        # most sequences have ended: the others move together
        dict(name="slots_compact", kind="compact", floats=16384, layers=24, slots=512, live=200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["conv", "conv_step", "ssm", "ssm", "ssm", "ssm_step", "ssm_step", "slots",
                       "compact"])
    ty = rng.choice(["f32", "f32", "bf16", "f16"])
    if kind in ("conv", "conv_step"):
        c = dict(kind=kind, type=ty, width=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.8,
                 bias=rng.random() < 0.8,
                 channels=rng.choice([2048, 4096, 8 * _log(rng, 4, 1024), _log(rng, 1, 8192)]))
        if kind == "conv_step":
            return dict(c, seqs=_log(rng, 1, 512))
        seqs = rng.choice([1, _log(rng, 1, 100)])
        return dict(c, seqs=seqs, tokens=max(_log(rng, 1, 8192), seqs), spread=rng.randint(0, 999))
    if kind in ("ssm", "ssm_step"):
        heads = rng.choice([32, 64, _log(rng, 1, 96)])
        head_dim = rng.choice([64, 64, 32, 128, _log(rng, 3, 128)])
        if rng.random() < 0.35:
            groups, state = heads, 1
        else:
            groups = rng.choice([g for g in range(1, heads + 1) if heads % g == 0 and g <= 16])
            state = rng.choice([16, 64, 128, _log(rng, 2, 256)])
        c = dict(kind=kind, type=ty, heads=heads, head_dim=head_dim, groups=groups, state=state,
                 gate=rng.random() < 0.8)
        one = heads * head_dim * state
        if kind == "ssm_step":
            return dict(c, seqs=_log(rng, 1, max(2, min(512, 128 * 64 * 64 * 128 // one))))
        seqs = rng.choice([1, _log(rng, 1, 48)])
        most = min(16384, 16384 * 64 * 64 // (heads * head_dim), 16384 * 64 * 64 * 128 // one)
        return dict(c, seqs=seqs, tokens=max(_log(rng, 1, max(2, most // 2)), seqs),
                    spread=rng.randint(0, 999))
    floats = rng.choice([8192, 16384, _log(rng, 5, 100000)])
    layers = rng.choice([1, 24, rng.randint(1, 32)])
    slots = _log(rng, 2, max(2, min(2000, 24 * 16384 * 512 // (floats * layers))))
    if kind == "slots":
        return dict(kind=kind, floats=floats, layers=layers, slots=slots,
                    pairs=_log(rng, 1, min(slots, 256)))
    return dict(kind=kind, floats=floats, layers=layers, slots=slots,
                live=rng.randint(1, slots))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """How the tokens fall to the sequences: one at least each, except that
    the second of four or more is empty; the same for every seed."""
    n, left = case["seqs"], case["tokens"]
    r = random.Random(case["spread"])
    empty = 1 if n >= 4 else -1
    w = [0.0 if b == empty else 0.2 + r.expovariate(1.0) for b in range(n)]
    lens = [0 if b == empty else 1 for b in range(n)]
    left -= sum(lens)
    total = sum(w)
    for b in range(n):
        lens[b] += int(left * w[b] / total)
    lens[0] += case["tokens"] - sum(lens)
    return lens


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 23)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _slots(g, seqs, spare):
    """Slots as a server hands them out: any order, some free."""
    return torch.randperm(seqs + spare, generator=g, device="cuda")[:seqs].to(torch.int32)


def _ragged(s, case):
    s["lens"] = _lengths(case)
    starts = [0]
    for n in s["lens"]:
        starts.append(starts[-1] + n)
    s["start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")


def _conv_inputs(case, seed):
    g, s = _generator(seed), dict(case)
    c, w, b, dtype = case["channels"], case["width"], case["seqs"], TYPES[case["type"]]
    rows = case["tokens"] if case["kind"] == "conv" else b
    s["x"] = _randn(g, rows, c).to(dtype)
    s["w"] = _randn(g, w, c) / math.sqrt(w)
    s["b"] = 0.1 * _randn(g, c) if case["bias"] else None
    s["slot"] = _slots(g, b, 3)
    s["pool"] = _randn(g, b + 3, w - 1, c)
    s["y"] = torch.empty_like(s["x"])
    if case["kind"] == "conv":
        _ragged(s, case)
    return s


def _ssm_inputs(case, seed):
    """Activations as in_proj and the convolution leave them; steps between
    0.001 and 0.1 and decay rates between 1 and 16, as such blocks start."""
    g, s = _generator(seed), dict(case)
    h, p, gr, n, b = (case[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    dtype = TYPES[case["type"]]
    rows = case["tokens"] if case["kind"] == "ssm" else b
    s["x"] = F.silu(_randn(g, rows, h * p)).to(dtype)
    s["z"] = _randn(g, rows, h * p).to(dtype) if case["gate"] else None
    s["B"] = F.silu(_randn(g, rows, gr * n)).to(dtype)
    s["C"] = F.silu(_randn(g, rows, gr * n)).to(dtype)
    s["dt"] = (0.5 * _randn(g, rows, h)).to(dtype)
    step = torch.exp(torch.rand(h, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = torch.log(torch.expm1(step))
    s["A"] = -(1.0 + 15.0 * torch.rand(h, generator=g, device="cuda"))
    s["D"] = 1.0 + 0.1 * _randn(g, h * p)
    s["slot"] = _slots(g, b, 2)
    s["pool"] = 0.2 * _randn(g, b + 2, h * p * n)
    s["y"] = torch.empty_like(s["x"])
    if case["kind"] == "ssm":
        _ragged(s, case)
    return s


def _slot_inputs(case, seed):
    g, s = _generator(seed), dict(case)
    s["pool"] = _randn(g, case["layers"], case["slots"], case["floats"])
    order = torch.randperm(case["slots"], generator=g, device="cuda").to(torch.int32)
    if case["kind"] == "slots":
        # beams: each goes on from a parent among all of them; every eighth
        # starts anew from zeros
        n = case["pairs"]
        s["dst"] = order[:n].contiguous()
        parent = torch.randint(0, n, (n,), generator=g, device="cuda")
        s["src"] = s["dst"][parent]
        s["src"][7::8] = -1
    else:
        s["table"] = torch.cat([order[:case["live"]],
                                torch.full((5,), -1, dtype=torch.int32, device="cuda")])
        s["table"] = s["table"][torch.randperm(s["table"].numel(), generator=g, device="cuda")]
        s["table"] = s["table"].contiguous()
        s["new"] = torch.empty_like(s["table"])
        s["count"] = torch.empty(1, dtype=torch.int32, device="cuda")
    return s


def _inputs(case, seed):
    if case["kind"] in ("conv", "conv_step"):
        return _conv_inputs(case, seed)
    return _ssm_inputs(case, seed) if case["kind"] in ("ssm", "ssm_step") else _slot_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["call"] = _call(s)  # the descriptor and workspace that a program keeps
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _library():
    path = os.path.join(os.getcwd(), "bitmamba.c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bitmamba_hip
    if not bitmamba_hip.lib().bm_hip_init():
        raise RuntimeError(bitmamba_hip.last_error())
    return bitmamba_hip


def _at(t):
    return None if t is None else t.data_ptr()


def _call(s):
    """The call of a pass, ready to be made, on the library's stream."""
    bh = _library()
    lib, kind = bh.lib(), s["kind"]
    if kind in ("conv", "conv_step"):
        c = s["channels"]
        d = bh.Conv(type=TYPE_IDS[s["type"]], channels=c, width=s["width"], silu=int(s["silu"]),
                    n_seqs=s["seqs"], n_tokens=s["x"].shape[0], seq_start=_at(s.get("start")),
                    slots=_at(s["slot"]), x=_at(s["x"]), x_stride=c, w=_at(s["w"]),
                    bias=_at(s["b"]), state=_at(s["pool"]), n_slots=s["pool"].shape[0],
                    state_stride=s["pool"].stride(0), y=_at(s["y"]), y_stride=c)
        f, d = (lib.bm_hip_conv_dev if kind == "conv" else lib.bm_hip_conv_step_dev), ctypes.byref(d)
        return lambda: bh.check(f(d, None), "conv")
    if kind in ("ssm", "ssm_step"):
        hp, gn = s["x"].shape[1], s["B"].shape[1]
        d = bh.Ssm(type=TYPE_IDS[s["type"]], n_heads=s["heads"], head_dim=s["head_dim"],
                   n_groups=s["groups"], d_state=s["state"], dt_softplus=1, n_seqs=s["seqs"],
                   n_tokens=s["x"].shape[0], seq_start=_at(s.get("start")), slots=_at(s["slot"]),
                   x=_at(s["x"]), x_stride=hp, B=_at(s["B"]), B_stride=gn, C=_at(s["C"]),
                   C_stride=gn, dt=_at(s["dt"]), dt_stride=s["heads"], z=_at(s["z"]), z_stride=hp,
                   A=_at(s["A"]), dt_bias=_at(s["dt_bias"]), D=_at(s["D"]), state=_at(s["pool"]),
                   n_slots=s["pool"].shape[0], state_stride=s["pool"].stride(0), y=_at(s["y"]),
                   y_stride=hp)
        r = ctypes.byref(d)
        if kind == "ssm_step":
            f = lib.bm_hip_ssm_step_dev
            return lambda: bh.check(f(r, None), "ssm_step")
        s["work"] = torch.empty(lib.bm_hip_ssm_workspace_bytes(r), dtype=torch.uint8, device="cuda")
        f, w = lib.bm_hip_ssm_dev, _at(s["work"])
        return lambda: bh.check(f(r, w, None), "ssm")
    layers, slots, floats = s["pool"].shape
    d = bh.Slots(base=_at(s["pool"]), n_slots=slots, n_layers=layers, slot_bytes=4 * floats,
                 slot_stride=4 * floats, layer_stride=4 * floats * slots)
    r = ctypes.byref(d)
    if kind == "slots":
        f, src, dst, n = lib.bm_hip_slots_copy_dev, _at(s["src"]), _at(s["dst"]), s["pairs"]
        return lambda: bh.check(f(r, 1, src, dst, n, None), "slots_copy")
    s["work"] = torch.empty(lib.bm_hip_slots_compact_workspace_bytes(slots), dtype=torch.uint8,
                            device="cuda")
    f, n, w = lib.bm_hip_slots_compact_dev, s["table"].numel(), _at(s["work"])
    table, new, count = _at(s["table"]), _at(s["new"]), _at(s["count"])
    return lambda: bh.check(f(r, 1, table, new, n, count, w, None), "slots_compact")


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _conv_plain(s):
    """Every token's window of taps, rows of the sequence's state before its
    first tokens, as one gather; then products and a sum."""
    w, slot, pool = s["width"], s["slot"].long(), s["pool"]
    if s["kind"] == "conv":
        start = s["start"].long()
        rows = torch.arange(s["x"].shape[0], device="cuda")
        seq = torch.searchsorted(start[1:].contiguous(), rows, right=True)
        ends = start[1:]
    else:
        rows = torch.arange(s["seqs"], device="cuda")
        seq, ends = rows, rows + 1
    b = torch.arange(s["seqs"], device="cuda")
    # each sequence's rows stand behind its w - 1 state rows
    at = rows + (w - 1) * (seq + 1)
    first = (ends - torch.bincount(seq, minlength=s["seqs"])) + (w - 1) * b
    tap = torch.arange(w, device="cuda")
    ext = torch.empty((rows.numel() + (w - 1) * s["seqs"], s["channels"]), device="cuda")
    ext[first[:, None] + tap[:w - 1]] = pool[slot]
    ext[at] = s["x"].float()
    y = (ext[at[:, None] - (w - 1) + tap] * s["w"]).sum(1)
    if s["b"] is not None:
        y = y + s["b"]
    if s["silu"]:
        y = y / (1.0 + torch.exp(-y))
    s["y"].copy_(y)
    pool[slot] = ext[(ends + (w - 1) * b)[:, None] + tap[:w - 1]]
    return {"y": s["y"], "state": pool}


def _steps(s, dt):
    """softplus(dt + bias), its exponential taken where it cannot overflow."""
    v = dt.float() + s["dt_bias"]
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _gated(s, y, x, z):
    y = y + s["D"] * x
    return y if z is None else y * z / (1.0 + torch.exp(-z))


def _step_plain(s):
    h, p, g, n, b = (s[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    slot, pool = s["slot"].long(), s["pool"]
    d = _steps(s, s["dt"])
    x = s["x"].float().view(b, h, p)
    bb = s["B"].float().view(b, g, 1, n).expand(b, g, h // g, n).reshape(b, h, 1, n)
    cc = s["C"].float().view(b, g, 1, n).expand(b, g, h // g, n).reshape(b, h, 1, n)
    st = pool[slot].view(b, h, p, n)
    st = st * torch.exp(s["A"] * d)[:, :, None, None] + (d[:, :, None] * x)[..., None] * bb
    y = (st * cc).sum(-1).view(b, h * p)
    z = None if s["z"] is None else s["z"].float()
    s["y"].copy_(_gated(s, y, s["x"].float(), z))
    pool[slot] = st.view(b, h * p * n)
    return {"y": s["y"], "state": pool}


def _scan_plain(s):
    """Chunks of tokens: products of C and B weighted by the decay between two
    tokens, and a state per chunk, joined over the chunks by the decay between
    two chunks.  Sequences are padded with steps of zero, which change nothing."""
    h, p, g, n, b = (s[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    q, dev = CHUNK, "cuda"
    nc = max(1, -(-max(s["lens"]) // q))
    start, slot, pool = s["start"].long(), s["slot"].long(), s["pool"]
    pos = torch.arange(nc * q, device=dev)
    inside = pos < (start[1:] - start[:-1])[:, None]
    row = torch.where(inside, start[:-1, None] + pos, 0)
    d = _steps(s, s["dt"])[row] * inside[..., None]
    xx = s["x"].float()
    # chunks by head: [b, nc, h, q, ...]
    x = xx[row].view(b, nc, q, h, p).transpose(2, 3).contiguous()
    bb = s["B"].float()[row].view(b, nc, q, g, n).transpose(2, 3).contiguous()
    cc = s["C"].float()[row].view(b, nc, q, g, n).transpose(2, 3).contiguous()
    d = d.view(b, nc, q, h).transpose(2, 3).contiguous()
    cum = torch.cumsum(d.double() * s["A"].double()[:, None], -1)
    later = torch.ones((q, q), dtype=torch.bool, device=dev).triu(1)
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(later, -math.inf)).float()
    cb = torch.matmul(cc, bb.transpose(-1, -2).contiguous())
    cb = cb[:, :, :, None].expand(b, nc, g, h // g, q, q).reshape(b, nc, h, q, q)
    dx = d[..., None] * x
    y = torch.matmul(cb * decay, dx)
    # what each chunk adds to the state, [b, nc, h, n, p], after the sequence's own
    left = torch.exp(cum[..., -1:] - cum).float()
    bh = bb[:, :, :, None].expand(b, nc, g, h // g, q, n).reshape(b, nc, h, q, n)
    ch = cc[:, :, :, None].expand(b, nc, g, h // g, q, n).reshape(b, nc, h, q, n)
    add = torch.matmul((bh * left[..., None]).transpose(-1, -2).contiguous(), dx)
    init = pool[slot].view(b, 1, h, p, n).transpose(-1, -2)
    add = torch.cat([init, add], 1).transpose(1, 2).reshape(b, h, nc + 1, n * p)
    # between chunks: state i before chunk i is sum_j<=i decay(j..i) add_j
    tot = torch.cumsum(F.pad(cum[..., -1].transpose(1, 2), (1, 0)), -1)
    far = torch.ones((nc + 1, nc + 1), dtype=torch.bool, device=dev).triu(1)
    over = torch.exp((tot[..., :, None] - tot[..., None, :]).masked_fill(far, -math.inf)).float()
    st = torch.matmul(over, add).view(b, h, nc + 1, n, p).transpose(1, 2)
    y = y + torch.matmul(ch, st[:, :nc].contiguous()) * torch.exp(cum).float()[..., None]
    y = y.transpose(2, 3).reshape(b, nc * q, h * p)[inside]
    z = None if s["z"] is None else s["z"].float()
    s["y"].copy_(_gated(s, y, xx, z))
    pool[slot] = st[:, nc].transpose(-1, -2).reshape(b, h * p * n)
    return {"y": s["y"], "state": pool}


def _slots_plain(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["pool"][:, dst] = s["pool"][:, src.clamp(min=0)] * (src >= 0).float()[:, None]
    return s["pool"]


def _compact_plain(s):
    """Live slots at or above the count of live ones go, in order, to the free
    ones below it."""
    table, slots = s["table"].long(), s["slots"]
    mark = torch.zeros(slots + 1, dtype=torch.int64, device="cuda")
    mark[torch.where(table < 0, slots, table)] = 1
    mark = mark[:slots]
    count = mark.sum()
    at = torch.arange(slots, device="cuda")
    free = torch.argsort(torch.where((mark == 0) & (at < count), at, at + slots))
    rank = torch.cumsum(mark * (at >= count), 0) - 1
    moves = (mark == 1) & (at >= count)
    to = torch.where(moves, free[rank.clamp(min=0)], at)
    # a slot that nothing moves to keeps what it holds
    new = torch.where(table < 0, table, to[table.clamp(min=0)])
    come = torch.cat([at, at[:1]]).scatter_(0, torch.where(moves, to, slots), at)[:slots]
    s["pool"].copy_(s["pool"][:, come])
    s["new"].copy_(new)
    s["count"].copy_(count.view(1))
    return {"pool": s["pool"], "new": s["new"], "count": s["count"]}


PLAIN = {"conv": _conv_plain, "conv_step": _conv_plain, "ssm": _scan_plain,
         "ssm_step": _step_plain, "slots": _slots_plain, "compact": _compact_plain}


def run(s):
    if not own:
        return PLAIN[s["kind"]](s)
    s["call"]()
    if s["kind"] == "slots":
        return s["pool"]
    if s["kind"] == "compact":
        return {"pool": s["pool"], "new": s["new"], "count": s["count"]}
    return {"y": s["y"], "state": s["pool"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("slots", "compact"):
        size = 4 * case["floats"] * case["layers"]
        if kind == "slots":
            n = case["pairs"]
            # an eighth of the slots written is cleared; parents read once
            parents = (n - n // 8) * 0.63
            return {"bytes": int(size * (n + parents) + 8 * n), "flops": 0}
        # every live slot beyond the count of live ones moves (the expectation)
        moves = case["live"] * (case["slots"] - case["live"]) / case["slots"]
        return {"bytes": int(2 * size * moves + 8 * case["live"] + 64), "flops": 0}
    size = 4 if case["type"] == "f32" else 2
    b = case["seqs"]
    if kind in ("conv", "conv_step"):
        c, w = case["channels"], case["width"]
        rows = case["tokens"] if kind == "conv" else b
        byt = 2 * rows * c * size + 4 * (w + 1) * c + 2 * 4 * b * (w - 1) * c
        return {"bytes": byt, "flops": rows * c * (2 * w + 4)}
    h, p, g, n = (case[k] for k in ("heads", "head_dim", "groups", "state"))
    rows = case["tokens"] if kind == "ssm" else b
    byt = rows * size * ((3 if case["gate"] else 2) * h * p + 2 * g * n + h)
    byt += 2 * 4 * b * h * p * n + 4 * (2 * h + h * p)
    return {"bytes": byt, "flops": rows * h * p * (5 * n + 6)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _conv_exact(s):
    pool, out = s["pool"].double(), []
    w, lens = s["w"].double(), s.get("lens") or [1] * s["seqs"]
    at = 0
    for b, n in enumerate(lens):
        slot = int(s["slot"][b])
        rows = torch.cat([pool[slot], s["x"][at:at + n].double()])
        y = sum(w[k] * rows[k:k + n] for k in range(s["width"]))
        y = y if s["b"] is None else y + s["b"].double()
        out.append(y * torch.sigmoid(y) if s["silu"] else y)
        pool[slot] = rows[n:]
        at += n
    return {"y": torch.cat(out), "state": pool}


def _ssm_exact(s):
    """The recurrence, one token of every sequence at a time."""
    h, p, g, n, b = (s[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    lens = s.get("lens") or [1] * b
    start = [sum(lens[:k]) for k in range(b)]
    x, bb, cc = s["x"].double().view(-1, h, p), s["B"].double().view(-1, g, n), s["C"].double().view(-1, g, n)
    step = F.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=1e9)
    decay = torch.exp(step * s["A"].double())
    pool = s["pool"].double().view(-1, h, p, n)
    y = torch.empty((x.shape[0], h, p), dtype=torch.float64, device="cuda")
    # the longest sequences first, so that those still running come first
    order = sorted(range(b), key=lambda k: -lens[k])
    slots = s["slot"].long()[torch.tensor(order, device="cuda")]
    state = pool[slots]
    base = torch.tensor([start[k] for k in order], device="cuda")
    for t in range(max(lens)):
        m = sum(lens[k] > t for k in order)
        r = base[:m] + t
        inp = (step[r][..., None] * x[r]).view(m, g, h // g, p, 1) * bb[r].view(m, g, 1, 1, n)
        state[:m] = state[:m] * decay[r][..., None, None] + inp.view(m, h, p, n)
        st = state[:m].view(m, g, (h // g) * p, n)
        y[r] = torch.matmul(st, cc[r].unsqueeze(-1)).view(m, h, p)
    pool[slots] = state
    y = y.view(-1, h * p) + s["D"].double() * s["x"].double()
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    return {"y": y, "state": pool.view(pool.shape[0], -1)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("conv", "conv_step"):
        return _conv_exact(s)
    if case["kind"] in ("ssm", "ssm_step"):
        return _ssm_exact(s)
    return None  # values are moved, none computed
