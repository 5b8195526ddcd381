"""The gated delta rule for many sequences, and the verification of drafted
tokens, as cases that can be timed: the rule for prompts of ragged lengths,
for the few drafted tokens of each sequence that are scored against states
that stay as they are, and for single tokens; the verification of ragged
drafts against the target's distributions, with the token that follows.

With own = False, run() computes an operator in its plain form, elementary
torch operations in 32 bits (log decays, the inverses of triangular matrices
and probabilities in 64); with own = True it makes the call that a user makes
of the library.  exact() is the definition in 64 bits, token by token.
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
CHUNK = 64  # tokens per chunk of the plain form
EPS = 1e-6  # beside the squares of a row of q or k


def listed():
    return [
        # one long document through a layer of 32 heads of 128, pairs of heads
        # with the same q and k
        dict(name="delta_long_bf16", kind="delta", type="bf16", heads=32, head_dim=128, groups=16,
             state=128, seqs=1, tokens=16384, gate=True, spread=0),
        # the prompt that comes before the first token, all in fp32
        dict(name="delta_prompt_1024_f32", kind="delta", type="f32", heads=32, head_dim=128,
             groups=32, state=128, seqs=1, tokens=1024, gate=True, spread=0),
        # sixteen ragged requests at 32 heads of 64, one of them empty
        dict(name="delta_ragged_bf16", kind="delta", type="bf16", heads=32, head_dim=64,
             groups=32, state=64, seqs=16, tokens=6001, gate=True, spread=3),
        # sizes that fit no tile, no gate
        dict(name="delta_odd_f16", kind="delta", type="f16", heads=6, head_dim=80, groups=3,
             state=100, seqs=9, tokens=1999, gate=False, spread=5),
        # four drafted tokens of each of 64 requests, and the one before them,
        # scored without touching the requests' states
        dict(name="delta_drafts_64", kind="delta_score", type="bf16", heads=32, head_dim=128,
             groups=16, state=128, seqs=64, tokens=320, gate=True, spread=0),
        # one request, one token: latency alone
        dict(name="delta_token_1", kind="delta_step", type="f32", heads=32, head_dim=128,
             groups=16, state=128, seqs=1, gate=True),
        # a serving batch, one token each: the states' bytes
        dict(name="delta_token_128", kind="delta_step", type="bf16", heads=32, head_dim=128,
             groups=16, state=128, seqs=128, gate=True),
        # one request with four drafted tokens, a draft model's logits: latency
        dict(name="verify_one_f32", kind="verify", type="f32", vocab=50257, seqs=1, drafts=4,
             ragged=False, draft="logits", weights=False, temp=0.8125, spread=0),
        # a serving batch with drafts of uneven lengths, probabilities of a
        # draft model's own sampler
        dict(name="verify_batch_bf16", kind="verify", type="bf16", vocab=50257, seqs=64, drafts=7,
             ragged=True, draft="weights", weights=False, temp=1.0, spread=1),
        # drafts looked up in the text so far: nothing but the tokens; the
        # target's probabilities as a filter left them
        dict(name="verify_lookup_f32", kind="verify", type="f32", vocab=32000, seqs=16, drafts=15,
             ragged=True, draft="none", weights=True, temp=1.0, spread=2),
        # greedy decoding of many requests
        dict(name="verify_greedy_f16", kind="verify", type="f16", vocab=50257, seqs=256, drafts=4,
             ragged=False, draft="none", weights=False, temp=0.0, spread=3),
        # the largest vocabulary that the sampler takes
        dict(name="verify_wide_f32", kind="verify", type="f32", vocab=256000, seqs=32, drafts=7,
             ragged=False, draft="logits", weights=False, temp=0.6875, spread=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "delta_score", "delta_step", "delta_step",
                       "verify", "verify", "verify"])
    ty = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "verify":
        vocab = rng.choice([50257, 32000, _log(rng, 50, 256000), _log(rng, 1000, 256000)])
        drafts = rng.choice([4, rng.randint(0, 15)])
        most = 32 * 8 * 256000 // (vocab * (drafts + 1))
        return dict(kind=kind, type=ty, vocab=vocab, seqs=_log(rng, 1, max(2, min(512, most))),
                    drafts=drafts, ragged=rng.random() < 0.6,
                    draft=rng.choice(["logits", "weights", "none"]), weights=rng.random() < 0.25,
                    temp=rng.choice([0.0, 1.0, rng.randint(5, 24) / 16]),
                    spread=rng.randint(0, 999))
    heads = rng.choice([16, 32, _log(rng, 1, 64)])
    head_dim = rng.choice([64, 128, 128, _log(rng, 5, 192)])
    groups = rng.choice([g for g in range(1, heads + 1) if heads % g == 0])
    state = rng.choice([64, 128, 128, _log(rng, 4, 256)])
    c = dict(kind=kind, type=ty, heads=heads, head_dim=head_dim, groups=groups, state=state,
             gate=rng.random() < 0.8)
    one = heads * head_dim * state
    full = 32 * 128 * 128
    if kind == "delta_step":
        return dict(c, seqs=_log(rng, 1, max(2, min(512, 128 * full // one))))
    if kind == "delta_score":
        seqs = _log(rng, 1, max(2, min(256, 64 * full // one)))
        return dict(c, seqs=seqs, tokens=seqs * rng.randint(1, 9), spread=0)
    seqs = rng.choice([1, _log(rng, 1, 48)])
    most = min(16384, 8192 * full // one, 8192 * 64 // heads)
    return dict(c, seqs=seqs, tokens=max(_log(rng, 1, max(2, most)), seqs),
                spread=rng.randint(0, 999))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """How the tokens fall to the sequences, the same for every seed: evenly
    where they are drafts; else unevenly, one at least each, except that the
    second of four or more is empty."""
    n, left = case["seqs"], case["tokens"]
    if case["kind"] == "delta_score":
        return [left // n] * n
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


def _drafts(case):
    """Rows of each sequence: its drafted tokens and one more."""
    r = random.Random(case["spread"])
    return [1 + (r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"])
            for _ in range(case["seqs"])]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 6007 + 41)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _starts(lens):
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _delta_inputs(case, seed):
    """q, k and v as a convolution with silu leaves them; steps between 0.001
    and 0.1 and decay rates between 1 and 16, as such layers start."""
    g, s = _generator(seed), dict(case)
    h, p, gr, n, b = (case[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    dtype = TYPES[case["type"]]
    rows = b if case["kind"] == "delta_step" else case["tokens"]
    s["q"] = F.silu(_randn(g, rows, gr * n)).to(dtype)
    s["k"] = F.silu(_randn(g, rows, gr * n)).to(dtype)
    s["v"] = F.silu(_randn(g, rows, h * p)).to(dtype)
    s["z"] = _randn(g, rows, h * p).to(dtype) if case["gate"] else None
    s["beta"] = _randn(g, rows, h).to(dtype)
    s["dt"] = (0.5 * _randn(g, rows, h)).to(dtype)
    step = torch.exp(torch.rand(h, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = torch.log(torch.expm1(step))
    s["A"] = -(1.0 + 15.0 * torch.rand(h, generator=g, device="cuda"))
    s["scale"] = n ** -0.5
    s["slot"] = torch.randperm(b + 2, generator=g, device="cuda")[:b].to(torch.int32)
    s["pool"] = 0.2 * _randn(g, b + 2, h * p * n)
    s["y"] = torch.empty_like(s["v"])
    if case["kind"] != "delta_step":
        s["lens"] = _lengths(case)
        s["start"] = _starts(s["lens"])
    return s


def _verify_inputs(case, seed):
    """A target's logits, a draft model's that are near them, and tokens drawn
    from the draft's."""
    g, s = _generator(seed), dict(case)
    v, dtype = case["vocab"], TYPES[case["type"]]
    s["lens"] = _drafts(case)
    s["start"] = _starts(s["lens"])
    rows = sum(s["lens"])
    target = 3.0 * _randn(g, rows, v)
    draft = target + 0.8 * _randn(g, rows, v)
    heat = 1.0 / max(case["temp"], 0.3)
    noise = -torch.log(torch.rand(rows, v, generator=g, device="cuda").clamp_(min=1e-30))
    s["tokens"] = torch.argmax(draft * heat - torch.log(noise), -1).to(torch.int32)
    if case["weights"]:
        target = torch.softmax(target * heat, -1)
    s["target"] = target.to(dtype)
    s["q"] = None
    if case["draft"] == "logits":
        s["q"] = draft.to(dtype)
    elif case["draft"] == "weights":
        s["q"] = torch.softmax(draft * heat, -1).to(dtype)
    s["u"] = torch.rand(rows, generator=g, device="cuda")
    b = case["seqs"]
    s["accepted"] = torch.empty(b, dtype=torch.int32, device="cuda")
    s["next"] = torch.empty(b, dtype=torch.int32, device="cuda")
    s["ratio"] = torch.zeros(rows, device="cuda")
    s["split"] = torch.empty(2 * b + 1, dtype=torch.int32, device="cuda")
    return s


def _inputs(case, seed):
    return _verify_inputs(case, seed) if case["kind"] == "verify" else _delta_inputs(case, seed)


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
    if kind == "verify":
        v = s["vocab"]
        d = bh.Verify(type=TYPE_IDS[s["type"]], vocab=v, n_seqs=s["seqs"],
                      n_rows=s["target"].shape[0], row_start=_at(s["start"]),
                      target=_at(s["target"]), target_stride=v, target_weights=int(s["weights"]),
                      draft=_at(s["q"]), draft_stride=v,
                      draft_weights=int(s["draft"] == "weights"), temp=s["temp"],
                      tokens=_at(s["tokens"]), u=_at(s["u"]), n_accepted=_at(s["accepted"]),
                      next_token=_at(s["next"]), ratio=_at(s["ratio"]),
                      split_start=_at(s["split"]))
        size, f = lib.bm_hip_verify_workspace_bytes, lib.bm_hip_verify_dev
    else:
        hp, gn, h = s["v"].shape[1], s["q"].shape[1], s["heads"]
        d = bh.Delta(type=TYPE_IDS[s["type"]], n_heads=h, head_dim=s["head_dim"],
                     n_groups=s["groups"], d_state=s["state"], dt_softplus=1, beta_sigmoid=1,
                     qk_norm=1, frozen=int(kind == "delta_score"), norm_eps=EPS, scale=s["scale"],
                     n_seqs=s["seqs"], n_tokens=s["v"].shape[0], seq_start=_at(s.get("start")),
                     slots=_at(s["slot"]), q=_at(s["q"]), q_stride=gn, k=_at(s["k"]), k_stride=gn,
                     v=_at(s["v"]), v_stride=hp, dt=_at(s["dt"]), dt_stride=h,
                     beta=_at(s["beta"]), beta_stride=h, z=_at(s["z"]), z_stride=hp,
                     A=_at(s["A"]), dt_bias=_at(s["dt_bias"]), state=_at(s["pool"]),
                     n_slots=s["pool"].shape[0], state_stride=s["pool"].stride(0), y=_at(s["y"]),
                     y_stride=hp)
        if kind == "delta_step":
            r, f = ctypes.byref(d), lib.bm_hip_delta_step_dev
            return lambda: bh.check(f(r, None), "delta_step")
        size, f = lib.bm_hip_delta_workspace_bytes, lib.bm_hip_delta_dev
    r = ctypes.byref(d)
    s["work"] = torch.empty(size(r), dtype=torch.uint8, device="cuda")
    w = _at(s["work"]) if s["work"].numel() else None
    return lambda: bh.check(f(r, w, None), kind)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _rates(s):
    """The log decay of every row and head in 64 bits, and its beta."""
    v = s["dt"].float() + s["dt_bias"]
    step = torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))
    return s["A"].double() * step.double(), 1.0 / (1.0 + torch.exp(-s["beta"].float()))


def _unit(t, heads):
    """Rows [.., groups, n] over their length, for every head of a group."""
    t = t * torch.rsqrt((t * t).sum(-1, keepdim=True) + EPS)
    return t.repeat_interleave(heads // t.shape[-2], -2)


def _outputs(s, y):
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1.0 + torch.exp(-z))
    s["y"].copy_(y)
    return s["y"] if s["kind"] == "delta_score" else {"y": s["y"], "state": s["pool"]}


def _step_plain(s):
    h, p, n, b = (s[k] for k in ("heads", "head_dim", "state", "seqs"))
    slot, pool = s["slot"].long(), s["pool"]
    log_decay, beta = _rates(s)
    q, k = (_unit(s[t].float().view(b, -1, n), h) for t in "qk")
    st = pool[slot].view(b, h, p, n) * torch.exp(log_decay).float()[..., None, None]
    miss = s["v"].float().view(b, h, p) - (st * k[:, :, None]).sum(-1)
    st = st + (beta[..., None] * miss)[..., None] * k[:, :, None]
    y = s["scale"] * (st * q[:, :, None]).sum(-1)
    pool[slot] = st.view(b, -1)
    return _outputs(s, y.view(b, -1))


def _inverse(low):
    """(I + low)^-1 of strictly lower triangular matrices [.., 64, 64]: blocks
    of 16 as products, since their powers end, then pairs of blocks."""
    n, size = low.shape[-1], 16
    blocks = low.unflatten(-1, (-1, size)).unflatten(-3, (-1, size))  # [.., i, 16, j, 16]
    power = -torch.diagonal(blocks, 0, -4, -2).movedim(-1, -3).contiguous()
    eye = torch.eye(size, dtype=low.dtype, device=low.device)
    inv = eye + power
    for _ in range(3):
        power = torch.matmul(power, power)
        inv = inv + torch.matmul(inv, power)
    while size < n:
        blocks = low.unflatten(-1, (-1, size)).unflatten(-3, (-1, size))
        below = torch.diagonal(blocks, -1, -4, -2).movedim(-1, -3)[..., ::2, :, :].contiguous()
        a, b = inv[..., ::2, :, :].contiguous(), inv[..., 1::2, :, :].contiguous()
        below = -torch.matmul(torch.matmul(b, below), a)
        inv = torch.cat([F.pad(a, (0, size)), torch.cat([below, b], -1)], -2)
        size *= 2
    return inv[..., 0, :, :]


def _delta_plain(s):
    """Chunks of tokens.  With c the sums of log decays within a chunk and S
    the state before it, what the rows write, w, solves
    w_i + beta_i sum_{j<i} e^{c_i - c_j} (k_i . k_j) w_j = beta_i (v_i - e^{c_i} k_i S):
    one triangular inverse per chunk and head, then a product per chunk in
    turn.  Sequences are padded with rows of zeros, which change nothing."""
    h, p, n, b = (s[k] for k in ("heads", "head_dim", "state", "seqs"))
    q0, dev = CHUNK, "cuda"
    nc = max(1, -(-max(s["lens"]) // q0))
    start, slot, pool = s["start"].long(), s["slot"].long(), s["pool"]
    pos = torch.arange(nc * q0, device=dev)
    inside = pos < (start[1:] - start[:-1])[:, None]
    row = torch.where(inside, start[:-1, None] + pos, 0)

    def chunks(t):  # [rows, h, ..] to [b, nc, h, 64, ..]
        t = t[row] * inside.view(inside.shape + (1,) * (t.dim() - 1))
        return t.view((b, nc, q0) + t.shape[2:]).transpose(2, 3).contiguous()

    log_decay, beta = (chunks(t) for t in _rates(s))
    q, k = (chunks(_unit(s[t].float().view(-1, s["groups"], n), h)) for t in "qk")
    v = chunks(s["v"].float().view(-1, h, p))
    cum = torch.cumsum(log_decay, -1)
    later = torch.ones((q0, q0), dtype=torch.bool, device=dev).triu(1)
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(later, -math.inf)).float()
    kt = k.transpose(-1, -2).contiguous()
    low = (beta[..., None] * torch.matmul(k, kt) * decay).tril(-1)
    inv = _inverse(low.double()).float()
    del low
    gain = torch.exp(cum).float()[..., None]
    writes = torch.matmul(inv, beta[..., None] * v)  # of a chunk that starts from zeros
    reads = torch.matmul(inv, beta[..., None] * gain * k)
    del inv
    left = torch.exp(cum[..., -1:] - cum).float()
    kt = kt * left[..., None, :]
    whole = torch.exp(cum[..., -1]).float()[..., None, None]
    st = pool[slot].view(b, h, p, n).transpose(-1, -2).contiguous()
    states, ws = [], []
    for c in range(nc):
        states.append(st)
        ws.append(writes[:, c] - torch.matmul(reads[:, c], st))
        st = st * whole[:, c] + torch.matmul(kt[:, c], ws[-1])
    del writes, reads
    y = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay, torch.stack(ws, 1))
    y = s["scale"] * (y + gain * torch.matmul(q, torch.stack(states, 1)))
    if s["kind"] == "delta":
        pool[slot] = st.transpose(-1, -2).reshape(b, -1)
    return _outputs(s, y.transpose(2, 3).reshape(b, nc * q0, h * p)[inside])


def _share(rows, weights, temp):
    """A row's probabilities in 64 bits; below a temperature of 0.05 all of it
    is at the largest logit, the first of equal ones."""
    if weights:
        w = rows.double()
        return w / w.sum(-1, keepdim=True)
    top = rows.max(-1, keepdim=True).values
    if temp < 0.05:
        at = torch.arange(rows.shape[-1], device=rows.device)
        best = torch.where(rows == top, at, rows.shape[-1]).min(-1, keepdim=True).values
        return (at == best).double()
    w = torch.exp((rows.double() - top.double()) * (1.0 / temp))
    return w / w.sum(-1, keepdim=True)


def _verify_plain(s):
    """Probabilities of all rows, a test per drafted token, then the token
    that follows from what the draft left of the first refused row."""
    dev, start = "cuda", s["start"].long()
    rows = torch.arange(s["target"].shape[0], device=dev)
    seq = torch.searchsorted(start[1:].contiguous(), rows, right=True)
    last = start[1:][seq] - 1
    token = s["tokens"].long()[:, None]
    p = _share(s["target"], s["weights"], s["temp"])
    if s["q"] is None:
        q = (torch.arange(s["vocab"], device=dev) == token).double()
    else:
        q = _share(s["q"], s["draft"] == "weights", s["temp"])
    pd, qd = (t.gather(1, token)[:, 0] for t in (p, q))
    ok = s["u"].double() * qd < pd
    s["ratio"].copy_(torch.where((rows < last) & (pd > 0.0), torch.clamp(pd / qd, max=1.0), 0.0))
    # the first row of a sequence that is refused, or its last
    stop = torch.where(ok & (rows < last), rows.numel(), rows)
    stop = torch.full((s["seqs"],), rows.numel(), device=dev).scatter_reduce(0, seq, stop, "amin")
    s["accepted"].copy_(stop - start[:-1])
    w = torch.where((stop == last[stop])[:, None], p[stop], torch.clamp(p[stop] - q[stop], min=0.0))
    w = torch.where(w.sum(-1, keepdim=True) == 0.0, p[stop], w)
    cum = torch.cumsum(w, -1)
    s["next"].copy_((cum <= (s["u"].double()[last[stop]] * cum[:, -1])[:, None]).sum(-1))
    s["split"][0::2] = s["start"]
    s["split"][1::2] = stop + 1
    return _verified(s)


def _verified(s):
    return {k: s[k] for k in ("accepted", "next", "ratio", "split")}


PLAIN = {"delta": _delta_plain, "delta_score": _delta_plain, "delta_step": _step_plain,
         "verify": _verify_plain}


def run(s):
    if not own:
        return PLAIN[s["kind"]](s)
    s["call"]()
    if s["kind"] == "verify":
        return _verified(s)
    return s["y"] if s["kind"] == "delta_score" else {"y": s["y"], "state": s["pool"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    b = case["seqs"]
    if case["kind"] == "verify":
        rows, v = sum(_drafts(case)), case["vocab"]
        # every row for its sum; of the draft no row of a sequence's last
        # token, and nothing where the target's largest logit decides
        greedy = case["temp"] < 0.05 and not case["weights"]
        drawn = 0 if case["draft"] == "none" or greedy else rows - b
        return {"bytes": (rows + drawn) * v * size + 12 * rows + 16 * b, "flops": 4 * (rows + drawn) * v}
    h, p, g, n = (case[k] for k in ("heads", "head_dim", "groups", "state"))
    rows = b if case["kind"] == "delta_step" else case["tokens"]
    byt = rows * size * ((3 if case["gate"] else 2) * h * p + 2 * g * n + 2 * h)
    byt += (1 if case["kind"] == "delta_score" else 2) * 4 * b * h * p * n + 8 * h
    return {"bytes": byt, "flops": rows * h * p * (7 * n + 6)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _delta_exact(s):
    """The recurrence, one token of every sequence at a time."""
    h, p, g, n, b = (s[k] for k in ("heads", "head_dim", "groups", "state", "seqs"))
    lens = s.get("lens") or [1] * b
    start = [sum(lens[:k]) for k in range(b)]
    q, k = (s[t].double().view(-1, g, n) for t in "qk")
    q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS) for t in (q, k))
    v = s["v"].double().view(-1, h, p)
    decay = torch.exp(F.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=1e9)
                      * s["A"].double())
    beta = torch.sigmoid(s["beta"].double())
    pool = s["pool"].double().view(-1, h, p, n)
    y = torch.empty_like(v)
    # the longest sequences first, so that those still running come first
    order = sorted(range(b), key=lambda k: -lens[k])
    slots = s["slot"].long()[torch.tensor(order, device="cuda")]
    state = pool[slots].view(b, g, -1, n)
    base = torch.tensor([start[k] for k in order], device="cuda")
    for t in range(max(lens)):
        m = sum(lens[k] > t for k in order)
        r = base[:m] + t
        kr = k[r].unsqueeze(-1)
        st = (state[:m].view(m, h, p * n) * decay[r][..., None]).view(m, g, -1, n)
        miss = v[r].view(m, g, -1) - torch.matmul(st, kr)[..., 0]
        w = (beta[r][..., None] * miss.view(m, h, p)).view(m, g, -1, 1)
        st = st + w * kr.transpose(-1, -2)
        y[r] = s["scale"] * torch.matmul(st, q[r].unsqueeze(-1)).view(m, h, p)
        state[:m] = st
    pool[slots] = state.view(b, h, p, n)
    y = y.view(-1, h * p)
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    return y if s["kind"] == "delta_score" else {"y": y, "state": pool.view(pool.shape[0], -1)}


def _verify_exact(s):
    """A sequence at a time."""
    accepted, following, split, row = [], [], [0], 0
    ratio = torch.zeros(s["ratio"].shape[0], dtype=torch.float64, device="cuda")
    tokens, u = s["tokens"].tolist(), s["u"].tolist()

    def distribution(r, is_draft):
        w = torch.zeros(s["vocab"], dtype=torch.float64, device="cuda")
        if is_draft and s["q"] is None:
            w[tokens[r]] = 1.0
            return w
        row = (s["q"] if is_draft else s["target"])[r].double()
        if s["draft"] == "weights" if is_draft else s["weights"]:
            return row / row.sum()
        if s["temp"] < 0.05:
            w[int((row == row.max()).nonzero()[0])] = 1.0
            return w
        return torch.softmax(row / s["temp"], 0)

    for n in s["lens"]:
        taken = n - 1
        for i in reversed(range(n - 1)):
            r = row + i
            p, q = (float(distribution(r, d)[tokens[r]]) for d in (False, True))
            ratio[r] = min(p, q) / q if q > 0.0 else float(p > 0.0)
            taken = taken if u[r] * q < p else i
        r = row + taken
        w = distribution(r, False)
        if taken < n - 1:
            rest = (w - distribution(r, True)).clamp(min=0.0)
            w = rest if float(rest.sum()) > 0.0 else w
        cum = torch.cumsum(w, 0)
        token = int((cum > u[row + n - 1] * cum[-1]).nonzero()[0])
        accepted.append(taken)
        following.append(token)
        split += [r + 1, row + n]
        row += n
    whole = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (accepted, following, split)]
    return {"accepted": whole[0], "next": whole[1], "ratio": ratio, "split": whole[2]}


def exact(case, seed):
    s = _inputs(case, seed)
    return _verify_exact(s) if case["kind"] == "verify" else _delta_exact(s)
