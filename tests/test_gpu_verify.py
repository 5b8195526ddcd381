"""Verification of drafted tokens against its definition in 64 bits, a sequence
at a time: which drafts stand, the token that follows, the ratios and the rows
that stand.  Tokens have to be equal.  The test and a draw compare sums of up to
256000 terms that are good to 2^-46 of the whole with a number of 24 bits; inputs
are drawn anew (from the next seed, before the call) where any comparison of the
oracle's is closer than 2^-40, so that no rounding can decide one."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import TYPES, at, f64, gpu
from test_zz_no_alloc import _hip_runtime, _ok

pytestmark = pytest.mark.gpu
CLOSE = 2.0 ** -40
MARK = -77


def note(msg):
    print("[case] " + msg, flush=True)


def shares(row, weights, temp):
    """Probabilities of a row; all zero where it has none."""
    if weights:
        w = np.where(np.isfinite(row) & (row > 0), row, 0.0)
    else:
        row = np.where(np.isnan(row), -np.inf, row)
        m = row.max()
        if m == -np.inf:
            return np.zeros_like(row)
        if np.float32(temp) < np.float32(0.05):
            w = np.zeros_like(row)
            w[int(np.argmax(row))] = 1.0
            return w
        with np.errstate(invalid="ignore"):
            w = np.exp(np.where(row == m, 0.0, (row - m) / float(np.float32(temp))))
    s = w.sum()
    return w / s if s > 0 else w


class VerifyCase:
    def __init__(self, type_name, vocab, lens, draft="logits", weights=False, temp=0.75, seed=0,
                 lead=0, row_pad=0, front=0, tail=0, spread=2.0, edit=None, noise=0.7):
        self.type, self.vocab, self.lens, self.temp, self.weights = type_name, vocab, lens, temp, weights
        self.draft_kind, self.edit = draft, edit
        self.args = (lead, row_pad, front, tail, spread, noise)
        self.starts = list(front + np.concatenate([[0], np.cumsum(lens)]).astype(int))
        for s in range(seed, seed + 50):
            self.draw(s)
            self.answer = self.want()
            if self.answer is not None:
                return
        raise AssertionError("no inputs without a close call")

    def draw(self, seed):
        lead, row_pad, front, tail, spread, noise = self.args
        r, V = np.random.default_rng(seed), self.vocab
        rows = front + sum(self.lens) + tail
        self.rows = rows
        t = spread * r.standard_normal((rows, V))
        d = t + noise * r.standard_normal((rows, V))
        heat = 1.0 / max(self.temp, 0.3)
        pick = np.argmax(d * heat + r.gumbel(size=d.shape), -1) if rows else np.zeros(0)
        soft = lambda v: np.exp(v * heat - (v * heat).max(-1, keepdims=True))
        target = soft(t) if self.weights else t
        draft = soft(d) if self.draft_kind == "weights" else d
        tokens = pick.astype(np.int32)
        u = r.random(rows).astype(np.float32)
        if self.edit:
            self.edit(target, draft, tokens, u)
        self.tokens, self.u = gpu(tokens, torch.int32), gpu(u, torch.float32)
        dt = TYPES[self.type][1]
        self.stride = lead + V + row_pad

        def rows_of(a):
            buf = torch.full((max(rows, 1), self.stride), 99.0, dtype=dt)
            buf[:rows, lead:lead + V] = torch.as_tensor(a).to(dt)
            buf = buf.cuda()
            return buf[:rows, lead:lead + V]

        self.target = rows_of(target)
        self.draft = None if self.draft_kind == "none" else rows_of(draft)

    def want(self):
        """None where a comparison is too close."""
        T = f64(self.target)
        D = None if self.draft is None else f64(self.draft)
        tokens, u = self.tokens.cpu().numpy(), self.u.cpu().numpy().astype(np.float64)
        greedy = not self.weights and np.float32(self.temp) < np.float32(0.05)
        accepted, nxt, ratio, split = [], [], {}, []
        for b in range(len(self.lens)):
            s, e = (min(max(v, 0), self.rows) for v in self.starts[b:b + 2])
            e = max(s, e)
            split.append(s)
            if e == s:
                accepted.append(0)
                nxt.append(-1)
                split.append(s)
                continue

            def q_of(r):
                if D is None:
                    q = np.zeros(self.vocab)
                    if 0 <= tokens[r] < self.vocab:
                        q[tokens[r]] = 1.0
                    return q
                return shares(D[r], self.draft_kind == "weights", self.temp)

            stop = None
            for r in range(s, e - 1):
                p, q = shares(T[r], self.weights, self.temp), q_of(r)
                inside = 0 <= tokens[r] < self.vocab
                pd, qd = (p[tokens[r]], q[tokens[r]]) if inside else (0.0, 0.0)
                if greedy:
                    stands = pd > 0
                    ratio[r] = 1.0 if stands else 0.0
                else:
                    stands = u[r] * qd < pd
                    ratio[r] = 0.0 if pd == 0 else (1.0 if pd >= qd else pd / qd)
                    if pd > 0 and qd > 0 and abs(u[r] * qd - pd) < CLOSE * pd:
                        return None
                if not stands and stop is None:
                    stop = r
            full = stop is None
            stop = e - 1 if full else stop
            accepted.append(stop - s)
            split.append(stop + 1)
            p = shares(T[stop], self.weights, self.temp)
            w = p
            if not full and not greedy:
                w = np.maximum(p - q_of(stop), 0.0)
                if 0 < w.sum() < 1e-9:
                    return None  # what is left of two equal rows is all rounding
                w = w if w.sum() > 0 else p
            if w.sum() == 0:
                nxt.append(-1)
                continue
            cum = np.cumsum(w)
            goal = u[e - 1] * cum[-1]
            over = (cum > goal) & (w > 0)
            if not greedy and (np.abs(cum[w > 0][:-1] - goal) < CLOSE * cum[-1]).any():
                return None
            nxt.append(int(np.argmax(w)) if greedy else
                       int(np.argmax(over)) if over.any() else int(np.nonzero(w > 0)[0][-1]))
        split.append(min(max(self.starts[-1], 0), self.rows))
        return accepted, nxt, ratio, split

    def descriptor(self, lib, ratio=True, split=True):
        n = len(self.lens)
        i32 = lambda k: torch.full((k,), MARK, dtype=torch.int32, device="cuda")
        self.d_start = gpu(np.array(self.starts), torch.int32)
        self.accepted, self.next, self.split = i32(n + 3), i32(n + 3), i32(2 * n + 4)
        self.ratio = torch.full((self.rows + 2,), float(MARK), device="cuda")
        d = bh.Verify(type=TYPES[self.type][0], vocab=self.vocab, n_seqs=n, n_rows=self.rows,
                      row_start=at(self.d_start), target=at(self.target), target_stride=self.stride,
                      target_weights=int(self.weights), draft=at(self.draft),
                      draft_stride=self.stride, draft_weights=int(self.draft_kind == "weights"),
                      temp=self.temp, tokens=at(self.tokens), u=at(self.u),
                      n_accepted=at(self.accepted), next_token=at(self.next),
                      ratio=at(self.ratio) if ratio else None,
                      split_start=at(self.split) if split else None)
        size = lib.bm_hip_verify_workspace_bytes(C.byref(d))
        self.work = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
        self.size = size
        return d

    def right(self, what):
        n = len(self.lens)
        accepted, nxt, ratio, split = self.answer
        assert self.accepted.tolist() == accepted + [MARK] * 3, what
        assert self.next.tolist() == nxt + [MARK] * 3, what
        assert self.split.tolist() == split + [MARK] * 3, what
        got = self.ratio.cpu().numpy()
        for r in range(self.rows + 2):
            if r in ratio:
                # two quotients and their own rounding
                assert abs(got[r] - ratio[r]) <= 2.0 ** -23 * ratio[r] + 2.0 ** -126, (what, r, got[r], ratio[r])
            else:
                assert got[r] == MARK, (what, r)
        assert (self.work[self.size:] == 0xFF).all()

    def check(self, lib, what, stream=None):
        d = self.descriptor(lib)
        torch.cuda.synchronize()
        bh.check(lib.bm_hip_verify_dev(C.byref(d), at(self.work), stream), "verify")
        torch.cuda.synchronize()
        self.right(what)


LENS = [5, 1, 0, 3, 9, 2, 1]


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("draft", ["logits", "weights", "none"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("temp", [0.0, 0.75])
def test_drafts(hip, type_name, draft, weights, temp):
    note("verify %s %s weights=%s temp=%g" % (type_name, draft, weights, temp))
    VerifyCase(type_name, 1000, LENS, draft, weights, temp, seed=3).check(hip, "drafts")


@pytest.mark.parametrize("vocab", [1, 2, 3, 15, 16, 17, 4095, 4096, 4097, 8192, 50257])
@pytest.mark.parametrize("type_name", ["f32", "bf16"])
def test_vocabularies(hip, vocab, type_name):
    for temp in (0.0, 1.5):
        note("vocabulary %d %s temp=%g" % (vocab, type_name, temp))
        VerifyCase(type_name, vocab, [3, 1, 2], temp=temp, seed=vocab).check(hip, "vocabulary")


def test_the_largest_vocabulary(hip):
    note("vocabulary 256000")
    for draft in ("logits", "none"):
        VerifyCase("f16", 256000, [2, 1], draft, seed=1).check(hip, "largest")


@pytest.mark.parametrize("type_name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lead,pad", [(1, 0), (0, 1), (3, 2), (2, 5), (7, 1)])
def test_rows_on_any_alignment(hip, type_name, lead, pad):
    note("alignment %s %d %d" % (type_name, lead, pad))
    VerifyCase(type_name, 4103, [3, 2], "weights", lead=lead, row_pad=pad, front=2, tail=1,
               seed=lead).check(hip, "alignment")


def test_long_and_many_sequences(hip):
    note("long")
    VerifyCase("f32", 130, [130, 3], seed=2, noise=0.1).check(hip, "long")
    VerifyCase("f32", 130, [70], temp=0.0, seed=2, noise=0.0).check(hip, "long, greedy")
    note("many")
    r = np.random.default_rng(0)
    VerifyCase("bf16", 67, [int(v) for v in r.integers(0, 6, 300)], "weights", seed=5).check(hip, "many")


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")])
def test_numbers_at_the_ends(hip, u):
    """Also what is no draw: a token with a probability follows all the same."""
    note("u = %r" % u)

    def edit(t, d, tokens, uu):
        uu[3] = u
        uu[6] = u
        t[3, :3] = t[6, :3] = -np.inf
        t[3, -2:] = t[6, -2:] = -np.inf

    c = VerifyCase("f32", 500, [4, 3], "none", seed=2, edit=edit)
    c.check(hip, "ends")
    assert all(3 <= v < 498 for v in c.next[:2].tolist()) or c.accepted[0] < 3


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("kind", ["masked", "nothing", "nan", "inf", "lowest", "draft outside",
                                  "same", "ties", "no draft left", "draft masked"])
@pytest.mark.parametrize("temp", [0.0, 0.75])
def test_rows_with_masks(hip, kind, temp):
    note("masks: %s temp=%g" % (kind, temp))

    def edit(t, d, tokens, u):
        V = t.shape[1]
        if kind == "masked":
            t[:, ::2] = -INF
        elif kind == "nothing":
            t[0] = t[3] = t[7] = -INF
        elif kind == "nan":
            t[:, ::3] = NAN
            d[:, 1::3] = NAN
            t[4] = NAN
        elif kind == "inf":
            t[:, 5::7] = INF
            d[2, 3] = INF
        elif kind == "lowest":
            t[:, ::2] = np.finfo(np.float32).min
            d[:, ::5] = np.finfo(np.float32).min
        elif kind == "draft outside":
            tokens[:] = np.where(np.arange(len(tokens)) % 2, V, -1)
            tokens[1] = 2 ** 31 - 1
        elif kind == "same":
            d[:] = t
        elif kind == "ties":
            t[:] = np.round(t)
            tokens[:] = np.argmax(t, -1)
        elif kind == "no draft left":
            t[:] = -INF
            t[:, 7] = 1.0
            d[:] = -INF
            d[:, 7] = 1.0
            tokens[:] = 3
        else:
            d[1] = d[4] = -INF

    VerifyCase("f32", 600, [4, 1, 4], temp=temp, seed=4, edit=edit).check(hip, kind)
    VerifyCase("f32", 600, [4, 1, 4], "none", temp=temp, seed=4, edit=edit).check(hip, kind + ", no q")


@pytest.mark.parametrize("kind", ["zeros", "odd", "draft zeros"])
def test_weights_that_are_none(hip, kind):
    note("weights: " + kind)

    def edit(t, d, tokens, u):
        if kind == "zeros":
            t[1] = t[4] = 0.0
        elif kind == "odd":
            t[:, ::4] = -1.0
            t[:, 1::8] = INF
            t[:, 2::8] = NAN
            d[:, ::3] = NAN
            d[:, 1::9] = -INF
        else:
            d[1] = d[3] = 0.0

    VerifyCase("f32", 600, [3, 1, 4], "weights", True, seed=4, edit=edit).check(hip, kind)


def test_outputs_that_are_left_out(hip):
    note("no ratio, no split")
    c = VerifyCase("f32", 300, [4, 2], seed=1)
    d = c.descriptor(hip, ratio=False, split=False)
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_verify_dev(C.byref(d), at(c.work), None))
    torch.cuda.synchronize()
    assert c.accepted.tolist()[:2] == c.answer[0] and c.next.tolist()[:2] == c.answer[1]
    assert (c.ratio == MARK).all() and (c.split == MARK).all()


def test_one_sequence_needs_no_starts(hip):
    note("no starts")
    c = VerifyCase("f32", 300, [6], seed=1)
    d = c.descriptor(hip)
    d.row_start = None
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_verify_dev(C.byref(d), at(c.work), None))
    torch.cuda.synchronize()
    c.right("alone")


def test_no_rows(hip):
    note("no rows")
    VerifyCase("f32", 300, [0, 0, 0], seed=1).check(hip, "none")


def test_a_workspace_of_a_larger_call(hip):
    note("larger workspace")
    big = VerifyCase("f32", 9000, [5, 5, 5], seed=1)
    big.descriptor(hip)
    for lens, vocab in (([2], 300), ([5, 5, 5], 4096), ([1, 9], 5000)):
        c = VerifyCase("f32", vocab, lens, seed=2)
        d = c.descriptor(hip)
        assert c.size <= big.size
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_verify_dev(C.byref(d), at(big.work), None))
        torch.cuda.synchronize()
        c.right("larger")


def test_replays_equal_the_eager_calls(hip):
    """Captured once; each replay reads tokens, numbers and starts anew."""
    note("replays")
    rt = _hip_runtime()
    s = C.c_void_p()
    _ok(rt.hipStreamCreateWithFlags(C.byref(s), 1), "hipStreamCreateWithFlags")
    cs = [VerifyCase("bf16", 5000, [4, 2, 5], "weights", seed=k) for k in (1, 60, 120)]
    c = cs[0]
    d = c.descriptor(hip)
    torch.cuda.synchronize()
    graph, exe = C.c_void_p(), C.c_void_p()
    _ok(rt.hipStreamBeginCapture(s, 1), "hipStreamBeginCapture")
    rc = hip.bm_hip_verify_dev(C.byref(d), at(c.work), s.value)
    _ok(rt.hipStreamEndCapture(s, C.byref(graph)), "hipStreamEndCapture")
    assert rc == 0, bh.last_error()
    _ok(rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0), "instantiate")
    try:
        for k, o in enumerate(cs + cs[:1]):
            for f in ("target", "draft", "tokens", "u"):
                getattr(c, f).copy_(getattr(o, f))
            for f in ("accepted", "next", "split", "ratio"):
                getattr(c, f).fill_(MARK)
            c.work.fill_(0xFF)
            torch.cuda.synchronize()
            _ok(rt.hipGraphLaunch(exe, s), "hipGraphLaunch")
            _ok(rt.hipStreamSynchronize(s), "sync")
            c.answer = o.answer if k < 3 else cs[0].want()
            c.right("replay %d" % k)
            (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
            if k == 0:
                cs[0].keep = (c.target.clone(), c.draft.clone(), c.tokens.clone(), c.u.clone())
    finally:
        rt.hipGraphExecDestroy(exe)
        rt.hipGraphDestroy(graph)
        rt.hipStreamDestroy(s)


def test_tokens_are_distributed_as_the_target(hip):
    """Many sequences with one draft each, drawn from q: the first token of each
    (the draft if it stands, else the one that follows) is distributed as p.
    With n draws a count is within 5 sqrt(n p (1 - p)) of n p but for one in
    1.7 million."""
    note("distribution")
    V, n = 12, 40000
    r = np.random.default_rng(0)
    p, q = (x / x.sum() for x in (r.random(V) ** 2 + 0.01, r.random(V) + 0.02))
    t = np.log(np.repeat(p[None], 2 * n, 0)).astype(np.float32)
    c = VerifyCase.__new__(VerifyCase)
    c.type, c.vocab, c.lens, c.temp, c.weights, c.draft_kind = "f32", V, [2] * n, 1.0, False, "weights"
    c.starts, c.rows, c.stride = list(range(0, 2 * n + 1, 2)), 2 * n, V
    c.target, c.draft = gpu(t, torch.float32), gpu(np.repeat(q[None], 2 * n, 0), torch.float32)
    tokens = r.choice(V, 2 * n, p=q)
    c.tokens, c.u = gpu(tokens, torch.int32), gpu(r.random(2 * n).astype(np.float32), torch.float32)
    d = c.descriptor(hip)
    torch.cuda.synchronize()
    bh.check(hip.bm_hip_verify_dev(C.byref(d), at(c.work), None))
    torch.cuda.synchronize()
    took = c.accepted[:n].cpu().numpy()
    first = np.where(took == 1, tokens[::2], c.next[:n].cpu().numpy())
    count = np.bincount(first, minlength=V)
    assert (np.abs(count - n * p) < 5 * np.sqrt(n * p * (1 - p)) + 1).all(), (count, n * p)
