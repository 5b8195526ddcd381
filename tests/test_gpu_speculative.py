"""Drafted decoding on device buffers, as a server would run it: the rows of all
sequences' drafts through the convolution (on copied slots) and the gated delta
rule (frozen slots), the verification, then the rows that stand once more on the
sequences' own slots by the verification's split_start.  The tokens have to be
those of decoding one by one, and the states theirs to fp32 rounding."""
import ctypes as C

import numpy as np
import pytest
import torch

import native
from native import bh
from recurrence import at, gpu

pytestmark = pytest.mark.gpu

V, D, H, P, G, N, W = 300, 48, 4, 24, 2, 40, 4
CH = 2 * G * N + H * P  # q, k and v go through the convolution


class Block:
    """One block and its head, all in fp32, with a convolution and a state slot
    per sequence and as many to spare."""

    def __init__(self, n, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.n = n
        self.embed, self.w_in = rnd(V, D), rnd(D, CH + H * P + 2 * H) / D ** 0.5
        self.w_out = 3.0 * rnd(H * P, V) / (H * P) ** 0.5
        self.conv_w, self.conv_b = rnd(W, CH) / W ** 0.5, 0.1 * rnd(CH)
        self.A = -torch.exp(rnd(H))
        self.dt_bias = rnd(H) - 2.0
        self.conv = torch.zeros(2 * n, (W - 1) * CH, device="cuda")
        self.state = torch.zeros(2 * n, H * P * N, device="cuda")
        self.own = torch.arange(n, dtype=torch.int32, device="cuda")
        self.spare = self.own + n
        # rows that stand on the own slots, the others nowhere
        self.split_slots = torch.full((2 * n,), -1, dtype=torch.int32, device="cuda")
        self.split_slots[0::2] = self.own

    def rows(self, lib, tokens, starts, n_seqs, conv_slots, state_slots, frozen=False, step=False):
        """Logits of all rows; the slots move on as the lists say."""
        T = tokens.numel()
        proj = (self.embed[tokens.long()] @ self.w_in).contiguous()
        x, z, dt, beta = proj.split([CH, H * P, H, H], 1)
        xc, y = torch.zeros(T, CH, device="cuda"), torch.zeros(T, H * P, device="cuda")
        ps = proj.shape[1]
        c = bh.Conv(type=bh.F32, channels=CH, width=W, silu=1, n_seqs=n_seqs, n_tokens=T,
                    seq_start=at(starts), slots=at(conv_slots), x=at(x), x_stride=ps,
                    w=at(self.conv_w), bias=at(self.conv_b), state=at(self.conv),
                    state_stride=self.conv.shape[1], n_slots=2 * self.n, y=at(xc), y_stride=CH)
        q, k, v = xc.split([G * N, G * N, H * P], 1)
        d = bh.Delta(type=bh.F32, n_heads=H, head_dim=P, n_groups=G, d_state=N, dt_softplus=1,
                     beta_sigmoid=1, qk_norm=1, frozen=int(frozen), norm_eps=1e-6,
                     scale=N ** -0.5, n_seqs=n_seqs, n_tokens=T, seq_start=at(starts),
                     slots=at(state_slots), q=at(q), k=at(k), v=at(v), dt=at(dt), beta=at(beta),
                     z=at(z), q_stride=CH, k_stride=CH, v_stride=CH, dt_stride=ps, beta_stride=ps,
                     z_stride=ps, A=at(self.A), dt_bias=at(self.dt_bias), state=at(self.state),
                     n_slots=2 * self.n, state_stride=self.state.shape[1], y=at(y), y_stride=H * P)
        torch.cuda.synchronize()
        if step:
            bh.check(lib.bm_hip_conv_step_dev(C.byref(c), None))
            bh.check(lib.bm_hip_delta_step_dev(C.byref(d), None))
        else:
            bh.check(lib.bm_hip_conv_dev(C.byref(c), None))
            work = torch.empty(lib.bm_hip_delta_workspace_bytes(C.byref(d)) + 1, dtype=torch.uint8,
                               device="cuda")
            bh.check(lib.bm_hip_delta_dev(C.byref(d), at(work), None))
        torch.cuda.synchronize()
        return y @ self.w_out


def starts_of(lens):
    return gpu(np.concatenate([[0], np.cumsum(lens)]), torch.int32)


@pytest.mark.parametrize("prompts,most", [([5, 40, 90, 1], 4), ([3], 7), ([70, 2, 33], 40)])
def test_drafted_decoding_is_decoding(hip, prompts, most):
    print("[case] prompts %s, up to %d drafts" % (prompts, most), flush=True)
    n, r = len(prompts), np.random.default_rng(len(prompts) + most)
    text = [list(map(int, r.integers(0, V, k + 1))) for k in prompts]
    total = 100

    def start(seed):
        b = Block(n, seed)
        rows = gpu(np.concatenate([t[:-1] for t in text]), torch.int32)
        b.rows(hip, rows, starts_of(prompts), n, b.own, b.own)
        return b

    # one by one, with numbers of which no two largest are too close to tell an
    # error from a rounding: by 1e-4 of the logits' spread, of sums of some hundred
    # terms that are good to 1e-6 of it
    for seed in range(7, 40):
        plain = start(seed)
        out = [t[-1:] for t in text]
        states, gap = [], 1e9
        for _ in range(total):
            states.append((plain.conv[:n].clone(), plain.state[:n].clone()))
            logits = plain.rows(hip, gpu(np.array([o[-1] for o in out]), torch.int32), None, n,
                                plain.own, plain.own, step=True)
            two = logits.topk(2, -1).values
            gap = min(gap, float(((two[:, 0] - two[:, 1]) / logits.std(-1)).min()))
            for o, t in zip(out, logits.argmax(-1).tolist()):
                o.append(t)
        if gap > 1e-4:
            break
    assert gap > 1e-4

    # by drafts, some of which are wrong
    b = start(seed)
    done = [0] * n  # tokens behind the prompt that stand
    i32 = lambda k: torch.full((k,), -5, dtype=torch.int32, device="cuda")
    while max(done) < total - most - 2:
        lens, rows = [], []
        for s in range(n):
            m = int(r.integers(0, most + 1))
            draft = [t if r.random() < 0.8 else int(r.integers(0, V))
                     for t in out[s][done[s] + 1:done[s] + 1 + m]]
            rows += [out[s][done[s]]] + draft
            lens.append(1 + len(draft))
        tokens, begin = gpu(np.array(rows), torch.int32), starts_of(lens)
        pool = bh.Slots(base=at(b.conv), n_slots=2 * n, n_layers=1, slot_bytes=4 * b.conv.shape[1],
                        slot_stride=4 * b.conv.shape[1])
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_slots_copy_dev(C.byref(pool), 1, at(b.own), at(b.spare), n, None))
        before = b.state.clone()
        logits = b.rows(hip, tokens, begin, n, b.spare, b.own, frozen=True).contiguous()
        assert torch.equal(before, b.state)
        # row i judges the token of row i + 1
        judged = torch.cat([tokens[1:], tokens[:1]])
        took, following, split = i32(n), i32(n), i32(2 * n + 1)
        u = torch.rand(len(rows), device="cuda")
        d = bh.Verify(type=bh.F32, vocab=V, n_seqs=n, n_rows=len(rows), row_start=at(begin),
                      target=at(logits), target_stride=V, temp=0.0, tokens=at(judged), u=at(u),
                      n_accepted=at(took), next_token=at(following), split_start=at(split))
        work = torch.empty(hip.bm_hip_verify_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        bh.check(hip.bm_hip_verify_dev(C.byref(d), at(work), None))
        torch.cuda.synchronize()
        b.rows(hip, tokens, split, 2 * n, b.split_slots, b.split_slots)
        at_row = 0
        for s in range(n):
            k = int(took[s])
            want = out[s][done[s] + 1:done[s] + 2 + k]
            assert rows[at_row + 1:at_row + 1 + k] + [int(following[s])] == want
            if k + 1 < lens[s]:  # the first that was refused was wrong
                assert rows[at_row + 1 + k] != want[-1]
            done[s] += k + 1
            at_row += lens[s]
            conv, state = states[done[s]][0][s], states[done[s]][1][s]
            # sums of some hundred terms in another order, a few dozen tokens long
            assert (b.conv[s] - conv).abs().max() <= 2.0 ** -16 * conv.abs().max()
            assert (b.state[s] - state).norm() <= 2.0 ** -14 * state.norm()
