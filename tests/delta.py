"""What the tests of the gated delta rule share: the calls, the rule in 64
bits, and the bound of the kernels' error.

Bounds.  u = 2^-24.  One row takes S[p] to a S[p] (I - b k k^T) + b v[p] k^T, and
with |k| <= 1 and 0 <= b <= 2 the matrix lengthens no vector, so an error in S[p]
(as a vector of d_state values) does not grow, and the rows' own errors add up.

Row after row (single tokens; sequences of up to 32 rows, eight at a time, whose
sums are the same with up to eight terms more): a product of N
factors is off by N u of the vectors' lengths, the decay by 10 u (1 + |A d|), the
other operations by a few u each: per row
    u ((N + 16) b |S| + (24 + 10 |A d|) (|S| + |b v|)).

In chunks of 64 rows, operands are two halves of 11 bits, off by 2^-22 of the
largest in a row of K, Q, T or A (|T| <= 1, since b <= 1 there), and of the
largest m in a column of S and of what is written.  K S: 2^-22 sqrt(N) m from
each side; T R: 2^-22 times the sum of 64 |R| from each side, 2^-15 m; A w
likewise, times |q| scale; K^T w: 2^-22 sqrt(64) sqrt(64) m.  Together below
kChunk = 2^-13 m per chunk, besides the rows' fp32 errors above.  These are worst
cases: 4096 products whose errors all point one way.  Independent ones add up as
their root, 64 times less, and the sum of a state's squared errors is held to
that: kSpread = 2^-19 of its length.
"""
import ctypes as C

import numpy as np
import torch

from native import bh
from recurrence import (MARK, TYPES, U, at, check_rows, close, columns, f64, gpu, half_step,
                        sequences, silu, softplus, tiny)

kChunk, kSpread = 2.0 ** -13, 2.0 ** -19
EPS = 1e-6


def rule(c, pool, seqs, fresh=None):
    """{row: y}, {row: bound}, new pool, {slot: bound}, in 64 bits."""
    H, P, G, N = c.H, c.P, c.G, c.N
    T = c.v.shape[0]
    v64 = lambda t, *sh: f64(t).reshape(T, *sh)
    q, k, v = v64(c.q, G, N), v64(c.k, G, N), v64(c.v, H, P)
    z = None if c.z is None else v64(c.z, H, P)
    if c.norm:
        q, k = (t / np.sqrt((t * t).sum(-1, keepdims=True) + c.eps) for t in (q, k))
    q, k = np.repeat(q, H // G, 1), np.repeat(k, H // G, 1)
    beta = np.ones((T, H)) if c.beta is None else v64(c.beta, H)
    if c.beta is not None and c.sigmoid:
        beta = 1.0 / (1.0 + np.exp(-beta))
    expo = np.zeros((T, H))
    if c.A is not None:
        d = v64(c.dt, H) + (0.0 if c.dt_bias is None else f64(c.dt_bias))
        expo = np.minimum(f64(c.A) * (softplus(d) if c.soft else d), 0.0)
    y, tol, stol = {}, {}, {}
    new = None if pool is None else pool.copy()
    for b, s, e, slot in seqs:
        S = np.zeros((H, P, N))
        if slot is not None and not (fresh is not None and fresh[b]):
            S = pool[slot].copy()
        n = e - s
        chunked = n > 32 and not c.step
        length, bv, out, own = [], [], [], np.zeros((n, H, P))
        for t in range(s, e):
            norm0 = np.sqrt((S * S).sum(-1))
            S = S * np.exp(expo[t])[:, None, None]
            w = beta[t][:, None] * (v[t] - (S * k[t][:, None]).sum(-1))
            S = S + w[..., None] * k[t][:, None]
            norm = np.sqrt((S * S).sum(-1))
            both = np.maximum(norm, norm0)
            add = np.abs(beta[t][:, None] * v[t])
            out.append(c.scale * (S * q[t][:, None]).sum(-1))
            own[t - s] = U * ((N + 16) * np.abs(beta[t])[:, None] * both +
                              (24 + 10 * np.abs(expo[t])[:, None]) * (both + add))
            length.append(both)
            bv.append(add)
        err = np.zeros((H, P))
        for i in range(n):
            t = s + i
            if chunked and i % 64 == 0:
                m = np.maximum(np.max(length[i:i + 64], 0), np.max(bv[i:i + 64], 0))
                err = err + kChunk * m
            err = err + own[i]
            qn = np.sqrt((q[t] * q[t]).sum(-1))[:, None] * abs(c.scale)
            tl = qn * (err + (N + 24) * U * length[i])
            o = out[i]
            if z is not None:
                g = silu(z[t])
                gate = (10 * U + (2.0 ** -20 + np.abs(z[t]) * 2.0 ** -23
                                  if chunked and c.type != "f32" else 0.0)) * np.abs(o * g)
                tl, o = tl * np.abs(g) + gate, o * g
            y[t], tol[t] = o, tl
        if slot is not None and not c.frozen and (n > 0 or (fresh is not None and fresh[b])):
            new[slot] = S
            stol[slot] = err[..., None] + 4 * U * np.abs(S)
    return y, tol, new, stol


class DeltaCase:
    def __init__(self, type_name, H, P, G, N, lens, gate=True, decay=True, bias=True, soft=True,
                 beta="sigmoid", norm=True, frozen=False, slots="shuffled", lead=0, row_pad=0,
                 front=0, tail=0, pool=True, seed=0, step=False, spare=2, slot_pad=0, rate=4.0,
                 scale=None, eps=EPS):
        r = np.random.default_rng(seed)
        self.type, self.step, self.soft, self.norm, self.frozen = type_name, step, soft, norm, frozen
        self.H, self.P, self.G, self.N, self.n = H, P, G, N, len(lens)
        self.scale = float(np.float32(N ** -0.5 if scale is None else scale))
        self.eps = float(np.float32(eps))
        n = self.n
        T = n if step else front + sum(lens) + tail
        self.n_tokens = T
        self.starts = (list(range(n + 1)) if step else
                       list(front + np.concatenate([[0], np.cumsum(lens)]).astype(int)))
        unit = lambda t: t / np.sqrt((t * t).sum(-1, keepdims=True)) * 0.99  # the types round
        q, k = (r.standard_normal((T, G, N)) + 0.3 for _ in range(2))
        if not norm:
            k = unit(k)
        b = r.standard_normal((T, H)) if beta == "sigmoid" else r.uniform(0, 1, (T, H))
        dt = r.standard_normal((T, H)) if soft else np.exp(r.uniform(-6, -1, (T, H)))
        parts = [r.standard_normal((T, H * P)), q.reshape(T, G * N), dt, k.reshape(T, G * N),
                 r.standard_normal((T, H * P)), b]
        self.buf, (self.z, self.q, self.dt, self.k, self.v, self.beta), self.stride = columns(
            parts, type_name, lead, row_pad)
        self.sigmoid = beta == "sigmoid"
        if beta is None:
            self.beta = None
        if not gate:
            self.z = None
        f32 = torch.float32
        self.A = gpu(-np.exp(r.uniform(np.log(0.01), np.log(rate), H)), f32) if decay else None
        self.dt_bias = gpu(r.uniform(-4, 0, H) if soft else 0.01 * r.random(H), f32) if bias else None
        self.n_slots = n + spare
        self.slots = [int(i) for i in r.permutation(self.n_slots)[:n]] if slots == "shuffled" else slots
        self.fresh = None
        self.pool_buf = gpu(r.standard_normal((self.n_slots, H * P * N + slot_pad)) * N ** -0.5,
                            f32) if pool else None
        self.ybuf, (self.y,), self.ystride = columns([np.full((T, H * P), MARK)], type_name, lead,
                                                     row_pad)
        self.work = None

    def descriptor(self):
        self.d_start = gpu(np.array(self.starts), torch.int32)
        self.d_slots = gpu(np.array(self.slots), torch.int32) if self.slots is not None and self.n else None
        self.d_fresh = gpu(np.array(self.fresh), torch.uint8) if self.fresh is not None else None
        s = self.stride
        return bh.Delta(type=TYPES[self.type][0], n_heads=self.H, head_dim=self.P, n_groups=self.G,
                        d_state=self.N, dt_softplus=int(self.soft), beta_sigmoid=int(self.sigmoid),
                        qk_norm=int(self.norm), frozen=int(self.frozen), norm_eps=self.eps,
                        scale=self.scale, n_seqs=self.n, n_tokens=self.n_tokens,
                        seq_start=at(self.d_start), slots=at(self.d_slots), fresh=at(self.d_fresh),
                        q=at(self.q), k=at(self.k), v=at(self.v), dt=at(self.dt),
                        beta=at(self.beta), z=at(self.z), q_stride=s, k_stride=s, v_stride=s,
                        dt_stride=s, beta_stride=s, z_stride=s, A=at(self.A),
                        dt_bias=at(self.dt_bias), state=at(self.pool_buf), n_slots=self.n_slots,
                        state_stride=0 if self.pool_buf is None else self.pool_buf.shape[1],
                        y=at(self.y), y_stride=self.ystride)

    def pool(self):
        row = self.H * self.P * self.N
        return f64(self.pool_buf[:, :row]).reshape(-1, self.H, self.P, self.N)

    def want(self):
        seqs = sequences(self.starts, self.slots, self.n_slots, self.n_tokens, self.pool_buf is not None)
        return rule(self, None if self.pool_buf is None else self.pool(), seqs,
                    None if self.step else self.fresh)

    def workspace(self, lib, d):
        """Filled with NaN: a call must not read what it has not written."""
        n = lib.bm_hip_delta_workspace_bytes(C.byref(d))
        self.work = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") if n else None
        return at(self.work)

    def call(self, lib, d, w, stream=None):
        if self.step:
            return lib.bm_hip_delta_step_dev(C.byref(d), stream)
        return lib.bm_hip_delta_dev(C.byref(d), w, stream)

    def run(self, lib, stream=None):
        d = self.descriptor()
        w = None if self.step else self.workspace(lib, d)
        torch.cuda.synchronize()
        bh.check(self.call(lib, d, w, stream), "delta")
        torch.cuda.synchronize()

    def check(self, lib, what):
        rows, tols, pool, stol = self.want()
        before = None if self.pool_buf is None else self.pool_buf.clone()
        self.run(lib)
        check_rows(self.ybuf, self.y, rows, tols, self.type, (self.H, self.P), what)
        if pool is None:
            return
        got = self.pool()
        for k in range(self.n_slots):
            if k in stol:
                close(got[k], pool[k], stol[k], "f32", "%s slot %d" % (what, k))
                off, all_of_it = np.linalg.norm(got[k] - pool[k]), np.linalg.norm(pool[k])
                assert off <= kSpread * all_of_it + 1e-30, "%s slot %d: %g of %g" % (what, k, off, all_of_it)
            else:
                assert torch.equal(before[k], self.pool_buf[k]), "%s: slot %d changed" % (what, k)
        row = self.H * self.P * self.N
        assert torch.equal(before[:, row:], self.pool_buf[:, row:])
