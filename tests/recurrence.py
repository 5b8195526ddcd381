"""What the tests of the batched recurrence share: device tensors, the calls,
and the operators in 64 bits with the bound of the kernels' fp32 error.

Bounds.  u = 2^-24 is the rounding of one fp32 operation.  A sum of products
of m factors in any order is off by at most about (m + terms) u times the sum
of the products' magnitudes; a recurrence over t tokens adds a product and a
sum per token.  The functions used have errors of a few u; softplus's error
and that of the exponent's products scale with the exponent: 8 u times the
summed |A| d.  The magnitudes come from the same recurrence on absolute
values.  The result's own rounding is half a step of its type.
"""
import ctypes as C

import numpy as np
import torch

import native
from native import bh

U = 2.0 ** -24
TYPES = {"f32": (bh.F32, torch.float32), "bf16": (bh.BF16, torch.bfloat16),
         "f16": (bh.F16, torch.float16)}
MARK = 77.0  # exact in every type


def at(t):
    return None if t is None else t.data_ptr()


def gpu(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).cuda()


def columns(parts, type_name, lead=0, row_pad=0):
    """The arrays side by side in one buffer of MARK: (views, row stride)."""
    dt = TYPES[type_name][1]
    rows = parts[0].shape[0]
    width = lead + sum(p.shape[1] for p in parts) + row_pad
    buf = torch.full((max(rows, 1), width), MARK, dtype=dt)
    views, c = [], lead
    for p in parts:
        buf[:rows, c:c + p.shape[1]] = torch.as_tensor(p).to(dt)
        views.append((c, p.shape[1]))
        c += p.shape[1]
    buf = buf.cuda()
    return buf, [buf[:, a:a + n] for a, n in views], width


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def half_step(type_name):
    return torch.finfo(TYPES[type_name][1]).eps / 2


def tiny(type_name):
    """Results below it may round to zero: fp16 keeps its subnormals, the
    functions' fp32 results do not."""
    f = torch.finfo(TYPES[type_name][1])
    return f.eps * f.tiny if type_name == "f16" else 4 * f.tiny


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1.0 + np.exp(-v))


def softplus(v):
    return np.maximum(v, 0.0) + np.log1p(np.exp(-np.abs(v)))


def sequences(starts, slots, n_slots, n_tokens, pool=True):
    """(b, first row, last row + 1, slot) of those that the call works on."""
    seen, out = set(), []
    for b in range(len(starts) - 1):
        s = min(max(starts[b], 0), n_tokens)
        e = max(s, min(max(starts[b + 1], 0), n_tokens))
        if not pool:
            out.append((b, s, e, None))
            continue
        k = slots[b] if slots is not None else b
        if 0 <= k < n_slots and k not in seen:
            seen.add(k)
            out.append((b, s, e, k))
    return out


def conv_ref(x, w, bias, act, seqs, pool, fresh=None):
    """{row: y}, {row: bound of |y|'s error before its own rounding}, new pool."""
    W = w.shape[0]
    y, tol = {}, {}
    new = None if pool is None else pool.copy()
    for b, s, e, slot in seqs:
        hist = np.zeros((W - 1, x.shape[1]))
        if slot is not None and not (fresh is not None and fresh[b]):
            hist = pool[slot].copy()
        rows = np.concatenate([hist, x[s:e]])
        for t in range(e - s):
            v = (rows[t:t + W] * w).sum(0) + (0.0 if bias is None else bias)
            mag = np.abs(rows[t:t + W] * w).sum(0) + (0.0 if bias is None else np.abs(bias))
            # the sum's error passes through silu with a slope below 1.1; the
            # function's own error is a few u of its value
            y[s + t] = silu(v) if act else v
            tol[s + t] = 1.1 * (W + 2) * U * mag + (8 * U * np.abs(silu(v)) if act else 0.0)
        if slot is not None:
            new[slot] = rows[e - s:]
    return y, tol, new


def ssm_ref(x, B, Cm, dt, z, A, dt_bias, D, soft, seqs, pool, fresh=None):
    """x, z [T][H][P], B, C [T][G][N], dt [T][H], pool [slots][H][P][N]:
    {row: y}, {row: bound}, new pool, {slot: bound}."""
    H, P = x.shape[1:]
    G, N = B.shape[1:]
    rep = H // G
    y, tol, stol = {}, {}, {}
    new = None if pool is None else pool.copy()
    for b, s, e, slot in seqs:
        S = np.zeros((H, P, N))
        if slot is not None and not (fresh is not None and fresh[b]):
            S = pool[slot].copy()
        M = np.abs(S)
        expo = np.zeros(H)
        for t in range(s, e):
            d = dt[t] + (0.0 if dt_bias is None else dt_bias)
            if soft:
                d = softplus(d)
            a = np.exp(A * d)[:, None, None]
            expo += np.abs(A) * np.abs(d)
            Bt, Ct = np.repeat(B[t], rep, 0)[:, None, :], np.repeat(Cm[t], rep, 0)[:, None, :]
            add = d[:, None, None] * x[t][:, :, None] * Bt
            S = a * S + add
            M = a * M + np.abs(add)
            v, mag = (S * Ct).sum(-1), (M * np.abs(Ct)).sum(-1)
            n = 2 * N + 8 * (t - s + 1) + 32
            err = (n + 8 * expo)[:, None] * U * mag
            if D is not None:
                v = v + D * x[t]
                err = err + 4 * U * np.abs(D * x[t])
            if z is not None:
                g = silu(z[t])
                err = err * np.abs(g) + 10 * U * np.abs(v * g)
                v = v * g
            y[t], tol[t] = v, err
        if slot is not None:
            new[slot] = S
            stol[slot] = (8 * (e - s) + 32 + 8 * expo)[:, None, None] * U * M
    return y, tol, new, stol


def close(got, want, tol, type_name, what):
    """|got - want| <= tol and the rounding of the result's type."""
    h = half_step(type_name)
    lim = tol * (1 + h) + h * np.abs(want) + tiny(type_name)
    bad = ~(np.abs(got - want) <= lim)
    if bad.any():
        i = tuple(int(k[0]) for k in np.nonzero(bad))
        raise AssertionError("%s: %d of %d off, first at %s: %r for %r, allowed %g" % (
            what, bad.sum(), bad.size, i, got[i], want[i], lim[i] if np.ndim(lim) else lim))


def check_rows(buf, view, rows, tols, type_name, shape, what):
    """Rows of y as wanted; every other value of its buffer still MARK."""
    got = f64(view)
    for t, want in rows.items():
        close(got[t].reshape(shape), want, tols[t], type_name, "%s row %d" % (what, t))
    rest = buf.clone()
    off = (view.data_ptr() - buf.data_ptr()) // buf.element_size()
    for t in rows:
        rest[t, off:off + view.shape[1]] = MARK
    assert (rest == MARK).all(), what + ": values outside the sequences' rows changed"


class ConvCase:
    def __init__(self, type_name, channels, width, lens, act=True, bias=True, slots="shuffled",
                 lead=0, row_pad=0, front=0, tail=0, pool=True, seed=0, step=False, spare=2,
                 slot_pad=0):
        r = np.random.default_rng(seed)
        self.type, self.step, self.act, self.width = type_name, step, act, width
        n = len(lens)
        T = n if step else front + sum(lens) + tail
        self.n_tokens = T
        self.starts = list(range(n + 1)) if step else list(front + np.concatenate([[0], np.cumsum(lens)]).astype(int))
        self.buf, (self.x,), self.stride = columns([r.standard_normal((T, channels))], type_name,
                                                   lead, row_pad)
        self.w = gpu(r.standard_normal((width, channels)), torch.float32)
        self.bias = gpu(r.standard_normal(channels), torch.float32) if bias else None
        self.n_slots = n + spare
        self.slots = [int(v) for v in r.permutation(self.n_slots)[:n]] if slots == "shuffled" else slots
        self.fresh = None
        row = (width - 1) * channels
        self.pool_buf = gpu(r.standard_normal((self.n_slots, row + slot_pad)), torch.float32) if pool else None
        self.ybuf, (self.y,), self.ystride = columns([np.full((T, channels), MARK)], type_name,
                                                     lead, row_pad)
        self.channels, self.n = channels, n

    def descriptor(self):
        self.d_start = gpu(np.array(self.starts), torch.int32)
        self.d_slots = gpu(np.array(self.slots), torch.int32) if self.slots is not None and self.n else None
        self.d_fresh = gpu(np.array(self.fresh), torch.uint8) if self.fresh is not None else None
        return bh.Conv(type=TYPES[self.type][0], channels=self.channels, width=self.width,
                       silu=int(self.act), n_seqs=self.n, n_tokens=self.n_tokens,
                       seq_start=at(self.d_start), slots=at(self.d_slots), fresh=at(self.d_fresh),
                       x=at(self.x), x_stride=self.stride, w=at(self.w), bias=at(self.bias),
                       state=at(self.pool_buf), n_slots=self.n_slots,
                       state_stride=0 if self.pool_buf is None else self.pool_buf.shape[1],
                       y=at(self.y), y_stride=self.ystride)

    def pool(self):
        row = (self.width - 1) * self.channels
        return f64(self.pool_buf[:, :row]).reshape(-1, self.width - 1, self.channels)

    def want(self):
        seqs = sequences(self.starts, self.slots, self.n_slots, self.n_tokens, self.pool_buf is not None)
        return conv_ref(f64(self.x), f64(self.w), None if self.bias is None else f64(self.bias),
                        self.act, seqs, None if self.pool_buf is None else self.pool(),
                        None if self.step else self.fresh)

    def run(self, lib, stream=None):
        d = self.descriptor()
        torch.cuda.synchronize()
        f = lib.bm_hip_conv_step_dev if self.step else lib.bm_hip_conv_dev
        bh.check(f(C.byref(d), stream), "conv")
        torch.cuda.synchronize()

    def check(self, lib, what):
        rows, tols, pool = self.want()
        pads = None if self.pool_buf is None else self.pool_buf.clone()
        self.run(lib)
        check_rows(self.ybuf, self.y, rows, tols, self.type, (self.channels,), what)
        if pool is not None:
            assert np.array_equal(self.pool(), pool), what + ": state"
            row = (self.width - 1) * self.channels
            assert torch.equal(pads[:, row:], self.pool_buf[:, row:])


class SsmCase:
    def __init__(self, type_name, H, P, G, N, lens, gate=True, skip=True, bias=True, soft=True,
                 slots="shuffled", lead=0, row_pad=0, front=0, tail=0, pool=True, seed=0,
                 step=False, spare=2, slot_pad=0, rate=4.0):
        r = np.random.default_rng(seed)
        self.type, self.step, self.soft = type_name, step, soft
        self.H, self.P, self.G, self.N, self.n = H, P, G, N, len(lens)
        n = self.n
        T = n if step else front + sum(lens) + tail
        self.n_tokens = T
        self.starts = list(range(n + 1)) if step else list(front + np.concatenate([[0], np.cumsum(lens)]).astype(int))
        dt = r.standard_normal((T, H)) if soft else np.exp(r.uniform(-6, -1, (T, H)))
        parts = [r.standard_normal((T, H * P)), r.standard_normal((T, H * P)),
                 r.standard_normal((T, G * N)), r.standard_normal((T, G * N)), dt]
        self.buf, (self.z, self.x, self.B, self.Cm, self.dt), self.stride = columns(
            parts, type_name, lead, row_pad)
        if not gate:
            self.z = None
        f32 = torch.float32
        self.A = gpu(-np.exp(r.uniform(np.log(0.2), np.log(rate), H)), f32)
        self.dt_bias = gpu(r.uniform(-4, 0, H) if soft else 0.01 * r.random(H), f32) if bias else None
        self.D = gpu(r.standard_normal((H, P)), f32) if skip else None
        self.n_slots = n + spare
        self.slots = [int(v) for v in r.permutation(self.n_slots)[:n]] if slots == "shuffled" else slots
        self.fresh = None
        self.pool_buf = gpu(r.standard_normal((self.n_slots, H * P * N + slot_pad)), f32) if pool else None
        self.ybuf, (self.y,), self.ystride = columns([np.full((T, H * P), MARK)], type_name, lead,
                                                     row_pad)
        self.work = None

    def descriptor(self):
        self.d_start = gpu(np.array(self.starts), torch.int32)
        self.d_slots = gpu(np.array(self.slots), torch.int32) if self.slots is not None and self.n else None
        self.d_fresh = gpu(np.array(self.fresh), torch.uint8) if self.fresh is not None else None
        s = self.stride
        return bh.Ssm(type=TYPES[self.type][0], n_heads=self.H, head_dim=self.P, n_groups=self.G,
                      d_state=self.N, dt_softplus=int(self.soft), n_seqs=self.n,
                      n_tokens=self.n_tokens, seq_start=at(self.d_start), slots=at(self.d_slots),
                      fresh=at(self.d_fresh), x=at(self.x), B=at(self.B), C=at(self.Cm),
                      dt=at(self.dt), z=at(self.z), x_stride=s, B_stride=s, C_stride=s,
                      dt_stride=s, z_stride=s, A=at(self.A), dt_bias=at(self.dt_bias),
                      D=at(self.D), state=at(self.pool_buf), n_slots=self.n_slots,
                      state_stride=0 if self.pool_buf is None else self.pool_buf.shape[1],
                      y=at(self.y), y_stride=self.ystride)

    def pool(self):
        row = self.H * self.P * self.N
        return f64(self.pool_buf[:, :row]).reshape(-1, self.H, self.P, self.N)

    def want(self):
        seqs = sequences(self.starts, self.slots, self.n_slots, self.n_tokens, self.pool_buf is not None)
        T, o = self.x.shape[0], lambda t: None if t is None else f64(t)
        v = lambda t, *sh: f64(t).reshape(T, *sh)
        return ssm_ref(v(self.x, self.H, self.P), v(self.B, self.G, self.N),
                       v(self.Cm, self.G, self.N), v(self.dt, self.H),
                       None if self.z is None else v(self.z, self.H, self.P), o(self.A),
                       o(self.dt_bias), o(self.D), self.soft, seqs,
                       None if self.pool_buf is None else self.pool(),
                       None if self.step else self.fresh)

    def workspace(self, lib, d):
        """Filled with NaN: a call must not read what it has not written."""
        n = lib.bm_hip_ssm_workspace_bytes(C.byref(d))
        self.work = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") if n else None
        return at(self.work)

    def run(self, lib, stream=None):
        d = self.descriptor()
        w = None if self.step else self.workspace(lib, d)
        torch.cuda.synchronize()
        if self.step:
            bh.check(lib.bm_hip_ssm_step_dev(C.byref(d), stream), "ssm_step")
        else:
            bh.check(lib.bm_hip_ssm_dev(C.byref(d), w, stream), "ssm")
        torch.cuda.synchronize()

    def check(self, lib, what):
        rows, tols, pool, stol = self.want()
        before = None if self.pool_buf is None else self.pool_buf.clone()
        self.run(lib)
        check_rows(self.ybuf, self.y, rows, tols, self.type, (self.H, self.P), what)
        if pool is not None:
            got = self.pool()
            row = self.H * self.P * self.N
            for k in range(self.n_slots):
                if k in stol:
                    close(got[k], pool[k], stol[k], "f32", "%s slot %d" % (what, k))
                else:
                    assert torch.equal(before[k], self.pool_buf[k]), "%s: slot %d changed" % (what, k)
            assert torch.equal(before[:, row:], self.pool_buf[:, row:])
