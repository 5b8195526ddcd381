// The gated delta rule for many sequences: the state S [head_dim][d_state] of a
// head is a table from keys to values, each row's key and value are written
// into it, and its query is read from it (include/bm_hip.h):
//
//   S = a S,  w = b (v - S k),  S = S + w k^T,  y = scale (S q) silu(z)
//
// State, sums and decays in fp32 or more; y rounded once.
#include <math.h>

#include "bm_dev.h"
#include "bm_mma.h"
#include "bm_seq.h"

namespace bm {

struct DeltaArgs {
  SeqView q;
  int heads, hd, groups, n;  // hd: head_dim, n: d_state
  bool softplus, sigmoid, norm, frozen;
  bool wide;  // four values of a row of Q or K lie on one load's alignment
  float eps, scale;
  const void *Q, *K, *v, *dt, *beta, *z;
  int64_t Qs, Ks, vs, dts, bs, zs;
  const float *A, *dt_bias;
  float* state;
  int64_t ss;
  void* y;
  int64_t ys;
};

// the exponent of a row's decay, at most 0 (NaN stays)
__device__ __forceinline__ float exponent_of(const DeltaArgs& a, float A, float dt, float bias) {
  if (!a.A) return 0.0f;
  dt += bias;
  const float p = A * (a.softplus ? softplus_f32(dt) : dt);
  return p > 0.0f ? 0.0f : p;
}
__device__ __forceinline__ float beta_of(const DeltaArgs& a, float b) {
  if (!a.beta) return 1.0f;
  return a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_f32(-b)) : b;
}
// 1 / sqrt(squares + eps); NaN where the squares' sum is not finite
__device__ __forceinline__ float unit_of(const DeltaArgs& a, float squares) {
  if (!a.norm) return 1.0f;
  return squares < __builtin_inff() ? __builtin_amdgcn_rsqf(squares + a.eps) : __builtin_nanf("");
}

// sum over teams of T neighbouring lanes, in every lane of the team
template <int T>
__device__ __forceinline__ float team_add(float v) {
  if (T > 1) v += __int_as_float(dpp_mov<0xB1>(__float_as_int(v)));
  if (T > 2) v += __int_as_float(dpp_mov<0x4E>(__float_as_int(v)));
  if (T > 4) v += __int_as_float(dpp_mov<0x141>(__float_as_int(v)));
  if (T > 8) v += __int_as_float(dpp_mov<0x140>(__float_as_int(v)));
#pragma unroll
  for (int m = 16; m < T; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// V neighbouring values of a row as the load leaves them
template <typename T, int V>
struct RawRow {
  Raw4<T> w;
};
template <typename T>
struct RawRow<T, 1> {
  uint32_t w;
};
template <typename T, int V>
__device__ __forceinline__ RawRow<T, V> load_values(__amdgpu_buffer_rsrc_t r, uint32_t off, int n,
                                                    int d_state, bool wide) {
  RawRow<T, V> o;
  if constexpr (V == 1) {
    o.w = load_raw<T>(r, n < d_state ? off : kNoColumn);
  } else if (wide) {
    o.w = load_raw4<T>(r, n < d_state ? off : kNoColumn);
  } else {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = load_raw<T>(r, n + i < d_state ? off + i * (uint32_t)sizeof(T) : kNoColumn);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i)
      o.w.w[i] = sizeof(T) == 2 ? v[2 * i & 3] | v[(2 * i + 1) & 3] << 16 : v[i];
  }
  return o;
}
template <typename T, int V>
__device__ __forceinline__ float value_of(const RawRow<T, V>& r, int i) {
  if constexpr (V == 1) return raw_f32<T>(r.w);
  else return raw4_f32<T>(r.w, i);
}

// ---------------------------------------------------------------------------
// Row after row.  A team of TEAM lanes holds one row of the state, V
// neighbouring values per lane and step of E; a wave takes 64 / TEAM rows at
// once and U such groups.  S k and S q are both taken from the state before
// the row, so that a row of the sequence reads it once:
//   S' q = a (S q) + w (k . q).
// ---------------------------------------------------------------------------
template <typename T, int TEAM, int V, int E, int U, bool STREAM, bool STEP>
__global__ __launch_bounds__(256) void k_delta_rows(DeltaArgs a) {
  constexpr int kRows = 64 / TEAM;
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p0 = (blockIdx.z * (blockDim.x >> 6) + wave) * (kRows * U) + lane / TEAM;
  const int nl = (lane % TEAM) * V;
  const int slots = first_slots(a.q);
  int t0 = b, t1 = b + 1;
  if (!STEP) {
    t0 = a.q.seq_start ? seq_row(a.q, b) : 0;
    t1 = a.q.seq_start ? seq_row(a.q, b + 1) : a.q.n_tokens;
  }
  const int slot = find_slot(a.q, b, slots);
  if (slot == kNoSlot) return;
  const bool keep = slot >= 0 && !(!STEP && a.q.fresh && a.q.fresh[b]);
  if (!STEP && t1 <= t0 && (keep || slot < 0)) return;  // no rows, and nothing to start from zeros
  const int g = h / (a.heads / a.groups);
  const float A = a.A ? a.A[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  // the head's part of the slot and of rows; what lies past them reads as
  // zeros and is not written
  const auto st = rows_at(a.state + (slot >= 0 ? (int64_t)slot * a.ss : 0) + (int64_t)h * a.hd * a.n,
                          slot >= 0 ? (uint32_t)(a.hd * a.n * 4) : 0);
  const uint32_t head = (uint32_t)(a.hd * sizeof(T)), gn = (uint32_t)(a.n * sizeof(T));
  const int64_t col = (int64_t)h * a.hd, gcol = (int64_t)g * a.n;

  float s[U][E][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
      const int p = p0 + u * kRows;
      load_floats<V, STREAM>(s[u][e], st,
                             keep && n < a.n ? (uint32_t)((p * a.n + n) * 4) : kNoColumn);
    }

  RawRow<T, V> kr[E], qr[E];
  uint32_t vr[U], zr[U], dtr = 0, br = 0;
  auto fetch = [&](int64_t t) {
    const auto bk = rows_at((const T*)a.K + t * a.Ks + gcol, gn);
    const auto bq = rows_at((const T*)a.Q + t * a.Qs + gcol, gn);
    const auto bv = rows_at((const T*)a.v + t * a.vs + col, head);
    const auto bz = rows_at((const T*)a.z + t * a.zs + col, a.z ? head : 0);
    const uint32_t one = sizeof(T);
    dtr = load_raw<T>(rows_at((const T*)a.dt + t * a.dts + h, a.A ? one : 0), 0);
    br = load_raw<T>(rows_at((const T*)a.beta + t * a.bs + h, a.beta ? one : 0), 0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
      kr[e] = load_values<T, V>(bk, (uint32_t)(n * sizeof(T)), n, a.n, a.wide);
      qr[e] = load_values<T, V>(bq, (uint32_t)(n * sizeof(T)), n, a.n, a.wide);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vr[u] = load_raw<T>(bv, (uint32_t)((p0 + u * kRows) * sizeof(T)));
      zr[u] = load_raw<T>(bz, (uint32_t)((p0 + u * kRows) * sizeof(T)));
    }
  };
  if (t0 < t1) fetch(t0);
  for (int64_t t = t0; t < t1; ++t) {
    float k[E][V], q[E][V], v[U], z[U], kk = 0.0f, qq = 0.0f, qk = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        k[e][i] = value_of<T, V>(kr[e], i);
        q[e][i] = value_of<T, V>(qr[e], i);
        kk = __builtin_fmaf(k[e][i], k[e][i], kk);
        qq = __builtin_fmaf(q[e][i], q[e][i], qq);
        qk = __builtin_fmaf(q[e][i], k[e][i], qk);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = raw_f32<T>(vr[u]);
      z[u] = raw_f32<T>(zr[u]);
    }
    const float beta = beta_of(a, raw_f32<T>(br));
    const Decay decay = decay_of(exponent_of(a, A, raw_f32<T>(dtr), bias));
    if (!STEP && t + 1 < t1) fetch(t + 1);
    const float uk = unit_of(a, team_add<TEAM>(kk));
    const float uq = a.scale * unit_of(a, team_add<TEAM>(qq));
    qk = team_add<TEAM>(qk) * uk * uq;
    const auto by = rows_at((const T*)a.y + t * a.ys + col, head);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sk = __builtin_fmaf(s[u][e][i], k[e][i], sk);
          sq = __builtin_fmaf(s[u][e][i], q[e][i], sq);
        }
      sk = team_add<TEAM>(sk) * uk;
      sq = team_add<TEAM>(sq) * uq;
      const float w = beta * (v[u] - __builtin_fmaf(sk, decay.lo, sk * decay.hi));
      const float wk = w * uk;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i)
          s[u][e][i] = __builtin_fmaf(s[u][e][i], decay.hi,
                                      __builtin_fmaf(s[u][e][i], decay.lo, wk * k[e][i]));
      float y = __builtin_fmaf(sq, decay.lo, sq * decay.hi);
      y = __builtin_fmaf(w, qk, y);
      if (a.z) y *= silu_f32(z[u]);
      const float out[1] = {y};
      store_row<T, 1>(by, lane % TEAM == 0 ? (uint32_t)((p0 + u * kRows) * sizeof(T)) : kNoColumn,
                      out);
    }
  }
  if (a.frozen) return;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
      const int p = p0 + u * kRows;
      store_floats<V, STREAM>(st, n < a.n ? (uint32_t)((p * a.n + n) * 4) : kNoColumn, s[u][e]);
    }
}

template <typename T, int TEAM, int V, int E, bool STEP>
static hipError_t launch_rows(const DeltaArgs& a, hipStream_t s) {
  constexpr int U = E >= 4 ? 2 : (E == 2 ? 4 : (TEAM >= 16 ? (STEP ? 8 : 4) : 2));
  constexpr int kRows = 64 / TEAM * U;  // rows of the state per wave
  const int waves = (a.hd + kRows - 1) / kRows;
  const int nw = waves < 4 ? waves : 4;
  const dim3 grid(a.q.n_seqs, a.heads, (waves + nw - 1) / nw);
  // as the scan's single tokens: states of 64 MiB or more go past the caches
  constexpr bool kLarge = STEP && V == 4 && TEAM >= 4;
  if (kLarge && (int64_t)a.q.n_seqs * a.heads * a.hd * a.n >= (1 << 24))
    return launch(k_delta_rows<T, TEAM, V, E, U, kLarge, STEP>, grid, dim3(64 * nw), 0, s, a);
  return launch(k_delta_rows<T, TEAM, V, E, U, false, STEP>, grid, dim3(64 * nw), 0, s, a);
}

template <typename T, bool STEP>
static hipError_t launch_rows_t(const DeltaArgs& a, hipStream_t s) {
  if (a.n % 4 == 0) {  // a state row's loads of four floats need no more than a float's alignment
    if (a.n <= 16) return launch_rows<T, 4, 4, 1, STEP>(a, s);
    if (a.n <= 32) return launch_rows<T, 8, 4, 1, STEP>(a, s);
    if (a.n <= 64) return launch_rows<T, 16, 4, 1, STEP>(a, s);
    if (a.n <= 128) return launch_rows<T, 16, 4, 2, STEP>(a, s);
    return launch_rows<T, 16, 4, 4, STEP>(a, s);
  }
  if (a.n <= 4) return launch_rows<T, 4, 1, 1, STEP>(a, s);
  if (a.n <= 16) return launch_rows<T, 16, 1, 1, STEP>(a, s);
  if (a.n <= 64) return launch_rows<T, 16, 1, 4, STEP>(a, s);
  return launch_rows<T, 64, 1, 4, STEP>(a, s);
}

static bool delta_fits(const char* name, const bm_hip_delta_t* op) {
  if (!op) {
    bm_set_error("%s: no descriptor", name);
    return false;
  }
  if (op->type < BM_HIP_F32 || op->type > BM_HIP_F16 || op->n_heads < 1 || op->n_heads > 65535 ||
      op->head_dim < 1 || op->head_dim > 65535 || op->n_groups < 1 ||
      op->n_heads % op->n_groups || op->d_state < 1 || op->d_state > 256 ||
      (int64_t)op->n_heads * op->head_dim > (1 << 21)) {
    bm_set_error("%s: invalid arguments (type=%d n_heads=%d head_dim=%d n_groups=%d d_state=%d)",
                 name, op->type, op->n_heads, op->head_dim, op->n_groups, op->d_state);
    return false;
  }
  return true;
}

}  // namespace bm

extern "C" size_t bm_hip_delta_workspace_bytes(const bm_hip_delta_t* op) {
  if (!bm::delta_fits("delta_workspace", op) || op->n_tokens < 0 || op->n_seqs < 0) return 0;
  return 0;
}

static int delta_call(const bm_hip_delta_t* op, void* workspace, void* stream, bool step) {
  const char* name = step ? "delta_step" : "delta";
  if (!bm::delta_fits(name, op)) return -2;
  const int64_t hp = (int64_t)op->n_heads * op->head_dim, gn = (int64_t)op->n_groups * op->d_state;
  const size_t elem = bm::type_bytes(op->type);
  const int64_t rows = step ? op->n_seqs : op->n_tokens;
  if (!bm::check_seqs(name, op->n_seqs, op->n_tokens, op->seq_start, op->slots, op->state,
                      op->state_stride, op->n_slots, hp * op->d_state, step))
    return -2;
  if ((op->qk_norm && !(op->norm_eps >= 0x1p-100f && op->norm_eps < INFINITY)) ||
      !isfinite(op->scale)) {
    bm_set_error("%s: norm_eps=%g (2^-100 and more) scale=%g", name, op->norm_eps, op->scale);
    return -2;
  }
  const struct {
    const char* name;
    const void* p;
    int64_t stride, width;
    bool given, own;  // own: each thread reads it only where it writes y
  } in[] = {{"q", op->q, op->q_stride, gn, true, false},
            {"k", op->k, op->k_stride, gn, true, false},
            {"v", op->v, op->v_stride, hp, true, true},
            {"dt", op->dt, op->dt_stride, op->n_heads, op->A != nullptr, false},
            {"beta", op->beta, op->beta_stride, op->n_heads, op->beta != nullptr, false},
            {"z", op->z, op->z_stride, hp, op->z != nullptr, op->z == op->v}};
  if (!bm::check_rows(name, "y", op->y, op->y_stride, hp, rows, elem)) return -2;
  for (const auto& t : in) {
    if (!t.given) continue;
    if (!bm::check_rows(name, t.name, t.p, t.stride, t.width, rows, elem) ||
        !bm::check_apart(name, t.name, t.p, t.stride, t.width, op->y, op->y_stride, hp, rows, elem,
                         step && t.own))
      return -2;
  }
  if (((uintptr_t)op->A | (uintptr_t)op->dt_bias) % 4) {
    bm_set_error("%s: A and dt_bias need addresses on 4 bytes", name);
    return -2;
  }
  (void)workspace;
  if (op->n_seqs == 0) return 0;
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  bm::DeltaArgs a;
  a.q = bm::SeqView{op->seq_start, op->state ? op->slots : nullptr, op->fresh, op->n_seqs,
                    op->n_tokens, op->state ? op->n_slots : 0};
  a.heads = op->n_heads;
  a.hd = op->head_dim;
  a.groups = op->n_groups;
  a.n = op->d_state;
  a.softplus = op->dt_softplus != 0;
  a.sigmoid = op->beta_sigmoid != 0;
  a.norm = op->qk_norm != 0;
  a.frozen = op->frozen != 0 || !op->state;
  a.wide = op->d_state % 4 == 0 && op->q_stride % 4 == 0 && op->k_stride % 4 == 0 &&
           ((uintptr_t)op->q | (uintptr_t)op->k) % (4 * elem) == 0;
  a.eps = op->norm_eps;
  a.scale = op->scale;
  a.Q = op->q;
  a.K = op->k;
  a.v = op->v;
  a.dt = op->dt;
  a.beta = op->beta;
  a.z = op->z;
  a.Qs = op->q_stride;
  a.Ks = op->k_stride;
  a.vs = op->v_stride;
  a.dts = op->dt_stride;
  a.bs = op->beta_stride;
  a.zs = op->z_stride;
  a.A = op->A;
  a.dt_bias = op->dt_bias;
  a.state = op->state;
  a.ss = op->state_stride;
  a.y = op->y;
  a.ys = op->y_stride;
  hipStream_t s = bm::stream_of(stream);
  hipError_t e;
  switch (op->type) {
    case BM_HIP_F32:
      e = step ? bm::launch_rows_t<float, true>(a, s) : bm::launch_rows_t<float, false>(a, s);
      break;
    case BM_HIP_BF16:
      e = step ? bm::launch_rows_t<__bf16, true>(a, s) : bm::launch_rows_t<__bf16, false>(a, s);
      break;
    default:
      e = step ? bm::launch_rows_t<_Float16, true>(a, s)
               : bm::launch_rows_t<_Float16, false>(a, s);
      break;
  }
  BM_HIP_CHECK_RET(e, -1);
  return 0;
}

extern "C" int bm_hip_delta_dev(const bm_hip_delta_t* op, void* workspace, void* stream) {
  return delta_call(op, workspace, stream, false);
}

extern "C" int bm_hip_delta_step_dev(const bm_hip_delta_t* op, void* stream) {
  return delta_call(op, nullptr, stream, true);
}
