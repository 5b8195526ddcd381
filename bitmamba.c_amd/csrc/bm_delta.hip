// The gated delta rule for many sequences: the state S [head_dim][d_state] of a
// head is a table from keys to values, each row's key and value are written
// into it, and its query is read from it (include/bm_hip.h):
//
//   S = a S,  w = b (v - S k),  S = S + w k^T,  y = scale (S q) silu(z)
//
// State, sums and decays in fp32 or more; y rounded once.
#include <math.h>

#include "bm_dev.h"
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
// (NaN for an infinite one, which would leave infinities of either sign)
__device__ __forceinline__ float beta_of(const DeltaArgs& a, float b) {
  if (!a.beta) return 1.0f;
  if (a.sigmoid) return __builtin_amdgcn_rcpf(1.0f + exp_f32(-b));
  return __builtin_fabsf(b) < __builtin_inff() ? b : __builtin_nanf("");
}
// what a row of q or k is multiplied by; NaN where its squares' sum is not finite
__device__ __forceinline__ float unit_of(const DeltaArgs& a, float squares) {
  const float unit = a.norm ? __builtin_amdgcn_rsqf(squares + a.eps) : 1.0f;
  return squares < __builtin_inff() ? unit : __builtin_nanf("");
}

// a permutation of all lanes of a row, in the form that an addition takes in
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over teams of T neighbouring lanes, in every lane of the team
template <int T>
__device__ __forceinline__ float team_add(float v) {
  if (T > 1) v += dpp_f32<0xB1>(v);
  if (T > 2) v += dpp_f32<0x4E>(v);
  if (T > 4) v += dpp_f32<0x141>(v);
  if (T > 8) v += dpp_f32<0x140>(v);
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
// One row per sequence.  A team of TEAM lanes holds one row of the state, V
// neighbouring values per lane and step of E; a wave takes 64 / TEAM rows at
// once and U such groups.  S k and S q are both taken from the state before
// the row, so that it is read once:
//   S' q = a (S q) + w (k . q).
// The state's bytes bound it: 128 sequences of 32 heads of 128 x 128 move 541 MB
// in 95 us, 5.7 TB/s; one sequence (4.3 MB) takes 4.2 us, a launch's latency.
// ---------------------------------------------------------------------------
template <typename T, int TEAM, int V, int E, int U, bool STREAM>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a) {
  constexpr int kRows = 64 / TEAM;
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p0 = (blockIdx.z * (blockDim.x >> 6) + wave) * (kRows * U) + lane / TEAM;
  const int nl = (lane % TEAM) * V;
  const int slot = find_slot(a.q, b, first_slots(a.q));
  if (slot == kNoSlot) return;
  const bool keep = slot >= 0;
  const int g = h / (a.heads / a.groups);
  const float A = a.A ? a.A[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  // the head's part of the slot and of rows; what lies past them reads as
  // zeros and is not written
  const auto st = rows_at(a.state + (keep ? (int64_t)slot * a.ss : 0) + (int64_t)h * a.hd * a.n,
                          keep ? (uint32_t)(a.hd * a.n * 4) : 0);
  const uint32_t head = (uint32_t)(a.hd * sizeof(T)), gn = (uint32_t)(a.n * sizeof(T));
  const int64_t t = b, col = (int64_t)h * a.hd, gcol = (int64_t)g * a.n;

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
  uint32_t vr[U], zr[U];
  const auto bk = rows_at((const T*)a.K + t * a.Ks + gcol, gn);
  const auto bq = rows_at((const T*)a.Q + t * a.Qs + gcol, gn);
  const auto bv = rows_at((const T*)a.v + t * a.vs + col, head);
  const auto bz = rows_at((const T*)a.z + t * a.zs + col, a.z ? head : 0);
  const auto by = rows_at((const T*)a.y + t * a.ys + col, head);
  const uint32_t one = sizeof(T);
  const uint32_t dtr = load_raw<T>(rows_at((const T*)a.dt + t * a.dts + h, a.A ? one : 0), 0);
  const uint32_t br = load_raw<T>(rows_at((const T*)a.beta + t * a.bs + h, a.beta ? one : 0), 0);
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

  float k[E][V], q[E][V], kk = 0.0f, qq = 0.0f, qk = 0.0f;
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
  const float beta = beta_of(a, raw_f32<T>(br));
  const Decay decay = decay_of(exponent_of(a, A, raw_f32<T>(dtr), bias));
  const float uk = unit_of(a, team_add<TEAM>(kk));
  const float uq = a.scale * unit_of(a, team_add<TEAM>(qq));
  qk = team_add<TEAM>(qk) * uk * uq;
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
    const float w = beta * (raw_f32<T>(vr[u]) - __builtin_fmaf(sk, decay.lo, sk * decay.hi));
    const float wk = w * uk;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i)
        s[u][e][i] = __builtin_fmaf(s[u][e][i], decay.hi,
                                    __builtin_fmaf(s[u][e][i], decay.lo, wk * k[e][i]));
    float y = __builtin_fmaf(sq, decay.lo, sq * decay.hi);
    y = __builtin_fmaf(w, qk, y);
    if (a.z) y *= silu_f32(raw_f32<T>(zr[u]));
    const float out[1] = {y};
    store_row<T, 1>(by, lane % TEAM == 0 ? (uint32_t)((p0 + u * kRows) * sizeof(T)) : kNoColumn,
                    out);
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

template <typename T, int TEAM, int V, int E>
static hipError_t launch_step(const DeltaArgs& a, hipStream_t s) {
  // Groups of rows per wave, with half and with twice as many: 128 sequences of 32
  // heads of 128 take, with 8 values of state, 13.5 us against 20.4 and 10.2, with 32
  // 26.8 (38.4, 25.8), with 64 47.6 (46.2, 48.5), with 128 94.7 (93.0, 91.8); 16
  // sequences with 64 values 9.4 (9.1, 10.9), with 128 13.1 (12.3, 14.5).
  constexpr int U = E >= 4 ? 2 : (E == 2 ? 4 : (TEAM >= 16 ? 8 : 2));
  constexpr int kRows = 64 / TEAM * U;  // rows of the state per wave
  const int waves = (a.hd + kRows - 1) / kRows;
  const int nw = waves < 4 ? waves : 4;
  const dim3 grid(a.q.n_seqs, a.heads, (waves + nw - 1) / nw);
  // States of 64 MiB or more go past the caches: 32 heads of 128 x 128 of 32, 64 and 128
  // sequences that lie in turn in memory take 28.3, 51.7 and 95.2 us, through
  // the caches 34.3, 58.3 and 105.4.
  constexpr bool kLarge = V == 4;
  if (kLarge && (int64_t)a.q.n_seqs * a.heads * a.hd * a.n >= (1 << 24))
    return launch(k_delta_step<T, TEAM, V, E, U, kLarge>, grid, dim3(64 * nw), 0, s, a);
  return launch(k_delta_step<T, TEAM, V, E, U, false>, grid, dim3(64 * nw), 0, s, a);
}

template <typename T>
static hipError_t launch_step_t(const DeltaArgs& a, hipStream_t s) {
  // Other teams, for 16 and for 128 sequences as above: 64 values in 8 lanes 9.3 and
  // 47.8 us (in 16: 9.4 and 47.6), 128 in 32 lanes 14.1 and 95.4 (13.1 and 94.7), 61
  // values one by one in 64 lanes 12.4 and 73.5 (in 16: 9.7 and 74.2).
  if (a.n % 4 == 0) {  // a state row's loads of four floats need no more than a float's alignment
    if (a.n <= 16) return launch_step<T, 4, 4, 1>(a, s);
    if (a.n <= 32) return launch_step<T, 8, 4, 1>(a, s);
    if (a.n <= 64) return launch_step<T, 16, 4, 1>(a, s);
    if (a.n <= 128) return launch_step<T, 16, 4, 2>(a, s);
    return launch_step<T, 16, 4, 4>(a, s);
  }
  if (a.n <= 4) return launch_step<T, 4, 1, 1>(a, s);
  if (a.n <= 16) return launch_step<T, 16, 1, 1>(a, s);
  if (a.n <= 64) return launch_step<T, 16, 1, 4>(a, s);
  return launch_step<T, 64, 1, 4>(a, s);
}

// ---------------------------------------------------------------------------
// A few rows per sequence: kFew at a time.  What the state of before them gives
// each row's key and query, X = [K Q]^T S, is one product on the matrix cores, in
// fp32 as the state is; with G = [K Q]^T [K Q] the rest needs no more than kFew
// numbers per row of the state.  With P_j the product of the decays up to row j
// and wu_i = (what row i wrote) / |k_i|, decayed up to j, row j writes and reads
//   w_j = b_j (v_j - (P_j X_j + sum_{i<j} G_ij wu_i) / |k_j|),
//   y_j = (P_j X'_j + sum_{i<=j} G'_ij wu_i) scale / |q_j|,
// and the state after them is P S + sum_i wu_i k_i^T, a product again.
//
// A wave takes M tiles of 16 rows of the state.  A lane of a 16x16x4
// product holds row (or column) lane % 16 of an operand at the step's value
// lane / 16, and rows 4 (lane / 16) .. + 3 of column lane % 16 of the result; four
// steps are four neighbours of a row, so that the state, n = 16 x + 4 (lane / 16)
// and on of row lane % 16, is operand and accumulator as it is loaded.
//
// 64 sequences of 5 rows, 32 heads of 128 x 128 in bf16, take 41 us frozen (134 MB
// read, 3.3 TB/s) and 103 us with the states written (268 MB): two waves per SIMD
// load, multiply (224 products of 32 cycles for four tiles) and store in turn.
// With keys and queries loaded before the state, and the next eight rows' during
// these, the latter takes 5 % less, and one sequence 4 to 15 % more.
// Row after row on the vector units they take 60 us frozen, bound by instructions.
// ---------------------------------------------------------------------------
typedef float v4f __attribute__((ext_vector_type(4)));
// Sequences of up to these rows go this way.  At 32 heads of 128 x 128 in bf16, all of
// the call: 64 sequences of 32 rows 163 us, of 33 rows, in chunks, 338; two
// sequences 27 and 24.
constexpr int kShort = 32;
constexpr int kFew = 8;

// keeps what is cheaply worked out anew from being held in registers over a loop
__device__ __forceinline__ uint32_t anew(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// x[i] of lane group j becomes x[j] of lane group i, groups of 16 lanes
__device__ __forceinline__ void transpose_groups(float (&x)[4]) {
  auto swap = [](auto how, float& a, float& b) {
    const auto r = how(__float_as_uint(a), __float_as_uint(b));
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
  };
  auto halves = [](uint32_t a, uint32_t b) {
    return __builtin_amdgcn_permlane32_swap(a, b, false, false);
  };
  auto rows = [](uint32_t a, uint32_t b) {
    return __builtin_amdgcn_permlane16_swap(a, b, false, false);
  };
  swap(halves, x[0], x[2]);
  swap(halves, x[1], x[3]);
  swap(rows, x[0], x[1]);
  swap(rows, x[2], x[3]);
}

// Two waves per SIMD, one with more than 128 values of state; twice as many of one
// tile, where rows on no load's alignment spill 19 to 29 registers.
template <typename T, int NX, int M, bool WIDE>
__global__ __launch_bounds__(64, (NX > 8 ? 1 : 2) * (M == 1 ? 2 : 1)) void k_delta_few(DeltaArgs a) {
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x, c = lane & 15, q = lane >> 4;
  const int first = blockIdx.z * (16 * M);
  const int t0 = a.q.seq_start ? seq_row(a.q, b) : 0;
  const int t1 = a.q.seq_start ? seq_row(a.q, b + 1) : a.q.n_tokens;
  if (t1 - t0 > kShort) return;
  const int slot = find_slot(a.q, b, first_slots(a.q));
  if (slot == kNoSlot) return;
  const bool keep = slot >= 0 && !(a.q.fresh && a.q.fresh[b]);
  if (t1 <= t0 && (keep || a.frozen || slot < 0)) return;
  const int g = h / (a.heads / a.groups);
  // the head's part of the slot; what lies past it reads as zeros and is not written
  float* const state = a.state + (slot >= 0 ? (int64_t)slot * a.ss : 0) + (int64_t)h * a.hd * a.n;
  const uint32_t state_bytes = (uint32_t)(a.hd * a.n * 4), head = (uint32_t)(a.hd * sizeof(T));
  const int p = first + lane;  // the lane's row of the state
  const uint32_t mine = lane < 16 * M ? (uint32_t)(p * sizeof(T)) : kNoColumn;
  const int64_t col = (int64_t)h * a.hd, gcol = (int64_t)g * a.n;
  auto place = [&](int m, int n) {
    return n < a.n ? (uint32_t)(((first + 16 * m + c) * a.n + n) * 4) : kNoColumn;
  };

  const auto to = rows_at(state, slot >= 0 ? state_bytes : 0);
  if (t1 <= t0) {  // no rows, and a state that begins with zeros
    const float zero[1] = {0.0f};
    for (int m = 0; m < M; ++m)
      for (int n = q; n < a.n; n += 4) store_floats<1>(to, place(m, n), zero);
    return;
  }
  v4f S[M][NX];
  const auto from = rows_at(state, keep ? state_bytes : 0);
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      const int n = 16 * x + 4 * q;
      if constexpr (WIDE) {
        S[m][x] = __builtin_bit_cast(
            v4f, __builtin_amdgcn_raw_buffer_load_b128(from, place(m, n), 0, 0));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[1];
          load_floats<1>(f, from, place(m, n + i));
          S[m][x][i] = f[0];
        }
      }
    }
  // each lane works out one row's decay and b
  static_assert(kShort <= 64, "one for each lane");
  const int64_t own = t0 + min(lane, t1 - t0 - 1);
  const float dt = a.A ? (float)((const T*)a.dt)[own * a.dts + h] : 0.0f;
  const Decay decays =
      decay_of(exponent_of(a, a.A ? a.A[h] : 0.0f, dt, a.dt_bias ? a.dt_bias[h] : 0.0f));
  const float betas = beta_of(a, a.beta ? (float)((const T*)a.beta)[own * a.bs + h] : 0.0f);

  int64_t t = t0;
  do {
    const int rows = min(kFew, (int)(t1 - t));
    // Rows past the last one are that one again: nothing of theirs is used.
    const int64_t r = t + min(c & 7, rows - 1);
    const T* src = c < 8 ? (const T*)a.K + r * a.Ks + gcol : (const T*)a.Q + r * a.Qs + gcol;
    const int nq = (int)anew(4 * q);
    v4f f[NX];
    if constexpr (WIDE) {
      Raw4<T> raw[NX];
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int n = 16 * x + nq;
        raw[x] = *(const Raw4<T>*)__builtin_assume_aligned(src + (n < a.n ? n : 0), 4 * sizeof(T));
      }
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[x][i] = 16 * x + nq < a.n ? raw4_f32<T>(raw[x], i) : 0.0f;
    } else {
      T raw[NX][4];
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[x][i] = src[min(16 * x + nq + i, a.n - 1)];
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[x][i] = 16 * x + nq + i < a.n ? (float)raw[x][i] : 0.0f;
    }
    T v[kFew], z[kFew];
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      const int64_t tj = t + min(j, rows - 1);
      v[j] = ((const T*)a.v + tj * a.vs + col)[min(p, a.hd - 1)];
      if (a.z) z[j] = ((const T*)a.z + tj * a.zs + col)[min(p, a.hd - 1)];
    }
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    v4f G = zero, X[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        G = __builtin_amdgcn_mfma_f32_16x16x4f32(f[x][i], f[x][i], G, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < M; ++m)
          X[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[x][i], S[m][x][i], X[m], 0, 0, 0);
      }
    const bool on = !a.frozen || t + kFew < t1;  // the state is needed again
    T kt[2][NX];
    if (on) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const T* k = (const T*)a.K + (t + min(4 * s + q, rows - 1)) * a.Ks + gcol;
#pragma unroll
        for (int x = 0; x < NX; ++x) kt[s][x] = k[min(16 * x + (int)anew(c), a.n - 1)];
      }
    }
    // 1 / |k| and scale / |q| of row 4 q + i, in lane 16 q + 4 q + i
    const float square = (c & 2) ? ((c & 1) ? G[3] : G[2]) : ((c & 1) ? G[1] : G[0]);
    const float units = unit_of(a, square) * (c < 8 ? 1.0f : a.scale);
    auto unit = [&](int i) { return lane_f32(units, 16 * (i >> 2) + i); };
    auto dot = [&](int i, int j) { return lane_f32(G[i & 3], 16 * (i >> 2) + j); };
    float seen[16];  // X of the lane's row of the state
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4] = {X[0][i], X[1][i], X[2][i], X[3][i]};
      transpose_groups(x);
#pragma unroll
      for (int m = 0; m < 4; ++m) seen[4 * m + i] = x[m];
    }
    Decay all = {1.0f, 0.0f};
    float wu[kFew];
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      wu[j] = 0.0f;
      if (j >= rows) continue;
      const int row = (int)(t - t0) + j;
      const Decay decay = {lane_f32(decays.hi, row), lane_f32(decays.lo, row)};
      const float hi = all.hi * decay.hi;
      const float lo = __builtin_fmaf(all.hi, decay.hi, -hi) +
                       __builtin_fmaf(all.hi, decay.lo, all.lo * decay.hi);
      all.hi = hi + lo;
      all.lo = (hi - all.hi) + lo;
      float sk = __builtin_fmaf(seen[j], all.lo, seen[j] * all.hi);
      float sq = __builtin_fmaf(seen[8 + j], all.lo, seen[8 + j] * all.hi);
#pragma unroll
      for (int i = 0; i < j; ++i) {
        wu[i] *= decay.hi;  // its rounding, 2^-25 of what a row wrote, at most 7 times
        sk = __builtin_fmaf(dot(j, i), wu[i], sk);
        sq = __builtin_fmaf(dot(8 + j, i), wu[i], sq);
      }
      const float uk = unit(j);
      wu[j] = lane_f32(betas, row) * __builtin_fmaf(-uk, sk, (float)v[j]) * uk;
      float y = __builtin_fmaf(dot(8 + j, j), wu[j], sq) * unit(8 + j);
      if (a.z) y *= silu_f32((float)z[j]);
      const float out[1] = {y};
      store_row<T, 1>(rows_at((const T*)a.y + (t + j) * a.ys + col, head), mine, out);
    }
    if (!on) return;
    float w[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[s][i] = wu[4 * s + i];
      transpose_groups(w[s]);
    }
#pragma unroll
    for (int x = 0; x < NX; ++x) {
#pragma unroll
      for (int m = 0; m < M; ++m)
        S[m][x] = __builtin_elementwise_fma(S[m][x], v4f{all.hi, all.hi, all.hi, all.hi},
                                            S[m][x] * all.lo);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < M; ++m)
          S[m][x] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kt[s][x], w[s][m], S[m][x], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);  // in place
    }
    t += kFew;
  } while (t < t1);
  if (a.frozen) return;
  const int nq = (int)anew(4 * q);
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      const int n = 16 * x + nq;
      if constexpr (WIDE) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, S[m][x]), to, place(m, n),
                                               0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f[1] = {S[m][x][i]};
          store_floats<1>(to, place(m, n + i), f);
        }
      }
    }
}

template <typename T, int NX, int M>
static hipError_t launch_few_m(const DeltaArgs& a, hipStream_t s) {
  const dim3 grid(a.q.n_seqs, a.heads, (a.hd + 16 * M - 1) / (16 * M));
  if (a.wide) return launch(k_delta_few<T, NX, M, true>, grid, dim3(64), 0, s, a);
  return launch(k_delta_few<T, NX, M, false>, grid, dim3(64), 0, s, a);
}
template <typename T, int NX>
static hipError_t launch_few(const DeltaArgs& a, hipStream_t s) {
  // One tile per wave while that is up to a wave per SIMD: the wave's own time counts
  // then, and not that each wave works out G.  Sequences of 5 rows, 32 heads of 128 x
  // 128, one tile against four: 1024 tiles 15.3 us against 19.2 (frozen 8.8 and
  // 9.6), 2048 tiles 28.7 against 27.6 (17.0 and 16.3), 4096 51.2 against 46.0.
  const int64_t tiles = (int64_t)a.q.n_seqs * a.heads * ((a.hd + 15) / 16);
  if (tiles <= 1024) return launch_few_m<T, NX, 1>(a, s);
  return launch_few_m<T, NX, (NX > 8 ? 2 : 4)>(a, s);
}

// ---------------------------------------------------------------------------
// Prompts: chunks of kC rows on the matrix cores.  A key is taken as r_i k_i with
// k_i of a length of 1 to 2 (r_i a power of two, and what norm_eps makes of it),
// and instead of w_i, what row i writes, r_i w_i is worked out, which is the size
// of what that leaves in the state whatever the key's length.  With c_i the sum of
// the exponents of a chunk's rows up to i and S the state before it, r w =: w solves
//   w_i + sum_{j<i} L_ij w_j = b_i r_i v_i - b_i r_i^2 e^{c_i} S k_i,
//   L_ij = b_i r_i^2 e^{c_i - c_j} (k_i . k_j),
// so with T = (I + L)^-1 (unit lower triangular) and A_ij = e^{c_i - c_j}
// (q_i . k_j) for j <= i, as products of kC rows
//   R = b r v - b r^2 e^c K S,  w = T R,
//   y = e^c Q S + A w,  S' = e^{c_C} S + K^T (e^{c_C - c} w).
// T and A need no state: the first launch makes them for all chunks and heads
// at once, the second walks each sequence's chunks.
//
// Precision.  MFMA operands are fp16.  A value is one half, or the sum of two
// (22 bits) where it is computed or fp32; what leaves fp16's range of exponents
// is scaled by powers of two: the rows of K, Q, T and A once, the columns of
// the state, R and w (one value of v each) as they grow and shrink.  b is in R, not
// in T: a value that is hardly written, or not at all, must not set that scale.
// The state itself stays in fp32 accumulators.  bf16 in three pieces is as exact
// and needs no scaling, but twice the products and 2.7 times the conversions.
//
// An infinity or NaN must not reach earlier rows of its chunk through a zero
// of T or A: a head's first row of that kind (k, a or b) ends what its chunk
// computes, and a column's (v, or what is computed from it) enters the
// products as zero; the rows from it on and the state become NaN.
// ---------------------------------------------------------------------------
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kC = 64;  // rows of a chunk
template <typename T>
constexpr int kHalves = sizeof(T) == 4 ? 2 : 1;  // of a value of K or Q
constexpr int kTri = 6 * 2 * 1024;  // bytes of T or A: blocks of 16 rows and 32 columns on and below the diagonal
// per place and head after T and A, 64 floats each: b r^2 e^c; b r; e^{c_C - c}; e^c of q; the
// scales of A and T; then the decay (two parts) and the first bad row
enum { kGrowK, kWrite, kLeft, kGrowQ, kFacA, kFacT, kMisc };
constexpr int kScalars = 7 * 256;

struct DeltaPlan {
  bool chunks;     // a sequence may have more than kShort rows
  bool by_rows;    // where a sequence's chunks lie: from row / 32, or from row / kC + b
  bool wide;       // eight values of a row of Q or K on one load's alignment
  int64_t units;   // chunks in the worst case
  int64_t places;
  uint8_t *heads, *keys;  // per place and head: T, A, scalars; per place and group: K, Q, K by columns
  int64_t head_bytes, key_bytes;
  size_t bytes;
};

// Operands.  A lane of a 16x16x32 product holds eight values of row (or column)
// lane % 16, at 8 (lane / 16) and on, and of a result rows 4 (lane / 16) .. + 3
// of column lane % 16.  Row r of tile t stands for row (of the chunk, or
// column of K) spread_row(t, r): the results of tiles 2s and 2s + 1 are then
// eight neighbours, 32 s + 8 (lane / 16) and on, and serve as operands as they are.
__host__ __device__ constexpr int spread_row(int t, int r) {
  return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
}
// where the block of T or A of row tile w and columns 32 s .. lies
__device__ __forceinline__ int tri_block(int w, int s) { return (w < 2 ? w : 2 * w - 2 + s) * 2048; }

// c += (sum of a) (sum of b) without the product of two second halves
template <int NA, int NB>
__device__ __forceinline__ v4f mfma_h(const v8h (&a)[NA], const v8h (&b)[NB], v4f c) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[j], c, 0, 0, 0);
  return c;
}

// two values as halves of a word: the nearest ones, and the nearest to what is left
template <int N>
__device__ __forceinline__ void halves2(uint32_t (&p)[N], float x, float y) {
  v2f v = {x, y};
  p[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2h));
  if constexpr (N == 2) {
    // x - half in one instruction; p[0] waits for x and y, so these do too
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(x) : "v"(p[0]), "v"(x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(y)
        : "v"(p[0]), "v"(y));
    v = v2f{x, y};
    p[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2h));
  }
}
template <int N>
__device__ __forceinline__ void halves8(v8h (&p)[N], const float (&v)[8]) {
  u32x4 w[N];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t o[N];
    halves2<N>(o, v[2 * e], v[2 * e + 1]);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i][e] = o[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = __builtin_bit_cast(v8h, w[i]);
}
template <int N>
__device__ __forceinline__ void halves8(v8h (&p)[N], v4f a, v4f b) {
  const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  halves8<N>(p, v);
}

// the larger magnitude, NaN if either is
__device__ __forceinline__ float max_abs(float m, float a) {
  return __builtin_elementwise_maximum(m, __builtin_fabsf(a));
}
// over the four lanes with one lane % 16, in each of them
template <typename F>
__device__ __forceinline__ float over_quads(float v, F f) {
  uint32_t b = __float_as_uint(v);
  const auto x = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  b = __float_as_uint(f(__uint_as_float(x[0]), __uint_as_float(x[1])));
  const auto y = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return f(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float quads_max(float v) {
  return over_quads(v, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
}
__device__ __forceinline__ float quads_add(float v) {
  return over_quads(v, [](float a, float b) { return a + b; });
}

// the power of two that takes a row's largest magnitude into 1 .. 2, and its inverse
struct Scale {
  float up, down;
};
__device__ __forceinline__ int exponent_bits(float v) { return (int)(__float_as_uint(v) >> 23 & 255); }
__device__ __forceinline__ Scale scale_of_bits(int bits) {
  const int e = min(max(bits, 1), 253);
  return Scale{__uint_as_float((uint32_t)(254 - e) << 23), __uint_as_float((uint32_t)e << 23)};
}
__device__ __forceinline__ Scale scale_of(float largest) { return scale_of_bits(exponent_bits(largest)); }
// the same for its length, given the sum of its squares; lengths below 2^-50,
// whose squares lose bits, go by the largest magnitude
__device__ __forceinline__ Scale scale_of_length(float largest, float squares) {
  const int e = exponent_bits(squares);
  return scale_of_bits(e < 27 || e == 255 ? exponent_bits(largest) : 127 + ((e - 127) >> 1));
}

// a value that all lanes share, in a scalar register: what a buffer's address or
// size is made of (quotients and clamps are worked out in vector registers, and
// a resource in those costs a loop around each access)
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// the block's LDS accesses are done; global ones stay in flight
__device__ __forceinline__ void lds_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ double scan_f64(double v) {  // running sums over the wave
  auto add = [&](auto dpp) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp((int)(uint32_t)b), hi = (uint32_t)dpp((int)(uint32_t)(b >> 32));
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);  // +0 without a source
  };
  add([](int x) { return dpp_or0<0x111>(x); });
  add([](int x) { return dpp_or0<0x112>(x); });
  add([](int x) { return dpp_or0<0x114>(x); });
  add([](int x) { return dpp_or0<0x118>(x); });
  add([](int x) { return dpp_or0<0x142, 0xa>(x); });
  add([](int x) { return dpp_or0<0x143, 0xc>(x); });
  return v;
}

constexpr int kRowL = kC + 4;  // floats of a row of L or T in LDS

// T = (I + L)^-1, both [kC][kRowL] in LDS, in fp32.  Blocks of 16 by
// substitution, a wave each; then blocks of 32 and the whole by
// [[B, 0], [M, D]]^-1 = [[B', 0], [-D' M B', D']], which keeps to the sizes that
// T itself has (sums of powers of L would not).
__device__ __forceinline__ void invert(const float* L, float* T, int wave, int lane) {
  const int c = lane & 15, q = lane >> 4;
  {
    const float* l = L + 16 * wave * kRowL + 16 * wave;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? -1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const float4 v = *(const float4*)(l + i * kRowL + j);
        s = __builtin_fmaf(v.x, x[j], s);
        if (j + 1 < i) s = __builtin_fmaf(v.y, x[j + 1], s);
        if (j + 2 < i) s = __builtin_fmaf(v.z, x[j + 2], s);
        if (j + 3 < i) s = __builtin_fmaf(v.w, x[j + 3], s);
      }
      x[i] = -s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((i & 3) == q) T[(16 * wave + i) * kRowL + 16 * wave + c] = x[i];
  }
  lds_sync();
  // d += block (bi, bk) of M times p, whose lane holds rows 4 q + i of 16
  auto times = [&](const float* M, int bi, int bk, const float (&p)[4], v4f d) {
    const float4 m = *(const float4*)(M + (16 * bi + c) * kRowL + 16 * bk + 4 * q);
    const float mv[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x4f32(mv[i], p[i], d, 0, 0, 0);
    return d;
  };
  auto block_of = [&](int bi, int bj, float (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = T[(16 * bi + 4 * q + i) * kRowL + 16 * bj + c];
  };
  auto put = [&](int bi, int bj, v4f d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) T[(16 * bi + 4 * q + i) * kRowL + 16 * bj + c] = -d[i];
  };
  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
  if (wave < 2) {
    const int bi = 2 * wave + 1, bj = 2 * wave;
    float p[4];
    block_of(bj, bj, p);
    const v4f m = times(L, bi, bj, p, zero);
    const float mv[4] = {m[0], m[1], m[2], m[3]};
    put(bi, bj, times(T, bi, bi, mv, zero));
  }
  lds_sync();
  {
    const int ra = wave >> 1, cb = wave & 1;
    v4f d = zero;
    for (int k = 0; k <= ra; ++k) {  // row k of L's block times column cb of T's first
      v4f m = zero;
      for (int e = cb; e < 2; ++e) {
        float p[4];
        block_of(e, cb, p);
        m = times(L, 2 + k, e, p, m);
      }
      const float mv[4] = {m[0], m[1], m[2], m[3]};
      d = times(T, 2 + ra, 2 + k, mv, d);
    }
    put(2 + ra, cb, d);
  }
  lds_sync();
}

// eight values of a row as the loads leave them
template <typename T, bool WIDE>
struct Eight {
  uint32_t w[WIDE ? 2 * sizeof(T) : 8];
};
template <typename T, bool WIDE>
__device__ __forceinline__ Eight<T, WIDE> load_eight(__amdgpu_buffer_rsrc_t r, uint32_t off, int n,
                                                     int d_state) {
  Eight<T, WIDE> o;
  if constexpr (WIDE) {
    const uint32_t at = n < d_state ? off : kNoColumn;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * k, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) o.w[4 * k + i] = v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      o.w[i] = load_raw<T>(r, n + i < d_state ? off + i * (uint32_t)sizeof(T) : kNoColumn);
  }
  return o;
}
template <typename T, bool WIDE>
__device__ __forceinline__ float eight_f32(const Eight<T, WIDE>& e, int i) {
  if constexpr (!WIDE) return raw_f32<T>(e.w[i]);
  else if constexpr (sizeof(T) == 4) return __uint_as_float(e.w[i]);
  else return (float)__builtin_bit_cast(T, (uint16_t)(e.w[i >> 1] >> (16 * (i & 1))));
}

// ---------------------------------------------------------------------------
// One chunk of one head: T, A and the rows' scalars; for a group's first head
// also K and Q as operands.  Wave w has the rows of tile w (spread_row).
// 16384 rows at 32 heads of 128 in 16 groups take 140 us: 415 MB written, 336 MB
// read, vector instructions on 43 % of the cycles.  An earlier form of 143 us took 120
// without the operands of K and Q, 127 without the inverse, 98 without both.  What
// it waits for are its own steps: with the heads of a group on one XCD it read 133 MB
// in the same time, with two and with three waves per SIMD too; four (128 registers,
// with spills) took 184 us.  A short prompt (1024 rows of fp32) takes 31 us.
// ---------------------------------------------------------------------------
template <typename T, int NK, bool WIDE>
__global__ __launch_bounds__(256) void k_delta_chunk(DeltaArgs a, DeltaPlan pl) {
  constexpr int KP = kHalves<T>, kTile = NK * KP * 1024;  // bytes of 16 rows
  constexpr int kShared = 4 * kTile > kC * kRowL * 4 ? 4 * kTile : kC * kRowL * 4;
  __shared__ __attribute__((aligned(16))) uint8_t shK[kShared];  // K; then T
  __shared__ __attribute__((aligned(16))) float shL[kC * kRowL];
  __shared__ __attribute__((aligned(16))) float shHi[kC], shLo[kC];
  __shared__ float shKk[kC], shKd[kC], shQf[kC];
  float* shT = (float*)shK;
  Unit u = find_unit(a.q, (int)wide_block(), kC);
  u = Unit{uniform(u.b), uniform(u.k), uniform(u.s), uniform(u.e)};
  if (u.b < 0 || u.e - u.s <= kShort) return;
  const int t0 = u.s + u.k * kC;
  if (t0 >= u.e) return;
  const int rows = min(kC, u.e - t0);
  const int64_t place = (pl.by_rows ? u.s / 32 : (int64_t)(u.s / kC) + u.b) + u.k;
  const int h = blockIdx.y, per = a.heads / a.groups, g = uniform(h / per);
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = uniform(tid >> 6);
  uint8_t* out = pl.heads + (place * a.heads + h) * pl.head_bytes;
  uint8_t* keys = pl.keys + (place * a.groups + g) * pl.key_bytes;
  const bool first_head = h == g * per;
  const int tiles = wave < 2 ? 2 : 4;  // of rows up to the wave's
  const int mine = spread_row(wave, r);

  // the wave's rows of K and Q, all loads before the first use
  Eight<T, WIDE> rk8[NK], rq8[NK];
  {
    const int half = 32 * (wave >> 1), have = uniform(max(0, min(32, rows - half)));
    const int64_t gcol = (int64_t)g * a.n;
    const auto bK = rows_of<T>((const T*)a.K + gcol, t0 + half, a.Ks, have);
    const auto bQ = rows_of<T>((const T*)a.Q + gcol, t0 + half, a.Qs, have);
    const uint32_t kr = (uint32_t)(mine - half) * (uint32_t)(a.Ks * sizeof(T)),
                   qr = (uint32_t)(mine - half) * (uint32_t)(a.Qs * sizeof(T));
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const int n = 32 * s + 8 * q;
      rk8[s] = load_eight<T, WIDE>(bK, kr + (uint32_t)(n * sizeof(T)), n, a.n);
    }
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const int n = 32 * s + 8 * q;
      rq8[s] = load_eight<T, WIDE>(bQ, qr + (uint32_t)(n * sizeof(T)), n, a.n);
    }
  }
  // row = lane, the same in every wave
  const int64_t row = t0 + min(lane, rows - 1);
  const float dt = a.A ? (float)((const T*)a.dt)[row * a.dts + h] : 0.0f;
  const float bt = a.beta ? (float)((const T*)a.beta)[row * a.bs + h] : 0.0f;
  const float expo = exponent_of(a, a.A ? a.A[h] : 0.0f, dt, a.dt_bias ? a.dt_bias[h] : 0.0f);
  const float beta = beta_of(a, bt);

  // K and Q as operands, rows scaled
  v8h qf[NK][KP];
  {
    float m = 0.0f, kk = 0.0f;
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = eight_f32<T, WIDE>(rk8[s], i);
        m = max_abs(m, v);
        kk = __builtin_fmaf(v, v, kk);
      }
    kk = quads_add(kk);
    const Scale sc = scale_of_length(quads_max(m), kk);
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = eight_f32<T, WIDE>(rk8[s], i) * sc.up;
      v8h p[KP];
      halves8<KP>(p, v);
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        *(v8h*)(shK + wave * kTile + (s * KP + i) * 1024 + lane * 16) = p[i];
        if (first_head) *(v8h*)(keys + wave * kTile + (s * KP + i) * 1024 + lane * 16) = p[i];
      }
    }
    float mq = 0.0f, qq = 0.0f;
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = eight_f32<T, WIDE>(rq8[s], i);
        mq = max_abs(mq, v);
        qq = __builtin_fmaf(v, v, qq);
      }
    const Scale sq = scale_of(quads_max(mq));
    qq = quads_add(qq);
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = eight_f32<T, WIDE>(rq8[s], i) * sq.up;
      halves8<KP>(qf[s], v);
      if (first_head)
#pragma unroll
        for (int i = 0; i < KP; ++i)
          *(v8h*)(keys + (4 + wave) * kTile + (s * KP + i) * 1024 + lane * 16) = qf[s][i];
    }
    if (q == 0) {
      shKk[mine] = kk;
      shKd[mine] = sc.down;
      shQf[mine] = a.scale * unit_of(a, qq) * sq.down;
    }
  }
  lds_sync();

  // the rows' scalars, in every wave alike
  const float squares = shKk[lane], rq = lane < rows ? shQf[lane] : 0.0f;
  const bool in = lane < rows;
  // b r and b r^2; not finite where b, the key or b |k|^2 is not
  const float rk = unit_of(a, squares) * shKd[lane], write = beta * rk, turn = write * rk;
  const bool bad = in && !(expo <= 0.0f && __builtin_fabsf(turn) < __builtin_inff());
  const uint64_t bads = __ballot(bad);
  const int first = bads ? __ffsll((unsigned long long)bads) - 1 : kC;
  const bool live = in && lane < first;
  double cum = live ? (double)expo * 1.4426950408889634 : 0.0;
  cum = scan_f64(cum < -256.0 ? -256.0 : cum);
  const double whole = __shfl(cum, 63);
  const float hi = (float)cum, grow = __builtin_amdgcn_exp2f(hi);
  shHi[lane] = hi;
  shLo[lane] = (float)(cum - (double)hi);
  float* scalars = (float*)(out + 2 * kTri);
  if (wave == 0) {
    scalars[kGrowK * 64 + lane] = live ? grow * turn : 0.0f;
    scalars[kWrite * 64 + lane] = live ? write : 0.0f;
    scalars[kLeft * 64 + lane] = live ? __builtin_amdgcn_exp2f((float)(whole - cum)) : 0.0f;
    scalars[kGrowQ * 64 + lane] = grow * rq;
    if (lane == 0) {
      const Decay d = decay_of((float)(whole * 0.6931471805599453));
      scalars[kMisc * 64] = d.hi;
      scalars[kMisc * 64 + 1] = d.lo;
      ((int*)scalars)[kMisc * 64 + 2] = first;
    }
  }
  const float bi = __shfl(live ? turn : 0.0f, mine), qi = __shfl(rq, mine);

  // (k_j . k_i) and (k_j . q_i): i a row of the wave's, by lane; j up to it
  v4f kk[4], kq[4];
  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    kk[t] = kq[t] = zero;
    if (t < tiles) {
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        v8h pj[KP], pi[KP];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          pj[i] = *(const v8h*)(shK + t * kTile + (s * KP + i) * 1024 + lane * 16);
          pi[i] = *(const v8h*)(shK + wave * kTile + (s * KP + i) * 1024 + lane * 16);
        }
        kk[t] = mfma_h(pj, pi, kk[t]);
        kq[t] = mfma_h(pj, qf[s], kq[t]);
      }
    }
  }
  if (first_head) {
    // K by columns: 16 columns of a tile and 32 rows each, as products with ones
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      const int t = 2 * x + (wave & 1), sp = wave >> 1;  // columns of step x
      v8h one;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        one[e] = spread_row(t, r) == 32 * x + 8 * q + e ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const uint8_t* at = shK + 2 * sp * kTile + (x * KP + i) * 1024 + lane * 16;
        const v4f c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const v8h*)at, one, zero, 0, 0, 0);
        const v4f c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const v8h*)(at + kTile), one, zero, 0, 0, 0);
        v8h o[1];
        halves8<1>(o, c0, c1);
        *(v8h*)(keys + 8 * kTile + ((t * 2 + sp) * KP + i) * 1024 + lane * 16) = o[0];
      }
    }
  }
  // L into LDS, A out
  const float ihi = shHi[mine], ilo = shLo[mine];
  float m8[2][8], ma = 0.0f;
#pragma unroll
  for (int sp = 0; sp < 2; ++sp) {
    if (2 * sp < tiles) {
      float l[8];
      const int j0 = 32 * sp + 8 * q;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 jh = *(const float4*)(shHi + j0 + 4 * k), jl = *(const float4*)(shLo + j0 + 4 * k);
        const float h4[4] = {jh.x, jh.y, jh.z, jh.w}, l4[4] = {jl.x, jl.y, jl.z, jl.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 4 * k + e;
          const float d = __builtin_amdgcn_exp2f((ihi - h4[e]) + (ilo - l4[e]));
          const float lv = bi * (d * kk[2 * sp + k][e]), mv = qi * (d * kq[2 * sp + k][e]);
          l[4 * k + e] = j < mine && mine < first ? lv : 0.0f;
          m8[sp][4 * k + e] = j <= mine && j < first ? mv : 0.0f;
          ma = max_abs(ma, m8[sp][4 * k + e]);
        }
      }
      *(float4*)(shL + mine * kRowL + j0) = make_float4(l[0], l[1], l[2], l[3]);
      *(float4*)(shL + mine * kRowL + j0 + 4) = make_float4(l[4], l[5], l[6], l[7]);
    }
  }
  auto put_tri = [&](uint8_t* at, float (&v)[2][8], float largest, int k) {
    const Scale sc = scale_of(quads_max(largest));
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
      if (2 * sp < tiles) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[sp][e] *= sc.up;
        v8h p[2];
        halves8<2>(p, v[sp]);
        uint8_t* o = at + tri_block(wave, sp) + lane * 16;
        *(v8h*)o = p[0];
        *(v8h*)(o + 1024) = p[1];
      }
    }
    if (q == 0) scalars[k * 64 + mine] = sc.down;
  };
  put_tri(out + kTri, m8, ma, kFacA);
  lds_sync();
  invert(shL, shT, wave, lane);
  float v8[2][8], mt = 0.0f;
#pragma unroll
  for (int sp = 0; sp < 2; ++sp) {
    if (2 * sp < tiles) {
      const int j0 = 32 * sp + 8 * q;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 x = *(const float4*)(shT + mine * kRowL + j0 + 4 * k);
        const float t4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v8[sp][4 * k + e] = j0 + 4 * k + e <= mine ? t4[e] : 0.0f;
          mt = max_abs(mt, v8[sp][4 * k + e]);
        }
      }
    }
  }
  put_tri(out, v8, mt, kFacT);
}

// ---------------------------------------------------------------------------
// A sequence's chunks in turn, for 16 rows of a head's state (16 columns of v),
// by two waves.  The first carries the state, all of whose columns it holds in
// accumulators, from chunk to chunk; the second, a chunk behind, makes y from
// the state and the w that the first leaves in LDS.  Nothing is exchanged
// between lanes: results serve as operands (spread_row).
//
// The state S and w (the prompts' r w, above) are held times a power of two per
// column, `unit`, so that the largest of S and w is at least kLow and S and w pass
// neither kTopS nor kTop: there two halves are good to 2^-23 of it.  w is looked at
// in every chunk; of S a bound is carried on, and its values looked at when that
// passes kTopS.  What leaves the range, or fp32, goes another way: a unit by the largest of S and b r v,
// and the chunk worked out anew.  (Where these are in range and w and S still below
// kLow, w is what is left of larger terms, and as good as they are.)
//
// Bound by the steps of a chunk, each of which waits for the one before: 2.35 us
// per chunk (600 us for 16384 rows at 32 heads of 128 x 128, on 256 blocks), of
// whose 5600 cycles the first wave spends 1300 on products and about as many on
// other instructions.  An earlier form of 603 us took 546 with all operands in the
// caches and 562 without the second wave.  Two blocks per SIMD pair did not pay: in
// 256 registers the operands of the next chunk no longer fit ahead (713 us), and
// staged in LDS by a third wave they took 643 us.  In fp32 with more than 128 values
// of state the operands do not fit 512 registers either: 488 of them spill, and 1024
// rows take 576 us where 128 values take 84.
// ---------------------------------------------------------------------------
constexpr float kTop = 32768.0f, kTopS = 16384.0f, kLow = 1.0f;
constexpr int kAim = 127 + 4, kTopAim = 127 + 10;  // exponent bits that a new unit gives the largest
// The first unit: the largest of a state and its first chunk's b r v are as a rule
// 2^-5 to 2^9.  To look at them all first takes 10 us more of 338 (64 prompts of 33
// rows at 32 heads of 128 x 128).
constexpr float kFirst = 32.0f;

// The power of two, of up to 2^-126 and 2^100, that takes a magnitude with the
// exponent bits e up to kAim's, where there is room to grow, or down to kTopAim's,
// where smaller values of the column lose least, as far as `unit` times it stays
// in that range.
__device__ __forceinline__ float to_range(int e, float unit) {
  const int ue = exponent_bits(unit), want = max(kAim, min(e, kTopAim));
  const int d = min(max(want - e, max(1 - ue, -126)), min(227 - ue, 100));
  return __uint_as_float((uint32_t)(127 + d) << 23);
}
__device__ __forceinline__ v4f mfma_one(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// c[.] += a[.] (sum of b), one product of halves after another, so that
// neighbours do not wait for each other
template <int M, int NA>
__device__ __forceinline__ void mfma_many(v4f (&c)[M], const v8h (&a)[M][NA], const v8h (&b)[2]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < 2 - i; ++j)
#pragma unroll
      for (int m = 0; m < M; ++m) c[m] = mfma_one(a[m][i], b[j], c[m]);
}

template <int NK>
struct ScanLds {
  static constexpr int kS = NK * 2 * 1024, kW = 2 * 2 * 1024;
  static constexpr int kBuffer = kS + kW + 3 * 64;  // S, w; per column: units of both, first bad row
};

template <typename T, int NK>
__global__ __launch_bounds__(128, 1) void k_delta_scan(
    DeltaArgs a, DeltaPlan pl, int64_t items, int slices, bool by_seq) {
  using L = ScanLds<NK>;
  constexpr int KP = kHalves<T>, NT = 2 * NK;
  __shared__ __attribute__((aligned(16))) uint8_t sh[2][L::kBuffer];
  const int64_t block = wide_block();
  const int64_t part = block / a.heads;
  const int h = uniform((int)(block - part * a.heads));
  const int64_t item = part / slices;
  const int slice = uniform((int)(part - item * slices));
  if (item >= items) return;
  int b, s, e;
  const int slots = first_slots(a.q);
  if (by_seq) {
    b = (int)item;
    s = a.q.seq_start ? seq_row(a.q, b) : 0;
    e = a.q.seq_start ? seq_row(a.q, b + 1) : a.q.n_tokens;
  } else {  // the sequence whose first row on a multiple of 32 this is
    if (32 * item >= a.q.n_tokens) return;
    b = find_row(a.q, (int)(32 * item), &e);
    if (b < 0) return;
    s = a.q.seq_start ? seq_row(a.q, b) : 0;
    if ((s + 31) / 32 != item) return;
  }
  b = uniform(b);
  s = uniform(s);
  e = uniform(e);
  if (e - s <= kShort) return;
  const int slot = uniform(find_slot(a.q, b, slots));
  if (slot == kNoSlot) return;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int g = uniform(h / (a.heads / a.groups));
  const int64_t place0 = pl.by_rows ? s / 32 : (int64_t)(s / kC) + b;
  const int chunks = (e - s + kC - 1) / kC;
  const int p = slice * 16 + r;
  const uint32_t col = p < a.hd ? (uint32_t)(((int64_t)h * a.hd + p) * sizeof(T)) : kNoColumn;
  // what the first launch left of a chunk
  const uint8_t* keys0 = pl.keys + (place0 * a.groups + g) * pl.key_bytes;
  const uint8_t* heads0 = pl.heads + (place0 * a.heads + h) * pl.head_bytes;
  const int64_t key_step = a.groups * pl.key_bytes, head_step = a.heads * pl.head_bytes;
  auto keys_of = [&](int c) { return rows_at(keys0 + c * key_step, (uint32_t)pl.key_bytes); };
  auto head_of = [&](int c) { return rows_at(heads0 + c * head_step, (uint32_t)pl.head_bytes); };
  auto operand = [&](__amdgpu_buffer_rsrc_t at, int off) {  // a kilobyte, 16 bytes per lane
    return __builtin_bit_cast(v8h, __builtin_amdgcn_raw_buffer_load_b128(at, lane * 16, off, 0));
  };
  auto scalars = [&](__amdgpu_buffer_rsrc_t at, int k, v4f (&v)[4]) {  // of the lane's rows of each tile
#pragma unroll
    for (int w = 0; w < 4; ++w)
      v[w] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(
                                         at, q * 32, 2 * kTri + k * 256 + spread_row(w, 0) * 4, 0));
  };
  auto triangle = [&](__amdgpu_buffer_rsrc_t at, int off, v8h (&f)[6][2]) {
#pragma unroll
    for (int k = 0; k < 6; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) f[k][i] = operand(at, off + k * 2048 + i * 1024);
  };
  // block (w, x) of T or A times rows 32 x .. of v, for all four row tiles
  auto times_triangle = [&](const v8h (&f)[6][2], const v8h (&v)[2][2], v4f (&o)[4]) {
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    // one product of halves after another, so that neighbours do not wait
#pragma unroll
    for (int w = 0; w < 4; ++w) o[w] = mfma_one(f[w < 2 ? w : 2 * w - 2][0], v[0][0], zero);
#pragma unroll
    for (int w = 2; w < 4; ++w) o[w] = mfma_one(f[2 * w - 1][0], v[1][0], o[w]);
#pragma unroll
    for (int w = 0; w < 4; ++w) o[w] = mfma_one(f[w < 2 ? w : 2 * w - 2][0], v[0][1], o[w]);
#pragma unroll
    for (int w = 2; w < 4; ++w) o[w] = mfma_one(f[2 * w - 1][0], v[1][1], o[w]);
#pragma unroll
    for (int w = 0; w < 4; ++w) o[w] = mfma_one(f[w < 2 ? w : 2 * w - 2][1], v[0][0], o[w]);
#pragma unroll
    for (int w = 2; w < 4; ++w) o[w] = mfma_one(f[2 * w - 1][1], v[1][0], o[w]);
  };
  // 16 values of v or z in the lane's column
  auto values = [&](const void* at, int64_t stride, int c, uint32_t (&v)[4][4]) {
    const uint32_t step = (uint32_t)(stride * sizeof(T)), at0 = anew(col + 8 * q * step);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = s + c * kC + 32 * half;
      const auto from = rows_of<T>(at, row, stride, at ? uniform(max(0, min(32, e - row))) : 0);
#pragma unroll
      for (int w = 2 * half; w < 2 * half + 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[w][i] = load_raw<T>(from, at0 + (spread_row(w & 1, 0) + i) * step);
    }
  };
  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};

  if (threadIdx.x < 64) {
    // ---- the state ----
    const bool keep = slot >= 0 && !(a.q.fresh && a.q.fresh[b]);
    const auto bst = rows_at(a.state + (slot >= 0 ? (int64_t)slot * a.ss : 0) +
                                 ((int64_t)h * a.hd + slice * 16) * a.n,
                             slot >= 0 ? (uint32_t)(min(16, a.hd - slice * 16) * a.n * 4) : 0);
    auto state_off = [&](uint32_t n0, int t, int i) {
      const int n = (int)n0 + spread_row(t, i);
      return n < a.n ? (uint32_t)((r * a.n + n) * 4) : kNoColumn;
    };
    v4f S[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        S[t][i] = keep ? load_row<float, 1>(bst, state_off(8 * q, t, i)).v[0] : 0.0f;
    // operands of the next chunk are loaded when those of this one are done with
    v8h kf[NK][4][KP], kt[2][NT][KP], tf[6][2];
    uint32_t vr[4][4];
    v4f grow[4], write[4], left[4], fac[4];
    auto fetch_k = [&](__amdgpu_buffer_rsrc_t k) {
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < KP; ++i) kf[x][w][i] = operand(k, ((w * NK + x) * KP + i) * 1024);
    };
    auto fetch_kt = [&](__amdgpu_buffer_rsrc_t k) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < KP; ++i)
            kt[x][t][i] = operand(k, (8 * NK * KP + (t * 2 + x) * KP + i) * 1024);
    };
    float unit = 1.0f, bound = 0.0f, lost = 0.0f;
    auto rescale = [&](float f) {
      unit *= f;
      bound *= f;
#pragma unroll
      for (int t = 0; t < NT; ++t) S[t] *= f;
    };
    auto largest = [&]() {  // of the state's column
      float m = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max_abs(m, S[t][i]);
      return quads_max(m);
    };
    {
      const auto k = keys_of(0);
      const auto o = head_of(0);
      fetch_k(k);
      values(a.v, a.vs, 0, vr);
      scalars(o, kGrowK, grow);
      scalars(o, kWrite, write);
      triangle(o, 0, tf);
      scalars(o, kFacT, fac);
      fetch_kt(k);
      scalars(o, kLeft, left);
    }
    // the unit by the largest finite of the state, ms, and of b r v
    auto aim = [&](bool off, float ms) {
      float mv = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) mv = fmaxf(mv, __builtin_fabsf(raw_f32<T>(vr[w][i]) * write[w][i]));
      if (__ballot(mv == __builtin_inff())) {
        mv = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = __builtin_fabsf(raw_f32<T>(vr[w][i]) * write[w][i]);
            mv = v < __builtin_inff() ? fmaxf(mv, v) : mv;
          }
      }
      mv = quads_max(mv);
      constexpr int kNone = -1000;
      int bits = max(mv > 0.0f ? exponent_bits(mv) + exponent_bits(unit) - 127 : kNone,
                     ms > 0.0f && ms < __builtin_inff() ? exponent_bits(ms) : kNone);
      off = off && bits != kNone;
      for (int k = 0; k < 2; ++k) {  // one power of two may not reach
        const float f = off ? to_range(bits, unit) : 1.0f;
        if (!__ballot(f != 1.0f)) break;
        rescale(f);
        bits += exponent_bits(f) - 127;
      }
    };
    bound = __builtin_inff();
    for (int c = 0; c < chunks; ++c) {
      const int next = c + 1 < chunks ? c + 1 : c;
      const auto head1 = head_of(next), keys1 = keys_of(next);
      const float* misc = (const float*)(heads0 + c * head_step + 2 * kTri) + kMisc * 64;
      const float dec_hi = misc[0], dec_lo = misc[1];
      const int first = ((const int*)misc)[2];
      uint8_t* buf = sh[c & 1];
      if (__ballot(!(bound <= kTopS))) {
        bound = largest();
        float f = bound > kTopS && bound < __builtin_inff() ? to_range(exponent_bits(bound), unit) : 1.0f;
        if (c == 0 && bound <= kTopS / kFirst) f = kFirst;
        rescale(f);
      }
      // K S, and S for the other wave
      v4f X[4];
      auto product = [&](auto keys) {
#pragma unroll
        for (int w = 0; w < 4; ++w) X[w] = zero;
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          v8h sf[2];
          halves8<2>(sf, S[2 * x], S[2 * x + 1]);
          *(v8h*)(buf + x * 2048 + lane * 16) = sf[0];
          *(v8h*)(buf + x * 2048 + 1024 + lane * 16) = sf[1];
          keys(x, sf);
        }
        if (q == 0) ((float*)(buf + L::kS + L::kW))[r] = __builtin_amdgcn_rcpf(unit);
      };
      product([&](int x, const v8h (&sf)[2]) { mfma_many(X, kf[x], sf); });
      __builtin_amdgcn_sched_barrier(0);
      fetch_k(keys1);
      // R = b r v - b r^2 e^c K S, w = T R
      v4f R[4], W[4];
      auto residue = [&]() {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            R[w][i] = __builtin_fmaf(-grow[w][i], X[w][i], raw_f32<T>(vr[w][i]) * write[w][i] * unit);
      };
      auto solve = [&]() {
        v8h rf[2][2];
        halves8<2>(rf[0], R[0], R[1]);
        halves8<2>(rf[1], R[2], R[3]);
        times_triangle(tf, rf, W);
        float m = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          W[w] *= fac[w];
#pragma unroll
          for (int i = 0; i < 4; ++i) m = max_abs(m, W[w][i]);
        }
        return quads_max(m);
      };
      residue();
      float mw = solve();
      int from = first;  // the column's rows from here on are NaN
      // (no w at all may also be values or a state too small for their halves)
      const bool over = !(mw <= kTop), faint = mw < kLow && unit < 0x1p100f && p < a.hd;
      if (__ballot(over || faint)) {
        const float ms = bound = largest(), unit0 = unit;
        const bool off = over || (faint && ms < kLow);
        if (__ballot(off)) aim(off, ms);
        if (__ballot(over || unit != unit0)) {  // all of it anew
          // infinities and NaN leave the products; `at` is the first row of one
          int at = kC;
          auto tame = [&](v4f (&v)[4]) {
            float m = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (!(__builtin_fabsf(v[w][i]) < __builtin_inff())) {
                  at = min(at, spread_row(w, 4 * q + i));
                  v[w][i] = 0.0f;
                }
                m = max_abs(m, v[w][i]);
              }
            return quads_max(m);
          };
          const auto k = keys_of(c);
          product([&](int x, const v8h (&sf)[2]) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              v8h kw[KP];
#pragma unroll
              for (int i = 0; i < KP; ++i) kw[i] = operand(k, ((w * NK + x) * KP + i) * 1024);
              X[w] = mfma_h(kw, sf, X[w]);
            }
          });
          residue();
          float m = tame(R), f = m > kTop ? to_range(exponent_bits(m), unit) : 1.0f;
          rescale(f);
#pragma unroll
          for (int w = 0; w < 4; ++w) R[w] *= f;
          (void)solve();
          mw = tame(W);
          f = mw > kTop ? to_range(exponent_bits(mw), unit) : 1.0f;
          rescale(f);
          mw *= f;
#pragma unroll
          for (int w = 0; w < 4; ++w) W[w] *= f;
          bound = largest();
          at = min(at, __shfl_xor(at, 16));
          from = min(from, min(at, __shfl_xor(at, 32)));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      values(a.v, a.vs, next, vr);
      scalars(head1, kGrowK, grow);
      scalars(head1, kWrite, write);
      triangle(head1, 0, tf);
      scalars(head1, kFacT, fac);
      // w for the other wave, and times e^{c_C - c} for the state
      v8h lf[2][2];
#pragma unroll
      for (int w = 0; w < 4; ++w) *(v4f*)(buf + L::kS + w * 1024 + lane * 16) = W[w];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        halves8<2>(lf[x], W[2 * x] * left[2 * x], W[2 * x + 1] * left[2 * x + 1]);
      if (q == 0) {
        ((float*)(buf + L::kS + L::kW))[16 + r] = __builtin_amdgcn_rcpf(unit);
        ((int*)(buf + L::kS + L::kW))[32 + r] = from;
      }
      // The decay as one float: what its rounding loses goes into the next one,
      // so that the product over all chunks is good to 2^-24.
      const float low = __builtin_fmaf(dec_hi, lost, dec_lo), decay = dec_hi + low;
      lost = decay > 0.0f ? ((dec_hi - decay) + low) * __builtin_amdgcn_rcpf(decay) : 0.0f;
      bound = __builtin_fmaf(bound, decay, 128.0f * mw);  // |K| < 2, 64 rows
      const float by = from < kC ? __builtin_nanf("") : decay;
#pragma unroll
      for (int t = 0; t < NT; ++t) S[t] *= by;
#pragma unroll
      for (int x = 0; x < 2; ++x) mfma_many(S, kt[x], lf[x]);
      __builtin_amdgcn_sched_barrier(0);
      fetch_kt(keys1);
      scalars(head1, kLeft, left);
      lds_sync();
    }
    if (a.frozen) return;
    const float down = __builtin_amdgcn_rcpf(unit);
    const uint32_t n0 = anew(8 * q);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float o[1] = {S[t][i] * down};
        store_row<float, 1>(bst, state_off(n0, t, i), o);
      }
  } else {
    // ---- y ----
    const uint32_t ys = (uint32_t)(a.ys * sizeof(T));
    v8h qf[NK][4][KP], af[6][2];
    uint32_t zr[4][4];
    v4f grow[4], fac[4];
    auto fetch_q = [&](int c) {
      const auto k = keys_of(c);
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < KP; ++i) qf[x][w][i] = operand(k, (((4 + w) * NK + x) * KP + i) * 1024);
    };
    fetch_q(0);
    for (int c = 0; c < chunks; ++c) {
      const int next = c + 1 < chunks ? c + 1 : c;
      const uint8_t* buf = sh[c & 1];
      const auto head = head_of(c);
      triangle(head, kTri, af);
      values(a.z, a.zs, c, zr);
      scalars(head, kGrowQ, grow);
      scalars(head, kFacA, fac);
      lds_sync();
      v4f X[4] = {zero, zero, zero, zero}, Y[4];
#pragma unroll
      for (int x = 0; x < NK; ++x) {
        const v8h sf[2] = {*(const v8h*)(buf + x * 2048 + lane * 16),
                           *(const v8h*)(buf + x * 2048 + 1024 + lane * 16)};
        mfma_many(X, qf[x], sf);
      }
      fetch_q(next);
      v8h wf[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        halves8<2>(wf[x], *(const v4f*)(buf + L::kS + 2 * x * 1024 + lane * 16),
                   *(const v4f*)(buf + L::kS + (2 * x + 1) * 1024 + lane * 16));
      times_triangle(af, wf, Y);
      const float* cols = (const float*)(buf + L::kS + L::kW);
      const float us = cols[r], uw = cols[16 + r];
      const int from = ((const int*)cols)[32 + r];
      float y[4][4];
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[w][i] = __builtin_fmaf(us * grow[w][i], X[w][i], uw * fac[w][i] * Y[w][i]);
      if (a.z) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[w][i] *= sizeof(T) == 4 ? silu_f32(raw_f32<T>(zr[w][i])) : silu_short(raw_f32<T>(zr[w][i]));
      }
      if (__ballot(from < kC)) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[w][i] = spread_row(w, 4 * q + i) < from ? y[w][i] : __builtin_nanf("");
      }
      const uint32_t at0 = anew(col + 8 * q * ys);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = s + c * kC + 32 * half;
        const auto by = rows_of<T>(a.y, row, a.ys, uniform(max(0, min(32, e - row))));
#pragma unroll
        for (int w = 2 * half; w < 2 * half + 2; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float o[1] = {y[w][i]};
            store_row<T, 1>(by, at0 + (spread_row(w & 1, 0) + i) * ys, o);
          }
      }
    }
  }
}

static int delta_nk(int n) { return n <= 64 ? 2 : (n <= 128 ? 4 : 8); }

template <typename T, int NK>
static hipError_t launch_chunks(const DeltaArgs& a, const DeltaPlan& pl, hipStream_t s) {
  const dim3 grid = wide_grid(pl.units, a.heads);
  const hipError_t e = pl.wide ? launch(k_delta_chunk<T, NK, true>, grid, dim3(256), 0, s, a, pl)
                               : launch(k_delta_chunk<T, NK, false>, grid, dim3(256), 0, s, a, pl);
  if (e != hipSuccess) return e;
  // of the sequences, or the rows on multiples of 32, whichever are fewer
  const int64_t marks = a.q.n_tokens / 32 + 1;
  const bool by_seq = a.q.n_seqs <= marks;
  const int64_t items = by_seq ? a.q.n_seqs : marks;
  const int slices = (a.hd + 15) / 16;
  return launch(k_delta_scan<T, NK>, wide_grid(items * slices * a.heads, 1), dim3(128), 0, s, a, pl,
                items, slices, by_seq);
}

template <typename T>
static hipError_t launch_delta(const DeltaArgs& a, const DeltaPlan& pl, bool step, hipStream_t s) {
  if (step) return launch_step_t<T>(a, s);
  if (a.q.seq_start || !pl.chunks) {
    const hipError_t e = a.n <= 64    ? launch_few<T, 4>(a, s)
                         : a.n <= 128 ? launch_few<T, 8>(a, s)
                                      : launch_few<T, 16>(a, s);
    if (e != hipSuccess || !pl.chunks) return e;
  }
  switch (delta_nk(a.n)) {
    case 2: return launch_chunks<T, 2>(a, pl, s);
    case 4: return launch_chunks<T, 4>(a, pl, s);
    default: return launch_chunks<T, 8>(a, pl, s);
  }
}

// The places of sequences of more than kShort rows: from row / kC + b on there
// are enough for any, from row / 32 on for those (n / 32 rounded down is at
// least n / kC rounded up then).  Both counts only grow with rows and sequences.
static DeltaPlan delta_plan(const bm_hip_delta_t* op, void* workspace) {
  DeltaPlan pl{};
  pl.chunks = op->n_tokens > kShort;
  if (!pl.chunks) return pl;
  const size_t elem = type_bytes(op->type);
  pl.wide = op->d_state % 8 == 0 && op->q_stride * elem % 4 == 0 && op->k_stride * elem % 4 == 0 &&
            ((uintptr_t)op->q | (uintptr_t)op->k) % 4 == 0;
  pl.units = unit_count(op->n_seqs, op->n_tokens, kC);
  const int64_t by_rows = op->n_tokens / 32 + 1;
  pl.by_rows = by_rows < pl.units;
  pl.places = pl.by_rows ? by_rows : pl.units;
  pl.head_bytes = 2 * kTri + kScalars;
  pl.key_bytes = (int64_t)12 * delta_nk(op->d_state) * (elem == 4 ? 2 : 1) * 1024;
  const size_t heads = (size_t)(pl.places * op->n_heads * pl.head_bytes);
  pl.heads = (uint8_t*)workspace;
  pl.keys = (uint8_t*)((uintptr_t)workspace + heads);
  pl.bytes = heads + (size_t)(pl.places * op->n_groups * pl.key_bytes);
  return pl;
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
  return bm::delta_plan(op, nullptr).bytes;
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
  const bm::DeltaPlan pl = bm::delta_plan(op, workspace);
  if (!step && pl.bytes && (!workspace || (uintptr_t)workspace % 256)) {
    bm_set_error("%s: a workspace of %zu bytes on 256 bytes is required", name, pl.bytes);
    return -2;
  }
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
    case BM_HIP_F32: e = bm::launch_delta<float>(a, pl, step, s); break;
    case BM_HIP_BF16: e = bm::launch_delta<__bf16>(a, pl, step, s); break;
    default: e = bm::launch_delta<_Float16>(a, pl, step, s); break;
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
