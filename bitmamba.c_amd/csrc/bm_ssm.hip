// The selective scan of the block (src/kernel.c:34-70, src/block.c:127-160)
// for many sequences, d_state values per channel, B and C shared by the heads
// of a group:
//
//   d = softplus(dt + dt_bias), a = exp(A d)
//   S[p][n] = a S[p][n] + d x[p] B[n]
//   y[p] = (sum_n C[n] S[p][n] + D[p] x[p]) z[p] / (1 + exp(-z[p]))
//
// State, sums and decays in fp32; y rounded once.
#include "bm_dev.h"
#include "bm_seq.h"

namespace bm {

struct SsmArgs {
  SeqView q;
  int heads, hd, groups, n;  // hd: head_dim, n: d_state
  bool softplus;
  const void *x, *B, *C, *dt, *z;
  int64_t xs, Bs, Cs, dts, zs;
  const float *A, *dt_bias, *D;
  float* state;
  int64_t ss;
  void* y;
  int64_t ys;
};

__device__ __forceinline__ float bias_of(const SsmArgs& a, int h) {
  return a.dt_bias ? a.dt_bias[h] : 0.0f;
}
__device__ __forceinline__ float step_of(const SsmArgs& a, float dt, float bias) {
  dt += bias;
  return a.softplus ? softplus_f32(dt) : dt;
}

// sum over teams of T neighbouring lanes, in every lane of the team: the
// order of adds is the same in every team
template <int T>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int m = 1; m < T; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// ---------------------------------------------------------------------------
// One token of each sequence.  A team of T lanes holds one channel's state
// row, V neighbouring values per lane and step of E; a wave takes 64 / T rows
// at once and U such groups of rows, all loads issued before the first use.
// Bound by the state's bytes, read and written once; at few sequences by one
// launch and the round trips slot -> state.  64 heads of 64, d_state 128,
// bf16, 128 sequences: 91 us, 540 MB at 5.9 TB/s; one value, fp32, one
// sequence: 2.9 us.
// ---------------------------------------------------------------------------
template <typename T, int TEAM, int V, int E, int U, bool STREAM>
__global__ __launch_bounds__(256) void k_ssm_step(SsmArgs a) {
  constexpr int kRows = 64 / TEAM;
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nw = blockDim.x >> 6;
  const int p0 = (blockIdx.z * nw + wave) * (kRows * U) + lane / TEAM;
  const int nl = (lane % TEAM) * V;
  const int slot = find_slot(a.q, b, first_slots(a.q));
  if (slot == kNoSlot) return;
  const int g = h / (a.heads / a.groups);
  const float d = step_of(a, (float)((const T*)a.dt)[(int64_t)b * a.dts + h], bias_of(a, h));
  const Decay decay = decay_of(a.A[h] * d);
  // the head's part of the slot, of x, z and y; what lies past them reads as
  // zeros and is not written
  const auto st = rows_at(a.state + (slot >= 0 ? (int64_t)slot * a.ss : 0) + (int64_t)h * a.hd * a.n,
                          slot >= 0 ? (uint32_t)(a.hd * a.n * 4) : 0);
  const uint32_t head = (uint32_t)(a.hd * sizeof(T));
  const auto bx = rows_at((const T*)a.x + (int64_t)b * a.xs + (int64_t)h * a.hd, head);
  const auto bz = rows_at((const T*)a.z + (int64_t)b * a.zs + (int64_t)h * a.hd, a.z ? head : 0);
  const auto by = rows_at((const T*)a.y + (int64_t)b * a.ys + (int64_t)h * a.hd, head);
  const auto bD = rows_at(a.D + (int64_t)h * a.hd, a.D ? (uint32_t)(a.hd * 4) : 0);
  const uint32_t gn = (uint32_t)(a.n * sizeof(T));
  const auto bB = rows_at((const T*)a.B + (int64_t)b * a.Bs + (int64_t)g * a.n, gn);
  const auto bC = rows_at((const T*)a.C + (int64_t)b * a.Cs + (int64_t)g * a.n, gn);
  float s[U][E][V], Bv[E][V], Cv[E][V];
  uint32_t x[U], z[U];
  float D[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = p0 + u * kRows;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
      load_floats<V, STREAM>(s[u][e], st, n < a.n ? (uint32_t)((p * a.n + n) * 4) : kNoColumn);
    }
    x[u] = load_raw<T>(bx, (uint32_t)(p * sizeof(T)));
    z[u] = load_raw<T>(bz, (uint32_t)(p * sizeof(T)));
    D[u] = __uint_as_float(load_raw<float>(bD, (uint32_t)(p * 4)));
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t n = (uint32_t)((nl + e * TEAM * V + i) * sizeof(T));
      Bv[e][i] = d * raw_f32<T>(load_raw<T>(bB, n));
      Cv[e][i] = raw_f32<T>(load_raw<T>(bC, n));
      // beyond d_state: zeros, whatever d is
      if (n >= gn) Bv[e][i] = 0.0f;
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = p0 + u * kRows;
    const float xf = raw_f32<T>(x[u]);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[u][e][i] = __builtin_fmaf(s[u][e][i], decay.hi,
                                    with_low(s[u][e][i], decay.lo, xf * Bv[e][i]));
        // beyond d_state nothing counts, even where x or the decay is infinite
        if (E * TEAM * V > 1 && (V == 1 || E > 1)) s[u][e][i] = n + i < a.n ? s[u][e][i] : 0.0f;
        sum = __builtin_fmaf(s[u][e][i], Cv[e][i], sum);
      }
      if (V > 1) sum = n < a.n ? sum : 0.0f;
      store_floats<V, STREAM>(st, n < a.n ? (uint32_t)((p * a.n + n) * 4) : kNoColumn, s[u][e]);
    }
    sum = __builtin_fmaf(D[u], xf, team_sum<TEAM>(sum));
    if (a.z) sum *= silu_f32(raw_f32<T>(z[u]));
    const float out[1] = {sum};
    store_row<T, 1>(by, lane % TEAM == 0 ? (uint32_t)(p * sizeof(T)) : kNoColumn, out);
  }
}

template <typename T, int TEAM, int V, int E>
static hipError_t launch_step(const SsmArgs& a, hipStream_t s) {
  constexpr int U = TEAM >= 16 ? 8 : (TEAM >= 4 ? 4 : 1);
  constexpr int kRows = 64 / TEAM * U;  // channels per wave
  const int waves = (a.hd + kRows - 1) / kRows;
  const int nw = waves < 4 ? waves : 4;
  const dim3 grid(a.q.n_seqs, a.heads, (waves + nw - 1) / nw);
  // States of 64 MiB or more, of which the caches keep nothing until the next
  // token of the layer, go past them (d_state 128, six layers in turn: 37.5
  // against 42.9 us at 100 MB, 16.5 against 13.6 us at 34 MB)
  constexpr bool kLarge = V == 4 && TEAM >= 4;
  if (kLarge && (int64_t)a.q.n_seqs * a.heads * a.hd * a.n >= (1 << 24))
    return launch(k_ssm_step<T, TEAM, V, E, U, kLarge>, grid, dim3(64 * nw), 0, s, a);
  return launch(k_ssm_step<T, TEAM, V, E, U, false>, grid, dim3(64 * nw), 0, s, a);
}

template <typename T>
static hipError_t launch_step_t(const SsmArgs& a, hipStream_t s) {
  if (a.n % 4 == 0) {  // a row's loads of four floats need no more than a float's alignment
    if (a.n <= 4) return launch_step<T, 1, 4, 1>(a, s);
    if (a.n <= 8) return launch_step<T, 2, 4, 1>(a, s);
    if (a.n <= 16) return launch_step<T, 4, 4, 1>(a, s);
    if (a.n <= 32) return launch_step<T, 8, 4, 1>(a, s);
    if (a.n <= 64) return launch_step<T, 16, 4, 1>(a, s);
    if (a.n <= 128) return launch_step<T, 32, 4, 1>(a, s);
    return launch_step<T, 64, 4, 1>(a, s);
  }
  if (a.n <= 1) return launch_step<T, 1, 1, 1>(a, s);
  if (a.n <= 2) return launch_step<T, 2, 1, 1>(a, s);
  if (a.n <= 4) return launch_step<T, 4, 1, 1>(a, s);
  if (a.n <= 8) return launch_step<T, 8, 1, 1>(a, s);
  if (a.n <= 16) return launch_step<T, 16, 1, 1>(a, s);
  if (a.n <= 32) return launch_step<T, 32, 1, 1>(a, s);
  if (a.n <= 64) return launch_step<T, 64, 1, 1>(a, s);
  return launch_step<T, 64, 1, 4>(a, s);
}

// ---------------------------------------------------------------------------
// Prompts.  The rows of a sequence are cut into units of `len` rows, where a
// sequence may have more than one in three launches:
//   the first pass runs every unit but a sequence's last from a zero state,
//   for the state it ends with and its whole decay;
//   the join turns these into the state that each unit starts from,
//     start_0 = the sequence's own, start_{j+1} = start_j decay_j + end_j;
//   the second pass runs all units from there and writes y.
// Otherwise the second pass alone runs.
//
// Workspace: per unit `ends` (laid out as the kernels hold a state) and
// `decays` (one per head).  A sequence's last unit has no end of its own: the
// first pass leaves the sequence's own state in its place.  A decay past fp32
// (A d > 0), which a state may still come through, being zero or small, is
// kept as minus its exponent.
// ---------------------------------------------------------------------------
struct ScanPlan {
  int len;         // rows per unit
  int64_t units;
  bool split;      // a sequence may have more than one unit
  bool by_rows;    // where a sequence's units lie in the workspace (ScanUnit)
  float* ends;
  float* decays;
};

// s times such a decay; t: the third part of its exponent, in powers of two.
// Three factors, none of them infinite, take every state but zero as far as the
// whole one would.
__device__ __forceinline__ float grown(float s, float t) {
  const float f = __builtin_amdgcn_exp2f(t < 127.0f ? t : 127.0f);
  return s * f * f * f;
}

struct ScanUnit {
  Unit u;
  int slot, t0, t1;
  int last;       // the sequence's last unit, counted from u.k's unit 0
  bool keep;      // starts from its slot's state
  // The place of the sequence's unit 0 in the workspace: its unit's index, or
  // 2 row / len.  The second leaves a sequence of two or more units the places
  // up to its end's, which are at least as many, and needs none for the others.
  int64_t place0;
};
// false: nothing to do (no such unit, or padding)
__device__ __forceinline__ bool scan_unit(const SeqView& q, int index, const ScanPlan& pl,
                                          ScanUnit& w) {
  const int len = pl.len, slots = first_slots(q);
  w.u = find_unit(q, index, len);
  if (w.u.b < 0) return false;
  w.t0 = w.u.s + w.u.k * len;
  w.last = w.u.e > w.u.s ? (w.u.e - w.u.s - 1) / len : 0;
  if (w.u.k > w.last) return false;
  w.t1 = w.u.e - w.t0 < len ? w.u.e : w.t0 + len;
  w.place0 = pl.by_rows ? 2 * (int64_t)(w.u.s / len) : (int64_t)index - w.u.k;
  w.slot = find_slot(q, w.u.b, slots);
  w.keep = w.slot >= 0 && !(q.fresh && q.fresh[w.u.b]);
  return w.slot != kNoSlot;
}

// ---- up to 8 state values per channel -------------------------------------
// A lane owns a channel with its state in registers and walks the unit's
// rows; a block is one wave.  What the channels of a head share per row --
// decay, d B[n], C[n] -- is worked out once per row and head into LDS.  2-4
// operations per state value and row against 12 bytes per channel and row:
// bound by memory, and in one short prompt by the round trips to it, so that
// the loads of a tile of kSmallRows rows are all issued before any is used,
// and the next tile's while one is worked on.  At 64 heads of 64 channels and
// one value, fp32, 1024 rows: 8 and 16 us for the two passes, 51 MB at 2.2
// TB/s; 6001 rows of 32 heads 55 us, 2.7 TB/s (tiles of 8 and 32 rows: 73 and
// 69 us; two or four channels per lane: 72 and 103).
constexpr int kSmallState = 8;
constexpr int kSmallRows = 16;
// of a row and head in LDS: decay, d B, C (in the first pass the exponent A d),
// and last the decay's low part
__host__ __device__ constexpr int small_entry(int ns) { return (2 + 2 * ns + 3) / 4 * 4; }

template <typename T, int NS, bool FULL>
__global__ __launch_bounds__(64) void k_scan_small(SsmArgs a, ScanPlan pl, int heads_max) {
  constexpr int tile = kSmallRows, EW = small_entry(NS);
  extern __shared__ float4 sh4[];
  float* sh = (float*)sh4;  // [tile][heads_max][EW]
  ScanUnit w;
  if (!scan_unit(a.q, blockIdx.x, pl, w)) return;
  if (!FULL && w.u.k == w.last) return;
  const int lane = threadIdx.x, channels = a.heads * a.hd;
  const int c0 = blockIdx.y * 64;
  const int c = c0 + lane;
  const bool on = c < channels;
  const int h0 = c0 / a.hd;
  const int h1 = (min(c0 + 64, channels) - 1) / a.hd;
  const int nh = h1 - h0 + 1;
  const int h = on ? c / a.hd : h0;
  const int per = a.heads / a.groups;
  const int64_t unit0 = w.place0, unit = unit0 + w.u.k;
  const int64_t unit_floats = (int64_t)channels * a.n;

  const uint32_t col = on ? (uint32_t)(c * sizeof(T)) : kNoColumn;
  const uint32_t xs = (uint32_t)(a.xs * sizeof(T)), zs = (uint32_t)(a.zs * sizeof(T)),
                 ys = (uint32_t)(a.ys * sizeof(T));
  uint32_t xr[tile], zr[tile];
  auto fetch = [&](int t) {
    const int rows = min(tile, w.t1 - t);
    const auto bx = rows_of<T>(a.x, t, a.xs, rows);
    const auto bz = rows_of<T>(a.z, t, a.zs, FULL && a.z ? rows : 0);
#pragma unroll
    for (int r = 0; r < tile; ++r) {
      xr[r] = load_raw<T>(bx, col + r * xs);
      if (FULL) zr[r] = load_raw<T>(bz, col + r * zs);
    }
  };
  if (w.t0 < w.t1) fetch(w.t0);

  float S[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) S[n] = 0.0f;
  // from the slot, or from the copy that the first pass made of it
  if (on && w.keep && (FULL ? w.last == 0 : w.u.k == 0)) {
    const float* st = a.state + (int64_t)w.slot * a.ss + (int64_t)c * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) S[n] = st[n];
  }
  if constexpr (!FULL) {
    if (w.u.k == 0) {
      float* e = pl.ends + (unit0 + w.last) * unit_floats + c;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        if (on && n < a.n) e[(int64_t)n * channels] = S[n];
        S[n] = 0.0f;
      }
    }
  } else if (w.last > 0 && on) {
    // the join, a few floats of each unit before this one: cheaper here than
    // a launch of its own (3 us against 4.7 and its gap)
    constexpr int kAhead = NS == 1 ? 16 : 4;
    const float* e = pl.ends + unit0 * unit_floats + c;
    const float* dec = pl.decays + unit0 * a.heads + h;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) S[n] = e[w.last * unit_floats + (int64_t)n * channels];
    for (int j0 = 0; j0 < w.u.k; j0 += kAhead) {
      float v[kAhead][NS], d[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int j = min(j0 + i, w.u.k - 1);
        d[i] = dec[(int64_t)j * a.heads];
#pragma unroll
        for (int n = 0; n < NS; ++n)
          v[i][n] = e[j * unit_floats + (int64_t)min(n, a.n - 1) * channels];
      }
      float least = 0.0f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) least = fminf(least, d[i]);
      if (__ballot(least < 0.0f)) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (j0 + i >= w.u.k) break;
#pragma unroll
          for (int n = 0; n < NS; ++n)
            S[n] = n < a.n ? (d[i] < 0.0f ? grown(S[n], d[i] * (kLog2e / -3.0f)) : S[n] * d[i]) +
                                 v[i][n]
                           : 0.0f;
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (j0 + i >= w.u.k) break;
#pragma unroll
        for (int n = 0; n < NS; ++n)
          S[n] = n < a.n ? __builtin_fmaf(S[n], d[i], v[i][n]) : 0.0f;
      }
    }
  }

  const float D = FULL && on && a.D ? a.D[c] : 0.0f;
  double total = 0.0;  // of the unit's exponents: its decay is rounded once
  for (int t = w.t0; t < w.t1; t += tile) {
    const int rows = min(tile, w.t1 - t);
    for (int i = lane; i < tile * nh; i += 64) {
      const int r = i / nh, hh = i - r * nh;
      float* s = sh + (r * heads_max + hh) * EW;
      if (r >= rows) {  // past the unit: leaves the state as it is
        s[0] = 1.0f;
#pragma unroll
        for (int n = 1; n < EW; ++n) s[n] = 0.0f;
        continue;
      }
      const int64_t row = t + r;
      const int g = (h0 + hh) / per;
      const float d = step_of(a, (float)((const T*)a.dt)[row * a.dts + h0 + hh],
                              bias_of(a, h0 + hh));
      const float Ad = a.A[h0 + hh] * d;
      const Decay decay = decay_of(Ad);
      s[0] = decay.hi;
      s[EW - 1] = decay.lo;
      if (!FULL) s[1 + NS] = Ad;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const bool have = n < a.n;
        s[1 + n] = have ? d * (float)((const T*)a.B)[row * a.Bs + (int64_t)g * a.n + n] : 0.0f;
        if (FULL)
          s[1 + NS + n] = have ? (float)((const T*)a.C)[row * a.Cs + (int64_t)g * a.n + n] : 0.0f;
      }
    }
    __syncthreads();
    float x[tile], z[tile];
#pragma unroll
    for (int r = 0; r < tile; ++r) {
      x[r] = raw_f32<T>(xr[r]);
      z[r] = FULL && a.z ? silu_f32(raw_f32<T>(zr[r])) : 1.0f;
    }
    if (t + tile < w.t1) fetch(t + tile);
    const auto by = rows_of<T>(a.y, t, a.ys, rows);
    float exponents = 0.0f, low = 0.0f;  // the tile's sums
#pragma unroll
    for (int r = 0; r < tile; ++r) {
      float e[EW];
      const float4* s = (const float4*)(sh + (r * heads_max + (h - h0)) * EW);
#pragma unroll
      for (int k = 0; k < EW / 4; ++k) *(float4*)(e + 4 * k) = s[k];
      float y = FULL ? D * x[r] : 0.0f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        S[n] = __builtin_fmaf(S[n], e[0], x[r] * e[1 + n]);
        // a value beyond d_state stays zero even where the decay is infinite
        if (NS > 2) S[n] = n < a.n ? S[n] : 0.0f;
        if (FULL) y = __builtin_fmaf(S[n], e[1 + NS + n], y);
      }
      low += e[EW - 1];
      if (!FULL) exponents += e[1 + NS];
      if (FULL) {
        const float out[1] = {y * z[r]};
        store_row<T, 1>(by, col + r * ys, out);
      }
    }
    // The tile's decays were the nearest floats.  What that left of them: for
    // the state from before the tile all of it, for what its rows added up to
    // 16 halves of 2^-24 too much (a second product per row instead took 57.5
    // against 56.0 us at 4 values, fp16, 6000 rows of 32 heads of 64; 52.3 now).
#pragma unroll
    for (int n = 0; n < NS; ++n) S[n] = with_low(S[n], low, S[n]);
    if (!FULL) total += (double)exponents;
    __syncthreads();
  }
  if (!on) return;
  if constexpr (!FULL) {
    float* e = pl.ends + unit * unit_floats + c;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) e[(int64_t)n * channels] = S[n];
    if (c % a.hd == 0) {
      const Decay all = decay_of((float)total);
      const float f = all.hi + all.lo;
      pl.decays[unit * a.heads + h] = f == __builtin_inff() ? (float)-total : f;
    }
  } else if (w.slot >= 0 && w.u.k == w.last) {
    float* st = a.state + (int64_t)w.slot * a.ss + (int64_t)c * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) st[n] = S[n];
  }
}

template <typename T, int NS>
static hipError_t launch_small(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  const int channels = a.heads * a.hd;
  const int by = (channels + 63) / 64;
  const int hm = (64 + a.hd - 2) / a.hd + 1;
  const int heads_max = hm < a.heads ? hm : a.heads;
  const int bytes = kSmallRows * heads_max * small_entry(NS) * 4;  // at most 80 KB
  if (bytes > 64 * 1024) {  // heads of one channel; once per process
    static const hipError_t raised[2] = {
        hipFuncSetAttribute((const void*)k_scan_small<T, NS, false>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024),
        hipFuncSetAttribute((const void*)k_scan_small<T, NS, true>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)};
    if (raised[0] != hipSuccess) return raised[0];
    if (raised[1] != hipSuccess) return raised[1];
  }
  const dim3 grid((unsigned)pl.units, by);
  if (pl.split) {
    const hipError_t e =
        launch(k_scan_small<T, NS, false>, grid, dim3(64), bytes, s, a, pl, heads_max);
    if (e != hipSuccess) return e;
  }
  return launch(k_scan_small<T, NS, true>, grid, dim3(64), bytes, s, a, pl, heads_max);
}

template <typename T>
static hipError_t launch_small_n(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  if (a.n == 1) return launch_small<T, 1>(a, pl, s);
  if (a.n == 2) return launch_small<T, 2>(a, pl, s);
  if (a.n <= 4) return launch_small<T, 4>(a, pl, s);
  return launch_small<T, 8>(a, pl, s);
}

// The join: a thread takes four neighbouring floats of a sequence's units in
// turn, kAhead of them loaded before the first is used.  A head's floats are
// head_floats.  Bound by reading and writing the states once: 4 TB/s at 31 MB.
__global__ __launch_bounds__(256) void k_scan_join(SeqView q, ScanPlan pl, int64_t unit_floats,
                                                   int blocks, int head_floats, int heads) {
  constexpr int kAhead = 8, V = 4;
  ScanUnit w;
  const int64_t block = wide_block();
  if (block >= pl.units * blocks) return;
  if (!scan_unit(q, (int)(block / blocks), pl, w) || w.u.k != 0 || w.last == 0) return;
  const int64_t at = (block % blocks * 256 + threadIdx.x) * V;
  if (at >= unit_floats) return;
  float* e = pl.ends + w.place0 * unit_floats + at;
  const float* dec = pl.decays + w.place0 * heads + at / head_floats;
  float S[V];
  load_f32<float, V>(S, e + w.last * unit_floats);
  for (int j0 = 0; j0 < w.last; j0 += kAhead) {
    float v[kAhead][V], d[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = min(j0 + i, w.last - 1);
      load_f32<float, V>(v[i], e + j * unit_floats);
      d[i] = dec[(int64_t)j * heads];
    }
    float least = 0.0f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) least = fminf(least, d[i]);
    if (__ballot(least < 0.0f)) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (j0 + i >= w.last) break;
        store_f32<float, V>(e + (j0 + i) * unit_floats, S);
#pragma unroll
        for (int k = 0; k < V; ++k)
          S[k] = (d[i] < 0.0f ? grown(S[k], d[i] * (-1.0f / 3.0f)) : S[k] * d[i]) + v[i][k];
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (j0 + i >= w.last) break;
      store_f32<float, V>(e + (j0 + i) * unit_floats, S);
#pragma unroll
      for (int k = 0; k < V; ++k) S[k] = __builtin_fmaf(S[k], d[i], v[i][k]);
    }
  }
  store_f32<float, V>(e + w.last * unit_floats, S);
}

// ---- more state values: chunks of kQ rows on the matrix cores --------------
//
// With c_i the sum of A d over the chunk's rows up to i,
//   y_i = sum_{j<=i} (C_i . B_j) e^{c_i - c_j} d_j x_j + e^{c_i} C_i . S
//   S'  = e^{c_Q} S + sum_j B_j (e^{c_Q - c_j} d_j x_j)
// A block takes one unit and up to four tiles of 32 channels of one group; a
// wave keeps its tile's state S [d_state][32] in accumulators over the whole
// unit.  B and C go through LDS once per chunk for all tiles.  Four waves and
// two blocks per CU beat one block of eight, whose waves all wait for the same
// barriers (second pass at d_state 128, bf16: 319 against 335 us then).
//
// What bounds it: per 32 rows and channels at d_state 128, bf16, 1004 vector
// instructions (splitting S, the decays, gates; 47 of them MFMAs).  With two
// waves per SIMD (220 registers) the vector pipe is busy 55 % of the time, the
// matrix pipe 19 %; leaving out all memory accesses took 228 us to 177.  Tried without
// gain: x and z a chunk ahead, a third wave per SIMD (spills), dot products in
// place of subtractions in the split, uniform row offsets, one exponential per
// row in place of one per pair.  64 heads of 64, d_state 128, one group, bf16,
// 16384 rows: 105 + 18 + 236 us for the passes and the join, 417 MB (82 us);
// 32 heads, d_state 64, fp32, 3001 rows: 23 + 10 + 40 us, 84 MB (16 us).
//
// Precision.  MFMA operands are bf16.  An fp32 value is carried as the sum of
// three bf16 pieces (8 bits each, the remainder of the piece before), fp16 as
// two, bf16 as one, all exact; of the products of two such sums those above
// 2^-24 of the whole are kept (piece indices that add up to less than 3), and
// everything is accumulated in fp32.  For a bf16 y the computed operands S and
// M have two pieces (off by 2^-18) and the gate a short exponential (silu_short),
// against y's rounding of 2^-9; the state itself always gets three pieces.
//
// Layouts (lane l, half h = l / 32; accumulator r of a 32x32 tile is row
// 8 (r / 4) + 4 h + r % 4, column l % 32).  The k order of a product is free
// as long as both operands use the same one, so the accumulators serve as
// operands as they are: k step s of 16 takes accumulators 8s .. 8s+7, that is
// rows 16 s + 4 h + {0..3} and 16 s + 8 + 4 h + {0..3}.  B, C and B^T are
// stored in LDS in that order, and x is loaded in it.
//
// Decays: c_i in fp64 over the chunk, kept as two floats, so that e^{c_i-c_j}
// is good to fp32 however large c is.  A row's exponent is held at -256
// powers of two, where its decay is long zero, so that the sums stay exact.
//
// Growth (A d > 0): a decay over several rows can be infinite where the state or
// x that it multiplies is zero or small, and multiplies what the products lose
// of pieces below 2^-126.  A chunk ends before its positive exponents sum up to
// kGrowth, for all the block's waves, since they share B and C.  Where that can
// happen each chunk waits for what the other waves say, 1 to 2 % of its time.
//
// Causality holds for infinities and NaN too: a product takes 0 for M above
// the diagonal, and 0 times such an x would reach earlier rows, so x enters
// that product as 0 and the rows from it on become NaN.  An fp32 x whose first
// piece is infinite (kInfinite and more) is treated the same.
constexpr int kQ = 32, kWaves = 4;
constexpr double kGrowth = 16.0;  // powers of two
constexpr float kInfinite = 0x1.ffp127f;  // rounds to an infinite bf16
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// bf16 pieces of two values, as the halves of a word each
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ void split2(uint32_t (&p)[N], float x, float y) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const v2f v = {x, y};
    p[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2bf));
    if (k + 1 < N) {
      x -= __uint_as_float(p[k] << 16);
      y -= __uint_as_float(p[k] & 0xffff0000u);
    }
  }
}
// of eight values, as MFMA operands
template <int N>
__device__ __forceinline__ void split8(v8bf (&p)[N], const float* v) {
  u32x4 w[N];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t q[N];
    split2<N>(q, v[2 * e], v[2 * e + 1]);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k][e] = q[k];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) p[k] = __builtin_bit_cast(v8bf, w[k]);
}

// c += (sum of a) (sum of b), pieces whose indices add up to less than ORD
template <int ORD, int NA, int NB>
__device__ __forceinline__ v16f mfma32(const v8bf (&a)[NA], const v8bf (&b)[NB], v16f c) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < ORD) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], c, 0, 0, 0);
  return c;
}

template <typename T>
struct Pieces;  // IN: of an input; Y: of what only y depends on
template <>
struct Pieces<float> {
  static constexpr int IN = 3, Y = 3;
};
template <>
struct Pieces<_Float16> {
  static constexpr int IN = 2, Y = 3;
};
template <>
struct Pieces<__bf16> {
  static constexpr int IN = 1, Y = 2;
};
constexpr int kStatePieces = 3;

// LDS of a block, in bytes
template <typename T, int NT>
struct MmLds {
  static constexpr int NP = 32 * NT;
  static constexpr int kRowB = (NP + 8) * 2;  // a row of B or C, padded by 16 bytes
  static constexpr int kRowT = (kQ + 8) * 2;  // a row of B^T
  static constexpr int kPieceB = kQ * kRowB, kPieceT = NP * kRowT;
  static constexpr int kRowCb = kQ + 4;  // floats
  static constexpr int kCb = kQ * kRowCb * 4;
  static constexpr int kScal = 5 * kQ * 4;  // per wave: c (two parts), d, e^c, e^{c_Q - c} d
  static constexpr int kApart = Pieces<T>::IN * (2 * kPieceB + kPieceT) + kCb + kWaves * kScal;
  // B by rows and B^T share a place where two blocks do not fit a CU
  // otherwise: the first is done with when C B^T is
  static constexpr bool kShared = kApart > 80 * 1024;
  static constexpr int kC = Pieces<T>::IN * (kShared && kPieceT > kPieceB ? kPieceT : kPieceB);
  static constexpr int kT = kShared ? 0 : kC + Pieces<T>::IN * kPieceB;
  static constexpr int kAfter = kC + Pieces<T>::IN * (kPieceB + (kShared ? 0 : kPieceT));
  static constexpr int kBytes = kAfter + kCb + kWaves * kScal;
};

// running sums over each half of the wave
__device__ __forceinline__ double half_scan(double v) {
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
  return v;
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane),
                 hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// keeps the compiler from working the offsets of 16 rows out ahead of the
// loop and holding them in registers
__device__ __forceinline__ uint32_t here(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// a state tile in `ends`
template <int NT>
__device__ __forceinline__ void put_tile(float* e, const v16f (&S)[NT]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(float4*)(e + (nt * 4 + q) * 256) =
          make_float4(S[nt][4 * q], S[nt][4 * q + 1], S[nt][4 * q + 2], S[nt][4 * q + 3]);
}
template <int NT>
__device__ __forceinline__ void get_tile(v16f (&S)[NT], const float* e) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 v = *(const float4*)(e + (nt * 4 + q) * 256);
      S[nt][4 * q] = v.x;
      S[nt][4 * q + 1] = v.y;
      S[nt][4 * q + 2] = v.z;
      S[nt][4 * q + 3] = v.w;
    }
}

template <typename T, int NT, bool FULL>
__global__ __launch_bounds__(64 * kWaves, NT < 8 ? 2 : 1) void k_scan_mm(SsmArgs a, ScanPlan pl, int tiles, int wide) {
  using L = MmLds<T, NT>;
  constexpr int IN = Pieces<T>::IN, YP = Pieces<T>::Y;
  constexpr bool kExact = YP == 3;  // y to better than bf16
  constexpr int kThreads = 64 * kWaves;
  constexpr int kBlocks = 64 * NT;  // 4x4 blocks of B (or C) in a chunk
  constexpr int kItems = ((FULL ? 2 : 1) * kBlocks + kThreads - 1) / kThreads;
  extern __shared__ float4 sh4[];
  uint8_t* shB = (uint8_t*)sh4;
  uint8_t* shC = shB + L::kC;
  uint8_t* shT = shB + L::kT;
  float* shCb = (float*)(shB + L::kAfter);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float* scal = (float*)((uint8_t*)shCb + L::kCb) + wave * (L::kScal / 4);
  float *shHi = scal, *shLo = scal + kQ, *shD = scal + 2 * kQ, *shE = scal + 3 * kQ,
        *shW = scal + 4 * kQ;

  ScanUnit w;
  if (!scan_unit(a.q, blockIdx.x, pl, w)) return;
  if (!FULL && w.u.k == w.last) return;
  const int g = blockIdx.y, per = a.heads / a.groups;
  const int ptiles = (a.hd + 31) / 32;
  const int item = blockIdx.z * kWaves + wave;  // tile of the group
  const bool active = item < tiles;
  const int h = g * per + (active ? item / ptiles : 0);
  const int pt = active ? item % ptiles : 0;
  const int p = pt * 32 + li;
  const bool on = active && p < a.hd;
  const int64_t c = (int64_t)h * a.hd + p;
  const int64_t unit0 = w.place0, unit = unit0 + w.u.k;
  constexpr int kTile = NT * 16 * 64;  // floats of a state tile in `ends`: [nt][r / 4][lane][4]
  const int64_t tile_at = ((int64_t)h * ptiles + pt) * kTile + 4 * lane;
  const int64_t unit_floats = (int64_t)a.heads * ptiles * kTile;

  v16f S[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[nt][r] = 0.0f;
  // the tile's part of the slot
  const auto bst = rows_at(a.state + (w.slot >= 0 ? (int64_t)w.slot * a.ss : 0) + (c - li) * a.n,
                           w.slot >= 0 && active ? (uint32_t)(min(32, a.hd - pt * 32) * a.n * 4) : 0);
  auto state_off = [&](int nt, int r) {
    const int n = nt * 32 + acc_row(r, half);
    return n < a.n ? (uint32_t)((li * a.n + n) * 4) : kNoColumn;
  };
  if (w.keep && (FULL ? w.last == 0 : w.u.k == 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[nt][r] = load_row<float, 1>(bst, state_off(nt, r)).v[0];
  }
  if constexpr (!FULL) {
    if (w.u.k == 0) {
      if (active) {
        float* e = pl.ends + (unit0 + w.last) * unit_floats + tile_at;
        put_tile(e, S);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 16; ++r) S[nt][r] = 0.0f;
      }
    }
  } else if (w.last > 0 && active) {
    get_tile(S, pl.ends + unit * unit_floats + tile_at);
  }

  const float A = a.A[h], bias = bias_of(a, h);
  const float Dp = FULL && on && a.D ? a.D[c] : 0.0f;
  double total = 0.0;  // of the unit's exponents, in powers of two

  const uint32_t xs = (uint32_t)(a.xs * sizeof(T)), zs = (uint32_t)(a.zs * sizeof(T)),
                 ys = (uint32_t)(a.ys * sizeof(T));
  const uint32_t col = (uint32_t)(c * sizeof(T));
  const uint32_t xoff = on ? col + 4 * half * xs : kNoColumn,
                 zoff = on ? col + 4 * half * zs : kNoColumn,
                 yoff = on ? col + 4 * half * ys : kNoColumn;
  // the next chunk's B, C and dt, and in the first pass x, are loaded while a
  // chunk is worked on; x and z of the second pass are not needed before B
  // and C have been through LDS
  uint32_t nx[16], ndt = 0;
  Raw4<T> nb[kItems][4];
  auto fetch_bc = [&](int t, int rows, auto load4) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int first = wave * 64 + k * kThreads;  // kBlocks: whole waves
      if (first >= (FULL ? 2 : 1) * kBlocks) break;
      const bool isC = first >= kBlocks;
      const int blk = tid + k * kThreads - (isC ? kBlocks : 0);
      const int n = blk % (8 * NT) * 4, j = blk / (8 * NT) * 4;
      const auto src = rows_of<T>(isC ? a.C : a.B, t, isC ? a.Cs : a.Bs, rows);
      const uint32_t stride = (uint32_t)((isC ? a.Cs : a.Bs) * sizeof(T));
      const uint32_t off = here(j * stride + (uint32_t)((g * a.n + n) * sizeof(T)));
#pragma unroll
      for (int q = 0; q < 4; ++q) nb[k][q] = load4(src, off + q * stride, n);
    }
  };
  auto fetch_x = [&](int t, int rows) {
    const auto bx = rows_of<T>(a.x, t, a.xs, rows);
    const uint32_t xo = here(xoff);
#pragma unroll
    for (int r = 0; r < 16; ++r) nx[r] = load_raw<T>(bx, xo + acc_row(r, 0) * xs);
  };
  auto fetch = [&](int t, int rows) {
    const auto bdt = rows_of<T>(a.dt, t, a.dts, rows);
    ndt = load_raw<T>(bdt, li * (uint32_t)(a.dts * sizeof(T)) + h * (uint32_t)sizeof(T));
    if (wide)
      fetch_bc(t, rows, [&](__amdgpu_buffer_rsrc_t r, uint32_t off, int n) {
        return load_raw4<T>(r, n < a.n ? off : kNoColumn);
      });
    if (!FULL) fetch_x(t, rows);
  };
  // value by value, where four do not lie on one load's alignment: not ahead
  auto fetch_narrow = [&](int t, int rows) {
    fetch_bc(t, rows, [&](__amdgpu_buffer_rsrc_t r, uint32_t off, int n) {
      Raw4<T> o;
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = load_raw<T>(r, n + i < a.n ? off + i * (uint32_t)sizeof(T) : kNoColumn);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i)
        o.w[i] = sizeof(T) == 2 ? v[2 * i & 3] | v[(2 * i + 1) & 3] << 16 : v[i];
      return o;
    });
  };
  // four values of four rows (or columns) of B or C as pieces in LDS: `at`
  // is the first one's place, rows `row` bytes and pieces `piece` bytes apart
  auto put = [&](uint8_t* at, int row, int piece, const Raw4<T> (&b)[4], bool turn) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = turn ? raw4_f32(b[i], q) : raw4_f32(b[q], i);
      uint32_t lo[IN], hi[IN];
      split2<IN>(lo, v[0], v[1]);
      split2<IN>(hi, v[2], v[3]);
#pragma unroll
      for (int pc = 0; pc < IN; ++pc) {
        const u32x2 o = {lo[pc], hi[pc]};
        *(u32x2*)(at + pc * piece + q * row) = o;
      }
    }
  };
  // four values' place in their 16: quarters 0, 2 | 1, 3
  auto place = [](int i) { return (i & ~15) + ((i >> 2) & 1) * 8 + ((i >> 3) & 1) * 4; };
  auto put_turned = [&](int id, const Raw4<T> (&b)[4]) {
    const int n = id % (8 * NT) * 4, j = id / (8 * NT) * 4;
    put(shT + n * L::kRowT + place(j) * 2, L::kRowT, L::kPieceT, b, true);
  };

  // A chunk's exponents, by lane li (both halves alike), and what is made of
  // them, in the wave's own part of LDS; out of dt fetched before.  Done ahead
  // of the chunk, in the shadow of the products before it.
  float eall = 1.0f;
  double whole = 0.0;
  auto exponents = [&](int rows) {
    const float d = li < rows ? step_of(a, raw_f32<T>(ndt), bias) : 0.0f;
    double cum = (double)A * (double)d * 1.4426950408889634;
    cum = cum < -256.0 ? -256.0 : (cum > 256.0 ? 256.0 : cum);
    const bool grows = __ballot(cum > 0.0) != 0;
    cum = half_scan(cum);
    whole = lane_f64(cum, kQ - 1);
    eall = __builtin_amdgcn_exp2f((float)whole);
    if (half == 0) {
      const float hi = (float)cum;
      shHi[li] = hi;
      shLo[li] = (float)(cum - (double)hi);
      shD[li] = d;
      shE[li] = __builtin_amdgcn_exp2f(hi);
      shW[li] = __builtin_amdgcn_exp2f((float)(whole - cum)) * d;
    }
    return grows;
  };
  // in the columns of C B^T that pad its rows, for each wave: whether any
  // exponent of its chunk is positive, the rows that can go together then, and
  // whether any can be positive: A > 0, or steps of either sign
  int *shGrows = (int*)shCb + kQ, *shRows = shGrows + 1, *shMay = shGrows + 2;
  const int pad = (lane & (kWaves - 1)) * L::kRowCb;
  auto ahead = [&](int rows) {
    const bool grows = exponents(rows);
    if (lane == 0) shGrows[wave * L::kRowCb] = grows;
  };

  if (w.t0 < w.t1) {
    fetch(w.t0, min(kQ, w.t1 - w.t0));
    ahead(min(kQ, w.t1 - w.t0));
  }
  if (lane == 0) shMay[wave * L::kRowCb] = !a.softplus || A > 0.0f;
  __syncthreads();
  const uint32_t may_grow = __ballot(shMay[pad]) != 0;
  int rows = 0;
  for (int t = w.t0; t < w.t1; t += rows) {
    rows = min(kQ, w.t1 - t);
    // the same in all waves; here(): one loop, not one for each of two values
    if (__builtin_amdgcn_readfirstlane(here(may_grow)) && __ballot(shGrows[pad])) {
      const float d = li < rows ? step_of(a, raw_f32<T>(ndt), bias) : 0.0f;
      const double up = half_scan((double)fminf(fmaxf(A * d * kLog2e, 0.0f), 256.0f));
      if (lane == 0) shRows[wave * L::kRowCb] = __popc((uint32_t)__ballot(up < kGrowth));
      __syncthreads();
      const int most = shRows[pad];
#pragma unroll
      for (int k = 0; k < kWaves; ++k) rows = min(rows, __builtin_amdgcn_readlane(most, k));
      rows = max(rows, 1);
      fetch(t, rows);
      (void)exponents(rows);
    }
    total += whole;
    // B and C into LDS
    if (!wide) fetch_narrow(t, rows);
    constexpr int kHeld = L::kShared && FULL ? kItems : 1;
    Raw4<T> held[kHeld][4];  // B, where its transpose has to wait
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int first = wave * 64 + k * kThreads;
      if (first >= (FULL ? 2 : 1) * kBlocks) break;
      const bool isC = first >= kBlocks;
      const int blk = tid + k * kThreads - (isC ? kBlocks : 0);
      const int n = blk % (8 * NT) * 4, j = blk / (8 * NT) * 4;
      if (FULL)
        put((isC ? shC : shB) + j * L::kRowB + place(n) * 2, L::kRowB, L::kPieceB, nb[k], false);
      if (L::kShared && FULL) {
#pragma unroll
        for (int q = 0; q < 4; ++q) held[k][q] = nb[k][q];
      } else if (!isC) {
        put_turned(blk, nb[k]);
      }
    }
    float x[16];
    if (!FULL)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = raw_f32<T>(nx[r]);
    uint32_t z[16];
    if (FULL) {
      fetch_x(t, rows);
      const auto bz = rows_of<T>(a.z, t, a.zs, a.z ? rows : 0);
      const uint32_t zo = here(zoff);
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = load_raw<T>(bz, zo + acc_row(r, 0) * zs);
    }
    const int next = t + rows, after = min(kQ, w.t1 - next);
    if (after > 0) fetch(next, after);
    __syncthreads();

    if constexpr (FULL) {
      // C B^T of the chunk: three 16x16 tiles on and below the diagonal
      if (wave < 3) {
        const int jt = wave == 2 ? 16 : 0, it = wave == 0 ? 0 : 16;
        const int lr = lane & 15, lg = lane >> 4;
        v4f cb = {0.0f, 0.0f, 0.0f, 0.0f};
        // operands of kAhead steps of 32 are read before the first is used
        constexpr int kAhead = IN == 1 ? (NT < 4 ? NT : 4) : 1;
#pragma unroll
        for (int k0 = 0; k0 < NT; k0 += kAhead) {
          v8bf pb[kAhead][IN], pc[kAhead][IN];
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int i = 0; i < IN; ++i) {
              const int at = (32 * (k0 + k) + 8 * lg) * 2;
              pb[k][i] = *(const v8bf*)(shB + i * L::kPieceB + (jt + lr) * L::kRowB + at);
              pc[k][i] = *(const v8bf*)(shC + i * L::kPieceB + (it + lr) * L::kRowB + at);
            }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int i = 0; i < IN; ++i)
#pragma unroll
              for (int j = 0; j < IN; ++j)
                if (i + j < YP)
                  cb = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pb[k][i], pc[k][j], cb, 0, 0, 0);
        }
        *(v4f*)(shCb + (it + lr) * L::kRowCb + jt + 4 * lg) = cb;
      }
      // C S, scaled by e^{c_i}
      v16f Y;
#pragma unroll
      for (int r = 0; r < 16; ++r) Y[r] = 0.0f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = S[nt][8 * s + e];
          v8bf ps[YP], pc[IN];
          split8<YP>(ps, v);
#pragma unroll
          for (int i = 0; i < IN; ++i)
            pc[i] = *(const v8bf*)(shC + i * L::kPieceB + li * L::kRowB + (32 * nt + 16 * s + 8 * half) * 2);
          Y = mfma32<YP>(pc, ps, Y);
        }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 e = *(const float4*)(shE + 8 * q + 4 * half);
        Y[4 * q] *= e.x;
        Y[4 * q + 1] *= e.y;
        Y[4 * q + 2] *= e.z;
        Y[4 * q + 3] *= e.w;
      }
      __syncthreads();  // C B^T is whole
      __builtin_amdgcn_sched_barrier(0);  // nothing that waits for x moves up
      if (L::kShared) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (tid + k * kThreads < kBlocks) put_turned(tid + k * kThreads, held[k]);
      }
      // M x within the chunk; a column with an infinite x or NaN is NaN from
      // that row on, and so is its state
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = raw_f32<T>(nx[r]);
      int first = kQ;
      // Not finite once any x is not, or is fp32 past bf16's range: at 4 x no
      // finite sum before it keeps such a one from overflowing.
      float probe = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) probe = __builtin_fmaf(x[r], IN == 3 ? 4.0f : 0.0f, probe);
      const bool odd = __ballot(!(__builtin_fabsf(probe) < __builtin_inff())) != 0;
      if (odd) {
        asm volatile("");  // a branch, not selects
#pragma unroll
        for (int r = 15; r >= 0; --r)
          if (!(__builtin_fabsf(x[r]) < kInfinite)) {
            first = acc_row(r, half);
            x[r] = 0.0f;
          }
        first = min(first, __shfl_xor(first, 32));
        if (first < kQ) eall = __builtin_nanf("");
      }
      const float hi = shHi[li], lo = shLo[li];
      const int diag = (int)here((uint32_t)(li - 4 * half));
      float m[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j0 = 8 * q + 4 * half;
        const float4 cb = *(const float4*)(shCb + li * L::kRowCb + j0);
        const float4 jh = *(const float4*)(shHi + j0), jl = *(const float4*)(shLo + j0),
                     jd = *(const float4*)(shD + j0);
        const float cbv[4] = {cb.x, cb.y, cb.z, cb.w}, h4[4] = {jh.x, jh.y, jh.z, jh.w},
                    l4[4] = {jl.x, jl.y, jl.z, jl.w}, d4[4] = {jd.x, jd.y, jd.z, jd.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f((hi - h4[i]) + (lo - l4[i]));
          float v = cbv[i] * (e * d4[i]);
          asm volatile("" : "+v"(v));  // a select, not a branch around the exponential
          m[4 * q + i] = 8 * q + i <= diag ? v : 0.0f;
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v8bf pm[YP], px[IN];
        split8<YP>(pm, m + 8 * s);
        split8<IN>(px, x + 8 * s);
        Y = mfma32<YP>(pm, px, Y);
      }
      const auto by = rows_of<T>(a.y, t, a.ys, rows);
      const uint32_t yo = here(yoff);
#pragma unroll
      for (int r = 0; r < 16; ++r) Y[r] = __builtin_fmaf(Dp, x[r], Y[r]);
      if (odd) {
        asm volatile("");
#pragma unroll
        for (int r = 0; r < 16; ++r) Y[r] = acc_row(r, half) < first ? Y[r] : __builtin_nanf("");
      }
      if (a.z)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          Y[r] *= kExact ? silu_f32(raw_f32<T>(z[r])) : silu_short(raw_f32<T>(z[r]));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float out[1] = {Y[r]};
        store_row<T, 1>(by, yo + acc_row(r, 0) * ys, out);
      }
      if (L::kShared) __syncthreads();  // B^T is whole
    }
    // the state
    {
      v8bf xw[2][kStatePieces];
      float v[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 e = *(const float4*)(shW + 8 * q + 4 * half);
        v[4 * q] = x[4 * q] * e.x;
        v[4 * q + 1] = x[4 * q + 1] * e.y;
        v[4 * q + 2] = x[4 * q + 2] * e.z;
        v[4 * q + 3] = x[4 * q + 3] * e.w;
      }
      split8<kStatePieces>(xw[0], v);
      split8<kStatePieces>(xw[1], v + 8);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) S[nt][r] *= eall;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          v8bf pb[IN];
#pragma unroll
          for (int i = 0; i < IN; ++i)
            pb[i] = *(const v8bf*)(shT + i * L::kPieceT + (32 * nt + li) * L::kRowT + (16 * s + 8 * half) * 2);
          S[nt] = mfma32<kStatePieces>(pb, xw[s], S[nt]);
        }
      }
      if (after > 0) ahead(after);
    }
    __syncthreads();  // the next chunk may overwrite LDS
  }

  if constexpr (!FULL) {
    if (!active) return;
    float* e = pl.ends + unit * unit_floats + tile_at;
    put_tile(e, S);
    const float sum = (float)total;
    if (pt == 0 && lane == 0)
      pl.decays[unit * a.heads + h] = sum >= 128.0f ? -sum : __builtin_amdgcn_exp2f(sum);
  } else if (w.slot >= 0 && w.u.k == w.last) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float out[1] = {S[nt][r]};
        store_row<float, 1>(bst, state_off(nt, r), out);
      }
  }
}

static int mm_ptiles(int hd) { return (hd + 31) / 32; }
static int mm_nt(int n) { return n <= 32 ? 1 : (n <= 64 ? 2 : (n <= 128 ? 4 : 8)); }
template <typename T, int NT>
static hipError_t launch_mm(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  const int tiles = a.heads / a.groups * mm_ptiles(a.hd);
  constexpr int bytes = MmLds<T, NT>::kBytes;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  const int wide = a.n % 4 == 0 && a.Bs % 4 == 0 && a.Cs % 4 == 0 &&
                   ((uintptr_t)a.B | (uintptr_t)a.C) % (4 * sizeof(T)) == 0;
  const dim3 grid((unsigned)pl.units, a.groups, (tiles + kWaves - 1) / kWaves);
  if (bytes > 64 * 1024) {  // once per process: a kernel's limit above the default
    static const hipError_t raised[2] = {
        hipFuncSetAttribute((const void*)k_scan_mm<T, NT, false>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
        hipFuncSetAttribute((const void*)k_scan_mm<T, NT, true>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes)};
    if (raised[0] != hipSuccess) return raised[0];
    if (raised[1] != hipSuccess) return raised[1];
  }
  if (pl.split) {
    hipError_t e =
        launch(k_scan_mm<T, NT, false>, grid, dim3(64 * kWaves), bytes, s, a, pl, tiles, wide);
    if (e != hipSuccess) return e;
    const int head = mm_ptiles(a.hd) * NT * 1024;
    const int64_t floats = (int64_t)a.heads * head;
    const int blocks = (int)((floats / 4 + 255) / 256);
    e = launch(k_scan_join, wide_grid(pl.units * blocks, 1), dim3(256), 0, s, a.q, pl, floats,
               blocks, head, a.heads);
    if (e != hipSuccess) return e;
  }
  return launch(k_scan_mm<T, NT, true>, grid, dim3(64 * kWaves), bytes, s, a, pl, tiles, wide);
}

template <typename T>
static hipError_t launch_mm_t(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  switch (mm_nt(a.n)) {
    case 1: return launch_mm<T, 1>(a, pl, s);
    case 2: return launch_mm<T, 2>(a, pl, s);
    case 4: return launch_mm<T, 4>(a, pl, s);
    default: return launch_mm<T, 8>(a, pl, s);
  }
}

// ---- the cut into units ----------------------------------------------------
// Units as short as it takes to fill the chip, no shorter than what a unit's
// prologue and the first pass are worth (32 rows; 128 on the matrix cores), at
// most 64 (32) of them in the longest sequence, and, where there are several
// sequences of which one may have almost all rows, no longer than 512 rows.
// The matrix kernel's fill stays a little below the 2048 waves that its second
// pass's registers let the chip hold, since one workgroup that finds no place
// then doubles the whole time: 219 against 330 us with 15 and 16 units of
// 16384 rows.
constexpr int kFillWaves = 1920, kSmallFillWaves = 2048;

static ScanPlan scan_plan(const bm_hip_ssm_t* op, size_t* bytes) {
  ScanPlan pl{};
  const int64_t channels = (int64_t)op->n_heads * op->head_dim;
  const bool small = op->d_state <= kSmallState;
  const int64_t waves = small ? (channels + 63) / 64
                              : (int64_t)op->n_heads * mm_ptiles(op->head_dim);
  const int step = small ? 32 : kQ, least = small ? 32 : 4 * kQ, most_units = small ? 64 : 32;
  const int64_t T = op->n_tokens;
  const int64_t fill = small ? kSmallFillWaves : kFillWaves;
  const int64_t want = fill / waves > 1 ? fill / waves : 1;
  int64_t len = ((T + want - 1) / want + step - 1) / step * step;
  const int64_t floor_len = ((T + most_units - 1) / most_units + step - 1) / step * step;
  if (len > 512 && op->n_seqs > 1) len = 512;  // uneven lengths: the longest is cut too
  if (len < floor_len) len = floor_len;
  if (len < least) len = least;
  pl.len = (int)len;
  pl.split = T > len;
  pl.units = unit_count(op->n_seqs, op->n_tokens, pl.len);
  const int64_t floats =
      small ? channels * op->d_state
            : (int64_t)op->n_heads * mm_ptiles(op->head_dim) * mm_nt(op->d_state) * 1024;
  // no more places than sequences of two units can take
  const int64_t by_rows = 2 * (T / pl.len) + 2;
  pl.by_rows = by_rows < pl.units;
  auto size_of = [&](int64_t places, size_t* ends) {
    *ends = align_up((size_t)places * floats * 4, 256);
    return *ends + (size_t)places * op->n_heads * 4;
  };
  size_t ends;
  (void)size_of(pl.by_rows ? by_rows : pl.units, &ends);
  pl.decays = (float*)ends;  // its offset, until the workspace is known
  // The size asked for is enough for any call of no more rows and sequences,
  // of which shorter ones can take more places: len does not grow evenly.
  // From its lines above T / len is at most `parts`, which, like the rule for
  // whether a sequence can be cut, never falls as T or n_seqs grows.
  const bool several = op->n_seqs > 1;
  int64_t parts = several && T / 512 > want ? T / 512 : want;
  if (parts > most_units) parts = most_units;
  if (parts > T / least) parts = T / least;
  const bool cut = T > least && (want > 1 || (several && T > 512));
  const int64_t places = parts + op->n_seqs < 2 * parts + 2 ? parts + op->n_seqs : 2 * parts + 2;
  size_t unused;
  *bytes = cut ? size_of(places, &unused) : 0;
  return pl;
}

template <typename T>
static hipError_t launch_scan_t(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  if (a.n > kSmallState) return launch_mm_t<T>(a, pl, s);
  return launch_small_n<T>(a, pl, s);
}

static bool shape_fits(const char* name, const bm_hip_ssm_t* op) {
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

extern "C" size_t bm_hip_ssm_workspace_bytes(const bm_hip_ssm_t* op) {
  if (!bm::shape_fits("ssm_workspace", op) || op->n_tokens < 0 || op->n_seqs < 0) return 0;
  size_t bytes = 0;
  (void)bm::scan_plan(op, &bytes);
  return bytes;
}

static int ssm_call(const bm_hip_ssm_t* op, void* workspace, void* stream, bool step) {
  const char* name = step ? "ssm_step" : "ssm";
  if (!bm::shape_fits(name, op)) return -2;
  const int64_t hp = (int64_t)op->n_heads * op->head_dim, gn = (int64_t)op->n_groups * op->d_state;
  const size_t elem = bm::type_bytes(op->type);
  const int64_t rows = step ? op->n_seqs : op->n_tokens;
  if (!bm::check_seqs(name, op->n_seqs, op->n_tokens, op->seq_start, op->slots, op->state,
                      op->state_stride, op->n_slots, hp * op->d_state, step))
    return -2;
  const struct {
    const char* name;
    const void* p;
    int64_t stride, width;
  } in[] = {{"x", op->x, op->x_stride, hp},
            {"B", op->B, op->B_stride, gn},
            {"C", op->C, op->C_stride, gn},
            {"dt", op->dt, op->dt_stride, op->n_heads},
            {"z", op->z, op->z_stride, hp}};
  if (!bm::check_rows(name, "y", op->y, op->y_stride, hp, rows, elem)) return -2;
  for (const auto& t : in) {
    if (!op->z && &t == &in[4]) continue;  // no gate
    if (!bm::check_rows(name, t.name, t.p, t.stride, t.width, rows, elem) ||
        !bm::check_apart(name, t.name, t.p, t.stride, t.width, op->y, op->y_stride, hp, rows, elem,
                         step && (&t == &in[0] || (&t == &in[4] && op->z == op->x))))
      return -2;
  }
  if (!op->A || ((uintptr_t)op->A | (uintptr_t)op->dt_bias | (uintptr_t)op->D) % 4) {
    bm_set_error("%s: A, dt_bias and D need addresses on 4 bytes, A is required", name);
    return -2;
  }
  bm::ScanPlan pl{};
  if (!step) {
    size_t bytes = 0;
    pl = bm::scan_plan(op, &bytes);
    if (pl.split && (!workspace || (uintptr_t)workspace % 256)) {
      bm_set_error("%s: a workspace of %zu bytes on 256 bytes is required", name, bytes);
      return -2;
    }
    pl.ends = (float*)workspace;
    pl.decays = (float*)((uintptr_t)workspace + (uintptr_t)pl.decays);
  }
  if (op->n_seqs == 0) return 0;
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  bm::SsmArgs a;
  a.q = bm::SeqView{op->seq_start, op->state ? op->slots : nullptr, op->fresh, op->n_seqs,
                    op->n_tokens, op->state ? op->n_slots : 0};
  a.heads = op->n_heads;
  a.hd = op->head_dim;
  a.groups = op->n_groups;
  a.n = op->d_state;
  a.softplus = op->dt_softplus != 0;
  a.x = op->x;
  a.B = op->B;
  a.C = op->C;
  a.dt = op->dt;
  a.z = op->z;
  a.xs = op->x_stride;
  a.Bs = op->B_stride;
  a.Cs = op->C_stride;
  a.dts = op->dt_stride;
  a.zs = op->z_stride;
  a.A = op->A;
  a.dt_bias = op->dt_bias;
  a.D = op->D;
  a.state = op->state;
  a.ss = op->state_stride;
  a.y = op->y;
  a.ys = op->y_stride;
  hipStream_t s = bm::stream_of(stream);
  hipError_t e;
  switch (op->type) {
    case BM_HIP_F32:
      e = step ? bm::launch_step_t<float>(a, s) : bm::launch_scan_t<float>(a, pl, s);
      break;
    case BM_HIP_BF16:
      e = step ? bm::launch_step_t<__bf16>(a, s) : bm::launch_scan_t<__bf16>(a, pl, s);
      break;
    default:
      e = step ? bm::launch_step_t<_Float16>(a, s) : bm::launch_scan_t<_Float16>(a, pl, s);
      break;
  }
  BM_HIP_CHECK_RET(e, -1);
  return 0;
}

extern "C" int bm_hip_ssm_dev(const bm_hip_ssm_t* op, void* workspace, void* stream) {
  return ssm_call(op, workspace, stream, false);
}

extern "C" int bm_hip_ssm_step_dev(const bm_hip_ssm_t* op, void* stream) {
  return ssm_call(op, nullptr, stream, true);
}
