// The selective scan of the block (src/kernel.c:34-70, src/block.c:127-160)
// for many sequences, d_state values per channel, B and C shared by the heads
// of a group:
//
//   d = softplus(dt + dt_bias), a = exp(A d)
//   S[p][n] = a S[p][n] + d x[p] B[n]
//   y[p] = (sum_n C[n] S[p][n] + D[p] x[p]) z[p] / (1 + exp(-z[p]))
//
// State, sums and decays in fp32; y rounded once.
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

__device__ __forceinline__ float step_of(const SsmArgs& a, float dt, int h) {
  if (a.dt_bias) dt += a.dt_bias[h];
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
// launch and the round trips slot -> state.
// ---------------------------------------------------------------------------
template <typename T, int TEAM, int V, int E, int U>
__global__ __launch_bounds__(256) void k_ssm_step(SsmArgs a) {
  constexpr int kRows = 64 / TEAM;
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nw = blockDim.x >> 6;
  const int p0 = (blockIdx.z * nw + wave) * (kRows * U) + lane / TEAM;
  const int nl = (lane % TEAM) * V;
  const int slot = find_slot(a.q, b);
  if (slot == kNoSlot) return;
  const int g = h / (a.heads / a.groups);
  const float d = step_of(a, (float)((const T*)a.dt)[(int64_t)b * a.dts + h], h);
  const float decay = exp_f32(a.A[h] * d);
  float* st = slot >= 0 ? a.state + (int64_t)slot * a.ss + (int64_t)h * a.hd * a.n : nullptr;
  const T* Bp = (const T*)a.B + (int64_t)b * a.Bs + (int64_t)g * a.n;
  const T* Cp = (const T*)a.C + (int64_t)b * a.Cs + (int64_t)g * a.n;
  const T* xp = (const T*)a.x + (int64_t)b * a.xs + (int64_t)h * a.hd;
  float s[U][E][V], x[U], Bv[E][V], Cv[E][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = p0 + u * kRows;
    x[u] = p < a.hd ? (float)xp[p] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int n = nl + e * TEAM * V;
#pragma unroll
      for (int i = 0; i < V; ++i) s[u][e][i] = 0.0f;
      if (st && p < a.hd && n < a.n) load_f32<float, V>(s[u][e], st + (int64_t)p * a.n + n);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = nl + e * TEAM * V + i;
      Bv[e][i] = n < a.n ? d * (float)Bp[n] : 0.0f;
      Cv[e][i] = n < a.n ? (float)Cp[n] : 0.0f;
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = p0 + u * kRows;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[u][e][i] = __builtin_fmaf(s[u][e][i], decay, x[u] * Bv[e][i]);
        sum = __builtin_fmaf(s[u][e][i], Cv[e][i], sum);
      }
    sum = team_sum<TEAM>(sum);
    if (p < a.hd) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int n = nl + e * TEAM * V;
        if (st && n < a.n) store_f32<float, V>(st + (int64_t)p * a.n + n, s[u][e]);
      }
      if (lane % TEAM == 0) {
        const int64_t c = (int64_t)h * a.hd + p;
        if (a.D) sum = __builtin_fmaf(a.D[c], x[u], sum);
        if (a.z) sum *= silu_f32((float)((const T*)a.z)[(int64_t)b * a.zs + c]);
        ((T*)a.y)[(int64_t)b * a.ys + c] = (T)sum;
      }
    }
  }
}

template <typename T, int TEAM, int V, int E>
static hipError_t launch_step(const SsmArgs& a, hipStream_t s) {
  constexpr int U = TEAM >= 4 ? 4 : 1;
  constexpr int kRows = 64 / TEAM * U;  // channels per wave
  const int waves = (a.hd + kRows - 1) / kRows;
  const int nw = waves < 4 ? waves : 4;
  hipLaunchKernelGGL((k_ssm_step<T, TEAM, V, E, U>),
                     dim3(a.q.n_seqs, a.heads, (waves + nw - 1) / nw), dim3(64 * nw), 0, s, a);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_step_t(const SsmArgs& a, hipStream_t s) {
  if (a.n % 4 == 0 && a.ss % 4 == 0 && (uintptr_t)a.state % 16 == 0) {
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
// Prompts.  The rows of a sequence are cut into units of `len` rows.  Every
// unit but a sequence's last is first run from a zero state for the state it
// ends with and its whole decay (pass FULL = false); the second pass runs all
// units, each from the state that its predecessors' results give,
//   S = S decay_j + end_j over the units j before it,
// and writes y.  Where no sequence can have two units there is one pass.
//
// Workspace: per unit, `ends` (the state's layout is the kernel's) and
// `decays` (one per head).  A sequence's last unit has no end of its own
// there: its place holds a copy of the state that the sequence starts from,
// since the slot is rewritten while other units still need it.
// ---------------------------------------------------------------------------
struct ScanPlan {
  int len;         // rows per unit
  int64_t units;
  bool split;      // a sequence may have more than one unit
  float* ends;
  float* decays;
};

struct ScanUnit {
  Unit u;
  int slot, t0, t1;
  int last;       // the sequence's last unit, counted from u.k's unit 0
  bool keep;      // starts from its slot's state
};
// false: nothing to do (no such unit, or padding)
__device__ __forceinline__ bool scan_unit(const SeqView& q, int index, int len, ScanUnit& w) {
  w.u = find_unit(q, index, len);
  if (w.u.b < 0) return false;
  w.t0 = w.u.s + w.u.k * len;
  w.last = w.u.e > w.u.s ? (w.u.e - w.u.s - 1) / len : 0;
  if (w.u.k > w.last) return false;
  w.t1 = w.u.e - w.t0 < len ? w.u.e : w.t0 + len;
  w.slot = find_slot(q, w.u.b);
  w.keep = w.slot >= 0 && !(q.fresh && q.fresh[w.u.b]);
  return w.slot != kNoSlot;
}

// ---- up to 8 state values per channel -------------------------------------
// A lane owns VC neighbouring channels with their state in registers and
// walks the unit's rows; a block is one wave.  What the channels of a head
// share per row -- decay, d B[n], C[n] -- is worked out once per row and head
// into LDS.  2-4 operations per state value and row against 12 bytes per
// channel and row: bound by memory.
constexpr int kSmallState = 8;
__host__ __device__ constexpr int small_entry(int ns) { return (1 + 2 * ns + 3) / 4 * 4; }
constexpr int kSmallRows = 16;  // rows of x and z in flight per lane

template <typename T, int NS, int VC, bool FULL>
__global__ __launch_bounds__(64) void k_scan_small(SsmArgs a, ScanPlan pl, int tile, int heads_max) {
  constexpr int EW = small_entry(NS);
  extern __shared__ float4 sh4[];
  float* sh = (float*)sh4;  // [tile][heads_max][EW]
  ScanUnit w;
  if (!scan_unit(a.q, blockIdx.x, pl.len, w)) return;
  if (!FULL && w.u.k == w.last) return;
  const int lane = threadIdx.x, channels = a.heads * a.hd;
  const int c0 = blockIdx.y * 64 * VC;
  const int c = c0 + lane * VC;
  const bool on = c < channels;  // VC divides head_dim where it is more than 1
  const int h0 = c0 / a.hd;
  const int h1 = (min(c0 + 64 * VC, channels) - 1) / a.hd;
  const int nh = h1 - h0 + 1;
  const int h = on ? c / a.hd : h0;
  const int per = a.heads / a.groups;
  const int64_t unit0 = (int64_t)blockIdx.x - w.u.k;

  float S[NS][VC];
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int i = 0; i < VC; ++i) S[n][i] = 0.0f;
  // from the slot, or from the copy that the first pass made of it
  if (on && w.keep && (FULL ? w.last == 0 : w.u.k == 0)) {
    const float* st = a.state + (int64_t)w.slot * a.ss + (int64_t)c * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < VC; ++i)
        if (n < a.n) S[n][i] = st[i * a.n + n];
  }
  if constexpr (!FULL) {
    if (w.u.k == 0) {
      if (on) {
        float* e = pl.ends + (unit0 + w.last) * channels * a.n;
#pragma unroll
        for (int n = 0; n < NS; ++n)
          if (n < a.n) store_f32<float, VC>(e + (int64_t)n * channels + c, S[n]);
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < VC; ++i) S[n][i] = 0.0f;
    }
  } else if (w.last > 0 && on) {
    const float* e = pl.ends + (unit0 + w.last) * channels * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) load_f32<float, VC>(S[n], e + (int64_t)n * channels + c);
    for (int j = 0; j < w.u.k; ++j) {
      e = pl.ends + (unit0 + j) * channels * a.n;
      const float dec = pl.decays[(unit0 + j) * a.heads + h];
#pragma unroll
      for (int n = 0; n < NS; ++n)
        if (n < a.n) {
          float v[VC];
          load_f32<float, VC>(v, e + (int64_t)n * channels + c);
#pragma unroll
          for (int i = 0; i < VC; ++i) S[n][i] = __builtin_fmaf(S[n][i], dec, v[i]);
        }
    }
  }

  float D[VC], all = 1.0f;
#pragma unroll
  for (int i = 0; i < VC; ++i) D[i] = FULL && on && a.D ? a.D[c + i] : 0.0f;
  const T* xp = (const T*)a.x + c;
  const T* zp = (const T*)a.z + c;
  T* yp = (T*)a.y + c;
  for (int t = w.t0; t < w.t1; t += tile) {
    const int rows = min(tile, w.t1 - t);
    for (int i = lane; i < rows * nh; i += 64) {
      const int r = i / nh, hh = i - r * nh;
      const int64_t row = t + r;
      const int g = (h0 + hh) / per;
      const float d = step_of(a, (float)((const T*)a.dt)[row * a.dts + h0 + hh], h0 + hh);
      float* s = sh + (r * heads_max + hh) * EW;
      s[0] = exp_f32(a.A[h0 + hh] * d);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const bool have = n < a.n;
        s[1 + n] = have ? d * (float)((const T*)a.B)[row * a.Bs + (int64_t)g * a.n + n] : 0.0f;
        if (FULL)
          s[1 + NS + n] = have ? (float)((const T*)a.C)[row * a.Cs + (int64_t)g * a.n + n] : 0.0f;
      }
    }
    __syncthreads();
    for (int r0 = 0; r0 < rows; r0 += kSmallRows) {
      float x[kSmallRows][VC], z[kSmallRows][VC];
#pragma unroll
      for (int r = 0; r < kSmallRows; ++r)
        if (on && r0 + r < rows) {
          load_f32<T, VC>(x[r], xp + (int64_t)(t + r0 + r) * a.xs);
          if (FULL && a.z) load_f32<T, VC>(z[r], zp + (int64_t)(t + r0 + r) * a.zs);
        }
#pragma unroll
      for (int r = 0; r < kSmallRows; ++r) {
        if (r0 + r >= rows) break;
        float e[EW];
        const float4* s = (const float4*)(sh + ((r0 + r) * heads_max + (h - h0)) * EW);
#pragma unroll
        for (int k = 0; k < EW / 4; ++k) *(float4*)(e + 4 * k) = s[k];
        float y[VC];
#pragma unroll
        for (int i = 0; i < VC; ++i) y[i] = FULL ? D[i] * x[r][i] : 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < VC; ++i) {
            S[n][i] = __builtin_fmaf(S[n][i], e[0], x[r][i] * e[1 + n]);
            // a value beyond d_state stays zero even where the decay is infinite
            if (NS > 2) S[n][i] = n < a.n ? S[n][i] : 0.0f;
            if (FULL) y[i] = __builtin_fmaf(S[n][i], e[1 + NS + n], y[i]);
          }
        all *= e[0];
        if (FULL) {
          if (a.z)
#pragma unroll
            for (int i = 0; i < VC; ++i) y[i] *= silu_f32(z[r][i]);
          if (on) store_f32<T, VC>(yp + (int64_t)(t + r0 + r) * a.ys, y);
        }
      }
    }
    __syncthreads();
  }
  if (!on) return;
  if constexpr (!FULL) {
    float* e = pl.ends + (int64_t)blockIdx.x * channels * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (n < a.n) store_f32<float, VC>(e + (int64_t)n * channels + c, S[n]);
    if (c % a.hd == 0) pl.decays[(int64_t)blockIdx.x * a.heads + h] = all;
  } else if (w.slot >= 0 && w.u.k == w.last) {
    float* st = a.state + (int64_t)w.slot * a.ss + (int64_t)c * a.n;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < VC; ++i)
        if (n < a.n) st[i * a.n + n] = S[n][i];
  }
}

template <typename T, int NS, int VC>
static hipError_t launch_small(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  const int span = 64 * VC, channels = a.heads * a.hd;
  const int by = (channels + span - 1) / span;
  const int hm = (span + a.hd - 2) / a.hd + 1;
  const int heads_max = hm < a.heads ? hm : a.heads;
  // rows per tile: 32, or what fits 32 KB (a row is at most 64 heads of 80 bytes)
  const int row = heads_max * small_entry(NS) * 4;
  int tile = 32;
  while (tile * row > 32768) tile /= 2;
  if (pl.split)
    hipLaunchKernelGGL((k_scan_small<T, NS, VC, false>), dim3((unsigned)pl.units, by), dim3(64),
                       tile * row, s, a, pl, tile, heads_max);
  hipLaunchKernelGGL((k_scan_small<T, NS, VC, true>), dim3((unsigned)pl.units, by), dim3(64),
                     tile * row, s, a, pl, tile, heads_max);
  return hipGetLastError();
}

template <typename T, int VC>
static hipError_t launch_small_n(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  if (a.n == 1) return launch_small<T, 1, VC>(a, pl, s);
  if (a.n == 2) return launch_small<T, 2, VC>(a, pl, s);
  if (a.n <= 4) return launch_small<T, 4, VC>(a, pl, s);
  return launch_small<T, 8, VC>(a, pl, s);
}

// ---- more state values: chunks of kQ rows on the matrix cores --------------
//
// With c_i the sum of A d over the chunk's rows up to i,
//   y_i = sum_{j<=i} (C_i . B_j) e^{c_i - c_j} d_j x_j + e^{c_i} C_i . S
//   S'  = e^{c_Q} S + sum_j B_j (e^{c_Q - c_j} d_j x_j)
// A block takes one unit and up to NW tiles of 32 channels of one group; a
// wave keeps its tile's state S [d_state][32] in accumulators over the whole
// unit.  B and C go through LDS once per chunk for all tiles.
//
// Precision.  MFMA operands are bf16.  An fp32 value is carried as the sum of
// three bf16 pieces (8 bits each, the remainder of the piece before), fp16 as
// two, bf16 as one, all exact; of the products of two such sums those above
// 2^-24 of the whole are kept (piece indices that add up to less than 3), and
// everything is accumulated in fp32.  For a bf16 y the computed operands S and
// M have two pieces (off by 2^-18, against y's rounding of 2^-9); the state
// itself always gets three.
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
// Causality holds for infinities and NaN too: a product takes 0 for M above
// the diagonal, and 0 times such an x would reach earlier rows, so x enters
// that product as 0 and the rows from it on become NaN.
constexpr int kQ = 32;
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// bf16 pieces of the elements [8 s, 8 s + 8) of v
template <int N>
__device__ __forceinline__ void split8(v8bf (&p)[N], const float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = v[e];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      p[k][e] = (__bf16)x;
      if (k + 1 < N) x -= (float)p[k][e];
    }
  }
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

// LDS of a block, in bytes.  B by rows and B^T share a place: the first is
// done with when C B^T is.
template <typename T, int NT>
struct MmLds {
  static constexpr int NP = 32 * NT;
  static constexpr int kRowB = (NP + 8) * 2;  // a row of B or C, padded by 16 bytes
  static constexpr int kRowT = (kQ + 8) * 2;  // a row of B^T
  static constexpr int kPieceB = kQ * kRowB, kPieceT = NP * kRowT;
  static constexpr int kB = Pieces<T>::IN * (kPieceB > kPieceT ? kPieceB : kPieceT);
  static constexpr int kC = Pieces<T>::IN * kPieceB;
  static constexpr int kRowCb = kQ + 4;  // floats
  static constexpr int kCb = kQ * kRowCb * 4;
  static constexpr int kScal = 5 * kQ * 4;  // per wave: c (two parts), d, e^c, e^{c_Q - c} d
  static constexpr int bytes(int nw) { return kB + kC + kCb + nw * kScal; }
};

template <typename T, int NT, int NW, bool FULL>
__global__ __launch_bounds__(64 * NW) void k_scan_mm(SsmArgs a, ScanPlan pl, int tiles, int wide) {
  using L = MmLds<T, NT>;
  constexpr int IN = Pieces<T>::IN, YP = Pieces<T>::Y;
  constexpr int kThreads = 64 * NW;
  constexpr int kBlocks = 64 * NT;  // 4x4 blocks of B (or C) in a chunk
  constexpr int kItems = ((FULL ? 2 : 1) * kBlocks + kThreads - 1) / kThreads;
  extern __shared__ float4 sh4[];
  uint8_t* shB = (uint8_t*)sh4;
  uint8_t* shC = shB + L::kB;
  float* shCb = (float*)(shC + L::kC);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, li = lane & 31;
  float* scal = (float*)((uint8_t*)shCb + L::kCb) + wave * (L::kScal / 4);
  float *shHi = scal, *shLo = scal + kQ, *shD = scal + 2 * kQ, *shE = scal + 3 * kQ,
        *shW = scal + 4 * kQ;

  ScanUnit w;
  if (!scan_unit(a.q, blockIdx.x, pl.len, w)) return;
  if (!FULL && w.u.k == w.last) return;
  const int g = blockIdx.y, per = a.heads / a.groups;
  const int ptiles = (a.hd + 31) / 32;
  const int item = blockIdx.z * NW + wave;  // tile of the group
  const bool active = item < tiles;
  const int h = g * per + (active ? item / ptiles : 0);
  const int pt = active ? item % ptiles : 0;
  const int p = pt * 32 + li;
  const bool on = active && p < a.hd;
  const int64_t c = (int64_t)h * a.hd + p;
  const int64_t unit0 = (int64_t)blockIdx.x - w.u.k;
  constexpr int kTile = NT * 16 * 64;  // floats of a state tile in `ends`
  const int64_t tile_at = ((int64_t)h * ptiles + pt) * kTile + lane;
  const int64_t unit_floats = (int64_t)a.heads * ptiles * kTile;

  v16f S[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[nt][r] = 0.0f;
  if (on && w.keep && (FULL ? w.last == 0 : w.u.k == 0)) {
    const float* st = a.state + (int64_t)w.slot * a.ss + c * a.n;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = nt * 32 + acc_row(r, half);
        if (n < a.n) S[nt][r] = st[n];
      }
  }
  if constexpr (!FULL) {
    if (w.u.k == 0) {
      if (active) {
        float* e = pl.ends + (unit0 + w.last) * unit_floats + tile_at;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            e[(nt * 16 + r) * 64] = S[nt][r];
            S[nt][r] = 0.0f;
          }
      }
    }
  } else if (w.last > 0 && active) {
    const float* e = pl.ends + (unit0 + w.last) * unit_floats + tile_at;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[nt][r] = e[(nt * 16 + r) * 64];
    for (int j = 0; j < w.u.k; ++j) {
      e = pl.ends + (unit0 + j) * unit_floats + tile_at;
      const float dec = pl.decays[(unit0 + j) * a.heads + h];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          S[nt][r] = __builtin_fmaf(S[nt][r], dec, e[(nt * 16 + r) * 64]);
    }
  }

  const float A = a.A[h];
  const float Dp = FULL && on && a.D ? a.D[c] : 0.0f;
  double total = 0.0;  // of the unit's exponents, in powers of two

  // the next chunk's values, loaded while a chunk is worked on
  T nx[16], nz[16], ndt = (T)0.0f;
  Pack<T, 4> nb[kItems][4];
  auto fetch = [&](int t) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int id = tid + k * kThreads;
      if (id >= (FULL ? 2 : 1) * kBlocks) continue;
      const bool isC = id >= kBlocks;
      const int blk = isC ? id - kBlocks : id;
      const int n = blk % (8 * NT) * 4, j = blk / (8 * NT) * 4;
      const T* src = (const T*)(isC ? a.C : a.B) + (int64_t)g * a.n + n;
      const int64_t stride = isC ? a.Cs : a.Bs;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool row = t + j + q < w.t1;
        const T* s = src + (int64_t)(t + j + q) * stride;
        if (wide) {
          if (row && n < a.n) nb[k][q] = *(const Pack<T, 4>*)s;
          else nb[k][q] = Pack<T, 4>{{(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f}};
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) nb[k][q].v[i] = row && n + i < a.n ? s[i] : (T)0.0f;
        }
      }
    }
    const T* xp = (const T*)a.x + c;
    const T* zp = (const T*)a.z + c;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t row = t + acc_row(r, half);
      const bool in = on && row < w.t1;
      nx[r] = in ? xp[row * a.xs] : (T)0.0f;
      if (FULL && a.z) nz[r] = in ? zp[row * a.zs] : (T)0.0f;
    }
    if (active && t + li < w.t1) ndt = ((const T*)a.dt)[(int64_t)(t + li) * a.dts + h];
  };
  if (w.t0 < w.t1) fetch(w.t0);

  for (int t = w.t0; t < w.t1; t += kQ) {
    // this chunk's values out of the fetched ones; B and C by rows into LDS
    float x[16], z[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = (float)nx[r];
      if (FULL) z[r] = (float)nz[r];
    }
    Pack<T, 4> b[kItems][4];
#pragma unroll
    for (int k = 0; k < kItems; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) b[k][q] = nb[k][q];
    const float d = active && t + li < w.t1 ? step_of(a, (float)ndt, h) : 0.0f;
    if (t + kQ < w.t1) fetch(t + kQ);
    if constexpr (FULL) {
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        const int id = tid + k * kThreads;
        if (id >= 2 * kBlocks) continue;
        const bool isC = id >= kBlocks;
        const int blk = isC ? id - kBlocks : id;
        const int n = blk % (8 * NT) * 4, j = blk / (8 * NT) * 4;
        // four values' place in their 16: quarters 0, 2 | 1, 3
        const int at = (n & ~15) + ((n >> 2) & 1) * 8 + ((n >> 3) & 1) * 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = (float)b[k][q].v[i];
#pragma unroll
          for (int pc = 0; pc < IN; ++pc) {
            Pack<__bf16, 4> o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o.v[i] = (__bf16)v[i];
              v[i] -= (float)o.v[i];
            }
            *(Pack<__bf16, 4>*)((isC ? shC : shB) + pc * L::kPieceB + (j + q) * L::kRowB + at * 2) = o;
          }
        }
      }
    }
    // the chunk's exponents, by lane li (both halves alike)
    double cum = (double)A * (double)d * 1.4426950408889634;
    cum = cum < -256.0 ? -256.0 : (cum > 256.0 ? 256.0 : cum);
#pragma unroll
    for (int m = 1; m < kQ; m <<= 1) {
      const double o = __shfl_up(cum, m, kQ);
      if (li >= m) cum += o;
    }
    const double whole = __shfl(cum, kQ - 1, kQ);
    total += whole;
    const float eall = __builtin_amdgcn_exp2f((float)whole);
    if (half == 0) {
      const float hi = (float)cum;
      shHi[li] = hi;
      shLo[li] = (float)(cum - (double)hi);
      shD[li] = d;
      shE[li] = __builtin_amdgcn_exp2f(hi);
      shW[li] = __builtin_amdgcn_exp2f((float)(whole - cum)) * d;
    }
    __syncthreads();

    v16f Y;
    if constexpr (FULL) {
      // C B^T of the chunk: three 16x16 tiles on and below the diagonal
      if (wave < 3) {
        const int jt = wave == 2 ? 16 : 0, it = wave == 0 ? 0 : 16;
        const int lr = lane & 15, lg = lane >> 4;
        v4f cb = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          v8bf pb[IN], pc[IN];
#pragma unroll
          for (int i = 0; i < IN; ++i) {
            pb[i] = *(const v8bf*)(shB + i * L::kPieceB + (jt + lr) * L::kRowB + (32 * k + 8 * lg) * 2);
            pc[i] = *(const v8bf*)(shC + i * L::kPieceB + (it + lr) * L::kRowB + (32 * k + 8 * lg) * 2);
          }
#pragma unroll
          for (int i = 0; i < IN; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j)
              if (i + j < YP) cb = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pb[i], pc[j], cb, 0, 0, 0);
        }
        *(v4f*)(shCb + (it + lr) * L::kRowCb + jt + 4 * lg) = cb;
      }
      // C S, scaled by e^{c_i}
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
      __syncthreads();  // C B^T is whole, B by rows is done with
    }
    // B^T into its place
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int id = tid + k * kThreads;
      if (id >= kBlocks) continue;  // C's
      const int n = id % (8 * NT) * 4, j = id / (8 * NT) * 4;
      const int at = (j & ~15) + ((j >> 2) & 1) * 8 + ((j >> 3) & 1) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = (float)b[k][q].v[i];
#pragma unroll
        for (int pc = 0; pc < IN; ++pc) {
          Pack<__bf16, 4> o;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            o.v[q] = (__bf16)v[q];
            v[q] -= (float)o.v[q];
          }
          *(Pack<__bf16, 4>*)(shB + pc * L::kPieceT + (n + i) * L::kRowT + at * 2) = o;
        }
      }
    }
    // the weighted x, for the state
    v8bf xw[2][kStatePieces];
    {
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
    }
    if constexpr (FULL) {
      // M x within the chunk
      bool odd = false;
#pragma unroll
      for (int r = 0; r < 16; ++r) odd |= !(__builtin_fabsf(x[r]) < __builtin_inff());
      int first = kQ;
      if (__ballot(odd)) {
#pragma unroll
        for (int r = 15; r >= 0; --r)
          if (!(__builtin_fabsf(x[r]) < __builtin_inff())) {
            first = acc_row(r, half);
            x[r] = 0.0f;
          }
        first = min(first, __shfl_xor(first, 32));
      }
      const float hi = shHi[li], lo = shLo[li];
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
          m[4 * q + i] = j0 + i <= li ? cbv[i] * (e * d4[i]) : 0.0f;
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v8bf pm[YP], px[IN];
        split8<YP>(pm, m + 8 * s);
        split8<IN>(px, x + 8 * s);
        Y = mfma32<YP>(pm, px, Y);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = acc_row(r, half);
        float v = i < first ? Y[r] : __builtin_nanf("");
        v = __builtin_fmaf(Dp, x[r], v);
        if (a.z) v *= silu_f32(z[r]);
        if (on && t + i < w.t1) ((T*)a.y)[(int64_t)(t + i) * a.ys + c] = (T)v;
      }
    }
    __syncthreads();  // B^T is whole
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) S[nt][r] *= eall;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v8bf pb[IN];
#pragma unroll
        for (int i = 0; i < IN; ++i)
          pb[i] = *(const v8bf*)(shB + i * L::kPieceT + (32 * nt + li) * L::kRowT + (16 * s + 8 * half) * 2);
        S[nt] = mfma32<kStatePieces>(pb, xw[s], S[nt]);
      }
    }
    __syncthreads();  // the next chunk may overwrite LDS
  }

  if constexpr (!FULL) {
    if (!active) return;
    float* e = pl.ends + (int64_t)blockIdx.x * unit_floats + tile_at;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) e[(nt * 16 + r) * 64] = S[nt][r];
    if (pt == 0 && lane == 0)
      pl.decays[(int64_t)blockIdx.x * a.heads + h] = __builtin_amdgcn_exp2f((float)total);
  } else if (on && w.slot >= 0 && w.u.k == w.last) {
    float* st = a.state + (int64_t)w.slot * a.ss + c * a.n;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = nt * 32 + acc_row(r, half);
        if (n < a.n) st[n] = S[nt][r];
      }
  }
}

static int mm_ptiles(int hd) { return (hd + 31) / 32; }
static int mm_nt(int n) { return n <= 32 ? 1 : (n <= 64 ? 2 : (n <= 128 ? 4 : 8)); }
// waves per block: eight where a group has that many tiles and the state
// leaves room for two waves per SIMD
static int mm_waves(int tiles, int nt) { return tiles > 4 && nt < 8 ? 8 : 4; }

template <typename T, int NT, int NW>
static hipError_t launch_mm(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  const int tiles = a.heads / a.groups * mm_ptiles(a.hd);
  constexpr int bytes = MmLds<T, NT>::bytes(NW);
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  const int wide = a.n % 4 == 0 && a.Bs % 4 == 0 && a.Cs % 4 == 0 &&
                   ((uintptr_t)a.B | (uintptr_t)a.C) % (4 * sizeof(T)) == 0;
  const dim3 grid((unsigned)pl.units, a.groups, (tiles + NW - 1) / NW);
  if (bytes > 64 * 1024) {  // once per process: a kernel's limit above the default
    static const hipError_t raised[2] = {
        hipFuncSetAttribute((const void*)k_scan_mm<T, NT, NW, false>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
        hipFuncSetAttribute((const void*)k_scan_mm<T, NT, NW, true>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes)};
    if (raised[0] != hipSuccess) return raised[0];
    if (raised[1] != hipSuccess) return raised[1];
  }
  if (pl.split)
    hipLaunchKernelGGL((k_scan_mm<T, NT, NW, false>), grid, dim3(64 * NW), bytes, s, a, pl, tiles,
                       wide);
  hipLaunchKernelGGL((k_scan_mm<T, NT, NW, true>), grid, dim3(64 * NW), bytes, s, a, pl, tiles,
                     wide);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_mm_t(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  const int nt = mm_nt(a.n);
  const bool w8 = mm_waves(a.heads / a.groups * mm_ptiles(a.hd), nt) == 8;
  switch (nt) {
    case 1: return w8 ? launch_mm<T, 1, 8>(a, pl, s) : launch_mm<T, 1, 4>(a, pl, s);
    case 2: return w8 ? launch_mm<T, 2, 8>(a, pl, s) : launch_mm<T, 2, 4>(a, pl, s);
    case 4: return w8 ? launch_mm<T, 4, 8>(a, pl, s) : launch_mm<T, 4, 4>(a, pl, s);
    default: return launch_mm<T, 8, 4>(a, pl, s);
  }
}

// ---- the cut into units ----------------------------------------------------
// Units as short as the chip needs to be filled (kFillWaves waves over all of
// them), but no shorter than what the first pass and the walk over a
// sequence's units are worth, and no more than 32 (64) of them in a sequence.
constexpr int kFillWaves = 2048;

static ScanPlan scan_plan(const bm_hip_ssm_t* op, size_t* bytes) {
  ScanPlan pl{};
  const int64_t channels = (int64_t)op->n_heads * op->head_dim;
  const bool small = op->d_state <= kSmallState;
  const int64_t waves = small ? (channels + 63) / 64
                              : (int64_t)op->n_heads * mm_ptiles(op->head_dim);
  const int step = small ? 32 : kQ, least = small ? 32 : 4 * kQ, most_units = small ? 64 : 32;
  const int64_t T = op->n_tokens;
  const int64_t want = kFillWaves / waves > 1 ? kFillWaves / waves : 1;
  int64_t len = (T / want + step) / step * step;
  const int64_t floor_len = (T / most_units + step) / step * step;
  if (len > 512) len = 512;  // uneven lengths: the longest sequence is cut too
  if (len < floor_len) len = floor_len;
  if (len < least) len = least;
  pl.len = (int)len;
  pl.split = T > len;
  pl.units = unit_count(op->n_seqs, op->n_tokens, pl.len);
  const int64_t floats =
      small ? channels * op->d_state
            : (int64_t)op->n_heads * mm_ptiles(op->head_dim) * mm_nt(op->d_state) * 1024;
  const size_t ends = align_up((size_t)pl.units * floats * 4, 256);
  *bytes = pl.split ? ends + (size_t)pl.units * op->n_heads * 4 : 0;
  pl.decays = (float*)ends;  // its offset, until the workspace is known
  return pl;
}

template <typename T>
static hipError_t launch_scan_t(const SsmArgs& a, const ScanPlan& pl, hipStream_t s) {
  if (a.n > kSmallState) return launch_mm_t<T>(a, pl, s);
  constexpr int V = 4;
  const bool wide = a.hd % V == 0 && a.xs % V == 0 && a.ys % V == 0 && (!a.z || a.zs % V == 0) &&
                    ((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.z) % (V * sizeof(T)) == 0;
  (void)wide;
  return launch_small_n<T, 1>(a, pl, s);
}

static bool shape_fits(const char* name, const bm_hip_ssm_t* op) {
  if (!op) {
    bm_set_error("%s: no descriptor", name);
    return false;
  }
  if (op->type < BM_HIP_F32 || op->type > BM_HIP_F16 || op->n_heads < 1 || op->n_heads > 65535 ||
      op->head_dim < 1 || op->head_dim > 65535 || op->n_groups < 1 ||
      op->n_heads % op->n_groups || op->d_state < 1 || op->d_state > 256 ||
      (int64_t)op->n_heads * op->head_dim > (1 << 22)) {
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
  if (!bm::check_rows(name, "y", op->y, op->y_stride, hp, elem)) return -2;
  for (const auto& t : in) {
    if (!op->z && &t == &in[4]) continue;  // no gate
    if (!bm::check_rows(name, t.name, t.p, t.stride, t.width, elem) ||
        !bm::check_apart(name, t.name, t.p, t.stride, t.width, op->y, op->y_stride, hp, rows, elem,
                         step && t.p == op->x))
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
    if (bytes && (!workspace || (uintptr_t)workspace % 256)) {
      bm_set_error("%s: a workspace of %zu bytes on 256 bytes is required", name, bytes);
      return -2;
    }
    if (pl.units > 0x7fffffff) {
      bm_set_error("%s: too many rows for one call", name);
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
