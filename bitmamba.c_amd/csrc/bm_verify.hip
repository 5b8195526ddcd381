// Verification of drafted tokens against the target's distributions, and the
// token that follows (include/bm_hip.h):
//
//   row i stands while u_i q_i(d_i) < p_i(d_i);  then a draw from
//   max(p - q, 0) of the first row that does not, or from p of the last.
//
// Three launches: the sum and maximum of every row in segments (k_verify_rows);
// what is decided from them, and the sum that the draw needs, in segments
// (k_verify_stop); the segment and the token of the draw (k_verify_draw).  A
// greedy target needs the first two only.
//
// A draw falls between two neighbouring tokens of up to 256000, so every
// error of a running sum moves draws by that much: exponentials and sums are in
// fp64, in an order that depends on the sizes alone.  The exponential's polynomial
// is off by 2^-46 of it, the rounding of its argument t, in bits, by |t| 2^-53 at most.
#include <math.h>

#include "bm_dev.h"
#include "bm_seq.h"

namespace bm {

constexpr int kSegment = 4096;  // values of a row per block
// threads and values of each: many of one row's values in flight where all rows
// are read, short chains where a sequence waits for one
constexpr int kRowsThreads = 256, kRowsValues = kSegment / kRowsThreads;
constexpr int kDrawThreads = 1024, kDrawValues = kSegment / kDrawThreads;
constexpr int kMaxVocab = 256000;
static_assert((kMaxVocab + kSegment - 1) / kSegment <= 64, "a segment per lane");

enum RowKind { kLogits, kWeights, kLargest, kToken };

// A row's segment, or a whole row: the largest value, the sum of 2^{(v - m) k}
// (of the values themselves for weights), and where the largest is first
struct RowSum {
  double s;
  float m;
  int at;
};
// What the draw of a sequence goes by
struct Draw {
  int row;             // -1: none
  float u;
  int p_kind, q_kind;  // q_kind -1: p alone
  float pm, qm;        // maxima
  int q_at;            // of a q that is 1 at one token
  int pad;
  double p_inv, q_inv;  // 1 / sum
};

struct VerifyArgs {
  SeqView q;
  int vocab, segments;
  int p_kind, q_kind;
  const void *p, *d;
  int64_t ps, ds;
  double k;  // log2(e) / temp
  const int32_t* tokens;
  const float* u;
  int32_t *accepted, *next, *split;
  float* ratio;
  RowSum* sums;  // [2][rows][segments]
  double* rest;  // [sequences][segments]
  Draw* draws;   // [sequences]
};

// 2^t for t at most 0 (NaN: 0): a polynomial on the fraction that is off by
// 2^-46 at most (fitted to 2^f on -1/2 .. 1/2 by exchange of its extrema)
__device__ __forceinline__ double exp2_f64(double t) {
  constexpr double c[10] = {0x1.0000000000039p+0,  0x1.62e42fefa3752p-1,  0x1.ebfbdff81570dp-3,
                            0x1.c6b08d70d2003p-5,  0x1.3b2ab72a1098dp-7,  0x1.5d87fd9011eeep-10,
                            0x1.43088fca9a183p-13, 0x1.ffce24611c0dap-17, 0x1.63edf1058a76ep-20,
                            0x1.b3f421492867dp-24};
  // the larger one, -1100 for NaN: one instruction, where fmax() takes two
  asm("v_max_f64 %0, %1, %2" : "=v"(t) : "v"(t), "s"(-1100.0));
  const double n = __builtin_rint(t), f = t - n;
  double r = c[9];
  // with the coefficient in scalar registers; the compiler copies each into the
  // result's registers first, two moves per step
#pragma unroll
  for (int i = 8; i >= 0; --i)
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(r), "v"(f), "s"(c[i]));
  return __builtin_ldexp(r, (int)n);
}
// What a row's shares are taken from: its largest value, or 0 where that is no
// finite one
struct Top {
  double m;
  bool odd;  // the largest is infinite: +inf has everything, or there is nothing
  float at;
};
__device__ __forceinline__ Top top_of(float m) {
  const bool odd = !(__builtin_fabsf(m) < __builtin_inff());
  return Top{odd ? 0.0 : (double)m, odd, m};
}
// a value's share of a row, up to the row's sum
__device__ __forceinline__ double share_of(int kind, float v, const Top& m, double k) {
  if (kind == kWeights) return v > 0.0f && v < __builtin_inff() ? (double)v : 0.0;
  if (m.odd) return m.at > 0.0f && v == m.at ? 1.0 : 0.0;
  return exp2_f64(((double)v - m.m) * k);
}

// the shares of N values; one branch for all of them
template <int N>
__device__ __forceinline__ void shares(double (&o)[N], int kind, const float (&v)[N], float largest,
                                       double k) {
  const Top top = top_of(largest);
  if (kind == kWeights) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = share_of(kWeights, v[j], top, k);
  } else if (top.odd) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = top.at > 0.0f && v[j] == top.at ? 1.0 : 0.0;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = exp2_f64(((double)v[j] - top.m) * k);
  }
}

// Values i .. i + N - 1 of a row on any alignment of T; `none` past its end.
// Words of four bytes are read, so a row of two-byte values that starts or ends
// within a word is read with its neighbour in that word.
template <int W>
struct alignas(4) Words {
  uint32_t w[W];
};
template <typename T, int N>
__device__ __forceinline__ void load_row_at(float (&o)[N], const T* row, int i, int vocab, float none) {
  static_assert(N % 4 == 0, "");
  if (i + N > vocab) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = i + j < vocab ? (float)row[i + j] : none;
    return;
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const Words<4> v = *(const Words<4>*)(row + i + j);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[j + k] = __uint_as_float(v.w[k]);
    }
  } else {
    const uintptr_t at = (uintptr_t)(row + i);
    const int odd = (int)(at >> 1 & 1);  // the same for the whole row, i being even
    const uint32_t* w = (const uint32_t*)(at - 2 * odd);
    constexpr int kWords = N / 2, kEach = kWords < 4 ? kWords : 4;
    uint32_t v[kWords + 1];
#pragma unroll
    for (int j = 0; j < kWords; j += kEach) {
      const Words<kEach> x = *(const Words<kEach>*)(w + j);
#pragma unroll
      for (int k = 0; k < kEach; ++k) v[j + k] = x.w[k];
    }
    v[kWords] = odd ? w[kWords] : 0;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const uint32_t x = odd ? __builtin_amdgcn_alignbit(v[j + 1], v[j], 16) : v[j];
      o[2 * j] = (float)__builtin_bit_cast(T, (uint16_t)x);
      o[2 * j + 1] = (float)__builtin_bit_cast(T, (uint16_t)(x >> 16));
    }
  }
}

// running sums over the wave on DPP
__device__ __forceinline__ double wave_scan_f64(double v) {
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
__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane),
                 hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) { return read_lane(wave_scan_f64(v), 63); }
__device__ __forceinline__ int wave_min_i32(int v) {
  v = min(v, dpp_mov<0xB1>(v));
  v = min(v, dpp_mov<0x4E>(v));
  v = min(v, dpp_mov<0x141>(v));
  v = min(v, dpp_mov<0x140>(v));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// what a sum to the largest value v counts in one to m
__device__ __forceinline__ double from_top(float v, float m, double k) {
  return v == m ? 1.0 : exp2_f64(((double)v - (double)m) * k);
}
// the maximum of four waves' and the sum to it
template <int N>
__device__ __forceinline__ RowSum join_sums(int kind, const RowSum (&v)[N], double k) {
  RowSum o = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (v[i].m > o.m) {  // the first of equal ones stays
      o.m = v[i].m;
      o.at = v[i].at;
    }
  o.s = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    o.s += kind == kWeights ? v[i].s : v[i].s * from_top(v[i].m, o.m, k);
  return o;
}

// ---------------------------------------------------------------------------
// One segment of one row of the target (y 0) or the draft (y 1).
// A pass over all rows: 480 rows of 256000 fp32 logits (491 MB) take 114 to 136 us,
// 3.6 to 4.3 TB/s, the vector units busy 83 % of it with exponentials in fp64;
// greedy rows in fp16 (129 MB) 33 to 38 us.  128 threads of 32 values take 30 us for
// those, but longer for fp32 and for few rows (one greedy sequence of 5: all of
// the call 8.6 us against 7.4).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kRowsThreads) void k_verify_rows(VerifyArgs a) {
  __shared__ RowSum part[kRowsThreads / 64];
  const bool draft = blockIdx.y != 0;
  const int64_t block = wide_block();
  const int64_t row = block / a.segments;
  if (row >= a.q.n_tokens) return;
  const int seg = (int)(block - row * a.segments);
  const int kind = draft ? a.q_kind : a.p_kind;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i0 = seg * kSegment + tid * kRowsValues;
  const float none = kind == kWeights ? 0.0f : -__builtin_inff();
  float v[kRowsValues];
  if (!draft) load_row_at<T>(v, (const T*)a.p + row * a.ps, i0, a.vocab, none);  // in the search's shadow
  int end;
  if (find_row(a.q, (int)row, &end) < 0 || (draft && row == end - 1)) return;
  if (draft) load_row_at<T>(v, (const T*)a.d + row * a.ds, i0, a.vocab, none);
  RowSum o{0.0, -__builtin_inff(), INT32_MAX};
#pragma unroll
  for (int j = 0; j < kRowsValues; ++j) o.m = fmaxf(o.m, v[j]);
  o.m = wave_max_f32(o.m);
  if (kind == kLargest) {
#pragma unroll
    for (int j = kRowsValues - 1; j >= 0; --j)
      if (v[j] == o.m) o.at = i0 + j;
    o.at = wave_min_i32(o.at);
  } else {
    double w[kRowsValues];
    shares(w, kind, v, o.m, a.k);
#pragma unroll
    for (int j = 0; j < kRowsValues; ++j) o.s += w[j];
    o.s = wave_sum_f64(o.s);
  }
  if (lane == 0) part[wave] = o;
  __syncthreads();
  if (tid == 0)
    a.sums[(row + (draft ? a.q.n_tokens : 0)) * a.segments + seg] =
        join_sums(kind == kLargest ? (int)kWeights : kind, part, a.k);
}

// a row's segments, one per lane, and the whole row, in all lanes
__device__ __forceinline__ RowSum load_sum(const VerifyArgs& a, int64_t row, bool draft) {
  const int lane = threadIdx.x & 63;
  RowSum o{0.0, -__builtin_inff(), INT32_MAX};
  if (lane < a.segments) o = a.sums[(row + (draft ? a.q.n_tokens : 0)) * a.segments + lane];
  return o;
}
__device__ __forceinline__ RowSum whole_sum(const VerifyArgs& a, int kind, RowSum o) {
  const float m = wave_max_f32(o.m);
  if (kind == kLargest) {
    o.at = wave_min_i32(o.m == m && m > -__builtin_inff() ? o.at : INT32_MAX);
    if (o.at == INT32_MAX) o.at = -1;
    o.s = o.at < 0 ? 0.0 : 1.0;
  } else {
    if (kind == kLogits) o.s *= from_top(o.m, m, a.k);
    o.s = wave_sum_f64(o.s);
  }
  o.m = m;
  return o;
}
// the probability of a token of the vocabulary, given its value and the row's sum
__device__ __forceinline__ double prob_of(const VerifyArgs& a, int kind, float v, const RowSum& r,
                                          int token) {
  if (kind == kToken) return 1.0;
  if (kind == kLargest) return token == r.at ? 1.0 : 0.0;
  return r.s > 0.0 ? share_of(kind, v, top_of(r.m), a.k) / r.s : 0.0;
}

// a token's weight in the draw
template <typename T, int N>
__device__ __forceinline__ void draw_weights(double (&w)[N], const VerifyArgs& a,
                                          const Draw& d, int i0) {
  float v[N];
  load_row_at<T>(v, (const T*)a.p + (int64_t)d.row * a.ps, i0, a.vocab,
            d.p_kind == kWeights ? 0.0f : -__builtin_inff());
  shares(w, d.p_kind, v, d.pm, a.k);
#pragma unroll
  for (int j = 0; j < N; ++j) w[j] *= d.p_inv;
  if (d.q_kind < 0) return;
  if (d.q_kind == kToken) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = i0 + j == d.q_at ? 0.0 : w[j];
    return;
  }
  load_row_at<T>(v, (const T*)a.d + (int64_t)d.row * a.ds, i0, a.vocab,
            d.q_kind == kWeights ? 0.0f : -__builtin_inff());
  double q[N];
  shares(q, d.q_kind, v, d.qm, a.k);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const double left = w[j] - q[j] * d.q_inv;
    w[j] = left > 0.0 ? left : 0.0;
  }
}

// ---------------------------------------------------------------------------
// The rows of a sequence in turn, a wave each, until one is refused; then a
// segment of the draw's weights.  Every block of a sequence decides for itself
// (a launch of its own would cost more than the few rows of a draft); the
// first writes what was decided, and goes through all rows for their ratios.
// Bound by the round trips of that chain: 6.6 us for one sequence of 5 rows, 12 us
// for 64 of up to 8.
// ---------------------------------------------------------------------------
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_verify_stop(VerifyArgs a, int blocks) {
  constexpr int kWavesV = THREADS / 64, kValues = kSegment / THREADS;
  __shared__ Draw shared;
  __shared__ int first;
  __shared__ double part[kWavesV];
  const int64_t block = wide_block();
  const int b = (int)(block / blocks), seg = (int)(block - (int64_t)b * blocks);
  if (b >= a.q.n_seqs) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int s = a.q.seq_start ? seq_row(a.q, b) : 0;
  const int e = a.q.seq_start ? max(s, seq_row(a.q, b + 1)) : a.q.n_tokens;
  const bool writer = seg == 0;
  if (writer && tid == 0 && a.split) {
    a.split[2 * (int64_t)b] = s;
    if (b == a.q.n_seqs - 1) a.split[2 * (int64_t)b + 2] = a.q.seq_start ? e : a.q.n_tokens;
  }
  if (e == s) {
    if (writer && tid == 0) {
      a.accepted[b] = 0;
      a.next[b] = -1;
      a.draws[b].row = -1;
      if (a.split) a.split[2 * (int64_t)b + 1] = s;
    }
    return;
  }
  const float u_last = a.u[e - 1];
  if (tid == 0) first = INT32_MAX;
  __syncthreads();
  for (int r0 = s; r0 < e; r0 += kWavesV) {
    const int row = r0 + wave;
    const bool have = row < e, last = row == e - 1;
    RowSum p{0.0, 0.0f, -1}, q{1.0, 0.0f, -1};
    int token = -1;
    if (have) {
      const bool drawn = !last && a.q_kind != kToken && a.p_kind != kLargest;
      // all loads of a row before anything is made of them
      if (!last) token = a.tokens[row];
      const float u = last ? 0.0f : a.u[row];
      p = load_sum(a, row, false);
      if (drawn) q = load_sum(a, row, true);
      const bool inside = token >= 0 && token < a.vocab;
      const float pv = inside ? (float)((const T*)a.p)[row * a.ps + token] : 0.0f;
      const float qv = inside && drawn ? (float)((const T*)a.d)[row * a.ds + token] : 0.0f;
      p = whole_sum(a, a.p_kind, p);
      bool stands = false;
      if (drawn) q = whole_sum(a, a.q_kind, q);
      if (!last) {
        const double pd = inside ? prob_of(a, a.p_kind, pv, p, token) : 0.0;
        const double qd = inside ? prob_of(a, a.q_kind, qv, q, token) : 0.0;
        stands = a.p_kind == kLargest ? pd > 0.0 : (double)u * qd < pd;
        if (writer && a.ratio && lane == 0)
          a.ratio[row] = pd > 0.0 ? (a.p_kind == kLargest || pd >= qd ? 1.0f : (float)(pd / qd)) : 0.0f;
      }
      if (!stands && lane == 0) atomicMin(&first, row);
    }
    __syncthreads();
    const int stop = first;  // read by all before any wave goes on to write it
    if (have && row == stop && lane == 0) {
      Draw d;
      d.row = p.s > 0.0 ? row : -1;
      d.u = u_last;
      d.p_kind = a.p_kind;
      d.pm = p.m;
      d.p_inv = p.s > 0.0 ? 1.0 / p.s : 0.0;
      d.q_kind = last ? -1 : (a.q_kind == kLargest ? (int)kToken : a.q_kind);
      d.qm = q.m;
      d.q_at = a.q_kind == kToken ? token : q.at;
      d.q_inv = q.s > 0.0 ? 1.0 / q.s : 0.0;
      d.pad = 0;
      shared = d;
      if (writer) {
        a.draws[b] = d;
        a.accepted[b] = row - s;
        if (a.p_kind == kLargest) a.next[b] = p.at;
        if (a.split) a.split[2 * (int64_t)b + 1] = row + 1;
      }
    }
    __syncthreads();
    if (stop != INT32_MAX && !(writer && a.ratio)) break;
  }
  if (a.p_kind == kLargest) return;
  const Draw d = shared;
  double sum = 0.0;
  if (d.row >= 0) {
    double w[kValues];
    draw_weights<T>(w, a, d, seg * kSegment + tid * kValues);
#pragma unroll
    for (int j = 0; j < kValues; ++j) sum += w[j];
  }
  sum = wave_sum_f64(sum);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = part[0];
#pragma unroll
    for (int i = 1; i < kWavesV; ++i) sum += part[i];
    a.rest[(int64_t)b * a.segments + seg] = sum;
  }
}

// ---------------------------------------------------------------------------
// The draw of one sequence: the segment in which the running sum passes u
// times the whole, then the token in it.  A launch's latency, 4 to 7 us.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kDrawThreads) void k_verify_draw(VerifyArgs a) {
  constexpr int kWavesV = kDrawThreads / 64;
  __shared__ double part[kWavesV];
  __shared__ int at[kWavesV], most[kWavesV];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Draw d = a.draws[b];
  if (d.row < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  double mine = lane < a.segments ? a.rest[(int64_t)b * a.segments + lane] : 0.0;
  if (__ballot(mine > 0.0) == 0) {  // the draft has all of it: from p
    d.q_kind = -1;
    if (lane < a.segments) {
      const RowSum o = a.sums[(int64_t)d.row * a.segments + lane];
      mine = o.s * d.p_inv;
      if (d.p_kind == kLogits) mine *= from_top(o.m, d.pm, a.k);
    }
  }
  const double run = wave_scan_f64(mine);
  const double want = (double)d.u * read_lane(run, 63);
  const uint64_t in = __ballot(mine > 0.0 && run > want);
  const uint64_t any = __ballot(mine > 0.0);
  const int seg = in ? __ffsll((unsigned long long)in) - 1
                     : (any ? 63 - __clzll((long long)any) : 0);
  const double before = seg > 0 ? read_lane(run, seg - 1) : 0.0;
  double w[kDrawValues], sum = 0.0;
  const int i0 = seg * kSegment + tid * kDrawValues;
  draw_weights<T>(w, a, d, i0);
#pragma unroll
  for (int j = 0; j < kDrawValues; ++j) sum += w[j];
  const double upto = wave_scan_f64(sum);
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  double c = before;
  for (int i = 0; i < wave; ++i) c += part[i];
  c += upto - sum;
  int got = INT32_MAX, last = -1;
#pragma unroll
  for (int j = 0; j < kDrawValues; ++j) {
    c += w[j];
    if (w[j] > 0.0) {
      last = i0 + j;
      if (got == INT32_MAX && c > want) got = i0 + j;
    }
  }
  got = wave_min_i32(got);
  last = -wave_min_i32(-last);
  if (lane == 0) {
    at[wave] = got;
    most[wave] = last;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kWavesV; ++i) {
      got = min(got, at[i]);
      last = max(last, most[i]);
    }
    a.next[b] = got != INT32_MAX ? got : last;
  }
}

template <typename T>
static hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const bool greedy = a.p_kind == kLargest, rows_of_draft = a.q_kind != kToken && !greedy;
  if (a.q.n_tokens > 0) {
    const hipError_t e = launch(k_verify_rows<T>, wide_grid((int64_t)a.q.n_tokens * a.segments,
                                                            rows_of_draft ? 2 : 1),
                                dim3(kRowsThreads), 0, s, a);
    if (e != hipSuccess) return e;
  }
  const int blocks = greedy ? 1 : a.segments;
  // Blocks that all run at once end sooner with more waves (one sequence of five
  // rows of 50257: 6.9 us with 1024 threads, 8.4 with 256); of more blocks each
  // wave repeats the decision (64 sequences: 22 and 12 us).
  const int64_t all = (int64_t)a.q.n_seqs * blocks;
  const dim3 grid = wide_grid(all, 1);
  const hipError_t e = all <= 256 ? launch(k_verify_stop<T, 1024>, grid, dim3(1024), 0, s, a, blocks)
                                  : launch(k_verify_stop<T, 256>, grid, dim3(256), 0, s, a, blocks);
  if (e != hipSuccess || greedy) return e;
  return launch(k_verify_draw<T>, dim3(a.q.n_seqs), dim3(kDrawThreads), 0, s, a);
}

struct VerifySpace {
  size_t sums, rest, draws, bytes;
};
static VerifySpace verify_space(int64_t rows, int64_t seqs, int vocab) {
  const int64_t segments = (vocab + kSegment - 1) / kSegment;
  VerifySpace v;
  v.sums = 0;
  v.rest = align_up((size_t)(2 * rows * segments) * sizeof(RowSum), 256);
  v.draws = v.rest + align_up((size_t)(seqs * segments) * sizeof(double), 256);
  v.bytes = v.draws + (size_t)seqs * sizeof(Draw);
  return v;
}

static bool verify_fits(const char* name, const bm_hip_verify_t* op) {
  if (!op) {
    bm_set_error("%s: no descriptor", name);
    return false;
  }
  if (op->type < BM_HIP_F32 || op->type > BM_HIP_F16 || op->vocab < 1 || op->vocab > kMaxVocab ||
      op->n_seqs < 0 || op->n_seqs > (1 << 20) || op->n_rows < 0 || op->n_rows >= (1 << 30)) {
    bm_set_error("%s: invalid arguments (type=%d vocab=%d n_seqs=%d n_rows=%d)", name, op->type,
                 op->vocab, op->n_seqs, op->n_rows);
    return false;
  }
  return true;
}

}  // namespace bm

extern "C" size_t bm_hip_verify_workspace_bytes(const bm_hip_verify_t* op) {
  if (!bm::verify_fits("verify_workspace", op)) return 0;
  return bm::verify_space(op->n_rows, op->n_seqs, op->vocab).bytes;
}

extern "C" int bm_hip_verify_dev(const bm_hip_verify_t* op, void* workspace, void* stream) {
  if (!bm::verify_fits("verify", op)) return -2;
  const size_t elem = bm::type_bytes(op->type);
  if (!op->row_start && op->n_seqs > 1) {
    bm_set_error("verify: %d sequences need row_start", op->n_seqs);
    return -2;
  }
  if (!bm::check_rows("verify", "target", op->target, op->target_stride, op->vocab, op->n_rows,
                      elem) ||
      (op->draft && !bm::check_rows("verify", "draft", op->draft, op->draft_stride, op->vocab,
                                    op->n_rows, elem)))
    return -2;
  if (!isfinite(op->temp) || op->temp < 0.0f) {
    bm_set_error("verify: temp=%g (0 and more)", op->temp);
    return -2;
  }
  if ((op->n_rows > 0 && (!op->tokens || !op->u)) ||
      (op->n_seqs > 0 && (!op->n_accepted || !op->next_token || !workspace)) ||
      (((uintptr_t)op->row_start | (uintptr_t)op->tokens | (uintptr_t)op->u |
        (uintptr_t)op->n_accepted | (uintptr_t)op->next_token | (uintptr_t)op->ratio |
        (uintptr_t)op->split_start) % 4) ||
      (uintptr_t)workspace % 256) {
    bm_set_error("verify: tokens, u, n_accepted, next_token and a workspace of %zu bytes are "
                 "required, lists on 4 bytes, the workspace on 256",
                 bm_hip_verify_workspace_bytes(op));
    return -2;
  }
  if (op->n_seqs == 0) return 0;
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  const bool greedy = op->temp < 0.05f;
  bm::VerifyArgs a;
  a.q = bm::SeqView{op->row_start, nullptr, nullptr, op->n_seqs, op->n_rows, 0};
  a.vocab = op->vocab;
  a.segments = (op->vocab + bm::kSegment - 1) / bm::kSegment;
  a.p_kind = op->target_weights ? bm::kWeights : (greedy ? bm::kLargest : bm::kLogits);
  a.q_kind = !op->draft ? bm::kToken
                        : (op->draft_weights ? bm::kWeights : (greedy ? bm::kLargest : bm::kLogits));
  a.p = op->target;
  a.d = op->draft;
  a.ps = op->target_stride;
  a.ds = op->draft_stride;
  a.k = greedy ? 1.0 : 1.4426950408889634 / (double)op->temp;
  a.tokens = op->tokens;
  a.u = op->u;
  a.accepted = op->n_accepted;
  a.next = op->next_token;
  a.split = op->split_start;
  a.ratio = op->ratio;
  const bm::VerifySpace space = bm::verify_space(op->n_rows, op->n_seqs, op->vocab);
  a.sums = (bm::RowSum*)((uint8_t*)workspace + space.sums);
  a.rest = (double*)((uint8_t*)workspace + space.rest);
  a.draws = (bm::Draw*)((uint8_t*)workspace + space.draws);
  hipStream_t s = bm::stream_of(stream);
  hipError_t e;
  switch (op->type) {
    case BM_HIP_F32: e = bm::launch_verify<float>(a, s); break;
    case BM_HIP_BF16: e = bm::launch_verify<__bf16>(a, s); break;
    default: e = bm::launch_verify<_Float16>(a, s); break;
  }
  BM_HIP_CHECK_RET(e, -1);
  return 0;
}
