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
// error of a running sum moves draws by that much: exponentials and sums are
// in fp64 (2^-47 of each), in an order that depends on the sizes alone.
#include <math.h>

#include "bm_dev.h"
#include "bm_seq.h"

namespace bm {

constexpr int kVerifyThreads = 256, kPerThread = 16;
constexpr int kSegment = kVerifyThreads * kPerThread;  // values of a row per block
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
  int row, last;       // row -1: none
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

// 2^t for t at most 0 (NaN: 0): the series of e^{f ln 2}, |f| <= 1/2, up to
// f^11, which leaves (ln 2 / 2)^12 / 12! < 2^-47
__device__ __forceinline__ double exp2_f64(double t) {
  constexpr double c1 = 0.693147180559945309417, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3,
                   c4 = c3 * c1 / 4, c5 = c4 * c1 / 5, c6 = c5 * c1 / 6, c7 = c6 * c1 / 7,
                   c8 = c7 * c1 / 8, c9 = c8 * c1 / 9, c10 = c9 * c1 / 10, c11 = c10 * c1 / 11;
  t = __builtin_fmax(t, -1100.0);
  const double n = __builtin_rint(t), f = t - n;
  double r = c11;
  r = __builtin_fma(r, f, c10);
  r = __builtin_fma(r, f, c9);
  r = __builtin_fma(r, f, c8);
  r = __builtin_fma(r, f, c7);
  r = __builtin_fma(r, f, c6);
  r = __builtin_fma(r, f, c5);
  r = __builtin_fma(r, f, c4);
  r = __builtin_fma(r, f, c3);
  r = __builtin_fma(r, f, c2);
  r = __builtin_fma(r, f, c1);
  r = __builtin_fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)n);
}
// a value's share of a row whose largest is m, before the sum divides it
__device__ __forceinline__ double share_of(int kind, float v, float m, double k) {
  if (kind == kWeights) return v > 0.0f && v < __builtin_inff() ? (double)v : 0.0;
  const double d = v == m ? 0.0 : (double)v - (double)m;  // infinite ones too
  return m == -__builtin_inff() ? 0.0 : exp2_f64(d * k);
}

// Values i .. i + 15 of a row on any alignment of T; `none` past its end.  Words
// of four bytes are read, so a row of two-byte values that starts or ends within
// a word is read with its neighbour in that word.
struct alignas(4) Words4 {
  uint32_t w[4];
};
template <typename T>
__device__ __forceinline__ void load16(float (&o)[kPerThread], const T* row, int i, int vocab,
                                       float none) {
  static_assert(kPerThread == 16, "");
  if (i + 16 > vocab) {
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = i + j < vocab ? (float)row[i + j] : none;
    return;
  }
  if constexpr (sizeof(T) == 4) {
    Words4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *(const Words4*)(row + i + 4 * j);
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = __uint_as_float(v[j >> 2].w[j & 3]);
  } else {
    const uintptr_t at = (uintptr_t)(row + i);
    const int odd = (int)(at >> 1 & 1);  // the same for the whole row, i being even
    const uint32_t* w = (const uint32_t*)(at - 2 * odd);
    const Words4 a = *(const Words4*)w, b = *(const Words4*)(w + 4);
    uint32_t v[9];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a.w[j];
      v[4 + j] = b.w[j];
    }
    v[8] = odd ? w[8] : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = odd ? __builtin_amdgcn_alignbit(v[j + 1], v[j], 16) : v[j];
      o[2 * j] = (float)__builtin_bit_cast(T, (uint16_t)x);
      o[2 * j + 1] = (float)__builtin_bit_cast(T, (uint16_t)(x >> 16));
    }
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = min(v, __shfl_xor(v, m));
  return v;
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
    o.s += kind == kWeights ? v[i].s
                            : v[i].s * (v[i].m == o.m ? 1.0 : exp2_f64(((double)v[i].m - o.m) * k));
  return o;
}

// ---------------------------------------------------------------------------
// One segment of one row of the target (z 0) or the draft (z 1).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void k_verify_rows(VerifyArgs a) {
  __shared__ RowSum part[kVerifyThreads / 64];
  const bool draft = blockIdx.y != 0;
  const int64_t block = wide_block();
  const int64_t row = block / a.segments;
  if (row >= a.q.n_tokens) return;
  int end;
  if (find_row(a.q, (int)row, &end) < 0 || (draft && row == end - 1)) return;
  const int seg = (int)(block - row * a.segments);
  const int kind = draft ? a.q_kind : a.p_kind;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i0 = seg * kSegment + tid * kPerThread;
  float v[kPerThread];
  load16<T>(v, (const T*)(draft ? a.d : a.p) + row * (draft ? a.ds : a.ps), i0, a.vocab,
            kind == kWeights ? 0.0f : -__builtin_inff());
  RowSum o{0.0, -__builtin_inff(), INT32_MAX};
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) o.m = fmaxf(o.m, v[j]);
  o.m = wave_max_f32(o.m);
  if (kind == kLargest) {
#pragma unroll
    for (int j = kPerThread - 1; j >= 0; --j)
      if (v[j] == o.m) o.at = i0 + j;
    o.at = wave_min_i32(o.at);
  } else {
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) o.s += share_of(kind, v[j], o.m, a.k);
    o.s = wave_sum_f64(o.s);
  }
  if (lane == 0) part[wave] = o;
  __syncthreads();
  if (tid == 0)
    a.sums[(row + (draft ? a.q.n_tokens : 0)) * a.segments + seg] =
        join_sums(kind == kLargest ? (int)kWeights : kind, part, a.k);
}

// a whole row, in all lanes
__device__ __forceinline__ RowSum row_sum(const VerifyArgs& a, int kind, int64_t row, bool draft) {
  const int lane = threadIdx.x & 63;
  RowSum o{0.0, -__builtin_inff(), INT32_MAX};
  if (lane < a.segments) o = a.sums[(row + (draft ? a.q.n_tokens : 0)) * a.segments + lane];
  const float m = wave_max_f32(o.m);
  if (kind == kLargest) {
    o.at = wave_min_i32(o.m == m && m > -__builtin_inff() ? o.at : INT32_MAX);
    if (o.at == INT32_MAX) o.at = -1;
    o.s = o.at < 0 ? 0.0 : 1.0;
  } else {
    if (kind == kLogits) o.s *= o.m == m ? 1.0 : exp2_f64(((double)o.m - m) * a.k);
    o.s = wave_sum_f64(lane < a.segments ? o.s : 0.0);
  }
  o.m = m;
  return o;
}
// the probability of a token, given the row's sum
template <typename T>
__device__ __forceinline__ double prob_of(const VerifyArgs& a, int kind, const T* row, RowSum r,
                                          int token) {
  if (token < 0 || token >= a.vocab) return 0.0;
  if (kind == kToken) return 1.0;
  if (kind == kLargest) return token == r.at ? 1.0 : 0.0;
  return r.s > 0.0 ? share_of(kind, (float)row[token], r.m, a.k) / r.s : 0.0;
}

// a token's weight in the draw
template <typename T>
__device__ __forceinline__ void weights16(double (&w)[kPerThread], const VerifyArgs& a,
                                          const Draw& d, int i0) {
  float v[kPerThread];
  load16<T>(v, (const T*)a.p + (int64_t)d.row * a.ps, i0, a.vocab,
            d.p_kind == kWeights ? 0.0f : -__builtin_inff());
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) w[j] = share_of(d.p_kind, v[j], d.pm, a.k) * d.p_inv;
  if (d.q_kind < 0) return;
  if (d.q_kind == kToken) {
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) w[j] = i0 + j == d.q_at ? 0.0 : w[j];
    return;
  }
  load16<T>(v, (const T*)a.d + (int64_t)d.row * a.ds, i0, a.vocab,
            d.q_kind == kWeights ? 0.0f : -__builtin_inff());
#pragma unroll
  for (int j = 0; j < kPerThread; ++j)
    w[j] = __builtin_fmax(w[j] - share_of(d.q_kind, v[j], d.qm, a.k) * d.q_inv, 0.0);
}

// ---------------------------------------------------------------------------
// The rows of a sequence in turn, a wave each, until one is refused; then a
// segment of the draw's weights.  Every block of a sequence decides for itself
// (a launch of its own would cost more than the few rows of a draft); the
// first writes what was decided, and goes through all rows for their ratios.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void k_verify_stop(VerifyArgs a, int blocks) {
  constexpr int kWavesV = kVerifyThreads / 64;
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
  if (tid == 0) first = INT32_MAX;
  __syncthreads();
  for (int r0 = s; r0 < e; r0 += kWavesV) {
    const int row = r0 + wave;
    const bool have = row < e, last = row == e - 1;
    RowSum p{0.0, 0.0f, -1}, q{1.0, 0.0f, -1};
    int token = -1;
    if (have) {
      p = row_sum(a, a.p_kind, row, false);
      bool stands = false;
      if (!last) {
        token = a.tokens[row];
        const double pd = prob_of<T>(a, a.p_kind, (const T*)a.p + row * a.ps, p, token);
        if (a.p_kind == kLargest) {
          stands = pd > 0.0;
          if (writer && a.ratio && lane == 0) a.ratio[row] = (float)pd;
        } else {
          if (a.q_kind != kToken) q = row_sum(a, a.q_kind, row, true);
          const double qd = prob_of<T>(a, a.q_kind, (const T*)a.d + row * a.ds, q, token);
          stands = (double)a.u[row] * qd < pd;
          if (writer && a.ratio && lane == 0)
            a.ratio[row] = pd > 0.0 ? (float)(pd < qd ? pd / qd : 1.0) : 0.0f;
        }
      }
      if (!stands && lane == 0) atomicMin(&first, row);
    }
    __syncthreads();
    const int stop = first;  // read by all before any wave goes on to write it
    if (have && row == stop && lane == 0) {
      Draw d;
      d.row = p.s > 0.0 ? row : -1;
      d.last = e - 1;
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
    double w[kPerThread];
    weights16<T>(w, a, d, seg * kSegment + tid * kPerThread);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) sum += w[j];
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

// running sums over the wave
__device__ __forceinline__ double wave_scan_f64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  return v;
}

// ---------------------------------------------------------------------------
// The draw of one sequence: the segment in which the running sum passes u
// times the whole, then the token in it.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void k_verify_draw(VerifyArgs a) {
  constexpr int kWavesV = kVerifyThreads / 64;
  __shared__ double part[kWavesV];
  __shared__ int at, most;
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
      if (d.p_kind == kLogits) mine *= o.m == d.pm ? 1.0 : exp2_f64(((double)o.m - d.pm) * a.k);
    }
  }
  const double run = wave_scan_f64(mine);
  const double want = (double)a.u[d.last] * __shfl(run, 63);
  const uint64_t in = __ballot(mine > 0.0 && run > want);
  const uint64_t any = __ballot(mine > 0.0);
  const int seg = in ? __ffsll((unsigned long long)in) - 1
                     : (any ? 63 - __clzll((long long)any) : 0);
  const double before = seg > 0 ? __shfl(run, seg - 1) : 0.0;
  if (tid == 0) {
    at = INT32_MAX;
    most = -1;
  }
  double w[kPerThread], sum = 0.0;
  const int i0 = seg * kSegment + tid * kPerThread;
  weights16<T>(w, a, d, i0);
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) sum += w[j];
  const double upto = wave_scan_f64(sum);
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  double c = before;
  for (int i = 0; i < wave; ++i) c += part[i];
  c += upto - sum;
  int got = INT32_MAX, last = -1;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    c += w[j];
    if (w[j] > 0.0) {
      last = i0 + j;
      if (got == INT32_MAX && c > want) got = i0 + j;
    }
  }
  if (got != INT32_MAX) atomicMin(&at, got);
  if (last >= 0) atomicMax(&most, last);
  __syncthreads();
  if (tid == 0) a.next[b] = at != INT32_MAX ? at : most;
}

template <typename T>
static hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const bool greedy = a.p_kind == kLargest, rows_of_draft = a.q_kind != kToken && !greedy;
  if (a.q.n_tokens > 0) {
    const hipError_t e = launch(k_verify_rows<T>, wide_grid((int64_t)a.q.n_tokens * a.segments,
                                                            rows_of_draft ? 2 : 1),
                                dim3(kVerifyThreads), 0, s, a);
    if (e != hipSuccess) return e;
  }
  const int blocks = greedy ? 1 : a.segments;
  const hipError_t e = launch(k_verify_stop<T>, wide_grid((int64_t)a.q.n_seqs * blocks, 1),
                              dim3(kVerifyThreads), 0, s, a, blocks);
  if (e != hipSuccess || greedy) return e;
  return launch(k_verify_draw<T>, dim3(a.q.n_seqs), dim3(kVerifyThreads), 0, s, a);
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
