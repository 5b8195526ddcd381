// The short causal convolution of the block (src/kernel.c:50-58) for many
// sequences: prompts of ragged lengths and single tokens, with the last
// width - 1 inputs of each sequence in its state slot.
//
//   y[t][c] = act(bias[c] + sum_k w[k][c] x[t - (W - 1) + k][c])
//
// 2 W + 4 operations per value read and written once: bound by memory.  A
// thread owns V neighbouring channels (16 bytes where the rows allow it) and
// walks a unit of kConvRows rows with the window in registers; the rows of a
// block's lanes are read whole, and each row is read 1 + (W - 1) / kConvRows
// times, the repeats out of L2.  4096 rows of 4096 channels, fp32: 32 us, 135
// MB at 4.2 TB/s; 1999 rows of 2307 channels, bf16, one channel per lane: 10
// us.  Stores of y past the caches take 26 us for the first, but the call and
// the scan that reads y then take 108 us together and not 105.
#include "bm_seq.h"

namespace bm {

constexpr int kConvRows = 16;  // rows per unit
constexpr int kConvBatch = 8;  // rows loaded together
constexpr int kConvSeqs = 4;   // single tokens per thread where there are many

template <int W, int V>
struct Taps {
  float w[W][V], b[V];
  bool silu;
  __device__ __forceinline__ Taps(const float* wp, const float* bp, int channels, int c, bool act)
      : silu(act) {
    const auto rw = rows_at(wp, (uint32_t)(W * channels * 4));
    const auto rb = rows_at(bp, bp ? (uint32_t)(channels * 4) : 0);  // none: zeros
#pragma unroll
    for (int k = 0; k < W; ++k) load_floats<V>(w[k], rw, (uint32_t)((k * channels + c) * 4));
    load_floats<V>(b, rb, (uint32_t)(c * 4));
  }
  // win: the W - 1 rows before x; moves x into it
  __device__ __forceinline__ void push(float (&win)[W - 1][V], const float (&x)[V],
                                       float (&y)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a = b[i];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) a = __builtin_fmaf(win[k][i], w[k][i], a);
      y[i] = __builtin_fmaf(x[i], w[W - 1][i], a);
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) win[k][i] = win[k + 1][i];
      win[W - 2][i] = x[i];
    }
    if (silu)
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = silu_f32(y[i]);
  }
};

struct ConvArgs {
  SeqView q;
  int channels;
  bool silu;
  const void* x;
  int64_t xs;
  const float *w, *bias;
  float* state;
  int64_t ss;
  void* y;
  int64_t ys;
  // the slot's rows; without one nothing is read (zeros) or written
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t slot_rows(int slot, int rows) const {
    return rows_at(state + (slot >= 0 ? (int64_t)slot * ss : 0),
                   slot >= 0 ? (uint32_t)(rows * channels * 4) : 0);
  }
};

template <typename T, int V>
__device__ __forceinline__ void unpack(float (&o)[V], const Pack<T, V>& p) {
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = (float)p.v[i];
}

template <typename T, int W, int V>
__global__ __launch_bounds__(256) void k_conv(ConvArgs a) {
  const int c = (blockIdx.y * 256 + threadIdx.x) * V;
  const int slots = first_slots(a.q);
  const Unit u = find_unit(a.q, (int)wide_block(), kConvRows);
  if (u.b < 0) return;
  if (u.k > (u.e > u.s ? (u.e - u.s - 1) / kConvRows : 0)) return;  // past its rows
  const int t0 = u.s + u.k * kConvRows, t1 = u.e - t0 < kConvRows ? u.e : t0 + kConvRows;
  const int slot = find_slot(a.q, u.b, slots);
  if (slot == kNoSlot || c >= a.channels) return;
  const uint32_t col = (uint32_t)(c * sizeof(T)), xs = (uint32_t)(a.xs * sizeof(T)),
                 ys = (uint32_t)(a.ys * sizeof(T)), row = (uint32_t)(a.channels * 4);
  const int rows = t1 - t0;
  const auto bx = rows_of<T>(a.x, t0, a.xs, rows);
  const auto by = rows_of<T>(a.y, t0, a.ys, rows);
  Pack<T, V> next[kConvBatch];
#pragma unroll
  for (int j = 0; j < kConvBatch; ++j) next[j] = load_row<T, V>(bx, col + j * xs);

  float win[W - 1][V], old[W - 1][V];
  Pack<T, V> end[W - 1];
  const auto st = a.slot_rows(slot, W - 1);
  if (u.k > 0) {
    const auto bw = rows_of<T>(a.x, t0 - (W - 1), a.xs, W - 1);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) unpack(win[k], load_row<T, V>(bw, col + k * xs));
  } else {
    // the sequence's first unit also replaces the state: the same thread has
    // read the old rows before it writes the new ones
    const bool keep = slot >= 0 && !(a.q.fresh && a.q.fresh[u.b]);
    const int n = u.e - u.s;
    const auto be = rows_of<T>(a.x, u.e - min(n, W - 1), a.xs, min(n, W - 1));
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      load_floats<V>(old[k], st, keep ? (uint32_t)(c * 4) + k * row : kNoColumn);
      const int back = n - (W - 1) < 0 ? n - (W - 1) : 0;  // rows that the old state keeps
      end[k] = load_row<T, V>(be, k + back >= 0 ? col + (k + back) * xs : kNoColumn);
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) win[k][i] = old[k][i];
  }
  const Taps<W, V> taps(a.w, a.bias, a.channels, c, a.silu);
  for (int t = 0; t < rows; t += kConvBatch) {
    Pack<T, V> now[kConvBatch];
#pragma unroll
    for (int j = 0; j < kConvBatch; ++j) now[j] = next[j];
    if (t + kConvBatch < rows)
#pragma unroll
      for (int j = 0; j < kConvBatch; ++j)
        next[j] = load_row<T, V>(bx, col + (t + kConvBatch + j) * xs);
#pragma unroll
    for (int j = 0; j < kConvBatch; ++j) {
      float x[V], o[V];
      unpack(x, now[j]);
      taps.push(win, x, o);
      store_row<T, V>(by, col + (t + j) * ys, o);
    }
  }
  if (u.k == 0) {
    const int n = u.e - u.s;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      float r[V];
      unpack(r, end[k]);
      // with fewer than W - 1 rows the first of the new state are old ones
#pragma unroll
      for (int o = k; o < W - 1; ++o)
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = n + k == o ? old[o][i] : r[i];
      store_floats<V>(st, (uint32_t)(c * 4) + k * row, r);
    }
  }
}

// One token of each sequence: bound by its state rows, read and written; at
// few sequences by one launch and the round trips slot -> rows.  A thread
// takes SEQS sequences, so that its taps are loaded once for them.  4096
// channels fp32, one sequence: 2.4 us; 4352 channels bf16, 512 sequences: 14.7
// us, 62 MB at 4.3 TB/s.
template <typename T, int W, int V, int SEQS>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs a) {
  const int c = (blockIdx.y * 256 + threadIdx.x) * V;
  const int first = first_slots(a.q);
  const uint32_t row = (uint32_t)(a.channels * 4), col = c < a.channels ? (uint32_t)(c * 4) : kNoColumn;
  const uint32_t at = c < a.channels ? (uint32_t)(c * sizeof(T)) : kNoColumn;
  int slot[SEQS];
  float win[SEQS][W - 1][V];
  Pack<T, V> x[SEQS];
#pragma unroll
  for (int q = 0; q < SEQS; ++q) {
    const int b = blockIdx.x * SEQS + q;
    slot[q] = b < a.q.n_seqs ? find_slot(a.q, b, first) : kNoSlot;
    const auto st = a.slot_rows(slot[q], W - 1);
    x[q] = load_row<T, V>(rows_of<T>(a.x, b, a.xs, slot[q] != kNoSlot), at);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load_floats<V>(win[q][k], st, col + k * row);
  }
  if (c >= a.channels) return;
  const Taps<W, V> taps(a.w, a.bias, a.channels, c, a.silu);
#pragma unroll
  for (int q = 0; q < SEQS; ++q) {
    const int b = blockIdx.x * SEQS + q;
    float r[V], o[V];
    unpack(r, x[q]);
    taps.push(win[q], r, o);
    const auto st = a.slot_rows(slot[q], W - 1);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store_floats<V>(st, col + k * row, win[q][k]);
    store_row<T, V>(rows_of<T>(a.y, b, a.ys, slot[q] != kNoSlot), at, o);
  }
}

template <typename T, int W, int V>
static hipError_t launch_conv(const ConvArgs& a, bool step, hipStream_t s) {
  const unsigned gy = (unsigned)((a.channels + 256 * V - 1) / (256 * V));
  if (step && (int64_t)a.q.n_seqs * gy >= 1024)  // one thread's work for four still fills the chip
    return launch(k_conv_step<T, W, V, kConvSeqs>,
                  dim3((a.q.n_seqs + kConvSeqs - 1) / kConvSeqs, gy), dim3(256), 0, s, a);
  if (step) return launch(k_conv_step<T, W, V, 1>, dim3(a.q.n_seqs, gy), dim3(256), 0, s, a);
  return launch(k_conv<T, W, V>, wide_grid(unit_count(a.q.n_seqs, a.q.n_tokens, kConvRows), gy),
                dim3(256), 0, s, a);
}

template <typename T, int V>
static hipError_t launch_conv_w(const ConvArgs& a, int width, bool step, hipStream_t s) {
  switch (width) {
    case 2: return launch_conv<T, 2, V>(a, step, s);
    case 3: return launch_conv<T, 3, V>(a, step, s);
    default: return launch_conv<T, 4, V>(a, step, s);
  }
}

template <typename T>
static hipError_t launch_conv_t(const ConvArgs& a, int width, bool step, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool wide = a.channels % V == 0 && a.xs % V == 0 && a.ys % V == 0 &&
                    ((uintptr_t)a.x | (uintptr_t)a.y) % 16 == 0;
  return wide ? launch_conv_w<T, V>(a, width, step, s) : launch_conv_w<T, 1>(a, width, step, s);
}

}  // namespace bm

static int conv_call(const bm_hip_conv_t* op, void* stream, bool step) {
  const char* name = step ? "conv_step" : "conv";
  if (!op) {
    bm_set_error("%s: no descriptor", name);
    return -2;
  }
  if (op->type < BM_HIP_F32 || op->type > BM_HIP_F16 || op->channels < 1 ||
      op->channels > (1 << 22) || op->width < 2 || op->width > 4 || !op->w ||
      (uintptr_t)op->w % 4 || (uintptr_t)op->bias % 4) {
    bm_set_error("%s: invalid arguments (type=%d channels=%d width=%d)", name, op->type,
                 op->channels, op->width);
    return -2;
  }
  const size_t elem = bm::type_bytes(op->type);
  const int64_t rows = step ? op->n_seqs : op->n_tokens;
  if (!bm::check_seqs(name, op->n_seqs, op->n_tokens, op->seq_start, op->slots, op->state,
                      op->state_stride, op->n_slots, (int64_t)(op->width - 1) * op->channels,
                      step) ||
      !bm::check_rows(name, "x", op->x, op->x_stride, op->channels, rows, elem) ||
      !bm::check_rows(name, "y", op->y, op->y_stride, op->channels, rows, elem) ||
      !bm::check_apart(name, "x", op->x, op->x_stride, op->channels, op->y, op->y_stride,
                       op->channels, rows, elem, step))
    return -2;
  if (op->n_seqs == 0) return 0;
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  bm::ConvArgs a;
  a.q = bm::SeqView{op->seq_start, op->state ? op->slots : nullptr, op->fresh, op->n_seqs,
                    op->n_tokens, op->state ? op->n_slots : 0};
  a.channels = op->channels;
  a.silu = op->silu != 0;
  a.x = op->x;
  a.xs = op->x_stride;
  a.w = op->w;
  a.bias = op->bias;
  a.state = op->state;
  a.ss = op->state_stride;
  a.y = op->y;
  a.ys = op->y_stride;
  hipStream_t s = bm::stream_of(stream);
  hipError_t e;
  switch (op->type) {
    case BM_HIP_F32: e = bm::launch_conv_t<float>(a, op->width, step, s); break;
    case BM_HIP_BF16: e = bm::launch_conv_t<__bf16>(a, op->width, step, s); break;
    default: e = bm::launch_conv_t<_Float16>(a, op->width, step, s); break;
  }
  BM_HIP_CHECK_RET(e, -1);
  return 0;
}

extern "C" int bm_hip_conv_dev(const bm_hip_conv_t* op, void* stream) {
  return conv_call(op, stream, false);
}

extern "C" int bm_hip_conv_step_dev(const bm_hip_conv_t* op, void* stream) {
  return conv_call(op, stream, true);
}
