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
// times, the repeats out of L2.
#include "bm_seq.h"

namespace bm {

constexpr int kConvRows = 32;  // rows per unit

template <int W, int V>
struct Taps {
  float w[W][V], b[V];
  bool silu;
  __device__ __forceinline__ Taps(const float* wp, const float* bp, int channels, int c, bool act)
      : silu(act) {
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) w[k][i] = wp[(size_t)k * channels + c + i];
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = bp ? bp[c + i] : 0.0f;
  }
  // win: the W - 1 rows before x; moves x into it
  __device__ __forceinline__ void push(float (&win)[W - 1][V], const float (&x)[V],
                                       float (&y)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a = b[i];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) a = __builtin_fmaf(win[k][i], w[k][i], a);
      a = __builtin_fmaf(x[i], w[W - 1][i], a);
      y[i] = silu ? silu_f32(a) : a;
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) win[k][i] = win[k + 1][i];
      win[W - 2][i] = x[i];
    }
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
};

template <typename T, int W, int V>
__global__ __launch_bounds__(256) void k_conv(ConvArgs a) {
  const int slots = first_slots(a.q);
  const Unit u = find_unit(a.q, blockIdx.x, kConvRows);
  if (u.b < 0) return;
  const int t0 = u.s + u.k * kConvRows, t1 = min(u.e, t0 + kConvRows);
  if (u.k > 0 && t0 >= t1) return;
  const int slot = find_slot(a.q, u.b, slots);
  if (slot == kNoSlot) return;
  const int c = (blockIdx.y * 256 + threadIdx.x) * V;
  if (c >= a.channels) return;
  const T* x = (const T*)a.x + c;
  T* y = (T*)a.y + c;
  float win[W - 1][V];
  if (u.k > 0) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      load_f32<T, V>(win[k], x + (int64_t)(t0 - (W - 1) + k) * a.xs);
  } else {
    // the sequence's first unit also replaces the state: the same thread has
    // read the old rows before it writes the new ones
    float* st = slot >= 0 ? a.state + (int64_t)slot * a.ss + c : nullptr;
    const bool keep = slot >= 0 && !(a.q.fresh && a.q.fresh[u.b]);
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) win[k][i] = keep ? st[(size_t)k * a.channels + i] : 0.0f;
    if (st) {
      const int n = u.e - u.s;
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        const int pos = n - (W - 1) + k;  // of the new row; negative: an old one
        float r[V];
        if (pos >= 0) {
          load_f32<T, V>(r, x + (int64_t)(u.s + pos) * a.xs);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            r[i] = 0.0f;
#pragma unroll
            for (int o = 0; o < W - 1; ++o) r[i] = o == W - 1 + pos ? win[o][i] : r[i];
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) st[(size_t)k * a.channels + i] = r[i];
      }
    }
  }
  const Taps<W, V> taps(a.w, a.bias, a.channels, c, a.silu);
  int t = t0;
  for (; t + 8 <= t1; t += 8) {
    float r[8][V], o[V];
#pragma unroll
    for (int j = 0; j < 8; ++j) load_f32<T, V>(r[j], x + (int64_t)(t + j) * a.xs);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      taps.push(win, r[j], o);
      store_f32<T, V>(y + (int64_t)(t + j) * a.ys, o);
    }
  }
  for (; t < t1; ++t) {
    float r[V], o[V];
    load_f32<T, V>(r, x + (int64_t)t * a.xs);
    taps.push(win, r, o);
    store_f32<T, V>(y + (int64_t)t * a.ys, o);
  }
}

// One token of each sequence: bound by its state rows, read and written; at
// few sequences by one launch and the round trips slot -> rows.
template <typename T, int W, int V>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs a) {
  const int b = blockIdx.x;
  const int c = (blockIdx.y * 256 + threadIdx.x) * V;
  const int slot = find_slot(a.q, b, first_slots(a.q));
  if (slot == kNoSlot || c >= a.channels) return;
  const Taps<W, V> taps(a.w, a.bias, a.channels, c, a.silu);
  float r[V], o[V], win[W - 1][V];
  load_f32<T, V>(r, (const T*)a.x + (int64_t)b * a.xs + c);
  float* st = slot >= 0 ? a.state + (int64_t)slot * a.ss + c : nullptr;
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) win[k][i] = st ? st[(size_t)k * a.channels + i] : 0.0f;
  taps.push(win, r, o);
  if (st)
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) st[(size_t)k * a.channels + i] = win[k][i];
  store_f32<T, V>((T*)a.y + (int64_t)b * a.ys + c, o);
}

template <typename T, int W, int V>
static hipError_t launch_conv(const ConvArgs& a, bool step, hipStream_t s) {
  const unsigned gy = (unsigned)((a.channels + 256 * V - 1) / (256 * V));
  if (step)
    hipLaunchKernelGGL((k_conv_step<T, W, V>), dim3(a.q.n_seqs, gy), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_conv<T, W, V>),
                       dim3((unsigned)unit_count(a.q.n_seqs, a.q.n_tokens, kConvRows), gy),
                       dim3(256), 0, s, a);
  return hipGetLastError();
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
      !bm::check_rows(name, "x", op->x, op->x_stride, op->channels, elem) ||
      !bm::check_rows(name, "y", op->y, op->y_stride, op->channels, elem) ||
      !bm::check_apart(name, "x", op->x, op->x_stride, op->channels, op->y, op->y_stride,
                       op->channels, rows, elem, step))
    return -2;
  if (op->n_seqs == 0) return 0;
  if (bm::unit_count(op->n_seqs, step ? 0 : op->n_tokens, bm::kConvRows) > 0x7fffffff) {
    bm_set_error("%s: too many rows for one call", name);
    return -2;
  }
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
