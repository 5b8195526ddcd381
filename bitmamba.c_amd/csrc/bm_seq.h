// What the batched recurrence kernels share: element types, the ragged rows
// of a call, the sequences' state slots, and the fp32 functions of the block.
#pragma once

#include <tuple>

#include "bm_common.h"
#include "bm_hip.h"

namespace bm {

// N elements of T at T's own alignment times N
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(float (&o)[N], const T* p) {
  const Pack<T, N> k = *(const Pack<T, N>*)p;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = (float)k.v[i];
}

// the one rounding of a result (to nearest even)
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&o)[N]) {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = (T)o[i];
  *(Pack<T, N>*)p = k;
}

// Up to 32 rows of a tensor as a buffer resource: an offset at or past its
// end reads zeros and writes nothing, so neither the last rows nor lanes
// without a column (offset kNoColumn) need a branch around a load, which would
// keep it from being issued with the others.  Row strides are below 2^24
// elements (check_rows), so 32 rows end below kNoColumn, and kNoColumn plus
// an offset within them does not wrap.
constexpr uint32_t kNoColumn = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* p, int64_t row,
                                                          int64_t stride, int rows) {
  return rows_at((const T*)p + row * stride, (uint32_t)rows * (uint32_t)stride * sizeof(T));
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_row(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  constexpr int B = sizeof(T) * N;
  static_assert(B == 2 || B == 4 || B == 8 || B == 16, "one load");
  if constexpr (B == 2) {
    return __builtin_bit_cast(Pack<T, N>, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
  } else if constexpr (B == 4) {
    return __builtin_bit_cast(Pack<T, N>, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
  } else if constexpr (B == 8) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
    return __builtin_bit_cast(Pack<T, N>, v);
  } else {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    return __builtin_bit_cast(Pack<T, N>, v);
  }
}
// A value or four of them as the load leaves them, for loads that are issued
// well ahead: as T they would be packed into pairs at once, which waits.
template <typename T>
__device__ __forceinline__ uint32_t load_raw(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  else return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}
template <typename T>
__device__ __forceinline__ float raw_f32(uint32_t v) {
  if constexpr (sizeof(T) == 2) return (float)__builtin_bit_cast(T, (uint16_t)v);
  else return __uint_as_float(v);
}
template <typename T>
struct Raw4 {
  uint32_t w[sizeof(T)];  // four values
};
template <typename T>
__device__ __forceinline__ Raw4<T> load_raw4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  Raw4<T> o;
  if constexpr (sizeof(T) == 2) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
    o.w[0] = v[0];
    o.w[1] = v[1];
  } else {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.w[i] = v[i];
  }
  return o;
}
template <typename T>
__device__ __forceinline__ float raw4_f32(const Raw4<T>& v, int i) {
  if constexpr (sizeof(T) == 2)
    return (float)__builtin_bit_cast(T, (uint16_t)(v.w[i >> 1] >> (16 * (i & 1))));
  else
    return __uint_as_float(v.w[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_row(__amdgpu_buffer_rsrc_t r, uint32_t off,
                                          const float (&o)[N]) {
  constexpr int B = sizeof(T) * N;
  static_assert(B == 2 || B == 4 || B == 8 || B == 16, "one store");
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = (T)o[i];
  if constexpr (B == 2) {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, k), r, off, 0, 0);
  } else if constexpr (B == 4) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, k), r, off, 0, 0);
  } else if constexpr (B == 8) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, k), r, off, 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, k), r, off, 0, 0);
  }
}

// V neighbouring floats (1, 4 or 8) on a multiple of 4 bytes; STREAM: past the caches, for what is
// read and written once and does not fit them
template <int V, bool STREAM = false>
__device__ __forceinline__ void load_floats(float (&o)[V], __amdgpu_buffer_rsrc_t r, uint32_t off) {
  constexpr int kAux = STREAM ? 2 : 0;  // the nt bit
  if constexpr (V == 1) {
    o[0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, kAux));
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * k, 0, kAux);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[k + i] = __uint_as_float(v[i]);
    }
  }
}
template <int V, bool STREAM = false>
__device__ __forceinline__ void store_floats(__amdgpu_buffer_rsrc_t r, uint32_t off,
                                             const float (&o)[V]) {
  constexpr int kAux = STREAM ? 2 : 0;
  if constexpr (V == 1) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[0]), r, off, 0, kAux);
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(o[k + i]);
      __builtin_amdgcn_raw_buffer_store_b128(v, r, off + 4 * k, 0, kAux);
    }
  }
}

// ---------------------------------------------------------------------------
// fp32 functions on the hardware's base-2 exponential (1 ulp): the argument's
// product with log2(e) is carried in two parts, so that its rounding, which
// would cost |x| / 2 ulps, stays out of the result.
// ---------------------------------------------------------------------------
constexpr float kLog2e = 0x1.715476p+0f, kLog2eLo = 0x1.4ae0cp-26f;
__device__ __forceinline__ float exp_f32(float x) {
  const float hi = x * kLog2e;
  const float lo = __builtin_fmaf(x, kLog2eLo, __builtin_fmaf(x, kLog2e, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  // 2^lo = 1 + lo ln2 for |lo| < 2^-17; lo of an infinite x is NaN
  const float r = e * __builtin_fmaf(lo, 0x1.62e43p-1f, 1.0f);
  return __builtin_fabsf(hi) < 256.0f ? r : e;
}
// exp(p) as hi, the nearest float, and lo, what that leaves, for a state that is
// multiplied by it row after row: the hardware's exponential is 0.12 units of
// 2^-24 too small on average just below 1, and even a rounded one keeps
// 2^-25 / (1 - a) of a steady state's value.  Below |p| = 1/16, where a decay's
// error outlives a few rows, exp(p) - 1 = p + (p^2 / 2 + p^3 / 6 + p^4 / 24), off
// by p^5 / 120 < 2^-26; above it lo is 0.
struct Decay {
  float hi, lo;
};
__device__ __forceinline__ Decay decay_of(float p) {
  const float t = __builtin_fmaf(__builtin_fmaf(p, 1.0f / 24.0f, 1.0f / 6.0f), p, 0.5f);
  const float s = p * p * t, m = p + s;  // |p| > |s| where neither is zero
  const float near1 = 1.0f + m, far = exp_f32(p);
  const bool near = __builtin_fabsf(p) < 0.0625f;
  return Decay{near ? near1 : far, near ? (m - (near1 - 1.0f)) + (s - (m - p)) : 0.0f};
}
// add + s lo, an infinite s left to the product with hi
__device__ __forceinline__ float with_low(float s, float lo, float add) {
  constexpr float kMax = 0x1.fffffep127f;
  return __builtin_fmaf(__builtin_amdgcn_fmed3f(s, -kMax, kMax), lo, add);
}
__device__ __forceinline__ float silu_f32(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + exp_f32(-x));
}
// the same to 2^-20 for |x| up to 8 and to |x| 2^-23 above, for what is rounded
// to bf16
__device__ __forceinline__ float silu_short(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e));
}
// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|) <= 1, by
// log(1 + e) = 2 artanh(s), s = e / (2 + e) <= 1/3: the series up to s^13
// leaves less than s^15 / 15 < 2^-26 of it
__device__ __forceinline__ float softplus_f32(float x) {
  const float e = exp_f32(-__builtin_fabsf(x)), q = 2.0f + e;
  float r = __builtin_amdgcn_rcpf(q);
  r = __builtin_fmaf(r, __builtin_fmaf(-q, r, 1.0f), r);
  const float s = e * r, s2 = s * s;
  float p = 1.0f / 13.0f;
  p = __builtin_fmaf(p, s2, 1.0f / 11.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 9.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 7.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 5.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 3.0f);
  p = __builtin_fmaf(p, s2, 1.0f);
  return __builtin_fmaf(2.0f * s, p, fmaxf(x, 0.0f));
}

// ---------------------------------------------------------------------------
// The rows and slots of a call
// ---------------------------------------------------------------------------
struct SeqView {
  const int32_t* seq_start;
  const int32_t* slots;
  const uint8_t* fresh;
  int n_seqs, n_tokens, n_slots;  // n_slots 0: no pool
};

__device__ __forceinline__ int seq_row(const SeqView& q, int i) {
  const int v = q.seq_start[i];
  return v < 0 ? 0 : (v > q.n_tokens ? q.n_tokens : v);
}

// Rows are handed out in units of `len` rows of one sequence: sequence b has
// the units from row(b) / len + b on.  That leaves it room for ceil(n / len)
// of its n rows and at least one unit, whatever row it starts at, so that no
// prefix sum over the sequences is needed; a unit past its rows is empty.
__host__ __device__ inline int64_t unit_count(int n_seqs, int n_tokens, int len) {
  return (int64_t)n_tokens / len + n_seqs;
}
// A grid of any number of blocks: x and z, since a launch has less than 2^32
// threads along x.  The last row of z may have blocks past the number.
constexpr int64_t kGridX = 1 << 20;
inline dim3 wide_grid(int64_t blocks, unsigned y) {
  return dim3((unsigned)(blocks < kGridX ? blocks : kGridX), y,
              (unsigned)((blocks + kGridX - 1) / kGridX));
}
__device__ __forceinline__ int64_t wide_block() {
  return (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
}
struct Unit {
  int b;     // sequence, -1: none
  int k;     // unit of it
  int s, e;  // its rows
};
// The unit's sequence by a search in steps of 63 (one load and ballot per
// level, the last of which also has the sequence's rows).  All lanes of the
// wave must call it with the same u.
__device__ __forceinline__ Unit find_unit(const SeqView& q, int u, int len) {
  if (!q.seq_start) return Unit{0, u, 0, q.n_tokens};
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.n_seqs;
  for (;;) {
    const int step = (hi - lo + 62) / 63;
    const int i = min(lo + lane * step, hi);
    const int row = seq_row(q, i);
    const int c = __popcll(__ballot(i < hi && row / len + i <= u));
    if (c == 0) return Unit{-1, 0, 0, 0};  // rows before the first sequence
    if (step == 1) {
      const int s = __builtin_amdgcn_readlane(row, c - 1), e = __builtin_amdgcn_readlane(row, c);
      // every counted start has i <= u, so b <= u and the unit's first row,
      // s + k len = s % len + (u - b) len, is not below 0 even where starts descend
      const int b = lo + c - 1;
      return Unit{b, u - (s / len + b), s, e < s ? s : e};
    }
    lo += (c - 1) * step;
    hi = min(hi, lo + step);
  }
}

// The sequence that a row belongs to, -1: none; all lanes with the same row.
// Its rows are s .. e - 1.
__device__ __forceinline__ int find_row(const SeqView& q, int row, int* e) {
  *e = q.n_tokens;
  if (!q.seq_start) return 0;
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.n_seqs;  // entries lo .. hi; the last is no sequence's first
  for (;;) {
    const int step = (hi - lo + 62) / 63;
    const int i = min(lo + lane * step, hi);
    const int r = seq_row(q, i);
    const int c = __popcll(__ballot(i < hi && r <= row));
    if (c == 0) return -1;
    if (step == 1) {
      *e = __builtin_amdgcn_readlane(r, c);
      return row < *e ? lo + c - 1 : -1;
    }
    lo += (c - 1) * step;
    hi = min(hi, lo + step);
  }
}

constexpr int kNoSlot = -1, kNoPool = -2;
// The slots of the first 64 sequences, one per lane: a load that waits for
// nothing, issued before the sequence is known.
__device__ __forceinline__ int first_slots(const SeqView& q) {
  const int lane = threadIdx.x & 63;
  return q.n_slots != 0 && q.slots ? q.slots[min(lane, q.n_seqs - 1)] : 0;
}
// The slot of sequence b; kNoSlot: padding.  All lanes of the wave must call
// it with the same b; first: first_slots().
__device__ __forceinline__ int find_slot(const SeqView& q, int b, int first) {
  if (q.n_slots == 0) return kNoPool;
  if (!q.slots) return b;  // checked by the host: n_seqs <= n_slots
  const int lane = threadIdx.x & 63;
  const int slot = b < 64 ? __builtin_amdgcn_readlane(first, b)
                          : __builtin_amdgcn_readfirstlane(q.slots[b]);
  if (slot < 0 || slot >= q.n_slots) return kNoSlot;
  bool taken = lane < b && first == slot;
  // Each block looks for itself, eight loads to a round trip: a step of the
  // scan with 64 heads of 64 and one value takes 18 us with a list and 15
  // without at 512 sequences, 180 and 94 at 4096 (272 by one load each).
  constexpr int kAhead = 8;
  for (int j = lane + 64; j < b; j += 64 * kAhead) {
    int v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = q.slots[min(j + 64 * k, b)];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) taken |= j + 64 * k < b && v[k] == slot;
  }
  return __ballot(taken) ? kNoSlot : slot;
}

// Device 0, the library's, current for a call made while another one is
class OnDevice {
 public:
  OnDevice() {
    if (hipGetDevice(&was_) == hipSuccess && was_ != 0) (void)hipSetDevice(0);
    else was_ = 0;
  }
  ~OnDevice() {
    if (was_ != 0) (void)hipSetDevice(was_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int was_ = 0;
};

// A launch by its own status: an error that an earlier call of the caller's
// left in this thread is not this one's.  The arguments are converted to the
// kernel's parameters.
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s,
                         const A&... args) {
  std::tuple<P...> v(static_cast<P>(args)...);
  void* p[sizeof...(P)];
  std::apply([&](auto&... e) { size_t i = 0; ((p[i++] = (void*)&e), ...); }, v);
  return hipLaunchKernel((const void*)kernel, grid, block, p, lds, s);
}

// Host checks shared by the descriptors; each sets the error and returns false.
inline size_t type_bytes(int type) { return type == BM_HIP_F32 ? 4 : 2; }
bool check_rows(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                int64_t rows, size_t elem);
bool check_apart(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                 const void* y, int64_t y_stride, int64_t y_width, int64_t rows, size_t elem,
                 bool same_ok);
bool check_seqs(const char* op, int n_seqs, int n_tokens, const int32_t* seq_start,
                const int32_t* slots, const float* state, int64_t state_stride, int n_slots,
                int64_t slot_floats, bool step);
hipStream_t stream_of(void* stream);  // nullptr: the library's

}  // namespace bm
