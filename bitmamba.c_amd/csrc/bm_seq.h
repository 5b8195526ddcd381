// What the batched recurrence kernels share: element types, the ragged rows
// of a call, the sequences' state slots, and the fp32 functions of the block.
#pragma once

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
__device__ __forceinline__ float silu_f32(float x) {
  // x rcp(1 + exp(-x)); -inf * 0 is 0 here, the limit
  const float r = x * __builtin_amdgcn_rcpf(1.0f + exp_f32(-x));
  return x < -126.0f ? -0.0f : r;
}
// log(1 + exp(x)) = max(x, 0) + log1p(exp(-|x|))
__device__ __forceinline__ float softplus_f32(float x) {
  return fmaxf(x, 0.0f) + log1pf(expf(-__builtin_fabsf(x)));
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
struct Unit {
  int b;     // sequence, -1: none
  int k;     // unit of it
  int s, e;  // its rows
};
// The unit's sequence by a search in steps of 64 (one load and ballot per
// level).  All lanes of the wave must call it with the same u.
__device__ __forceinline__ Unit find_unit(const SeqView& q, int u, int len) {
  if (!q.seq_start) return Unit{0, u, 0, q.n_tokens};
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.n_seqs;
  do {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const bool below = i < hi && seq_row(q, i) / len + i <= u;
    const int c = __popcll(__ballot(below));
    if (c == 0) return Unit{-1, 0, 0, 0};  // rows before the first sequence
    lo += (c - 1) * step;
    hi = min(hi, lo + step);
  } while (hi - lo > 1);
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int s = __builtin_amdgcn_readfirstlane(seq_row(q, lo));
  const int e = __builtin_amdgcn_readfirstlane(seq_row(q, lo + 1));
  return Unit{lo, u - (s / len + lo), s, e < s ? s : e};
}

constexpr int kNoSlot = -1, kNoPool = -2;
// The slot of sequence b; kNoSlot: padding.  All lanes of the wave must call
// it with the same b.
__device__ __forceinline__ int find_slot(const SeqView& q, int b) {
  if (q.n_slots == 0) return kNoPool;
  if (!q.slots) return b;  // checked by the host: n_seqs <= n_slots
  const int lane = threadIdx.x & 63;
  const int slot = __builtin_amdgcn_readfirstlane(q.slots[b]);
  if (slot < 0 || slot >= q.n_slots) return kNoSlot;
  bool taken = false;
  for (int j = lane; j < b; j += 64) taken |= q.slots[j] == slot;
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

// Host checks shared by the descriptors; each sets the error and returns false.
inline size_t type_bytes(int type) { return type == BM_HIP_F32 ? 4 : 2; }
bool check_rows(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                size_t elem);
bool check_apart(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                 const void* y, int64_t y_stride, int64_t y_width, int64_t rows, size_t elem,
                 bool same_ok);
bool check_seqs(const char* op, int n_seqs, int n_tokens, const int32_t* seq_start,
                const int32_t* slots, const float* state, int64_t state_stride, int n_slots,
                int64_t slot_floats, bool step);
hipStream_t stream_of(void* stream);  // nullptr: the library's

}  // namespace bm
