// Moving the slots of state pools: copying, forking, reordering, clearing and
// compacting.  Nothing is computed, so everything is bound by the bytes read
// and written.
#include "bm_seq.h"

namespace bm {

constexpr int kMaxPairs = 1024, kMaxPools = 8, kMaxCompact = 65536;

struct PoolView {
  uint8_t* base;
  int64_t slot_bytes, slot_stride, layer_stride;
};

__device__ __forceinline__ uint4 zero_of(const uint4*) { return make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ uint32_t zero_of(const uint32_t*) { return 0; }
__device__ __forceinline__ uint8_t zero_of(const uint8_t*) { return 0; }

// ---------------------------------------------------------------------------
// Copy of n pairs at once.  A block owns `cols` neighbouring words of W in
// one layer for all pairs: it reads them of every source into registers, E
// words per thread, waits for them, and only then writes any of them.  So
// each pair reads what stood there before the call, whatever the lists
// say, in one pass and without a second buffer.
//
// Several pairs with one dst: the first that moves anything counts.  The
// block finds it in a hash table of the destinations in LDS (at most half of
// its places taken).
//
// 64 pairs of 24 layers of 64 KB, some with one source: 32 us, 156 MB of
// different bytes at 4.9 TB/s.
// ---------------------------------------------------------------------------
constexpr int kHash = 2 * kMaxPairs;

template <typename W, int E>
__global__ __launch_bounds__(256) void k_slots_copy(PoolView pool, int n_slots,
                                                    const int32_t* __restrict__ src,
                                                    const int32_t* __restrict__ dst, int n,
                                                    int log_cols, int log_hash) {
  __shared__ int key[kHash], first[kHash], from[kMaxPairs], into[kMaxPairs];
  const int tid = threadIdx.x, places = 1 << log_hash;
  for (int i = tid; i < places; i += 256) {
    key[i] = -1;
    first[i] = kMaxPairs;
  }
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const int s = src[i], d = dst[i];
    const bool moves = s >= -1 && s < n_slots && d >= 0 && d < n_slots;
    from[i] = s;
    into[i] = -1;
    if (!moves) continue;
    int at = (int)(((uint32_t)d * 2654435761u) >> (32 - log_hash));
    for (int tries = 0; tries < places; ++tries) {  // at most n places are taken
      const int was = atomicCAS(&key[at], -1, d);
      if (was == -1 || was == d) break;
      at = (at + 1) & (places - 1);
    }
    atomicMin(&first[at], i);
  }
  __syncthreads();
  for (int i = tid; i < places; i += 256)
    if (key[i] >= 0) into[first[i]] = key[i];
  __syncthreads();

  const int64_t words = pool.slot_bytes / (int64_t)sizeof(W);
  const int64_t col0 = wide_block() << log_cols;
  uint8_t* layer = pool.base + (int64_t)blockIdx.y * pool.layer_stride;
  W v[E];
  int to[E];
  const int64_t col = col0 + (tid & ((1 << log_cols) - 1));  // 256 is a multiple of the columns,
  const int first_pair = tid >> log_cols;                     // or one pair has them all
  const bool many = log_cols > 8;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int item = tid + 256 * e;
    const int i = many ? item >> log_cols : first_pair + (e << (8 - log_cols));
    const int64_t at = many ? col0 + (item & ((1 << log_cols) - 1)) : col;
    to[e] = i < n && at < words ? into[i] : -1;
    if (to[e] < 0) continue;
    const int s = from[i];
    v[e] = s < 0 ? zero_of((const W*)nullptr)
                 : ((const W*)(layer + (int64_t)s * pool.slot_stride))[at];
  }
  // every load of the block has returned before its first store
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (to[e] < 0) continue;
    const int64_t at = many ? col0 + ((tid + 256 * e) & ((1 << log_cols) - 1)) : col;
    ((W*)(layer + (int64_t)to[e] * pool.slot_stride))[at] = v[e];
  }
}

template <typename W, int E>
static hipError_t launch_copy_e(const PoolView& p, int n_layers, int n_slots, const int32_t* src,
                                const int32_t* dst, int n, hipStream_t s) {
  // the columns of a block: a power of two, all pairs' words in its registers
  const int64_t words = p.slot_bytes / (int64_t)sizeof(W);
  int lc = 0, lh = 6;
  while ((2 << lc) * n <= 256 * E && ((int64_t)1 << lc) < words) ++lc;
  while ((1 << lh) < 2 * n) ++lh;
  const int64_t blocks = (words + ((int64_t)1 << lc) - 1) >> lc;
  if (blocks > kGridX * 65535) return hipErrorInvalidValue;
  return launch(k_slots_copy<W, E>, wide_grid(blocks, n_layers), dim3(256), 0, s, p, n_slots, src,
                dst, n, lc, lh);
}

// Words per thread: as many as leave the chip at least two workgroups per CU,
// since each of them works the lists out for itself.
template <typename W>
static hipError_t launch_copy_w(const PoolView& p, int n_layers, int n_slots, const int32_t* src,
                                const int32_t* dst, int n, hipStream_t s) {
  const int64_t items = p.slot_bytes / (int64_t)sizeof(W) * n * n_layers;
  if (n > 512 || items >= 512 * 256 * 16)
    return launch_copy_e<W, 16>(p, n_layers, n_slots, src, dst, n, s);
  if (n > 128 || items >= 512 * 256 * 4)
    return launch_copy_e<W, 4>(p, n_layers, n_slots, src, dst, n, s);
  return launch_copy_e<W, 1>(p, n_layers, n_slots, src, dst, n, s);
}

// the widest word that every slot's start and size fit
static int word_of(const PoolView& p, int n_layers) {
  const uint64_t bits = (uint64_t)(uintptr_t)p.base | (uint64_t)p.slot_bytes |
                        (uint64_t)p.slot_stride | (n_layers > 1 ? (uint64_t)p.layer_stride : 0);
  return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1);
}

static hipError_t launch_copy(const PoolView& p, int n_layers, int n_slots, const int32_t* src,
                              const int32_t* dst, int n, hipStream_t s) {
  switch (word_of(p, n_layers)) {
    case 16: return launch_copy_w<uint4>(p, n_layers, n_slots, src, dst, n, s);
    case 4: return launch_copy_w<uint32_t>(p, n_layers, n_slots, src, dst, n, s);
    default: return launch_copy_w<uint8_t>(p, n_layers, n_slots, src, dst, n, s);
  }
}

// ---------------------------------------------------------------------------
// Compaction.  One block finds the moves: a bitmap of the live slots, its
// running count, and from them for each live slot at or above `live` its rank
// among those, which is the rank of the free slot below `live` that it goes
// to.  Sources and destinations are disjoint, so the moves themselves are a
// plain copy.  200 of 512 slots of 24 layers of 64 KB live: 7 us for the list,
// latency of one block's five barriers, and 83 us for 383 MB, 4.6 TB/s.
// ---------------------------------------------------------------------------
struct Moves {
  int32_t count;
  int32_t pad[3];
  // then int32_t src[n_slots / 2], dst[n_slots / 2]
};
__host__ __device__ inline int moves_cap(int n_slots) { return n_slots / 2 + 1; }

__global__ __launch_bounds__(1024) void k_slots_plan(const int32_t* slots,
                                                     int32_t* new_slots, int n, int n_slots,
                                                     int32_t* n_live, Moves* mv) {
  constexpr int kWords = kMaxCompact / 32;
  __shared__ uint32_t bits[kWords];
  __shared__ int before[kWords];  // live slots below the word
  __shared__ int wave_sum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kWords; i += 1024) bits[i] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) {
    const int s = slots[i];
    if (s >= 0 && s < n_slots) atomicOr(&bits[s >> 5], 1u << (s & 31));
  }
  __syncthreads();
  // two words per thread; running count over the wave, then over the waves
  const int c0 = __popc(bits[2 * tid]), c1 = __popc(bits[2 * tid + 1]);
  int sum = c0 + c1;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(sum, m);
    if (lane >= m) sum += o;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int base = 0, live = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    base += w < wave ? wave_sum[w] : 0;
    live += wave_sum[w];
  }
  before[2 * tid] = base + sum - c0 - c1;
  before[2 * tid + 1] = base + sum - c1;
  __syncthreads();
  auto rank = [&](int s) {  // live slots below s
    return before[s >> 5] + __popc(bits[s >> 5] & ((1u << (s & 31)) - 1));
  };
  const int stay = live < n_slots ? rank(live) : live;  // live slots below `live`
  const int cap = moves_cap(n_slots);
  int32_t* src = (int32_t*)(mv + 1);
  int32_t* dst = src + cap;
  for (int s = tid; s < n_slots; s += 1024) {
    const bool on = bits[s >> 5] >> (s & 31) & 1;
    const int r = rank(s);
    if (on && s >= live) src[r - stay] = s;
    if (!on && s < live) dst[s - r] = s;
  }
  if (tid == 0) {
    mv->count = live - stay;
    if (n_live) *n_live = live;
  }
  // dst, written by this block, is read again below
  __threadfence();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int i = tid; i < n; i += 1024) {
    const int s = slots[i];
    const bool on = s >= 0 && s < n_slots;
    new_slots[i] = on && s >= live ? __hip_atomic_load(dst + (rank(s) - stay), __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT)
                                   : s;
  }
}

// the moves of every layer, in runs of 1024 words, over however many blocks
// there are
template <typename W>
__global__ __launch_bounds__(256) void k_slots_move(PoolView pool, int n_layers, int n_slots,
                                                    const Moves* __restrict__ mv) {
  constexpr int kRun = 1024;
  const int32_t* src = (const int32_t*)(mv + 1);
  const int32_t* dst = src + moves_cap(n_slots);
  const int64_t words = pool.slot_bytes / (int64_t)sizeof(W);
  const int64_t runs = (words + kRun - 1) / kRun;
  const int64_t total = runs * n_layers * mv->count;
  for (int64_t r = blockIdx.x; r < total; r += gridDim.x) {
    const int64_t m = r / (runs * n_layers), in = r % (runs * n_layers);
    uint8_t* layer = pool.base + in / runs * pool.layer_stride;
    const W* from = (const W*)(layer + (int64_t)src[m] * pool.slot_stride);
    W* to = (W*)(layer + (int64_t)dst[m] * pool.slot_stride);
    const int64_t w0 = in % runs * kRun + threadIdx.x;
    W v[kRun / 256];
#pragma unroll
    for (int e = 0; e < kRun / 256; ++e)
      if (w0 + 256 * e < words) v[e] = from[w0 + 256 * e];
#pragma unroll
    for (int e = 0; e < kRun / 256; ++e)
      if (w0 + 256 * e < words) to[w0 + 256 * e] = v[e];
  }
}

template <typename W>
static hipError_t launch_move(const PoolView& p, int n_layers, int n_slots, int most,
                              const Moves* mv, hipStream_t s) {
  const int64_t words = p.slot_bytes / (int64_t)sizeof(W);
  const int64_t runs = (words + 1023) / 1024 * n_layers;
  const int64_t total = runs > 4096 ? 4096 : runs * most;
  return launch(k_slots_move<W>, dim3((unsigned)(total < 4096 ? total : 4096)), dim3(256), 0, s, p,
                n_layers, n_slots, mv);
}

static bool pools_fit(const char* name, const bm_hip_slots_t* pools, int n_pools) {
  if (!pools || n_pools < 1 || n_pools > kMaxPools) {
    bm_set_error("%s: 1 to %d pools (%d)", name, kMaxPools, n_pools);
    return false;
  }
  for (int i = 0; i < n_pools; ++i) {
    const bm_hip_slots_t& p = pools[i];
    const int64_t most = (int64_t)1 << 46;
    if (!p.base || p.n_slots < 1 || p.n_slots != pools[0].n_slots || p.n_layers < 1 ||
        p.n_layers > 65535 || p.slot_bytes < 1 || p.slot_bytes > ((int64_t)1 << 40) ||
        p.slot_stride < p.slot_bytes || p.slot_stride > most || p.layer_stride > most ||
        p.layer_stride < 0) {
      bm_set_error("%s: pool %d: %d slots of %lld bytes, stride %lld, %d layers, stride %lld", name,
                   i, p.n_slots, (long long)p.slot_bytes, (long long)p.slot_stride, p.n_layers,
                   (long long)p.layer_stride);
      return false;
    }
    // layers either follow each other or lie within a slot's stride
    const int64_t span = (int64_t)(p.n_slots - 1) * p.slot_stride + p.slot_bytes;
    const bool blocks = p.layer_stride >= span;
    const bool inside = p.layer_stride >= p.slot_bytes &&
                        (p.n_layers - 1) * p.layer_stride + p.slot_bytes <= p.slot_stride;
    if (p.n_layers > 1 && !blocks && !inside) {
      bm_set_error("%s: pool %d: the slots of its layers overlap (layer stride %lld)", name, i,
                   (long long)p.layer_stride);
      return false;
    }
  }
  return true;
}

static PoolView view_of(const bm_hip_slots_t& p) {
  return PoolView{(uint8_t*)p.base, p.slot_bytes, p.slot_stride, p.layer_stride};
}

}  // namespace bm

extern "C" int bm_hip_slots_copy_dev(const bm_hip_slots_t* pools, int n_pools, const int32_t* src,
                                     const int32_t* dst, int n, void* stream) {
  if (!bm::pools_fit("slots_copy", pools, n_pools)) return -2;
  if (n < 0 || n > bm::kMaxPairs || (n > 0 && (!src || !dst)) ||
      ((uintptr_t)src | (uintptr_t)dst) % 4) {
    bm_set_error("slots_copy: invalid lists (0 to %d pairs, n=%d)", bm::kMaxPairs, n);
    return -2;
  }
  if (n == 0) return 0;
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  hipStream_t s = bm::stream_of(stream);
  for (int i = 0; i < n_pools; ++i)
    BM_HIP_CHECK_RET(bm::launch_copy(bm::view_of(pools[i]), pools[i].n_layers, pools[i].n_slots,
                                     src, dst, n, s),
                     -1);
  return 0;
}

extern "C" size_t bm_hip_slots_compact_workspace_bytes(int n_slots) {
  if (n_slots < 1 || n_slots > bm::kMaxCompact) return 0;
  return sizeof(bm::Moves) + 2 * sizeof(int32_t) * (size_t)bm::moves_cap(n_slots);
}

extern "C" int bm_hip_slots_compact_dev(const bm_hip_slots_t* pools, int n_pools,
                                        const int32_t* slots, int32_t* new_slots, int n,
                                        int32_t* n_live, void* workspace, void* stream) {
  if (!bm::pools_fit("slots_compact", pools, n_pools)) return -2;
  const int n_slots = pools[0].n_slots;
  if (n < 0 || n_slots > bm::kMaxCompact || (n > 0 && (!slots || !new_slots)) || !workspace ||
      (uintptr_t)workspace % 16 ||
      ((uintptr_t)slots | (uintptr_t)new_slots | (uintptr_t)n_live) % 4) {
    bm_set_error("slots_compact: invalid arguments (n=%d n_slots=%d)", n, n_slots);
    return -2;
  }
  const uintptr_t t0 = (uintptr_t)slots, t1 = (uintptr_t)new_slots, len = (uintptr_t)n * 4;
  if (t0 != t1 && t0 < t1 + len && t1 < t0 + len) {
    bm_set_error("slots_compact: new_slots overlaps slots in part");
    return -2;
  }
  if (!bm_hip_init()) return -1;
  bm::OnDevice dev;
  hipStream_t s = bm::stream_of(stream);
  bm::Moves* mv = (bm::Moves*)workspace;
  BM_HIP_CHECK_RET(bm::launch(bm::k_slots_plan, dim3(1), dim3(1024), 0, s, slots, new_slots, n,
                              n_slots, n_live, mv),
                   -1);
  const int most = n < n_slots / 2 ? n : n_slots / 2;  // moves: live ones above as many free ones
  if (most == 0) return 0;
  for (int i = 0; i < n_pools; ++i) {
    const bm::PoolView p = bm::view_of(pools[i]);
    hipError_t e;
    switch (bm::word_of(p, pools[i].n_layers)) {
      case 16: e = bm::launch_move<uint4>(p, pools[i].n_layers, n_slots, most, mv, s); break;
      case 4: e = bm::launch_move<uint32_t>(p, pools[i].n_layers, n_slots, most, mv, s); break;
      default: e = bm::launch_move<uint8_t>(p, pools[i].n_layers, n_slots, most, mv, s); break;
    }
    BM_HIP_CHECK_RET(e, -1);
  }
  return 0;
}
