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
// Prompts, token by token: a wave holds R channels of a head, their state
// values over its lanes.
// ---------------------------------------------------------------------------
constexpr int kPlainRows = 4;

template <typename T>
__global__ __launch_bounds__(64) void k_ssm_plain(SsmArgs a) {
  const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int p0 = blockIdx.z * kPlainRows;
  const int slot = find_slot(a.q, b);
  if (slot == kNoSlot) return;
  const int s = a.q.seq_start ? seq_row(a.q, b) : 0;
  const int e = a.q.seq_start ? seq_row(a.q, b + 1) : a.q.n_tokens;
  const int g = h / (a.heads / a.groups);
  float* st = slot >= 0 ? a.state + (int64_t)slot * a.ss + (int64_t)h * a.hd * a.n : nullptr;
  const bool keep = slot >= 0 && !(a.q.fresh && a.q.fresh[b]);
  float S[kPlainRows][4];
#pragma unroll
  for (int r = 0; r < kPlainRows; ++r)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = lane + 64 * k;
      S[r][k] = keep && p0 + r < a.hd && n < a.n ? st[(int64_t)(p0 + r) * a.n + n] : 0.0f;
    }
  for (int t = s; t < e; ++t) {
    const float d = step_of(a, (float)((const T*)a.dt)[(int64_t)t * a.dts + h], h);
    const float decay = exp_f32(a.A[h] * d);
    float Bv[4], Cv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = lane + 64 * k;
      const int64_t o = (int64_t)g * a.n + n;
      Bv[k] = n < a.n ? d * (float)((const T*)a.B)[(int64_t)t * a.Bs + o] : 0.0f;
      Cv[k] = n < a.n ? (float)((const T*)a.C)[(int64_t)t * a.Cs + o] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kPlainRows; ++r) {
      if (p0 + r >= a.hd) break;
      const int64_t c = (int64_t)h * a.hd + p0 + r;
      const float x = (float)((const T*)a.x)[(int64_t)t * a.xs + c];
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        S[r][k] = __builtin_fmaf(S[r][k], decay, x * Bv[k]);
        sum = __builtin_fmaf(S[r][k], Cv[k], sum);
      }
      sum = team_sum<64>(sum);
      if (lane == 0) {
        if (a.D) sum = __builtin_fmaf(a.D[c], x, sum);
        if (a.z) sum *= silu_f32((float)((const T*)a.z)[(int64_t)t * a.zs + c]);
        ((T*)a.y)[(int64_t)t * a.ys + c] = (T)sum;
      }
    }
  }
  if (st)
#pragma unroll
    for (int r = 0; r < kPlainRows; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = lane + 64 * k;
        if (p0 + r < a.hd && n < a.n) st[(int64_t)(p0 + r) * a.n + n] = S[r][k];
      }
}

template <typename T>
static hipError_t launch_scan_t(const SsmArgs& a, void* workspace, hipStream_t s) {
  (void)workspace;
  hipLaunchKernelGGL((k_ssm_plain<T>),
                     dim3(a.q.n_seqs, a.heads, (a.hd + kPlainRows - 1) / kPlainRows), dim3(64), 0,
                     s, a);
  return hipGetLastError();
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
  return 0;
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
  if (!step && bm_hip_ssm_workspace_bytes(op) && (!workspace || (uintptr_t)workspace % 256)) {
    bm_set_error("%s: a workspace on 256 bytes is required", name);
    return -2;
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
      e = step ? bm::launch_step_t<float>(a, s) : bm::launch_scan_t<float>(a, workspace, s);
      break;
    case BM_HIP_BF16:
      e = step ? bm::launch_step_t<__bf16>(a, s) : bm::launch_scan_t<__bf16>(a, workspace, s);
      break;
    default:
      e = step ? bm::launch_step_t<_Float16>(a, s) : bm::launch_scan_t<_Float16>(a, workspace, s);
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
