// Log probabilities of given tokens, the entropy of each row and its most likely tokens, from
// materialised logits, with the gradient.
//
// With m = max_j z_j, s = sum_j exp(z_j - m), u = sum_j exp(z_j - m) (z_j - m):
//   log p_t = (z_t - m) - log s,   H = -sum_j p_j log p_j = log s - u / s,
// so one pass over a row with a running maximum and sums gives both; a masked logit (-inf) adds
// nothing to either sum. The alternatives are the top_k largest logits, equal ones in the order of
// their index. The gradient of g log p_t + e H + sum_i a_i log p_{k_i} is
//   dz_j = -p_j (g + sum_i a_i + e (log p_j + H)) + g [j = t] + sum_i a_i [j = k_i].
// Sums and statistics are fp32; m and s are kept apart for the backward pass (their sum m + log s
// would round away the low bits of log s).
#include <climits>

#include "common.cuh"

namespace nfb {

enum LogprobSite : uint32_t { kSiteTarget = 1 };
constexpr int kMaxTop = 32;

struct LpArgs {
  const void* logits;
  const int64_t* targets;  // null: none
  float *logprobs, *entropy, *stats;  // stats: (m, s) per row
  float* top_logprobs;
  int64_t* top_tokens;
  uint32_t* status;
  int64_t rows, ld, ignore_index;
  int V, top_k;
};

struct Stat { float m, s, u; };  // u: sum of exp(z - m) (z - m)

// (x - m) clamped so that a masked logit gives 0 * finite, not 0 * inf; NaN passes through.
__device__ __forceinline__ float clamp_low(float d) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(d), "f"(-1e4f));
  return r;
}

__device__ __forceinline__ Stat stat_merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  const float base = m == -INFINITY ? 0.f : m;
  const float da = clamp_low(a.m - base), db = clamp_low(b.m - base);
  const float ea = expf(da), eb = expf(db);
  // exp(z - m) (z - m) = exp(d) exp(z - m') ((z - m') + d) for m = m' - d
  return {m, a.s * ea + b.s * eb, ea * (a.u + a.s * da) + eb * (b.u + b.s * db)};
}

template <typename T>
__global__ void __launch_bounds__(512) logprobs_kernel(const LpArgs a) {
  __shared__ Stat red[16];
  __shared__ float red_v[16];
  __shared__ int red_i[16];
  __shared__ float best_v;
  __shared__ int best_i;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  Stat st{-INFINITY, 0.f, 0.f};
  for (int j = threadIdx.x; j < a.V; j += blockDim.x) {
    const float z = to_f32(x[j]);
    // the element's own statistics: NaN must reach the sums, so s is exp(z - z) rather than 1
    const float d = clamp_low(z - (z == -INFINITY ? 0.f : z));
    st = stat_merge(st, Stat{z, expf(d), 0.f});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = stat_merge(st, Stat{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                             __shfl_xor_sync(0xffffffffu, st.u, o)});
  if (lane == 0) red[warp] = st;
  __syncthreads();
  st = red[0];
  for (int w = 1; w < warps; ++w) st = stat_merge(st, red[w]);
  const float m = st.m == -INFINITY ? 0.f : st.m, log_s = logf(st.s);
  if (threadIdx.x == 0) {
    a.stats[2 * row] = m;
    a.stats[2 * row + 1] = st.s;
    // a row without a finite logit has no distribution: its entropy is 0
    a.entropy[row] = st.s == 0.f ? 0.f : log_s - st.u / st.s;
    if (a.targets) {
      const int64_t t = a.targets[row];
      float lp = 0.f;
      if (t != a.ignore_index) {
        if (t < 0 || t >= a.V) {
          set_status(a.status, kBadArgument, kSiteTarget);
          lp = __int_as_float(0x7fffffff);
        } else {
          const float z = to_f32(x[t]);
          lp = st.s == 0.f ? -INFINITY : (z - m) - log_s;
        }
      }
      a.logprobs[row] = lp;
    }
  }
  // top_k rounds of the largest (value, lowest index) behind the last one
  float last_v = INFINITY;
  int last_i = -1;
  for (int k = 0; k < a.top_k; ++k) {
    float bv = -INFINITY;
    int bi = INT_MAX;
    for (int j = threadIdx.x; j < a.V; j += blockDim.x) {
      const float z = to_f32(x[j]);
      const bool behind = z < last_v || (z == last_v && j > last_i);
      if (behind && (z > bv || (z == bv && j < bi))) { bv = z; bi = j; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xffffffffu, bv, o);
      const int i = __shfl_xor_sync(0xffffffffu, bi, o);
      if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
    }
    if (lane == 0) { red_v[warp] = bv; red_i[warp] = bi; }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < warps; ++w)
        if (red_v[w] > bv || (red_v[w] == bv && red_i[w] < bi)) { bv = red_v[w]; bi = red_i[w]; }
      best_v = bv;
      best_i = bi;
      a.top_tokens[row * a.top_k + k] = bi == INT_MAX ? 0 : bi;  // only rows with NaN run out of values
      a.top_logprobs[row * a.top_k + k] = st.s == 0.f ? -INFINITY : (bv - m) - log_s;
    }
    __syncthreads();
    last_v = best_v;
    last_i = best_i;
  }
}

struct LpBwdArgs {
  const void* logits;
  const int64_t *targets, *top_tokens;
  const float *g_logprobs, *g_entropy, *g_top;  // null: no gradient from that output
  const float *stats, *entropy;
  void* d_logits;
  int64_t rows, ld, ignore_index;
  int V, top_k;
};

template <typename T>
__global__ void __launch_bounds__(512) logprobs_bwd_kernel(const LpBwdArgs a) {
  __shared__ int s_idx[kMaxTop + 1];
  __shared__ float s_g[kMaxTop + 1];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.ld;
  T* dx = (T*)a.d_logits + row * a.V;
  const int n_fix = a.top_k + 1;
  if (threadIdx.x < n_fix) {  // entry 0: the target; then the alternatives
    int j = -1;
    float g = 0.f;
    if (threadIdx.x == 0) {
      if (a.g_logprobs && a.targets[row] != a.ignore_index && a.targets[row] >= 0 && a.targets[row] < a.V) {
        j = (int)a.targets[row];
        g = a.g_logprobs[row];
      }
    } else if (a.g_top) {
      j = (int)a.top_tokens[row * a.top_k + threadIdx.x - 1];
      g = a.g_top[row * a.top_k + threadIdx.x - 1];
    }
    s_idx[threadIdx.x] = j;
    s_g[threadIdx.x] = g;
  }
  __syncthreads();
  float whole = 0.f;
  for (int i = 0; i < n_fix; ++i) whole += s_g[i];
  const float m = a.stats[2 * row], s = a.stats[2 * row + 1], log_s = logf(s);
  const float e = a.g_entropy ? a.g_entropy[row] : 0.f, H = a.entropy[row];
  const float inv = s == 0.f ? 0.f : 1.f / s;
  for (int j = threadIdx.x; j < a.V; j += blockDim.x) {
    const float d = clamp_low(to_f32(x[j]) - m);
    const float p = s == 0.f ? 0.f : expf(d) * inv;
    float g = s == 0.f ? 0.f : -p * (whole + e * ((d - log_s) + H));
    if (s != 0.f)
      for (int i = 0; i < n_fix; ++i)
        if (s_idx[i] == j) g += s_g[i];
    dx[j] = from_f32<T>(g);
  }
}

}  // namespace nfb

using namespace nfb;

NFB_API int nfb_logprobs_fwd(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t V, const int64_t* targets,
                             int64_t ignore_index, int top_k, float* logprobs, float* entropy, float* stats,
                             float* top_logprobs, int64_t* top_tokens, uint32_t* status, void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX - 4096 || top_k < 0 || top_k > kMaxTop || top_k > V)
    return (int)cudaErrorInvalidValue;
  const LpArgs a{logits, targets, logprobs, entropy, stats, top_logprobs, top_tokens, status,
                 rows, ld, ignore_index, (int)V, top_k};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == kF32) logprobs_kernel<float><<<(unsigned)rows, 512, 0, st>>>(a);
  else if (dtype == kBF16) logprobs_kernel<__nv_bfloat16><<<(unsigned)rows, 512, 0, st>>>(a);
  else if (dtype == kF16) logprobs_kernel<__half><<<(unsigned)rows, 512, 0, st>>>(a);
  else return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}

NFB_API int nfb_logprobs_bwd(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t V, const int64_t* targets,
                             int64_t ignore_index, int top_k, const int64_t* top_tokens, const float* g_logprobs,
                             const float* g_entropy, const float* g_top, const float* stats, const float* entropy,
                             void* d_logits, void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX - 4096 || top_k < 0 || top_k > kMaxTop || top_k > V)
    return (int)cudaErrorInvalidValue;
  const LpBwdArgs a{logits, targets, top_tokens, g_logprobs, g_entropy, g_top, stats, entropy, d_logits,
                    rows, ld, ignore_index, (int)V, top_k};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == kF32) logprobs_bwd_kernel<float><<<(unsigned)rows, 512, 0, st>>>(a);
  else if (dtype == kBF16) logprobs_bwd_kernel<__nv_bfloat16><<<(unsigned)rows, 512, 0, st>>>(a);
  else if (dtype == kF16) logprobs_bwd_kernel<__half><<<(unsigned)rows, 512, 0, st>>>(a);
  else return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}
