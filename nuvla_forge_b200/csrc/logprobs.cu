// Log probabilities of given tokens, the entropy of each row and its most likely tokens, from
// materialised logits, with the gradient.
//
// With m = max_j z_j, r = sum of exp(z_j - m) over all j but one that has the maximum, and
// u = sum_j exp(z_j - m) (z_j - m):
//   log p_t = (z_t - m) - log(1 + r),   H = -sum_j p_j log p_j = log(1 + r) - u / (1 + r),
// so one pass over a row with a running maximum and sums gives both; a masked logit (-inf) adds
// nothing to either sum. The sum is kept as its excess over 1 because a trained head often has a
// row's mass on one token: then log p_t = -r + ..., and a sum near 1 would have lost the digits of r.
// The alternatives are the top_k largest logits, equal ones in the order of their index. The gradient
// of g log p_t + e H + sum_i a_i log p_{k_i} is
//   dz_j = -p_j (g + sum_i a_i + e (log p_j + H)) + g [j = t] + sum_i a_i [j = k_i].
// Sums and statistics are fp32; m and r are kept apart for the backward pass.
#include <climits>
#include <cooperative_groups.h>

#include "common.cuh"

namespace nfb {

namespace cg = cooperative_groups;

enum LogprobSite : uint32_t { kSiteTarget = 1 };
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.44269504088896340736f;

struct LpArgs {
  const void* logits;
  const int64_t* targets;  // null: none
  float *logprobs, *entropy, *stats;  // stats: (m, r) of each row, or null
  float* top_logprobs;
  int64_t* top_tokens;
  uint32_t* status;
  int64_t rows, ld, ignore_index;
  int V, top_k, split;  // split: CTAs (one cluster) a row
};

struct Stat { float m, s, u; };  // maximum; sums of exp(z - m) and of exp(z - m) (z - m)
struct RowStat { float m, r, u; };  // the same with r = s - 1; r = -1: no finite logit

// z - m clamped so that a masked logit gives 0 * finite, not 0 * inf; NaN passes through. (The
// difference is taken before the factor log2(e): a row at the type's lowest value stays finite.)
__device__ __forceinline__ float below_max(float z, float m) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z - m), "f"(-1e4f));
  return r;
}
__device__ __forceinline__ float exp_of(float d) {  // relative: 2^-22 of ex2, |d| 2^-24 of the rounded product
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * kLog2e));
  return y;
}
__device__ __forceinline__ float or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// `a` moved to the maximum m: exp(d + c) (d + c) with c = a.m - m.
__device__ __forceinline__ Stat stat_at(Stat a, float m) {
  const float c = below_max(a.m, or_zero(m)), e = exp_of(c);
  return {m, a.s * e, e * (a.u + a.s * c)};
}
// The statistics of two disjoint parts of a row together.
__device__ __forceinline__ RowStat row_merge(RowStat a, RowStat b) {
  if (b.m > a.m) {
    const RowStat t = a;
    a = b;
    b = t;
  }
  const float c = below_max(b.m, or_zero(a.m)), e = exp_of(c), s = 1.f + b.r;
  return {a.m, a.r + s * e, a.u + e * (b.u + s * c)};
}

// Order of the alternatives as one number: the value (zeros of both signs alike), then the lower index.
__device__ __forceinline__ uint64_t rank_key(float z, int j) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return (uint64_t)(b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}

// Largest of a 16-byte vector's values, NaN left out; pairs of 16-bit values at a time.
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(&v);
    const T2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
}

// The row is read once here, so it leaves no lines in L1; it stays in the L2 for a backward pass.
__device__ __forceinline__ uint4 ld_row(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The k-th largest of the warp's 32 values (counted with repetition).
__device__ __forceinline__ float kth_of_warp(float v, int k) {
  const uint32_t b = __float_as_uint(v + 0.f);
  const uint32_t key = b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  bool in = true;
  uint32_t best = 0;
  if (k <= 16) {
    for (int i = 0; i < k; ++i) {  // the largest one leaves
      best = __reduce_max_sync(0xffffffffu, in ? key : 0u);
      const uint32_t who = __ballot_sync(0xffffffffu, in && key == best);
      in = in && (int)(threadIdx.x & 31) != __ffs(who) - 1;
    }
  } else {
    for (int i = k; i <= 32; ++i) {  // the smallest one leaves
      best = __reduce_min_sync(0xffffffffu, in ? key : 0xFFFFFFFFu);
      const uint32_t who = __ballot_sync(0xffffffffu, in && key == best);
      in = in && (int)(threadIdx.x & 31) != __ffs(who) - 1;
    }
  }
  return __uint_as_float(best ^ ((best >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// Forward. A CTA (or a cluster of them, where there are few rows) streams over a row: each thread
// keeps sums against its own running maximum, so the row is read once, no thread waits for a common
// maximum, and few registers leave room for the loads of many rows in flight.
//
// Alternatives: the k-th largest of the maxima of 32 groups of threads bounds the k-th largest logit
// from below. The bound is taken after every thread's first vectors and renewed as the row goes by (a
// group maximum that is read late is only a lower bound, so nobody waits); a thread whose vectors of a
// round reach it notes their place and maximum, some k (1 + log(rounds)) notes a row. At the end the
// notes that reach the final bound are read again, from the L2, a warp for each note and a lane for
// each value, and the candidates (about k) are ranked against one another. (Looking at the values when
// they come, unrolled over a thread's vectors, filled the loop with code that crowded the instruction
// cache: 15% of the stalls.) If values equal to the bound overflow (a constant or fully masked row),
// those above it are ranked and the first ones equal to it taken in the order of the row; if even the
// greater ones overflow (sorted rows), k rounds of a block-wide maximum remain.
//
// What bounds it: for 16-bit logits the HBM's rate leaves 11 issue slots of an SM for a warp's 32 values,
// and the sums take 8 with one exponential among them. Without alternatives 16384 x 32000 bf16 take
// 178 us (5.9 TB/s, 92% of the measured copy rate) at 1965 MHz, 203 us once the power limit holds the SMs
// near 1680 MHz; with 5 the issue slots bind (84% busy): 233 us. With many alternatives (1500 x 150001:
// 91 us with none, 124 us with 20, 206 us with 32) the search for the bound and the notes bind, and for
// rows of a few hundred logits (100000 x 300: 142 us, with 5 alternatives 285 us; the bytes take 9 us) the
// block's fixed work, 5 us a row without and 10 us with alternatives.
constexpr int kLpUnroll = 4, kLpAbove = 512, kLpEqual = 128;

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1536 / NT) logprobs_kernel(const LpArgs a) {
  constexpr int VE = 16 / sizeof(T), kWarps = NT / 32, kGroup = NT / 32;  // 32 groups of kGroup threads
  constexpr int kNotes = NT == 64 ? 256 : NT == 128 ? 768 : 1024;  // 32 alternatives leave some 130 (1 + log(rounds))
  __shared__ Stat s_stat[kWarps];
  __shared__ float s_group[32];
  __shared__ int s_noted, s_above, s_equal;   // notes; candidates above the bound and equal to it
  __shared__ float2 s_note[kNotes];         // a thread's maximum in a round, and the number of its first vector
  __shared__ uint64_t s_cand[kLpAbove + kLpEqual];
  __shared__ uint64_t s_best[kMaxTop];        // keys of the alternatives, descending; 0: none
  __shared__ uint64_t s_round[kWarps];
  __shared__ RowStat s_row;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = a.split == 1 ? blockIdx.x : blockIdx.x / a.split;
  const int rank = a.split == 1 ? 0 : blockIdx.x % a.split;
  const T* x = (const T*)a.logits + row * a.ld;
  const int k = a.top_k;
  // rows begin anywhere: values in front of the first 16-byte boundary and behind the last one are
  // taken one by one by the first threads
  const int head = min(a.V, (int)((-reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)));
  const int vecs = (a.V - head) / VE;
  const int per = (vecs + a.split - 1) / a.split;
  const int first = min(vecs, rank * per), last = min(vecs, first + per);
  const int lo = rank == 0 ? 0 : head + first * VE, hi = rank == a.split - 1 ? a.V : head + last * VE;
  const int n_front = head + first * VE - lo, n_back = hi - (head + last * VE);
  const int single = tid < n_front ? lo + tid : tid - n_front < n_back ? head + last * VE + (tid - n_front) : -1;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  if (tid < kMaxTop) s_best[tid] = 0;
  if (tid == 0) s_noted = s_above = s_equal = 0;

  float mx = single >= 0 ? to_f32(x[single]) : -INFINITY;
  Stat st{-INFINITY, 0.f, 0.f};
  {
    const float z = mx;
    st.m = mx = fmaxf(mx, -INFINITY);  // NaN left out
    const float d = below_max(z, or_zero(mx));
    if (single >= 0) {
      st.s = exp_of(d);
      st.u = st.s * d;
    }
  }
  const int rounds = (last - first + NT * kLpUnroll - 1) / (NT * kLpUnroll);
  float bound = INFINITY;
  volatile float* group = s_group;
  auto publish = [&](float m) {  // this thread's group maximum so far
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane % kGroup == 0) group[tid / kGroup] = m;
  };
#pragma unroll 1
  for (int turn = 0; turn < rounds; ++turn) {
    const int base = first + turn * (NT * kLpUnroll), v0 = base + tid;
    uint4 w[kLpUnroll];
    if (base + NT * kLpUnroll <= last) {
#pragma unroll
      for (int i = 0; i < kLpUnroll; ++i) w[i] = ld_row(xv + v0 + i * NT);
    } else {
#pragma unroll
      for (int i = 0; i < kLpUnroll; ++i) {
        const uint32_t none = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
        w[i] = make_uint4(none, none, none, none);  // -inf
        if (v0 + i * NT < last) w[i] = ld_row(xv + v0 + i * NT);
      }
    }
    float m = vec_max<T>(w[0]);
#pragma unroll
    for (int i = 1; i < kLpUnroll; ++i) m = fmaxf(m, vec_max<T>(w[i]));
    if (m > mx) {
      mx = m;
      st = stat_at(st, mx);
    }
    if (k > 0) {
      // rounds 0, 2, 8, 32, ..., or with many alternatives 0, 1, 2, 4, ... (1500 x 150001 with 32: 206 us, 286 us)
      if ((turn & (turn - 1)) == 0 && (turn == 0 || k > 8 || (turn & 0x2AAAAAAA))) {
        publish(mx);
        if (turn == 0) __syncthreads();
        bound = kth_of_warp(group[lane], k);
      }
      if (m >= bound) {
        const int at = atomicAdd(&s_noted, 1);
        if (at < kNotes) s_note[at] = make_float2(m, __int_as_float(v0));
      }
    }
    const float ref = or_zero(mx);
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < kLpUnroll; ++i) {
      float z[VE];
      unpack16<T>(w[i], z);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = below_max(z[e], ref), p = exp_of(d);
        s += p;
        u = fmaf(p, d, u);
      }
    }
    st.s += s;
    st.u += u;
  }
  // the warps' sums, then the row's by the warp that has the maximum
  {
    Stat t = stat_at(st, warp_max(st.m));
    t.s = warp_sum(t.s);
    t.u = warp_sum(t.u);
    if (lane == 0) s_stat[warp] = t;
  }
  if (k > 0) publish(mx);
  __syncthreads();
  {
    Stat t = lane < kWarps ? s_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    const float m = warp_max(t.m);
    const int owner = __ffs(__ballot_sync(0xffffffffu, t.m == m)) - 1;
    if (warp == owner) {
      t = stat_at(t, m);
      const float sum = warp_sum(t.s), u = warp_sum(t.u);
      float r = sum - 1.f;
      if (sum < 2.f && m != -INFINITY) {
        // the sum may be little more than 1: everything but the maximum again, by whole warps where that
        // is exact enough, and value by value (a lane each) for the thread that has the maximum
        const int src = __ffs(__ballot_sync(0xffffffffu, mx == m)) - 1, src_tid = tid - lane + src;
        r = (lane < kWarps && lane != owner ? t.s : 0.f) + (lane != src ? stat_at(st, m).s : 0.f);
        const int n = max(0, (last - first - src_tid + NT - 1) / NT) * VE;
        bool left_out = false;
#pragma unroll 4
        for (int e0 = 0; e0 < n; e0 += 32) {
          const int e = e0 + lane;
          const float z = e < n ? to_f32(x[head + (first + src_tid + e / VE * NT) * VE + e % VE]) : -INFINITY;
          const uint32_t hit = __ballot_sync(0xffffffffu, z == m);
          if (e < n && (left_out || lane != __ffs(hit) - 1)) r += exp_of(below_max(z, m));
          left_out = left_out || hit != 0;
        }
        const int one = __shfl_sync(0xffffffffu, single, src);
        if (one >= 0 && lane == 0) {
          const float z = to_f32(x[one]);
          if (left_out || z != m) r += exp_of(below_max(z, m));
        }
        r = warp_sum(r);
      }
      if (lane == 0) s_row = {m, r, u};
    }
  }
  auto rank_in = [&](const uint64_t* list, int n, uint64_t mine) {
    int better = 0;
    for (int o = 0; o < n; ++o) better += list[o] > mine;
    if (better < k) s_best[better] = mine;
  };
  if (k > 0) {
    bound = kth_of_warp(group[lane], k);
    auto take = [&](float z, int j) {
      if (z > bound) {
        const int at = atomicAdd(&s_above, 1);
        if (at < kLpAbove) s_cand[at] = rank_key(z, j);
      } else if (z == bound) {
        const int at = atomicAdd(&s_equal, 1);
        if (at < kLpEqual) s_cand[kLpAbove + at] = rank_key(z, j);
      }
    };
    if (single >= 0) take(to_f32(x[single]), single);
    // lane l of a warp has value l of the vectors from number v0 on, NT apart
    const int lane_v = lane / VE * NT, lane_e = lane % VE;
    const bool lane_on = lane < kLpUnroll * VE;
    const int notes = s_noted;
    if (notes <= kNotes) {
      for (int i0 = warp; i0 < notes; i0 += 4 * kWarps) {
        int j[4];
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 n = i0 + i * kWarps < notes ? s_note[i0 + i * kWarps] : make_float2(-INFINITY, 0.f);
          const int v = __float_as_int(n.y) + lane_v;
          j[i] = i0 + i * kWarps < notes && n.x >= bound && lane_on && v < last ? head + v * VE + lane_e : -1;
          if (j[i] >= 0) z[i] = to_f32(x[j[i]]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j[i] >= 0) take(z[i], j[i]);
      }
    } else {  // too many: every round of the lanes that reach the bound
      for (uint32_t who = __ballot_sync(0xffffffffu, mx >= bound); who; who &= who - 1) {
        for (int turn = 0; turn < rounds; ++turn) {
          const int v = first + turn * (NT * kLpUnroll) + (tid - lane + __ffs(who) - 1) + lane_v;
          const int j = head + v * VE + lane_e;
          if (lane_on && v < last) take(to_f32(x[j]), j);
        }
      }
    }
    __syncthreads();
    const int above = s_above, equal = s_equal;
    if (above >= k ? above <= kLpAbove : equal <= kLpEqual) {
      // rank those above the bound, and those equal to it where they are needed
      const int n = above >= k ? above : above + equal;
      for (int i = tid; i < n; i += NT) {
        const uint64_t mine = s_cand[i < above ? i : kLpAbove + (i - above)];
        int better = 0;
        for (int o = 0; o < above; ++o) better += s_cand[o] > mine;
        if (i >= above)
          for (int o = 0; o < equal; ++o) better += s_cand[kLpAbove + o] > mine;
        if (better < k) s_best[better] = mine;
      }
    } else if (above < k) {
      if (tid < above) rank_in(s_cand, above, s_cand[tid]);
      int found = above;  // the first equal ones in the order of the row
      for (int j0 = lo; j0 < hi && found < k; j0 += NT) {
        const int j = j0 + tid;
        const float z = j < hi ? to_f32(x[j]) : 0.f;
        const uint32_t hit = __ballot_sync(0xffffffffu, j < hi && z == bound);
        if (lane == 0) s_round[warp] = __popc(hit);
        __syncthreads();
        int at = found;
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) at += (int)s_round[w];
          found += (int)s_round[w];
        }
        at += __popc(hit & ((1u << lane) - 1));
        if ((hit >> lane & 1) && at < k) s_best[at] = rank_key(z, j);
        __syncthreads();
      }
    } else {
      uint64_t below = ~0ull;
      for (int r = 0; r < k; ++r) {
        uint64_t best = 0;
        auto look = [&](float z, int j) {
          const uint64_t key = rank_key(z, j);
          if (z == z && key < below && key > best) best = key;
        };
        if (single >= 0) look(to_f32(x[single]), single);
        for (int v = first + tid; v < last; v += NT) {
          float z[VE];
          unpack16<T>(__ldg(xv + v), z);
#pragma unroll
          for (int e = 0; e < VE; ++e) look(z[e], head + v * VE + e);
        }
        best = warp_max_key(best);
        if (lane == 0) s_round[warp] = best;
        __syncthreads();
        best = warp_max_key(lane < kWarps ? s_round[lane] : 0);
        if (tid == 0) s_best[r] = best;
        below = best;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  RowStat t = s_row;
  if (a.split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0 && warp == 0) {
      for (int r = 1; r < a.split; ++r) t = row_merge(t, *cluster.map_shared_rank(&s_row, r));
      if (k > 0) {  // the CTAs' lists, ranked again
        for (int r = 0; r < a.split; ++r)
          if (lane < k) s_cand[r * k + lane] = cluster.map_shared_rank(s_best, r)[lane];
        __syncwarp();
        if (lane < k) s_best[lane] = 0;
        __syncwarp();
        for (int i = lane; i < a.split * k; i += 32) {
          const uint64_t mine = s_cand[i];
          int better = 0;
          for (int o = 0; o < a.split * k; ++o) better += s_cand[o] > mine;
          if (mine != 0 && better < k) s_best[better] = mine;
        }
        __syncwarp();
      }
    }
    cluster.sync();  // the other CTAs' shared memory has been read
    if (rank != 0) return;
  }
  if (warp != 0) return;
  const float m = or_zero(t.m), log_s = log1pf(t.r);
  const bool none = t.r == -1.f;  // no finite logit: no distribution, its entropy is 0
  if (lane == 0) {
    if (a.stats) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = t.r;
    }
    a.entropy[row] = none ? 0.f : log_s - t.u / (1.f + t.r);
    if (a.targets) {
      const int64_t j = a.targets[row];
      float lp = 0.f;
      if (j != a.ignore_index) {
        if (j < 0 || j >= a.V) {
          set_status(a.status, kBadArgument, kSiteTarget);
          lp = __int_as_float(0x7fffffff);
        } else {
          lp = none ? -INFINITY : (to_f32(x[j]) - m) - log_s;
        }
      }
      a.logprobs[row] = lp;
    }
  }
  if (lane < k) {
    const uint64_t key = s_best[lane];  // 0: only a row with NaN runs out of values
    a.top_tokens[row * k + lane] = key == 0 ? 0 : (int)~(uint32_t)key;
    a.top_logprobs[row * k + lane] = none ? -INFINITY : (key_value(key) - m) - log_s;
  }
}

struct LpBwdArgs {
  const void* logits;
  const int64_t *targets, *top_tokens;
  const float *g_logprobs, *g_entropy, *g_top;  // null: no gradient from that output
  const float *stats, *entropy;
  void* d_logits;
  int64_t rows, ld, ignore_index;
  int V, top_k, chunks, per;  // CTAs a row; values of a chunk
};

// Backward: a stream over the row, bound by its bytes (each logit read, each gradient written: 16384 x
// 32000 bf16 in 312 us, 6.7 TB/s, the measured copy rate). With d = z - m the gradient apart from the
// given tokens is exp(d) (c1 d + c0), c0 and c1 of the row, which one warp prepares while the first
// logits are on their way. The given tokens' places are written
// again by the first threads, each with its whole value (a token may be the target and an alternative),
// rounded once.
// Rows whose distance differs from V by no multiple of 16 bytes (logits cut from an odd padded vocabulary) are
// read and written value by value: 8192 x 32000 bf16 646 us, against 161 us dense or cut from 32008.
// 40 registers: 16384 x 32000 bf16 312 us; 32 and a spill 321 us, 48 320 us, 64 349 us (fewer CTAs).
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(NT, 1536 / NT) logprobs_bwd_kernel(const LpBwdArgs a) {
  constexpr int VE = 16 / sizeof(T), kVecs = 4;
  __shared__ int s_idx[kMaxTop + 1];
  __shared__ float s_g[kMaxTop + 1];
  __shared__ float s_c0, s_c1, s_log;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x - row * a.chunks);
  const T* x = (const T*)a.logits + row * a.ld;
  T* dx = (T*)a.d_logits + row * a.V;
  const int begin = chunk * a.per, end = min(a.V, begin + a.per);
  // VEC: x and dx begin at the same distance from a 16-byte boundary
  const int head = VEC ? min(end, begin + (int)((-reinterpret_cast<uintptr_t>(x + begin) & 15) / sizeof(T))) : end;
  const int vecs = (end - head) / VE, tail = head + vecs * VE;
  uint4 w[kVecs];
  if constexpr (VEC) {
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if ((int)threadIdx.x + i * NT < vecs) w[i] = __ldcs(xv + threadIdx.x + i * NT);
  }
  const float m = a.stats[2 * row], r = a.stats[2 * row + 1];
  const float e = a.g_entropy ? a.g_entropy[row] : 0.f, H = a.entropy[row];
  const bool none = r == -1.f;  // no finite logit: no gradient
  const float inv = none ? 0.f : 1.f / (1.f + r);
  const int n_fix = a.top_k + 1;
  if (threadIdx.x < 32) {
    // entry 0: the target; then the alternatives
    float whole = 0.f;
    for (int i = threadIdx.x; i < n_fix; i += 32) {
      int j = -1;
      float g = 0.f;
      if (i == 0) {
        if (a.g_logprobs) {
          const int64_t t = a.targets[row];
          if (t != a.ignore_index && t >= 0 && t < a.V) {
            j = (int)t;
            g = a.g_logprobs[row];
          }
        }
      } else if (a.g_top) {
        j = (int)a.top_tokens[row * a.top_k + i - 1];
        g = a.g_top[row * a.top_k + i - 1];
      }
      s_idx[i] = j;
      s_g[i] = g;
      whole += g;
    }
    whole = warp_sum(whole);
    if (threadIdx.x == 0) {
      const float log_s = log1pf(r);
      s_log = log_s;
      s_c0 = none ? 0.f : -(whole + e * (H - log_s)) * inv;
      s_c1 = -e * inv;
    }
  }
  __syncthreads();
  const float c0 = s_c0, c1 = s_c1, log_s = s_log;
  auto grad = [&](float z) {
    const float d = below_max(z, m);
    return exp_of(d) * fmaf(c1, d, c0);
  };
  if constexpr (VEC) {
    if ((int)threadIdx.x < head - begin) dx[begin + threadIdx.x] = from_f32<T>(grad(to_f32(x[begin + threadIdx.x])));
    if ((int)threadIdx.x < end - tail) dx[tail + threadIdx.x] = from_f32<T>(grad(to_f32(x[tail + threadIdx.x])));
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    uint4* dv = reinterpret_cast<uint4*>(dx + head);
    for (int v0 = threadIdx.x;;) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        if (v0 + i * NT < vecs) {
          float z[VE];
          unpack16<T>(w[i], z);
#pragma unroll
          for (int k = 0; k < VE; ++k) z[k] = grad(z[k]);
          dv[v0 + i * NT] = pack16<T>(z);
        }
      }
      v0 += kVecs * NT;
      if (v0 >= vecs) break;
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
        if (v0 + i * NT < vecs) w[i] = __ldcs(xv + v0 + i * NT);
    }
  } else {
    for (int j = begin + threadIdx.x; j < end; j += NT) dx[j] = from_f32<T>(grad(to_f32(x[j])));
  }
  __syncthreads();
  if ((int)threadIdx.x < n_fix && !none) {
    const int j = s_idx[threadIdx.x];
    if (j >= begin && j < end) {
      float own = 0.f, others = 0.f;
      for (int i = 0; i < n_fix; ++i) (s_idx[i] == j ? own : others) += s_g[i];
      // own - p own as own (1 - p), with 1 - p from the excess r: p may be nearly 1
      const float d = below_max(to_f32(x[j]), m);
      dx[j] = from_f32<T>(own * ((r - expm1f(d)) * inv) - exp_of(d) * inv * (others + e * ((d - log_s) + H)));
    }
  }
}

}  // namespace nfb

using namespace nfb;

namespace {

template <typename T, int NT>
int launch_fwd_nt(LpArgs& a, cudaStream_t st) {
  // a cluster for each row while the rows leave SMs idle and each CTA keeps two vectors a thread (one row
  // of 150000 fp32 logits 10.8 us, undivided 22.4 us; of 32000 bf16 6.6 us against 7.4 us)
  const int64_t vecs = a.V / (int64_t)(16 / sizeof(T));
  a.split = 1;
  while (a.split < 8 && a.rows * a.split * 2 <= 2 * nfb_num_sms() && vecs >= (int64_t)a.split * 4 * NT) a.split *= 2;
  if (a.rows * a.split > INT_MAX) return (int)cudaErrorInvalidValue;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * a.split));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = a.split > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, logprobs_kernel<T, NT>, a);
}

// Threads a row: few for short rows and where many rows fill the GPU anyway (less waiting for one
// another: 16384 x 32000 bf16 with 5 alternatives 229 us with 128, 266 us with 256; 20000 x 2000 fp16
// 57 us with 64, 89 us with 128), many for few rows or long ones (64 x 32000 bf16: 7.6 us with 256, 8.2 us
// with 128; 1500 x 150001 with 32 alternatives 211 us against 461 us, whose notes overflow).
// Above 128 KB a row 256 threads cost little with few alternatives (4000 x 80001 bf16 with 5: 139 us, 134 us
// with 128; 1000 x 150001 fp32 with none: 117 us, 107 us) and save much with many (the latter with 32:
// 390 us, 1199 us).
template <typename T>
int launch_fwd(LpArgs& a, cudaStream_t st) {
  const int64_t bytes = a.V * (int64_t)sizeof(T);
  if (bytes < 8192) return launch_fwd_nt<T, 64>(a, st);
  if (bytes < 16384 || (bytes <= 131072 && a.rows >= 12 * (int64_t)nfb_num_sms())) return launch_fwd_nt<T, 128>(a, st);
  return launch_fwd_nt<T, 256>(a, st);
}

template <typename T, int NT>
int launch_bwd_nt(LpBwdArgs& a, cudaStream_t st) {
  // four vectors a thread, twice where the CTAs are more than run at once: what a CTA prepares weighs half
  // (16384 x 32000 bf16 321 us, with one round 336 us, both at 32 registers; one row of 32000 3.5 us with
  // one round, 4.3 with two)
  constexpr int64_t kRound = 64 * NT / (int64_t)sizeof(T);
  int64_t chunk = kRound;
  if (a.rows * ((a.V + kRound - 1) / kRound) > 1536 / NT * (int64_t)nfb_num_sms()) chunk *= 2;
  a.chunks = (int)((a.V + chunk - 1) / chunk);
  // chunks of whole 16-byte pieces and of like size
  a.per = (int)((((int64_t)a.V + a.chunks - 1) / a.chunks + 7) / 8 * 8);
  if (a.rows * a.chunks > INT_MAX) return (int)cudaErrorInvalidValue;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.d_logits)) & 15) == 0 &&
                   (a.ld - a.V) * (int64_t)sizeof(T) % 16 == 0;
  const unsigned grid = (unsigned)(a.rows * a.chunks);
  if (vec) logprobs_bwd_kernel<T, NT, true><<<grid, NT, 0, st>>>(a);
  else logprobs_bwd_kernel<T, NT, false><<<grid, NT, 0, st>>>(a);
  return (int)cudaGetLastError();
}

// Threads a CTA: few for short rows, so that as many rows are under way as threads allow and fewer idle
// (20000 x 2000 fp16 35 us with 64, 44 us with 128, 64 us with 256; 6000 x 8003 bf16 38 us with 128,
// 42 us with 256); of no weight where a row has several chunks.
template <typename T>
int launch_bwd(LpBwdArgs& a, cudaStream_t st) {
  const int64_t bytes = a.V * (int64_t)sizeof(T);
  if (bytes <= 8192) return launch_bwd_nt<T, 64>(a, st);
  if (bytes <= 16384) return launch_bwd_nt<T, 128>(a, st);
  return launch_bwd_nt<T, 256>(a, st);
}

}  // namespace

NFB_API int nfb_logprobs_fwd(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t V, const int64_t* targets,
                             int64_t ignore_index, int top_k, float* logprobs, float* entropy, float* stats,
                             float* top_logprobs, int64_t* top_tokens, uint32_t* status, void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX - (1 << 20) || top_k < 0 || top_k > kMaxTop || top_k > V)
    return (int)cudaErrorInvalidValue;
  LpArgs a{logits, targets, logprobs, entropy, stats, top_logprobs, top_tokens, status,
           rows, ld, ignore_index, (int)V, top_k, 1};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return launch_fwd<float>(a, st);
    case kBF16: return launch_fwd<__nv_bfloat16>(a, st);
    case kF16: return launch_fwd<__half>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}

NFB_API int nfb_logprobs_bwd(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t V, const int64_t* targets,
                             int64_t ignore_index, int top_k, const int64_t* top_tokens, const float* g_logprobs,
                             const float* g_entropy, const float* g_top, const float* stats, const float* entropy,
                             void* d_logits, void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX - (1 << 20) || top_k < 0 || top_k > kMaxTop || top_k > V)
    return (int)cudaErrorInvalidValue;
  LpBwdArgs a{logits, targets, top_tokens, g_logprobs, g_entropy, g_top, stats, entropy, d_logits,
              rows, ld, ignore_index, (int)V, top_k, 1, 0};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return launch_bwd<float>(a, st);
    case kBF16: return launch_bwd<__nv_bfloat16>(a, st);
    case kF16: return launch_bwd<__half>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}
