// Paged key-value cache: appending rotated keys and values, and attention of one new token per
// sequence over the pages.
//
// Cache layout: k and v pools [n_pages, page_size, Hkv, D] (the projection-native order of the
// model's attention), a table [B, W] of page ids, and a length per sequence; token p of sequence b
// lives in page table[b, p / page_size], slot p % page_size. Lengths and page ids live on the
// device, so nothing here waits for the host. Every id and position that a kernel reads from memory
// is checked before it is used as an index; a bad one sets the status word (code 3) and its access
// is skipped.
#include <climits>

#include "common.cuh"

namespace nfb {

// Sites of the status word.
enum PagedSite : uint32_t { kSiteAppendPos = 1, kSiteAppendPage = 2, kSiteAppendRope = 3, kSiteAttnLen = 4, kSiteAttnPage = 5 };

// ---------------------------------------------------------------------------------------------
// Append. A new token t of sequence b (t < counts[b]) has position p = starts[b] + t. Its key is
// rotated by p, k' = R(p) k, and k' and v are stored in the cache; its query, when given, is
// rotated the same way. R turns `half` pairs of each head's first 2 * half values by the angles of
// row p of the cos / sin tables:
//   a' = a cos - b sin,  b' = b cos + a sin,
// with (a, b) = (x[i], x[half + i]), or neighbours (x[2i], x[2i + 1]). The angles come as fp32
// tables, so far positions lose nothing to a product p * frequency in fp32; the turn is computed
// in fp32 and rounded once to the storage type.
//
// One unit of work is V pairs (two vectors) of a rotated head or one vector of what is copied as it
// is; a block of 256 threads takes the units of one token, or of several where a token has few.
// ---------------------------------------------------------------------------------------------
struct AppendArgs {
  const void *q, *k, *v;
  void *q_out, *k_cache, *v_cache;
  const int32_t *table, *starts, *counts;
  const float *cos, *sin;
  uint32_t* status;
  int64_t tokens;  // B * T
  int T, Hq, Hkv, D, half, interleaved, page_size, n_pages, table_width, rope_rows;
  int units, units_rot, tokens_per_block;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh, t_sb;
};

template <typename T, int V> struct alignas(V * sizeof(T)) Chunk { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> chunk_load(const T* p) {
  Chunk<T, V> c;
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(&c) = *reinterpret_cast<const uint4*>(p);
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) c.v[i] = p[i];
  }
  return c;
}

template <typename T, int V>
__device__ __forceinline__ void chunk_store(T* p, const Chunk<T, V>& c) {
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&c);
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = c.v[i];
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  const int local = threadIdx.x / a.units;
  const int64_t token = (int64_t)blockIdx.x * a.tokens_per_block + local;
  if (local >= a.tokens_per_block || token >= a.tokens) return;
  const int b = (int)(token / a.T), t = (int)(token - (int64_t)b * a.T);
  const bool live = a.counts == nullptr || t < a.counts[b];
  const int64_t pos = (int64_t)a.starts[b] + t;
  // where the token goes; page < 0: nowhere
  int page = -1, slot = 0;
  if (live) {
    if (pos < 0 || pos >= (int64_t)a.table_width * a.page_size) {
      set_status(a.status, kBadArgument, kSiteAppendPos);
    } else {
      page = a.table[(int64_t)b * a.t_sb + pos / a.page_size];
      slot = (int)(pos % a.page_size);
      if (page < 0 || page >= a.n_pages) {
        set_status(a.status, kBadArgument, kSiteAppendPage);
        page = -1;
      }
    }
  }
  int64_t row = pos;
  if (a.half > 0 && (row < 0 || row >= a.rope_rows)) {
    // padding behind the count takes the table's last row; a live token must have a row of its own
    if (live) {
      set_status(a.status, kBadArgument, kSiteAppendRope);
      page = -1;
    }
    row = row < 0 ? 0 : a.rope_rows - 1;
  }
  const int n_pair = a.half / V;
  const int rot_units = (a.Hq + a.Hkv) * a.units_rot;
  for (int u = a.tokens_per_block > 1 ? threadIdx.x - local * a.units : threadIdx.x; u < a.units;
       u += a.tokens_per_block > 1 ? a.units : blockDim.x) {
    const T* src;
    T* dst;
    int e;  // index of the unit within its head
    bool rot = false;
    if (u < rot_units) {
      int h = u / a.units_rot;
      e = u - h * a.units_rot;
      rot = e < n_pair;
      if (h < a.Hq) {
        src = (const T*)a.q + b * a.q_sb + t * a.q_st + h * a.q_sh;
        dst = (T*)a.q_out + (token * a.Hq + h) * a.D;
      } else {
        if (page < 0) continue;
        h -= a.Hq;
        src = (const T*)a.k + b * a.k_sb + t * a.k_st + h * a.k_sh;
        dst = (T*)a.k_cache + page * a.kc_sp + slot * a.kc_ss + h * a.kc_sh;
      }
    } else {
      if (page < 0) continue;
      const int w = u - rot_units, per = a.D / V;
      const int h = w / per;
      e = w - h * per;
      src = (const T*)a.v + b * a.v_sb + t * a.v_st + h * a.v_sh;
      dst = (T*)a.v_cache + page * a.vc_sp + slot * a.vc_ss + h * a.vc_sh;
      chunk_store<T, V>(dst + e * V, chunk_load<T, V>(src + e * V));
      continue;
    }
    if (!rot) {
      const int off = 2 * a.half + (e - n_pair) * V;
      chunk_store<T, V>(dst + off, chunk_load<T, V>(src + off));
      continue;
    }
    const int o1 = a.interleaved ? 2 * e * V : e * V;
    const int o2 = a.interleaved ? o1 + V : a.half + e * V;
    Chunk<T, V> c1 = chunk_load<T, V>(src + o1), c2 = chunk_load<T, V>(src + o2);
    const float* cs = a.cos + row * a.half + e * V;
    const float* sn = a.sin + row * a.half + e * V;
    float x[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = to_f32(c1.v[i]);
      x[V + i] = to_f32(c2.v[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : V + i;
      const float c = cs[i], s = sn[i];
      // selected by constant indices in both layouts, so x stays in registers
      const float xa = a.interleaved ? x[2 * i] : x[i], xb = a.interleaved ? x[2 * i + 1] : x[V + i];
      const T ra = from_f32<T>(xa * c - xb * s), rb = from_f32<T>(xb * c + xa * s);
      if (a.interleaved) {
        if (ia < V) c1.v[ia < V ? ia : 0] = ra; else c2.v[ia >= V ? ia - V : 0] = ra;
        if (ib < V) c1.v[ib < V ? ib : 0] = rb; else c2.v[ib >= V ? ib - V : 0] = rb;
      } else {
        c1.v[i] = ra;
        c2.v[i] = rb;
      }
    }
    chunk_store<T, V>(dst + o1, c1);
    chunk_store<T, V>(dst + o2, c2);
  }
}

// ---------------------------------------------------------------------------------------------
// Attention of one query per sequence and head over the sequence's cached tokens:
//   z_j = scale q . k_j,  out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  m = max_j z_j;
// a sequence of length 0 gives a row of zeros.
//
// Work split. The work is the list of (sequence, unit, tile of 16 tokens) in that order, a unit
// being one key head with a block of its query heads. The kernel's CTAs divide the
// list into equal runs, so a batch of ragged lengths is as balanced as one long sequence, with no
// knowledge of the lengths on the host: each CTA finds its first sequence with a warp scan over the
// lengths. A (sequence, unit) covered by one CTA is finished there; where several CTAs share it,
// each leaves its running maximum, sum and unnormalised fp32 output in a slot of the workspace (at
// most two slots a CTA: its first and its last run), and attn_join_kernel combines them in the
// order of the list, so results do not depend on timing.
// ---------------------------------------------------------------------------------------------
constexpr int kTile = 16;
constexpr int kAttnWarps = 4;

struct AttnArgs {
  const void *q, *k_cache, *v_cache;
  void* out;
  const int32_t *table, *lengths;
  float *ws_o, *ws_ml;  // [2 * ctas][rows][D] and [2 * ctas][rows][2]
  uint32_t* status;
  int B, Hq, Hkv, D, G;        // G = Hq / Hkv query heads per key head
  int rows, subs, units;       // query heads a unit covers; units per key head; units per sequence
  int ctas, min_tiles;
  int page_size, n_pages, table_width;
  int64_t q_sb, q_sh, o_sb, o_sh, kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh, t_sb;
  float scale_log2;            // scale * log2(e): exponentials are taken to base 2
};

__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) {
  const int64_t cap = min((int64_t)a.table_width * a.page_size, (int64_t)INT_MAX - 2 * kTile);
  int n = a.lengths[b];
  if (n < 0 || n > cap) {
    set_status(a.status, kBadArgument, kSiteAttnLen);
    n = n < 0 ? 0 : (int)cap;
  }
  return n;
}
__device__ __forceinline__ int seq_tiles(const AttnArgs& a, int b) { return (seq_len(a, b) + kTile - 1) / kTile; }

__device__ __forceinline__ int64_t warp_incl_scan(int64_t v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// Tiles of all sequences before `upto` (warp-collective).
__device__ __forceinline__ int64_t tiles_before(const AttnArgs& a, int upto) {
  int64_t n = 0;
  for (int b = threadIdx.x & 31; b < upto; b += 32) n += seq_tiles(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

__device__ __forceinline__ int64_t tiles_per_cta(const AttnArgs& a, int64_t all) {
  const int64_t total = all * a.units;
  return max((int64_t)a.min_tiles, (total + a.ctas - 1) / a.ctas);
}

// The sequence that holds list position pos, and the tiles before it (warp-collective).
__device__ __forceinline__ void find_seq(const AttnArgs& a, int64_t pos, int& b, int64_t& before) {
  int64_t done = 0;
  const int lane = threadIdx.x & 31;
  b = a.B;
  before = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int64_t t = base + lane < a.B ? seq_tiles(a, base + lane) : 0;
    const int64_t incl = done + warp_incl_scan(t);
    const uint32_t hit = __ballot_sync(0xffffffffu, pos < incl * a.units);
    if (hit) {
      const int l = __ffs(hit) - 1;
      b = base + l;
      before = __shfl_sync(0xffffffffu, incl - t, l);
      return;
    }
    done = __shfl_sync(0xffffffffu, incl, 31);
  }
}

// One CTA's part of one (sequence, unit).
struct Part {
  int b, kvh, row0, rows;  // sequence, key head, first query head and number of query heads
  int tile0, tile1, len;
  int slot;                // workspace slot, or -1: the CTA covers all of it and finishes the rows
};

// Walks the CTA's run of the list.
template <typename F>
__device__ __forceinline__ void for_each_part(const AttnArgs& a, F&& f) {
  const int64_t total = tiles_before(a, a.B) * a.units;
  const int64_t per = tiles_per_cta(a, total / a.units);
  int64_t pos = (int64_t)blockIdx.x * per;
  const int64_t end = min(pos + per, total);
  if (pos >= end) return;
  const int64_t first = pos;
  int b;
  int64_t before;
  find_seq(a, pos, b, before);
  int len = seq_len(a, b), tiles = (len + kTile - 1) / kTile;
  const int64_t off = pos - before * a.units;
  int unit = (int)(off / tiles), tile = (int)(off - (int64_t)unit * tiles);
  while (true) {
    const int n = (int)min((int64_t)(tiles - tile), end - pos);
    Part p;
    p.b = b;
    p.kvh = unit / a.subs;
    const int sub = unit - p.kvh * a.subs;
    p.row0 = p.kvh * a.G + sub * a.rows;
    p.rows = min(a.rows, a.G - sub * a.rows);
    p.tile0 = tile;
    p.tile1 = tile + n;
    p.len = len;
    p.slot = n == tiles ? -1 : (int)(2 * blockIdx.x + (pos == first ? 0 : 1));
    f(p);
    pos += n;
    if (pos >= end) break;
    tile = 0;
    if (++unit == a.units) {
      unit = 0;
      do {
        ++b;
        len = seq_len(a, b);
      } while (len == 0);
      tiles = (len + kTile - 1) / kTile;
    }
  }
}

// exp2 of a difference to the running maximum; a maximum of -inf (all scores -inf) stands for 0.
__device__ __forceinline__ float max_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// Plain kernel for any type, width up to 32 * DP and stride: a warp takes every fourth tile of the
// run, a lane the values lane, lane + 32, ... of a head; fp32 products and warp sums. 4 tokens are
// loaded at a time. It serves fp32 caches and what the tensor-core kernel does not tile.
template <typename T, int DP, int GC>
__global__ void __launch_bounds__(32 * kAttnWarps) attn_plain_kernel(const AttnArgs a) {
  __shared__ float s_o[kAttnWarps][GC][32 * DP];
  __shared__ float s_m[kAttnWarps][GC], s_l[kAttnWarps][GC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for_each_part(a, [&](const Part& p) {
    float q[GC][DP], o[GC][DP], m[GC], l[GC];
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int i = 0; i < DP; ++i) {
        const int d = lane + 32 * i;
        o[g][i] = 0.f;
        q[g][i] = g < p.rows && d < a.D
                      ? to_f32(((const T*)a.q)[p.b * a.q_sb + (p.row0 + g) * a.q_sh + d]) * a.scale_log2 : 0.f;
      }
    }
    const int tok1 = min(p.tile1 * kTile, p.len);
    for (int tile = p.tile0 + warp; tile < p.tile1; tile += kAttnWarps) {
#pragma unroll 1
      for (int j0 = 0; j0 < kTile; j0 += 4) {
        float kv[4][DP], vv[4][DP];
        bool ok[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = tile * kTile + j0 + j;
          ok[j] = tok < tok1;
          int page = 0, slot = 0;
          if (ok[j]) {
            page = a.table[(int64_t)p.b * a.t_sb + tok / a.page_size];
            slot = tok % a.page_size;
            if (page < 0 || page >= a.n_pages) {
              set_status(a.status, kBadArgument, kSiteAttnPage);
              ok[j] = false;
            }
          }
          const T* kp = (const T*)a.k_cache + page * a.kc_sp + slot * a.kc_ss + p.kvh * a.kc_sh;
          const T* vp = (const T*)a.v_cache + page * a.vc_sp + slot * a.vc_ss + p.kvh * a.vc_sh;
#pragma unroll
          for (int i = 0; i < DP; ++i) {
            const int d = lane + 32 * i;
            const bool in = ok[j] && d < a.D;
            kv[j][i] = in ? to_f32(kp[d]) : 0.f;
            vv[j][i] = in ? to_f32(vp[d]) : 0.f;
          }
        }
#pragma unroll
        for (int g = 0; g < GC; ++g) {
          if (g >= p.rows) break;
          float s[4];
          float mx = m[g];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float d = 0.f;
#pragma unroll
            for (int i = 0; i < DP; ++i) d = fmaf(q[g][i], kv[j][i], d);
            d = warp_sum(d);
            s[j] = ok[j] ? d : -INFINITY;
            mx = fmaxf(mx, s[j]);
          }
          const float base = max_or_zero(mx);
          const float alpha = exp2f(m[g] - base);
          m[g] = mx;
          l[g] *= alpha;
#pragma unroll
          for (int i = 0; i < DP; ++i) o[g][i] *= alpha;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = exp2f(s[j] - base);
            l[g] += e;
#pragma unroll
            for (int i = 0; i < DP; ++i) o[g][i] = fmaf(e, vv[j][i], o[g][i]);
          }
        }
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      if (lane == 0) {
        s_m[warp][g] = m[g];
        s_l[warp][g] = l[g];
      }
#pragma unroll
      for (int i = 0; i < DP; ++i) s_o[warp][g][lane + 32 * i] = o[g][i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.rows * a.D; i += blockDim.x) {
      const int g = i / a.D, d = i - g * a.D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) mx = fmaxf(mx, s_m[w][g]);
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float e = exp2f(s_m[w][g] - max_or_zero(mx));
        sum += s_l[w][g] * e;
        acc += s_o[w][g][d] * e;
      }
      if (p.slot < 0) {
        ((T*)a.out)[p.b * a.o_sb + (p.row0 + g) * a.o_sh + d] = from_f32<T>(sum == 0.f ? 0.f : acc / sum);
      } else {
        const int64_t r = (int64_t)p.slot * a.rows + g;
        a.ws_o[r * a.D + d] = acc;
        if (d == 0) {
          a.ws_ml[2 * r] = mx;
          a.ws_ml[2 * r + 1] = sum;
        }
      }
    }
    __syncthreads();
  });
}

// Combines the parts of each (sequence, query head) that several CTAs share, in list order, and
// writes the zero rows of empty sequences. One block per sequence and query head.
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
  const int b = blockIdx.x / a.Hq, h = blockIdx.x - b * a.Hq;
  const int tiles = seq_tiles(a, b);
  T* out = (T*)a.out + b * a.o_sb + h * a.o_sh;
  if (tiles == 0) {
    for (int d = threadIdx.x; d < a.D; d += blockDim.x) out[d] = from_f32<T>(0.f);
    return;
  }
  const int kvh = h / a.G, sub = (h - kvh * a.G) / a.rows, g = h - kvh * a.G - sub * a.rows;
  const int64_t before = tiles_before(a, b);
  const int64_t per = tiles_per_cta(a, before + tiles_before(a, a.B) - before);
  const int64_t s0 = before * a.units + (int64_t)(kvh * a.subs + sub) * tiles, s1 = s0 + tiles;
  const int64_t c0 = s0 / per, c1 = (s1 - 1) / per;
  if (c0 == c1) return;  // finished by the one CTA that had it
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float m = -INFINITY, sum = 0.f, acc = 0.f;
    for (int64_t c = c0; c <= c1; ++c) {
      // the first CTA has the rows in its last slot unless its run starts there
      const int64_t r = (2 * c + (c * per < s0 ? 1 : 0)) * a.rows + g;
      const float pm = a.ws_ml[2 * r], pl = a.ws_ml[2 * r + 1], po = a.ws_o[r * a.D + d];
      const float mx = fmaxf(m, pm), base = max_or_zero(mx);
      const float e0 = exp2f(m - base), e1 = exp2f(pm - base);
      sum = sum * e0 + pl * e1;
      acc = acc * e0 + po * e1;
      m = mx;
    }
    out[d] = from_f32<T>(sum == 0.f ? 0.f : acc / sum);
  }
}

}  // namespace nfb

using namespace nfb;

namespace {

template <typename T, int V>
int launch_append(AppendArgs& a, cudaStream_t st) {
  a.units_rot = a.half / V + (a.D - 2 * a.half) / V;
  const int64_t units = (int64_t)(a.Hq + a.Hkv) * a.units_rot + (int64_t)a.Hkv * (a.D / V);
  if (units > INT_MAX / 2) return (int)cudaErrorInvalidValue;
  a.units = (int)units;
  a.tokens_per_block = units >= 256 ? 1 : 256 / (int)units;
  const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > INT_MAX) return (int)cudaErrorInvalidValue;
  append_kernel<T, V><<<(unsigned)blocks, 256, 0, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int DP>
int launch_plain(const AttnArgs& a, cudaStream_t st) {
  if (a.rows == 1) attn_plain_kernel<T, DP, 1><<<a.ctas, 32 * kAttnWarps, 0, st>>>(a);
  else attn_plain_kernel<T, DP, 4><<<a.ctas, 32 * kAttnWarps, 0, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T>
int launch_attn(const AttnArgs& a, cudaStream_t st) {
  int rc;
  if (a.D <= 64) rc = launch_plain<T, 2>(a, st);
  else if (a.D <= 128) rc = launch_plain<T, 4>(a, st);
  else rc = launch_plain<T, 8>(a, st);
  if (rc != 0) return rc;
  attn_join_kernel<T><<<(unsigned)(a.B * a.Hq), 128, 0, st>>>(a);
  return (int)cudaGetLastError();
}

// The split of a call into units and CTAs; the same for the workspace query and the launch.
void plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t capacity, int sms, AttnArgs& a) {
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.G = (int)(Hq / Hkv);
  a.rows = a.G == 1 ? 1 : 4;
  a.subs = (a.G + a.rows - 1) / a.rows;
  a.units = a.Hkv * a.subs;
  a.min_tiles = kAttnWarps;
  const int64_t most = B * a.units * ((capacity + kTile - 1) / kTile);
  const int64_t want = (most + a.min_tiles - 1) / a.min_tiles;
  const int64_t slots = (int64_t)sms * 4;
  a.ctas = (int)(want < 1 ? 1 : want < slots ? want : slots);
}

}  // namespace

// dims: B, T, Hq, Hkv, D, half, interleaved, page_size, n_pages, table_width, rope_rows, then the
// strides q (b, t, h), k (b, t, h), v (b, t, h), k_cache (page, slot, head), v_cache (page, slot,
// head), table (b), all in elements.
NFB_API int nfb_append_kv(int dtype, const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                          void* v_cache, const int32_t* table, const int32_t* starts, const int32_t* counts,
                          const float* cos, const float* sin, const int64_t* dims, uint32_t* status, void* stream) {
  AppendArgs a;
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_cache = k_cache; a.v_cache = v_cache;
  a.table = table; a.starts = starts; a.counts = counts; a.cos = cos; a.sin = sin; a.status = status;
  const int64_t B = dims[0];
  for (int i = 0; i < 11; ++i)
    if (dims[i] < 0 || dims[i] > INT_MAX) return (int)cudaErrorInvalidValue;
  a.T = (int)dims[1]; a.Hq = (int)dims[2]; a.Hkv = (int)dims[3]; a.D = (int)dims[4]; a.half = (int)dims[5];
  a.interleaved = (int)dims[6]; a.page_size = (int)dims[7]; a.n_pages = (int)dims[8];
  a.table_width = (int)dims[9]; a.rope_rows = (int)dims[10];
  a.q_sb = dims[11]; a.q_st = dims[12]; a.q_sh = dims[13];
  a.k_sb = dims[14]; a.k_st = dims[15]; a.k_sh = dims[16];
  a.v_sb = dims[17]; a.v_st = dims[18]; a.v_sh = dims[19];
  a.kc_sp = dims[20]; a.kc_ss = dims[21]; a.kc_sh = dims[22];
  a.vc_sp = dims[23]; a.vc_ss = dims[24]; a.vc_sh = dims[25];
  a.t_sb = dims[26];
  a.tokens = B * a.T;
  if (a.tokens == 0 || a.D == 0 || a.Hkv == 0) return 0;
  if (2 * a.half > a.D || a.page_size < 1 || (a.half > 0 && (a.rope_rows < 1 || !cos || !sin)))
    return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return launch_append<float, 1>(a, st);
    case kBF16: return launch_append<__nv_bfloat16, 1>(a, st);
    case kF16: return launch_append<__half, 1>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}

NFB_API int64_t nfb_paged_attn_ws(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t capacity) {
  AttnArgs a;
  plan(B, Hq, Hkv, D, capacity, nfb_num_sms(), a);
  return (int64_t)2 * a.ctas * a.rows * (D + 2);
}

// dims: B, Hq, Hkv, D, page_size, n_pages, table_width, then the strides q (b, h), out (b, h),
// k_cache (page, slot, head), v_cache (page, slot, head), table (b), all in elements.
NFB_API int nfb_paged_attn(int dtype, const void* q, const void* k_cache, const void* v_cache, const int32_t* table,
                           const int32_t* lengths, void* out, float* ws, const int64_t* dims, float scale,
                           uint32_t* status, void* stream) {
  AttnArgs a;
  for (int i = 0; i < 7; ++i)
    if (dims[i] < 0 || dims[i] > INT_MAX) return (int)cudaErrorInvalidValue;
  const int64_t B = dims[0], Hq = dims[1], Hkv = dims[2], D = dims[3];
  if (B == 0 || Hq == 0) return 0;
  if (Hkv < 1 || Hq % Hkv || D < 1 || D > 256 || dims[4] < 1 || B * Hq > INT_MAX) return (int)cudaErrorInvalidValue;
  plan(B, Hq, Hkv, D, dims[4] * dims[6], nfb_num_sms(), a);
  a.page_size = (int)dims[4]; a.n_pages = (int)dims[5]; a.table_width = (int)dims[6];
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.out = out; a.table = table; a.lengths = lengths;
  a.ws_o = ws;
  a.ws_ml = ws + (int64_t)2 * a.ctas * a.rows * D;
  a.status = status;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.q_sb = dims[7]; a.q_sh = dims[8]; a.o_sb = dims[9]; a.o_sh = dims[10];
  a.kc_sp = dims[11]; a.kc_ss = dims[12]; a.kc_sh = dims[13];
  a.vc_sp = dims[14]; a.vc_ss = dims[15]; a.vc_sh = dims[16];
  a.t_sb = dims[17];
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return launch_attn<float>(a, st);
    case kBF16: return launch_attn<__nv_bfloat16>(a, st);
    case kF16: return launch_attn<__half>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}
