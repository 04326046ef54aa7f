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
// The call is bound by its bytes (each input read, each output written once), so it is shaped like a
// copy: one unit of work a thread, no loop, no shared memory, few registers, the data on its way
// before the token's place is looked up. A unit is two vectors (of 16 bytes where everything is
// aligned) of one head: V pairs of a rotated head, or what is copied as it is. At 40 registers 12 blocks
// of 128 threads are resident. 8 contexts of 3392 tokens, 16 + 8 heads of 128, take 70 us (6.3 TB/s, 98%
// of the measured copy rate). With hardware divisions it was 78 us, bound by instruction issue; threads
// that kept the angles for several heads or tokens took 79 to 114 us, for want of loads in flight.
// ---------------------------------------------------------------------------------------------
constexpr int kAppendThreads = 128;

// Division of numbers below 2^31 by a fixed one: n / d = n m >> (31 + s) with s = ceil(log2 d) and
// m = ceil(2^(31 + s) / d), since then m d - 2^(31 + s) < d <= 2^s and n (m d - 2^(31 + s)) < 2^(31 + s).
struct FastDiv {
  uint32_t d, m, s;
  __host__ void set(uint32_t div) {
    d = div;
    s = 0;
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ int quot(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> (31 + s)); }
};

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out, *k_cache, *v_cache;
  const int32_t *table, *starts, *counts;
  const float *cos, *sin;
  uint32_t* status;
  int token0, tokens;             // the launch's tokens, of B * T
  FastDiv by_units, by_T, by_rot, by_v, by_page;
  int T, Hq, Hkv, D, half, interleaved, page_size, n_pages, table_width, rope_rows;
  int units, units_rot, units_v;  // of a token; of a head of q or k; of a head of v
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
__device__ __forceinline__ Chunk<T, V> chunk_load_once(const T* p) {
  if constexpr (V * sizeof(T) == 16) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    return *reinterpret_cast<Chunk<T, V>*>(&u);
  } else {
    return chunk_load<T, V>(p);
  }
}

// Turns V pairs: (x1[i], x2[i]), or the neighbours among the 2 V values of x1, x2.
template <typename T, int V, bool PAIRS>
__device__ __forceinline__ void turn(Chunk<T, V>& c1, Chunk<T, V>& c2, const float* c, const float* s) {
  float x[2 * V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    x[i] = to_f32(c1.v[i]);
    x[V + i] = to_f32(c2.v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = PAIRS ? 2 * i : i, ib = PAIRS ? 2 * i + 1 : V + i;
    const T ra = from_f32<T>(x[ia] * c[i] - x[ib] * s[i]), rb = from_f32<T>(x[ib] * c[i] + x[ia] * s[i]);
    (ia < V ? c1.v[ia % V] : c2.v[ia % V]) = ra;
    (ib < V ? c1.v[ib % V] : c2.v[ib % V]) = rb;
  }
}

template <typename T, int V, bool PAIRS>
__global__ void __launch_bounds__(kAppendThreads, 12) append_kernel(const AppendArgs a) {
  const int idx = blockIdx.x * kAppendThreads + threadIdx.x;
  const int local = a.by_units.quot(idx);
  if (local >= a.tokens) return;
  int u = idx - local * a.units;
  const int token = a.token0 + local, b = a.by_T.quot(token), t = token - b * a.T;
  const bool live = a.counts == nullptr || t < a.counts[b];
  const int q_units = a.Hq * a.units_rot, k_units = a.Hkv * a.units_rot;
  const int kind = u < q_units ? 0 : u < q_units + k_units ? 1 : 2;
  if (kind != 0 && !live) return;
  u -= kind == 0 ? 0 : kind == 1 ? q_units : q_units + k_units;
  const int h = kind == 2 ? a.by_v.quot(u) : a.by_rot.quot(u), e = u - h * (kind == 2 ? a.units_v : a.units_rot);
  // the unit's vectors: a rotated pair of vectors, or up to two neighbours of the rest
  const int n_pair = kind == 2 ? 0 : a.half / V;
  const bool turned = e < n_pair;
  const int rest = (kind == 2 ? 0 : 2 * a.half) + (e - n_pair) * 2 * V;
  const int o1 = turned ? (PAIRS ? 2 * e * V : e * V) : rest;
  const int o2 = turned ? (PAIRS ? o1 + V : a.half + e * V) : rest + V;
  const bool two = turned || o2 < a.D;
  const T* src = kind == 0   ? (const T*)a.q + b * a.q_sb + t * a.q_st + h * a.q_sh
                 : kind == 1 ? (const T*)a.k + b * a.k_sb + t * a.k_st + h * a.k_sh
                             : (const T*)a.v + b * a.v_sb + t * a.v_st + h * a.v_sh;
  Chunk<T, V> c1 = chunk_load_once<T, V>(src + o1), c2;
  if (two) c2 = chunk_load_once<T, V>(src + o2);
  const int64_t pos = (int64_t)a.starts[b] + t;
  int64_t row = pos;
  bool stored = live;
  if (a.half > 0 && (pos < 0 || pos >= a.rope_rows)) {
    // padding behind the count takes the tables' nearest row; a live token must have its own
    if (live) set_status(a.status, kBadArgument, kSiteAppendRope);
    stored = false;
    row = pos < 0 ? 0 : a.rope_rows - 1;
  }
  T* dst;
  if (kind == 0) {
    dst = (T*)a.q_out + ((int64_t)token * a.Hq + h) * a.D;
  } else {
    if (!stored) return;
    if (pos < 0 || pos >= (int64_t)a.table_width * a.page_size) {
      set_status(a.status, kBadArgument, kSiteAppendPos);
      return;
    }
    const int w = pos <= INT_MAX ? a.by_page.quot((int)pos) : (int)(pos / a.page_size);
    const int slot = (int)(pos - (int64_t)w * a.page_size);
    const int page = a.table[(int64_t)b * a.t_sb + w];
    if (page < 0 || page >= a.n_pages) {
      set_status(a.status, kBadArgument, kSiteAppendPage);
      return;
    }
    dst = kind == 1 ? (T*)a.k_cache + page * a.kc_sp + slot * a.kc_ss + h * a.kc_sh
                    : (T*)a.v_cache + page * a.vc_sp + slot * a.vc_ss + h * a.vc_sh;
  }
  if (turned) {
    const float *cos = a.cos + row * a.half + e * V, *sin = a.sin + row * a.half + e * V;
    float cs[V], sn[V];
#pragma unroll
    for (int k = 0; k < V; k += (V % 4 == 0 ? 4 : 1)) {
      if constexpr (V % 4 == 0) {
        *reinterpret_cast<float4*>(cs + k) = __ldg(reinterpret_cast<const float4*>(cos + k));
        *reinterpret_cast<float4*>(sn + k) = __ldg(reinterpret_cast<const float4*>(sin + k));
      } else {
        cs[k] = __ldg(cos + k);
        sn[k] = __ldg(sin + k);
      }
    }
    turn<T, V, PAIRS>(c1, c2, cs, sn);
  }
  chunk_store<T, V>(dst + o1, c1);
  if (two) chunk_store<T, V>(dst + o2, c2);
}

// ---------------------------------------------------------------------------------------------
// Attention of one query per sequence and head over the sequence's cached tokens:
//   z_j = scale q . k_j,  out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  m = max_j z_j;
// a sequence of length 0 gives a row of zeros.
//
// Work split. The work is the list of (sequence, unit, tile of 16 tokens) in that order, a unit
// being one key head with a block of its query heads. The kernel's CTAs divide the list into runs that
// do not care where sequences end, so a batch of ragged lengths is as balanced as one long sequence,
// with no knowledge of the lengths on the host: each CTA finds its first sequence with a warp scan over
// the lengths. A (sequence, unit) covered by one CTA is finished there; where several CTAs share it,
// each leaves its running maximum, sum and unnormalised fp32 output in a slot of the workspace (at
// most two slots a CTA: its first and its last run), and attn_join_kernel combines them in the
// order of the list, so results do not depend on timing.
//
// Where there are many (sequence, unit) pairs, each has a CTA of its own for its first `head` tiles
// (no search, no shared rows as long as that is all), and the list holds what lies behind them.
// ---------------------------------------------------------------------------------------------
constexpr int kTile = 16;
constexpr int kAttnWarps = 4;
// Resident CTAs an SM of the tensor-core kernel, by its registers.
__host__ __device__ constexpr int attn_ctas(int D, int NG) { return NG > 1 ? 2 : D <= 64 ? 4 : 3; }

struct AttnArgs {
  const void *q, *k_cache, *v_cache;
  void* out;
  const int32_t *table, *lengths;
  float *ws_o, *ws_ml;  // [2 * (mains + ctas)][rows][D] and [2 * (mains + ctas)][rows][2]
  uint32_t* status;
  int B, Hq, Hkv, D, G;        // G = Hq / Hkv query heads per key head
  int rows, subs, units;       // query heads a unit covers; units per key head; units per sequence
  int mains, head;             // CTAs that each have the first `head` tiles of a (sequence, unit), or 0, 0
  int ctas, big, min_tiles;    // CTAs that divide the list, and how many of them take the larger runs
  float share;                 // of the list that those take
  int cap;                     // tokens that a row of the table has room for
  int page_size, n_pages, table_width;
  int64_t q_sb, q_sh, o_sb, o_sh, kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh, t_sb;
  float scale_log2;            // scale * log2(e): exponentials are taken to base 2
};

__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) {
  int n = a.lengths[b];
  if (n < 0 || n > a.cap) {
    set_status(a.status, kBadArgument, kSiteAttnLen);
    n = n < 0 ? 0 : a.cap;
  }
  return n;
}
__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
// Tiles of a sequence that are in the list.
__device__ __forceinline__ int listed_tiles(const AttnArgs& a, int len) { return max(0, tiles_of(len) - a.head); }

// The list's division (positions fit 31 bits: the host sees to it): the first `big` CTAs take `per`
// tiles each, the others, which start as those end, `small` tiles. SMs do not run at one speed (the
// first CTAs of one long sequence ended between 50 and 82 us), so the small runs fill what is left.
struct Division {
  int per, small, big;
  __device__ __forceinline__ Division(const AttnArgs& a, int total) {
    big = a.big;
    const int rest = a.ctas - a.big;
    if (rest == 0) {
      per = max(a.min_tiles, (int)(((uint32_t)total + a.ctas - 1) / (uint32_t)a.ctas));
      small = 1;
    } else {
      per = max(a.min_tiles, (int)((float)total * a.share / (float)big) + 1);
      const int left = total - (int)min((int64_t)total, (int64_t)per * big);
      small = max(a.min_tiles, (int)(((uint32_t)left + rest - 1) / (uint32_t)rest));
    }
  }
  __device__ __forceinline__ int64_t begin(int c) const {
    return c < big ? (int64_t)c * per : (int64_t)big * per + (int64_t)(c - big) * small;
  }
  __device__ __forceinline__ int size(int c) const { return c < big ? per : small; }
  __device__ __forceinline__ int cta_of(int pos) const {
    const int64_t edge = (int64_t)big * per;
    return pos < edge ? (int)((uint32_t)pos / (uint32_t)per) : big + (int)((uint32_t)(pos - edge) / (uint32_t)small);
  }
};

// Where a CTA's run begins: the sequence that holds its first position, that sequence's length and the
// listed tiles before it; false where the list ends before. Warp-collective; the lengths of up to 128
// sequences are read once, of more twice.
struct Start { int pos, size, total, b, len, before; };
__device__ __forceinline__ bool find_start(const AttnArgs& a, int cta, Start& st) {
  constexpr int kHeld = 4;
  const int lane = threadIdx.x & 31;
  int held[kHeld];
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = 32 * i + lane < a.B ? seq_len(a, 32 * i + lane) : 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) all += listed_tiles(a, held[i]);
  for (int s = 32 * kHeld + lane; s < a.B; s += 32) all += listed_tiles(a, seq_len(a, s));
  st.total = (int)__reduce_add_sync(0xffffffffu, all) * a.units;
  const Division div(a, st.total);
  const int64_t pos = div.begin(cta);
  if (pos >= st.total) return false;
  st.pos = (int)pos;
  st.size = min(div.size(cta), st.total - st.pos);
  int done = 0;
#pragma unroll 1
  for (int base = 0; base < a.B; base += 32) {
    int len = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) len = base == 32 * i ? held[i] : len;
    if (base >= 32 * kHeld) len = base + lane < a.B ? seq_len(a, base + lane) : 0;
    const int mine = listed_tiles(a, len);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    incl += done;
    const uint32_t hit = __ballot_sync(0xffffffffu, st.pos < incl * a.units);
    if (hit) {
      const int s = __ffs(hit) - 1;
      st.b = base + s;
      st.len = __shfl_sync(0xffffffffu, len, s);
      st.before = __shfl_sync(0xffffffffu, incl - mine, s);
      return true;
    }
    done = __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// A CTA's run of the list, one (sequence, unit) at a time: the fields describe the current part.
struct Parts {
  int b, kvh, row0, rows;  // sequence, key head, first query head and number of query heads
  int tile0, tile1, len;
  int slot;                // workspace slot, or -1: the CTA covers all of the unit and finishes its rows
  int unit, tiles;         // tiles: of the sequence, in the list
  int left;                // tiles of the run behind this part

  __device__ __forceinline__ void set_heads(const AttnArgs& a) {
    kvh = unit / a.subs;
    const int sub = unit - kvh * a.subs;
    row0 = kvh * a.G + sub * a.rows;
    rows = min(a.rows, a.G - sub * a.rows);
  }
  __device__ __forceinline__ void set(const AttnArgs& a, int tile, int free_slot) {
    set_heads(a);
    const int n = min(tiles - tile, left);
    tile0 = a.head + tile;
    tile1 = tile0 + n;
    left -= n;
    // all of the listed tiles: the unit is finished, or (its head being elsewhere) has a slot by its number
    slot = n < tiles ? a.mains + free_slot : a.head == 0 ? -1 : a.mains + 2 * a.ctas + b * a.units + unit;
  }
  // False: the CTA has nothing to do. (All warps of the CTA compute the same.)
  __device__ __forceinline__ bool first(const AttnArgs& a) {
    if ((int)blockIdx.x < a.mains) {
      b = blockIdx.x / a.units;
      unit = blockIdx.x - b * a.units;
      set_heads(a);
      len = seq_len(a, b);
      left = tile0 = 0;
      tile1 = min(tiles_of(len), a.head);
      slot = tiles_of(len) > a.head ? (int)blockIdx.x : -1;
      return len > 0;
    }
    Start st;
    if (!find_start(a, blockIdx.x - a.mains, st)) return false;
    left = st.size;
    b = st.b;
    len = st.len;
    tiles = listed_tiles(a, len);
    const int off = st.pos - st.before * a.units;
    unit = (int)((uint32_t)off / (uint32_t)tiles);
    set(a, off - unit * tiles, 2 * (blockIdx.x - a.mains));
    return true;
  }
  __device__ __forceinline__ bool next(const AttnArgs& a) {
    if (left == 0) return false;
    if (++unit == a.units) {
      unit = 0;
      do {
        ++b;
        len = seq_len(a, b);
        tiles = listed_tiles(a, len);
      } while (tiles == 0);
    }
    set(a, 0, 2 * (blockIdx.x - a.mains) + 1);
    return true;
  }
};

// Rows of zeros for the empty sequences, dealt out over the CTAs.
template <typename T>
__device__ __forceinline__ void zero_empty(const AttnArgs& a) {
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (seq_len(a, b) != 0) continue;
    for (int i = threadIdx.x; i < a.Hq * a.D; i += blockDim.x) {
      const int h = i / a.D;
      ((T*)a.out)[b * a.o_sb + h * a.o_sh + (i - h * a.D)] = from_f32<T>(0.f);
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
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Parts p;
  for (bool more = p.first(a); more; more = p.next(a)) {
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
  }
  zero_empty<T>(a);
}

// Tensor-core kernel for 16-bit caches. A warp takes tiles of 16 tokens and multiplies them with
// mma.m16n8k16, the tokens and values on the 16-row side and 8 query heads on the 8-column side:
//   S^T = K Q^T    (16 tokens x 8 heads x 16 values a step),
//   O^T += V^T P^T (16 values x 8 heads x 16 tokens a step).
// The work is bound by the cache's bytes (2 Hq / Hkv products for each value read), so the small
// warp-level shape is the right one: the 128 rows of a tcgen05 tile would stay empty.
//
// K: the product does not care which value a k index stands for, so a lane's 16-byte piece of a key
// row (values 8j.. of each 32) is the A fragment of two steps, with Q held in the same order. V is
// read transposed by ldmatrix. Weights leave the S^T fragments for the P^T ones by an 8 x 8 transpose
// in registers, and each head's maximum and sum live in the lanes that hold its columns of O^T.
//
// 64 sequences of 3392 tokens, 16 query and 8 key heads of 128, take 137 us (6.45 TB/s, the measured
// copy rate); with lengths spread from 0 up 75 us (5.9 TB/s), the rest being the kernel's start, its
// tail and the join; one sequence of 131001 tokens 89 us (6.05 TB/s).
//
// The weights p = exp(z - m) would lose 8 bits (bf16) as an operand, so they go in as two: hi, p
// rounded a little low so that p - hi > 0, and the rest; one step is two products, 2^-16 of p is left,
// and an infinite value stays infinite because both parts are positive. Sums of weights use the fp32
// values. The running maximum moves only when a score passes it by more than kRoom (a factor of 2^8):
// the sums have the room, and the rescaling, with its exchange between lanes, becomes rare.
//
// fp16 has the digits (2^-20 of p) but not the range: its parts of a p below 2^-4 would be subnormal, and
// a p below 2^-25 gone from the values while it stays in the sum. So they are 2^14 p, as large as fp16
// holds with a factor of 2 left for the lazy maximum (p <= 2), and the output is scaled back. Left of p
// are 2^-20 p or 2^-39, whichever is more: the 2^17 smallest weights of a long cache add up to 2^-22.
// (An infinite value stays infinite down to p = 2^-28; below, the second part may be 0.) Scale and room cost
// nothing: 512 ragged sequences of up to 2000 tokens 298 us, as with unscaled parts and a room of 2^8.
template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static constexpr float kLow = 1.f - 0x1p-8f, kScale = 1.f, kRoom = 8.f;
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
};
template <> struct Mma<__half> {
  static constexpr float kLow = 1.f - 0x1p-10f, kScale = 0x1p14f, kRoom = 1.f;
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
};

// Asynchronous copies of 16 bytes to shared memory; off: nothing is read and zeros are stored.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ldmatrix4t(uint32_t p) {
  uint4 v;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared-memory layout of a tile: 16 rows of keys, then 16 of values, kPitch bytes each; the 16-byte
// pieces of a row are permuted by the row so that the fragment reads (two key rows by four pieces,
// eight value rows by one piece at a time) touch every bank once.
template <int D> struct Tile {
  static constexpr int kPieces = D / 8;                              // 16-byte pieces of a row
  static constexpr int kPitch = D == 32 ? 64 : D == 64 ? 128 : 256;  // D = 96: padded, the permutation needs it
  static constexpr int kV = kTile * kPitch, kStage = 2 * kV;
  static constexpr int kCopies = kTile * kPieces / 32;               // 16-byte copies a lane makes for each of K and V
  static __device__ __forceinline__ int k_at(int t, int piece) {
    return t * kPitch + ((D == 32 ? piece : piece ^ ((t & 1) << 2)) << 4);
  }
  static __device__ __forceinline__ int v_at(int t, int piece) {
    return kV + t * kPitch + ((D == 32 ? piece ^ (t >> 1 & 3) : piece ^ (t & 7)) << 4);
  }
};
// Tiles in each warp's ring.
template <int D> constexpr int ring_stages() { return D <= 64 ? 3 : 2; }
template <int D> constexpr int attn_smem() {
  return kAttnWarps * (ring_stages<D>() * Tile<D>::kStage + 4 * (D + 4) * 4) + 256;
}

// The fetching side of a warp: it walks the run on its own, the ring's depth ahead of the products and
// across the borders of parts.
template <typename T, int D, bool PAGE16>
struct TileFetch {
  using L = Tile<D>;
  static constexpr int S = ring_stages<D>();
  static constexpr int kRows = 32 / L::kPieces;  // whole rows a copy, so that pointers advance by equal steps (D = 96: 24 lanes)
  const AttnArgs& a;
  const int lane, warp;
  Parts p;
  bool more;        // p is a part with tiles left to fetch
  int next;         // next tile of it
  const T *kb, *vb; // this lane's piece of the part's key head, in page 0
  // where the tiles are: PAGE16: lane i has (page, slot) of tile first + 4 i, `have` of them left; else
  // lane i < 16 of token i of the next tile. page -1: not to be read.
  int pg, sl, have;
  uint64_t masks;   // live tokens of the tiles in the ring, 16 bits each, oldest first

  __device__ __forceinline__ TileFetch(const AttnArgs& a_, const Parts& p_, bool any)
      : a(a_), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), p(p_), more(any), masks(0) { if (any) enter(); }

  // Begins at the current part's first tile for this warp, or that of a later part.
  __device__ __forceinline__ void enter() {
    while (p.tile0 + warp >= p.tile1) {
      more = p.next(a);
      if (!more) return;
    }
    next = p.tile0 + warp;
    have = 0;
    kb = (const T*)a.k_cache + p.kvh * a.kc_sh;
    vb = (const T*)a.v_cache + p.kvh * a.vc_sh;
    kb += lane / L::kPieces * a.kc_ss + lane % L::kPieces * 8;
    vb += lane / L::kPieces * a.vc_ss + lane % L::kPieces * 8;
  }

  __device__ __forceinline__ void lookup(int tok, bool on) {
    pg = -1;
    sl = 0;
    if (on) {
      const int w = tok / a.page_size;
      sl = tok - w * a.page_size;
      pg = a.table[(int64_t)p.b * a.t_sb + w];
      if (pg < 0 || pg >= a.n_pages) {
        set_status(a.status, kBadArgument, kSiteAttnPage);
        pg = -1;
      }
    }
  }

  // Starts the warp's copies of the next tile into the ring at `stage`.
  __device__ __forceinline__ void fetch(uint32_t stage) {
    uint32_t mask = 0;
    if (more) {
      int page = 0, slot = 0;
      if constexpr (PAGE16) {
        if (have == 0) {
          const int tile = next + lane * kAttnWarps;
          lookup(tile * kTile, tile < p.tile1);
          have = 32;
        }
        page = __shfl_sync(0xffffffffu, pg, 32 - have);
        slot = __shfl_sync(0xffffffffu, sl, 32 - have);
        --have;
        mask = page < 0 ? 0u : (1u << min(kTile, p.len - next * kTile)) - 1u;
      } else {
        const int tok = next * kTile + lane;
        lookup(tok, lane < kTile && tok < p.len);
        mask = __ballot_sync(0xffffffffu, pg >= 0) & 0xFFFFu;
      }
      if (PAGE16 && mask == 0xFFFFu) {
        const T* kp = kb + (int64_t)page * a.kc_sp + (int64_t)slot * a.kc_ss;
        const T* vp = vb + (int64_t)page * a.vc_sp + (int64_t)slot * a.vc_ss;
        const int t0 = lane / L::kPieces, piece = lane % L::kPieces;
        if (32 % L::kPieces == 0 || t0 < kRows) {
#pragma unroll
          for (int t = 0; t < kTile; t += kRows) {
            cp16(stage + L::k_at(t + t0, piece), kp);
            kp += kRows * a.kc_ss;
          }
#pragma unroll
          for (int t = 0; t < kTile; t += kRows) {
            cp16(stage + L::v_at(t + t0, piece), vp);
            vp += kRows * a.vc_ss;
          }
        }
      } else {
        // (from the head's first value again)
        const T* k0 = (const T*)a.k_cache + p.kvh * a.kc_sh;
        const T* v0 = (const T*)a.v_cache + p.kvh * a.vc_sh;
#pragma unroll
        for (int i = 0; i < L::kCopies; ++i) {
          const int u = i * 32 + lane, t = u / L::kPieces, piece = u - t * L::kPieces;
          const int tp = PAGE16 ? page : __shfl_sync(0xffffffffu, pg, t);
          const int64_t ts = PAGE16 ? slot + t : __shfl_sync(0xffffffffu, sl, t);
          const bool on = mask >> t & 1;
          cp16_if(stage + L::k_at(t, piece), on ? k0 + tp * a.kc_sp + ts * a.kc_ss + piece * 8 : k0, on);
          cp16_if(stage + L::v_at(t, piece), on ? v0 + tp * a.vc_sp + ts * a.vc_ss + piece * 8 : v0, on);
        }
      }
      next += kAttnWarps;
      if (next >= p.tile1) {
        more = p.next(a);
        if (more) enter();
      }
    }
    cp_commit();
    masks = masks >> 16 | (uint64_t)mask << (16 * (S - 1));
  }
};

template <typename T, int D, int NG, bool PAGE16>
__global__ void __launch_bounds__(32 * kAttnWarps, attn_ctas(D, NG)) attn_mma_kernel(const AttnArgs a) {
  using W = TileFetch<T, D, PAGE16>;
  using L = Tile<D>;
  constexpr int KC = D / 32, MT = D / 16;
  constexpr int kPitchO = D + 4;  // floats of a row of s_o
  extern __shared__ unsigned char smem_raw[];
  __shared__ float s_m[kAttnWarps][8 * NG], s_l[kAttnWarps][8 * NG];
  // rows begin at multiples of their pitch, so that a piece's index can be xor-ed into its address
  unsigned char* smem = smem_raw + (-(uint32_t)__cvta_generic_to_shared(smem_raw) & 255u);
  static_assert(W::S <= 4, "masks");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(smem) + warp * W::S * L::kStage;
  const uint32_t ring1 = ring0 + W::S * L::kStage;
  float* s_o = reinterpret_cast<float*>(smem + kAttnWarps * W::S * L::kStage);  // [warp][4 heads][kPitchO]
  // this lane's places in a tile: key pieces of tokens r and r + 8, and its row address for ldmatrix
  const int k_lane = L::k_at(r, j);
  const int v_lane = L::v_at((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);
  uint32_t stage = ring0;
  Parts p;
  bool more = p.first(a);
  W w(a, p, more);
#pragma unroll 1
  for (int i = 0; i < W::S; ++i) w.fetch(ring0 + i * L::kStage);
  for (; more; more = p.next(a)) {
    uint4 q[NG][KC];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int row = g * 8 + r;
        q[g][c] = make_uint4(0, 0, 0, 0);
        if (row < p.rows) {
          const T* qp = (const T*)a.q + p.b * a.q_sb + (p.row0 + row) * a.q_sh + 32 * c + 8 * j;
          q[g][c] = *reinterpret_cast<const uint4*>(qp);
        }
      }
    float o[NG][MT][4];            // values 16 t + r (+ 8) of heads 2j, 2j + 1
    float m[NG][2], l[NG][2];      // of heads 2j, 2j + 1; the sum over this lane's tokens only
    float base[NG][2];             // m, or 0 while it is -inf
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      m[g][0] = m[g][1] = -INFINITY;
      base[g][0] = base[g][1] = 0.f;
      l[g][0] = l[g][1] = 0.f;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[g][t][0] = o[g][t][1] = o[g][t][2] = o[g][t][3] = 0.f;
    }
#pragma unroll 1
    for (int tile = p.tile0 + warp; tile < p.tile1; tile += kAttnWarps) {
      cp_wait<W::S - 1>();
      __syncwarp();
      const uint32_t mask = (uint32_t)w.masks & 0xFFFFu;
      float s[NG][2][4];           // two sums, so that products need not wait for one another
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][0][i] = s[g][1][i] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 x = lds16((stage + k_lane) ^ (c << 6)), y = lds16(((stage + k_lane) ^ (c << 6)) + 8 * L::kPitch);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          Mma<T>::run(s[g][0], x.x, y.x, x.y, y.y, q[g][c].x, q[g][c].y);
          Mma<T>::run(s[g][1], x.z, y.z, x.w, y.w, q[g][c].z, q[g][c].w);
        }
      }
      uint32_t hi[NG][2], lo[NG][2];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = (s[g][0][i] + s[g][1][i]) * a.scale_log2;
        if (mask != 0xFFFFu) {
#pragma unroll
          for (int i = 0; i < 4; ++i) z[i] = mask >> (r + 8 * (i >> 1)) & 1 ? z[i] : -INFINITY;
        }
        float mx[2] = {fmaxf(z[0], z[2]), fmaxf(z[1], z[3])};
        if (__any_sync(0xffffffffu, mx[0] > m[g][0] + Mma<T>::kRoom || mx[1] > m[g][1] + Mma<T>::kRoom)) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], x));
            const float mn = fmaxf(m[g][n], mx[n]), alpha = ex2(m[g][n] - max_or_zero(mn));
            m[g][n] = mn;
            base[g][n] = max_or_zero(mn);
            l[g][n] *= alpha;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              o[g][t][n] *= alpha;
              o[g][t][n + 2] *= alpha;
            }
          }
        }
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = ex2(z[i] - base[g][i & 1]);
        l[g][0] += e[0] + e[2];
        l[g][1] += e[1] + e[3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr float kScale = Mma<T>::kScale, kHi = Mma<T>::kLow * kScale;
          const uint32_t x = Mma<T>::pack(e[2 * h] * kHi, e[2 * h + 1] * kHi);
          const float2 f = Mma<T>::unpack(x);
          hi[g][h] = transpose8x8(x);
          lo[g][h] = transpose8x8(Mma<T>::pack(fmaf(e[2 * h], kScale, -f.x), fmaf(e[2 * h + 1], kScale, -f.y)));
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const uint4 x = ldmatrix4t((stage + v_lane) ^ (t << 5));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          Mma<T>::run(o[g][t], x.x, x.y, x.z, x.w, hi[g][0], hi[g][1]);
          Mma<T>::run(o[g][t], x.x, x.y, x.z, x.w, lo[g][0], lo[g][1]);
        }
      }
      __syncwarp();  // every lane has read the tile
      w.fetch(stage);
      stage = stage + L::kStage == ring1 ? ring0 : stage + L::kStage;
    }
    // the warps' results, joined in order, 4 heads at a time
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[g][n] += __shfl_xor_sync(0xffffffffu, l[g][n], x);
        if (r == 0) {
          s_m[warp][g * 8 + 2 * j + n] = m[g][n];
          s_l[warp][g * 8 + 2 * j + n] = l[g][n];
        }
      }
#pragma unroll
    for (int h4 = 0; h4 < 2 * NG; ++h4) {
      if (4 * h4 >= p.rows) break;
      if ((j >> 1) == (h4 & 1)) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float* so = s_o + (warp * 4 + 2 * (j & 1) + n) * kPitchO + r;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            so[16 * t] = o[h4 / 2][t][n] * (1.f / Mma<T>::kScale);
            so[16 * t + 8] = o[h4 / 2][t][n + 2] * (1.f / Mma<T>::kScale);
          }
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < min(4, p.rows - 4 * h4) * (D / 4); i += blockDim.x) {
        const int gl = i / (D / 4), d = i % (D / 4) * 4, g = 4 * h4 + gl;
        float mx = -INFINITY;
#pragma unroll
        for (int y = 0; y < kAttnWarps; ++y) mx = fmaxf(mx, s_m[y][g]);
        float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < kAttnWarps; ++y) {
          const float e = ex2(s_m[y][g] - max_or_zero(mx));
          const float4 x = *reinterpret_cast<const float4*>(s_o + (y * 4 + gl) * kPitchO + d);
          sum += s_l[y][g] * e;
          acc[0] += x.x * e; acc[1] += x.y * e; acc[2] += x.z * e; acc[3] += x.w * e;
        }
        if (p.slot < 0) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          T* op = (T*)a.out + p.b * a.o_sb + (p.row0 + g) * a.o_sh + d;
          const uint2 y = make_uint2(Mma<T>::pack(acc[0] * inv, acc[1] * inv), Mma<T>::pack(acc[2] * inv, acc[3] * inv));
          *reinterpret_cast<uint2*>(op) = y;
        } else {
          const int64_t rr = (int64_t)p.slot * a.rows + g;
          *reinterpret_cast<float4*>(a.ws_o + rr * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          if (d == 0) {
            a.ws_ml[2 * rr] = mx;
            a.ws_ml[2 * rr + 1] = sum;
          }
        }
      }
      __syncthreads();
    }
  }
  zero_empty<T>(a);
}

// Combines the parts of each (sequence, query head) that several CTAs share, in list order. One block
// of NT threads per sequence and query head; threads take the parts' rows, VEC values each, in as many
// interleaved sums as the block has room for. Each thread's first rows are on their way before the
// weights of the parts (up to NT at once) are known.
template <typename T, int VEC, int NT>
__global__ void __launch_bounds__(NT) attn_join_kernel(const AttnArgs a) {
  constexpr int kAhead = 4, kWarps = NT / 32;
  __shared__ float s_w[NT];
  __shared__ float s_red[2][kWarps];
  __shared__ alignas(16) float s_acc[NT * VEC];
  const int b = blockIdx.x / a.Hq, h = blockIdx.x - b * a.Hq;
  const int kvh = h / a.G, sub = (h - kvh * a.G) / a.rows, g = h - kvh * a.G - sub * a.rows;
  const int tiles = listed_tiles(a, seq_len(a, b));
  int c0 = 0, c1 = 0, first = 0;
  if (tiles > 0) {
    uint32_t sum_before = 0, sum_all = 0;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < a.B; i += 32) {
      const int t = listed_tiles(a, seq_len(a, i));
      sum_all += t;
      sum_before += i < b ? t : 0;
    }
    const int total = (int)__reduce_add_sync(0xffffffffu, sum_all) * a.units;
    const Division div(a, total);
    const int s0 = (int)__reduce_add_sync(0xffffffffu, sum_before) * a.units + (kvh * a.subs + sub) * tiles;
    c0 = div.cta_of(s0);
    c1 = div.cta_of(s0 + tiles - 1);
    // the first CTA has the rows in its last slot unless its run starts there
    first = 2 * c0 + (div.begin(c0) < s0 ? 1 : 0);
  }
  // launched while the main kernel still runs; its parts are complete behind this point
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tiles == 0 || (a.head == 0 && c0 == c1)) return;  // finished by the one CTA that had it, or empty
  const int heads = a.head > 0 ? 1 : 0, pair = b * a.units + kvh * a.subs + sub;  // parts in front of the list's
  auto row_of = [&](int i) {
    const int slot = i < heads              ? pair
                     : heads == 1 && c0 == c1 ? a.mains + 2 * a.ctas + pair
                                              : a.mains + (i == heads ? first : 2 * (c0 + i - heads));
    return (int64_t)slot * a.rows + g;
  };
  const int n = heads + c1 - c0 + 1;
  const int lanes = (a.D + VEC - 1) / VEC, warp = threadIdx.x >> 5;
  const int nway = lanes >= NT ? 1 : NT / lanes;
  const int way = threadIdx.x / lanes, d = (threadIdx.x - way * lanes) * VEC;
  const bool on = way < nway;
  float m = -INFINITY, sum = 0.f, acc[VEC], more = 0.f;  // more: VEC = 1 and a head wider than the block
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  auto add = [&](const float (&x)[VEC], float f) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] += x[e] * f;
  };
  auto get = [&](int i, float (&x)[VEC]) {
    const float* src = a.ws_o + row_of(i) * a.D + d;
    if constexpr (VEC == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src);
    else x[0] = *src;
  };
  for (int i0 = 0; i0 < n; i0 += NT) {
    const int k = min(NT, n - i0);
    float x[kAhead][VEC];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (on && way + u * nway < k) get(i0 + way + u * nway, x[u]);
    const int64_t r = row_of(i0 + min((int)threadIdx.x, k - 1));
    const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * r);
    const float pm = (int)threadIdx.x < k ? ml.x : -INFINITY, pl = (int)threadIdx.x < k ? ml.y : 0.f;
    const float wm = warp_max(pm);
    if ((threadIdx.x & 31) == 0) s_red[0][warp] = wm;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mn = fmaxf(mn, s_red[0][w]);
    const float alpha = exp2f(m - max_or_zero(mn)), w = exp2f(pm - max_or_zero(mn));
    m = mn;
    s_w[threadIdx.x] = w;
    const float wl = warp_sum(pl * w);
    if ((threadIdx.x & 31) == 0) s_red[1][warp] = wl;
    __syncthreads();
    sum *= alpha;
#pragma unroll
    for (int y = 0; y < kWarps; ++y) sum += s_red[1][y];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= alpha;
    more *= alpha;
    if (on) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (way + u * nway < k) add(x[u], s_w[way + u * nway]);
#pragma unroll 4
      for (int i = way + kAhead * nway; i < k; i += nway) {
        get(i0 + i, x[0]);
        add(x[0], s_w[i]);
      }
      if (VEC == 1 && d + NT < a.D)
        for (int i = 0; i < k; ++i) more += a.ws_o[row_of(i0 + i) * a.D + d + NT] * s_w[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) s_acc[threadIdx.x * VEC + e] = acc[e];
  __syncthreads();
  if (way != 0 || d >= a.D) return;
  T* out = (T*)a.out + b * a.o_sb + h * a.o_sh;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float y = acc[e];
    for (int w = 1; w < nway; ++w) y += s_acc[w * lanes * VEC + d + e];
    out[d + e] = from_f32<T>(y * inv);
  }
  if (VEC == 1 && d + NT < a.D) out[d + NT] = from_f32<T>(more * inv);
}

}  // namespace nfb

using namespace nfb;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int V>
int launch_append(AppendArgs& a, cudaStream_t st) {
  const int rest = (a.D - 2 * a.half) / V;
  a.units_rot = a.half / V + (rest + 1) / 2;
  a.units_v = (a.D / V + 1) / 2;
  const int64_t units = (int64_t)(a.Hq + a.Hkv) * a.units_rot + (int64_t)a.Hkv * a.units_v;
  if (units > INT_MAX / 2) return (int)cudaErrorInvalidValue;
  a.units = (int)units;
  a.by_units.set((uint32_t)units);
  a.by_T.set((uint32_t)a.T);
  a.by_rot.set((uint32_t)a.units_rot);
  a.by_v.set((uint32_t)a.units_v);
  a.by_page.set((uint32_t)a.page_size);
  // thread numbers are kept below 2^31: more tokens take more launches
  const int all = a.tokens, most = (int)((INT_MAX - kAppendThreads) / units);
  for (a.token0 = 0; a.token0 < all; a.token0 += a.tokens) {
    a.tokens = all - a.token0 < most ? all - a.token0 : most;
    const unsigned blocks = (unsigned)(((int64_t)a.tokens * units + kAppendThreads - 1) / kAppendThreads);
    if (a.interleaved) append_kernel<T, V, true><<<blocks, kAppendThreads, 0, st>>>(a);
    else append_kernel<T, V, false><<<blocks, kAppendThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    if (a.token0 > INT_MAX - a.tokens) break;
  }
  return 0;
}

template <typename T, int DP>
int launch_plain(const AttnArgs& a, cudaStream_t st) {
  if (a.rows == 1) attn_plain_kernel<T, DP, 1><<<a.mains + a.ctas, 32 * kAttnWarps, 0, st>>>(a);
  else attn_plain_kernel<T, DP, 4><<<a.mains + a.ctas, 32 * kAttnWarps, 0, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int D, int NG, bool PAGE16>
int launch_mma_one(const AttnArgs& a, cudaStream_t st) {
  constexpr int kSmem = attn_smem<D>();
  static uint64_t ready = 0;  // one bit per device (an attribute set twice does no harm)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(attn_mma_kernel<T, D, NG, PAGE16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess && dev < 64) ready |= 1ull << dev;
  }
  if (e != cudaSuccess) return (int)e;
  attn_mma_kernel<T, D, NG, PAGE16><<<a.mains + a.ctas, 32 * kAttnWarps, kSmem, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int D>
int launch_mma(const AttnArgs& a, cudaStream_t st) {
  const bool p16 = a.page_size % kTile == 0;
  if (a.rows <= 8) return p16 ? launch_mma_one<T, D, 1, true>(a, st) : launch_mma_one<T, D, 1, false>(a, st);
  return p16 ? launch_mma_one<T, D, 2, true>(a, st) : launch_mma_one<T, D, 2, false>(a, st);
}

template <typename T, int VEC, int NT>
int launch_join(const AttnArgs& a, cudaStream_t st) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hq));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, attn_join_kernel<T, VEC, NT>, a);
}

template <typename T>
int launch_attn(const AttnArgs& a, bool mma, cudaStream_t st) {
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (mma) {
      switch (a.D) {
        case 32: rc = launch_mma<T, 32>(a, st); break;
        case 64: rc = launch_mma<T, 64>(a, st); break;
        case 96: rc = launch_mma<T, 96>(a, st); break;
        default: rc = launch_mma<T, 128>(a, st); break;
      }
    }
  }
  if (!mma) {
    if (a.D <= 64) rc = launch_plain<T, 2>(a, st);
    else if (a.D <= 128) rc = launch_plain<T, 4>(a, st);
    else rc = launch_plain<T, 8>(a, st);
  }
  if (rc != 0 || a.ctas == 0 || (a.mains == 0 && a.ctas == 1)) return rc;  // nothing to join
  // (the second threshold: one long sequence has tens of parts a head)
  const bool vec = a.D % 4 == 0 && aligned16(a.ws_o), wide = a.ctas >= 16 * (int64_t)a.B * a.units;
  if (vec) return wide ? launch_join<T, 4, 512>(a, st) : launch_join<T, 4, 128>(a, st);
  return launch_join<T, 1, 128>(a, st);
}

// The split of a call into units and CTAs; false where positions of the list would not fit 31 bits.
// Many (sequence, unit) pairs: one CTA for each with up to 8192 tokens, the list for the rest (512 ragged
// sequences of up to 2000: 295 us, 7.1 TB/s, divided 366 us; 256 of up to 3000: 227 us against 263 us; one
// of 60000 among 255 of up to 1000: 145 us against 137 us). The same for short caches, up to 48 tiles a
// sequence, however few (400 tokens, 8 sequences of 8 key heads of 128: 7.7 us, divided 9.8 us; but 1000
// tokens, 4 sequences: 12.5 us, divided 9.8 us). Else the list is divided over as many CTAs as the GPU
// holds; where there is much work for each of them, they take 80% of it and as many smaller runs follow
// (64 ragged sequences of up to 3392: 75 us against 84; all of 3392: 138 us against 139; 16 of 6000, 8
// heads of 96: 62 us against 69).
bool plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t capacity, bool mma, int sms, AttnArgs& a) {
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.G = (int)(Hq / Hkv);
  if (mma) {
    a.subs = (a.G + 15) / 16;
    a.rows = (a.G + a.subs - 1) / a.subs;
  } else {
    a.rows = a.G == 1 ? 1 : 4;
    a.subs = (a.G + a.rows - 1) / a.rows;
  }
  a.units = a.Hkv * a.subs;
  a.cap = (int)(capacity < INT_MAX - 2 * kTile ? capacity : INT_MAX - 2 * kTile);
  const int64_t pairs = B * a.units, per_seq = (a.cap + kTile - 1) / kTile;
  const int64_t slots = (int64_t)sms * (mma ? attn_ctas(a.D, a.rows <= 8 ? 1 : 2) : 4);
  constexpr int kHead = 512;
  a.min_tiles = kAttnWarps;
  a.share = 0.f;
  a.mains = a.head = 0;
  const bool few_tiles = per_seq <= 48;
  if (few_tiles || (pairs >= 4 * slots && (per_seq <= kHead || pairs * a.rows * (D + 2) * 8 <= (64 << 20)))) {
    a.mains = (int)pairs;
    a.head = few_tiles ? 48 : kHead;
    a.ctas = a.big = per_seq <= a.head ? 0 : (int)slots;
    return pairs <= INT_MAX - slots && (a.ctas == 0 || per_seq * pairs <= INT_MAX);
  }
  if (per_seq * pairs > INT_MAX) return false;
  const int64_t want = (pairs * per_seq + a.min_tiles - 1) / a.min_tiles;
  if (want >= 2 * slots && pairs * per_seq >= 96 * slots) {
    a.big = (int)slots;
    a.ctas = (int)(2 * slots);
    a.share = 0.8f;
  } else {
    a.ctas = a.big = (int)(want < 1 ? 1 : want < slots ? want : slots);
  }
  return true;
}

int64_t ws_floats(const AttnArgs& a) { return a.ctas == 0 ? 0 : 2 * ((int64_t)a.mains + a.ctas) * a.rows * (a.D + 2); }

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
  if (B * a.T > INT_MAX) return (int)cudaErrorInvalidValue;
  a.tokens = (int)(B * a.T);
  if (a.tokens == 0 || a.D == 0 || a.Hkv == 0) return 0;
  if (2 * a.half > a.D || a.page_size < 1 || (a.half > 0 && (a.rope_rows < 1 || !cos || !sin)))
    return (int)cudaErrorInvalidValue;
  // 16-byte vectors where every row, and every half of a rotated one, begins on 16 bytes
  const int V = dtype == kF32 ? 4 : 8;
  bool vec = a.D % V == 0 && a.half % V == 0 && aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache) &&
             (!q || (aligned16(q) && aligned16(q_out))) && (a.half == 0 || (aligned16(cos) && aligned16(sin)));
  for (int i = q ? 11 : 14; i < 26; ++i) vec = vec && dims[i] % V == 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return vec ? launch_append<float, 16 / sizeof(float)>(a, st) : launch_append<float, 1>(a, st);
    case kBF16: return vec ? launch_append<__nv_bfloat16, 16 / sizeof(__nv_bfloat16)>(a, st) : launch_append<__nv_bfloat16, 1>(a, st);
    case kF16: return vec ? launch_append<__half, 16 / sizeof(__half)>(a, st) : launch_append<__half, 1>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}

NFB_API int64_t nfb_paged_attn_ws(int mma, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t capacity) {
  if (B < 1 || Hq < 1 || Hkv < 1 || D < 1) return 0;  // nothing to launch (and a division by no heads below)
  AttnArgs a;
  return plan(B, Hq, Hkv, D, capacity, mma != 0, nfb_num_sms(), a) ? ws_floats(a) : -1;
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
  // the tensor-core kernel reads 16-byte pieces of rows of 16-bit values
  bool mma = dtype != kF32 && (D == 32 || D == 64 || D == 96 || D == 128) && aligned16(q) && aligned16(k_cache) &&
             aligned16(v_cache) && aligned16(ws) && dims[9] % 4 == 0 && dims[10] % 4 == 0 &&
             (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  const int piece[] = {7, 8, 11, 12, 13, 14, 15, 16};
  for (int i : piece) mma = mma && dims[i] % 8 == 0;
  if (!plan(B, Hq, Hkv, D, dims[4] * dims[6], mma, nfb_num_sms(), a)) return (int)cudaErrorInvalidValue;
  a.page_size = (int)dims[4]; a.n_pages = (int)dims[5]; a.table_width = (int)dims[6];
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.out = out; a.table = table; a.lengths = lengths;
  a.ws_o = ws;
  a.ws_ml = ws + 2 * ((int64_t)a.mains + a.ctas) * a.rows * D;
  a.status = status;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.q_sb = dims[7]; a.q_sh = dims[8]; a.o_sb = dims[9]; a.o_sh = dims[10];
  a.kc_sp = dims[11]; a.kc_ss = dims[12]; a.kc_sh = dims[13];
  a.vc_sp = dims[14]; a.vc_ss = dims[15]; a.vc_sh = dims[16];
  a.t_sb = dims[17];
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case kF32: return launch_attn<float>(a, mma, st);
    case kBF16: return launch_attn<__nv_bfloat16>(a, mma, st);
    case kF16: return launch_attn<__half>(a, mma, st);
  }
  return (int)cudaErrorInvalidValue;
}
