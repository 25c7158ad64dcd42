// Operators over a paged KV cache that the caller holds: the step plan, the
// append of normalised and rotated keys, page means, and attention on CUDA
// cores (every type, float32 caches in particular).
//
// A cache is pages of P positions: value d of position r of page p, KV head g
// is at p * page_stride + g * head_stride + r * token_stride + d. A request's
// table maps its logical page t / P to a page of the pool. Entries outside
// [0, num_pages) stand for no page: their positions are not attended and
// nothing is written there, whatever a table holds.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "tma.cuh"

namespace tcu {

typedef __nv_bfloat16 bf16;

// Division of t < 2^31 by a run-time constant d: floor(t / d) =
// (t * m) >> 32 >> s with m = ceil(2^(32 + s) / d), s = ceil(log2 d), where m
// needs 33 bits; the missing top bit is the "+ t" (the usual round-up method).
struct FastDiv {
  uint32_t d, m, s;
  __host__ static FastDiv of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    const uint64_t m = ((1ull << 32) * ((1ull << s) - d)) / d + 1;
    return FastDiv{d, (uint32_t)m, s};
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t t) const {
#ifdef __CUDA_ARCH__
    const uint32_t h = __umulhi(t, m);
#else
    const uint32_t h = (uint32_t)(((uint64_t)t * m) >> 32);
#endif
    return (uint32_t)(((uint64_t)h + t) >> s);
  }
};

struct PagedView {
  void* k;
  void* v;
  int num_pages, P, kvh, hd;
  int64_t sp, sh, st;  // strides of a page, a head, a position, in values
  FastDiv divP;
};

// Values of a row, four at a time, as float32.
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const bf16* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
}

// One rounding (to nearest even) to the stored type.
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(bf16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__half* p, float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// ---------------------------------------------------------------------------
// The step plan.
//
//   have_i = ceil(held_i / P), pages_i = ceil((held_i + fresh_i) / P)
//   start_i = sum of the earlier fresh, taken_i = sum of the earlier pages - have
//   table_i[have_i + j] = free[taken_i + j]
//   token start_i + j: position held_i + j, slot = table_i[pos / P] * P + pos % P
//
// Requests are planned in order up to the first that does not fit (tokens,
// free pages or table width) or whose counts are negative. All arithmetic is
// on integers, so every CTA scans the n requests for itself (two L2 reads
// each) and the step needs one launch and no communication: CTA c then fills
// the tokens [c * tile, (c + 1) * tile) and CTA 0 the per-request outputs.
struct PlanArgs {
  int n, P, width, n_free, capacity;
  const int *held, *fresh;
  int* tables;
  int64_t table_stride;
  const int* free_pages;
  int *starts, *lengths, *positions;
  int64_t* slots;
  int* counts;
  FastDiv divP;
};

constexpr int PLAN_THREADS = 256;
constexpr int PLAN_TILE = 1024;  // tokens a CTA fills

struct PlanSum {
  long long tok, pg;
};

__global__ void __launch_bounds__(PLAN_THREADS) k_plan_step(PlanArgs a) {
  __shared__ PlanSum wsum[PLAN_THREADS / 32];
  __shared__ int s_start[PLAN_THREADS + 1], s_page[PLAN_THREADS], s_held[PLAN_THREADS];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t_lo = (long long)blockIdx.x * PLAN_TILE, t_hi = min((long long)a.capacity, t_lo + PLAN_TILE);
  long long tok0 = 0, pg0 = 0;  // totals of the requests before this tile
  int planned = 0;
  bool open = true;
  for (int i0 = 0; i0 < a.n && open; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    int held = 0, fresh = 0;
    bool bad = false;
    long long have = 0, pages = 0;
    if (i < a.n) {
      held = a.held[i];
      fresh = a.fresh[i];
      bad = held < 0 || fresh < 0 || (long long)held + fresh > 0x7fffffffll;
      if (!bad) {
        have = ((long long)held + a.P - 1) / a.P;
        pages = ((long long)held + fresh + a.P - 1) / a.P;
        bad = pages > a.width;
      }
    }
    // Inclusive sums of this tile.
    long long ct = bad ? 0 : fresh, cp = bad ? 0 : pages - have;
    const int need = (int)cp;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, ct, o), v = __shfl_up_sync(0xffffffffu, cp, o);
      if (lane >= o) {
        ct += u;
        cp += v;
      }
    }
    if (tid == 0) s_bad = PLAN_THREADS;
    if (lane == 31) wsum[warp] = PlanSum{ct, cp};
    __syncthreads();
    for (int w = 0; w < warp; w++) {
      ct += wsum[w].tok;
      cp += wsum[w].pg;
    }
    bad = bad || tok0 + ct > a.capacity || pg0 + cp > a.n_free;
    if (i < a.n && bad) atomicMin(&s_bad, tid);
    __syncthreads();
    const int good = min(s_bad, min(PLAN_THREADS, a.n - i0));  // requests of this tile that are planned
    const bool mine = tid < good;
    const int start = (int)(tok0 + ct) - (mine ? fresh : 0);
    const int page0 = (int)(pg0 + cp) - need;
    if (mine) {
      s_start[tid] = start;
      s_page[tid] = page0;
      s_held[tid] = held;
    }
    if (mine && tid == good - 1) s_start[good] = start + fresh;
    if (blockIdx.x == 0 && i < a.n) {
      if (mine) {
        a.starts[i] = start;
        a.lengths[i] = held + fresh;
      } else {
        a.lengths[i] = held;
      }
    }
    if (blockIdx.x == 0 && mine)
      for (int j = 0; j < need; j++) a.tables[(int64_t)i * a.table_stride + have + j] = a.free_pages[page0 + j];
    __syncthreads();
    // This CTA's tokens among the tile's.
    if (good > 0) {
      const long long lo = max(t_lo, (long long)s_start[0]), hi = min(t_hi, (long long)s_start[good]);
      for (long long t = lo + tid; t < hi; t += PLAN_THREADS) {
        int l = 0, r = good - 1;  // the last request that starts at or before t (empty ones in front of it lose)
        while (l < r) {
          const int m = (l + r + 1) >> 1;
          if (s_start[m] <= (int)t) l = m; else r = m - 1;
        }
        const int h = s_held[l], pos = h + (int)t - s_start[l];
        const int first_new = (int)(((long long)h + a.P - 1) / a.P), page = (int)a.divP.div(pos);
        // Pages this step adds come from the free list: the table may not be written yet.
        const int id = page >= first_new ? a.free_pages[s_page[l] + page - first_new] : a.tables[(int64_t)(i0 + l) * a.table_stride + page];
        a.positions[t] = pos;
        a.slots[t] = id < 0 ? -1 : (int64_t)id * a.P + (pos - page * a.P);
      }
      const int last = good - 1;
      // Totals after the tile's planned requests.
      if (tid == last) wsum[0] = PlanSum{tok0 + ct, pg0 + cp};
      __syncthreads();
      tok0 = wsum[0].tok;
      pg0 = wsum[0].pg;
    }
    planned += good;
    open = good == PLAN_THREADS;
    __syncthreads();
  }
  if (blockIdx.x == 0) {
    // Requests from the first that did not fit on.
    for (int i = planned + tid; i <= a.n; i += PLAN_THREADS) {
      a.starts[i] = (int)tok0;
      if (i < a.n) a.lengths[i] = a.held[i];
    }
    if (tid == 0) {
      a.counts[0] = planned;
      a.counts[1] = (int)tok0;
      a.counts[2] = (int)pg0;
    }
  }
  for (long long t = max(t_lo, tok0) + tid; t < t_hi; t += PLAN_THREADS) {
    a.positions[t] = -1;
    a.slots[t] = -1;
  }
}

// ---------------------------------------------------------------------------
// Append: q and k normalised per head and rotated, q to its output, k and v
// to the cache, in one pass.
//
//   rms:   y = x / sqrt(mean x^2 + eps) * w
//   layer: y = (x - mean) / sqrt(mean (x - mean)^2 + eps) * w
//   pair (a, b) of rotary pair i at position p, (c, s) = table[p][i]:
//          a' = a c - b s, b' = b c + a s
//   split halves: a = y[i], b = y[i + pairs]; adjacent: a = y[2i], b = y[2i + 1].
//
// Float32 throughout, rounded once when stored. LPH lanes share one head of
// one token, four values a lane and chunk; the partner of a rotary pair comes
// from shared memory. Bytes bound it: each value is read and written once.
enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

struct AppendArgs {
  int T, H, KVH, hd;
  const void* qkv;
  int64_t qkv_stride;
  const int* positions;
  const int64_t* slots;
  const float2* table;
  int max_positions, pairs, adjacent;
  int norm;
  float eps;
  const float *qw, *kw;
  int64_t w_stride;  // hd, or 0 when the heads share their weights
  void* q_out;
  int64_t q_stride;
  PagedView kv;
};

constexpr int APPEND_THREADS = 256;

template <typename TQ, typename TK, int LPH, int CH>
__global__ void __launch_bounds__(APPEND_THREADS) k_append(AppendArgs a) {
  constexpr int GROUPS = APPEND_THREADS / LPH;
  __shared__ __align__(16) float stage[GROUPS][LPH * CH * 4 + 4];
  const int grp = threadIdx.x / LPH, lane = threadIdx.x % LPH;
  const int heads = a.H + 2 * a.KVH;
  const int64_t item = (int64_t)blockIdx.x * GROUPS + grp;
  const int t = (int)(item / heads), h = (int)(item % heads);
  int pos = -1;
  int64_t slot = -1;
  if (t < a.T) {
    pos = a.positions[t];
    slot = a.slots[t];
  }
  // Padding, and positions or slots outside the table and the pool: nothing is written.
  const bool live = slot >= 0 && slot < (int64_t)a.kv.num_pages * a.kv.P && pos >= 0 && (a.pairs == 0 || pos < a.max_positions);
  const bool rot = h < a.H + a.KVH;
  float x[CH][4];
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int d = (c * LPH + lane) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && d < a.hd) v = load4(reinterpret_cast<const TQ*>(a.qkv) + (int64_t)t * a.qkv_stride + (int64_t)h * a.hd + d);
    x[c][0] = v.x;
    x[c][1] = v.y;
    x[c][2] = v.z;
    x[c][3] = v.w;
  }
  if (a.norm != NORM_NONE) {
    const float inv = 1.f / (float)a.hd;
    float mean = 0.f;
    if (a.norm == NORM_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < CH; c++) s += (x[c][0] + x[c][1]) + (x[c][2] + x[c][3]);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      mean = s * inv;
    }
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        if ((c * LPH + lane) * 4 + j < a.hd) s = fmaf(x[c][j] - mean, x[c][j] - mean, s);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (rot) {
      const float r = rsqrtf(fmaf(s, inv, a.eps));
      const float* w = h < a.H ? a.qw + h * a.w_stride : a.kw + (h - a.H) * a.w_stride;
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int d = (c * LPH + lane) * 4;
        if (d < a.hd) {
          const float4 wv = *reinterpret_cast<const float4*>(w + d);
          x[c][0] = (x[c][0] - mean) * r * wv.x;
          x[c][1] = (x[c][1] - mean) * r * wv.y;
          x[c][2] = (x[c][2] - mean) * r * wv.z;
          x[c][3] = (x[c][3] - mean) * r * wv.w;
        }
      }
    }
  }
  if (a.pairs > 0) {
    float* st = stage[grp];
#pragma unroll
    for (int c = 0; c < CH; c++) *reinterpret_cast<float4*>(st + (c * LPH + lane) * 4) = make_float4(x[c][0], x[c][1], x[c][2], x[c][3]);
    __syncwarp();
    if (live && rot) {
      const float2* tab = a.table + (int64_t)pos * a.pairs;
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int d = (c * LPH + lane) * 4 + j;
          if (d < 2 * a.pairs) {
            const bool second = a.adjacent ? (d & 1) : d >= a.pairs;
            const int i = a.adjacent ? d >> 1 : (second ? d - a.pairs : d);
            const float2 cs = tab[i];
            const float other = st[a.adjacent ? d ^ 1 : (second ? d - a.pairs : d + a.pairs)];
            x[c][j] = second ? fmaf(x[c][j], cs.x, other * cs.y) : fmaf(x[c][j], cs.x, -(other * cs.y));
          }
        }
    }
  }
  if (!live) return;
  const int64_t page = slot / a.kv.P, row = slot - page * a.kv.P;
  const int g = h < a.H + a.KVH ? h - a.H : h - a.H - a.KVH;
  const int64_t off = page * a.kv.sp + (int64_t)g * a.kv.sh + row * a.kv.st;
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int d = (c * LPH + lane) * 4;
    if (d >= a.hd) continue;
    const float4 v = make_float4(x[c][0], x[c][1], x[c][2], x[c][3]);
    if (h < a.H)
      store4(reinterpret_cast<TQ*>(a.q_out) + (int64_t)t * a.q_stride + (int64_t)h * a.hd + d, v);
    else
      store4(reinterpret_cast<TK*>(rot ? a.kv.k : a.kv.v) + off + d, v);
  }
}

// ---------------------------------------------------------------------------
// Page means: for every slot that is the last of its page, the mean key of
// the page for each KV head (float32 sum in position order of each lane's
// rows, rounded once). One warp takes 32 slots and one KV head.
struct MeansArgs {
  int T;
  const int64_t* slots;
  void* means;  // [num_pages][kvh][hd]
  PagedView kv;
};

template <typename TK>
__global__ void __launch_bounds__(128) k_page_means(MeansArgs a) {
  const int warp = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int g = blockIdx.y, P = a.kv.P;
  const int64_t t = (int64_t)warp * 32 + lane;
  int64_t slot = t < a.T ? a.slots[t] : -1;
  if (slot >= (int64_t)a.kv.num_pages * P) slot = -1;
  const int64_t my_page = slot < 0 ? -1 : slot / P;
  uint32_t todo = __ballot_sync(0xffffffffu, slot >= 0 && slot - my_page * P == P - 1);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t page = __shfl_sync(0xffffffffu, my_page, src);
    const TK* base = reinterpret_cast<const TK*>(a.kv.k) + page * a.kv.sp + (int64_t)g * a.kv.sh;
    TK* out = reinterpret_cast<TK*>(a.means) + (page * a.kv.kvh + g) * a.kv.hd;
    for (int d0 = 0; d0 < a.kv.hd; d0 += 128) {
      const int d = d0 + lane * 4;
      if (d >= a.kv.hd) continue;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < P; r++) {
        const float4 v = load4(base + (int64_t)r * a.kv.st + d);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const float n = (float)P;
      store4(out + d, make_float4(s.x / n, s.y / n, s.z / n, s.w / n));
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.
//
// Query j of request i (rows starts[i] + j of q) is at position
// lengths[i] - (starts[i + 1] - starts[i]) + j and attends to the positions
// up to its own. A "row" is one query and one of the G = H / KVH query heads
// of a KV head. The history is cut into parts handled by separate CTAs; each
// leaves (sum_t 2^(s_t - m) v_t, m, sum_t 2^(s_t - m)) of its rows, with s in
// units of log2 (the scale carries log2 e), and k_attend_join adds the parts
// up in part order. A row that sees nothing leaves m = -inf and l = 0 and its
// output is zero.
struct AttendArgs {
  int n, T, H, KVH, G, hd, max_fresh;
  const void* q;
  int64_t q_ts, q_hs;
  void* out;
  int64_t o_ts, o_hs;
  const int *starts, *lengths, *tables;
  int64_t table_stride;
  int width;          // entries of a table
  const int* prefix;  // pages all requests share, logical pages [0, prefix_pages)
  int prefix_pages;
  int max_length;     // positions from here on are not attended
  float scale;        // scale * log2 e
  PagedView kv;
  // Parts: [T * H rows][slots], the prefix's first, then the request's own.
  float* part_o;   // [row][slot][hd]
  float2* part_ml; // [row][slot] (m, l)
  int slots, prefix_slots;
  int prefix_chunk, own_chunk;  // positions per part
  // Sparse: the pages each (query, KV head) reads (ascending, -1 behind them).
  const int* pages;  // [T][KVH][budget]
  int budget;
};

struct Query {
  int token;     // row of q, -1: none
  int request;
  int pos;       // its position
};

// Query j of request i.
__device__ __forceinline__ Query query_at(const AttendArgs& a, int i, int j) {
  const int s = a.starts[i], fresh = a.starts[i + 1] - s;
  const int token = s + j;
  if (j >= fresh || s < 0 || token >= a.T) return Query{-1, i, -1};
  return Query{token, i, min(a.lengths[i] - fresh + j, a.max_length - 1)};
}

// The request of row `token` of q: the last i with starts[i] <= token.
__device__ __forceinline__ Query query_of(const AttendArgs& a, int token) {
  if (token >= a.T || token >= a.starts[a.n] || token < a.starts[0]) return Query{-1, 0, -1};
  int l = 0, r = a.n - 1;
  if (token < a.n && a.starts[token] == token && a.starts[token + 1] == token + 1) l = r = token;  // one token each
  while (l < r) {
    const int m = (l + r + 1) >> 1;
    if (a.starts[m] <= token) l = m; else r = m - 1;
  }
  const int fresh = a.starts[l + 1] - a.starts[l];
  const int j = token - a.starts[l];
  if (j >= a.max_fresh || j >= fresh) return Query{-1, l, -1};
  return Query{token, l, min(a.lengths[l] - fresh + j, a.max_length - 1)};
}

// Where position index u of a part's history lies: offset of the row in the
// cache, and its position t. Negative page ids and ids past the pool give -1.
enum { SRC_PREFIX = 0, SRC_OWN = 1, SRC_LIST = 2 };

template <int SRC>
__device__ __forceinline__ int64_t source_at(const AttendArgs& a, const int* ids, const int* table, int u, int& t) {
  const int b = (int)a.kv.divP.div(u), r = u - b * a.kv.P;
  int id;
  if (SRC == SRC_LIST) {
    const int j = b < a.budget ? ids[b] : -1;
    if (j < 0 || j >= a.width) {
      t = 0x7fffffff;
      return -1;
    }
    t = j * a.kv.P + r;
    id = table[j];
  } else {
    t = u;
    if (SRC == SRC_OWN && b >= a.width) return -1;
    id = ids[b];
  }
  if (id < 0 || id >= a.kv.num_pages) return -1;
  return (int64_t)id * a.kv.sp + (int64_t)r * a.kv.st;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / l, 0 for a row that saw nothing; NaN stays NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

// CUDA-core parts. A warp holds four groups of eight lanes; a group takes
// every fourth position of its warp's share and keeps a softmax state of its
// own for each of R rows, so that nothing is exchanged until the end: dot
// products need three shuffles, the running sums none. The groups' states
// are joined through shared memory in a fixed order.
//
// grid: x = request * row tiles + row tile (own history: rows of a request;
// list: rows of a query, x counts queries; prefix: x = row tile of all rows),
// y = KV head, z = part.
constexpr int CC_WARPS = 4;
constexpr int CC_GROUPS = CC_WARPS * 4;

template <typename TQ, typename TK, int NCH, int R, int SRC>
__global__ void __launch_bounds__(CC_WARPS * 32) k_attend_cc(AttendArgs a, int row_tiles) {
  extern __shared__ __align__(16) float cc_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int grp = lane >> 3, l8 = lane & 7;
  const int g = blockIdx.y, part = blockIdx.z;
  const int hd = a.hd;
  // Rows of this CTA: (query, head) pairs r0 .. r0 + R - 1 of the row space.
  int limit[R], row_out[R];  // last position seen; token * H + head, or -1
  int request = 0, token0 = -1, most = -1;
  const int tile = SRC == SRC_PREFIX ? blockIdx.x : blockIdx.x % row_tiles;
  if (SRC != SRC_PREFIX) request = blockIdx.x / row_tiles;
  const TQ* qp[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int row = tile * R + r;
    Query q;
    int hh;
    if (SRC == SRC_PREFIX) {
      q = query_of(a, row / a.G);
      hh = row % a.G;
    } else if (SRC == SRC_OWN) {
      q = row / a.G < a.max_fresh ? query_at(a, request, row / a.G) : Query{-1, request, -1};
      hh = row % a.G;
    } else {  // "request" counts (request, query) pairs here
      q = query_at(a, request / a.max_fresh, request % a.max_fresh);
      if (row >= a.G) q.token = -1;
      hh = row;
    }
    limit[r] = q.token < 0 ? -1 : q.pos;
    row_out[r] = q.token < 0 ? -1 : q.token * a.H + g * a.G + hh;
    qp[r] = q.token < 0 ? nullptr : reinterpret_cast<const TQ*>(a.q) + (int64_t)q.token * a.q_ts + (int64_t)(g * a.G + hh) * a.q_hs;
    if (q.token >= 0) {
      token0 = q.token;
      most = max(most, q.pos);
    }
  }
  if (token0 < 0) return;
  const int prefix_end = a.prefix_pages * a.kv.P;
  int u0, u1;
  const int* ids;
  const int* table = nullptr;
  if (SRC == SRC_PREFIX) {
    u0 = part * a.prefix_chunk;
    u1 = min(min(u0 + a.prefix_chunk, prefix_end), most + 1);
    ids = a.prefix;
  } else if (SRC == SRC_OWN) {
    u0 = prefix_end + part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, most + 1);
    ids = a.tables + (int64_t)request * a.table_stride;
  } else {
    u0 = part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, a.budget * a.kv.P);
    ids = a.pages + ((int64_t)token0 * a.KVH + g) * a.budget;
    table = a.tables + (int64_t)(request / a.max_fresh) * a.table_stride;
  }
  if (SRC == SRC_OWN && u0 >= u1 && !(part == 0 && a.slots == 1)) return;  // k_attend_join counts the parts by the same rule

  float q[R][NCH][4], o[R][NCH][4], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int d = (c * 8 + l8) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (qp[r] && d < hd) v = load4(qp[r] + d);
      q[r][c][0] = v.x * a.scale;
      q[r][c][1] = v.y * a.scale;
      q[r][c][2] = v.z * a.scale;
      q[r][c][3] = v.w * a.scale;
#pragma unroll
      for (int j = 0; j < 4; j++) o[r][c][j] = 0.f;
    }
  }
  const TK* kb = reinterpret_cast<const TK*>(a.kv.k) + (int64_t)g * a.kv.sh;
  const TK* vb = reinterpret_cast<const TK*>(a.kv.v) + (int64_t)g * a.kv.sh;
  constexpr int U = 2;  // positions of a group per round
  for (int u = u0 + warp * 4 + grp; u - grp < u1; u += CC_GROUPS * U) {
    float4 kx[U][NCH], vx[U][NCH];
    int t[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int ui = u + i * CC_GROUPS;
      t[i] = 0x7fffffff;
      int64_t off = -1;
      if (ui < u1) off = source_at<SRC>(a, ids, table, ui, t[i]);
      if (off < 0) t[i] = 0x7fffffff;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int d = (c * 8 + l8) * 4;
        // Positions no row sees are not read: whatever lies there stays out.
        const bool on = t[i] <= most && d < hd;
        kx[i][c] = on ? load4(kb + off + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        vx[i][c] = on ? load4(vb + off + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      float s[U];
#pragma unroll
      for (int i = 0; i < U; i++) {
        float d = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
          d = fmaf(q[r][c][0], kx[i][c].x, d);
          d = fmaf(q[r][c][1], kx[i][c].y, d);
          d = fmaf(q[r][c][2], kx[i][c].z, d);
          d = fmaf(q[r][c][3], kx[i][c].w, d);
        }
        s[i] = d;
      }
#pragma unroll
      for (int i = 0; i < U; i++) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 4);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
        if (t[i] > limit[r]) s[i] = -INFINITY;
      }
      float mx = m[r];
#pragma unroll
      for (int i = 0; i < U; i++) mx = fmaxf(mx, s[i]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      const float alpha = ex2(m[r] - ref);
      float p[U], add = 0.f;
#pragma unroll
      for (int i = 0; i < U; i++) {
        p[i] = ex2(s[i] - ref);
        add += p[i];
      }
      m[r] = mx;
      l[r] = fmaf(l[r], alpha, add);
#pragma unroll
      for (int c = 0; c < NCH; c++) {
#pragma unroll
        for (int j = 0; j < 4; j++) o[r][c][j] *= alpha;
#pragma unroll
        for (int i = 0; i < U; i++) {
          o[r][c][0] = fmaf(p[i], vx[i][c].x, o[r][c][0]);
          o[r][c][1] = fmaf(p[i], vx[i][c].y, o[r][c][1]);
          o[r][c][2] = fmaf(p[i], vx[i][c].z, o[r][c][2]);
          o[r][c][3] = fmaf(p[i], vx[i][c].w, o[r][c][3]);
        }
      }
    }
  }
  // Join the sixteen groups' states, one row at a time.
  const int width = NCH * 32;
  float* so = cc_smem;                       // [16][width]
  float* sml = cc_smem + CC_GROUPS * width;  // [16][2]
  const int gi = warp * 4 + grp;
#pragma unroll
  for (int r = 0; r < R; r++) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NCH; c++) *reinterpret_cast<float4*>(so + gi * width + (c * 8 + l8) * 4) = make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]);
    if (l8 == 0) {
      sml[2 * gi] = m[r];
      sml[2 * gi + 1] = l[r];
    }
    __syncthreads();
    if (row_out[r] < 0) continue;  // the same for every thread
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < CC_GROUPS; i++) mx = fmaxf(mx, sml[2 * i]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float w[CC_GROUPS], ls = 0.f;
#pragma unroll
    for (int i = 0; i < CC_GROUPS; i++) {
      w[i] = ex2(sml[2 * i] - ref);
      ls = fmaf(sml[2 * i + 1], w[i], ls);
    }
    const int64_t slot = (int64_t)row_out[r] * a.slots + (SRC == SRC_OWN ? a.prefix_slots : 0) + part;
    const bool direct = a.slots == 1;  // the only part: the output itself
    const float inv = inverse_sum(ls);
    TQ* out = reinterpret_cast<TQ*>(a.out) + (int64_t)(row_out[r] / a.H) * a.o_ts + (int64_t)(row_out[r] % a.H) * a.o_hs;
    for (int d = threadIdx.x; d < hd; d += CC_WARPS * 32) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < CC_GROUPS; i++) s = fmaf(so[i * width + d], w[i], s);
      if (direct)
        store_as(out + d, s * inv);
      else
        a.part_o[slot * hd + d] = s;
    }
    if (threadIdx.x == 0 && !direct) a.part_ml[slot] = make_float2(mx, ls);
  }
}

// Parts of a row with its last position pos: the prefix's, then its own.
__device__ __forceinline__ int own_parts(const AttendArgs& a, int pos) {
  const int n = pos + 1 - a.prefix_pages * a.kv.P;
  return n <= 0 ? 0 : (n + a.own_chunk - 1) / a.own_chunk;
}

// Adds up the parts of one row (warp per row): out = sum_j w_j o_j / sum_j w_j
// l_j with w_j = 2^(m_j - max m), in part order. grid: x = request * max_fresh
// + query, y = heads / 4. Positions of one request may use different numbers
// of parts; the request's largest position decides which were written.
template <typename TQ, int LIST>
__global__ void __launch_bounds__(128) k_attend_join(AttendArgs a) {
  const int i = blockIdx.x / a.max_fresh, j = blockIdx.x % a.max_fresh;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.H) return;
  const Query q = query_at(a, i, j);
  if (q.token < 0) return;
  const int np = a.prefix_slots, no = LIST ? a.slots : own_parts(a, q.pos);
  const int64_t row = (int64_t)q.token * a.H + h;
  const float2* ml = a.part_ml + row * a.slots;
  const int parts = LIST ? no : np + no;
  float mx = -INFINITY;
  for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, ml[p].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  for (int p = 0; p < parts; p++) l = fmaf(ml[p].y, ex2(ml[p].x - ref), l);
  const float inv = inverse_sum(l);
  TQ* out = reinterpret_cast<TQ*>(a.out) + (int64_t)q.token * a.o_ts + (int64_t)h * a.o_hs;
  const float* po = a.part_o + row * a.slots * a.hd;
  for (int d = lane; d < a.hd; d += 32) {
    float s = 0.f;
    for (int p = 0; p < parts; p++) s = fmaf(po[(int64_t)p * a.hd + d], ex2(ml[p].x - ref), s);
    store_as(out + d, s * inv);
  }
}

// ---------------------------------------------------------------------------
// Page choice of sparse attention.
//
// score(b) = max over the KV head's query heads h of q_h . mean_b, in float64:
// products of the stored types are exact and the sum is good to 2^-52 of its
// terms, so the order of pages does not depend on how the sum was taken.
// Candidates: first <= b < npages - last; a key orders them (NaN lowest).
struct ChooseArgs {
  int first, last, top;
  const void* means;       // [num_pages][KVH][hd]
  unsigned long long* keys;  // [T][KVH][width]
  int width;
  int* pages;              // [T][KVH][budget]
};

__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(s == s)) return 1ull;
  s += 0.0;  // -0 and +0 are one value
  const unsigned long long u = (unsigned long long)__double_as_longlong(s);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// grid: x = request * max_fresh + query, y = KV head, z = 64-page tile; eight
// lanes a page.
template <typename TQ, typename TK>
__global__ void __launch_bounds__(128) k_page_scores(AttendArgs a, ChooseArgs c) {
  extern __shared__ double qs[];  // [G][hd]
  const Query q = query_at(a, blockIdx.x / a.max_fresh, blockIdx.x % a.max_fresh);
  if (q.token < 0 || q.pos < 0) return;
  const int g = blockIdx.y, hd = a.hd;
  const int npages = q.pos / a.kv.P + 1;
  const int lo = max(c.first, (int)blockIdx.z * 64), hi = min(min(npages - c.last, c.width), (int)blockIdx.z * 64 + 64);
  if (lo >= hi) return;
  for (int e = threadIdx.x; e < a.G * hd; e += 128) {
    const int h = e / hd, d = e % hd;
    qs[e] = (double)(float)(reinterpret_cast<const TQ*>(a.q)[(int64_t)q.token * a.q_ts + (int64_t)(g * a.G + h) * a.q_hs + d]);
  }
  __syncthreads();
  const int* table = a.tables + (int64_t)q.request * a.table_stride;
  const int l8 = threadIdx.x & 7;
  for (int b0 = blockIdx.z * 64; b0 < (int)blockIdx.z * 64 + 64; b0 += 16) {
    const int b = b0 + (threadIdx.x >> 3);
    const int id = b >= lo && b < hi ? table[b] : -1;
    const bool on = id >= 0 && id < a.kv.num_pages;
    const TK* mp = reinterpret_cast<const TK*>(c.means) + ((int64_t)(on ? id : 0) * a.KVH + g) * hd;
    double best = 0.0;
    for (int h = 0; h < a.G; h++) {
      double s = 0.0;
      for (int d = l8 * 4; d < hd; d += 32) {
        const float4 v = on ? load4(mp + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        const double* x = qs + h * hd + d;
        s = fma(x[0], (double)v.x, s);
        s = fma(x[1], (double)v.y, s);
        s = fma(x[2], (double)v.z, s);
        s = fma(x[3], (double)v.w, s);
      }
      s += __shfl_xor_sync(0xffffffffu, s, 4);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      // The largest of the heads; a NaN makes the page NaN.
      best = h == 0 || s > best || !(s == s) ? (h > 0 && !(best == best) ? best : s) : best;
    }
    if (l8 == 0 && b >= lo && b < hi) c.keys[((int64_t)q.token * a.KVH + g) * c.width + b] = on ? score_key(best) : 0ull;
  }
}

// One CTA per (query, KV head): the key of the top-th candidate by radix
// selection (eight bits a pass, histograms in shared memory), then the chosen
// pages in ascending order; candidates equal to that key are taken from the
// lowest page on. grid: x = request * max_fresh + query, y = KV head.
constexpr int CHOOSE_THREADS = 256;

__global__ void __launch_bounds__(CHOOSE_THREADS) k_page_choose(AttendArgs a, ChooseArgs c) {
  __shared__ int hist[256];
  __shared__ int wsum[CHOOSE_THREADS / 32], wtie[CHOOSE_THREADS / 32];
  __shared__ unsigned long long s_prefix;
  __shared__ int s_want;
  const Query q = query_at(a, blockIdx.x / a.max_fresh, blockIdx.x % a.max_fresh);
  if (q.token < 0) return;
  const int g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* out = c.pages + ((int64_t)q.token * a.KVH + g) * a.budget;
  const int npages = q.pos < 0 ? 0 : min(q.pos / a.kv.P + 1, c.width);
  const int lo = min(c.first, npages), hi = max(lo, npages - c.last);
  const unsigned long long* keys = c.keys + ((int64_t)q.token * a.KVH + g) * c.width;
  unsigned long long thr = 0;  // every candidate with a larger key is taken
  int ties = 0;                // and this many with this key
  if (hi - lo <= c.top) {
    ties = hi - lo;  // all: the keys do not matter
  } else if (c.top > 0) {
    unsigned long long prefix = 0;
    int want = c.top;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int e = tid; e < 256; e += CHOOSE_THREADS) hist[e] = 0;
      __syncthreads();
      for (int b = lo + tid; b < hi; b += CHOOSE_THREADS) {
        const unsigned long long k = keys[b];
        if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, left = want;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        s_prefix = prefix | ((unsigned long long)d << shift);
        s_want = left;
      }
      __syncthreads();
      prefix = s_prefix;
      want = s_want;
    }
    thr = prefix;
    ties = want;
  }
  const bool all = hi - lo <= c.top;
  int done = 0, tied = 0;  // pages written, ties seen
  for (int b0 = 0; b0 < npages; b0 += CHOOSE_THREADS) {
    const int b = b0 + tid;
    const bool inside = b >= lo && b < hi;
    const unsigned long long k = inside && !all ? keys[b] : 0;
    const bool tie = inside && !all && c.top > 0 && k == thr;
    const uint32_t tb = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) wtie[warp] = __popc(tb);
    __syncthreads();
    int before = tied + __popc(tb & ((1u << lane) - 1));
    int tie_total = 0;
    for (int w = 0; w < CHOOSE_THREADS / 32; w++) {
      if (w < warp) before += wtie[w];
      tie_total += wtie[w];
    }
    const bool take = b < npages && (!inside || all || (c.top > 0 && k > thr) || (tie && before < ties));
    const uint32_t kb = __ballot_sync(0xffffffffu, take);
    if (lane == 0) wsum[warp] = __popc(kb);
    __syncthreads();
    int at = done + __popc(kb & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < CHOOSE_THREADS / 32; w++) {
      if (w < warp) at += wsum[w];
      total += wsum[w];
    }
    if (take && at < a.budget) out[at] = b;
    done += total;
    tied += tie_total;
    __syncthreads();
  }
  for (int e = done + tid; e < a.budget; e += CHOOSE_THREADS) out[e] = -1;
}

}  // namespace tcu
