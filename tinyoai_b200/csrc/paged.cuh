// Operators over a paged KV cache that the caller holds: the step plan, the
// append of normalised and rotated keys, page means, page choice, and attention
// on CUDA cores (float32 caches).
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
// needs 33 bits; the missing top bit is the "+ t" (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
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
  int small;  // 1: the pool has fewer than 2^31 positions
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

__device__ __forceinline__ void unpack2(__half, uint32_t r, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ void unpack2(bf16, uint32_t r, float& lo, float& hi) {
  lo = __uint_as_float(r << 16);
  hi = __uint_as_float(r & 0xffff0000u);
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
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  store4(p, make_float4(x[0], x[1], x[2], x[3]));
  store4(p + 4, make_float4(x[4], x[5], x[6], x[7]));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
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
// the tokens [c * tile, (c + 1) * tile) and CTA 0 the per-request outputs. Where
// an output is an input's own array, one CTA does all: others could read what
// CTA 0 has written (it reads a tile of requests before it writes any of it).
// Latency bounds it, a chain of three or four L2 reads: 3.4 us for 64 decoding
// requests, 6.2 us for 1,024 with 13,312 token places (a call takes 9 us of
// the host's time from Python).
struct PlanArgs {
  int n, P, width, n_free, capacity;
  int tile;  // tokens a CTA fills
  const int *held, *fresh;
  int* tables;
  int64_t table_stride;
  const int* free_pages;
  int *starts, *lengths, *positions;
  int64_t* slots;
  int* counts;
  FastDiv divP;
};

constexpr int PLAN_TILE = 1024;

struct PlanSum {
  long long tok, pg;
};

// PLAN_THREADS: 256, or 1024 so that up to 1,024 requests are one tile (a
// tile's chain of loads, barriers and searches takes about 3 us).
template <int PLAN_THREADS>
__global__ void __launch_bounds__(PLAN_THREADS) k_plan_step(PlanArgs a) {
  pdl_wait();
  __shared__ PlanSum wsum[PLAN_THREADS / 32];
  __shared__ int s_start[PLAN_THREADS + 1], s_page[PLAN_THREADS], s_held[PLAN_THREADS];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t_lo = (long long)blockIdx.x * a.tile, t_hi = min((long long)a.capacity, t_lo + a.tile);
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
// Float32 throughout, rounded once when stored. Each value is read and written
// once. A CTA takes one token at a time and a share of its heads; LPH lanes
// hold a head, eight values each, the next token's heads already on their
// way. A lane has the same features of every head, so it keeps their cosines,
// sines and shared norm weights in registers. Instructions count here beside
// bytes (4,096 bfloat16 rows of 32 + 8 + 8 heads of 128, 103 MB: 33 us with a
// rotary pair's other value fetched from another lane and addresses taken
// anew for every token, 22.8 so, 15.7 at the copy rate): where pairs come in
// fours a lane holds both values of four pairs, two runs of four features.
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

// Eight stored values, as loaded.
template <typename T>
struct Raw8 {
  uint4 v;
  __device__ __forceinline__ void stream(const T* p) { v = ld_stream16(p); }  // read once, and not moved among other such loads
  __device__ __forceinline__ void get(float (&x)[8]) const {
    unpack2(T(), v.x, x[0], x[1]);
    unpack2(T(), v.y, x[2], x[3]);
    unpack2(T(), v.z, x[4], x[5]);
    unpack2(T(), v.w, x[6], x[7]);
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void stream(const float* p) {
    const uint4 u = ld_stream16(p), w = ld_stream16(p + 4);
    a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
    b = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};

template <typename T>
__device__ __forceinline__ void load4to(const T* p, float* x) {
  const float4 v = load4(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}

// Where a rotary pair's other value is: in the same lane, in its second run of
// four features (TURN_RUNS) or beside the first (TURN_BESIDE), or anywhere
// (TURN_SHARED: through shared memory).
enum { TURN_NONE = 0, TURN_RUNS = 1, TURN_BESIDE = 2, TURN_SHARED = 3 };

// Four stored values, as loaded.
template <typename T>
struct Raw4 {
  uint2 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint2(0, 0); }
  __device__ __forceinline__ void get(float* x) const {
    unpack2(T(), v.x, x[0], x[1]);
    unpack2(T(), v.y, x[2], x[3]);
  }
};
template <>
struct Raw4<float> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = load4(p); }
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
};

// u c + v s, both products and the sum rounded, as the sessions' own rotation
// rounds them (rope_pair in attention.cuh): a batch step that appends here
// stores the keys, binary16 ones too, that it would store there.
__device__ __forceinline__ float turned(float u, float c, float v, float s) { return __fadd_rn(__fmul_rn(u, c), __fmul_rn(v, s)); }

// grid: x = tokens x, x + gridDim.x, ...; y = share of the heads (heads_per_cta of them).
template <typename TQ, typename TK, int LPH, int TURN, int NORM>
__global__ void __launch_bounds__(APPEND_THREADS, 3) k_append(AppendArgs a, int heads_per_cta) {
  constexpr int GROUPS = APPEND_THREADS / LPH;
  constexpr int HEADS = sizeof(TQ) == 4 ? 2 : 3;  // heads of a group of lanes at a time
  __shared__ __align__(16) float stage[TURN == TURN_SHARED ? GROUPS : 1][LPH * 8 + 4];
  const int grp = threadIdx.x / LPH, lane = threadIdx.x % LPH;
  const int h0 = blockIdx.y * heads_per_cta, h1 = min(a.H + 2 * a.KVH, h0 + heads_per_cta);
  // This lane's features: four from da and four from db on.
  const bool turns = TURN == TURN_RUNS && lane < a.pairs / 4;
  const int da = turns ? lane * 4 : TURN == TURN_RUNS ? 2 * a.pairs + (lane - a.pairs / 4) * 8 : lane * 8;
  const int db = turns ? a.pairs + lane * 4 : da + 4;
  const float inv = 1.f / (float)a.hd;
  pdl_wait();
  struct Head {
    Raw4<TQ> lo, hi;
  };
  for (int hb = h0; hb < h1; hb += GROUPS * HEADS) {
    // What does not change from token to token. A lane without work has on false.
    bool on[HEADS], rot[HEADS], is_q[HEADS];
    int in_at[HEADS];       // of the row
    int64_t out_at[HEADS];  // of the query row, or of the slot's place in the cache
    TK* cache[HEADS];
    const float* weight[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
      const int h = hb + i * GROUPS + grp, g = h < a.H + a.KVH ? h - a.H : h - a.H - a.KVH;
      on[i] = h < h1 && da < a.hd;
      rot[i] = h < a.H + a.KVH;
      is_q[i] = h < a.H;
      in_at[i] = h * a.hd;
      out_at[i] = is_q[i] ? (int64_t)h * a.hd : (int64_t)g * a.kv.sh;
      cache[i] = reinterpret_cast<TK*>(rot[i] ? a.kv.k : a.kv.v);
      weight[i] = is_q[i] ? a.qw + h * a.w_stride : a.kw + g * a.w_stride;
    }
    Head coming[HEADS];
    auto fetch = [&](int t) {
      const TQ* src = reinterpret_cast<const TQ*>(a.qkv) + (int64_t)t * a.qkv_stride;
#pragma unroll
      for (int i = 0; i < HEADS; i++) {
        if (on[i]) {
          coming[i].lo.load(src + in_at[i] + da);
          coming[i].hi.load(src + in_at[i] + db);
        } else {
          coming[i].lo.zero();
          coming[i].hi.zero();
        }
      }
    };
    int t = blockIdx.x, pos_coming = a.positions[t];
    int64_t slot_coming = a.slots[t];
    fetch(t);
    for (; t < a.T; t += gridDim.x) {
      const int pos = pos_coming;
      const int64_t slot = slot_coming;
      Head raw[HEADS];
#pragma unroll
      for (int i = 0; i < HEADS; i++) raw[i] = coming[i];
      const int next = t + gridDim.x;
      if (next < a.T) {  // on its way while this token is worked on
        fetch(next);
        pos_coming = a.positions[next];
        slot_coming = a.slots[next];
      }
      // Padding, and positions or slots outside the table and the pool: nothing is written.
      const bool live = slot >= 0 && slot < (int64_t)a.kv.num_pages * a.kv.P && pos >= 0 && (TURN == TURN_NONE || pos < a.max_positions);
      if (!live) continue;
      // Cosines and sines of this lane's pairs, or (TURN_SHARED) of its features.
      float cs[8], sn[8];
      const float2* tab = a.table + (int64_t)pos * a.pairs;
      if (TURN == TURN_RUNS || TURN == TURN_BESIDE) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = lane * 4 + e;
          const float2 v = i < a.pairs ? tab[i] : make_float2(1.f, 0.f);
          cs[e] = v.x;
          sn[e] = v.y;
        }
      } else if (TURN == TURN_SHARED) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int f = da + e;
          const bool second = f >= a.pairs;
          const float2 v = f < 2 * a.pairs ? tab[second ? f - a.pairs : f] : make_float2(1.f, 0.f);
          cs[e] = v.x;
          sn[e] = second ? v.y : -v.y;
        }
      }
      const int64_t page = a.kv.small ? (int64_t)a.kv.divP.div((uint32_t)slot) : slot / a.kv.P;
      const int64_t kv_off = page * a.kv.sp + (slot - page * a.kv.P) * a.kv.st;
      TQ* q_out = reinterpret_cast<TQ*>(a.q_out) + (int64_t)t * a.q_stride;
      // Every lane takes part in the shuffles, with or without work.
#pragma unroll
      for (int i = 0; i < HEADS; i++) {
        float x[8];
        raw[i].lo.get(x);
        raw[i].hi.get(x + 4);
        if (NORM != NORM_NONE) {
          float mean = 0.f, s = 0.f;
          if (NORM == NORM_LAYER) {
            float z = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
            mean = z * inv;
            if (rot[i])
#pragma unroll
              for (int e = 0; e < 8; e++) x[e] -= mean;
          }
          if (on[i])
#pragma unroll
            for (int e = 0; e < 8; e++) s = fmaf(x[e], x[e], s);
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (rot[i] && on[i]) {
            const float r = rsqrtf(fmaf(s, inv, a.eps));
            float w[8];
            load4to(weight[i] + da, w);
            load4to(weight[i] + db, w + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * r * w[e];
          }
        }
        if (TURN == TURN_RUNS) {
          if (rot[i] && turns)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float u = x[e], v = x[4 + e];
              x[e] = turned(u, cs[e], v, -sn[e]);
              x[4 + e] = turned(v, cs[e], u, sn[e]);
            }
        } else if (TURN == TURN_BESIDE) {
          if (rot[i])
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (lane * 4 + e < a.pairs) {
                const float u = x[2 * e], v = x[2 * e + 1];
                x[2 * e] = turned(u, cs[e], v, -sn[e]);
                x[2 * e + 1] = turned(v, cs[e], u, sn[e]);
              }
        } else if (TURN == TURN_SHARED) {
          float* st = stage[grp];
          __syncwarp();
          *reinterpret_cast<float4*>(st + da) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(st + da + 4) = make_float4(x[4], x[5], x[6], x[7]);
          __syncwarp();
          if (rot[i])
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const int f = da + e;
              if (f < 2 * a.pairs) x[e] = turned(x[e], cs[e], st[f >= a.pairs ? f - a.pairs : f + a.pairs], sn[e]);
            }
        }
        if (on[i]) {
          const float4 lo = make_float4(x[0], x[1], x[2], x[3]), hi = make_float4(x[4], x[5], x[6], x[7]);
          if (is_q[i]) {
            store4(q_out + out_at[i] + da, lo);
            store4(q_out + out_at[i] + db, hi);
          } else {
            store4(cache[i] + kv_off + out_at[i] + da, lo);
            store4(cache[i] + kv_off + out_at[i] + db, hi);
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Page means: for every slot that is the last of its page, the mean key of
// the page for each KV head, float32 sums rounded once. WARPS warps take 32
// slots and one KV head: hd / 8 lanes hold a position's features, eight each,
// and the sets of lanes that fit take alternate positions, a page of 32 in
// one go. The sets' sums are added in a fixed order. One warp where there are
// slots enough to fill the GPU (16,384 of the 3B shape: 23 us, with four 32),
// four, which share each page, where there are not (256 slots: 4.9 us, with one 7.9).
struct MeansArgs {
  int T;
  const int64_t* slots;
  void* means;  // [num_pages][kvh][hd]
  PagedView kv;
};

template <typename TK, int WARPS>
__global__ void __launch_bounds__(128) k_page_means(MeansArgs a) {
  constexpr int LANES = WARPS * 32;
  __shared__ __align__(16) float sums[128][8];
  const int tid = threadIdx.x % LANES, lane = tid & 31, base_row = threadIdx.x - tid;
  const int g = blockIdx.y, P = a.kv.P, lpr = a.kv.hd / 8, sets = LANES / lpr;
  const int64_t t = ((int64_t)blockIdx.x * (128 / LANES) + threadIdx.x / LANES) * 32 + lane;
  pdl_wait();
  int64_t slot = t < a.T ? a.slots[t] : -1;
  if (slot >= (int64_t)a.kv.num_pages * P) slot = -1;
  const int my_page = slot < 0 ? -1 : (int)(slot / P);
  uint32_t todo = __ballot_sync(0xffffffffu, slot >= 0 && slot - (int64_t)my_page * P == P - 1);  // the same in all WARPS warps
  const int r0 = tid / lpr, d = (tid - r0 * lpr) * 8;
  constexpr int U = WARPS > 1 ? 4 : sizeof(TK) == 4 ? 8 : 16;
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t page = __shfl_sync(0xffffffffu, my_page, src);
    const TK* base = reinterpret_cast<const TK*>(a.kv.k) + page * a.kv.sp + (int64_t)g * a.kv.sh + d;
    float s[8] = {};
    if (r0 < sets) {
      for (int r = r0; r < P; r += U * sets) {
        // Rows behind the page's last are read as that one and not added.
        Raw8<TK> x[U];
#pragma unroll
        for (int i = 0; i < U; i++) x[i].stream(base + (int64_t)min(r + i * sets, P - 1) * a.kv.st);
#pragma unroll
        for (int i = 0; i < U; i++) {
          float y[8];
          x[i].get(y);
          if (r + i * sets < P)
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] += y[e];
        }
      }
    }
    store8(&sums[threadIdx.x][0], s);
    if (WARPS > 1) __syncthreads(); else __syncwarp();
    // One feature a thread: the sets' sums in order.
    for (int f = tid; f < a.kv.hd; f += LANES) {
      float x = 0.f;
      for (int i = 0; i < min(sets, P); i++) x += sums[base_row + i * lpr + (f >> 3)][f & 7];
      store_as(reinterpret_cast<TK*>(a.means) + (page * a.kv.kvh + g) * a.kv.hd + f, x / (float)P);
    }
    if (WARPS > 1) __syncthreads(); else __syncwarp();
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
// units of log2 (the scale carries log2 e) and both sums times 2^weight_bias,
// and k_attend_join adds the parts up in part order. A row that sees nothing leaves m = -inf and l = 0 and its
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
  int own_begin;                // where the requests' own parts begin: behind the prefix, or 0 (all of the history)
  // 1: a row's parts are a cluster's CTAs, which join them through each
  // other's shared memory and write the output; nothing goes to part_*.
  int cluster;
  // Sparse: the pages each (query, KV head) reads (ascending, -1 behind them).
  const int* pages;  // [T][KVH][budget]
  int budget;
  // 1: launched behind the prefix's kernel to run beside it (see overlap_begin).
  int overlap;
};

// Kernels here are launched so that they may start while the one before them
// on the stream drains (programmatic dependent launch), and wait for it
// before they read anything. The kernel of the requests' own positions reads
// nothing the prefix's kernel writes and is bound by other parts of the GPU:
// it starts as soon as every CTA of that one has (which had waited for all
// earlier work), runs beside it, and its last CTA ends after it, so that what
// follows finds both complete.
__device__ __forceinline__ void overlap_begin(const AttendArgs& a) {
  if (!a.overlap) pdl_wait();
}
__device__ __forceinline__ void overlap_end(const AttendArgs& a) {
  if (a.overlap && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) pdl_wait();
}

struct Query {
  int token;     // row of q, -1: none
  int request;
  int pos;       // its position, -1 for every negative one
};

// Query j of request i.
__device__ __forceinline__ Query query_at(const AttendArgs& a, int i, int j) {
  const int s = a.starts[i], fresh = a.starts[i + 1] - s;
  const int token = s + j;
  if (j >= fresh || s < 0 || token >= a.T) return Query{-1, i, -1};
  return Query{token, i, max(min(a.lengths[i] - fresh + j, a.max_length - 1), -1)};
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
  return Query{token, l, max(min(a.lengths[l] - fresh + j, a.max_length - 1), -1)};
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
    if (SRC == SRC_OWN && b < a.prefix_pages) {
      id = a.prefix[b];
    } else {
      if (SRC == SRC_OWN && b >= a.width) return -1;
      id = ids[b];
    }
  }
  if (id < 0 || id >= a.kv.num_pages) return -1;
  return (int64_t)id * a.kv.sp + (int64_t)r * a.kv.st;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights that become 16-bit operands are 2^(score - m + weight_bias): binary16
// has no values below 2^-24, so that weights relative to a largest of 1 would
// lose bits from 2^-14 of it on and vanish from the products, though not from
// their float32 sum, below 2^-25. A long light tail behind a heavy position is
// made of such weights. With 2^14 (float32 rows) both pieces of a weight keep
// their bits down to 2^-17 of the largest and 2^-39 of it is the error of
// any other; with 2^11 (binary16 rows, whose shared prefix needs the rest of
// the range for a reference that lags behind, paged_tc.cuh) it is 11 bits down to
// 2^-25, and 2^-36. Both sums of a row carry the factor, which cancels; kernels
// whose parts are joined have the same. bfloat16 has float32's exponents.
template <typename TQ, typename TK>
__host__ __device__ constexpr float weight_bias() {
  return sizeof(TK) == 4 || __is_same(TK, bf16) ? 0.f : sizeof(TQ) == 4 ? 14.f : 11.f;
}

// 1 / l, 0 for a row that saw nothing; NaN stays NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

// A matrix product takes in every position of its tile, those a row does not
// attend to with weight 0; an infinity or NaN among their values makes the
// row's sums NaN. Such rows (not finite, and short of the part's last
// position) are summed again by this: a warp adds 2^(score - m + weight_bias) v
// over the part's positions up to `last` one by one, score and m in units of
// log2, and writes the sums to dst. The part is the tiles of `tile` positions every `step`
// from u0 on, up to u1.
template <typename TQ, typename TK, int HD, int SRC>
__device__ __noinline__ void sum_row(const AttendArgs& a, int row, int g, int request, int u0, int u1, int tile, int step, int last, float m, float* dst) {
  constexpr int NCH = (HD + 127) / 128;
  const int lane = threadIdx.x & 31;
  const TQ* qp = reinterpret_cast<const TQ*>(a.q) + (int64_t)(row / a.H) * a.q_ts + (int64_t)(row % a.H) * a.q_hs;
  const TK* kb = reinterpret_cast<const TK*>(a.kv.k) + (int64_t)g * a.kv.sh;
  const TK* vb = reinterpret_cast<const TK*>(a.kv.v) + (int64_t)g * a.kv.sh;
  const int* ids = SRC == SRC_PREFIX ? a.prefix : a.tables + (int64_t)request * a.table_stride;
  float4 q[NCH], o[NCH];
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    const int d = (c * 32 + lane) * 4;
    q[c] = d < a.hd ? load4(qp + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  for (int ub = u0; ub < u1 && ub <= last; ub += step)
    for (int u = ub; u < min(ub + tile, u1) && u <= last; u++) {
      int t;
      const int64_t off = source_at<SRC>(a, ids, nullptr, u, t);
      if (off < 0) continue;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int d = (c * 32 + lane) * 4;
        if (d < a.hd) {
          const float4 k = load4(kb + off + d);
          s = fmaf(q[c].x, k.x, fmaf(q[c].y, k.y, fmaf(q[c].z, k.z, fmaf(q[c].w, k.w, s))));
        }
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float p = ex2(fmaf(s, a.scale, -ref) + weight_bias<TQ, TK>());
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int d = (c * 32 + lane) * 4;
        if (d < a.hd) {
          const float4 v = load4(vb + off + d);
          o[c].x = fmaf(p, v.x, o[c].x);
          o[c].y = fmaf(p, v.y, o[c].y);
          o[c].z = fmaf(p, v.z, o[c].z);
          o[c].w = fmaf(p, v.w, o[c].w);
        }
      }
    }
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    const int d = (c * 32 + lane) * 4;
    if (d < a.hd) *reinterpret_cast<float4*>(dst + d) = o[c];
  }
}

// The parts of a cluster's rows, joined: row r of part p is at rows + r * stride
// (m, l, then hd sums) of the shared memory of the cluster's CTA p. CTA p
// writes the features p * 4, (p + parts) * 4, ... of every row, each from all
// parts in part order. Every thread of every CTA of the cluster calls this.
template <typename TQ, typename RowOut>
__device__ __forceinline__ void cluster_join(const AttendArgs& a, float* rows, int stride, int count, RowOut row_out) {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  uint32_t rank, parts;
  asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %cluster_nctarank;" : "=r"(parts));
  const uint32_t base = smem_u32(rows);
  const int quads = (a.hd / 4 + (int)parts - 1) / (int)parts;  // of a CTA
  for (int e = threadIdx.x; e < count * quads; e += blockDim.x) {
    const int r = e / quads, d = ((e - r * quads) * (int)parts + (int)rank) * 4, row = row_out(r);
    if (row < 0 || d >= a.hd) continue;
    const uint32_t at = base + (uint32_t)(r * stride) * 4;
    float m[8], l[8], mx = -INFINITY;
#pragma unroll
    for (int p = 0; p < 8; p++) {
      m[p] = -INFINITY;
      l[p] = 0.f;
      if (p < (int)parts) {
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(p));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m[p]) : "r"(there));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l[p]) : "r"(there + 4));
      }
      mx = fmaxf(mx, m[p]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 8; p++)
      if (p < (int)parts) {
        const float w = ex2(m[p] - ref);
        uint32_t there;
        float x[4];
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at + 8 + d * 4), "r"(p));
#pragma unroll
        for (int i = 0; i < 4; i++) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[i]) : "r"(there + 4 * i));
        ls = fmaf(l[p], w, ls);
        s.x = fmaf(x[0], w, s.x);
        s.y = fmaf(x[1], w, s.y);
        s.z = fmaf(x[2], w, s.z);
        s.w = fmaf(x[3], w, s.w);
      }
    const float inv = inverse_sum(ls);
    store4(reinterpret_cast<TQ*>(a.out) + (int64_t)(row / a.H) * a.o_ts + (int64_t)(row % a.H) * a.o_hs + d, make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv));
  }
  // Nobody leaves while its shared memory is read.
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CUDA-core parts. A warp holds four groups of eight lanes; a group takes
// every fourth position of its warp's share and keeps a softmax state of its
// own for each of R rows, so that nothing is exchanged until the end: dot
// products need three shuffles, the running sums none. The groups' states
// are joined through shared memory in a fixed order. Float32 multiply-adds
// bound it where several rows share positions, bytes otherwise; small steps
// are bound by the chain of starts, table, keys and join: 12 us for eight
// requests of up to four tokens over 592 positions, 4 KV heads of 64.
//
// grid: x = request * row tiles + row tile (own history: rows of a request;
// list: rows of a query, x counts queries; prefix: x = row tile of all rows),
// y = KV head, z = part.
constexpr int CC_WARPS = 4;
constexpr int CC_GROUPS = CC_WARPS * 4;

template <int NCH, int R, int SRC>
__global__ void __launch_bounds__(CC_WARPS * 32) k_attend_cc(AttendArgs a, int row_tiles) {
  pdl_wait();
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
  const float* qp[R];
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
    qp[r] = q.token < 0 ? nullptr : reinterpret_cast<const float*>(a.q) + (int64_t)q.token * a.q_ts + (int64_t)(g * a.G + hh) * a.q_hs;
    if (q.token >= 0) {
      token0 = q.token;
      most = max(most, q.pos);
    }
  }
  if (token0 < 0) return;  // the same for all of a cluster
  const int prefix_end = a.prefix_pages * a.kv.P;
  int u0, u1;
  const int* ids;
  const int* table = nullptr;
  if (SRC == SRC_PREFIX) {
    u0 = part * a.prefix_chunk;
    u1 = min(min(u0 + a.prefix_chunk, prefix_end), most + 1);
    ids = a.prefix;
  } else if (SRC == SRC_OWN) {
    u0 = a.own_begin + part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, most + 1);
    ids = a.tables + (int64_t)request * a.table_stride;
  } else {
    u0 = part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, a.budget * a.kv.P);
    ids = a.pages + ((int64_t)token0 * a.KVH + g) * a.budget;
    table = a.tables + (int64_t)(request / a.max_fresh) * a.table_stride;
  }
  if (SRC == SRC_OWN && u0 >= u1 && !(part == 0 && a.slots == 1) && !a.cluster) return;  // k_attend_join counts the parts by the same rule

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
  const float* kb = reinterpret_cast<const float*>(a.kv.k) + (int64_t)g * a.kv.sh;
  const float* vb = reinterpret_cast<const float*>(a.kv.v) + (int64_t)g * a.kv.sh;
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
          if (SRC != SRC_LIST && t[i] > limit[r]) continue;  // zero times an infinity is none; a list's rows share a limit
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
    float* out = reinterpret_cast<float*>(a.out) + (int64_t)(row_out[r] / a.H) * a.o_ts + (int64_t)(row_out[r] % a.H) * a.o_hs;
    float* mine = cc_smem + CC_GROUPS * (width + 2) + r * (width + 2);  // this part of the row, for its cluster
    for (int d = threadIdx.x; d < hd; d += CC_WARPS * 32) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < CC_GROUPS; i++) s = fmaf(so[i * width + d], w[i], s);
      if (a.cluster)
        mine[2 + d] = s;
      else if (direct)
        out[d] = s * inv;
      else
        a.part_o[slot * hd + d] = s;
    }
    if (threadIdx.x == 0) {
      if (a.cluster)
        mine[0] = mx, mine[1] = ls;
      else if (!direct)
        a.part_ml[slot] = make_float2(mx, ls);
    }
  }
  if (a.cluster) {
    float* rows = cc_smem + CC_GROUPS * (width + 2);
    cluster_join<float>(a, rows, width + 2, R, [&](int r) {
      int x = -1;
#pragma unroll
      for (int i = 0; i < R; i++)
        if (i == r) x = row_out[i];
      return x;
    });
  }
}

// Parts of a row with its last position pos: the prefix's, then its own.
__device__ __forceinline__ int own_parts(const AttendArgs& a, int pos) {
  const int n = pos + 1 - a.own_begin;
  return n <= 0 ? 0 : (n + a.own_chunk - 1) / a.own_chunk;
}

// Adds up the parts of one row (warp per row): out = sum_j w_j o_j / sum_j w_j
// l_j with w_j = 2^(m_j - max m), in part order; a part without weight adds
// nothing, whatever it holds. grid: x = request * max_fresh + query, y = heads / 4.
template <typename TQ, int LIST>
__global__ void __launch_bounds__(128) k_attend_join(AttendArgs a) {
  pdl_wait();
  const int i = blockIdx.x / a.max_fresh, j = blockIdx.x % a.max_fresh;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.H) return;
  const Query q = query_at(a, i, j);
  if (q.token < 0) return;
  const int parts = LIST ? a.slots : a.prefix_slots + own_parts(a, q.pos);
  const int64_t row = (int64_t)q.token * a.H + h;
  const float2* ml = a.part_ml + row * a.slots;
  float mx = -INFINITY;
  for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, ml[p].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = mx == -INFINITY ? 0.f : mx;
  const float* po = a.part_o + row * a.slots * a.hd;
  TQ* out = reinterpret_cast<TQ*>(a.out) + (int64_t)q.token * a.o_ts + (int64_t)h * a.o_hs;
  for (int d0 = 0; d0 < a.hd; d0 += 128) {
    const int d = d0 + lane * 4;
    float l = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < parts; p0 += 32) {
      const float2 mine = p0 + lane < parts ? ml[p0 + lane] : make_float2(-INFINITY, 0.f);
      const float w = ex2(mine.x - ref);
      const int n = min(32, parts - p0);
      for (int p1 = 0; p1 < n; p1 += 8) {
        float wp[8];
        float4 x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          // Not held back by the part's statistics, which are on their way too.
          x[e] = p1 + e < n && d < a.hd ? *reinterpret_cast<const float4*>(po + (int64_t)(p0 + p1 + e) * a.hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          wp[e] = __shfl_sync(0xffffffffu, w, (p1 + e) & 31);
          l = fmaf(__shfl_sync(0xffffffffu, mine.y, (p1 + e) & 31), wp[e], l);
          if (wp[e] == 0.f) continue;
          s.x = fmaf(x[e].x, wp[e], s.x);
          s.y = fmaf(x[e].y, wp[e], s.y);
          s.z = fmaf(x[e].z, wp[e], s.z);
          s.w = fmaf(x[e].w, wp[e], s.w);
        }
      }
    }
    const float inv = inverse_sum(l);
    if (d < a.hd) store4(out + d, make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv));
  }
}

// ---------------------------------------------------------------------------
// Page choice of sparse attention.
//
// score(b) = max over the KV head's query heads h of q_h . mean_b, of which
// the order is wanted in float64. The scores are first taken in float32 with
// a bound on their error, eps = c sum_d |q_d| |mean_d| (the largest over
// heads and pages; c counts every rounding of the products and sums). With s
// the top-th largest float32 score, pages above s + 2 eps are certainly among
// the best and pages below s - 2 eps certainly not; only those between, seldom
// more than the page at the border itself, are scored again in float64, where
// products of the stored types are exact and the sum is good to 2^-52 of its
// terms. A bound that is not finite (infinite or NaN means) sends every page
// to float64.
struct ChooseArgs {
  int first, last, top;
  const void* means;         // [num_pages][KVH][hd]
  float* scores;             // [T][KVH][width]; NaN: no page, or a NaN score
  float* eps;                // [T][KVH][tiles]
  unsigned long long* keys;  // [T][KVH][width], of the pages scored again
  int width, tiles, per;     // a scoring CTA takes `per` pages, tiles of them cover a table
  int* pages;                // [T][KVH][budget]
};

// The bound on a score's error from most, the largest sum |q_d| |mean_d|: c
// above, (2 hd + 32) steps of 2^-23, covers hd products and additions (the
// tensor core's may truncate) and the 22-bit split of float32 queries. Two errors
// are no part of the sum: products that end among float32's subnormal numbers
// or below (2^-126 each), and what the split leaves out of values far below a
// query's largest, 2^-25 of the step `scale` its pieces are counted in, times a
// binary16 mean (0: not split).
__device__ __forceinline__ float score_error(float most, int hd, float scale) {
  return fmaf(most, (float)(2 * hd + 32) * 1.1920929e-7f, (float)hd * fmaf(scale, 0x1p-9f, 0x1p-125f));
}

// Candidate pages [lo, hi) of a query.
struct Candidates {
  int npages, lo, hi;
};
__device__ __forceinline__ Candidates candidates_of(const AttendArgs& a, const ChooseArgs& c, int pos) {
  Candidates x;
  x.npages = pos < 0 ? 0 : min((int)a.kv.divP.div(pos) + 1, c.width);
  x.lo = min(c.first, x.npages);
  x.hi = max(x.lo, x.npages - c.last);
  return x;
}

// Float32 scores on CUDA cores (float32 caches), eight lanes a page.
// grid: x = request * max_fresh + query, y = KV head, z = page tile.
__global__ void __launch_bounds__(128) k_page_scores_cc(AttendArgs a, ChooseArgs c) {
  extern __shared__ __align__(16) float cq[];  // [G][hd]
  __shared__ float s_eps[4];
  pdl_wait();
  const Query q = query_at(a, blockIdx.x / a.max_fresh, blockIdx.x % a.max_fresh);
  if (q.token < 0) return;
  const int g = blockIdx.y, hd = a.hd;
  const Candidates cand = candidates_of(a, c, q.pos);
  const int lo = max(cand.lo, (int)blockIdx.z * c.per), hi = min(cand.hi, (int)blockIdx.z * c.per + c.per);
  if (lo >= hi || cand.hi - cand.lo <= c.top) return;  // nothing to choose here
  for (int e = threadIdx.x * 4; e < a.G * hd; e += 128 * 4) {
    const int h = e / hd, d = e - h * hd;
    *reinterpret_cast<float4*>(cq + e) = load4(reinterpret_cast<const float*>(a.q) + (int64_t)q.token * a.q_ts + (int64_t)(g * a.G + h) * a.q_hs + d);
  }
  __syncthreads();
  const int* table = a.tables + (int64_t)q.request * a.table_stride;
  const int l8 = threadIdx.x & 7;
  float most = 0.f;
  for (int b0 = blockIdx.z * c.per; b0 < hi; b0 += 16) {
    const int b = b0 + (threadIdx.x >> 3);
    const int id = b >= lo && b < hi ? table[b] : -1;
    const bool on = id >= 0 && id < a.kv.num_pages;
    const float* mp = reinterpret_cast<const float*>(c.means) + ((int64_t)(on ? id : 0) * a.KVH + g) * hd;
    float best = -INFINITY;
    bool nan = false;
    for (int h = 0; h < a.G; h++) {
      float s = 0.f, z = 0.f;
      for (int d = l8 * 4; d < hd; d += 32) {
        const float4 v = on ? load4(mp + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 x = *reinterpret_cast<const float4*>(cq + h * hd + d);
        s = fmaf(x.x, v.x, fmaf(x.y, v.y, fmaf(x.z, v.z, fmaf(x.w, v.w, s))));
        z = fmaf(fabsf(x.x), fabsf(v.x), fmaf(fabsf(x.y), fabsf(v.y), fmaf(fabsf(x.z), fabsf(v.z), fmaf(fabsf(x.w), fabsf(v.w), z))));
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        z += __shfl_xor_sync(0xffffffffu, z, o);
      }
      nan |= !(s == s);
      best = fmaxf(best, s);
      most = z > most || !(z == z) ? z : most;
    }
    if (l8 == 0 && b >= lo && b < hi) c.scores[((int64_t)q.token * a.KVH + g) * c.width + b] = on && !nan ? best : NAN;
  }
  // NaN outlives the maximum: it has the largest bits of the positive floats.
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
  if ((threadIdx.x & 31) == 0) s_eps[threadIdx.x >> 5] = __uint_as_float(w);
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t x = 0;
    for (int i = 0; i < 4; i++) x = max(x, __float_as_uint(s_eps[i]));
    c.eps[((int64_t)q.token * a.KVH + g) * c.tiles + blockIdx.z] = score_error(__uint_as_float(x), hd, 0.f);
  }
}

// Order-preserving keys; NaN is 1, below every number, and no page 0.
__device__ __forceinline__ uint32_t score_key32(float s) {
  if (!(s == s)) return 1u;
  return float_order_key(s + 0.f);  // -0 and +0 are one value
}
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(s == s)) return 1ull;
  s += 0.0;
  const unsigned long long u = (unsigned long long)__double_as_longlong(s);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

constexpr int CHOOSE_MAX = 1024;    // threads of a choosing CTA at most
constexpr int CHOOSE_CACHE = 8192;  // scores a CTA keeps in shared memory; others are read again from L2
constexpr int CHOOSE_OPEN = 64;     // pages at the border that are ordered at once
constexpr int RADIX_BITS = 11, RADIX_BINS = 1 << RADIX_BITS;

struct ChooseShared {
  int hist[RADIX_BINS];
  int sums[CHOOSE_MAX / 32], result[2];
  int sure, open;
  uint32_t eps;
  int list[CHOOSE_OPEN];
  unsigned long long key[CHOOSE_OPEN];
};

// The top `stop` of `bits` bits of the want-th largest key (1 <= want <= number
// of keys) among the entries that `each(f)` calls f(key) for on every thread,
// by digits of 11 bits from the highest on; `want` becomes how many of the keys
// with these bits are wanted. Eleven
// bits: scores share their exponents, and eight would put most of them on a
// few bins, where the counts' updates queue up.
template <int CHOOSE_THREADS, typename Key, typename Each>
__device__ __forceinline__ Key radix_select(ChooseShared& sh, int bits, int stop, int& want, Each each) {
  constexpr int BINS_PER = RADIX_BINS / CHOOSE_THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Key prefix = 0;
  int done = 0;  // bits of the prefix
  while (done < stop) {
    const int n = min(RADIX_BITS, bits - done), shift = bits - done - n;
#pragma unroll
    for (int i = 0; i < BINS_PER; i++) sh.hist[tid + i * CHOOSE_THREADS] = 0;
    __syncthreads();
    each([&](Key k) {
      if (done == 0 || (k >> (shift + n)) == (prefix >> (shift + n))) atomicAdd(&sh.hist[(int)((k >> shift) & ((Key(1) << n) - 1))], 1);
    });
    __syncthreads();
    int mine = 0;
#pragma unroll
    for (int i = 0; i < BINS_PER; i++) mine += sh.hist[tid * BINS_PER + i];
    int up = mine;  // entries in this thread's bins and above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_down_sync(0xffffffffu, up, o);
      if (lane + o < 32) up += x;
    }
    if (lane == 0) sh.sums[warp] = up;
    __syncthreads();
    for (int w = warp + 1; w < CHOOSE_THREADS / 32; w++) up += sh.sums[w];
    if (up >= want && up - mine < want) {  // one thread
      int left = want - (up - mine), d = BINS_PER - 1;
      while (sh.hist[tid * BINS_PER + d] < left) left -= sh.hist[tid * BINS_PER + d--];
      sh.result[0] = tid * BINS_PER + d;
      sh.result[1] = left;
    }
    __syncthreads();
    prefix |= (Key)sh.result[0] << shift;
    want = sh.result[1];
    done += n;
  }
  return prefix;
}

// One CTA per (query, KV head): a narrow interval around the top-th key by
// radix selection, the pages in and around it ordered in float64, then the
// chosen pages in ascending order. Latency bounds it (17 us from cold caches
// for 512 lists of up to 1,024 pages, which all SMs hold at once). 256 threads, or 1,024 where tables have
// more than 1,024 pages (32 lists of 4,096 pages: 12 us, with 256 threads 17).
// grid: x = request * max_fresh + query, y = KV head.
template <typename TQ, typename TK, int CHOOSE_THREADS>
__global__ void __launch_bounds__(CHOOSE_THREADS) k_page_choose(AttendArgs a, ChooseArgs c) {
  __shared__ ChooseShared sh;
  extern __shared__ uint32_t cache[];  // keys, min(width, CHOOSE_CACHE)
  pdl_wait();
  const Query q = query_at(a, blockIdx.x / a.max_fresh, blockIdx.x % a.max_fresh);
  if (q.token < 0) return;
  const int g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t at = (int64_t)q.token * a.KVH + g;
  int* out = c.pages + at * a.budget;
  const Candidates cand = candidates_of(a, c, q.pos);
  const int npages = cand.npages, lo = cand.lo, hi = cand.hi;
  const bool all = hi - lo <= c.top, choose = !all && c.top > 0;
  const float* scores = c.scores + at * c.width;
  unsigned long long* keys = c.keys + at * c.width;
  const int kept = min(hi, min(c.width, CHOOSE_CACHE));
  auto key32 = [&](int b) { return b < kept ? cache[b] : score_key32(scores[b]); };
  // Keys above in_above: certainly in; below out_below: certainly not; those
  // between are open (all of them, where the bound is not finite).
  uint32_t in_above = 0xffffffffu, out_below = 0;
  auto is_open = [&](uint32_t k) { return k <= in_above && k >= out_below; };
  unsigned long long thr = 0;  // open pages with a larger key are taken (~0: all open pages),
  int ties = 0;                // and this many with this one
  if (choose) {
    if (tid == 0) {
      sh.eps = 0;
      sh.sure = sh.open = 0;
    }
#pragma unroll 4
    for (int b = lo + tid; b < kept; b += CHOOSE_THREADS) cache[b] = score_key32(scores[b]);
    uint32_t e = 0;
    for (int i = lo / c.per + tid; i <= (hi - 1) / c.per; i += CHOOSE_THREADS) e = max(e, __float_as_uint(c.eps[at * c.tiles + i]) & 0x7fffffffu);
    e = __reduce_max_sync(0xffffffffu, e);
    __syncthreads();
    if (lane == 0 && e) atomicMax(&sh.eps, e);
    // The upper 22 bits of the top-th largest float32 score's key: it lies in
    // [prefix, prefix + 1023], about the width of the error bound.
    int want = c.top;
    const uint32_t prefix = radix_select<CHOOSE_THREADS, uint32_t>(sh, 32, 2 * RADIX_BITS, want, [&](auto f) {
#pragma unroll 4
      for (int b = lo + tid; b < hi; b += CHOOSE_THREADS) f(key32(b));
    });
    const float eps = __uint_as_float(sh.eps);
    const float low = float_from_order_key(prefix), high = float_from_order_key(prefix | 1023u);
    if (eps < INFINITY && prefix > 1u && fabsf(low) < INFINITY && fabsf(high) < INFINITY) {
      // Rounded outwards by the additions' own half steps.
      in_above = score_key32(high + (2.f * eps + 2e-7f * fabsf(high)));
      out_below = max(2u, score_key32(low - (2.f * eps + 2e-7f * fabsf(low))));
    }
    // Pages certainly in, and pages that float64 has to order.
    int sure = 0;
#pragma unroll 4
    for (int b = lo + tid; b < hi; b += CHOOSE_THREADS) {
      const uint32_t x = key32(b);
      sure += x > in_above;
      if (is_open(x)) {
        const int i = atomicAdd(&sh.open, 1);
        if (i < CHOOSE_OPEN) sh.list[i] = b;
      }
    }
    sure = __reduce_add_sync(0xffffffffu, sure);
    if (lane == 0 && sure) atomicAdd(&sh.sure, sure);
    __syncthreads();
    want = c.top - sh.sure;
    const int open = sh.open;
    if (open == want) {
      ties = want;
      thr = ~0ull;
    } else {
      // Float64 keys, a warp a page.
      const int* table = a.tables + (int64_t)q.request * a.table_stride;
      auto exact_key = [&](int b) {
        const int id = table[b];
        if (id < 0 || id >= a.kv.num_pages) return 0ull;
        const TK* mp = reinterpret_cast<const TK*>(c.means) + ((int64_t)id * a.KVH + g) * a.hd;
        double best = 0.0;
        for (int h = 0; h < a.G; h++) {
          const TQ* qp = reinterpret_cast<const TQ*>(a.q) + (int64_t)q.token * a.q_ts + (int64_t)(g * a.G + h) * a.q_hs;
          double s = 0.0;
          for (int d = lane * 4; d < a.hd; d += 128) {
            const float4 u = load4(qp + d), v = load4(mp + d);
            s = fma((double)u.x, (double)v.x, s);
            s = fma((double)u.y, (double)v.y, s);
            s = fma((double)u.z, (double)v.z, s);
            s = fma((double)u.w, (double)v.w, s);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          // The largest of the heads; a NaN makes the page NaN.
          if (h == 0 || (best == best && (s > best || !(s == s)))) best = s;
        }
        return score_key(best);
      };
      if (open <= CHOOSE_OPEN) {  // a few pages at the border: each counts those above it
        for (int i = warp; i < open; i += CHOOSE_THREADS / 32) {
          const int b = sh.list[i];
          const unsigned long long k = exact_key(b);
          if (lane == 0) {
            sh.key[i] = k;
            keys[b] = k;
          }
        }
        __syncthreads();
        if (tid < open) {
          const unsigned long long k = sh.key[tid];
          int above = 0, same = 0;
          for (int i = 0; i < open; i++) {
            above += sh.key[i] > k;
            same += sh.key[i] == k;
          }
          if (above < want && above + same >= want) {  // this key is the border; equal ones write the same
            sh.result[0] = tid;
            sh.result[1] = want - above;
          }
        }
        __syncthreads();
        thr = sh.key[sh.result[0]];
        ties = sh.result[1];
      } else {
        for (int b0 = lo + warp * 32; b0 < hi; b0 += CHOOSE_THREADS) {
          const int mine = b0 + lane;
          uint32_t todo = __ballot_sync(0xffffffffu, mine < hi && is_open(key32(min(mine, hi - 1))));
          while (todo) {
            const int b = b0 + __ffs(todo) - 1;
            todo &= todo - 1;
            const unsigned long long k = exact_key(b);
            if (lane == 0) keys[b] = k;
          }
        }
        __syncthreads();
        thr = radix_select<CHOOSE_THREADS, unsigned long long>(sh, 64, 64, want, [&](auto f) {
          for (int b = lo + tid; b < hi; b += CHOOSE_THREADS)
            if (is_open(key32(b))) f(keys[b]);
        });
        ties = want;
      }
    }
  }
  // The chosen pages in order: each thread looks through a run of pages (an
  // odd number, so that a warp's reads of the scores fall on different banks),
  // and one sum over the threads says where its pages go. Ties go to the lower
  // pages: their count before a thread's run needs a sum of its own.
  const bool keyed = choose && thr != ~0ull;
  const int per = ((npages + CHOOSE_THREADS - 1) / CHOOSE_THREADS) | 1;
  const int b0 = min(npages, tid * per), b1 = min(npages, b0 + per);
  // -1: not taken, 0: a tie, 1: taken.
  auto verdict = [&](int b) {
    if (b < lo || b >= hi || all) return 1;
    if (!choose) return -1;
    const uint32_t x = key32(b);
    if (!is_open(x)) return x > in_above ? 1 : -1;
    if (!keyed) return 1;
    const unsigned long long k = keys[b];
    return k > thr ? 1 : k == thr ? 0 : -1;
  };
  auto sum_before = [&](int mine, int& total) {
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh.sums[warp] = x;
    __syncthreads();
    int before = x - mine;
    total = 0;
    for (int w = 0; w < CHOOSE_THREADS / 32; w++) {
      if (w < warp) before += sh.sums[w];
      total += sh.sums[w];
    }
    return before;
  };
  int tied = 0, total;
  if (keyed) {
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += verdict(b) == 0;
    tied = sum_before(mine, total);
  }
  int mine = 0;
  for (int b = b0, t = tied; b < b1; b++) {
    const int v = verdict(b);
    mine += v > 0 || (v == 0 && t++ < ties);
  }
  int to = sum_before(mine, total);
  for (int b = b0, t = tied; b < b1; b++) {
    const int v = verdict(b);
    if (v > 0 || (v == 0 && t++ < ties)) {
      if (to < a.budget) out[to] = b;
      to++;
    }
  }
  for (int e = total + tid; e < a.budget; e += CHOOSE_THREADS) out[e] = -1;
}

}  // namespace tcu
