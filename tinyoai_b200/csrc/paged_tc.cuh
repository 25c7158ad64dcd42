// Attention of many query rows to the prefix they share (16-bit caches) on
// the 5th-generation tensor cores.
//
// All rows of a step (queries x the G query heads of a KV head) read the same
// keys, so they fill 128-row tcgen05 tiles, and each 128-position block of
// keys and values is fetched by TMA once per CTA:
//   S = Q K^T   M = 128 rows, N = 128 positions, K = head size; Q and K in
//               shared memory (128-byte swizzle), S in TMEM;
//   P = 2^(S scale - m)  one thread per row, packed to 16 bits over S's own
//               TMEM columns;
//   O += P V    A = P from TMEM, B = V as stored (features contiguous), O in
//               TMEM.
// Two streams of this run against each other so that one stream's softmax
// covers the other's products: two tiles of rows over the same blocks
// (more than 128 rows) or one tile of rows over alternate blocks, each
// stream then leaving a partial result of its own. Warps 0-3 and 4-7 are the
// streams' softmax, warp 8 issues the TMA loads (from the moment the page ids
// are there, while the others bring the queries), warp 9 the products.
//
// A row's reference m moves only when a block's maximum passes it by more
// than a factor 2^lag, which spares the multiplication of O in TMEM for almost
// every block; the sums stay exact in float32 since the same m enters numerator
// and denominator. bfloat16: lag 8; binary16: lag 4, whose largest weight
// 2^(4 + weight_bias) = 2^15 is within the type. A stream's
// product S(i + 1) overwrites the columns of P(i): the tensor core runs a
// CTA's products in the order they are issued, P(i) V before S(i + 1).
//
// 1,024 rows (256 queries x 4) over 32,768 positions, 8 KV heads of 128: 160 us,
// 860 TFLOP/s. A pair of blocks takes about 4,000 cycles of which the products
// are 2,048 at the peak rate, the exponentials 2,048 of the special function
// units, shared memory's reads and TMA's writes 2,048; what is left is the
// chain product - softmax - product of each stream. Taking a part of the
// exponentials on the multiply-add pipes (a polynomial) made it slower
// (177 -> 184 us with every fourth), as did one vote for every 32 columns (250).
//
// Copies read this GPU's own memory into this CTA's shared memory; page ids
// that name no page become a coordinate behind the last page, which TMA fills
// with zeros, and their positions are masked. Every wait is bounded; one that
// runs out ends the CTA with NaN results.
#pragma once
#include <cuda.h>

#include "paged.cuh"
#include "paged_mma.cuh"
#include "ring.h"
#include "tcgen05.cuh"

namespace tcu {

constexpr int PT_ROWS = 128, PT_KEYS = 128;
constexpr int PT_THREADS = 320;
// Registers a thread: leaves an SM 16,896 of them and 23 KB of shared memory,
// one CTA of k_attend_mma beside this kernel's.
#define PT_REGS 152
constexpr int PT_IDS = 1024;      // page ids of a part
constexpr int PT_SUB = 16384;     // bytes of 128 rows of 64 values
constexpr int PT_MAX_STAGES = 4;

struct PagedTcArgs {
  int per;         // blocks of a part
  int blocks;      // blocks of the prefix
  int split_keys;  // 1: both streams have the same rows and take alternate blocks
  int stages;      // of the K ring, and of the V ring
  int box;         // rows of one TMA box: min(page, 128)
  int hdp;         // head size rounded up to 16
};

struct PtShared {
  uint64_t k_full[PT_MAX_STAGES], k_empty[PT_MAX_STAGES], v_full[PT_MAX_STAGES], v_empty[PT_MAX_STAGES];
  uint64_t s_full[2], p_full[2], o_done[2], gone;
  uint32_t tmem;
  int err;
  int row[2 * PT_ROWS], limit[2 * PT_ROWS];
  int ids[PT_IDS];
};

__host__ __device__ constexpr size_t pt_smem(int sub, int split_keys, int stages) {
  return (size_t)sub * PT_SUB * ((split_keys ? 1 : 2) + 2 * stages) + 1024 + sizeof(PtShared);
}

constexpr size_t PT_MAX_SMEM = 227 * 1024;
static_assert(pt_smem(2, 0, 2) <= PT_MAX_SMEM && pt_smem(1, 0, 4) <= PT_MAX_SMEM, "shared memory of the prefix kernel");

// One box of a [features, positions, heads, pages] tensor.
__device__ __forceinline__ void pt_load(void* dst, const CUtensorMap* map, int x, int row, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// After a wait that ran out: what was issued must have landed before the CTA
// leaves (bounded as well).
__device__ __forceinline__ void pt_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = global_ns();
  while (!mbar_try_wait(bar, parity))
    if (global_ns() - t0 > TCU_WAIT_NS) return;
}

// a * b + c and a + b on two floats at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

// Masks 64 scores of positions key0 ..: past column `seen`, and of pages that are none.
__device__ __forceinline__ void pt_mask_bits(const AttendArgs& a, const PtShared& sh, int key0, int seen, int prefix_end, int blk0, uint32_t* bits) {
  const int lane = threadIdx.x & 31, first = (int)a.kv.divP.div(blk0 * PT_KEYS);
#pragma unroll
  for (int w = 0; w < 2; w++) {
    const int key = key0 + w * 32 + lane;
    const uint32_t there = __ballot_sync(0xffffffffu, key < prefix_end && sh.ids[min((int)a.kv.divP.div(min(key, prefix_end - 1)) - first, PT_IDS - 1)] >= 0);
    const int n = min(max(seen + 1 - 32 * w, 0), 32);
    bits[w] = there & (n == 32 ? 0xffffffffu : (1u << n) - 1);
  }
}
__device__ __forceinline__ void pt_mask(const AttendArgs& a, const PtShared& sh, uint32_t (&s)[PT_KEYS / 2], int key0, int seen, int prefix_end, int blk0) {
  uint32_t bits[2];
  pt_mask_bits(a, sh, key0, seen, prefix_end, blk0, bits);
#pragma unroll
  for (int q = 0; q < PT_KEYS / 2; q++)
    if (!(bits[q >> 5] >> (q & 31) & 1)) s[q] = 0xff800000u;
}

__device__ __forceinline__ void pt_ld16(uint32_t taddr, uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
        "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
      : "r"(taddr));
  tc_wait_ld();
}

// This lane's first n columns from taddr on, times f.
__device__ __forceinline__ void pt_scale_rows(uint32_t taddr, int n, float f) {
  for (int q = 0; q < n; q += 16) {
    uint32_t x[16];
    pt_ld16(taddr + q, x);
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr + q), "r"(x[0]),
        "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]),
        "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15])
        : "memory");
  }
}

template <typename T, int SUB>
__global__ void __maxnreg__(PT_REGS) k_attend_prefix_tc(const __grid_constant__ AttendArgs a, const __grid_constant__ PagedTcArgs p, const __grid_constant__ CUtensorMap kmap,
                                                                     const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ uint8_t pt_mem[];
  pdl_wait();
  pdl_launch_dependents();  // the requests' own positions
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_mem) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = base;
  uint8_t* ks = qs + (size_t)(p.split_keys ? 1 : 2) * SUB * PT_SUB;
  uint8_t* vs = ks + (size_t)p.stages * SUB * PT_SUB;
  PtShared& sh = *reinterpret_cast<PtShared*>(vs + (size_t)p.stages * SUB * PT_SUB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = blockIdx.y, part = blockIdx.z;
  const int blk0 = part * p.per, nblk = min(p.per, p.blocks - blk0);
  const int prefix_end = a.prefix_pages * a.kv.P;
  const int tiles = p.split_keys ? 1 : 2;

  // The rows, the page ids, the barriers.
  int valid = 0, none = 0;
  if (tid < tiles * PT_ROWS) {
    const int row = blockIdx.x * tiles * PT_ROWS + tid;
    const Query q = query_of(a, row / a.G);
    sh.row[tid] = q.token < 0 ? -1 : q.token * a.H + g * a.G + row % a.G;
    sh.limit[tid] = q.token < 0 ? -1 : q.pos;
    valid = q.token >= 0;
  }
  const int first = (int)a.kv.divP.div(blk0 * PT_KEYS);
  {
    const int last = (int)a.kv.divP.div(min(prefix_end, (blk0 + nblk) * PT_KEYS) - 1);
    for (int e = tid; e <= last - first; e += PT_THREADS) {
      int id = a.prefix[first + e];
      if (id < 0 || id >= a.kv.num_pages) {
        id = -1;
        none = 1;
      }
      sh.ids[e] = id;
    }
  }
  if (tid == 0) {
    sh.err = 0;
    for (int i = 0; i < p.stages; i++) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int t = 0; t < 2; t++) {
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_full[t], 4);
      mbar_init(&sh.o_done[t], 1);
    }
    mbar_init(&sh.gone, 1);
    fence_barrier_init();
  }
  if (!__syncthreads_or(valid)) return;  // padding rows only
  const bool bad = __syncthreads_or(none) != 0;
  // TMEM columns: S of stream t at t * 128, P over its second half, O of stream t at 256 + t * 128.
  const int count[2] = {p.split_keys ? (nblk + 1) / 2 : nblk, p.split_keys ? nblk / 2 : nblk};
  uint32_t tmem = 0;
  if (warp != 8) {  // the loads of keys and values begin at once
    if (warp == 9) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // Queries, swizzled as the descriptors read them; a negative scale is taken
    // into their sign, so that the largest score is the largest S.
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    for (int e = tid < 256 ? tid : tiles * PT_ROWS * SUB * 8; e < tiles * PT_ROWS * SUB * 8; e += 256) {
      const int rr = e / (SUB * 8), ch = e % (SUB * 8), row = sh.row[rr], d = ch * 8;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row >= 0 && d < a.hd)
        x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (int64_t)(row / a.H) * a.q_ts + (int64_t)(row % a.H) * a.q_hs + d);
      x.x ^= flip;
      x.y ^= flip;
      x.z ^= flip;
      x.w ^= flip;
      const int t = rr / PT_ROWS, r = rr % PT_ROWS;
      *reinterpret_cast<uint4*>(qs + (size_t)(t * SUB + (ch >> 3)) * PT_SUB + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    named_bar_sync(1, PT_THREADS - 32);
    tc_fence_after();
    tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
  }

  int sent_k = 0, sent_v = 0;  // blocks of keys and of values whose copies were queued (by warp 8's first lane)
  if (warp == 8) {
    if (lane == 0) {
      const uint32_t bytes = (uint32_t)SUB * PT_SUB;
      const int boxes = PT_KEYS / p.box;
      bool ok = true;
      for (int b = 0; b < nblk && ok; b++) {
        const int st = b % p.stages, round = b / p.stages;
        const int key0 = (blk0 + b) * PT_KEYS;
#pragma unroll 1
        for (int kv = 0; kv < 2; kv++) {
          uint64_t* full = kv ? &sh.v_full[st] : &sh.k_full[st];
          if (round > 0) ok = mbar_wait(kv ? &sh.v_empty[st] : &sh.k_empty[st], (round - 1) & 1, &sh.err);
          if (!ok) break;
          mbar_expect_tx(full, bytes);
          uint8_t* dst = (kv ? vs : ks) + (size_t)st * SUB * PT_SUB;
          for (int x = 0; x < boxes; x++) {
            const int key = key0 + x * p.box;
            const int pg = (int)a.kv.divP.div(key), row0 = key - pg * a.kv.P;
            int id = key < prefix_end ? sh.ids[pg - first] : -1;
            if (id < 0) id = a.kv.num_pages;  // behind the pool: zeros
            for (int s = 0; s < SUB; s++) pt_load(dst + (size_t)s * PT_SUB + x * p.box * 128, kv ? &vmap : &kmap, s * 64, row0, g, id, full);
          }
          if (kv) sent_v++; else sent_k++;
        }
      }
    }
  } else if (warp == 9) {
    // The whole warp runs the schedule, so that descriptors stay in uniform
    // registers; its elected lane issues the products and their commits.
    const uint32_t type = __is_same(T, bf16) ? (1u << 7) | (1u << 10) : 0u;
    const uint32_t id_s = (1u << 4) | type | ((uint32_t)(PT_KEYS >> 3) << 17) | ((uint32_t)(PT_ROWS >> 4) << 24);
    const uint32_t id_o = (1u << 4) | type | (1u << 16) | ((uint32_t)(p.hdp >> 3) << 17) | ((uint32_t)(PT_ROWS >> 4) << 24);
    const int ksteps = p.hdp / 16;
    // Descriptors of the first tile of each operand; steps add to the address field (16-byte units).
    const uint64_t q_desc = tc_smem_desc(smem_u32(qs)), k_desc = tc_smem_desc(smem_u32(ks)), v_desc = tc_smem_desc_mn(smem_u32(vs), PT_SUB);
    const bool leader = tc_elect();
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, &sh.err)); };
    auto scores = [&](int t, int i) {
      const int b = p.split_keys ? 2 * i + t : i, st = b % p.stages;
      wait(&sh.k_full[st], (b / p.stages) & 1);
      if (!ok) return;
      tc_fence_after();
      const uint64_t qd = q_desc + (uint64_t)((p.split_keys ? 0 : t) * (SUB * PT_SUB >> 4)), kd = k_desc + (uint64_t)(st * (SUB * PT_SUB >> 4));
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < SUB * 4; kk++) {
          const uint64_t off = (kk >> 2) * (PT_SUB >> 4) + (kk & 3) * 2;
          if (kk < ksteps) tc_mma(tmem + t * 128, qd + off, kd + off, id_s, kk > 0 ? 1u : 0u);
        }
        tc_commit(&sh.s_full[t]);
        if ((p.split_keys || t == 1) && b + p.stages < nblk) tc_commit(&sh.k_empty[st]);
      }
      __syncwarp();
    };
    auto values = [&](int t, int i) {
      const int b = p.split_keys ? 2 * i + t : i, st = b % p.stages;
      wait(&sh.v_full[st], (b / p.stages) & 1);
      wait(&sh.p_full[t], i & 1);
      if (!ok) return;
      tc_fence_after();
      const uint64_t vd = v_desc + (uint64_t)(st * (SUB * PT_SUB >> 4));
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < PT_KEYS / 16; kk++)
          tc_mma_ta(tmem + 256 + t * 128, tmem + t * 128 + PT_KEYS / 2 + kk * 8, vd + (uint64_t)(kk * (2048 >> 4)), id_o, i > 0 || kk > 0 ? 1u : 0u);
        if ((p.split_keys || t == 1) && b + p.stages < nblk) tc_commit(&sh.v_empty[st]);
        if (i == count[t] - 1) tc_commit(&sh.o_done[t]);
      }
      __syncwarp();
    };
#pragma unroll
    for (int t = 0; t < 2; t++)
      if (count[t] > 0) scores(t, 0);
    for (int i = 0; i < count[0]; i++) {
#pragma unroll
      for (int t = 0; t < 2; t++)
        if (i < count[t]) {
          values(t, i);
          if (i + 1 < count[t]) scores(t, i + 1);
        }
    }
  } else {
    const int t = warp >> 2, r = tid & 127;
    const int at = p.split_keys ? r : tid;  // this thread's row
    const int row = sh.row[at], limit = sh.limit[at];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + t * 128 + lanes, to = tmem + 256 + t * 128 + lanes;
    // Not zero, so that a masked score times it stays -inf.
    const float scale = fmaxf(fabsf(a.scale), 1.17549435e-38f);
    constexpr float BIAS = weight_bias<T, T>(), LAG = BIAS == 0.f ? 8.f : 4.f;
    // From here on a score's rounding to float32 shows in its weight: the
    // reference does not lag, and a score is rounded as the reference was before
    // that is taken off, so that no weight passes 2^BIAS.
    constexpr float LARGE = 262144.f;
    static_assert(BIAS == 0.f || BIAS + LAG < 16.f, "the largest binary16 weight");
    float m = -INFINITY, l = 0.f, lag = LAG;
    bool ok = true, large = false;  // large: a row of the warp has such scores
    for (int i = 0; i < count[t]; i++) {
      const int key0 = (blk0 + (p.split_keys ? 2 * i + t : i)) * PT_KEYS;
      ok = mbar_wait(&sh.s_full[t], i & 1, &sh.err);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // First the row's maximum, 64 columns at a time (all 128 would not stay
      // in registers); the second half is still there for its weights.
      constexpr int HALF = PT_KEYS / 2;
      uint32_t s[HALF];
      const int seen = min(limit, prefix_end - 1) - key0;  // columns up to here are this row's
      const bool special = bad || __any_sync(0xffffffffu, seen < PT_KEYS - 1);
      auto load = [&](int half) {
        tc_ld32(ts + half * HALF, s);
        tc_ld32(ts + half * HALF + 32, s + 32);
        tc_wait_ld();
        if (special) pt_mask(a, sh, s, key0 + half * HALF, seen - half * HALF, prefix_end, blk0);
      };
      float mx = -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        load(half);
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < HALF; q += 8)
#pragma unroll
          for (int z = 0; z < 4; z++) x[z] = fmaxf(x[z], fmaxf(__uint_as_float(s[q + z]), __uint_as_float(s[q + 4 + z])));
        mx = fmaxf(mx, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
      }
      mx *= scale;
      const bool move = mx > m + lag;  // from -inf as well
      if (__any_sync(0xffffffffu, move)) {
        const float alpha = move ? (m == -INFINITY ? 0.f : ex2(m - mx)) : 1.f;
        if (move) m = mx;
        if (move) lag = fabsf(m) < LARGE ? LAG : 0.f;
        large = __any_sync(0xffffffffu, lag == 0.f);
        l *= alpha;
        // S(i) is complete, so P(i - 1) V is, which was issued before it.
        if (i > 0) pt_scale_rows(to, p.hdp, alpha);
      }
      const float ref = m == -INFINITY ? 0.f : m;
      const float mul = large ? 1.f : scale, add = large ? BIAS : BIAS - ref;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      // Weights of the second half, then of the first, packed into the
      // second half of S's columns, which is read by then.
#pragma unroll
      for (int half = 1; half >= 0; half--) {
        if (half == 0) load(0);
        if (large)
#pragma unroll
          for (int q = 0; q < HALF; q++) s[q] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(s[q]), scale), ref));
        uint32_t w[HALF / 2];
#pragma unroll
        for (int q = 0; q < HALF; q += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[q]), __uint_as_float(s[q + 1])), make_float2(mul, mul), make_float2(add, add));
          const float2 e = make_float2(ex2(x.x), ex2(x.y));
          sum[(q / 2) & 1] = add2(sum[(q / 2) & 1], e);
          w[q / 2] = pack2<T>(e.x, e.y);
        }
        tc_st32(ts + HALF + half * (HALF / 2), w);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[t]);
    }
    if (ok && count[t] > 0) ok = mbar_wait(&sh.o_done[t], 0, &sh.err);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    const int64_t slot = (int64_t)(row < 0 ? 0 : row) * a.slots + (p.split_keys ? 2 * part + t : part);
    float odd = 0.f;  // NaN once a sum is not finite
    for (int q = 0; q < p.hdp; q += 16) {
      uint32_t x[16] = {};
      if (count[t] > 0) pt_ld16(to + q, x);
      if (row >= 0) {
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (q + e < a.hd) *reinterpret_cast<uint4*>(a.part_o + slot * a.hd + q + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
#pragma unroll
        for (int e = 0; e < 16; e++) odd = fmaf(__uint_as_float(x[e]), 0.f, odd);
      }
    }
    // Rows that the part's last positions, which are not theirs, left without a finite sum.
    const int part_end = min(prefix_end, (blk0 + nblk) * PT_KEYS);
    uint32_t again = __ballot_sync(0xffffffffu, row >= 0 && limit < part_end - 1 && odd != odd);
    if (again) {
      __syncwarp();  // the first sums are written
      for (; again; again &= again - 1) {
        const int from = __ffs(again) - 1, at_row = __shfl_sync(0xffffffffu, row, from), tile = blk0 + (p.split_keys ? t : 0);
        sum_row<T, T, SUB * 64, SRC_PREFIX>(a, at_row, g, 0, tile * PT_KEYS, part_end, PT_KEYS, (p.split_keys ? 2 : 1) * PT_KEYS,
                                            __shfl_sync(0xffffffffu, limit, from), __shfl_sync(0xffffffffu, m, from),
                                            a.part_o + __shfl_sync(0xffffffffu, slot, from) * a.hd);
      }
    }
    if (row >= 0) a.part_ml[slot] = ok ? make_float2(m, l) : make_float2(NAN, NAN);
  }
  tc_fence_before();
  __syncthreads();
  // Every copy and product was waited for above, unless a wait ran out. Then
  // some may be on their way still, whichever warp gave up.
  if (*(volatile int*)&sh.err) {
    if (warp == 8 && lane == 0)
      for (int st = 0; st < p.stages; st++) {
        const int pk = ring_last_parity(sent_k, st, p.stages), pv = ring_last_parity(sent_v, st, p.stages);
        if (pk >= 0) pt_drain(&sh.k_full[st], pk);
        if (pv >= 0) pt_drain(&sh.v_full[st], pv);
      }
    if (warp == 9 && tc_elect()) {  // the lane that issued the products
      tc_commit(&sh.gone);
      pt_drain(&sh.gone, 0);
    }
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace tcu
