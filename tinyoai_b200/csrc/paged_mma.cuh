// Attention over 16-bit paged caches for few query rows at a time (decode
// steps, selected pages): the cache streams once from HBM through registers
// into warp-level matrix instructions.
//
// Bytes bound this: a step reads 4 * hd bytes of cache per position and KV
// head and spends 4 * hd flops per query head on them, far below what a
// 128-row tcgen05 tile needs to be worth filling (G = H / KVH rows). So a
// warp takes 16 positions at a time and computes S^T = K Q^T and O^T = V^T P^T
// with m16n8k16: positions (then features) are the 16 rows, query rows the 8
// columns. Operands come straight from global memory, with no shared memory
// and no data exchange in between:
//  - K (rows = positions, k = features): a lane loads 16 bytes of a position,
//    eight neighbouring features, and takes them as its k entries of two
//    steps; Q is read with the same order of features, which a sum over
//    features does not notice.
//  - V^T (rows = features, k = positions): a lane loads the same eight
//    features of four positions and interleaves them pairwise; feature 2j and
//    2j + 1 of the eight become rows r and r + 8 of product j.
//  - P^T leaves the first product with positions in rows; one 8 x 8 transpose
//    within the warp (movmatrix) gives the second product's operand.
// The softmax statistics are float32, one running maximum per warp and query
// row; the weights are rounded to the cache's type as operands (binary16: times
// 2^weight_bias, paged.cuh). Float32 queries over a binary16 cache keep 22 bits:
// q * 2^sx and the weights are each two binary16 values and each product two
// instructions.
//
// A CTA's warps take alternate 16-position tiles of the CTA's part and join
// their states through shared memory in warp order. Four CTAs (16 warps of
// 8 KB in flight) an SM: 64 requests x 8 KV heads that read 66 pages of 32
// positions of 128 features each (553 MB) take 90 us, 6.1 TB/s of the 6.56 a
// copy reaches; 256 requests of up to 1,024 positions (537 MB) 98 us.
#pragma once
#include "../../include/tinyoai_cuda.h"
#include "paged.cuh"

namespace tcu {

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<bf16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

constexpr int MM_WARPS = 4;
constexpr int MM_IDS = 1024;  // page ids of a part, copied to shared memory (a part has at most this many pages)

// Shared memory: the queries [PIECES][8 NT columns][HD + 32] 16-bit values (the pad puts
// the two rows a quarter warp reads on different banks), then, when the loop
// is over, the warps' outputs [MM_WARPS][8 NT][HD + 4] float32 and their (m, l),
// and the CTA's joint rows [8 NT][HD + 2] where a cluster joins them.
template <int HD, int NT, int PIECES>
constexpr size_t mm_smem(bool cluster) {
  const size_t q = (size_t)PIECES * 8 * NT * (HD + 32) * 2, o = (size_t)(MM_WARPS * (HD + 4 + 2) + (cluster ? HD + 2 : 0)) * 8 * NT * 4;
  return q > o ? q : o;
}

// Query rows col -> (token * H + head, -1: none) into shared memory [PIECES][cols][HD + 32],
// float32 ones as pairs of binary16 values of q * 2^sx. scale[col] = s * 2^-sx.
template <typename TQ, typename TK, int HD, int PIECES>
__device__ __forceinline__ void mm_load_queries(const AttendArgs& a, TK* qs, const int* rows, float* scale, int cols, float s) {
  constexpr int QS = HD + 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.hd;
  if (PIECES == 1) {
    constexpr int CH = HD / 8;
    for (int e = tid; e < cols * CH; e += MM_WARPS * 32) {
      const int col = e / CH, d = (e % CH) * 8, row = rows[col];
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row >= 0 && d < hd)
        x = *reinterpret_cast<const uint4*>(reinterpret_cast<const TQ*>(a.q) + (int64_t)(row / a.H) * a.q_ts + (int64_t)(row % a.H) * a.q_hs + d);
      *reinterpret_cast<uint4*>(qs + col * QS + d) = x;
    }
    for (int col = tid; col < cols; col += MM_WARPS * 32) scale[col] = s;
  } else {
    for (int col = warp; col < cols; col += MM_WARPS) {
      const int row = rows[col];
      float x[(HD + 31) / 32], mx = 0.f;
#pragma unroll
      for (int i = 0; i < (HD + 31) / 32; i++) {
        const int d = lane + 32 * i;
        x[i] = row >= 0 && d < hd ? (float)(reinterpret_cast<const TQ*>(a.q)[(int64_t)(row / a.H) * a.q_ts + (int64_t)(row % a.H) * a.q_hs + d]) : 0.f;
        mx = fmaxf(mx, fabsf(x[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // 2^sx brings the largest value into [2^13, 2^14). Infinite or NaN rows stay as they are.
      int ex = 0;
      if (mx > 0.f && mx < INFINITY) frexpf(mx, &ex);
      const int sx = mx > 0.f && mx < INFINITY ? min(max(14 - ex, -126), 126) : 0;
      const float up = __int_as_float((127 + sx) << 23);
#pragma unroll
      for (int i = 0; i < (HD + 31) / 32; i++) {
        const int d = lane + 32 * i;
        if (d < HD) {
          const float y = x[i] * up;
          const __half h = __float2half_rn(y);
          const float rest = y - __half2float(h);
          reinterpret_cast<__half*>(qs)[col * QS + d] = h;
          reinterpret_cast<__half*>(qs)[cols * QS + col * QS + d] = __float2half_rn(rest == rest ? rest : 0.f);
        }
      }
      if (lane == 0) scale[col] = s * __int_as_float((127 - sx) << 23);
    }
  }
}

// grid as k_attend_cc's, with row tiles of 8 * NT rows.
template <typename TQ, typename TK, int HD, int NT, int SRC>
__device__ __forceinline__ void mm_part(const AttendArgs& a, int row_tiles) {
  constexpr int COLS = 8 * NT, KG = (HD + 31) / 32, VG = (HD + 63) / 64;
  constexpr int PIECES = sizeof(TQ) == 4 ? 2 : 1;
  constexpr int QS = HD + 32;
  extern __shared__ __align__(16) uint8_t mm_mem[];
  __shared__ int s_limit[COLS], s_row[COLS], s_ids[MM_IDS];
  __shared__ float s_scale[COLS];
  TK* qs = reinterpret_cast<TK*>(mm_mem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int g = blockIdx.y, part = blockIdx.z, hd = a.hd;
  const int tile = SRC == SRC_PREFIX ? blockIdx.x : blockIdx.x % row_tiles;
  const int request = SRC == SRC_PREFIX ? 0 : blockIdx.x / row_tiles;
  if (tid < COLS) {
    const int row = tile * COLS + tid;
    Query q;
    int hh = row % a.G;
    if (SRC == SRC_PREFIX) {
      q = query_of(a, row / a.G);
    } else if (SRC == SRC_OWN) {
      q = row / a.G < a.max_fresh ? query_at(a, request, row / a.G) : Query{-1, request, -1};
    } else {  // "request" counts (request, query) pairs
      q = query_at(a, request / a.max_fresh, request % a.max_fresh);
      if (row >= a.G) q.token = -1;
    }
    s_limit[tid] = q.token < 0 ? -2 : q.pos;  // -2: no row, -1: a row that sees nothing
    s_row[tid] = q.token < 0 ? -1 : q.token * a.H + g * a.G + hh;
  }
  __syncthreads();
  int most = -2, least = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < COLS; i++) {
    const int x = s_limit[i];
    most = max(most, x);
    if (x > -2) least = min(least, x);
  }
  if (most == -2) return;
  int u0, u1;
  const int prefix_end = a.prefix_pages * a.kv.P;
  if (SRC == SRC_PREFIX) {
    u0 = part * a.prefix_chunk;
    u1 = min(min(u0 + a.prefix_chunk, prefix_end), most + 1);
  } else if (SRC == SRC_OWN) {
    u0 = a.own_begin + part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, most + 1);
    if (u0 >= u1 && !(part == 0 && a.slots == 1) && !a.cluster) return;  // k_attend_join counts the parts by the same rule
  } else {
    u0 = part * a.own_chunk;
    u1 = min(u0 + a.own_chunk, a.budget * a.kv.P);
  }
  // The part's page ids (-1: no page) and, for a list, the pages' first positions.
  const int b0 = (int)a.kv.divP.div(u0);
  __shared__ int s_first[SRC == SRC_LIST ? MM_IDS : 1];
  {
    const int nb = u1 > u0 ? (int)a.kv.divP.div(u1 - 1) - b0 + 1 : 0;
    if (SRC == SRC_LIST) {
      const int token = s_row[0] / a.H;
      const int* list = a.pages + ((int64_t)token * a.KVH + g) * a.budget;
      const int* table = a.tables + (int64_t)(request / a.max_fresh) * a.table_stride;
      for (int e = tid; e < nb; e += MM_WARPS * 32) {
        const int j = list[b0 + e];
        int id = j >= 0 && j < a.width ? table[j] : -1;
        if (id >= a.kv.num_pages) id = -1;
        s_ids[e] = id;
        s_first[e] = id < 0 ? 0 : j * a.kv.P;
      }
    } else {
      const int* ids = SRC == SRC_PREFIX ? a.prefix : a.tables + (int64_t)request * a.table_stride;
      for (int e = tid; e < nb; e += MM_WARPS * 32) {
        const int b = b0 + e;
        int id = SRC == SRC_PREFIX || b < a.width ? ids[b] : -1;
        if (SRC == SRC_OWN && b < a.prefix_pages) id = a.prefix[b];
        if (id >= a.kv.num_pages) id = -1;
        s_ids[e] = id;
      }
    }
  }
  mm_load_queries<TQ, TK, HD, PIECES>(a, qs, s_row, s_scale, COLS, a.scale);
  __syncthreads();
  float o[VG][4][NT][4], m[NT][2], l[NT][2], sc[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      m[t][e] = -INFINITY;
      l[t][e] = 0.f;
      sc[t][e] = s_scale[t * 8 + 2 * c + e];
      lim[t][e] = s_limit[t * 8 + 2 * c + e];
#pragma unroll
      for (int v = 0; v < VG; v++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          o[v][j][t][e] = 0.f;
          o[v][j][t][2 + e] = 0.f;
        }
    }
  const TK* kb = reinterpret_cast<const TK*>(a.kv.k) + (int64_t)g * a.kv.sh;
  const TK* vb = reinterpret_cast<const TK*>(a.kv.v) + (int64_t)g * a.kv.sh;
  const bool aligned = (a.kv.P & 15) == 0;  // a 16-position tile lies in one page
  constexpr int NOWHERE = 0x7ffffff0;       // behind every position, with room for a tile
  for (int ub = u0 + warp * 16; ub < u1; ub += MM_WARPS * 16) {
    // Cache rows: positions r and r + 8 of the tile for K, 2c, 2c + 1, 2c + 8 and 2c + 9 for V.
    int64_t ko[2], vo[4];
    int tk[2], tv[4];
    if (aligned) {
      const int b = (int)a.kv.divP.div(ub), row0 = ub - b * a.kv.P, id = s_ids[b - b0];
      const int64_t base = (int64_t)id * a.kv.sp + (int64_t)row0 * a.kv.st;
      const int t0 = id < 0 ? NOWHERE : SRC == SRC_LIST ? s_first[b - b0] + row0 : ub;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        ko[i] = base + (int64_t)(r + 8 * i) * a.kv.st;
        tk[i] = t0 + r + 8 * i;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int x = 2 * c + (i & 1) + (i >> 1) * 8;
        vo[i] = base + (int64_t)x * a.kv.st;
        tv[i] = t0 + x;
      }
    } else {
      auto at = [&](int u, int64_t& off, int& t) {
        off = 0;
        t = NOWHERE;
        if (u >= u1) return;
        const int b = (int)a.kv.divP.div(u), row = u - b * a.kv.P, id = s_ids[b - b0];
        if (id < 0) return;
        off = (int64_t)id * a.kv.sp + (int64_t)row * a.kv.st;
        t = SRC == SRC_LIST ? s_first[b - b0] + row : u;
      };
#pragma unroll
      for (int i = 0; i < 2; i++) at(ub + r + 8 * i, ko[i], tk[i]);
#pragma unroll
      for (int i = 0; i < 4; i++) at(ub + 2 * c + (i & 1) + (i >> 1) * 8, vo[i], tv[i]);
    }
    // Positions no row sees are not read: whatever lies there stays out of the products.
    uint4 kx[2][KG], vx[VG][4];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int q = 0; q < KG; q++) {
        const int d = q * 32 + c * 8;
        kx[i][q] = tk[i] <= most && d < hd ? ld_stream16(kb + ko[i] + d) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
    for (int v = 0; v < VG; v++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int d = v * 64 + r * 8;
        vx[v][i] = tv[i] <= most && d < hd ? ld_stream16(vb + vo[i] + d) : make_uint4(0, 0, 0, 0);
      }
    // The instruction's additions truncate. Float32 results want better than
    // a chain of them: there each product starts from zero and is added here.
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; t++) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
    for (int q = 0; q < KG; q++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          const uint4 y = *reinterpret_cast<const uint4*>(qs + (p * COLS + t * 8 + r) * QS + q * 32 + c * 8);
          if (PIECES == 1) {
            mma16816<TK>(s[t], kx[0][q].x, kx[1][q].x, kx[0][q].y, kx[1][q].y, y.x, y.y);
            mma16816<TK>(s[t], kx[0][q].z, kx[1][q].z, kx[0][q].w, kx[1][q].w, y.z, y.w);
          } else {
            float u[4] = {}, w[4] = {};
            mma16816<TK>(u, kx[0][q].x, kx[1][q].x, kx[0][q].y, kx[1][q].y, y.x, y.y);
            mma16816<TK>(w, kx[0][q].z, kx[1][q].z, kx[0][q].w, kx[1][q].w, y.z, y.w);
#pragma unroll
            for (int e = 0; e < 4; e++) s[t][e] += u[e] + w[e];
          }
        }
    // Scores in units of log2; rows: positions r (entries 0, 1) and r + 8 (2, 3).
    float alpha[NT][2];
    uint32_t ph[NT][2], pl[NT][2];
    const bool masked = tk[1] > least || tk[0] > least;
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        s[t][e] *= sc[t][e];
        s[t][2 + e] *= sc[t][e];
        if (masked) {
          if (tk[0] > lim[t][e]) s[t][e] = -INFINITY;
          if (tk[1] > lim[t][e]) s[t][2 + e] = -INFINITY;
        }
        float mx = fmaxf(s[t][e], s[t][2 + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = fmaxf(mx, m[t][e]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        alpha[t][e] = ex2(m[t][e] - ref);
        m[t][e] = mx;
        // Two subtractions, so that a large score's rounding cannot lift its weight.
        s[t][e] = ex2((s[t][e] - ref) + weight_bias<TQ, TK>());
        s[t][2 + e] = ex2((s[t][2 + e] - ref) + weight_bias<TQ, TK>());
        l[t][e] = fmaf(l[t][e], alpha[t][e], s[t][e] + s[t][2 + e]);
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t h = pack2<TK>(s[t][2 * i], s[t][2 * i + 1]);
        ph[t][i] = transpose8x8(h);
        if (PIECES == 2) {
          const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&h));
          pl[t][i] = transpose8x8(pack2<TK>(s[t][2 * i] - hf.x, s[t][2 * i + 1] - hf.y));
        }
      }
    }
#pragma unroll
    for (int v = 0; v < VG; v++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t x0 = j == 0 ? vx[v][0].x : j == 1 ? vx[v][0].y : j == 2 ? vx[v][0].z : vx[v][0].w;
        const uint32_t x1 = j == 0 ? vx[v][1].x : j == 1 ? vx[v][1].y : j == 2 ? vx[v][1].z : vx[v][1].w;
        const uint32_t x2 = j == 0 ? vx[v][2].x : j == 1 ? vx[v][2].y : j == 2 ? vx[v][2].z : vx[v][2].w;
        const uint32_t x3 = j == 0 ? vx[v][3].x : j == 1 ? vx[v][3].y : j == 2 ? vx[v][3].z : vx[v][3].w;
        const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
        const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          if (PIECES == 1) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
              o[v][j][t][e] *= alpha[t][e];
              o[v][j][t][2 + e] *= alpha[t][e];
            }
            mma16816<TK>(o[v][j][t], a0, a1, a2, a3, ph[t][0], ph[t][1]);
          } else {
            float u[4] = {};
            mma16816<TK>(u, a0, a1, a2, a3, pl[t][0], pl[t][1]);
            mma16816<TK>(u, a0, a1, a2, a3, ph[t][0], ph[t][1]);
#pragma unroll
            for (int e = 0; e < 2; e++) {
              o[v][j][t][e] = fmaf(o[v][j][t][e], alpha[t][e], u[e]);
              o[v][j][t][2 + e] = fmaf(o[v][j][t][2 + e], alpha[t][e], u[2 + e]);
            }
          }
        }
      }
  }
  // Each lane's sums cover its own positions.
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
    }
  __syncthreads();  // the queries are read
  constexpr int OS = HD + 4;
  float* so = reinterpret_cast<float*>(mm_mem);
  float2* sml = reinterpret_cast<float2*>(so + MM_WARPS * COLS * OS);
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = t * 8 + 2 * c + e;
      float* dst = so + (warp * COLS + col) * OS;
#pragma unroll
      for (int v = 0; v < VG; v++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int d = v * 64 + r * 8 + 2 * j;
          if (d < HD) *reinterpret_cast<float2*>(dst + d) = make_float2(o[v][j][t][e], o[v][j][t][2 + e]);
        }
      if (r == 0) sml[warp * COLS + col] = make_float2(m[t][e], l[t][e]);
    }
  if (SRC != SRC_LIST && least < min(u1 - 1, most)) {  // some row is short of positions that entered its products
    __syncwarp();
    for (int col = 0; col < COLS; col++) {
      if (s_row[col] < 0 || s_limit[col] >= u1 - 1) continue;
      float* dst = so + (warp * COLS + col) * OS;
      bool odd = false;
      for (int d = lane; d < hd; d += 32) odd |= !(fabsf(dst[d]) < INFINITY);
      if (__any_sync(0xffffffffu, odd))
        sum_row<TQ, TK, HD, SRC>(a, s_row[col], g, request, u0 + warp * 16, u1, 16, MM_WARPS * 16, s_limit[col], sml[warp * COLS + col].x, dst);
    }
  }
  __syncthreads();
  const bool direct = a.slots == 1;  // the only part: the output itself
  float* rows = so + MM_WARPS * COLS * (OS + 2);  // this part of the rows, for its cluster
  for (int e = tid; e < COLS * (HD / 4); e += MM_WARPS * 32) {
    const int col = e / (HD / 4), d = (e % (HD / 4)) * 4, row = s_row[col];
    if (row < 0 || d >= hd) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < MM_WARPS; w++) mx = fmaxf(mx, sml[w * COLS + col].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < MM_WARPS; w++) {
      const float2 ml = sml[w * COLS + col];
      const float f = ex2(ml.x - ref);
      const float4 y = *reinterpret_cast<const float4*>(so + (w * COLS + col) * OS + d);
      ls = fmaf(ml.y, f, ls);
      x.x = fmaf(y.x, f, x.x);
      x.y = fmaf(y.y, f, x.y);
      x.z = fmaf(y.z, f, x.z);
      x.w = fmaf(y.w, f, x.w);
    }
    if (a.cluster) {
      float* mine = rows + col * (HD + 2);
      mine[2 + d] = x.x;
      mine[3 + d] = x.y;
      mine[4 + d] = x.z;
      mine[5 + d] = x.w;
      if (d == 0) mine[0] = mx, mine[1] = ls;
    } else if (direct) {
      const float inv = inverse_sum(ls);
      TQ* out = reinterpret_cast<TQ*>(a.out) + (int64_t)(row / a.H) * a.o_ts + (int64_t)(row % a.H) * a.o_hs + d;
      store4(out, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    } else {
      const int64_t slot = (int64_t)row * a.slots + (SRC == SRC_OWN ? a.prefix_slots : 0) + part;
      *reinterpret_cast<float4*>(a.part_o + slot * hd + d) = x;
      if (d == 0) a.part_ml[slot] = make_float2(mx, ls);
    }
  }
  if (a.cluster) cluster_join<TQ>(a, rows, HD + 2, COLS, [&](int r) { return s_row[r]; });
}

template <typename TQ, typename TK, int HD, int NT, int SRC>
__global__ void __launch_bounds__(MM_WARPS * 32, NT == 1 && HD <= 128 ? 4 : NT == 4 || HD > 128 ? 2 : 3) k_attend_mma(const __grid_constant__ AttendArgs a, int row_tiles) {
  overlap_begin(a);
  mm_part<TQ, TK, HD, NT, SRC>(a, row_tiles);
  overlap_end(a);
}

// Float32 scores of pages (16-bit caches): the first product of the attention
// with mean keys in the place of keys, and the same product of magnitudes for
// the error bound. The means' bytes and their latency bound it: 84 MB, 256
// bytes from one place at a time, in 30 us with a tile of 16 pages in flight
// beside the one worked on and four CTAs an SM (45 us with seven CTAs and none
// in flight beside it; 120 us with the scores taken in float64 at once).
// grid: x = request * max_fresh + query, y = KV head, z = page tile.
template <typename TQ, typename TK, int HD>
__global__ void __launch_bounds__(MM_WARPS * 32, HD <= 128 ? 4 : 2) k_page_scores_mma(AttendArgs a, ChooseArgs c) {
  constexpr int PIECES = sizeof(TQ) == 4 ? 2 : 1;
  constexpr int KG = (HD + 31) / 32, QS = HD + 32;
  extern __shared__ __align__(16) uint8_t mm_mem[];  // [PIECES][groups of 8][HD + 32]
  __shared__ int s_row[TCU_PAGED_MAX_GROUP];
  __shared__ float s_scale[TCU_PAGED_MAX_GROUP];
  __shared__ uint32_t s_eps[MM_WARPS];
  TK* qs = reinterpret_cast<TK*>(mm_mem);
  pdl_wait();
  const Query q = query_at(a, blockIdx.x / a.max_fresh, blockIdx.x % a.max_fresh);
  if (q.token < 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, cc = lane & 3;
  const int g = blockIdx.y, hd = a.hd, groups = (a.G + 7) / 8;
  const Candidates cand = candidates_of(a, c, q.pos);
  const int lo = max(cand.lo, (int)blockIdx.z * c.per), hi = min(cand.hi, (int)blockIdx.z * c.per + c.per);
  if (lo >= hi || cand.hi - cand.lo <= c.top) return;  // nothing to choose here
  const int* table = a.tables + (int64_t)q.request * a.table_stride;
  // A warp takes every fourth tile of 16 pages; the next tile's means are on
  // their way while it works on one, and the ids of the one after that.
  constexpr int STEP = 16 * MM_WARPS;
  auto ids = [&](int b0, int (&id)[2]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int b = b0 + r + 8 * i;
      id[i] = b >= lo && b < hi ? table[b] : -1;
      if (id[i] >= a.kv.num_pages) id[i] = -1;
    }
  };
  auto means = [&](const int (&id)[2], uint4 (&x)[2][KG]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const TK* mp = reinterpret_cast<const TK*>(c.means) + ((int64_t)max(id[i], 0) * a.KVH + g) * hd;
#pragma unroll
      for (int k = 0; k < KG; k++) {
        const int d = k * 32 + cc * 8;
        x[i][k] = id[i] >= 0 && d < hd ? ld_stream16(mp + d) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  const int first = blockIdx.z * c.per + warp * 16;
  int id[2], id_next[2], id_after[2];
  uint4 kx[2][KG], kn[2][KG];
  ids(first, id);
  ids(first + STEP, id_next);
  means(id, kx);
  if (tid < groups * 8) s_row[tid] = tid < a.G ? q.token * a.H + g * a.G + tid : -1;
  __syncthreads();
  mm_load_queries<TQ, TK, HD, PIECES>(a, qs, s_row, s_scale, groups * 8, 1.f);
  __syncthreads();
  float most = 0.f;
  for (int b0 = first; b0 < hi; b0 += STEP) {
    means(id_next, kn);
    ids(b0 + 2 * STEP, id_after);
    float best[2] = {-INFINITY, -INFINITY};
    uint32_t nan = 0;
    for (int n = 0; n < groups; n++) {
      float s[4] = {}, z[4] = {};
#pragma unroll
      for (int k = 0; k < KG; k++)
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          const uint4 y = *reinterpret_cast<const uint4*>(qs + (p * groups * 8 + n * 8 + r) * QS + k * 32 + cc * 8);
          const uint4 u = kx[0][k], v = kx[1][k];
          constexpr uint32_t M = 0x7fff7fffu;
          mma16816<TK>(s, u.x, v.x, u.y, v.y, y.x, y.y);
          mma16816<TK>(s, u.z, v.z, u.w, v.w, y.z, y.w);
          mma16816<TK>(z, u.x & M, v.x & M, u.y & M, v.y & M, y.x & M, y.y & M);
          mma16816<TK>(z, u.z & M, v.z & M, u.w & M, v.w & M, y.z & M, y.w & M);
        }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int col = n * 8 + 2 * cc + (e & 1);
        if (col < a.G) {
          const float x = s[e] * s_scale[col], w = z[e] * s_scale[col];
          if (!(x == x)) nan |= 1u << (e >> 1);
          best[e >> 1] = fmaxf(best[e >> 1], x);
          most = w > most || !(w == w) ? w : most;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], o));
        nan |= __shfl_xor_sync(0xffffffffu, nan, o);
      }
      const int b = b0 + r + 8 * i;
      if (cc == 0 && b >= lo && b < hi) c.scores[((int64_t)q.token * a.KVH + g) * c.width + b] = id[i] >= 0 && !(nan >> i & 1) ? best[i] : NAN;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      id[i] = id_next[i];
      id_next[i] = id_after[i];
#pragma unroll
      for (int k = 0; k < KG; k++) kx[i][k] = kn[i][k];
    }
  }
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
  if (lane == 0) s_eps[warp] = w;
  __syncthreads();
  if (tid == 0) {
    uint32_t x = 0;
    for (int i = 0; i < MM_WARPS; i++) x = max(x, s_eps[i]);
    float scale = 0.f;  // of the coarsest split
    if (PIECES == 2)
      for (int i = 0; i < a.G; i++) scale = fmaxf(scale, s_scale[i]);
    c.eps[((int64_t)q.token * a.KVH + g) * c.tiles + blockIdx.z] = score_error(__uint_as_float(x), hd, scale);
  }
}

}  // namespace tcu
