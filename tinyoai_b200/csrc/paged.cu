// Host side of the paged-cache operators declared in include/tinyoai_cuda.h
// (section "Operators over a paged KV cache the caller holds"): argument
// checks, kernel selection, workspace layout and launches. Nothing here
// allocates, synchronises or keeps anything between calls.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "../../include/tinyoai_cuda.h"
#include "paged.cuh"
#include "paged_mma.cuh"
#include "paged_tc.cuh"
#include "status.h"
#include "tma_host.h"

using namespace tcu;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

#define TRY(x)                   \
  do {                           \
    int r_ = (x);                \
    if (r_ != TCU_OK) return r_; \
  } while (0)
#define CK(x)                                                                                                        \
  do {                                                                                                               \
    cudaError_t e_ = (x);                                                                                            \
    if (e_ != cudaSuccess) return fail(TCU_ECUDA, "%s (%s:%d): %s", #x, __FILE__, __LINE__, cudaGetErrorString(e_)); \
  } while (0)

// Makes `device` current for one call and puts the caller's device back.
struct OnDevice {
  int before = -1, rc = TCU_OK;
  explicit OnDevice(int device) {
    rc = require_device(device);
    if (rc != TCU_OK) return;
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != device) {
      before = cur;
      if (cudaSetDevice(device) != cudaSuccess) rc = fail(TCU_ECUDA, "device %d cannot be made current", device);
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// A pointer the kernels read or write: memory of this device, aligned.
int check_ptr(const char* name, const void* p, int device, size_t align) {
  if (!p) return fail(TCU_EINVAL, "%s is null", name);
  if (reinterpret_cast<uintptr_t>(p) % align) return fail(TCU_EINVAL, "%s is not %zu-byte aligned", name, align);
  cudaPointerAttributes pa;
  cudaError_t e = cudaPointerGetAttributes(&pa, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TCU_EINVAL, "%s: %s", name, cudaGetErrorString(e));
  }
  if ((pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged) || pa.device != device)
    return fail(TCU_EINVAL, "%s must be device memory on device %d", name, device);
  return TCU_OK;
}

// Whether two of n1 x n2 rows of `hd` values, s1 and s2 apart, share values.
bool rows_overlap(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t hd) {
  if (n1 < 2) s1 = 0;
  if (n2 < 2) s2 = 0;
  if (s1 > s2) std::swap(s1, s2), std::swap(n1, n2);
  if ((n1 > 1 && s1 < hd) || (n2 > 1 && s2 < hd)) return true;
  // Rows i s1 and j s2 meet where they are nearer than hd: none do where the
  // steps of s2 pass all rows of s1, the common case.
  for (int64_t j = 1; n1 > 1 && j < n2 && j * s2 < (n1 - 1) * s1 + hd; j++) {
    const int64_t r = j * s2 % s1;
    if (r < hd || (s1 - r < hd && j * s2 / s1 + 1 < n1)) return true;
  }
  return false;
}

// Rows read and rows written of one call: `dims` of them in each dimension,
// `from` and `to` apart, of r and w bytes. False where they are known to share
// bytes without being the same rows (each is then read before it is written):
// decided for steps that agree, which views of one buffer have.
struct Rows {
  const void* at;
  int64_t step[2];  // bytes
  int64_t bytes;
};
bool same_or_apart(const Rows& in, const Rows& out, const int64_t (&dims)[2]) {
  int64_t end_in = in.bytes, end_out = out.bytes;
  bool equal = true;
  for (int i = 0; i < 2; i++) {
    end_in += (dims[i] - 1) * in.step[i];
    end_out += (dims[i] - 1) * out.step[i];
    equal = equal && (dims[i] == 1 || in.step[i] == out.step[i]);
  }
  const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(out.at) - reinterpret_cast<uintptr_t>(in.at));
  if (d == 0 || d >= end_in || -d >= end_out || !equal) return true;
  // Row (i, j) of the output begins d + di s0 + dj s1 behind one of the input.
  const int64_t s0 = dims[0] > 1 ? out.step[0] : 0, s1 = dims[1] > 1 ? out.step[1] : 0;
  for (int64_t dj = -(dims[1] - 1); dj < dims[1]; dj++) {
    const int64_t rest = d + dj * s1;
    const int64_t near = s0 > 0 ? -rest / s0 : 0;
    for (int64_t di = near - 1; di <= near + 1; di++) {
      if (di <= -dims[0] || di >= dims[0]) continue;
      const int64_t gap = rest + di * s0;
      if (gap < in.bytes && -gap < out.bytes) return false;
    }
  }
  return true;
}

int elem_bytes(int dtype) { return dtype == TCU_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == TCU_F32 || dtype == TCU_F16 || dtype == TCU_BF16; }

// Rows are the cache's type, or float32 over a binary16 cache (what the
// models of this library compute and store).
int check_pair(int rows, int cache) {
  if (!dtype_ok(rows) || !dtype_ok(cache)) return fail(TCU_EUNSUP, "paged operators take float32, binary16 and bfloat16 values");
  if (rows != cache && !(rows == TCU_F32 && cache == TCU_F16))
    return fail(TCU_EUNSUP, "rows have the cache's type, or are float32 over a binary16 cache");
  return TCU_OK;
}

int check_kv(const tcu_paged_kv* kv) {
  if (!kv) return fail(TCU_EINVAL, "null cache");
  if (!dtype_ok(kv->dtype)) return fail(TCU_EUNSUP, "paged operators take float32, binary16 and bfloat16 values");
  if (kv->num_pages < 1 || kv->page_tokens < 1 || kv->kv_heads < 1) return fail(TCU_EINVAL, "the cache has no pages, positions or heads");
  if (kv->page_tokens > TCU_PAGED_MAX_PAGE_TOKENS) return fail(TCU_EINVAL, "%d positions a page, at most %d", kv->page_tokens, TCU_PAGED_MAX_PAGE_TOKENS);
  if (kv->kv_heads > 65535) return fail(TCU_EINVAL, "%d KV heads, at most 65535", kv->kv_heads);
  if (kv->head_dim < 8 || kv->head_dim > TCU_PAGED_MAX_HEAD_DIM || kv->head_dim % 8)
    return fail(TCU_EUNSUP, "head size %d is not a multiple of 8 in 8..%d", kv->head_dim, TCU_PAGED_MAX_HEAD_DIM);
  const int64_t per16 = 16 / elem_bytes(kv->dtype);
  if (kv->page_stride < 0 || kv->head_stride < 0 || kv->token_stride < 0) return fail(TCU_EINVAL, "negative cache stride");
  if (kv->page_stride % per16 || kv->head_stride % per16 || kv->token_stride % per16)
    return fail(TCU_EINVAL, "cache strides must be multiples of 16 bytes");
  return TCU_OK;
}

PagedView view_of(const tcu_paged_kv* kv) {
  PagedView v;
  v.k = kv->k;
  v.v = kv->v;
  v.num_pages = kv->num_pages;
  v.P = kv->page_tokens;
  v.kvh = kv->kv_heads;
  v.hd = kv->head_dim;
  v.sp = kv->page_stride;
  v.sh = kv->head_stride;
  v.st = kv->token_stride;
  v.divP = FastDiv::of((uint32_t)kv->page_tokens);
  v.small = (int64_t)kv->num_pages * kv->page_tokens < 0x7fffffffll;
  return v;
}

// Queues a kernel that may start while the one before it on the stream
// drains (every kernel here waits for that one before it reads, paged.cuh), in
// clusters of `cluster` CTAs along z. carveout: the share of an SM's cache that
// this launch wants as shared memory (percent, -1: left to the driver).
template <typename... P, typename... A>
int launch_cluster(const char* name, void (*kern)(P...), dim3 grid, int cluster, int carveout, int block, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[3];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    cudaLaunchAttribute& c = attr[cfg.numAttrs++];
    c.id = cudaLaunchAttributeClusterDimension;
    c.val.clusterDim.x = c.val.clusterDim.y = 1;
    c.val.clusterDim.z = (unsigned)cluster;
  }
  if (carveout >= 0) {
    cudaLaunchAttribute& c = attr[cfg.numAttrs++];
    c.id = cudaLaunchAttributePreferredSharedMemoryCarveout;
    c.val.sharedMemCarveout = (unsigned)carveout;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TCU_ECUDA, "%s: %s", name, cudaGetErrorString(e));
  }
  return TCU_OK;
}

template <typename... P, typename... A>
int launch(const char* name, void (*kern)(P...), dim3 grid, int block, size_t smem, cudaStream_t s, const A&... args) {
  return launch_cluster(name, kern, grid, 1, -1, block, smem, s, args...);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int SM_COUNT = 148;  // B200

// ---------------------------------------------------------------------------
// Append

template <typename TQ, typename TK>
int launch_append(const AppendArgs& a, cudaStream_t s) {
  const int heads = a.H + 2 * a.KVH;
  auto go = [&](auto kern, int lph) {
    // A CTA takes all heads of a token where there are tokens enough to fill
    // the GPU, otherwise as many as its groups of lanes hold at once; three
    // CTAs an SM go through the tokens.
    const int groups = APPEND_THREADS / lph;
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(ceil_div(heads, groups), ceil_div(8 * SM_COUNT, a.T)));
    const int per = (int)(ceil_div(ceil_div(heads, shares), groups) * groups);
    const int64_t y = ceil_div(heads, per), x = std::min<int64_t>(a.T, std::max<int64_t>(1, 3 * SM_COUNT / y));
    return launch("k_append", kern, dim3((unsigned)x, (unsigned)y), APPEND_THREADS, 0, s, a, per);
  };
  auto pick_norm = [&](auto turn, auto norm) {
    constexpr int TURN = decltype(turn)::value, NORM = decltype(norm)::value;
    if (a.hd <= 64) return go(k_append<TQ, TK, 8, TURN, NORM>, 8);
    if (a.hd <= 128) return go(k_append<TQ, TK, 16, TURN, NORM>, 16);
    return go(k_append<TQ, TK, 32, TURN, NORM>, 32);
  };
  auto pick = [&](auto turn) {
    if (a.norm == NORM_RMS) return pick_norm(turn, std::integral_constant<int, NORM_RMS>());
    if (a.norm == NORM_LAYER) return pick_norm(turn, std::integral_constant<int, NORM_LAYER>());
    return pick_norm(turn, std::integral_constant<int, NORM_NONE>());
  };
  if (a.pairs == 0) return pick(std::integral_constant<int, TURN_NONE>());
  if (a.adjacent) return pick(std::integral_constant<int, TURN_BESIDE>());
  if (a.pairs % 4 == 0) return pick(std::integral_constant<int, TURN_RUNS>());
  return pick(std::integral_constant<int, TURN_SHARED>());
}

template <typename TK>
int launch_means(const MeansArgs& a, cudaStream_t s) {
  if (ceil_div(a.T, 128) * a.kv.kvh < 2 * SM_COUNT)
    return launch("k_page_means", k_page_means<TK, 4>, dim3((unsigned)ceil_div(a.T, 32), a.kv.kvh), 128, 0, s, a);
  return launch("k_page_means", k_page_means<TK, 1>, dim3((unsigned)ceil_div(a.T, 128), a.kv.kvh), 128, 0, s, a);
}

// ---------------------------------------------------------------------------
// Attention

// Positions of a request in attention: the end of a part, up to as long again,
// stays a 32-bit number.
constexpr int64_t MAX_POSITIONS = 1ll << 30;

struct AttendPlan {
  int prefix_rows = 0, prefix_chunk = 0, prefix_slots = 0, own_rows = 0, own_chunk = 0, own_slots = 0, slots = 0;
  bool tc = false;      // the prefix on tcgen05
  bool cluster = false; // the parts of a row are joined within a cluster
  int own_begin = 0;
  int score_per = 64, score_tiles = 0;  // pages of a scoring CTA, and such shares of a table
  PagedTcArgs tc_args{};
  int tc_tiles = 0, tc_parts = 0;
  size_t part_o = 0, part_ml = 0, keys = 0, scores = 0, eps = 0, bytes = 0;  // offsets of the workspace regions, and their size
};


// Positions per part: enough CTAs for four on each SM, but parts of at least
// 128 positions, whose own cost (its queries, its partial) a shorter one
// would not earn back, and of at most MM_IDS pages.
int chunk_of(int64_t positions, int64_t ctas_per_part, int P) {
  const int64_t want = std::max<int64_t>(1, 4LL * SM_COUNT / std::max<int64_t>(1, ctas_per_part));
  int64_t c = std::max<int64_t>(128, ceil_div(ceil_div(positions, want), 64) * 64);
  // Up to 4,096 positions: eight parts at most, which a cluster joins.
  if (positions <= 4096) c = std::max<int64_t>(c, ceil_div(ceil_div(positions, 8), 64) * 64);
  c = std::min<int64_t>(c, std::max<int64_t>(64, (int64_t)(MM_IDS - 2) * P / 64 * 64));
  return (int)std::min<int64_t>(c, MAX_POSITIONS);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Query rows a CTA takes: CUDA cores 4 (their state lives in registers, hd
// values each), matrix instructions 8, 16 or 32.
int rows_per_cta(const tcu_paged_kv* kv, int64_t rows) {
  if (kv->dtype == TCU_F32) return kv->head_dim <= 128 ? 4 : 2;
  if (rows <= 8) return 8;
  return rows <= 16 || kv->head_dim > 128 ? 16 : 32;
}

// Whether the prefix goes to k_attend_prefix_tc, and how it is cut. The kernel
// takes 16-bit rows and caches of one type, head sizes 64..128, pages that
// tile 128 positions (or that 128 positions tile), strides TMA can describe,
// and is worth its set-up from TC_MIN_ROWS rows and TC_MIN_BLOCKS blocks on.
constexpr int TC_MIN_ROWS = 33, TC_MIN_BLOCKS = 4;

void plan_tc(const tcu_paged_kv* kv, const tcu_paged_queries* q, int prefix_pages, AttendPlan* p) {
  const int P = kv->page_tokens, hd = kv->head_dim;
  const int64_t rows = (int64_t)q->rows * (q->heads / kv->kv_heads), shared = (int64_t)prefix_pages * P;
  const int64_t blocks = ceil_div(shared, PT_KEYS);
  if (kv->dtype == TCU_F32 || q->dtype != kv->dtype || hd < 64 || hd > 128 || P % 8 || (P <= PT_KEYS ? PT_KEYS % P : P % PT_KEYS)) return;
  if (rows < TC_MIN_ROWS || blocks < TC_MIN_BLOCKS) return;
  const int64_t strides[3] = {kv->token_stride, kv->head_stride, kv->page_stride};
  const int64_t dims[3] = {P, kv->kv_heads, kv->num_pages};
  for (int i = 0; i < 3; i++)
    if (strides[i] * 2 >= (1LL << 40) || (dims[i] > 1 && strides[i] == 0)) return;
  p->tc = true;
  const int split = rows <= PT_ROWS;
  p->tc_tiles = (int)ceil_div(rows, split ? PT_ROWS : 2 * PT_ROWS);
  const int64_t units = (int64_t)p->tc_tiles * kv->kv_heads;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)(PT_IDS - 2) * P / PT_KEYS));
  // Blocks per part: waves of one CTA per SM, three blocks' worth of set-up,
  // and the join's traffic of every part. A block takes 1.3 us on an SM whose
  // products never wait (half of that where the streams share the blocks) and
  // about 2.5 as they do, but with 2.5 second waves look cheaper than they are:
  // 256 requests over 32,768 positions take 175 us in 4 parts (128 CTAs) and 191
  // in the 9 (288 CTAs, 2 waves) that 2.5 would choose, 242 and 272 with up to
  // 1,024 positions of their own each, which run on the SMs left over (times in
  // a graph); the seven other shapes tried chose the same parts with both.
  double best = 1e30;
  const double join = 1e-6 * q->rows * q->heads * hd * 8 / 4.0 * (split ? 2 : 1);  // us a part at 4 TB/s
  for (int64_t parts = ceil_div(blocks, most); parts <= std::min<int64_t>(blocks, ceil_div(blocks, most) + 64); parts++) {
    const int64_t per = ceil_div(blocks, parts), real = ceil_div(blocks, per);
    const double us = (double)ceil_div(units * real, SM_COUNT) * (1.3 * (split ? ceil_div(per, 2) : per) + 4.0) + join * real;
    if (us < best) {
      best = us;
      p->tc_args.per = (int)per;
      p->tc_parts = (int)real;
    }
  }
  const int sub = hd > 64 ? 2 : 1;
  p->tc_args.blocks = (int)blocks;
  p->tc_args.split_keys = split;
  p->tc_args.stages = sub == 2 ? 2 : 4;
  p->tc_args.box = std::min(P, PT_KEYS);
  p->tc_args.hdp = (hd + 15) / 16 * 16;
  p->prefix_slots = p->tc_parts * (split ? 2 : 1);
}

AttendPlan plan_attend(const tcu_paged_kv* kv, const tcu_paged_queries* q, int prefix_pages, int max_length, int budget) {
  AttendPlan p;
  const int G = q->heads / kv->kv_heads, P = kv->page_tokens;
  const int64_t T = q->rows;
  if (budget > 0) {
    p.own_rows = rows_per_cta(kv, G);
    const int64_t most = (int64_t)std::max(1, std::min(budget, q->table_width)) * P;  // a list holds no more pages than a table
    p.own_chunk = chunk_of(most, T * kv->kv_heads * ceil_div(G, p.own_rows), P);
    p.own_slots = (int)ceil_div(most, p.own_chunk);
  } else {
    const int64_t shared = (int64_t)prefix_pages * P;
    p.prefix_rows = rows_per_cta(kv, T * G);
    p.own_rows = rows_per_cta(kv, (int64_t)q->max_fresh * G);
    plan_tc(kv, q, prefix_pages, &p);
    const int64_t own_tiles = (int64_t)q->requests * ceil_div((int64_t)q->max_fresh * G, p.own_rows);
    if (shared > 0 && !p.tc) {
      // One kernel over each request's whole history reads the prefix
      // own_tiles times through L2, a kernel of its own for the prefix
      // prefix_tiles times, and costs a launch and a join: about 6 us, in
      // which L2 moves some 32 MB.
      const int64_t prefix_tiles = ceil_div(T * G, p.prefix_rows), bytes = 2 * shared * kv->kv_heads * kv->head_dim * elem_bytes(kv->dtype);
      if ((own_tiles - prefix_tiles) * bytes > (32 << 20)) {
        p.prefix_chunk = chunk_of(shared, prefix_tiles * kv->kv_heads, P);
        p.prefix_slots = (int)ceil_div(shared, p.prefix_chunk);
      }
    }
    p.own_begin = p.prefix_slots > 0 ? (int)shared : 0;
    const int64_t own = std::max<int64_t>(0, (int64_t)max_length - p.own_begin);
    p.own_chunk = chunk_of(own, own_tiles * kv->kv_heads, P);
    p.own_slots = (int)ceil_div(own, p.own_chunk);
  }
  // Up to eight parts of one kernel: a cluster joins them.
  p.cluster = p.prefix_slots == 0 && p.own_slots > 1 && p.own_slots <= 8;
  p.slots = std::max(1, p.prefix_slots + p.own_slots);
  size_t off = 0;
  const size_t rows = (p.slots > 1 && !p.cluster) || p.tc ? (size_t)T * q->heads : 0;
  p.part_o = off;
  off += align256(rows * p.slots * kv->head_dim * sizeof(float));
  p.part_ml = off;
  off += align256(rows * p.slots * sizeof(float2));
  if (budget > 0) {
    p.keys = off;
    const size_t lists = (size_t)T * kv->kv_heads;
    off += align256(lists * q->table_width * sizeof(unsigned long long));
    p.scores = off;
    off += align256(lists * q->table_width * sizeof(float));
    p.eps = off;
    // Scoring CTAs: up to four for each SM (its room), of 64 pages at least.
    const int64_t shares = std::max<int64_t>(1, 4 * SM_COUNT / std::max<int64_t>(1, (int64_t)lists));
    p.score_per = (int)(ceil_div(std::max<int64_t>(1, ceil_div(q->table_width, shares)), 64) * 64);
    p.score_tiles = (int)ceil_div(q->table_width, p.score_per);
    off += align256(lists * p.score_tiles * sizeof(float));
  }
  p.bytes = off;
  return p;
}

// x of the grid and row tiles for CTAs of `rows` rows.
template <int SRC>
int64_t grid_x(const AttendArgs& a, int rows, int* tiles) {
  if (SRC == SRC_PREFIX) {
    *tiles = (int)ceil_div((int64_t)a.T * a.G, rows);
    return *tiles;
  }
  *tiles = (int)ceil_div(SRC == SRC_OWN ? (int64_t)a.max_fresh * a.G : a.G, rows);
  return (int64_t)a.n * (SRC == SRC_OWN ? 1 : a.max_fresh) * *tiles;
}

// Once per kernel and device: lets the kernel have up to `most` bytes of
// dynamic shared memory.
template <auto Kern>
int prepare_kernel(size_t most) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  CK(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return TCU_OK;
  CK(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  done.fetch_or(bit, std::memory_order_release);
  return TCU_OK;
}

template <int NCH, int R, int SRC>
int launch_cc_r(const AttendArgs& a, int parts, cudaStream_t s) {
  int tiles;
  const int64_t x = grid_x<SRC>(a, R, &tiles);
  const size_t smem = sizeof(float) * (CC_GROUPS + (a.cluster ? R : 0)) * (NCH * 32 + 2);
  return launch_cluster("k_attend_cc", k_attend_cc<NCH, R, SRC>, dim3((unsigned)x, a.KVH, parts), a.cluster ? parts : 1, -1, CC_WARPS * 32, smem, s, a, tiles);
}

template <typename TQ, typename TK, int HD, int NT, int SRC>
int launch_mma_n(const AttendArgs& a, int parts, cudaStream_t s) {
  int tiles;
  const int64_t x = grid_x<SRC>(a, 8 * NT, &tiles);
  const size_t smem = mm_smem<HD, NT, sizeof(TQ) == 4 ? 2 : 1>(a.cluster);
  constexpr auto kern = k_attend_mma<TQ, TK, HD, NT, SRC>;
  TRY((prepare_kernel<kern>(mm_smem<HD, NT, sizeof(TQ) == 4 ? 2 : 1>(true))));
  // Beside the prefix's kernel: half of the cache as shared memory, which this
  // kernel's own four CTAs fill: 256 requests over 32,768 shared positions take
  // 242 us in a graph, with the driver's choice 271, with all of it (no cache left for its
  // loads) 282. Alone it is left to the driver: half would keep a second CTA of
  // the larger variants off an SM (64 requests of 2,048 positions, heads of 256
  // in groups of 16: 219 us, 130 so).
  return launch_cluster("k_attend_mma", kern, dim3((unsigned)x, a.KVH, parts), a.cluster ? parts : 1, a.overlap ? 50 : -1, MM_WARPS * 32, smem, s, a, tiles);
}

template <typename TQ, typename TK, int HD, int SRC>
int launch_mma(const AttendArgs& a, int rows, int parts, cudaStream_t s) {
  if (rows == 8) return launch_mma_n<TQ, TK, HD, 1, SRC>(a, parts, s);
  if (rows == 16) return launch_mma_n<TQ, TK, HD, 2, SRC>(a, parts, s);
  if constexpr (HD <= 128) return launch_mma_n<TQ, TK, HD, 4, SRC>(a, parts, s);
  return fail(TCU_EINVAL, "no kernel for %d rows", rows);
}

// The parts of one source of positions: CUDA cores for float32 caches, matrix
// instructions for 16-bit ones.
template <typename TQ, typename TK, int SRC>
int launch_parts(const AttendArgs& a, int rows, int parts, cudaStream_t s) {
  if (parts == 0) return TCU_OK;
  if constexpr (sizeof(TK) == 4) {
    const int nch = (a.hd + 31) / 32;
    if (nch <= 2) return launch_cc_r<2, 4, SRC>(a, parts, s);
    if (nch <= 3) return launch_cc_r<3, 4, SRC>(a, parts, s);
    if (nch <= 4) return launch_cc_r<4, 4, SRC>(a, parts, s);
    return launch_cc_r<8, 2, SRC>(a, parts, s);
  } else {
    if (a.hd <= 64) return launch_mma<TQ, TK, 64, SRC>(a, rows, parts, s);
    if (a.hd <= 96) return launch_mma<TQ, TK, 96, SRC>(a, rows, parts, s);
    if (a.hd <= 128) return launch_mma<TQ, TK, 128, SRC>(a, rows, parts, s);
    return launch_mma<TQ, TK, 256, SRC>(a, rows, parts, s);
  }
}

// The cache as a tensor of [features, positions, heads, pages] and 64 x box x 1 x 1 boxes.
int cache_map(CUtensorMap* map, const AttendArgs& a, void* base, int box, bool is_bf16) {
  const auto encode = tensor_map_encoder();
  if (!encode) return fail(TCU_ECUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[4] = {(cuuint64_t)a.hd, (cuuint64_t)a.kv.P, (cuuint64_t)a.kv.kvh, (cuuint64_t)a.kv.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)a.kv.st * 2, (cuuint64_t)a.kv.sh * 2, (cuuint64_t)a.kv.sp * 2};
  for (int i = 0; i < 3; i++)
    if (dims[i + 1] == 1 && strides[i] == 0) strides[i] = 16;  // a dimension of one has no step
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, boxes, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TCU_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return TCU_OK;
}

template <typename T>
int launch_prefix_tc(const AttendArgs& a, const AttendPlan& p, cudaStream_t s) {
  CUtensorMap km, vm;
  const bool is_bf16 = std::is_same<T, bf16>::value;
  TRY(cache_map(&km, a, a.kv.k, p.tc_args.box, is_bf16));
  TRY(cache_map(&vm, a, a.kv.v, p.tc_args.box, is_bf16));
  const int sub = a.hd > 64 ? 2 : 1;
  const size_t smem = pt_smem(sub, p.tc_args.split_keys, p.tc_args.stages);
  const dim3 grid(p.tc_tiles, a.KVH, p.tc_parts);
  if (sub == 2) {
    TRY((prepare_kernel<k_attend_prefix_tc<T, 2>>(PT_MAX_SMEM)));
    return launch("k_attend_prefix_tc", k_attend_prefix_tc<T, 2>, grid, PT_THREADS, smem, s, a, p.tc_args, km, vm);
  }
  TRY((prepare_kernel<k_attend_prefix_tc<T, 1>>(PT_MAX_SMEM)));
  return launch("k_attend_prefix_tc", k_attend_prefix_tc<T, 1>, grid, PT_THREADS, smem, s, a, p.tc_args, km, vm);
}

template <typename TQ, typename TK>
int launch_attend(AttendArgs a, const AttendPlan& p, cudaStream_t s) {
  if (p.tc) {
    if constexpr (std::is_same<TQ, TK>::value && sizeof(TK) == 2) TRY(launch_prefix_tc<TK>(a, p, s));
  } else {
    TRY((launch_parts<TQ, TK, SRC_PREFIX>(a, p.prefix_rows, p.prefix_slots, s)));
  }
  a.overlap = p.tc;
  TRY((launch_parts<TQ, TK, SRC_OWN>(a, p.own_rows, p.own_slots, s)));
  if (p.cluster || (!p.tc && p.prefix_slots + p.own_slots == 1)) return TCU_OK;  // the output is written
  return launch("k_attend_join", k_attend_join<TQ, 0>, dim3((unsigned)((int64_t)a.n * a.max_fresh), (a.H + 3) / 4), 128, 0, s, a);
}

int launch_scores_cc(const AttendArgs& a, const ChooseArgs& c, unsigned queries, cudaStream_t s) {
  TRY((prepare_kernel<k_page_scores_cc>(sizeof(float) * TCU_PAGED_MAX_GROUP * TCU_PAGED_MAX_HEAD_DIM)));
  return launch("k_page_scores_cc", k_page_scores_cc, dim3(queries, a.KVH, c.tiles), 128, sizeof(float) * a.G * a.hd, s, a, c);
}

template <typename TQ, typename TK, int HD>
int launch_scores(const AttendArgs& a, const ChooseArgs& c, unsigned queries, cudaStream_t s) {
  constexpr size_t row = (sizeof(TQ) == 4 ? 2 : 1) * (HD + 32) * 2;
  TRY((prepare_kernel<k_page_scores_mma<TQ, TK, HD>>(row * TCU_PAGED_MAX_GROUP)));
  return launch("k_page_scores_mma", k_page_scores_mma<TQ, TK, HD>, dim3(queries, a.KVH, c.tiles), MM_WARPS * 32, row * ((a.G + 7) / 8 * 8), s, a, c);
}

template <typename TQ, typename TK>
int launch_sparse(const AttendArgs& a, const ChooseArgs& c, const AttendPlan& p, cudaStream_t s) {
  const unsigned queries = (unsigned)((int64_t)a.n * a.max_fresh);
  // No query has more than width pages: with room for all, none is scored.
  if (c.top > 0 && c.width - c.first - c.last > c.top) {
    if constexpr (sizeof(TK) == 4)
      TRY(launch_scores_cc(a, c, queries, s));
    else if (a.hd <= 64)
      TRY((launch_scores<TQ, TK, 64>(a, c, queries, s)));
    else if (a.hd <= 96)
      TRY((launch_scores<TQ, TK, 96>(a, c, queries, s)));
    else if (a.hd <= 128)
      TRY((launch_scores<TQ, TK, 128>(a, c, queries, s)));
    else
      TRY((launch_scores<TQ, TK, 256>(a, c, queries, s)));
  }
  const size_t cache = sizeof(uint32_t) * std::min(c.width, CHOOSE_CACHE);
  if (c.width <= 1024)
    TRY((launch("k_page_choose", k_page_choose<TQ, TK, 256>, dim3(queries, a.KVH), 256, cache, s, a, c)));
  else
    TRY((launch("k_page_choose", k_page_choose<TQ, TK, 1024>, dim3(queries, a.KVH), 1024, cache, s, a, c)));
  TRY((launch_parts<TQ, TK, SRC_LIST>(a, p.own_rows, p.own_slots, s)));
  if (p.cluster || p.own_slots == 1) return TCU_OK;  // the output is written
  return launch("k_attend_join", k_attend_join<TQ, 1>, dim3(queries, (a.H + 3) / 4), 128, 0, s, a);
}

int check_queries(const tcu_paged_kv* kv, const tcu_paged_queries* q) {
  if (!q) return fail(TCU_EINVAL, "null queries");
  TRY(check_pair(q->dtype, kv->dtype));
  if (q->requests < 0 || q->rows < 0 || q->table_width < 0) return fail(TCU_EINVAL, "negative count");
  if (q->heads < 1 || q->heads % kv->kv_heads) return fail(TCU_EINVAL, "%d query heads over %d KV heads", q->heads, kv->kv_heads);
  if (q->heads / kv->kv_heads > TCU_PAGED_MAX_GROUP) return fail(TCU_EUNSUP, "%d query heads a KV head, at most %d", q->heads / kv->kv_heads, TCU_PAGED_MAX_GROUP);
  if (q->max_fresh < 1) return fail(TCU_EINVAL, "max_fresh %d", q->max_fresh);
  if (q->table_stride < q->table_width) return fail(TCU_EINVAL, "table stride %lld below the width %d", (long long)q->table_stride, q->table_width);
  if ((int64_t)q->table_width * kv->page_tokens > MAX_POSITIONS) return fail(TCU_EINVAL, "tables of %d pages pass 2^30 positions", q->table_width);
  const int G = q->heads / kv->kv_heads;
  if ((int64_t)q->requests * q->max_fresh * G > 0x7fffffffll || (int64_t)q->rows * q->heads > 0x7fffffffll)
    return fail(TCU_EINVAL, "too many rows for one call");
  const int64_t per16 = 16 / elem_bytes(q->dtype);
  if (q->q_token_stride % per16 || q->q_head_stride % per16 || q->out_token_stride % per16 || q->out_head_stride % per16)
    return fail(TCU_EINVAL, "query and output strides must be multiples of 16 bytes");
  if (q->q_token_stride < 0 || q->q_head_stride < 0 || q->out_token_stride < 0 || q->out_head_stride < 0) return fail(TCU_EINVAL, "negative query stride");
  if (rows_overlap(q->rows, q->out_token_stride, q->heads, q->out_head_stride, kv->head_dim)) return fail(TCU_EINVAL, "output rows overlap");
  if (!(q->scale == q->scale)) return fail(TCU_EINVAL, "scale is not a number");
  return TCU_OK;
}

int check_query_ptrs(const tcu_paged_kv* kv, const tcu_paged_queries* q, int device) {
  TRY(check_ptr("k", kv->k, device, 16));
  TRY(check_ptr("v", kv->v, device, 16));
  TRY(check_ptr("q", q->q, device, 16));
  TRY(check_ptr("out", q->out, device, 16));
  TRY(check_ptr("starts", q->starts, device, 4));
  TRY(check_ptr("lengths", q->lengths, device, 4));
  if (q->table_width > 0) TRY(check_ptr("tables", q->tables, device, 4));
  const int64_t es = elem_bytes(q->dtype), dims[2] = {q->rows, q->heads};
  if (!same_or_apart(Rows{q->q, {q->q_token_stride * es, q->q_head_stride * es}, kv->head_dim * es},
                     Rows{q->out, {q->out_token_stride * es, q->out_head_stride * es}, kv->head_dim * es}, dims))
    return fail(TCU_EINVAL, "out overlaps q");
  return TCU_OK;
}

AttendArgs attend_args(const tcu_paged_kv* kv, const tcu_paged_queries* q, const AttendPlan& p, void* workspace) {
  AttendArgs a{};
  a.n = q->requests;
  a.T = q->rows;
  a.H = q->heads;
  a.KVH = kv->kv_heads;
  a.G = q->heads / kv->kv_heads;
  a.hd = kv->head_dim;
  a.max_fresh = q->max_fresh;
  a.q = q->q;
  a.q_ts = q->q_token_stride;
  a.q_hs = q->q_head_stride;
  a.out = q->out;
  a.o_ts = q->out_token_stride;
  a.o_hs = q->out_head_stride;
  a.starts = q->starts;
  a.lengths = q->lengths;
  a.tables = q->tables;
  a.table_stride = q->table_stride;
  a.width = q->table_width;
  a.scale = (float)((double)q->scale * 1.4426950408889634);
  a.kv = view_of(kv);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(w + p.part_o);
  a.part_ml = reinterpret_cast<float2*>(w + p.part_ml);
  a.slots = p.slots;
  a.prefix_slots = p.prefix_slots;
  a.prefix_chunk = p.prefix_chunk;
  a.own_chunk = p.own_chunk;
  a.own_begin = p.own_begin;
  a.cluster = p.cluster;
  return a;
}

int check_workspace(const AttendPlan& p, void* workspace, uint64_t bytes, int device) {
  if (p.bytes == 0) return TCU_OK;
  if (bytes < p.bytes) return fail(TCU_EINVAL, "workspace of %llu bytes, %llu needed", (unsigned long long)bytes, (unsigned long long)p.bytes);
  return check_ptr("workspace", workspace, device, 256);
}

int check_prefix(const tcu_paged_kv* kv, int32_t prefix_pages, int32_t max_length) {
  if (prefix_pages < 0 || (int64_t)prefix_pages * kv->page_tokens > MAX_POSITIONS) return fail(TCU_EINVAL, "prefix of %d pages", prefix_pages);
  if (max_length < 0) return fail(TCU_EINVAL, "max_length %d", max_length);
  return TCU_OK;
}

// Positions a request can hold: what its table (or the prefix) maps.
int length_bound(const tcu_paged_kv* kv, const tcu_paged_queries* q, int prefix_pages, int max_length) {
  const int64_t mapped = (int64_t)std::max(prefix_pages, q->table_width) * kv->page_tokens;
  return (int)(max_length > 0 ? std::min<int64_t>(max_length, mapped) : mapped);
}

int check_sparse(const tcu_paged_kv* kv, int32_t first, int32_t last, int32_t top) {
  if (first < 0 || last < 1 || top < 0) return fail(TCU_EINVAL, "first %d and top %d must not be negative, last %d must be at least 1", first, top, last);
  if ((int64_t)first + last + top > TCU_PAGED_MAX_SELECTED)
    return fail(TCU_EINVAL, "%lld pages a query, at most %d", (long long)first + last + top, TCU_PAGED_MAX_SELECTED);
  if (((int64_t)first + last + top) * kv->page_tokens > MAX_POSITIONS)
    return fail(TCU_EINVAL, "%lld pages of %d positions a query pass 2^30", (long long)first + last + top, kv->page_tokens);
  return TCU_OK;
}

// The arrays of a plan lie apart, but for lengths or starts that are an input's
// own array (a decode loop's lengths are the next step's held): *in_place.
int check_plan_arrays(const PlanArgs& a, bool* in_place) {
  struct Array {
    const char* name;
    const void* at;
    int64_t bytes;
    bool output;
  };
  const int64_t n = a.n, cap = a.capacity;
  const Array arrays[] = {{"held", a.held, 4 * n, false},         {"fresh", a.fresh, 4 * n, false},          {"free_pages", a.free_pages, 4ll * a.n_free, false},
                          {"starts", a.starts, 4 * (n + 1), true}, {"lengths", a.lengths, 4 * n, true},       {"positions", a.positions, 4 * cap, true},
                          {"slots", a.slots, 8 * cap, true},       {"counts", a.counts, 12, true}};
  for (const Array& x : arrays) {
    if (x.bytes == 0) continue;
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x.at), x1 = x0 + x.bytes;
    for (const Array& y : arrays) {
      if (&y == &x) break;
      const uintptr_t y0 = reinterpret_cast<uintptr_t>(y.at), y1 = y0 + y.bytes;
      if (!(x.output || y.output) || x0 >= y1 || y0 >= x1) continue;
      if (x0 == y0 && !y.output && ((x.at == a.lengths && (y.at == a.held || y.at == a.fresh)) || (x.at == a.starts && y.at == a.fresh)))
        *in_place = true;
      else
        return fail(TCU_EINVAL, "%s and %s overlap", y.name, x.name);
    }
    // The tables' rows, not what lies between them.
    const uintptr_t t0 = reinterpret_cast<uintptr_t>(a.tables);
    const uint64_t row = 4ull * a.width, step = 4ull * a.table_stride;
    if (n == 0 || row == 0 || x1 <= t0 || x0 >= t0 + (n - 1) * step + row) continue;
    const uint64_t into = x0 < t0 ? 0 : (x0 - t0) % step;
    if (into < row || into + x.bytes > step) return fail(TCU_EINVAL, "tables and %s overlap", x.name);
  }
  return TCU_OK;
}

}  // namespace

extern "C" {

int tcu_plan_step(int32_t device, void* stream, int32_t n, const int32_t* held, const int32_t* fresh, int32_t page_tokens, int32_t* tables,
                  int32_t table_width, int64_t table_stride, const int32_t* free_pages, int32_t n_free, int32_t capacity, int32_t* starts,
                  int32_t* lengths, int32_t* positions, int64_t* slots, int32_t* counts) {
  if (n < 0 || n_free < 0 || capacity < 0 || table_width < 0) return fail(TCU_EINVAL, "negative count");
  if (page_tokens < 1 || page_tokens > TCU_PAGED_MAX_PAGE_TOKENS)
    return fail(TCU_EINVAL, "%d positions a page, 1..%d are possible", page_tokens, TCU_PAGED_MAX_PAGE_TOKENS);
  if (table_stride < table_width) return fail(TCU_EINVAL, "table stride %lld below the width %d", (long long)table_stride, table_width);
  if (!starts || !counts || (n > 0 && (!held || !fresh || !lengths)) || (capacity > 0 && (!positions || !slots)) ||
      (n > 0 && table_width > 0 && !tables) || (n_free > 0 && !free_pages))
    return fail(TCU_EINVAL, "null argument");
  OnDevice on(device);
  TRY(on.rc);
  TRY(check_ptr("starts", starts, device, 4));
  TRY(check_ptr("counts", counts, device, 4));
  if (n > 0) {
    TRY(check_ptr("held", held, device, 4));
    TRY(check_ptr("fresh", fresh, device, 4));
    TRY(check_ptr("lengths", lengths, device, 4));
    if (table_width > 0) TRY(check_ptr("tables", tables, device, 4));
  }
  if (n_free > 0) TRY(check_ptr("free_pages", free_pages, device, 4));
  if (capacity > 0) {
    TRY(check_ptr("positions", positions, device, 4));
    TRY(check_ptr("slots", slots, device, 8));
  }
  PlanArgs a{};
  a.n = n;
  a.P = page_tokens;
  a.width = table_width;
  a.n_free = n_free;
  a.capacity = capacity;
  a.held = held;
  a.fresh = fresh;
  a.tables = tables;
  a.table_stride = table_stride;
  a.free_pages = free_pages;
  a.starts = starts;
  a.lengths = lengths;
  a.positions = positions;
  a.slots = slots;
  a.counts = counts;
  a.divP = FastDiv::of((uint32_t)page_tokens);
  bool in_place = false;
  TRY(check_plan_arrays(a, &in_place));
  a.tile = in_place ? std::max(capacity, 1) : PLAN_TILE;
  const unsigned grid = (unsigned)std::max<int64_t>(1, ceil_div(capacity, a.tile));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return n <= 256 && capacity / grid <= PLAN_TILE ? launch("k_plan_step", k_plan_step<256>, dim3(grid), 256, 0, s, a) : launch("k_plan_step", k_plan_step<1024>, dim3(grid), 1024, 0, s, a);
}

int tcu_paged_append(int32_t device, void* stream, const tcu_paged_kv* kv, int32_t dtype, int32_t rows, int32_t heads, const void* qkv,
                     int64_t qkv_stride, const int32_t* positions, const int64_t* slots, const tcu_rotary* rotary, const tcu_head_norm* norm,
                     void* q_out, int64_t q_stride) {
  TRY(check_kv(kv));
  TRY(check_pair(dtype, kv->dtype));
  if (rows < 0 || heads < 1) return fail(TCU_EINVAL, "%d rows of %d heads", rows, heads);
  const int hd = kv->head_dim;
  const int64_t width = ((int64_t)heads + 2 * kv->kv_heads) * hd, per16 = 16 / elem_bytes(dtype);
  if ((int64_t)rows * (heads + 2 * kv->kv_heads) > 0x7fffffffll) return fail(TCU_EINVAL, "too many rows for one call");
  if (qkv_stride < width || q_stride < (int64_t)heads * hd) return fail(TCU_EINVAL, "a row's stride is below its width");
  if (qkv_stride % per16 || q_stride % per16) return fail(TCU_EINVAL, "row strides must be multiples of 16 bytes");
  if (rows_overlap(kv->num_pages, kv->page_stride, kv->kv_heads, kv->head_stride, hd) ||
      rows_overlap(kv->num_pages, kv->page_stride, kv->page_tokens, kv->token_stride, hd) ||
      rows_overlap(kv->kv_heads, kv->head_stride, kv->page_tokens, kv->token_stride, hd))
    return fail(TCU_EINVAL, "the cache's rows overlap: it cannot be appended to");
  AppendArgs a{};
  if (rotary && rotary->pairs > 0) {
    if (rotary->pairs * 2 > hd) return fail(TCU_EINVAL, "%d rotary pairs in a head of %d", rotary->pairs, hd);
    if (rotary->max_positions < 1 || !rotary->table) return fail(TCU_EINVAL, "empty rotary table");
    a.table = reinterpret_cast<const float2*>(rotary->table);
    a.max_positions = rotary->max_positions;
    a.pairs = rotary->pairs;
    a.adjacent = rotary->adjacent != 0;
  } else if (rotary && rotary->pairs < 0) {
    return fail(TCU_EINVAL, "%d rotary pairs", rotary->pairs);
  }
  if (norm && norm->kind != TCU_NORM_NONE) {
    if (norm->kind != TCU_NORM_RMS && norm->kind != TCU_NORM_LAYER) return fail(TCU_EINVAL, "unknown norm %d", norm->kind);
    if (!(norm->eps >= 0) || std::isinf(norm->eps)) return fail(TCU_EINVAL, "norm epsilon %g", norm->eps);
    if (norm->head_stride != 0 && norm->head_stride != hd) return fail(TCU_EINVAL, "norm weights are shared (stride 0) or per head (stride %d)", hd);
    a.norm = norm->kind == TCU_NORM_RMS ? NORM_RMS : NORM_LAYER;
    a.eps = (float)norm->eps;
    a.qw = norm->q_weight;
    a.kw = norm->k_weight;
    a.w_stride = norm->head_stride;
  }
  if (rows > 0 && (!qkv || !positions || !slots || !q_out || !kv->k || !kv->v)) return fail(TCU_EINVAL, "null argument");
  OnDevice on(device);
  TRY(on.rc);
  if (rows == 0) return TCU_OK;
  TRY(check_ptr("k", kv->k, device, 16));
  TRY(check_ptr("v", kv->v, device, 16));
  TRY(check_ptr("qkv", qkv, device, 16));
  TRY(check_ptr("q_out", q_out, device, 16));
  const int64_t es = elem_bytes(dtype), one_row[2] = {rows, 1};
  if (!same_or_apart(Rows{qkv, {qkv_stride * es, 0}, width * es}, Rows{q_out, {q_stride * es, 0}, (int64_t)heads * hd * es}, one_row))
    return fail(TCU_EINVAL, "q_out overlaps qkv");
  TRY(check_ptr("positions", positions, device, 4));
  TRY(check_ptr("slots", slots, device, 8));
  if (a.pairs) TRY(check_ptr("rotary table", a.table, device, 8));
  if (a.norm) {
    TRY(check_ptr("q_weight", a.qw, device, 16));
    TRY(check_ptr("k_weight", a.kw, device, 16));
  }
  a.T = rows;
  a.H = heads;
  a.KVH = kv->kv_heads;
  a.hd = hd;
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.positions = positions;
  a.slots = slots;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.kv = view_of(kv);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TCU_F32 && kv->dtype == TCU_F32) return launch_append<float, float>(a, s);
  if (dtype == TCU_F32) return launch_append<float, __half>(a, s);
  if (dtype == TCU_F16) return launch_append<__half, __half>(a, s);
  return launch_append<bf16, bf16>(a, s);
}

int tcu_paged_means(int32_t device, void* stream, const tcu_paged_kv* kv, int32_t rows, const int64_t* slots, void* means) {
  TRY(check_kv(kv));
  if (rows < 0) return fail(TCU_EINVAL, "%d rows", rows);
  if (rows > 0 && (!slots || !means || !kv->k)) return fail(TCU_EINVAL, "null argument");
  OnDevice on(device);
  TRY(on.rc);
  if (rows == 0) return TCU_OK;
  TRY(check_ptr("k", kv->k, device, 16));
  TRY(check_ptr("slots", slots, device, 8));
  TRY(check_ptr("means", means, device, 16));
  MeansArgs a{};
  a.T = rows;
  a.slots = slots;
  a.means = means;
  a.kv = view_of(kv);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv->dtype == TCU_F32) return launch_means<float>(a, s);
  if (kv->dtype == TCU_F16) return launch_means<__half>(a, s);
  return launch_means<bf16>(a, s);
}

int tcu_paged_attend_workspace(const tcu_paged_kv* kv, const tcu_paged_queries* q, int32_t prefix_pages, int32_t max_length, uint64_t* bytes) {
  if (!bytes) return fail(TCU_EINVAL, "null argument");
  TRY(check_kv(kv));
  TRY(check_queries(kv, q));
  TRY(check_prefix(kv, prefix_pages, max_length));
  *bytes = plan_attend(kv, q, prefix_pages, length_bound(kv, q, prefix_pages, max_length), 0).bytes;
  return TCU_OK;
}

int tcu_paged_attend(int32_t device, void* stream, const tcu_paged_kv* kv, const tcu_paged_queries* q, const int32_t* prefix,
                     int32_t prefix_pages, int32_t max_length, void* workspace, uint64_t workspace_bytes) {
  TRY(check_kv(kv));
  TRY(check_queries(kv, q));
  TRY(check_prefix(kv, prefix_pages, max_length));
  if (prefix_pages > 0 && !prefix) return fail(TCU_EINVAL, "prefix is null");
  OnDevice on(device);
  TRY(on.rc);
  if (q->requests == 0 || q->rows == 0) return TCU_OK;
  TRY(check_query_ptrs(kv, q, device));
  if (prefix_pages > 0) TRY(check_ptr("prefix", prefix, device, 4));
  const int bound = length_bound(kv, q, prefix_pages, max_length);
  const AttendPlan p = plan_attend(kv, q, prefix_pages, bound, 0);
  TRY(check_workspace(p, workspace, workspace_bytes, device));
  AttendArgs a = attend_args(kv, q, p, workspace);
  a.prefix = prefix;
  a.prefix_pages = prefix_pages;
  a.max_length = bound;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (q->dtype == TCU_F32 && kv->dtype == TCU_F32) return launch_attend<float, float>(a, p, s);
  if (q->dtype == TCU_F32) return launch_attend<float, __half>(a, p, s);
  if (q->dtype == TCU_F16) return launch_attend<__half, __half>(a, p, s);
  return launch_attend<bf16, bf16>(a, p, s);
}

int tcu_paged_attend_sparse_workspace(const tcu_paged_kv* kv, const tcu_paged_queries* q, int32_t first, int32_t last, int32_t top, uint64_t* bytes) {
  if (!bytes) return fail(TCU_EINVAL, "null argument");
  TRY(check_kv(kv));
  TRY(check_queries(kv, q));
  TRY(check_sparse(kv, first, last, top));
  *bytes = plan_attend(kv, q, 0, 0, first + last + top).bytes;
  return TCU_OK;
}

int tcu_paged_attend_sparse(int32_t device, void* stream, const tcu_paged_kv* kv, const tcu_paged_queries* q, const void* means, int32_t first,
                            int32_t last, int32_t top, int32_t* pages, void* workspace, uint64_t workspace_bytes) {
  TRY(check_kv(kv));
  TRY(check_queries(kv, q));
  TRY(check_sparse(kv, first, last, top));
  OnDevice on(device);
  TRY(on.rc);
  if (q->requests == 0 || q->rows == 0) return TCU_OK;
  TRY(check_query_ptrs(kv, q, device));
  TRY(check_ptr("means", means, device, 16));
  TRY(check_ptr("pages", pages, device, 4));
  const AttendPlan p = plan_attend(kv, q, 0, 0, first + last + top);
  TRY(check_workspace(p, workspace, workspace_bytes, device));
  AttendArgs a = attend_args(kv, q, p, workspace);
  a.max_length = q->table_width * kv->page_tokens;
  a.pages = pages;
  a.budget = first + last + top;
  ChooseArgs c{};
  c.first = first;
  c.last = last;
  c.top = top;
  c.means = means;
  c.keys = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(workspace) + p.keys);
  c.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.scores);
  c.eps = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.eps);
  c.width = q->table_width;
  c.per = p.score_per;
  c.tiles = p.score_tiles;
  c.pages = pages;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (q->dtype == TCU_F32 && kv->dtype == TCU_F32) return launch_sparse<float, float>(a, c, p, s);
  if (q->dtype == TCU_F32) return launch_sparse<float, __half>(a, c, p, s);
  if (q->dtype == TCU_F16) return launch_sparse<__half, __half>(a, c, p, s);
  return launch_sparse<bf16, bf16>(a, c, p, s);
}

}  // extern "C"
