// Attention of a few new tokens per request (the drafted tokens of a speculative step, a short
// continuation) over the paged cache, with the kv axis split over CTAs.
//
//   out[r, h] = sum_t softmax_t(q[r, h] . K[t, h / G] * sm_scale) V[t, h / G],   t <= len_i - n_i + j
//
// for row j of request i. The work of a batch is K/V traffic: every row of the cache is needed once,
// whatever the number of new tokens, so the plan cuts requests along the kv axis until all SMs
// stream, and a merge kernel folds the partial (max, sum, output) states. An item of the plan is
// (request, q tile, page range): the tile's tokens and the G q heads of a kv head are stacked into
// rows (row = token * G + head), so one pass over a K/V tile serves all of them.
#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "common.cuh"

namespace dsv {
namespace {

constexpr int32_t kChunkMagic = 0x44534331;  // "DSC1"
// header: magic, items, merge rows, q tokens per tile, batch, offset of the items, offset of the merge
// rows, q heads, kv heads, head_dim, partial rows, page size, dtype, nnz, kernel (+ 4: some tile has many parts), entries of kv_indices
constexpr int kPlanHeader = 16;
// request, first q token, q tokens, first page | end page, partial row or -1, first q row, first entry of the page list |
// pages of the request, first q token behind which the request's tokens lie (n_new - q0), 2 unused: all that a CTA needs but the last
// page's length, so that it begins after two dependent loads instead of four
constexpr int kItemInts = 12;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct ChunkParams {
  const void* q;
  const void* pages;
  const int32_t* kv_indices;
  const int32_t* kv_last_page_len;
  void* out;
  float* lse;
  const int32_t* items;
  float* part_o;   // [partial rows][Hq][D]
  float* part_ml;  // [partial rows][Hq][2]
  int64_t q_stride, out_stride, page_stride;  // elements
  int n_q_heads, n_kv_heads, head_dim, page_size, num_pages, nnz;
  float scale_log2;
  int* status;
};

// What a CTA knows about its item after the bounds checks.
struct Item {
  int q_row0;    // first q row (global) of the tile
  int nq;        // tokens of the tile
  int n_rows;    // nq * G
  int ip0;       // first entry of the request's page list
  int tok_begin, tok_end;  // kv tokens [begin, end) of this part
  int limit0;    // last kv position the tile's first token sees
  int slot;      // first partial row, -1: write the result
};

__device__ __forceinline__ bool load_item(const ChunkParams& p, int index, Item& it) {
  const int4* raw = reinterpret_cast<const int4*>(p.items + (int64_t)index * kItemInts);
  const int4 a = __ldg(raw), b = __ldg(raw + 1), c = __ldg(raw + 2);
  const int req = a.x, nq = a.z, pb = a.w, pe = b.x, n_pages = c.x, left = c.y;
  if (nq < 1 || nq > left || b.z < 0 || b.z + nq > p.nnz || pb < 0 || pe > n_pages || pb > pe) return false;
  const int kv_len = n_pages > 0 ? (n_pages - 1) * p.page_size + __ldg(p.kv_last_page_len + req) : 0;
  it.q_row0 = b.z;
  it.nq = nq;
  it.n_rows = nq * (p.n_q_heads / p.n_kv_heads);
  it.ip0 = b.w;
  it.limit0 = kv_len - left;
  it.tok_begin = pb * p.page_size;
  // what lies behind the last token's limit is not needed by any row of the tile
  it.tok_end = max(it.tok_begin, min(pe * p.page_size, it.limit0 + nq));
  it.slot = b.y;
  return true;
}

}  // namespace
}  // namespace dsv
#include "chunk_tma.cuh"
#include "chunk_tc.cuh"
namespace dsv {
namespace {

// ---- the general kernel: every type, head_dim, page size and pool stride --------------------------
// CTA of 128 threads: 16 rows of one kv head, 8 threads a row. 32 kv tokens at a time are widened to
// fp32 in shared memory; a thread computes 4 of its row's 32 scores, the row's softmax runs over the 8
// lanes, and the thread keeps head_dim / 8 elements of the row's output in registers. fp32
// multiply-adds and the shared-memory loads that feed them bound it: it serves fp32 caches and shapes that the tensor-core kernels do not
// take. One fp32 request of 65,536 tokens, 4 new, 32 / 8 heads of 128: 516 us (1.0 TB/s, 8.3 TFLOP/s); 8 bf16 requests of 8192, 4 new,
// 32 / 8 heads of 96: 337 us (9.6 TFLOP/s).
constexpr int kSimpleThreads = 128, kSimpleRows = 16, kSimpleTok = 32;

template <typename T, int DMAX>
__global__ void __launch_bounds__(kSimpleThreads)
chunk_simple_kernel(const ChunkParams p, int row_blocks) {
  constexpr int N = Vec16<T>::N;
  constexpr int NV = DMAX / 32;  // float4 of the output per thread
  constexpr int LD = DMAX + 4;   // row pitch: float4 loads of 8 lanes x 4 rows fall in different banks
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;                             // [16][LD]
  float* sk = sq + kSimpleRows * LD;          // [32][LD]
  float* sv = sk + kSimpleTok * LD;           // [32][LD]
  float* sp = sv + kSimpleTok * LD;           // [16][33]
  const int G = p.n_q_heads / p.n_kv_heads, D = p.head_dim;
  const int tid = threadIdx.x;
  int b = blockIdx.x;
  const int rb = b % row_blocks;
  b /= row_blocks;
  const int kv_head = b % p.n_kv_heads;
  Item it;
  if (!load_item(p, b / p.n_kv_heads, it)) {
    if (tid == 0) record_status(p.status, ST_BAD_PLAN);
    return;
  }
  const int row0 = rb * kSimpleRows;
  if (row0 >= it.n_rows) return;
  const int row = tid >> 3, c = tid & 7;
  const int r = row0 + row;
  const bool live = r < it.n_rows;
  const int tok = live ? r / G : 0, head = live ? r % G : 0;
  const int limit = it.limit0 + tok;

  const int vec = D / N;  // 16-byte vectors of a head row
  const T* q = reinterpret_cast<const T*>(p.q);
  for (int x = tid; x < kSimpleRows * vec; x += kSimpleThreads) {
    const int rr = x / vec, v = x % vec, gr = row0 + rr;
    float f[N];
    if (gr < it.n_rows) {
      Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4*>(q + (int64_t)(it.q_row0 + gr / G) * p.q_stride +
                                                           (int64_t)(kv_head * G + gr % G) * D) + v), f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sq[rr * LD + v * N + e] = f[e] * p.scale_log2;
  }
  float m = -INFINITY, l = 0.f;
  float4 o[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);

  const T* pages = reinterpret_cast<const T*>(p.pages);
  const int64_t half = (int64_t)p.page_size * p.n_kv_heads * D;
  for (int t0 = it.tok_begin; t0 < it.tok_end; t0 += kSimpleTok) {
    const int n = min(kSimpleTok, it.tok_end - t0);
    __syncthreads();  // the previous tile is no longer read
    for (int x = tid; x < 2 * kSimpleTok * vec; x += kSimpleThreads) {
      const int kv = x / (kSimpleTok * vec), y = x % (kSimpleTok * vec), tt = y / vec, v = y % vec;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 0.f;
      if (tt < n) {
        const int t = t0 + tt;
        int page = __ldg(p.kv_indices + it.ip0 + t / p.page_size);
        if (page < 0 || page >= p.num_pages) {
          record_status(p.status, ST_BAD_PAGE_ID);
          page = 0;
        }
        Vec16<T>::unpack(ld_stream16(pages + (int64_t)page * p.page_stride + kv * half +
                                     ((int64_t)(t % p.page_size) * p.n_kv_heads + kv_head) * D + v * N), f);
      }
      float* dst = (kv ? sv : sk) + tt * LD + v * N;
#pragma unroll
      for (int e = 0; e < N; ++e) dst[e] = f[e];
    }
    __syncthreads();
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d = 0; d < D; d += 4) {
      const float4 a = *reinterpret_cast<const float4*>(sq + row * LD + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 k = *reinterpret_cast<const float4*>(sk + (c + 8 * i) * LD + d);
        s[i] = fmaf(a.x, k.x, fmaf(a.y, k.y, fmaf(a.z, k.z, fmaf(a.w, k.w, s[i]))));
      }
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + c + 8 * i;
      if (t >= it.tok_end || t > limit || !live) s[i] = -INFINITY;
      mx = fmaxf(mx, s[i]);
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float off = mx == -INFINITY ? 0.f : mx;  // a row that has seen nothing yet
    const float keep = exp2f(m - off);
    m = mx;
    l *= keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = exp2f(s[i] - off);
      l += s[i];
      sp[row * 33 + c + 8 * i] = s[i];
    }
    __syncwarp();  // a row's 8 threads are in one warp
#pragma unroll
    for (int i = 0; i < NV; ++i) { o[i].x *= keep; o[i].y *= keep; o[i].z *= keep; o[i].w *= keep; }
    // only what the row sees: a later token's V may hold anything, 0 * inf included
    const int seen = live ? min(n, limit - t0 + 1) : 0;
    for (int tt = 0; tt < seen; ++tt) {
      const float w = sp[row * 33 + tt];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int d = (i * 8 + c) * 4;
        if (d < D) {
          const float4 v = *reinterpret_cast<const float4*>(sv + tt * LD + d);
          o[i].x = fmaf(w, v.x, o[i].x); o[i].y = fmaf(w, v.y, o[i].y);
          o[i].z = fmaf(w, v.z, o[i].z); o[i].w = fmaf(w, v.w, o[i].w);
        }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int x = 1; x < 8; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if (!live) return;
  const int qh = kv_head * G + head;
  if (it.slot < 0) {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* dst = reinterpret_cast<T*>(p.out) + (int64_t)(it.q_row0 + tok) * p.out_stride + (int64_t)qh * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = (i * 8 + c) * 4;
      if (d < D) {
        dst[d] = from_f32<T>(o[i].x * inv); dst[d + 1] = from_f32<T>(o[i].y * inv);
        dst[d + 2] = from_f32<T>(o[i].z * inv); dst[d + 3] = from_f32<T>(o[i].w * inv);
      }
    }
    if (p.lse != nullptr && c == 0)
      p.lse[(int64_t)(it.q_row0 + tok) * p.n_q_heads + qh] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
  } else {
    const int64_t at = (int64_t)(it.slot + tok) * p.n_q_heads + qh;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = (i * 8 + c) * 4;
      if (d < D) *reinterpret_cast<float4*>(p.part_o + at * D + d) = o[i];
    }
    if (c == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
  }
}

// ---- merge of the parts of a split tile -----------------------------------------------------------
// W warps per (split q row, q head) take its parts round robin, 4 in flight each, and are joined in shared
// memory. merge row: {q row, first partial row, parts, partial rows per part}. W = 8 when some row has more
// than 8 parts (one warp took 11 us for the 74 parts of a 64k-token request, a chain of 19 loads), else 1
// (8 warps for the 2 parts of each of 37,000 rows took 40 us longer).
constexpr int kMergeThreads = 256;

template <typename T, int W>
__global__ void __launch_bounds__(kMergeThreads)
chunk_merge_kernel(const int4* __restrict__ rows, int units, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                   T* __restrict__ out, float* __restrict__ lse, int64_t out_stride, int n_q_heads, int head_dim) {
  constexpr int U = kMergeThreads / 32 / W;  // units of a CTA
  __shared__ float4 s_acc[U][W][64];  // head_dim <= 256
  __shared__ float s_m[U][W], s_l[U][W];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W, sub = (threadIdx.x >> 5) / W;
  const int unit = min((int)blockIdx.x * U + sub, units - 1);  // the last CTA may do a unit twice
  const int4 mr = __ldg(rows + unit / n_q_heads);
  const int qh = unit % n_q_heads;
  const int64_t first = (int64_t)mr.y * n_q_heads + qh, step = (int64_t)mr.w * n_q_heads;
  float m = -INFINITY, l = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int s0 = warp; s0 < mr.z; s0 += 4 * W) {
    float2 ml[4];
    float4 v[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i * W;
      ml[i] = make_float2(-INFINITY, 0.f);
      v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < mr.z) {
        ml[i] = __ldg(reinterpret_cast<const float2*>(part_ml + (first + s * step) * 2));
        const float4* po = reinterpret_cast<const float4*>(part_o + (first + s * step) * head_dim);
        if (lane * 4 < head_dim) v[i][0] = __ldg(po + lane);
        if (lane * 4 + 128 < head_dim) v[i][1] = __ldg(po + lane + 32);
      }
    }
    const float mx = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
    const float off = mx == -INFINITY ? 0.f : mx;
    const float keep = exp2f(m - off);
    m = mx;
    l *= keep;
#pragma unroll
    for (int k = 0; k < 2; ++k) { acc[k].x *= keep; acc[k].y *= keep; acc[k].z *= keep; acc[k].w *= keep; }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = exp2f(ml[i].x - off);
      l = fmaf(ml[i].y, w, l);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        acc[k].x = fmaf(w, v[i][k].x, acc[k].x); acc[k].y = fmaf(w, v[i][k].y, acc[k].y);
        acc[k].z = fmaf(w, v[i][k].z, acc[k].z); acc[k].w = fmaf(w, v[i][k].w, acc[k].w);
      }
    }
  }
  s_acc[sub][warp][lane] = acc[0];
  s_acc[sub][warp][lane + 32] = acc[1];
  if (lane == 0) { s_m[sub][warp] = m; s_l[sub][warp] = l; }
  __syncthreads();
  float mx = -INFINITY, lsum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[sub][w]);
  const float off = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int w = 0; w < W; ++w) lsum = fmaf(s_l[sub][w], exp2f(s_m[sub][w] - off), lsum);
  for (int d = warp * 32 + lane; d < head_dim; d += W * 32) {
    float res = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) res = fmaf(reinterpret_cast<const float*>(s_acc[sub][w])[d], exp2f(s_m[sub][w] - off), res);
    out[(int64_t)mr.x * out_stride + (int64_t)qh * head_dim + d] = from_f32<T>(lsum == 0.f ? 0.f : res / lsum);
  }
  if (lse != nullptr && warp == 0 && lane == 0)
    lse[(int64_t)mr.x * n_q_heads + qh] = lsum == 0.f ? -INFINITY : (mx + log2f(lsum)) * kLn2;
}

template <typename T>
void launch_merge(const int4* rows, int units, bool many, const ChunkParams& p, cudaStream_t st) {
  if (many)
    chunk_merge_kernel<T, 8><<<units, kMergeThreads, 0, st>>>(rows, units, p.part_o, p.part_ml, (T*)p.out, p.lse, p.out_stride, p.n_q_heads, p.head_dim);
  else
    chunk_merge_kernel<T, 1><<<(units + 7) / 8, kMergeThreads, 0, st>>>(rows, units, p.part_o, p.part_ml, (T*)p.out, p.lse, p.out_stride, p.n_q_heads, p.head_dim);
}

template <typename T, int DMAX>
cudaError_t launch_simple(const ChunkParams& p, int n_items, int tile_tokens, cudaStream_t st) {
  const int row_blocks = (tile_tokens * (p.n_q_heads / p.n_kv_heads) + kSimpleRows - 1) / kSimpleRows;
  const int64_t grid = (int64_t)n_items * p.n_kv_heads * row_blocks;
  const size_t smem = ((size_t)(kSimpleRows + 2 * kSimpleTok) * (DMAX + 4) + kSimpleRows * 33) * sizeof(float);
  cudaError_t e = allow_smem<chunk_simple_kernel<T, DMAX>>(smem);
  if (e != cudaSuccess) return e;
  chunk_simple_kernel<T, DMAX><<<(unsigned)grid, kSimpleThreads, smem, st>>>(p, row_blocks);
  return cudaGetLastError();
}
int ilog2_exact(int x) {  // log2 of a power of two, -1 otherwise
  if (x <= 0 || (x & (x - 1)) != 0) return -1;
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
enum : int { kSimple = 0, kMma = 1, kTc = 2, kManyParts = 4 };  // kernel of a plan, and whether its merge takes eight warps a row
// kv heads of a CTA of the mma.sync kernel
int heads_per_cta(int n_kv_heads) {
  int hb = 8;
  while (hb > 1 && n_kv_heads % hb != 0) hb >>= 1;
  return hb;
}

template <typename T, int D>
cudaError_t launch_tma(const CUtensorMap& map, const ChunkParams& p, const chunk_tma::Split& sp, int n_items, cudaStream_t st) {
  const size_t smem = (size_t)512 * D * chunk_tma::kStages + 1024 + 64;
  cudaError_t e = allow_smem<chunk_tma::chunk_tma_kernel<T, D>>(smem);
  if (e != cudaSuccess) return e;
  chunk_tma::chunk_tma_kernel<T, D><<<(unsigned)(n_items * (p.n_kv_heads >> sp.hb_log2)), chunk_tma::kThreads, smem, st>>>(map, p, sp);
  return cudaGetLastError();
}

template <typename T, int D, bool MERGED>
cudaError_t launch_tc(const chunk_tc::Maps& m, const ChunkParams& p, int ps_log2, int n_items, cudaStream_t st) {
  const size_t smem = (size_t)2 * 128 * D * 2 + (size_t)(2 + chunk_tc::kVStages) * chunk_tc::kBN * D * 2 + 256 + 1024;
  cudaError_t e = allow_smem<chunk_tc::chunk_tc_kernel<T, D, MERGED>>(smem);
  if (e != cudaSuccess) return e;
  chunk_tc::chunk_tc_kernel<T, D, MERGED><<<(unsigned)(n_items * p.n_kv_heads), chunk_tc::kThreads, smem, st>>>(m.q, m.k, m.v, p, ps_log2);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_tc_d(const chunk_tc::Maps& m, const ChunkParams& p, int ps_log2, int n_items, cudaStream_t st) {
  if (p.head_dim == 64) return launch_tc<T, 64, false>(m, p, ps_log2, n_items, st);
  return p.page_size >= 16 ? launch_tc<T, 128, true>(m, p, ps_log2, n_items, st) : launch_tc<T, 128, false>(m, p, ps_log2, n_items, st);
}

template <typename T>
cudaError_t launch_simple_d(const ChunkParams& p, int n_items, int tile_tokens, cudaStream_t st) {
  if (p.head_dim <= 64) return launch_simple<T, 64>(p, n_items, tile_tokens, st);
  if (p.head_dim <= 128) return launch_simple<T, 128>(p, n_items, tile_tokens, st);
  return launch_simple<T, 256>(p, n_items, tile_tokens, st);
}

int chunk_plan(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host, int batch, int n_q_heads, int n_kv_heads, int head_dim,
               int page_size, int dtype, int sm_count, int64_t workspace_capacity, int32_t* plan_host, int64_t plan_capacity_i32,
               int64_t* plan_used_i32, int64_t* workspace_bytes) {
  DSV_REQUIRE(qo_indptr_host && kv_indptr_host && plan_host && plan_used_i32 && workspace_bytes,
              "chunk_plan: null pointer argument");
  DSV_REQUIRE(batch >= 0, "chunk_plan: negative batch");
  DSV_REQUIRE(dtype_ok(dtype), "chunk_plan: unknown dtype %d", dtype);
  DSV_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0,
              "chunk_plan: n_q_heads (%d) must be a positive multiple of n_kv_heads (%d)", n_q_heads, n_kv_heads);
  DSV_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256, "chunk_plan: head_dim %d must be a multiple of 8, at most 256",
              head_dim);
  DSV_REQUIRE(page_size > 0, "chunk_plan: page_size must be positive");
  if (sm_count <= 0) sm_count = 148;
  const int G = n_q_heads / n_kv_heads;
  // Rows of a q tile: all new tokens of a request where they fit, so that its K/V is read once.
  const bool tensor = dtype != DSV_F32 && (head_dim == 64 || head_dim == 128) && G <= 128 && ilog2_exact(page_size) >= 3;
  int most = 0;
  for (int i = 0; i < batch; ++i) most = std::max(most, qo_indptr_host[i + 1] - qo_indptr_host[i]);
  // up to 16 rows: mma.sync, all heads of a page in one CTA; more: tcgen05, one kv head per CTA
  const int kind = !tensor ? kSimple : (int64_t)most * G <= 16 ? kMma : kTc;
  const int tile = std::max(1, kind == kMma ? 16 / G : kind == kTc ? (most > 128 / G ? 2 * (128 / G) : 128 / G) : kSimpleRows / G);
  const int ctas_per_item = kind == kMma ? n_kv_heads / heads_per_cta(n_kv_heads)
                            : kind == kTc ? n_kv_heads : n_kv_heads * ((tile * G + kSimpleRows - 1) / kSimpleRows);

  struct Tile { int req, q0, nq, pages; };
  std::vector<Tile> tiles;
  int64_t total_pages = 0, n_tiles = 0;
  int max_pages = 0;
  bool fits = true;
  DSV_REQUIRE(qo_indptr_host[0] == 0 && kv_indptr_host[0] >= 0, "chunk_plan: indptr must begin at 0");
  for (int i = 0; i < batch; ++i) {
    const int n = qo_indptr_host[i + 1] - qo_indptr_host[i], np = kv_indptr_host[i + 1] - kv_indptr_host[i];
    DSV_REQUIRE(n >= 0 && np >= 0, "chunk_plan: indptr not monotone at %d", i);
    // (positions are 32-bit in the kernels, which step past the end by up to a tile of 128 and a lane's box)
    DSV_REQUIRE((int64_t)np * page_size <= (1ll << 31) - 1024, "chunk_plan: request %d is longer than 2^31 - 1024 tokens", i);
    // whole tiles are the least that a plan can have: one that the caller has no room for takes no memory either
    n_tiles += (n + (int64_t)tile - 1) / tile;
    if (kPlanHeader + kItemInts * n_tiles > plan_capacity_i32) {
      fits = false;
      continue;
    }
    for (int q0 = 0; q0 < n; q0 += std::min(tile, n - q0)) {
      const int nq = std::min(tile, n - q0);
      // pages that the tile's last token can see if the last page is full (the kernel knows its true length)
      const int64_t seen = (int64_t)np * page_size - n + q0 + nq;
      const int pages = (int)std::max<int64_t>(0, std::min<int64_t>(np, (seen + page_size - 1) / page_size));
      tiles.push_back({i, q0, nq, pages});
      total_pages += pages;
      max_pages = std::max(max_pages, pages);
    }
  }
  if (!fits) {
    *plan_used_i32 = kPlanHeader + kItemInts * n_tiles;
    *workspace_bytes = 0;
    return fail(DSV_E_WORKSPACE, "chunk_plan: plan needs %lld int32, capacity %lld", (long long)*plan_used_i32, (long long)plan_capacity_i32);
  }
  // Part length: compared on a model of the launch. A CTA costs the bytes it streams plus a fixed
  // overhead (fill and drain of its ring, q), a launch that splits anything a merge and the partial
  // states' way to memory and back. CTAs fill `slots` at a time; the last round is half empty on average.
  auto count_items = [&](int c) {
    int64_t k = 0;
    for (const Tile& t : tiles) k += std::max(1, (t.pages + c - 1) / c);
    return k;
  };
  const double page_cost = (double)2 * page_size * n_kv_heads * head_dim * elem_size(dtype) / ctas_per_item;
  // in bytes of streaming; the general kernel is bound by arithmetic: there a CTA's cost is counted in tokens
  const double unit = kind == kSimple ? page_cost / page_size * 32 : 128.0 * 1024;
  const double overhead = unit, merge_cost = 1.5 * unit;
  const int64_t slots = (int64_t)sm_count * (kind == kSimple ? 4 : 1);
  const int64_t most_items = std::max<int64_t>((int64_t)4 * sm_count, (int64_t)tiles.size());
  const int min_chunk = std::max(1, (kind == kSimple ? 32 : 128) / page_size);
  int chunk = std::max(min_chunk, max_pages);
  double best = -1.0;
  auto consider = [&](int64_t c64) {
    const int c = (int)std::min<int64_t>(std::max<int64_t>(c64, min_chunk), std::max(min_chunk, max_pages));
    const int64_t k = count_items(c);
    if (k > most_items) return;
    int64_t rows = 0, merged = 0;  // partial states, and the q rows that they belong to
    if (k > (int64_t)tiles.size()) {
      for (const Tile& t : tiles) {
        const int64_t parts = std::max(1, (t.pages + c - 1) / c);
        if (parts > 1) { rows += parts * t.nq; merged += t.nq; }
      }
      // a split that the caller has no room for is none (whole tiles need no workspace)
      if (rows > workspace_capacity / ((int64_t)n_q_heads * (head_dim + 2) * (int64_t)sizeof(float)) ||
          kPlanHeader + kItemInts * k + 4 * merged > plan_capacity_i32)
        return;
    }
    const int64_t ctas = k * ctas_per_item;
    const double longest = std::min(c, max_pages) * page_cost + overhead;
    double cost = ctas <= slots ? longest
                                : std::max(longest, ((double)total_pages * ctas_per_item * page_cost + (double)ctas * overhead) / (double)slots) + 0.5 * longest;
    if (rows > 0) cost += merge_cost + 2.0 * (double)rows * n_q_heads * (head_dim + 2) * sizeof(float) / sm_count;
    if (best < 0.0 || cost < best) { best = cost; chunk = c; }
  };
  if (!tiles.empty()) {
    for (int parts = 1; parts <= 8; ++parts) consider((max_pages + parts - 1) / parts);
    for (int rounds = 1; rounds <= 4; ++rounds) {
      const int64_t c = (total_pages * ctas_per_item + rounds * slots - 1) / (rounds * slots);
      consider(c);
      consider(c + std::max<int64_t>(1, c / 16));
      consider(c + std::max<int64_t>(1, c / 6));
      consider(c + std::max<int64_t>(1, c / 3));
    }
  }
  const int64_t n_items = count_items(chunk);
  int64_t merge_rows = 0, part_rows = 0, most_parts = 0;
  for (const Tile& t : tiles) {
    const int64_t parts = std::max(1, (t.pages + chunk - 1) / chunk);
    most_parts = std::max(most_parts, parts);
    if (parts > 1) { merge_rows += t.nq; part_rows += parts * t.nq; }
  }
  const int64_t need = kPlanHeader + kItemInts * n_items + 4 * merge_rows;
  *plan_used_i32 = need;
  *workspace_bytes = part_rows * n_q_heads * (head_dim + 2) * (int64_t)sizeof(float);
  if (need > plan_capacity_i32)
    return fail(DSV_E_WORKSPACE, "chunk_plan: plan needs %lld int32, capacity %lld", (long long)need,
                (long long)plan_capacity_i32);
  DSV_REQUIRE(part_rows < (1ll << 31) && n_items * std::max(n_kv_heads * 8, ctas_per_item) < (1ll << 31) &&
                  merge_rows * n_q_heads < (1ll << 31), "chunk_plan: too many partial states");
  struct Out { int len; int32_t v[6]; };
  std::vector<Out> items;
  items.reserve((size_t)n_items);
  int32_t* merge = plan_host + kPlanHeader + kItemInts * n_items;
  int64_t at_merge = 0, at_part = 0;
  for (const Tile& t : tiles) {
    const int parts = std::max(1, (t.pages + chunk - 1) / chunk);
    const int base = t.pages / parts, extra = t.pages % parts;
    int at = 0;
    for (int s = 0; s < parts; ++s) {
      const int len = base + (s < extra ? 1 : 0);
      items.push_back({len, {t.req, t.q0, t.nq, at, at + len, parts > 1 ? (int32_t)(at_part + (int64_t)s * t.nq) : -1}});
      at += len;
    }
    if (parts > 1) {
      for (int j = 0; j < t.nq; ++j) {
        int32_t* m = merge + 4 * at_merge++;
        m[0] = qo_indptr_host[t.req] + t.q0 + j; m[1] = (int32_t)(at_part + j); m[2] = parts; m[3] = t.nq;
      }
      at_part += (int64_t)parts * t.nq;
    }
  }
  std::stable_sort(items.begin(), items.end(), [](const Out& a, const Out& b) { return a.len > b.len; });  // longest first
  for (int k = 0; k < kPlanHeader; ++k) plan_host[k] = 0;
  plan_host[0] = kChunkMagic; plan_host[1] = (int32_t)n_items; plan_host[2] = (int32_t)merge_rows; plan_host[3] = tile;
  plan_host[4] = batch; plan_host[5] = kPlanHeader; plan_host[6] = (int32_t)(kPlanHeader + kItemInts * n_items);
  plan_host[7] = n_q_heads; plan_host[8] = n_kv_heads; plan_host[9] = head_dim; plan_host[10] = (int32_t)part_rows;
  plan_host[11] = page_size; plan_host[12] = dtype; plan_host[13] = batch > 0 ? qo_indptr_host[batch] : 0;
  plan_host[14] = kind + (most_parts > 8 ? kManyParts : 0); plan_host[15] = batch > 0 ? kv_indptr_host[batch] : 0;
  for (int64_t k = 0; k < n_items; ++k) {
    int32_t* it = plan_host + kPlanHeader + kItemInts * k;
    for (int j = 0; j < 6; ++j) it[j] = items[k].v[j];
    const int req = it[0], q0 = it[1];
    it[6] = qo_indptr_host[req] + q0;
    it[7] = kv_indptr_host[req];
    it[8] = kv_indptr_host[req + 1] - kv_indptr_host[req];
    it[9] = qo_indptr_host[req + 1] - qo_indptr_host[req] - q0;
    it[10] = it[11] = 0;
  }
  return DSV_OK;
}

}  // namespace
}  // namespace dsv

extern "C" {

int dsv_chunk_plan_within(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host, int batch, int n_q_heads,
                          int n_kv_heads, int head_dim, int page_size, int dtype, int sm_count,
                          int64_t workspace_capacity, int32_t* plan_host, int64_t plan_capacity_i32,
                          int64_t* plan_used_i32, int64_t* workspace_bytes) {
  using namespace dsv;
  DSV_REQUIRE(workspace_capacity >= 0, "chunk_plan: negative workspace_capacity");
  try {
    return chunk_plan(qo_indptr_host, kv_indptr_host, batch, n_q_heads, n_kv_heads, head_dim, page_size, dtype, sm_count, workspace_capacity,
                      plan_host, plan_capacity_i32, plan_used_i32, workspace_bytes);
  } catch (const std::exception& e) {  // no exception leaves a C entry
    return fail(DSV_E_WORKSPACE, "chunk_plan: %s", e.what());
  }
}

int dsv_chunk_plan(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host, int batch, int n_q_heads,
                   int n_kv_heads, int head_dim, int page_size, int dtype, int sm_count, int32_t* plan_host,
                   int64_t plan_capacity_i32, int64_t* plan_used_i32, int64_t* workspace_bytes) {
  return dsv_chunk_plan_within(qo_indptr_host, kv_indptr_host, batch, n_q_heads, n_kv_heads, head_dim, page_size, dtype, sm_count,
                               INT64_MAX, plan_host, plan_capacity_i32, plan_used_i32, workspace_bytes);
}

int dsv_paged_chunk_attention(const void* q, int64_t q_stride_tok, const int32_t* qo_indptr, const void* pages_layer,
                              int64_t page_stride, int64_t num_pages, const int32_t* kv_indices,
                              const int32_t* kv_indptr, const int32_t* kv_last_page_len, void* out,
                              int64_t out_stride_tok, float* lse, const int32_t* plan_host, const int32_t* plan_dev,
                              void* workspace, int64_t workspace_bytes, int batch, int nnz, int n_q_heads,
                              int n_kv_heads, int head_dim, int page_size, int dtype, float sm_scale, void* stream) {
  using namespace dsv;
  DSV_REQUIRE(dtype_ok(dtype), "chunk: unknown dtype %d", dtype);
  DSV_REQUIRE(batch >= 0 && nnz >= 0, "chunk: negative batch or nnz");
  if (batch == 0 || nnz == 0) return DSV_OK;
  DSV_REQUIRE(q && qo_indptr && pages_layer && kv_indptr && kv_last_page_len && out && plan_host && plan_dev,
              "chunk: null pointer argument");
  DSV_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0, "chunk: bad head counts");
  DSV_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256, "chunk: head_dim %d must be a multiple of 8, at most 256",
              head_dim);
  DSV_REQUIRE(page_size > 0, "chunk: page_size must be positive");
  DSV_REQUIRE(num_pages > 0 && num_pages < (1ll << 30), "chunk: num_pages (%lld) out of range", (long long)num_pages);
  DSV_REQUIRE(plan_host[0] == kChunkMagic && plan_host[4] == batch && plan_host[7] == n_q_heads &&
                  plan_host[8] == n_kv_heads && plan_host[9] == head_dim && plan_host[11] == page_size && plan_host[12] == dtype,
              "chunk: plan does not belong to this call");
  DSV_REQUIRE(nnz >= plan_host[13], "chunk: the plan covers %d rows, q has %d", plan_host[13], nnz);
  const int n_items = plan_host[1], merge_rows = plan_host[2];
  const int64_t part_rows = plan_host[10];
  DSV_REQUIRE(n_items >= 0 && merge_rows >= 0 && part_rows >= 0 && plan_host[3] > 0, "chunk: corrupt plan");
  if (n_items == 0) return DSV_OK;
  DSV_REQUIRE(kv_indices != nullptr || plan_host[15] == 0, "chunk: null pointer argument");  // no request has a page: an empty list
  const int es = elem_size(dtype);
  DSV_REQUIRE(aligned16(q) && aligned16(pages_layer) && aligned16(out) && (q_stride_tok * es) % 16 == 0 &&
                  (out_stride_tok * es) % 16 == 0 && (page_stride * es) % 16 == 0,
              "chunk: pointers and strides must be 16-byte aligned");
  DSV_REQUIRE(q_stride_tok >= (int64_t)n_q_heads * head_dim && out_stride_tok >= (int64_t)n_q_heads * head_dim,
              "chunk: token stride smaller than a row");
  DSV_REQUIRE(page_stride >= (int64_t)2 * page_size * n_kv_heads * head_dim, "chunk: page_stride smaller than one page");
  const int64_t ws_need = part_rows * n_q_heads * (head_dim + 2) * (int64_t)sizeof(float);
  if (ws_need > 0 && (workspace == nullptr || workspace_bytes < ws_need))
    return fail(DSV_E_WORKSPACE, "chunk: workspace needs %lld bytes, got %lld", (long long)ws_need, (long long)workspace_bytes);
  DSV_REQUIRE(ws_need == 0 || aligned16(workspace), "chunk: workspace must be 16-byte aligned");
  ChunkParams p;
  p.q = q; p.pages = pages_layer; p.kv_indices = kv_indices;
  p.kv_last_page_len = kv_last_page_len; p.out = out; p.lse = lse; p.items = plan_dev + plan_host[5];
  DSV_REQUIRE(aligned16(p.items) && aligned16(plan_dev + plan_host[6]), "chunk: device plan must be 16-byte aligned");
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + part_rows * n_q_heads * head_dim;
  p.q_stride = q_stride_tok; p.out_stride = out_stride_tok; p.page_stride = page_stride;
  p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim; p.page_size = page_size;
  p.num_pages = (int)num_pages; p.nnz = nnz; p.scale_log2 = sm_scale * kLog2e; p.status = device_status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  const int ps_log2 = ilog2_exact(page_size);
  // a pool with gaps between its pages has no tensor map, and the tensor-core kernels scale a row's largest score, which has to stay
  // its largest: the general kernel takes any plan and scales q
  const int kind = page_stride == (int64_t)2 * page_size * n_kv_heads * head_dim && sm_scale > 0.f ? plan_host[14] & ~kManyParts : kSimple;
  DSV_REQUIRE(kind >= kSimple && kind <= kTc && (kind == kSimple || (ps_log2 >= 3 && dtype != DSV_F32 && (head_dim == 64 || head_dim == 128))),
              "chunk: corrupt plan");
  if (kind == kMma) {
    const int hb = heads_per_cta(n_kv_heads);
    const chunk_tma::Split sp = {ilog2_exact(hb), ps_log2};
    CUtensorMap map;
    if (!chunk_tma::make_tensor_map(&map, pages_layer, num_pages, page_size, n_kv_heads, head_dim, hb, dtype == DSV_BF16))
      return fail(DSV_E_CUDA, "chunk: tensor map of the pages rejected");
    if (dtype == DSV_F16)
      e = head_dim == 128 ? launch_tma<__half, 128>(map, p, sp, n_items, st) : launch_tma<__half, 64>(map, p, sp, n_items, st);
    else
      e = head_dim == 128 ? launch_tma<__nv_bfloat16, 128>(map, p, sp, n_items, st) : launch_tma<__nv_bfloat16, 64>(map, p, sp, n_items, st);
  } else if (kind == kTc) {
    chunk_tc::Maps maps;
    if (!chunk_tma::encode_tiled_fn() || !chunk_tc::make_maps(chunk_tma::encode_tiled_fn(), maps, p, head_dim == 128 && page_size >= 16, dtype == DSV_BF16))
      return fail(DSV_E_CUDA, "chunk: tensor maps rejected");
    e = dtype == DSV_F16 ? launch_tc_d<__half>(maps, p, ps_log2, n_items, st) : launch_tc_d<__nv_bfloat16>(maps, p, ps_log2, n_items, st);
  } else switch (dtype) {
    case DSV_F32: e = launch_simple_d<float>(p, n_items, plan_host[3], st); break;
    case DSV_F16: e = launch_simple_d<__half>(p, n_items, plan_host[3], st); break;
    default: e = launch_simple_d<__nv_bfloat16>(p, n_items, plan_host[3], st);
  }
  if (e != cudaSuccess) return fail(DSV_E_CUDA, "chunk launch failed: %s", cudaGetErrorString(e));
  if (merge_rows > 0) {
    const int4* rows = reinterpret_cast<const int4*>(plan_dev + plan_host[6]);
    const int units = merge_rows * n_q_heads;
    const bool many = (plan_host[14] & kManyParts) != 0;
    switch (dtype) {
      case DSV_F32: launch_merge<float>(rows, units, many, p, st); break;
      case DSV_F16: launch_merge<__half>(rows, units, many, p, st); break;
      default: launch_merge<__nv_bfloat16>(rows, units, many, p, st);
    }
    DSV_CUDA(cudaGetLastError());
  }
  return DSV_OK;
}

}  // extern "C"
