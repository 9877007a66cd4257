// Chunk attention for 16-bit K/V and at most 16 rows ((token, q head) pairs of a kv head) per item, on the
// tensor cores (mma.sync), K/V staged by TMA.
//
// A CTA owns one item of the plan for `hb` kv heads: 8 consumer warps and a producer warp, 1 CTA per SM,
// a 3-deep ring of 512 * D bytes per stage (128 (head, token) rows of K and of V). The warps are split over
// heads first, then over the 16-token groups of a stage (ts): hb * ts = 8; the ts warps of a head merge at the end.
// Per 16 tokens: S = Q K^T as mma.sync.m16n8k16, causal / length mask where a row's limit falls into the group,
// online softmax on the fragments, O += P V. One 16-row MMA tile covers all rows, so the arithmetic is a few
// percent of the time that the tile's bytes take. With 17 rows and more it would read its tile from shared
// memory once per 16 rows: those go to the tcgen05 kernel.
// Two requests of about 100 kv tokens, 2-4 of them new, 8 q / 2 kv heads of 64: 6.5 us, the latency of one launch and one ring fill.
// 32 q / 8 kv heads of 128, bf16: one request of 65,536 tokens, 4 new, 60 us with the merge (4.5 TB/s); 128 requests of 512-4096 tokens, 1-4 new,
// 216 us (5.7 TB/s, 0.87 of a copy; the tcgen05 kernel on the same caches with 5 new: 237 us).
#pragma once

#include <cuda.h>

#include "tcgen05.cuh"

namespace dsv {
namespace chunk_tma {

using namespace ptx;

constexpr int kConsumerWarps = 8;
constexpr int kConsumerThreads = kConsumerWarps * 32;
constexpr int kThreads = kConsumerThreads + 32;
constexpr int kStages = 3;
constexpr float kGrow = 8.f;  // log2 units

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
// The halves of a pair that are no finite numbers (an exponent of all ones), as a mask.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return ((w & E) == E ? 0x0000ffffu : 0u) | (((w >> 16) & E) == E ? 0xffff0000u : 0u);
}

struct Split {
  int hb_log2, ps_log2;  // kv heads of a CTA, page size
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_tma_kernel(const __grid_constant__ CUtensorMap tmap, const ChunkParams p, const Split sp) {
  constexpr int DH = D / 64;            // 64-element halves of head_dim
  constexpr int KSTEPS = D / 16;
  constexpr int HALF = 128 * D * 2;     // K (or V) part of a stage
  constexpr int STAGE = 2 * HALF;

  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;  // swizzle atoms are 1024-byte aligned
  unsigned char* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_full = smem_base + kStages * STAGE;  // kStages x 8 bytes
  const uint32_t bar_empty = bar_full + kStages * 8;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hb_log = sp.hb_log2, hb = 1 << hb_log;
  const int ng = kConsumerWarps >> hb_log, ttok = 16 * ng;  // 16-token groups and tokens of a stage
  const int ps_log = sp.ps_log2, ps = 1 << ps_log;
  const int bt_log = min(ps_log, 4), bt = 1 << bt_log;      // tokens per TMA box
  const int bpg = 16 >> bt_log;                               // boxes per 16-token group
  const int box_bytes = DH * hb * bt * 128;
  const int G = p.n_q_heads / p.n_kv_heads;
  const int n_groups = p.n_kv_heads >> hb_log;
  const int kv_group = blockIdx.x % n_groups;                 // the kv heads of an item are adjacent CTAs

  Item it;
  if (!load_item(p, blockIdx.x / n_groups, it) || it.n_rows > 16) {
    if (tid == 0) record_status(p.status, ST_BAD_PLAN);
    return;
  }
  const int n_tiles = (it.tok_end - it.tok_begin + ttok - 1) / ttok;
  const int ts = ng;  // warps of a kv head: one 16-token group of a stage each

  if (tid == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, kConsumerWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();

  // ============================ producer warp ============================================
  if (warp == kConsumerWarps) {
    const int32_t* idx = p.kv_indices + it.ip0;
    const int n_boxes = ng * bpg;  // boxes per tile and per K/V half (<= 16)
    int tile = 0;
    for (; tile < n_tiles; ++tile) {
      const int s = tile % kStages;
      const int tok0 = it.tok_begin + tile * ttok + lane * bt;  // first token of this lane's box
      const bool mine = lane < n_boxes && tok0 < it.tok_end;
      int page = 0;
      if (mine) {
        page = __ldg(idx + (tok0 >> ps_log));
        if (page < 0 || page >= p.num_pages) {
          record_status(p.status, ST_BAD_PAGE_ID);
          page = 0;
        }
      }
      if (tile >= kStages) {
        if (!warp_wait(bar_empty + 8 * s, ((tile / kStages) - 1) & 1, p.status)) break;
      }
      const unsigned live = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) mbar_expect_tx(bar_full + 8 * s, (uint32_t)(__popc(live) * 2 * box_bytes));
      __syncwarp();
      if (mine) {
        const uint32_t dst = smem_base + s * STAGE + lane * box_bytes;
        const int in_page = tok0 & (ps - 1);
        tma_load_5d(dst, &tmap, bar_full + 8 * s, 0, in_page, kv_group * hb, 0, 2 * page);
        tma_load_5d(dst + HALF, &tmap, bar_full + 8 * s, 0, in_page, kv_group * hb, 0, 2 * page + 1);
      }
    }
    // the CTA does not end before its copies, whatever became of a consumer's wait
    for (int k = max(tile - kStages, 0); k < tile; ++k) warp_wait(bar_full + 8 * (k % kStages), (k / kStages) & 1, p.status);
    return;
  }

  // ============================ consumer warps ===========================================
  const int g = lane >> 2, tg = lane & 3;
  const int head_local = warp & (hb - 1), sub = warp >> hb_log;
  const int kv_head = kv_group * hb + head_local;
  const int r0 = g, r1 = r0 + 8;  // this lane's rows
  const int t_r0 = r0 / G, t_r1 = r1 / G;
  // last kv position that a row sees in this part; -1 for rows that are not there
  const int lim0 = r0 < it.n_rows ? min(it.limit0 + t_r0, it.tok_end - 1) : -1;
  const int lim1 = r1 < it.n_rows ? min(it.limit0 + t_r1, it.tok_end - 1) : -1;
  const int lim_first = min(it.limit0, it.tok_end - 1);  // smallest limit of the live rows; the largest is tok_end - 1

  uint32_t qa[KSTEPS][4];
  {
    const T* q0 = reinterpret_cast<const T*>(p.q) + (int64_t)(it.q_row0 + t_r0) * p.q_stride + (int64_t)(kv_head * G + r0 % G) * D;
    const T* q1 = reinterpret_cast<const T*>(p.q) + (int64_t)(it.q_row0 + t_r1) * p.q_stride + (int64_t)(kv_head * G + r1 % G) * D;
    const bool a0 = r0 < it.n_rows, a1 = r1 < it.n_rows;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const int d0 = kk * 16 + tg * 2;
      qa[kk][0] = a0 ? *reinterpret_cast<const uint32_t*>(q0 + d0) : 0u;
      qa[kk][2] = a0 ? *reinterpret_cast<const uint32_t*>(q0 + d0 + 8) : 0u;
      qa[kk][1] = a1 ? *reinterpret_cast<const uint32_t*>(q1 + d0) : 0u;
      qa[kk][3] = a1 ? *reinterpret_cast<const uint32_t*>(q1 + d0 + 8) : 0u;
    }
  }

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float sc = p.scale_log2;

  // Row (128 bytes) of token tl of a 16-token group, head head_local, half dh, inside the group:
  //   ((box * DH + dh) * hb + head_local) * bt + token_in_box, box = tl >> bt_log.
  // ldmatrix lane roles: K matrices (tok lo, c), (tok lo, c+1), (tok hi, c), (tok hi, c+1);
  //                      V matrices (tok lo, c), (tok hi, c), (tok lo, c+1), (tok hi, c+1).
  const int lr = lane & 7, lm = lane >> 3;
  const int k_tl = lr + ((lm >> 1) << 3), k_cx = lm & 1;
  const int v_tl = lr + ((lm & 1) << 3), v_cx = lm >> 1;
  auto row_of = [&](int tl, int dh) { return (((tl >> bt_log) * DH + dh) * hb + head_local) * bt + (tl & (bt - 1)); };
  // Offset of this lane's first 16-byte chunk; the chunk index enters by XOR (128-byte swizzle), and chunk 2 k + cx
  // differs from chunk cx in the bits of 32 k, so a step's addresses are offset ^ (32 k).
  uint32_t k_off[DH], v_off[DH];
#pragma unroll
  for (int dh = 0; dh < DH; ++dh) {
    const int kr = row_of(k_tl, dh), vr = row_of(v_tl, dh);
    k_off[dh] = kr * 128 + ((k_cx ^ (kr & 7)) << 4);
    v_off[dh] = HALF + vr * 128 + ((v_cx ^ (vr & 7)) << 4);
  }

  // One step: a group of 16 tokens.
  auto step = [&](const int stage, const int grp, const int wt0) {
    const uint32_t kbase = smem_base + stage * STAGE + (uint32_t)(grp * bpg * box_bytes);
    const uint32_t vbase = kbase + HALF;
    const bool masked = wt0 + 15 > lim_first;
    bool poisoned = false;  // V of a token that some row does not see is not a number
    if (masked) {
      unsigned char* vg = smem + (vbase - smem_base);
      const int live = it.tok_end - wt0;
      if (live < 16) {
        // whole boxes were brought (or none): tokens past the end hold whatever was there. Clear them in V so
        // that 0 * garbage cannot produce a NaN (every warp that reads them writes the same zeros).
        for (int x = lane; x < (16 - live) * DH * 8; x += 32) {
          const int ch = x & 7, dh = (x >> 3) % DH, tl = live + (x >> 3) / DH;
          *reinterpret_cast<uint4*>(vg + row_of(tl, dh) * 128 + ch * 16) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      for (int x = lane; x < 16 * DH * 8; x += 32) {
        const int ch = x & 7, dh = (x >> 3) % DH, tl = (x >> 3) / DH;
        const uint4 v = *reinterpret_cast<const uint4*>(vg + row_of(tl, dh) * 128 + ch * 16);
        poisoned |= (not_finite<T>(v.x) | not_finite<T>(v.y) | not_finite<T>(v.z) | not_finite<T>(v.w)) != 0;
      }
      poisoned = __any_sync(0xffffffffu, poisoned);
    }
    float s[2][4];  // [8-token column block][row g: 2 tokens, row g + 8: 2 tokens]
#pragma unroll
    for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      uint32_t b[4];
      ldmatrix_x4(b, (kbase + k_off[kk >> 2]) ^ ((kk & 3) << 5));
      mma16816<T>(s[0], qa[kk], b[0], b[1]);
      mma16816<T>(s[1], qa[kk], b[2], b[3]);
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = wt0 + 8 * i + 2 * tg;
        if (c > lim0) s[i][0] = -INFINITY;
        if (c + 1 > lim0) s[i][1] = -INFINITY;
        if (c > lim1) s[i][2] = -INFINITY;
        if (c + 1 > lim1) s[i][3] = -INFINITY;
      }
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][1]));
      mx1 = fmaxf(mx1, fmaxf(s[i][2], s[i][3]));
    }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    // The reference maximum moves only when a row maximum outgrew it by 2^8 (P stays below 2^8, its rounding is
    // relative), so O is rescaled a few times per request instead of at every new maximum.
    const float t0m = mx0 * sc, t1m = mx1 * sc;
    const bool grow0 = t0m > m0 + kGrow || (m0 == -INFINITY && t0m > m0), grow1 = t1m > m1 + kGrow || (m1 == -INFINITY && t1m > m1);
    if (__any_sync(0xffffffffu, grow0 || grow1)) {
      const float f0 = grow0 ? ex2(m0 - t0m) : 1.f, f1 = grow1 ? ex2(m1 - t1m) : 1.f;
      m0 = grow0 ? t0m : m0;
      m1 = grow1 ? t1m : m1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) { o[j][0] *= f0; o[j][1] *= f0; o[j][2] *= f1; o[j][3] *= f1; }
    }
    const float off0 = m0 == -INFINITY ? 0.f : -m0, off1 = m1 == -INFINITY ? 0.f : -m1;
    // P is rounded to the 16-bit type of V, as the tensor core needs it; the sum l is not
    uint32_t pa[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = ex2(fmaf(s[i][0], sc, off0)), b = ex2(fmaf(s[i][1], sc, off0));
      const float c = ex2(fmaf(s[i][2], sc, off1)), d = ex2(fmaf(s[i][3], sc, off1));
      l0 += a + b;
      l1 += c + d;
      pa[i * 2] = pack2<T>(a, b);
      pa[i * 2 + 1] = pack2<T>(c, d);
    }
#pragma unroll
    for (int jn = 0; jn < D / 16; ++jn) {
      uint32_t v[4];
      ldmatrix_x4_trans(v, (kbase + v_off[jn >> 2]) ^ ((jn & 3) << 5));
      if (poisoned) {  // a zero weight must not meet an infinity: such values are added below
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] &= ~not_finite<T>(v[k]);
      }
      mma16816<T>(o[2 * jn], pa, v[0], v[1]);
      mma16816<T>(o[2 * jn + 1], pa, v[2], v[3]);
    }
    if (poisoned) {  // the rest, token by token, only into the rows that see it
#pragma unroll 1
      for (int tl = 0; tl < 16; ++tl) {
        const int from = g * 4 + ((tl & 7) >> 1);
        const float2 w0 = unpack2<T>(__shfl_sync(0xffffffffu, tl < 8 ? pa[0] : pa[2], from));
        const float2 w1 = unpack2<T>(__shfl_sync(0xffffffffu, tl < 8 ? pa[1] : pa[3], from));
        const float a = (tl & 1) ? w0.y : w0.x, b = (tl & 1) ? w1.y : w1.x;
        const bool see0 = wt0 + tl <= lim0, see1 = wt0 + tl <= lim1;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const int d = j * 8 + tg * 2, row = row_of(tl, d >> 6);
          const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + (vbase - smem_base) + row * 128 +
                                                                ((((d & 63) >> 3) ^ (row & 7)) << 4) + (d & 7) * 2);
          const uint32_t odd = not_finite<T>(w);
          const float2 v = unpack2<T>(w);
          if (odd & 0xffffu) {
            if (see0) o[j][0] = fmaf(a, v.x, o[j][0]);
            if (see1) o[j][2] = fmaf(b, v.x, o[j][2]);
          }
          if (odd >> 16) {
            if (see0) o[j][1] = fmaf(a, v.y, o[j][1]);
            if (see1) o[j][3] = fmaf(b, v.y, o[j][3]);
          }
        }
      }
    }
  };

  bool ok = true;
  for (int tile = 0; tile < n_tiles; ++tile) {
    const int s = tile % kStages;
    if (!warp_wait(bar_full + 8 * s, (tile / kStages) & 1, p.status)) {
      ok = false;  // (still passes the barriers below: warps whose waits succeeded meet there)
      break;
    }
    const int t0 = it.tok_begin + tile * ttok + 16 * sub;  // this warp's group of the stage
    if (t0 < it.tok_end) step(s, sub, t0);
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_empty + 8 * s);  // this warp is done with the stage
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

  // ---- merge the warps that share rows and write, through shared memory ---------------------
  // every issued copy has been waited for above so the ring is free
  asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumerThreads) : "memory");
  constexpr int LD = D + 4;
  float* sc_o = reinterpret_cast<float*>(smem);        // [warp][16][LD]
  float* sc_ml = sc_o + kConsumerWarps * 16 * LD;      // [warp][16][2]
#pragma unroll
  for (int j = 0; j < D / 8; ++j) {
    *reinterpret_cast<float2*>(&sc_o[(warp * 16 + g) * LD + j * 8 + tg * 2]) = make_float2(o[j][0], o[j][1]);
    *reinterpret_cast<float2*>(&sc_o[(warp * 16 + g + 8) * LD + j * 8 + tg * 2]) = make_float2(o[j][2], o[j][3]);
  }
  if (tg == 0) {
    *reinterpret_cast<float2*>(&sc_ml[(warp * 16 + g) * 2]) = make_float2(m0, l0);
    *reinterpret_cast<float2*>(&sc_ml[(warp * 16 + g + 8) * 2]) = make_float2(m1, l1);
  }
  asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumerThreads) : "memory");

  if (!ok) return;
  // four consecutive elements of a row per thread
  const int quads = D / 4;
  for (int x = tid; x < hb * it.n_rows * quads; x += kConsumerThreads) {
    const int d = (x % quads) * 4, y = x / quads, r = y % it.n_rows, hl = y / it.n_rows;
    float mx = -INFINITY;
    for (int s2 = 0; s2 < ts; ++s2) mx = fmaxf(mx, sc_ml[((hl + s2 * hb) * 16 + r) * 2]);
    const float off = mx == -INFINITY ? 0.f : mx;
    float lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s2 = 0; s2 < ts; ++s2) {
      const int at = (hl + s2 * hb) * 16 + r;
      const float a = ex2(sc_ml[at * 2] - off);
      lsum = fmaf(sc_ml[at * 2 + 1], a, lsum);
      const float4 v = *reinterpret_cast<const float4*>(&sc_o[at * LD + d]);
      acc.x = fmaf(v.x, a, acc.x); acc.y = fmaf(v.y, a, acc.y);
      acc.z = fmaf(v.z, a, acc.z); acc.w = fmaf(v.w, a, acc.w);
    }
    const int tok = r / G, qh = (kv_group * hb + hl) * G + r % G;
    if (it.slot < 0) {
      const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
      T* dst = reinterpret_cast<T*>(p.out) + (int64_t)(it.q_row0 + tok) * p.out_stride + (int64_t)qh * D + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      if (p.lse != nullptr && d == 0)
        p.lse[(int64_t)(it.q_row0 + tok) * p.n_q_heads + qh] = lsum == 0.f ? -INFINITY : (mx + log2f(lsum)) * kLn2;
    } else {
      const int64_t at = (int64_t)(it.slot + tok) * p.n_q_heads + qh;
      *reinterpret_cast<float4*>(p.part_o + at * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mx, lsum);
    }
  }
}

// ---- host: the tensor map of one layer's pages ----------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// (64 elements, token in page, kv head, 64-element half of head_dim, 2 * page + {K, V}): one box is the
// [16 tokens x hb heads x head_dim] slab of a page's K or V, token-major per head, 128-byte swizzled.
inline bool make_tensor_map(CUtensorMap* map, const void* pages_layer, int64_t num_pages, int page_size, int n_kv_heads,
                            int head_dim, int hb, bool bf16) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return false;
  const cuuint64_t half_stride = (cuuint64_t)page_size * n_kv_heads * head_dim * 2;
  const cuuint64_t dims[5] = {64, (cuuint64_t)page_size, (cuuint64_t)n_kv_heads, (cuuint64_t)(head_dim / 64), (cuuint64_t)(2 * num_pages)};
  const cuuint64_t strides[4] = {(cuuint64_t)n_kv_heads * head_dim * 2, (cuuint64_t)head_dim * 2, 128, half_stride};
  const cuuint32_t box[5] = {64, (cuuint32_t)(page_size < 16 ? page_size : 16), (cuuint32_t)hb, (cuuint32_t)(head_dim / 64), 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
            const_cast<void*>(pages_layer), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace chunk_tma
}  // namespace dsv
