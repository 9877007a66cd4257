// Chunk attention for 16-bit K/V on the 5th-generation tensor cores, the kv axis split over CTAs.
//
// One CTA owns one item of the plan and one kv head: up to two q tiles of 128 / G tokens (the G q heads of the
// kv head stacked with the tokens into the 128 rows of an MMA) and a range of kv tokens, walked in tiles of
// 128. Its work is a sequence of units, alternating between two sets of (S, O) accumulators in TMEM:
//   two q tiles:  unit u = (kv tile u / 2, q tile u % 2)
//   one q tile:   unit u = (kv tile u, set u % 2): the even and the odd kv tiles are two partial softmaxes,
//                 joined in the epilogue
// so in either case one set's softmax warps work while the tensor core runs the other set's products:
//     S = Q K^T     tcgen05.mma (M = 128, N = 128), operands in 128B-swizzled shared memory, S in TMEM
//     softmax       thread = row = TMEM lane; the mask, a reference maximum that moves only when outgrown by
//                   2^8, P = 2^(S * scale - m) in 16 bits written over S
//     O += P V      tcgen05.mma with A = P from TMEM, B = the V tile read MN-major
// A padded MMA tile costs 2 x 512 cycles per 128 tokens, a third of the time that the tile's 64 KB take at
// full HBM speed (2850 cycles per SM), so even a few live rows are bound by the K/V traffic; warps without a
// live row only pass the barriers. K and V arrive in boxes of 16 tokens x head_dim (4 KB for head_dim 128).
//
// Measured (bf16, 8 kv heads of 128): one request of 65,536 tokens, 5 of them new, 32 q heads: 55 us with the merge, 4.9 TB/s;
// 128 requests of 512-4096 tokens, 1-8 new, 64 q heads (1.24 GB): 239 us, 5.2 TB/s. A 64 KB tile takes 1.58 us per SM in
// the steady state (6 TB/s), the rest is each CTA's fill and drain, about 6 us; CTAs that stay and carry their rings over
// several items were slower (60 and 264 us: their softmax warps spill). 16 requests of 3000-8192 tokens with 100-257 new ones
// (206 GFLOP): 340-344 us, bound by the softmax between the products.
#pragma once

#include <cuda.h>

#include "tcgen05.cuh"

namespace dsv {
namespace chunk_tc {

using namespace ptx;

constexpr int kBN = 128;      // kv tokens per tile
constexpr int kVStages = 3;
constexpr int kThreads = 352;  // 2 x 4 softmax warps, q + K producer, MMA warp, V producer
constexpr float kGrow = 8.f;   // log2 units

template <typename T, int D, bool MERGED>
__global__ void __launch_bounds__(kThreads, 1)
chunk_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const ChunkParams p, const int ps_log) {
  constexpr int DH = D / 64;
  constexpr int QTILE = 128 * D * 2;      // one q tile: [DH][128 rows][128 B]
  constexpr int KVTILE = kBN * D * 2;
  constexpr int HALF_ROWS = 128 * 128;
  static_assert(!MERGED || D == 128, "merged boxes hold both halves of a 128-element head");
  // K stage: [DH][128 tokens][128 B], or merged [16 groups][DH][8 tokens][128 B]
  constexpr int K_GROUP = MERGED ? 2048 : 1024;
  constexpr int K_HALF = MERGED ? 1024 : HALF_ROWS;
  // V stage: [DH][128 tokens][128 B], or merged [8 boxes][DH][16 tokens][128 B]
  constexpr int V_STEP = MERGED ? 4096 : 2048;
  constexpr int V_HALF = MERGED ? 2048 : HALF_ROWS;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr uint32_t IDESC_QK = instr_desc(kBf16 ? 1 : 0, 0, kBN, 128);
  constexpr uint32_t IDESC_PV = instr_desc(kBf16 ? 1 : 0, 1, D, 128);
  constexpr uint32_t COL_O = 128, COL_SET = 256;  // set x owns TMEM columns [256 x, 256 x + 256): S / P, then O

  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = p.n_q_heads / p.n_kv_heads, tq = 128 / G;
  const int kv_head = blockIdx.x % p.n_kv_heads;  // the kv heads of an item are adjacent CTAs
  const int ps = 1 << ps_log, bt = min(ps, 16), n_boxes = kBN / bt;

  if (warp == 9 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];\n prefetch.tensormap [%1];\n prefetch.tensormap [%2];\n" ::"l"(&q_map), "l"(&k_map), "l"(&v_map));
  }
  Item it;
  if (!load_item(p, blockIdx.x / p.n_kv_heads, it) || it.nq > 2 * tq) {
    if (tid == 0) record_status(p.status, ST_BAD_PLAN);
    return;
  }
  const bool dual = it.nq > tq;           // two q tiles
  const int n_tiles = (it.tok_end - it.tok_begin + kBN - 1) / kBN;
  const int units = dual ? 2 * n_tiles : n_tiles;

  // shared memory: q tiles, K stages (2 with two q tiles, 3 with one), V stages, barriers
  const int k_stages = dual ? 2 : 3;
  const uint32_t q_smem = base, k_smem = q_smem + (dual ? 2 : 1) * QTILE, v_smem = base + 2 * QTILE + 2 * KVTILE;
  const uint32_t bars = v_smem + kVStages * KVTILE;
  const uint32_t bar_q = bars, bar_kfull = bars + 8, bar_kempty = bars + 32, bar_vfull = bars + 56, bar_vempty = bars + 80,
                 bar_sfull = bars + 104, bar_pfull = bars + 120, bar_odone = bars + 136;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (bars - base) + 152);
  volatile int* poison = reinterpret_cast<volatile int*>(smem + (bars - base) + 156);
  volatile int* gave_up = poison + 1;  // some wait ran out

  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < 3; ++s) {
      mbar_init(bar_kfull + 8 * s, 1);
      mbar_init(bar_kempty + 8 * s, 1);
      mbar_init(bar_vfull + 8 * s, 1);
      mbar_init(bar_vempty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_pfull + 8 * s, 4);  // one arrival per softmax warp
      mbar_init(bar_odone + 8 * s, 1);
    }
    *poison = 0;
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) {  // TMEM: all 512 columns (one CTA per SM)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_u32(const_cast<uint32_t*>(tmem_slot))),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;   // every wait of this warp has ended
  int issued = 0;   // tiles that a producer has asked for, or whether the issuer has issued anything

  if (warp == 8 || warp == 10) {
    // ================================ TMA producers: warp 8 = q + K ring, warp 10 = V ring =======
    if (warp == 8 && lane == 0 && units > 0) {
      mbar_expect_tx(bar_q, (uint32_t)(DH * G * tq * 128 * (dual ? 2 : 1)));
      for (int x = 0; x < (dual ? 2 : 1); ++x)
        for (int dh = 0; dh < DH; ++dh)
          tma_load_4d(q_smem + x * QTILE + dh * HALF_ROWS, &q_map, bar_q, 0, kv_head * G, dh, it.q_row0 + x * tq);
    }
    const int32_t* idx = p.kv_indices + it.ip0;
    const int kv = warp == 10 ? 1 : 0;
    const int n_stages = kv ? kVStages : k_stages;
    const uint32_t ring = kv ? v_smem : k_smem, bar_full = kv ? bar_vfull : bar_kfull, bar_empty = kv ? bar_vempty : bar_kempty;
    auto page_of = [&](int tile) {  // page of this lane's box
      const int tok = it.tok_begin + tile * kBN + lane * bt;
      if (lane >= n_boxes || tok >= it.tok_end) return -1;
      int page = __ldg(idx + (tok >> ps_log));
      if (page < 0 || page >= p.num_pages) {
        record_status(p.status, ST_BAD_PAGE_ID);
        page = 0;
      }
      return page;
    };
    int page = n_tiles > 0 ? page_of(0) : -1;
    for (int tile = 0; tile < n_tiles; ++tile) {
      const int s = tile % n_stages, round = tile / n_stages;
      const int next = tile + 1 < n_tiles ? page_of(tile + 1) : -1;  // looked up ahead of the wait
      if (round > 0 && !warp_wait(bar_empty + 8 * s, (round - 1) & 1, p.status)) { ok = false; break; }
      const unsigned live = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) mbar_expect_tx(bar_full + 8 * s, (uint32_t)(__popc(live) * DH * bt * 128));
      __syncwarp();
      if (page >= 0) {
        const int in_page = (it.tok_begin + tile * kBN + lane * bt) & (ps - 1);
        if constexpr (MERGED) {  // bt = 16: one 4 KB box per 16 tokens
          const uint32_t dst = ring + (uint32_t)(s * KVTILE + lane * 4096);
          if (kv) tma_load_5d(dst, &v_map, bar_full + 8 * s, 0, in_page, kv_head, 0, 2 * page + 1);
          else tma_load_5d(dst, &k_map, bar_full + 8 * s, 0, 0, 2 * kv_head, in_page >> 3, 2 * page);
        } else {
          for (int dh = 0; dh < DH; ++dh)
            tma_load_5d(ring + (uint32_t)(s * KVTILE + dh * HALF_ROWS + lane * bt * 128), &v_map, bar_full + 8 * s, 0, in_page,
                        kv_head, dh, 2 * page + kv);
        }
      }
      page = next;
      issued = tile + 1;
    }
  } else if (warp == 9) {
    // ================================ MMA issuer (one thread) ===================================
    if (lane == 0 && units > 0) {
      ok = mbar_wait(bar_q, 0, p.status);
      issued = ok ? 1 : 0;
      auto issue_qk = [&](int u) {  // S_x = Q K_tile^T; wait for the K tile on its first use
        const int x = u & 1, tile = dual ? u >> 1 : u, s = tile % k_stages;
        if (!dual || x == 0) {
          if (!mbar_wait(bar_kfull + 8 * s, (tile / k_stages) & 1, p.status)) return false;
          tc_fence_after();
        }
        const uint32_t d = tmem + x * COL_SET;
        const uint64_t qa = smem_desc(q_smem + (dual ? x * QTILE : 0), 16, 1024), kb = smem_desc(k_smem + s * KVTILE, 16, K_GROUP);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t qoff = (uint64_t)(((kk >> 2) * HALF_ROWS + (kk & 3) * 32) / 16);
          const uint64_t koff = (uint64_t)(((kk >> 2) * K_HALF + (kk & 3) * 32) / 16);
          if (kk == 0) umma_ss(d, qa + qoff, kb + koff, IDESC_QK, 0u);
          else umma_ss_acc(d, qa + qoff, kb + koff, IDESC_QK);
        }
        tc_commit(bar_sfull + 8 * x);
        if (!dual || x == 1) tc_commit(bar_kempty + 8 * s);  // last reader of this K stage
        return true;
      };
      for (int u = 0; ok && u < min(2, units); ++u) ok = issue_qk(u);
      for (int u = 0; ok && u < units; ++u) {
        const int x = u & 1, i = u >> 1, tile = dual ? i : u, s = tile % kVStages;
        if (!dual || x == 0) ok = mbar_wait(bar_vfull + 8 * s, (tile / kVStages) & 1, p.status);
        if (ok) ok = mbar_wait(bar_pfull + 8 * x, i & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        const int ksteps = (min(kBN, it.tok_end - it.tok_begin - tile * kBN) + 15) >> 4;  // 16-token steps with a token of this part
        const uint32_t a = tmem + x * COL_SET, d = a + COL_O;
        const uint64_t vb = smem_desc(v_smem + s * KVTILE, V_HALF, 1024);
        if (ksteps == kBN / 16 && i > 0) {  // the common case, fully unrolled
#pragma unroll
          for (int kt = 0; kt < kBN / 16; ++kt) umma_ts_acc(d, a + kt * 8, vb + (uint64_t)(kt * V_STEP / 16), IDESC_PV);
        } else {
          for (int kt = 0; kt < ksteps; ++kt)
            umma_ts(d, a + kt * 8, vb + (uint64_t)(kt * V_STEP / 16), IDESC_PV, (i > 0 || kt > 0) ? 1u : 0u);
        }
        tc_commit(bar_odone + 8 * x);
        if (!dual || x == 1) tc_commit(bar_vempty + 8 * s);  // last reader of this V stage
        if (u + 2 < units) ok = issue_qk(u + 2);  // behind P V in issue order, so S / P of the set may be overwritten
      }
    }
  } else {
    // ================================ softmax / epilogue =========================================
    const int x = warp >> 2, row = tid & 127;  // set of this warp group; TMEM lane and MMA row
    const int my_units = (units + 1 - x) >> 1;
    const int tok_local = (dual ? x * tq : 0) + row / G, head = row % G;
    const bool live = row < G * tq && tok_local < it.nq;
    const bool warp_live = __any_sync(0xffffffffu, live);
    // last kv position this row sees in this part; the region that some live row of the item does not see
    const int limit = live ? min(it.limit0 + tok_local, it.tok_end - 1) : -1;
    const int hidden = max(it.limit0 + 1, it.tok_begin);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + x * COL_SET, o_addr = s_addr + COL_O;
    const float sc = p.scale_log2;
    float m_used = -INFINITY, l = 0.f;
    for (int i = 0; i < my_units; ++i) {
      if (!warp_wait(bar_sfull + 8 * x, i & 1, p.status)) { ok = false; break; }
      tc_fence_after();
      const int tile = dual ? i : 2 * i + x;
      const int t0 = it.tok_begin + tile * kBN;
      if (warp_live) {
        // the whole S row in registers: four 32-column loads in flight, one wait
        uint32_t r[kBN];
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
        tmem_wait_ld();
        if (t0 + kBN - 1 > limit) {
#pragma unroll
          for (int k = 0; k < kBN; ++k)
            if (t0 + k > limit) r[k] = 0xff800000u;  // -inf
        }
        float m8[8];  // eight independent chains of three-input maxima
#pragma unroll
        for (int k = 0; k < 8; ++k) m8[k] = __uint_as_float(r[k]);
#pragma unroll
        for (int k = 8; k + 15 < kBN; k += 16) {
#pragma unroll
          for (int j = 0; j < 8; ++j) m8[j] = fmax3(m8[j], __uint_as_float(r[k + 2 * j]), __uint_as_float(r[k + 2 * j + 1]));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) m8[j] = fmaxf(m8[j], __uint_as_float(r[kBN - 8 + j]));  // 8 + 7 * 16 = 120 done
        const float m_tile = fmaxf(fmax3(m8[0], m8[1], m8[2]), fmaxf(fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * sc;
        float factor = 1.f;
        if (m_tile > m_used + kGrow || (m_used == -INFINITY && m_tile > -INFINITY)) {
          factor = (m_used == -INFINITY) ? 0.f : exp2f(m_used - m_tile);
          m_used = m_tile;
        }
        // (O is free: S of this unit was issued behind the set's previous P V, and completions are in issue order)
        if (i > 0 && __any_sync(0xffffffffu, factor != 1.f)) {
          l *= factor;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
            tmem_st32(o_addr + c * 32, o);
          }
        }
        const float off = (m_used == -INFINITY) ? 0.f : m_used;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float x0, x1, a, b;
            ffma2(x0, x1, __uint_as_float(r[c * 32 + 2 * k]), __uint_as_float(r[c * 32 + 2 * k + 1]), sc, sc, -off, -off);
            a = ex2(x0);
            b = ex2(x1);
            fadd2(ls[2 * (k & 1)], ls[2 * (k & 1) + 1], ls[2 * (k & 1)], ls[2 * (k & 1) + 1], a, b);
            pk[k] = pack2<T>(a, b);
          }
          tmem_st16(s_addr + c * 16, pk);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        tmem_wait_st();
      }
      // V of tokens that a row does not see meets a zero weight: rows past the end of this part hold whatever was
      // there and are cleared; values of the hidden region that are no finite numbers are cleared too and handed to
      // the rows that do see them in the epilogue. All groups that use the tile write the same zeros, each before it
      // releases its own P.
      const int cols = min(kBN, it.tok_end - t0);
      const int z1 = (cols + 15) & ~15, z0 = max(0, min(hidden - t0, cols));
      if (z0 < z1) {
        const int vs = tile % kVStages;
        if (!warp_wait(bar_vfull + 8 * vs, (tile / kVStages) & 1, p.status)) { ok = false; break; }
        constexpr uint32_t E = kBf16 ? 0x7f80u : 0x7c00u;
        bool found = false;
        for (int z = row; z < (z1 - z0) * DH * 8; z += 128) {
          const int ch = z & 7, dh = (z >> 3) % DH, rr = z0 + (z >> 3) / DH;
          const int at = MERGED ? (rr >> 4) * V_STEP + dh * V_HALF + (rr & 15) * 128 : dh * HALF_ROWS + rr * 128;
          uint4* v = reinterpret_cast<uint4*>(smem + (v_smem - base) + vs * KVTILE + at + ch * 16);
          if (rr >= cols) {
            *v = make_uint4(0, 0, 0, 0);
            continue;
          }
          const uint4 a = *v;
          const uint32_t w[4] = {a.x, a.y, a.z, a.w};
          uint32_t m[4], any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            m[k] = ((w[k] & E) == E ? 0xffffu : 0u) | (((w[k] >> 16) & E) == E ? 0xffff0000u : 0u);
            any |= m[k];
          }
          if (any) {
            found = true;
            *v = make_uint4(w[0] & ~m[0], w[1] & ~m[1], w[2] & ~m[2], w[3] & ~m[3]);
          }
        }
        if (found) *poison = 1;
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_pfull + 8 * x);
    }
    // (a group without a unit waits for the other's only one: it is about to write where q lies)
    if (ok && units > 0) ok = my_units > 0 ? warp_wait(bar_odone + 8 * x, (my_units - 1) & 1, p.status) : warp_wait(bar_odone, 0, p.status);
    tc_fence_after();

    // ---- epilogue. Two q tiles: a group writes its own rows. One q tile: both groups publish (m, l) of their half
    // of the kv tiles, then group x writes the columns [x D / 2, (x + 1) D / 2) of the joined result.
    float wa = 1.f, wb = 0.f, m_all = m_used, l_all = l;
    int c0 = 0, c1 = D / 32;
    uint32_t oa = o_addr, ob = 0;
    if (dual) {
      // `poison` of both groups: a value that the other one cleared first is not found by this one. (Parts without a hidden
      // region look for none.)
      if (hidden < it.tok_end) asm volatile("bar.sync 1, 256;\n" ::: "memory");
    } else {
      float2* ml = reinterpret_cast<float2*>(smem + (q_smem - base));  // q is no longer read
      ml[x * 128 + row] = make_float2(m_used, l);
      tc_fence_before();
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      tc_fence_after();
      const float2 a = ml[row], b = ml[128 + row];
      m_all = fmaxf(a.x, b.x);
      const float off = m_all == -INFINITY ? 0.f : m_all;
      wa = exp2f(a.x - off);
      wb = exp2f(b.x - off);
      l_all = a.y * wa + b.y * wb;
      oa = tmem + lane_base + COL_O;
      ob = oa + COL_SET;
      c0 = x * (D / 64);
      c1 = c0 + D / 64;
    }
    if (ok && warp_live) {
      const bool use_a = dual ? my_units > 0 : units > 0, use_b = !dual && units > 1;
      const bool fix = *poison != 0;
      const int qh = kv_head * G + head;
      const int64_t at = (int64_t)(it.slot + tok_local) * p.n_q_heads + qh;
      const float inv = it.slot >= 0 ? 1.f : l_all == 0.f ? 0.f : 1.f / l_all;
      T* dst = reinterpret_cast<T*>(p.out) + (int64_t)(it.q_row0 + tok_local) * p.out_stride + (int64_t)qh * D;
#pragma unroll 1
      for (int c = c0; c < c1; ++c) {
        uint32_t o[32], o2[32];
        if (use_a) tmem_ld32(oa + c * 32, o);
        if (use_b) tmem_ld32(ob + c * 32, o2);
        tmem_wait_ld();
        float f[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          // a set that never ran holds nothing; one whose rows saw nothing holds 0
          float v = use_a ? __uint_as_float(o[k]) * wa : 0.f;
          if (use_b) v = fmaf(__uint_as_float(o2[k]), wb, v);
          f[k] = v;
        }
        if (live) {
          if (fix) {
            for (int t = hidden; t <= limit; ++t) {
              const int page = __ldg(p.kv_indices + it.ip0 + (t >> ps_log));
              if (page < 0 || page >= p.num_pages) continue;
              const T* v = reinterpret_cast<const T*>(p.pages) + (int64_t)page * p.page_stride +
                           ((int64_t)(ps + (t & (ps - 1))) * p.n_kv_heads + kv_head) * D + c * 32;
#pragma unroll 1
              for (int k = 0; k < 32; ++k) {
                const float e = to_f32(v[k]);
                if (!isfinite(e)) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) f[j] += j == k ? e : 0.f;
                }
              }
            }
          }
          if (it.slot < 0) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = pack2<T>(f[v * 8 + 2 * k] * inv, f[v * 8 + 2 * k + 1] * inv);
              *reinterpret_cast<uint4*>(dst + c * 32 + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<float4*>(p.part_o + at * D + c * 32 + v * 4) = make_float4(f[v * 4], f[v * 4 + 1], f[v * 4 + 2], f[v * 4 + 3]);
          }
        }
      }
      if (live && (dual || x == 0)) {
        if (it.slot >= 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_all, l_all);
        else if (p.lse != nullptr)
          p.lse[(int64_t)(it.q_row0 + tok_local) * p.n_q_heads + qh] = l_all == 0.f ? -INFINITY : (m_all + log2f(l_all)) * kLn2;
      }
    }
  }

  // ---- teardown: everyone meets here, then the allocating warp frees TMEM ----------------------
  if (!ok) *gave_up = 1;
  tc_fence_before();
  __syncthreads();
  if (*gave_up) {  // a CTA that gave up still sees its copies and products end, within the same limits
    if (warp == 8 || warp == 10) {
      const int n_stages = warp == 10 ? kVStages : k_stages;
      const uint32_t full = warp == 10 ? bar_vfull : bar_kfull;
      for (int k = max(issued - n_stages, 0); k < issued; ++k) warp_wait(full + 8 * (k % n_stages), (k / n_stages) & 1, p.status);
      if (warp == 8 && units > 0) warp_wait(bar_q, 0, p.status);
    }
    __syncthreads();
    if (warp == 9 && lane == 0 && issued) {
      tc_commit(bar_q);  // the barrier's second phase: all products issued so far
      mbar_wait(bar_q, 1, p.status);
    }
    __syncthreads();
  }
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- host: tensor maps ------------------------------------------------------------------------------
struct Maps {
  CUtensorMap q, k, v;
};

// q: (64 elements, head, 64-element half, token), box (64, G, 1, 128 / G) -> rows token * G + head. Pages: as the
// boxes of K and V want them; merged (head_dim 128, pages of 16 tokens or more): K with the token index split into
// (token mod 8, token / 8) and the half of head_dim between, so that a box lands as [8-token group][half][8 tokens]
// [128 B], which one K-major descriptor walks; V as [half][16 tokens][128 B].
template <typename Fn>
bool make_maps(Fn enc, Maps& m, const ChunkParams& p, bool merged, bool bf16) {
  const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const cuuint64_t D = p.head_dim, H = p.n_kv_heads, ps = p.page_size, P2 = 2 * (cuuint64_t)p.num_pages;
  const int G = p.n_q_heads / p.n_kv_heads;
  auto go = [&](CUtensorMap* map, int rank, const void* at, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    return enc(map, dt, rank, const_cast<void*>(at), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  const cuuint64_t qd[4] = {64, (cuuint64_t)p.n_q_heads, D / 64, (cuuint64_t)p.nnz};
  const cuuint64_t qs[3] = {D * 2, 128, (cuuint64_t)p.q_stride * 2};
  const cuuint32_t qb[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)(128 / G)};
  if (!go(&m.q, 4, p.q, qd, qs, qb)) return false;
  const cuuint64_t half = ps * H * D * 2;
  const cuuint64_t vd[5] = {64, ps, H, D / 64, P2}, vs[4] = {H * D * 2, D * 2, 128, half};
  const cuuint32_t vb[5] = {64, (cuuint32_t)(ps < 16 ? ps : 16), 1, merged ? 2u : 1u, 1};
  if (!go(&m.v, 5, p.pages, vd, vs, vb)) return false;
  m.k = m.v;
  if (merged) {
    const cuuint64_t kd[5] = {64, 8, 2 * H, ps / 8, P2}, ks[4] = {H * D * 2, 128, 8 * H * D * 2, half};
    const cuuint32_t kb[5] = {64, 8, 2, 2, 1};
    if (!go(&m.k, 5, p.pages, kd, ks, kb)) return false;
  }
  return true;
}

}  // namespace chunk_tc
}  // namespace dsv
