// Temperature / top-p sampling and the verification of drafted tokens.
//
// A row of logits gives weights w_v = exp((l_v - max l) / T). Tokens are ranked by value, lower index
// first among equals; token v is kept when the weights ranked before it sum to at most top_p times the
// whole sum. With Z the sum of the kept weights, p_v = w_v / Z for kept v and 0 otherwise. A draw with
// u in [0, 1) takes the first v in INDEX order whose running sum of p exceeds u times the whole.
//
// Which token a draw takes depends on ~1e5 borders per row: rounded sums would move some of them and the
// result would depend on how a row is cut among threads. Weights are therefore 64-bit fixed point
// (units of 2^-44 of the largest weight, evaluated in double): integer sums are exact and associative,
// so every cut of the row, and every order of the atomics, gives the same token. 2^18 entries of
// weight one still fit 63 bits, hence the bound on the vocabulary. Sums in double (one walk, before the
// largest logit is known) and in fp32 (drafts) decide only where the answer lies farther from a border
// than they can differ from the integers; what comes closer, below 1 % of ordinary rows, goes the exact
// way. So the token depends neither on the launch nor on which way a row went.
//
// A row is read from HBM once: a cluster of up to 8 CTAs keeps it in shared memory, or, with many rows,
// finds it in L2 again. The largest logit, the weight sums, the top-p border and the draw each walk it
// there. Sums and histograms of a cluster's CTAs meet through distributed shared memory.
//
// The top-p border is found without sorting: a histogram of weight over 2048 bins of (max - l) / T gives
// the bin of the border; the members of that bin are then split 2048 ways again by (value, index) until
// one token is left (two or three times).
//
// Bound by the arithmetic of the FP64 weights (about 28 instructions an entry; issue slots 64 % busy, the FP64 pipe 40 %), few rows by
// the chain of exchanges (2 us each). Measured: 1 row of 128,256 bf16 logits 16 us, 128 rows 91 us, 1024 rows without a border 160 us
// (1.6 TB/s); 64 rows of 32,003 fp32 with probabilities 34 us; verification of 128 requests with 0-7 drafts each (128,256,
// bf16) 165 us, 52 of them the streaming decision (4.1 TB/s), the rest one draw per request. Slower: 1024 rows whose border lies in a
// flat tail around zero 2.4 ms (count_border crosses the 16-bit values 2048 at a time, and most of them lie around zero); drafts at
// temperatures of 0.1 and below, where the streaming decision leaves most of them open: 240-345 us for 128 requests.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dsv {
namespace {

constexpr int kBins = 2048;
constexpr int kMaxCtas = 8;   // of a cluster (the portable limit)
constexpr int kMaxWarps = 16;
constexpr int kList = 256;    // members of the border's bin that are ranked directly
constexpr int kSub = 16;      // subsegments of a warp's part of a row
constexpr int kMaxVocab = 1 << 18, kIndexBits = 18;
constexpr double kOne = 17592186044416.0;          // 2^44: the fixed-point weight of the largest logit
constexpr double kProbOne = 1152921504606846976.0;  // 2^60: fixed-point probabilities of the residual
constexpr float kWindow = 8.f;                      // nats below the top that the first histogram covers
constexpr int kTable = 64;
typedef unsigned long long u64;
constexpr u64 kRaw = 0x4330000000000000ull;  // 2^52 as a double: integers sit behind it

// 2^(j / 64)
__constant__ double kPowers[kTable] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int vocab;
  const float* temperature;
  const float* top_p;
  const float* uniform;
  int32_t* tokens;       // sample: per row; verify: per request
  float* probs;          // sample, optional
  int64_t probs_stride;
  // verification only
  const int32_t* indptr;
  const int32_t* draft;  // token ids of the step's rows
  const float* draft_probs;
  int64_t draft_stride;
  uint8_t* ok;           // per row: the draft that follows it is accepted
  int32_t* accepted;
  int batch, nnz;
  int slice;             // entries of a CTA
  int cap;               // entries of a warp's list
  int* status;
};

// What the CTAs of a cluster show one another. Every exchange uses a slot of its own, so one cluster
// barrier per exchange is enough.
struct Slot {
  u64 a, b, c;
};
struct Shared {
  uint32_t hist_lo[kBins], hist_hi[kBins];
  double table[kTable];  // 2^(j / 64)
  Slot slot[36];
  u64 warp_a[kMaxWarps], warp_b[kMaxWarps], warp_c[kMaxWarps];
  u64 seg[kMaxWarps * kSub];  // mass of the subsegments
  u64 list[kList];       // this CTA's members of the border's bin
  u64 all_key[kList], all_w[kList];
  int n_list;
  int32_t tie;
  int near_n[kMaxWarps];
  u64 border, kept;
};

struct QuickShared {
  Slot slot[2];
  u64 warp_a[kMaxWarps], warp_b[kMaxWarps], warp_c[kMaxWarps], warp_d[kMaxWarps];
};

// ---- cluster plumbing ------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  if (cluster_size() == 1) {
    __syncthreads();
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {  // the same shared-memory object of CTA `rank`
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t ld_remote32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld_remote64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += shfl_xor64(v, o);
  return v;
}
// The cluster's sum / maximum / minimum of one integer per CTA (lane r asks CTA r: one round trip).
__device__ __forceinline__ u64 cluster_sum(const u64* p, int upto) {
  const uint32_t lane = threadIdx.x & 31;
  u64 v = (int)lane < upto ? ld_remote64(remote(p, lane)) : 0;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += shfl_xor64(v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ u64 cluster_max(const u64* p) {
  const uint32_t lane = threadIdx.x & 31;
  u64 v = lane < cluster_size() ? ld_remote64(remote(p, lane)) : 0;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = max(v, shfl_xor64(v, o));
  return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ u64 cluster_min(const u64* p) {
  const uint32_t lane = threadIdx.x & 31;
  u64 v = lane < cluster_size() ? ld_remote64(remote(p, lane)) : ~0ull;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = min(v, shfl_xor64(v, o));
  return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// order-preserving integer of a number (NaN excluded by the callers); 16 bits for 16-bit types
template <typename T>
__device__ __forceinline__ uint32_t order_key(float x) {
  x += 0.f;  // -0 ranks with +0
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t b = __half_as_ushort(__float2half_rn(x));
    return (b & 0x8000u) ? b ^ 0xffffu : b | 0x8000u;
  } else {
    const uint32_t b = __float_as_uint(x);
    const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return sizeof(T) == 2 ? k >> 16 : k;
  }
}
// (value, index) as one integer, larger = ranked earlier; unique within a row
template <typename T>
__device__ __forceinline__ u64 rank_key(float l, int index) {
  return ((u64)order_key<T>(l) << kIndexBits) | (u64)(kMaxVocab - 1 - index);
}

template <typename T>
__device__ __forceinline__ float key_value(uint32_t k) {  // the number of an order key
  if constexpr (std::is_same<T, __half>::value) {
    return __half2float(__ushort_as_half((unsigned short)((k & 0x8000u) ? k & 0x7fffu : k ^ 0xffffu)));
  } else {
    if (sizeof(T) == 2) k = (k & 0x8000u) ? k << 16 : (k << 16) | 0xffffu;
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
  }
}

// What is known of a row: its largest logit and the scale of its exponent. Fixed-point weights are
// 2^44 2^((l c - K) / 64).
struct RowScale {
  float top;     // largest logit that is a number
  float cutoff;  // entries below have weight 0 (2^-60 and less)
  float t;       // temperature
  float c32;     // log2(e) / T
  double c;      // 64 log2(e) / T
  double magic;  // 1.5 * 2^52 - K, K = round(top c): added to l c it leaves the rounded l c - K in the low word
};
__device__ __forceinline__ RowScale row_scale(float top, float temperature) {
  RowScale s;
  s.top = top;
  s.t = fminf(fmaxf(temperature, 1e-30f), 1e36f);  // (so that the cutoff below stays finite)
  s.c = 92.332482616893657 / (double)s.t;
  s.c32 = 1.442695041f / s.t;
  // A temperature so small that one unit in the last place of the top already gives weight 0 gives the same weights
  // as 2^37 / |top|, which keeps the exponents in range.
  if (fabs((double)top * s.c) > 137438953472.0) s.c = 137438953472.0 / fabs((double)top);
  const float a = fabsf(top), ulp = a > 0.f ? a - __uint_as_float(__float_as_uint(a) - 1u) : 1.4e-45f;  // (finite for the largest number too)
  s.cutoff = top - fmaxf(64.f * s.t, 2.f * ulp);
  s.magic = 6755399441055744.0 - rint((double)top * s.c);
  return s;
}
// The fixed-point weight of the top, 2^44 2^((top c - K) / 64), as a number.
__device__ __forceinline__ double top_weight(const RowScale& s) {
  return kOne * exp2(fma((double)s.top, s.c, s.magic - 6755399441055744.0) * 0.015625);
}
// Fixed-point weight behind kRaw (subtract it; sums may subtract it once per entry). With l c = N + r, |r| <= 1/2:
// 2^((N - K) / 64) from a table of 2^(j / 64) and an exponent, e^(r ln 2 / 64) by its Taylor series to the fourth power (the table-driven
// exponential of P. T. P. Tang, ACM TOMS 15, 1989) (its argument is
// below 0.0055: the next term is under 2^-44). Eight FP64 instructions: 128,256 entries keep one SM's FP64 units
// busy for 8 us, 1.5 times what its share of HBM takes to bring them in 16 bits.
__device__ __forceinline__ u64 raw_weight(float l, const RowScale& s, const double* __restrict__ table) {
  const double x = (double)fmaxf(l, s.cutoff);  // NaN and -inf too: weight 0
  const double m = fma(x, s.c, s.magic);
  const double r = fma(x, s.c, s.magic - m);
  constexpr double a = 0.010830424696249145;  // ln 2 / 64
  double e = fma(r, a * a * a * a / 24.0, a * a * a / 6.0);
  e = fma(r, e, a * a / 2.0);
  e = fma(r, e, a);
  e = fma(r, e, 1.0);
  const int n = __double2loint(m);
  const double t = table[n & (kTable - 1)];
  const double scaled = __hiloint2double(__double2hiint(t) + ((n >> 6) << 20) + (44 << 20), __double2loint(t));
  return (u64)__double_as_longlong(fma(scaled, e, 4503599627370496.0));  // + 2^52: rounded to an integer
}
__device__ __forceinline__ double weight(float l, const RowScale& s) {  // in units of the largest, for single entries
  const double x = ((double)fmaxf(l, s.cutoff) - (double)s.top) * s.c;
  return exp2(fmax(x, -64000.0) * 0.015625);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// A CTA's slice of a row as 16-byte vectors, aligned as in global memory: vector v holds the entries first + v * N and
// on; what lies before and behind the slice reads as -inf (no token). kShared: in shared memory, else in global memory
// (where the first pass has left it in L2). Rows at the ends of the number range are rewritten as they are read, without
// changing an order or a weight: +inf entries become 0 and all others -inf; a row below -1e38 is scaled by 1/4 (with its
// temperature).
enum : int { kAsIs = 0, kInfinite = 1, kQuartered = 2 };
__device__ __forceinline__ float rewritten(float l, int how) {
  return how == kInfinite ? (l == INFINITY ? 0.f : -INFINITY) : how == kQuartered ? l * 0.25f : l;
}
template <typename T, int NT, bool kShared>
struct Slice {
  static constexpr int N = Vec16<T>::N;
  const uint4* g;  // in global memory
  const uint4* v;  // where walks after the first read it
  int n_vec, first;
  int seg, sub;    // vectors of a warp's contiguous segment, of a subsegment
  int lead, tail;  // entries of the first and of the last vector that lie outside
  int limit;       // entries of the row
  int how;
  __device__ __forceinline__ void mask(int i, float (&f)[N]) const {
    if (i == 0 || i == n_vec - 1) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if ((i == 0 && k < lead) || (i == n_vec - 1 && k >= N - tail)) f[k] = -INFINITY;
    }
  }
  __device__ __forceinline__ void finish(int i, float (&f)[N]) const {
    mask(i, f);
    if (how != kAsIs) {
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = rewritten(f[k], how);
    }
  }
  __device__ __forceinline__ void get(int i, float (&f)[N]) const {
    Vec16<T>::unpack(kShared ? v[i] : ld_stream16(v + i), f);
    finish(i, f);
  }
  // of(values, first index) for the vectors [a, b), lane by lane; from L2 two vectors are on their way while one is used.
  template <typename F>
  __device__ __forceinline__ void each(int a, int b, int step, F of) const {
    float f[N];
    if (kShared) {
      for (int i = a; i < b; i += step) {
        get(i, f);
        of(f, first + i * N);
      }
      return;
    }
    uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0, u2 = u0;
    if (a < b) u0 = ld_stream16(v + a);
    if (a + step < b) u1 = ld_stream16(v + a + step);
    for (int i = a; i < b; i += step) {
      if (i + 2 * step < b) u2 = ld_stream16(v + i + 2 * step);
      Vec16<T>::unpack(u0, f);
      finish(i, f);
      of(f, first + i * N);
      u0 = u1;
      u1 = u2;
    }
  }
  // of(vector, its number): the 16-byte vectors themselves, neighbours' entries in the first and the last one included.
  template <typename F>
  __device__ __forceinline__ void each_raw(int a, int b, F of) const {
    if (kShared) {
      for (int i = a; i < b; i += 32) of(v[i], i);
      return;
    }
    uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0, u2 = u0, u3 = u0;
    if (a < b) u0 = ld_stream16(v + a);
    if (a + 32 < b) u1 = ld_stream16(v + a + 32);
    if (a + 64 < b) u2 = ld_stream16(v + a + 64);
    for (int i = a; i < b; i += 32) {
      if (i + 96 < b) u3 = ld_stream16(v + i + 96);
      of(u0, i);
      u0 = u1;
      u1 = u2;
      u2 = u3;
    }
  }
  // The same for the warp's 32 lanes together: of(values, first index) runs in all of them, with -inf behind the end.
  template <typename F>
  __device__ __forceinline__ void each_warp(int a, int b, F of) const {
    const int lane = threadIdx.x & 31;
    float f[N];
    uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0, u2 = u0;
    if (!kShared && a + lane < b) u0 = ld_stream16(v + a + lane);
    if (!kShared && a + 32 + lane < b) u1 = ld_stream16(v + a + 32 + lane);
    for (int i0 = a; i0 < b; i0 += 32) {
      const int i = i0 + lane;
      if (kShared) u0 = v[min(i, b - 1)];
      else if (i + 64 < b) u2 = ld_stream16(v + i + 64);
      Vec16<T>::unpack(u0, f);
      finish(i, f);
      if (i >= b) {
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = -INFINITY;
      }
      of(f, first + i * N);
      u0 = u1;
      u1 = u2;
    }
  }
  __device__ __forceinline__ int begin(int warp) const { return min(warp * seg, n_vec); }
  __device__ __forceinline__ int end(int warp) const { return min(warp * seg + seg, n_vec); }
  // Sum of `of(values, first index)` over every subsegment of the warp, into sh.seg; the warp's total.
  template <typename F>
  __device__ __forceinline__ u64 sum(Shared& sh, F of) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = end(warp);
    u64 total = 0;
    int at = begin(warp);
    for (int k = 0; k < kSub; ++k) {
      const int stop = min(at + sub, e);
      u64 x = 0;
      each(at + lane, stop, 32, [&](const float (&f)[N], int i) { x += of(f, i); });
      if (at < stop) x = warp_sum(x);
      if (lane == 0) sh.seg[warp * kSub + k] = x;
      total += x;
      at = stop;
    }
    return total;
  }
};

template <int N>
__device__ __forceinline__ float largest(const float (&f)[N]) {  // NaN ignored
  float m = fmaxf(f[0], f[1]);
#pragma unroll
  for (int i = 2; i < N; ++i) m = fmaxf(m, f[i]);
  return m;
}

// of(value, place) for the entries of a vector that `in` marks: one by one where they are few, side by side where many.
template <int N, typename F>
__device__ __forceinline__ void marked(const float (&f)[N], unsigned in, F of) {
  if (__popc(in) > 2) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in >> i & 1) of(f[i], i);
    return;
  }
  while (in) {
    const int i = __ffs(in) - 1;
    in &= in - 1;
    float l = f[0];
#pragma unroll
    for (int j = 1; j < N; ++j) l = i == j ? f[j] : l;
    of(l, i);
  }
}

// Geometry of the slice; `first_walk` brings it in.
template <typename T, int NT, bool kShared>
__device__ __forceinline__ Slice<T, NT, kShared> make_slice(const T* row, int vocab, int slice, uint4* buf) {
  constexpr int N = Vec16<T>::N, W = NT / 32;
  const int begin = min((int)cluster_rank() * slice, vocab), n = min(begin + slice, vocab) - begin;
  const T* src = row + begin;
  Slice<T, NT, kShared> sl;
  sl.lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  sl.g = reinterpret_cast<const uint4*>(src - sl.lead);
  sl.v = kShared ? buf : sl.g;
  sl.first = begin - sl.lead;
  sl.n_vec = n > 0 ? (sl.lead + n + N - 1) / N : 0;
  sl.tail = sl.n_vec * N - sl.lead - n;
  sl.seg = ((sl.n_vec + W * 32 - 1) / (W * 32)) * 32;
  sl.sub = max(64, ((sl.seg + kSub * 32 - 1) / (kSub * 32)) * 32);
  sl.limit = vocab;
  sl.how = kAsIs;
  return sl;
}

// The one walk over HBM: of(values, first index, first vector of the warp's turn) for the warp's segment, its 32 lanes together,
// -inf behind the end; four vectors a lane on their way. A shared slice gets its copy.
template <typename T, int NT, bool kShared, typename F>
__device__ __forceinline__ void first_walk(const Slice<T, NT, kShared>& sl, uint4* buf, F of) {
  constexpr int N = Vec16<T>::N, DEPTH = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, a = sl.begin(warp), b = sl.end(warp);
  const unsigned inner = (unsigned)max(min(b, sl.n_vec - 1) - 1, 0);  // vectors 1 .. inner need no mask
  uint4 u[DEPTH];
#pragma unroll
  for (int k = 0; k < DEPTH; ++k) {
    u[k] = make_uint4(0, 0, 0, 0);
    if (a + 32 * k + lane < b) u[k] = ld_stream16(sl.g + a + 32 * k + lane);
  }
  for (int i0 = a; i0 < b; i0 += 32 * DEPTH) {
#pragma unroll
    for (int k = 0; k < DEPTH; ++k) {
      const int at = i0 + 32 * k, i = at + lane;
      if (at >= b) break;
      const uint4 now = u[k];
      if (i + 32 * DEPTH < b) u[k] = ld_stream16(sl.g + i + 32 * DEPTH);
      if (kShared && i < b) buf[i] = now;
      float f[N];
      Vec16<T>::unpack(now, f);
      if ((unsigned)(i - 1) >= inner) {  // the slice's first or last vector, or behind the segment
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (i >= b || (i == 0 && j < sl.lead) || (i == sl.n_vec - 1 && j >= N - sl.tail)) f[j] = -INFINITY;
      }
      of(f, sl.first + i * N, at);
    }
  }
}

// How a row at the end of the number range is rewritten from here on, and its rewritten top.
template <typename T, int NT, bool kShared>
__device__ __forceinline__ float settle(Slice<T, NT, kShared>& sl, float top) {
  sl.how = top == INFINITY ? kInfinite : top < -1e38f && top > -INFINITY ? kQuartered : kAsIs;
  return rewritten(top, sl.how);
}

// Greedy walk: the row's largest entry that is a number and its lowest index (-1: there is none). Slot 0.
template <typename T, int NT, bool kShared, typename S>
__device__ int greedy_walk(const Slice<T, NT, kShared>& sl, uint4* buf, float& top, S& sh) {
  constexpr int N = Vec16<T>::N;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float best = -INFINITY;
  int at = 0x7fffffff;
  first_walk(sl, buf, [&](const float (&f)[N], int i0, int) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f[i] > best) { best = f[i]; at = i0 + i; }  // ascending: the first of equal ones stays
  });
  // (value, lowest index) as one integer; 0: nothing
  u64 k = at == 0x7fffffff ? 0 : ((u64)order_key<float>(best) << 32) | (u64)(0xffffffffu - (uint32_t)at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, shfl_xor64(k, o));
  if (lane == 0) sh.warp_a[warp] = k;
  __syncthreads();
  if (warp == 0) {
    k = lane < NT / 32 ? sh.warp_a[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = max(k, shfl_xor64(k, o));
    if (lane == 0) sh.slot[0].a = k;
  }
  cluster_sync();
  k = cluster_max(&sh.slot[0].a);
  top = k ? key_value<float>((uint32_t)(k >> 32)) : -INFINITY;
  return k ? (int)(0xffffffffu - (uint32_t)k) : -1;
}

__device__ __forceinline__ double as_double(u64 v) { return __longlong_as_double((long long)v); }
__device__ __forceinline__ u64 as_bits(double v) { return (u64)__double_as_longlong(v); }
// 2^n of an integer below 1024; 0 far below.
__device__ __forceinline__ double power(double n) {
  return n > -1022.0 ? __hiloint2double((1023 + (int)n) << 20, 0) : 0.0;
}

// 2^(l c / 64 - e) as the product of two doubles, magic = 1.5 * 2^52 - 64 e: raw_weight without the fixed point.
__device__ __forceinline__ void double_weight(float l, double c, double magic, const double* __restrict__ table, double& scaled, double& series) {
  const double x = (double)l, w = fma(x, c, magic), r = fma(x, c, magic - w);
  constexpr double a = 0.010830424696249145;
  double y = fma(r, a * a * a * a / 24.0, a * a * a / 6.0);
  y = fma(r, y, a * a / 2.0);
  y = fma(r, y, a);
  series = fma(r, y, 1.0);
  const int n = __double2loint(w);
  const double p = table[n & (kTable - 1)];
  scaled = __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));  // the weight is scaled * series
}

// Sum of the row's weights in double, and its top, from the first walk. Every warp measures against a power of two of its
// own, 2^E near its first entries' maximum (a double's range leaves 600 factors of two to both sides), so nothing has to be known
// before; the powers are joined exactly. `far`: an entry outgrew that range, or l c leaves the integers of a double: the sum
// does not hold.
struct Walk {
  float top;
  bool far;
  double e;              // the row's power
  double total;          // weights of the row in units of 2^e
  double inc;            // lane r: those of the CTAs up to r
};
constexpr double kReach = 600.0;

// Joins (mass, power) over the warp: the largest power, the masses and their running sums in it. Powers are integers, or (kReal) not.
template <bool kReal = false>
__device__ __forceinline__ void join(double& mass, double& e, double& inc, int lane) {
  double g = e;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) g = fmax(g, __shfl_xor_sync(0xffffffffu, g, o));
  mass = g > -INFINITY && e > -INFINITY ? mass * (kReal ? (double)exp2f((float)(e - g)) : power(e - g)) : 0.0;
  e = g;
  inc = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
}

// (Slot 0. sh.warp_a / b keep every warp's mass and power, sh.seg the subsegments' masses as doubles in the warp's power.)
template <typename T, int NT, bool kShared>
__device__ Walk weight_walk(const Slice<T, NT, kShared>& sl, uint4* buf, float temperature, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float t = fminf(fmaxf(temperature, 1e-30f), 1e36f);
  const double c = 92.332482616893657 / (double)t;
  if (threadIdx.x < kTable) sh.table[threadIdx.x] = kPowers[threadIdx.x];
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  float top = -INFINITY, cutoff = 0.f;
  double e = -INFINITY, magic = 0.0, mass = 0.0, part = 0.0, odd = 0.0;
  bool far = false;
  int sub = 0, next = sl.begin(warp) + sl.sub;
  if (lane < kSub) sh.seg[warp * kSub + lane] = 0;
  __syncwarp();
  auto close = [&]() {  // end of a subsegment
    part += odd;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) sh.seg[warp * kSub + sub] = as_bits(part);
    mass += part;
    part = odd = 0.0;
    ++sub;
  };
  first_walk(sl, buf, [&](const float (&f)[N], int, int at) {
    if (at >= next) {
      close();
      next += sl.sub;
    }
    float m = largest(f);
    top = fmaxf(top, m);
    if (e == -INFINITY) {  // warp-uniform: until there is an entry to measure against
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const double x = (double)m * c * 0.015625;
      if (m > -INFINITY) {
        e = fabs(x) < 1e6 ? rint(x) : 0.0;
        far |= !(fabs(x) < 1e6);
        const float reach = 0.69f * (float)kReach * t;  // what lies farther below counts as much as that: less than can be drawn
        cutoff = m - reach;
        far |= !(reach < 1e37f && cutoff > -3e38f && cutoff < m);
        magic = 6755399441055744.0 - 64.0 * e;
      }
    }
    if (e > -INFINITY && !far) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        double scaled, series;
        double_weight(fmaxf(f[i], cutoff), c, magic, sh.table, scaled, series);
        if (i & 1) odd = fma(scaled, series, odd);
        else part = fma(scaled, series, part);
      }
    }
  });
  close();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // An entry more than kReach above the warp's first ones makes the sum meaningless (it may have wrapped an exponent).
  far |= top > -INFINITY && !(((double)top * c * 0.015625 - e) < kReach);
  far = __any_sync(0xffffffffu, far);
  if (lane == 0) {
    sh.warp_a[warp] = as_bits(far ? 0.0 : mass);
    sh.warp_b[warp] = as_bits(e);
    sh.warp_c[warp] = (u64)__float_as_uint(top) | (far ? 1ull << 32 : 0);
  }
  __syncthreads();
  double inc;
  if (warp == 0) {
    const bool in = lane < NT / 32;
    mass = in ? as_double(sh.warp_a[lane]) : 0.0;
    e = in ? as_double(sh.warp_b[lane]) : -INFINITY;
    top = in ? __uint_as_float((uint32_t)sh.warp_c[lane]) : -INFINITY;
    far = __any_sync(0xffffffffu, in && (sh.warp_c[lane] >> 32) != 0);
    join(mass, e, inc, lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const double all = __shfl_sync(0xffffffffu, inc, 31);
    if (lane == 0) {
      sh.slot[0].a = as_bits(all);
      sh.slot[0].b = as_bits(e);
      sh.slot[0].c = (u64)__float_as_uint(top) | (far ? 1ull << 32 : 0);
    }
  }
  cluster_sync();
  Walk w;
  const uint32_t n = cluster_size();
  const bool in = (uint32_t)lane < n;
  mass = in ? as_double(ld_remote64(remote(&sh.slot[0].a, lane))) : 0.0;
  e = in ? as_double(ld_remote64(remote(&sh.slot[0].b, lane))) : -INFINITY;
  const u64 x = in ? ld_remote64(remote(&sh.slot[0].c, lane)) : (u64)__float_as_uint(-INFINITY);
  join(mass, e, inc, lane);
  w.top = __uint_as_float((uint32_t)x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w.top = fmaxf(w.top, __shfl_xor_sync(0xffffffffu, w.top, o));
  w.far = __any_sync(0xffffffffu, (x >> 32) != 0) || w.top == INFINITY || w.top < -1e38f;
  w.e = e;
  w.total = __shfl_sync(0xffffffffu, inc, 31);
  w.inc = inc;
  return w;
}

// First lane whose running sum exceeds the target; where rounding leaves none, the first that reaches the whole.
__device__ __forceinline__ int pick(double inc, double target, double& rest) {
  const double all = __shfl_sync(0xffffffffu, inc, 31);
  const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
  const int who = __ffs(hit ? hit : __ballot_sync(0xffffffffu, inc == all)) - 1;
  const double before = __shfl_sync(0xffffffffu, inc, max(who - 1, 0));
  rest = fmax(who > 0 ? target - before : target, 0.0);
  return who;
}

// The top's weight in the walk's units.
__device__ __forceinline__ double top_units(const Walk& w, float temperature) {
  const double c = 92.332482616893657 / (double)fminf(fmaxf(temperature, 1e-30f), 1e36f);
  return exp2((double)w.top * c * 0.015625 - w.e);
}
// How far a running sum in double, or u times the whole, may lie from the one in fixed-point weights, in the walk's units: an entry's
// two masses differ by at most 2^-45 of the top (its rounding, or all of a smaller one), which makes 2^-44 an entry for a running sum
// and a target together, taken twice; 2^-32 of the whole covers the additions (2^18 roundings of 2^-53) and the series (2^-43).
__device__ __forceinline__ double sum_margin(const Walk& w, float temperature, int vocab) {
  return (double)vocab * 0x1p-43 * top_units(w, temperature) + w.total * 0x1p-32;
}

// floor(x all) for x in [0, 1], exact (24 bits times 63); 0 for NaN and below, all above.
__device__ __forceinline__ u64 fraction_of(float x, u64 all) {
  if (!(x > 0.f)) return 0;
  if (x >= 1.f) return all;
  const uint32_t b = __float_as_uint(x), e = b >> 23;
  const u64 m = e ? (b & 0x7fffffu) | 0x800000u : b;
  const int shift = 150 - (int)max(e, 1u);  // x = m 2^-shift, 24 <= shift <= 149
  const u64 hi = __umul64hi(m, all), lo = m * all;  // hi < 2^24
  return shift < 64 ? (hi << (64 - shift)) | (lo >> shift) : hi >> min(shift - 64, 63);
}

// The entry of a vector whose mass holds the target, `run` the sum before the vector: written, and true, where the target is farther
// than the margin from both ends of that mass.
template <int N>
__device__ __forceinline__ bool take(const double (&m)[N], double run, double target, double margin, int first, int32_t* out) {
  double to_low = 0.0, to_high = 0.0;
  int i = -1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (m[j] > 0.0 && (i < 0 || run <= target)) {
      i = j;
      to_low = target - run;
      to_high = m[j] - to_low;
    }
    run += m[j];
  }
  const bool sure = to_low > margin && to_high > margin;
  if (sure) *out = first + i;
  return sure;
}

// The draw of a row without a cut from the sums that weight_walk left: only the subsegment that holds the target is read again.
// (Every CTA joins the same numbers in the same order, so exactly one of them finds the target its own.) The sums are grouped by the
// launch and count weights that cannot be drawn, so they decide only where the target lies farther than `sum_margin` from both ends
// of the token's mass; there the fixed-point sums give the same token. false (in all threads of the cluster): they do not. Slot 35.
template <typename T, int NT, bool kShared>
__device__ __forceinline__ bool draw_in_subsegment(const Slice<T, NT, kShared>& sl, const Walk& walk, float temperature, float u, int32_t* out,
                                                   Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31;
  const float t = fminf(fmaxf(temperature, 1e-30f), 1e36f);
  const double c = 92.332482616893657 / (double)t;
  double rest, inc, margin = sum_margin(walk, temperature, sl.limit);
  const int owner = pick(walk.inc, u > 0.f ? fmin((double)u, 1.0) * walk.total : 0.0, rest);
  if (owner != (int)cluster_rank()) return true;
  const bool in = lane < NT / 32;
  const double own_e = in ? as_double(sh.warp_b[lane]) : -INFINITY;
  double mass = in ? as_double(sh.warp_a[lane]) : 0.0, e = own_e;
  join(mass, e, inc, lane);
  const int w = pick(inc, rest * power(walk.e - e), rest);
  const double e_w = __shfl_sync(0xffffffffu, own_e, w);
  rest *= power(e - e_w);
  margin *= power(walk.e - e) * power(e - e_w);
  inc = lane < kSub ? as_double(sh.seg[w * kSub + lane]) : 0.0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  const int k = pick(inc, rest, rest);
  const float lowest = walk.top - 31.2f * t;  // weights below 2^-45 of the largest cannot be drawn
  const double magic = 6755399441055744.0 - 64.0 * e_w;
  const int a = min(sl.begin(w) + k * sl.sub, sl.end(w)), b = min(a + sl.sub, sl.end(w));
  for (int v0 = a; v0 < b; v0 += 32) {
    const int v = v0 + lane;
    double m[N], total = 0.0;
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = -INFINITY;
    if (v < b) sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = 0.0;
      if (f[i] >= lowest) {
        double scaled, series;
        double_weight(f[i], c, magic, sh.table, scaled, series);
        m[i] = scaled * series;
      }
      total += m[i];
    }
    inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, inc > rest);
    if (hit) {
      const int who = __ffs(hit) - 1;
      const double before = __shfl_up_sync(0xffffffffu, inc, 1);
      bool sure = false;
      if (lane == who) sure = take(m, lane > 0 ? before : 0.0, rest, margin, sl.first + v * N, out);
      return __any_sync(0xffffffffu, sure) != 0;
    }
    rest = fmax(rest - __shfl_sync(0xffffffffu, inc, 31), 0.0);
  }
  return false;  // among weights that cannot be drawn
}
template <typename T, int NT, bool kShared>
__device__ bool draw_all(const Slice<T, NT, kShared>& sl, const Walk& walk, float temperature, float u, int32_t* out, Shared& sh) {
  if (threadIdx.x < 32) {
    const bool sure = draw_in_subsegment(sl, walk, temperature, u, out, sh);
    if (threadIdx.x == 0) sh.slot[35].a = sure ? 0 : 1;
  }
  cluster_sync();
  return cluster_max(&sh.slot[35].a) == 0;
}

// Sums over the cluster of up to three integers per warp (in its lane 0), through slot `s`: the wholes, and what the CTAs
// before this one have of the first. The warps' first integers stay in sh.warp_a.
template <int NT>
__device__ Slot cluster_total(u64 a, u64 b, u64 c, Shared& sh, int s, u64& before) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) { sh.warp_a[warp] = a; sh.warp_b[warp] = b; sh.warp_c[warp] = c; }
  __syncthreads();
  if (warp < 3) {
    const u64 v = warp_sum(lane < NT / 32 ? (warp == 0 ? sh.warp_a : warp == 1 ? sh.warp_b : sh.warp_c)[lane] : 0);
    if (lane == 0) (warp == 0 ? sh.slot[s].a : warp == 1 ? sh.slot[s].b : sh.slot[s].c) = v;
  }
  cluster_sync();
  const uint32_t n = cluster_size();
  if (n == 1) {
    before = 0;
    return sh.slot[s];
  }
  u64 v = lane < n ? ld_remote64(remote(&sh.slot[s].a, lane)) : 0, w = lane < n ? ld_remote64(remote(&sh.slot[s].b, lane)) : 0,
      y = lane < n ? ld_remote64(remote(&sh.slot[s].c, lane)) : 0, x = lane < cluster_rank() ? v : 0;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) { v += shfl_xor64(v, o); w += shfl_xor64(w, o); x += shfl_xor64(x, o); y += shfl_xor64(y, o); }
  Slot all;
  all.a = __shfl_sync(0xffffffffu, v, 0);
  all.b = __shfl_sync(0xffffffffu, w, 0);
  all.c = __shfl_sync(0xffffffffu, y, 0);
  before = __shfl_sync(0xffffffffu, x, 0);
  return all;
}

// Histogram entries are 64 bits in two words: the low word's atomic tells whether it wrapped.
__device__ __forceinline__ void hist_add(Shared& sh, int bin, u64 w) {
  const uint32_t lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
  const uint32_t old = atomicAdd(&sh.hist_lo[bin], lo);
  const uint32_t up = hi + (old + lo < old ? 1u : 0u);
  if (up) atomicAdd(&sh.hist_hi[bin], up);
}
template <int NT>
__device__ __forceinline__ void hist_clear(Shared& sh) {
  for (int i = threadIdx.x; i < kBins / 4; i += NT) {
    reinterpret_cast<uint4*>(sh.hist_lo)[i] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(sh.hist_hi)[i] = make_uint4(0, 0, 0, 0);
  }
}

// First bin of the cluster's summed histogram whose inclusive running sum exceeds a limit, the sum before it and its own
// mass; -1: none, `before` is the whole. Each CTA sums its share of the bins over the cluster; mass_of(bin, sum) makes a mass of a
// bin's sum. Slots s to s + 2.
template <int NT, typename F>
__device__ int hist_find(Shared& sh, int s, u64 limit, u64& before, u64& mass, F mass_of) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = cluster_size(), rank = cluster_rank();
  constexpr int MAX = kBins / NT;
  const int bins = kBins / c, per = max(1, bins / NT);  // bins of this CTA, of a thread
  cluster_sync();  // all histograms are complete
  u64 v[MAX], mine = 0;
  const int b0 = threadIdx.x * per;
#pragma unroll
  for (int i = 0; i < MAX; ++i) {
    v[i] = 0;
    if (i < per && b0 + i < bins) {
      const int b = rank * bins + b0 + i;
      if (c == 1) {
        v[i] = ((u64)sh.hist_hi[b] << 32) + sh.hist_lo[b];
      } else {
        uint32_t lo[kMaxCtas], hi[kMaxCtas];  // all in flight at once
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) {
          lo[r] = r < c ? ld_remote32(remote(&sh.hist_lo[b], r)) : 0;
          hi[r] = r < c ? ld_remote32(remote(&sh.hist_hi[b], r)) : 0;
        }
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) v[i] += ((u64)hi[r] << 32) + lo[r];
      }
      v[i] = mass_of(b, v[i]);
    }
    mine += v[i];
  }
  const u64 inc = warp_scan(mine, lane), warp_mass = __shfl_sync(0xffffffffu, inc, 31);
  if (threadIdx.x == 0) sh.slot[s + 1].a = ~0ull;
  u64 cta_before, base = 0;
  const Slot all = cluster_total<NT>(warp_mass, 0, 0, sh, s, cta_before);
  for (int w = 0; w < warp; ++w) base += sh.warp_a[w];
  u64 at = cta_before + base + inc - mine;
  if (at <= limit && at + mine > limit) {
#pragma unroll
    for (int i = 0; i < MAX; ++i) {
      if (at <= limit && at + v[i] > limit) {
        sh.slot[s + 1].a = (u64)(rank * bins + b0 + i);
        sh.slot[s + 1].b = at;
        sh.slot[s + 2].a = v[i];
      }
      at += v[i];
    }
  }
  before = all.a;
  if (all.a <= limit) return -1;
  cluster_sync();
  const uint32_t l = lane < c ? lane : 0;
  const u64 x = ld_remote64(remote(&sh.slot[s + 1].a, l)), y = ld_remote64(remote(&sh.slot[s + 1].b, l)),
            z = ld_remote64(remote(&sh.slot[s + 2].a, l));
  const int from = __ffs(__ballot_sync(0xffffffffu, x != ~0ull)) - 1;
  before = __shfl_sync(0xffffffffu, y, from);
  mass = __shfl_sync(0xffffffffu, z, from);
  return (int)__shfl_sync(0xffffffffu, x, from);
}

// A warp's entries within kWindow nats of the top, in index order. They are a small part of most rows, and where all of them
// are held and the border lies among them, nothing behind them is looked at again.
struct Entry {
  u64 w;
  float l;
  int i;
};
struct Near {
  Entry* all;  // of the CTA: `cap` for each warp
  int cap, n;  // entries of this warp (n > cap: not all are held)
  bool usable;
  __device__ __forceinline__ Entry* mine() const { return all + (threadIdx.x >> 5) * cap; }
};

// The kept tokens: those above `value`, and of those equal to it the ones up to index `index`.
struct Kept {
  float value;
  int index;
  u64 total;  // sum of the kept weights
  __device__ __forceinline__ bool holds(float l, int i) const { return l > value || (l == value && i <= index); }
};
template <typename T>
__device__ __forceinline__ void set_border(Kept& k, u64 key) {
  k.value = key_value<T>((uint32_t)(key >> kIndexBits));
  k.index = kMaxVocab - 1 - (int)(key & (kMaxVocab - 1));
}

// First index whose running sum of mass exceeds a target; sh.seg holds the masses of the subsegments, `mine` (per warp)
// their sum. target_of(whole) gives the target, below the whole. The CTA that holds the index writes it to *out. Returns the
// whole; 0: there is no mass. One slot.
template <typename T, int NT, bool kShared, typename M, typename F>
__device__ u64 locate(const Slice<T, NT, kShared>& sl, Shared& sh, int slot, u64 mine, M mass, F target_of, int32_t* out) {
  constexpr int N = Vec16<T>::N, PER = NT / 32 * kSub / 32;  // subsegments of a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 before;
  const u64 all = cluster_total<NT>(mine, 0, 0, sh, slot, before).a;
  if (all == 0 || warp != 0) return all;
  u64 target = target_of(all);
  u64 own[PER], sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) { own[k] = sh.seg[lane * PER + k]; sum += own[k]; }
  u64 inc = warp_scan(sum, lane);
  const u64 cta = __shfl_sync(0xffffffffu, inc, 31);
  if (target < before || target - before >= cta) return all;  // another CTA's
  target -= before;
  const int who = __ffs(__ballot_sync(0xffffffffu, inc > target)) - 1;
  int which = 0;
  u64 run = inc - sum;  // of the lane that holds it: its subsegment and what lies before
  if (lane == who) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (which == k && run + own[k] <= target) { run += own[k]; which = k + 1; }
    }
  }
  which = who * PER + __shfl_sync(0xffffffffu, which, who);
  target -= __shfl_sync(0xffffffffu, run, who);
  const int w = which / kSub, a = min(sl.begin(w) + which % kSub * sl.sub, sl.end(w)), b = min(a + sl.sub, sl.end(w));
  for (int v0 = a; v0 < b; v0 += 32) {
    const int v = v0 + lane;
    u64 m[N], total = 0;
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = -INFINITY;
    if (v < b) sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = f[i] > -INFINITY ? mass(f[i], sl.first + v * N + i) : 0;
      total += m[i];
    }
    inc = warp_scan(total, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        run = inc - total;
        int i = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          run += m[k];
          if (run <= target) i = k + 1;
        }
        *out = sl.first + v * N + i;
      }
      break;
    }
    target -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return all;
}

// The border among the entries that the CTAs' lists hold (kList at most, behind a cluster barrier): every CTA fetches them all, a thread
// weighs what ranks before its entry.
template <typename T>
__device__ void rank_members(u64 limit, u64 kept, const RowScale& s, Kept& k, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = cluster_size();
  const int mine = lane < c ? (int)ld_remote32(remote(&sh.n_list, lane)) : 0;
  const int upto = (int)warp_scan((u64)mine, lane), members = __shfl_sync(0xffffffffu, upto, 31);
  if (warp < c) {  // warp r fetches CTA r's
    const int n = __shfl_sync(0xffffffffu, mine, warp), first = __shfl_sync(0xffffffffu, upto, warp) - n;
    for (int i = lane; i < n; i += 32) {
      const u64 key = ld_remote64(remote(&sh.list[i], warp));
      sh.all_key[first + i] = key;
      sh.all_w[first + i] = raw_weight(key_value<T>((uint32_t)(key >> kIndexBits)), s, sh.table) - kRaw;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < members; i += blockDim.x) {
    const u64 key = sh.all_key[i];
    u64 above = 0;
    for (int j = 0; j < members; ++j) above += sh.all_key[j] > key ? sh.all_w[j] : 0;
    if (above <= limit && above + sh.all_w[i] > limit) {  // the last kept one
      sh.border = key;
      sh.kept = above + sh.all_w[i];
    }
  }
  __syncthreads();
  set_border<T>(k, sh.border);
  k.total = kept + sh.kept;
}

// The border falls among `count` entries equal to `value`: the ones with the lowest indices are kept, as many as begin within the
// limit. k.total comes with what ranks before them. Slots 14 and 15.
template <typename T, int NT, bool kShared>
__device__ void keep_ties(const Slice<T, NT, kShared>& sl, float value, u64 limit, u64 count, const RowScale& s, Kept& k, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const u64 w = raw_weight(value, s, sh.table) - kRaw, n = limit / w + 1;
  k.value = value;
  k.total += n * w;
  if (n >= count) {
    k.index = kMaxVocab;
    return;
  }
  if (threadIdx.x == 0) sh.tie = -1;
  const u64 mine = sl.sum(sh, [&](const float (&f)[N], int) {
    int x = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) x += f[i] == value ? 1 : 0;
    return (u64)x;
  });
  locate(sl, sh, 14, mine, [&](float l, int) { return l == value ? (u64)1 : 0; }, [&](u64) { return n - 1; }, &sh.tie);
  __syncthreads();
  if (threadIdx.x == 0) sh.slot[15].a = (u64)(sh.tie + 1);
  cluster_sync();
  k.index = (int)cluster_max(&sh.slot[15].a) - 1;
}

// Border of a row of 16-bit logits that lies behind the list: entries are counted by their very value, 2048 order keys (16 factors
// of two in bf16, 2 in fp16) at a time, and a bin's mass is its count times one weight. Eight instructions per entry instead of the 45
// of weighing each; the members of a bin are equal, so only their indices are left to look at. false: the border lies on a zero, whose
// two signs are one value. Slots 3 to 8 in turn.
template <typename T, int NT, bool kShared>
__device__ bool count_border(const Slice<T, NT, kShared>& sl, const RowScale& s, u64 limit, Kept& k, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k.total = 0;
  int key0 = (int)order_key<T>(s.top);
  for (int round = 0; key0 >= 0; ++round, key0 -= kBins) {
    hist_clear<NT>(sh);
    __syncthreads();
    sl.each_raw(sl.begin(warp) + lane, sl.end(warp), [&](const uint4& u, int i) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      const bool edge = i == 0 || i == sl.n_vec - 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t neg = (w[j] >> 15) & 0x00010001u;               // signs
        const uint32_t key = w[j] ^ (neg * 0xffffu | 0x80008000u);     // order keys of both halves
        const uint32_t a = (uint32_t)key0 - (key & 0xffffu), b = (uint32_t)key0 - (key >> 16);
        bool in_a = a < (uint32_t)kBins, in_b = b < (uint32_t)kBins;
        if (edge) {
          const int at = i * N + 2 * j;
          in_a = in_a && at >= sl.lead && at < sl.n_vec * N - sl.tail;
          in_b = in_b && at + 1 >= sl.lead && at + 1 < sl.n_vec * N - sl.tail;
        }
        if (in_a) atomicAdd(&sh.hist_lo[a], 1u);
        if (in_b) atomicAdd(&sh.hist_lo[b], 1u);
      }
    });
    u64 before, mass;
    const int bin = hist_find<NT>(sh, 3 + 3 * (round & 1), limit, before, mass,
                                  [&](int b, u64 n) { return n ? n * (raw_weight(key_value<T>((uint32_t)(key0 - b)), s, sh.table) - kRaw) : 0; });
    limit -= before;
    k.total += before;
    if (bin >= 0) {
      const float value = key_value<T>((uint32_t)(key0 - bin));
      if (value == 0.f) return false;
      keep_ties(sl, value, limit, mass / (raw_weight(value, s, sh.table) - kRaw), s, k, sh);
      return true;
    }
    cluster_sync();  // the slots of the round before last are free
  }
  return false;  // cannot happen with top_p < 1
}

// Top-p border of the row. `known`: the sum of its weights in units of the fixed-point weights, or -1. Without a cut the masses of
// the subsegments are left in sh.seg (`mine`: the warp's). Slots 2 to 30.
template <typename T, int NT, bool kShared>
__device__ Kept find_kept(const Slice<T, NT, kShared>& sl, const RowScale& s, float top_p, double known, Near& near, Shared& sh, u64& mine) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Kept k;
  k.value = -INFINITY;
  k.index = -1;
  const int w0 = sl.begin(warp), w1 = sl.end(warp);
  u64 before;
  mine = 0;
  near.n = 0;
  near.usable = false;
  if (!(top_p < 1.f)) {  // NaN: no cut
    mine = sl.sum(sh, [&](const float (&f)[N], int) {
      u64 x = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) x += raw_weight(f[i], s, sh.table);
      return x - N * kRaw;
    });
    k.total = cluster_total<NT>(mine, 0, 0, sh, 2, before).a;
    return k;
  }
  // One walk gives the sum and the list of the tokens near the top (and the sum of all, where that is not known).
  float from = INFINITY, base = s.top, to = s.top - kWindow * s.t, scale = (float)kBins / (kWindow * s.t);
  u64 whole_mass = 0, sum = 0;
  Entry* list = near.mine();
  sl.each_warp(w0, w1, [&](const float (&f)[N], int i0) {
    if (known < 0.0) {
#pragma unroll
      for (int i = 0; i < N; ++i) whole_mass += raw_weight(f[i], s, sh.table);
      whole_mass -= N * kRaw;
    }
    if (__any_sync(0xffffffffu, largest(f) >= to)) {
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) in |= f[i] >= to ? 1u << i : 0u;
      const int n = __popc(in);
      int at = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += t;
      }
      const int total = __shfl_sync(0xffffffffu, at, 31);
      at += near.n - n;
      while (in) {
        const int i = __ffs(in) - 1;
        in &= in - 1;
        float l = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) l = i == j ? f[j] : l;
        const u64 w = raw_weight(l, s, sh.table) - kRaw;  // evaluated again
        sum += w;
        if (at < near.cap) list[at] = {w, l, i0 + i};
        ++at;
      }
      near.n += total;
    }
  });
  if (lane == 0) sh.near_n[warp] = near.n;
  int put = 0;  // the cluster's entries, should they be few
  if (lane == 0 && near.n > 0) put = atomicAdd(&sh.n_list, near.n);
  put = __shfl_sync(0xffffffffu, put, 0);
  __syncwarp();  // the entries were written by other lanes, and a shuffle orders no memory
  for (int i = lane; i < min(near.n, near.cap); i += 32)
    if (put + i < kList) sh.list[put + i] = rank_key<T>(list[i].l, list[i].i);
  Slot whole = cluster_total<NT>(warp_sum(sum), warp_sum(whole_mass), (u64)near.n + (near.n > near.cap ? 1ull << 40 : 0), sh, 2, before);
  if (known >= 0.0) whole.b = (u64)known;
  k.total = whole.b;
  u64 limit = fraction_of(top_p, whole.b), mass, kept = 0;
  near.usable = limit < whole.a && whole.c < 1ull << 40;
  if constexpr (sizeof(T) == 2) {
    if (!near.usable && sl.how == kAsIs && count_border(sl, s, limit, k, sh)) return k;
    k.value = -INFINITY;
    k.index = -1;
    k.total = whole.b;
  }
  int bin = -1, window = 0;
  if (!(near.usable && whole.c <= kList)) {
    cluster_sync();
    // Histograms over windows of kWindow nats, the last one to where weights end. (The tail of a vocabulary is most of its
    // entries and seldom holds the border.)
    for (; bin < 0; ++window) {
      if (window > 0 || limit >= whole.a) {
        if (window == 0) {
          limit -= whole.a;
          kept = whole.a;
          window = 1;
        }
        if (window == 3) {  // cannot happen with top_p < 1: the whole exceeds the limit
          k.total = kept;
          return k;
        }
        from = base = to;
        to = window == 1 ? s.top - 2.f * kWindow * s.t : s.cutoff;
        scale = (float)kBins / (window == 1 ? kWindow * s.t : (64.f - 2.f * kWindow) * s.t);
      }
      hist_clear<NT>(sh);  // (every CTA has read it: the cluster barrier in cluster_total)
      __syncthreads();
      auto count = [&](float l, u64 w) { hist_add(sh, min((int)((base - l) * scale), kBins - 1), w); };
      if (near.usable) {
        for (int i = lane; i < near.n; i += 32) count(list[i].l, list[i].w);
      } else {
        sl.each(w0 + lane, w1, 32, [&](const float (&f)[N], int) {
          unsigned in = 0;
          if (largest(f) < to) return;
#pragma unroll
          for (int i = 0; i < N; ++i) in |= f[i] >= to && f[i] < from && f[i] > s.cutoff ? 1u << i : 0u;
          marked(f, in, [&](float l, int) { count(l, raw_weight(l, s, sh.table) - kRaw); });
        });
      }
      bin = hist_find<NT>(sh, 3 + 3 * window, limit, before, mass, [](int, u64 w) { return w; });
      limit -= before;
      kept += before;
    }
  }
  if (near.usable && whole.c <= kList) {  // few: every CTA ranks all of them
    rank_members<T>(limit, kept, s, k, sh);
    return k;
  }
  // Members of the border's bin: listed, and the range of their rank keys. In the row the values around the bin are found by two
  // comparisons, with room for the rounding of the bin's arithmetic, the members among them by their bin.
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  const float width = 1.f / scale, slack = 1e-6f * (fabsf(base) + (float)(bin + 1) * width);
  const float v_hi = base - (float)bin * width + slack, v_lo = bin == kBins - 1 ? to : base - (float)(bin + 1) * width - slack;
  u64 lo = ~0ull, hi = 0;
  auto member = [&](float l, int i) {
    if (min((int)((base - l) * scale), kBins - 1) != bin) return;
    const u64 key = rank_key<T>(l, i);
    lo = min(lo, key);
    hi = max(hi, key);
    const int at = atomicAdd(&sh.n_list, 1);
    if (at < kList) sh.list[at] = key;
  };
  if (near.usable) {
    for (int i = lane; i < near.n; i += 32) member(list[i].l, list[i].i);
  } else {
    sl.each(w0 + lane, w1, 32, [&](const float (&f)[N], int i0) {
      if (largest(f) < v_lo) return;
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) in |= f[i] <= v_hi && f[i] >= v_lo ? 1u << i : 0u;
      while (in) {
        const int i = __ffs(in) - 1;
        in &= in - 1;
        float l = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) l = i == j ? f[j] : l;
        if (l >= to && l < from && l > s.cutoff) member(l, i0 + i);
      }
    });
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lo = min(lo, shfl_xor64(lo, o)); hi = max(hi, shfl_xor64(hi, o)); }
  if (lane == 0) { sh.warp_a[warp] = lo; sh.warp_b[warp] = hi; }
  __syncthreads();
  if (warp == 0) {
    lo = lane < NT / 32 ? sh.warp_a[lane] : ~0ull;
    hi = lane < NT / 32 ? sh.warp_b[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { lo = min(lo, shfl_xor64(lo, o)); hi = max(hi, shfl_xor64(hi, o)); }
    if (lane == 0) {
      sh.slot[12].a = lo;
      sh.slot[12].b = hi;
      sh.slot[13].a = (u64)sh.n_list;
    }
  }
  cluster_sync();  // also: every CTA has read the histogram that is cleared next
  lo = cluster_min(&sh.slot[12].a);
  hi = cluster_max(&sh.slot[12].b);
  const int c = cluster_size();
  const int members = (int)cluster_sum(&sh.slot[13].a, c);
  if (members <= kList) {
    rank_members<T>(limit, kept, s, k, sh);
    return k;
  }
  if ((lo >> kIndexBits) == (hi >> kIndexBits)) {  // many, but of one value (16-bit logits)
    k.total = kept;
    keep_ties(sl, key_value<T>((uint32_t)(lo >> kIndexBits)), limit, members, s, k, sh);
    return k;
  }
  for (int s0 = 16;; s0 += 3) {  // 50 bits of rank key, 11 a round: five rounds at most
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
    hist_clear<NT>(sh);
    __syncthreads();
    sl.each(w0 + lane, w1, 32, [&](const float (&f)[N], int i0) {
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) in |= f[i] <= v_hi && f[i] >= v_lo && f[i] > s.cutoff ? 1u << i : 0u;
      while (in) {
        const int i = __ffs(in) - 1;
        in &= in - 1;
        float l = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) l = i == j ? f[j] : l;
        const u64 key = rank_key<T>(l, i0 + i);
        if (key >= lo && key <= hi) hist_add(sh, (int)((hi - key) >> shift), raw_weight(l, s, sh.table) - kRaw);
      }
    });
    bin = hist_find<NT>(sh, s0, limit, before, mass, [](int, u64 w) { return w; });
    if (bin < 0) {  // cannot happen: the members' mass exceeds the limit
      k.total = kept + before;
      return k;
    }
    limit -= before;
    kept += before;
    hi -= (u64)bin << shift;
    const u64 wide = (1ull << shift) - 1;
    lo = hi - lo > wide ? hi - wide : lo;
    if (shift == 0) {
      set_border<T>(k, hi);
      k.total = kept + mass;
      return k;
    }
  }
}

// The same with a border that does not depend on the launch. `known` comes from sums in double, so that the limit top_p * known may lie to
// the other side of a token's mass than the one of the fixed-point sum: a border that close to an end of its token's mass (the two
// sums differ by 2^-45 of the top, half a unit, an entry, and 2^-33 of the whole, see sum_margin) is searched again with that sum.
template <typename T, int NT, bool kShared>
__device__ __forceinline__ Kept settled_border(const Slice<T, NT, kShared>& sl, const RowScale& s, float top_p, double known, Near& near, Shared& sh,
                                               u64& mine) {
  for (;;) {
    const Kept k = find_kept(sl, s, top_p, known, near, sh, mine);
    if (!(top_p < 1.f) || known < 0.0) return k;
    const u64 limit = fraction_of(top_p, (u64)known), margin = (u64)sl.limit + (u64)(known * 0x1p-32);
    const u64 below = k.total - (raw_weight(k.value, s, sh.table) - kRaw);  // ranked before the last kept token
    if (limit > below + margin && limit + margin < k.total) return k;
    known = -1.0;
    cluster_sync();  // the others may still read this CTA's slots and list
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
  }
}

// One entry's mass in a draw.
struct Mass {
  RowScale s;
  Kept kept;
  double inv_z;         // 1 / Z in units of 2^-44, residual only
  const float* minus;   // row of the draft distribution to subtract, or null
  int one_hot;          // or the token whose draft probability is 1, or -1
  bool residual;
  __device__ __forceinline__ u64 of_kept(float l, int i, const double* table) const { return of_weight(raw_weight(l, s, table) - kRaw, i); }
  __device__ __forceinline__ u64 of_weight(u64 w, int i) const {
    if (residual && w) {
      const double q = minus != nullptr ? (double)__ldg(minus + i) : i == one_hot ? 1.0 : 0.0;
      const double r = (double)w * inv_z - q;
      w = r > 0.0 ? (u64)__double2ull_rn(r * kProbOne) : 0;
    }
    return w;
  }
};

// First index whose running sum of mass exceeds u * (whole sum); false when there is no mass. `ready`: sh.seg holds the masses
// of the subsegments already, `mine` the warp's.
template <typename T, int NT, bool kShared>
__device__ bool draw(const Slice<T, NT, kShared>& sl, const Mass& mass, const Near& near, float u, bool ready, u64 mine, int slot, int32_t* out,
                     Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto target_of = [&](u64 all) { return min(fraction_of(u, all), all - 1); };
  if (near.usable) {  // every kept token is in the lists
    auto of = [&](const Entry& e) { return mass.kept.holds(e.l, e.i) ? mass.of_weight(e.w, e.i) : 0; };
    const Entry* list = near.mine();
    mine = 0;
    for (int i = lane; i < near.n; i += 32) mine += of(list[i]);
    u64 before;
    const u64 all = cluster_total<NT>(warp_sum(mine), 0, 0, sh, slot, before).a;
    if (all == 0 || warp != 0) return all != 0;
    u64 target = target_of(all);
    const u64 own = lane < NT / 32 ? sh.warp_a[lane] : 0;
    u64 inc = warp_scan(own, lane);
    const u64 cta = __shfl_sync(0xffffffffu, inc, 31);
    if (target < before || target - before >= cta) return true;  // another CTA's
    target -= before;
    const int w = __ffs(__ballot_sync(0xffffffffu, inc > target)) - 1;
    target -= __shfl_sync(0xffffffffu, inc - own, w);
    list = near.all + w * near.cap;
    const int n = sh.near_n[w];
    for (int i0 = 0; i0 < n; i0 += 32) {
      const u64 m = i0 + lane < n ? of(list[i0 + lane]) : 0;
      inc = warp_scan(m, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
      if (hit) {
        if (lane == 0) *out = list[i0 + __ffs(hit) - 1].i;
        break;
      }
      target -= __shfl_sync(0xffffffffu, inc, 31);
    }
    return true;
  }
  if (!ready) {
    mine = sl.sum(sh, [&](const float (&f)[N], int at) {
      if (largest(f) < mass.kept.value) return (u64)0;
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) in |= f[i] >= mass.kept.value && mass.kept.holds(f[i], at + i) ? 1u << i : 0u;
      u64 x = 0;
      marked(f, in, [&](float l, int i) { x += mass.of_kept(l, at + i, sh.table); });
      return x;
    });
  }
  return locate(sl, sh, slot, mine, [&](float l, int i) { return mass.kept.holds(l, i) ? mass.of_kept(l, i, sh.table) : 0; }, target_of, out) != 0;
}

// The lists lie at the start of the dynamic shared memory, the slice behind them.
template <int NT>
__device__ __forceinline__ uint4* slice_of(unsigned char* dyn, const SampleParams& p) {
  return reinterpret_cast<uint4*>(dyn + (size_t)p.cap * (NT / 32) * sizeof(Entry));
}

// The draw of a row without a cut from max(p - q, 0), in double like weight_walk: masses of the subsegments, then the one that holds
// the target again. As in draw_all the sums decide only away from the ends of the token's mass: p of an entry differs from the
// fixed-point one by 2^-45 of the top's p and by the relative difference of the two wholes, which makes twice sum_margin here, in
// units of the whole. false (in all threads of the cluster): they do not, or hardly anything is left. Slots 33 and 35.
template <typename T, int NT, bool kShared>
__device__ bool draw_rest(const Slice<T, NT, kShared>& sl, const Walk& walk, float temperature, const float* q, int one_hot, float u,
                          int32_t* out, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float t = fminf(fmaxf(temperature, 1e-30f), 1e36f), lowest = walk.top - 31.2f * t;
  const double c = 92.332482616893657 / (double)t, magic = 6755399441055744.0 - 64.0 * walk.e, inv = 1.0 / walk.total;
  const bool wide = q != nullptr && ((reinterpret_cast<uintptr_t>(q + sl.first) & 15) == 0);
  auto rest_of = [&](const float (&f)[N], int i0, double (&m)[N]) {
    float d[N];
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = i0 + i == one_hot ? 1.f : 0.f;
    if (q != nullptr) {
      const bool inside = i0 >= 0 && i0 + N <= sl.limit;
      if (wide && inside) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(q + i0 + i));
          d[i] = x.x; d[i + 1] = x.y; d[i + 2] = x.z; d[i + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = f[i] >= lowest ? __ldg(q + i0 + i) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double scaled, series;
      double_weight(fmaxf(f[i], lowest), c, magic, sh.table, scaled, series);
      const double y = fma(scaled * series, inv, -(double)d[i]);
      m[i] = f[i] >= lowest && y > 0.0 ? y : 0.0;
    }
  };
  double mass = 0.0;
  const int e = sl.end(warp);
  int at = sl.begin(warp);
  __syncthreads();  // weight_walk's masses in sh.seg are no longer needed
  for (int k = 0; k < kSub; ++k) {
    const int stop = min(at + sl.sub, e);
    double x = 0.0;
    sl.each(at + lane, stop, 32, [&](const float (&f)[N], int i0) {
      double m[N];
      rest_of(f, i0, m);
#pragma unroll
      for (int i = 0; i < N; ++i) x += m[i];
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) sh.seg[warp * kSub + k] = as_bits(x);
    mass += x;
    at = stop;
  }
  if (lane == 0) sh.warp_a[warp] = as_bits(mass);
  __syncthreads();
  double inc, same = 0.0;
  if (warp == 0) {
    mass = lane < NT / 32 ? as_double(sh.warp_a[lane]) : 0.0;
    same = 0.0;
    join(mass, same, inc, lane);
    const double all = __shfl_sync(0xffffffffu, inc, 31);
    if (lane == 0) sh.slot[33].a = as_bits(all);
  }
  cluster_sync();
  mass = lane < (int)cluster_size() ? as_double(ld_remote64(remote(&sh.slot[33].a, lane))) : 0.0;
  same = 0.0;
  join(mass, same, inc, lane);
  const double all = __shfl_sync(0xffffffffu, inc, 31), margin = 2.0 * sum_margin(walk, temperature, sl.limit) * inv;
  if (!(all > margin)) return false;
  // (warp 0 of the CTA that holds the target; the answer of the others is yes)
  auto settle_token = [&]() {
    double rest;
    if (pick(inc, u > 0.f ? fmin((double)u, 1.0) * all : 0.0, rest) != (int)cluster_rank()) return true;
    mass = lane < NT / 32 ? as_double(sh.warp_a[lane]) : 0.0;
    join(mass, same, inc, lane);
    const int w = pick(inc, rest, rest);
    mass = lane < kSub ? as_double(sh.seg[w * kSub + lane]) : 0.0;
    join(mass, same, inc, lane);
    const int k = pick(inc, rest, rest), a = min(sl.begin(w) + k * sl.sub, sl.end(w)), b = min(a + sl.sub, sl.end(w));
    for (int v0 = a; v0 < b; v0 += 32) {
      const int v = v0 + lane;
      float f[N];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = -INFINITY;
      if (v < b) sl.get(v, f);
      double m[N], total = 0.0;
      rest_of(f, sl.first + min(v, b - 1) * N, m);
#pragma unroll
      for (int i = 0; i < N; ++i) total += m[i];
      mass = total;
      join(mass, same, inc, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, inc > rest);
      if (hit) {
        const int who = __ffs(hit) - 1;
        const double before = __shfl_up_sync(0xffffffffu, inc, 1);
        bool sure = false;
        if (lane == who) sure = take(m, lane > 0 ? before : 0.0, rest, margin, sl.first + v * N, out);
        return __any_sync(0xffffffffu, sure) != 0;
      }
      rest = fmax(rest - __shfl_sync(0xffffffffu, inc, 31), 0.0);
    }
    return false;
  };
  if (warp == 0) {
    const bool sure = settle_token();
    if (lane == 0) sh.slot[35].a = sure ? 0 : 1;
  }
  cluster_sync();
  return cluster_max(&sh.slot[35].a) == 0;
}

// The sum of weight_walk in units of the fixed-point weights, -1 where it does not hold.
__device__ __forceinline__ double in_fixed_units(const Walk& w, const RowScale& s) {
  return w.far ? -1.0 : w.total * exp2(44.0 + (w.e - (6755399441055744.0 - s.magic) * 0.015625));
}

template <typename T, int NT, bool kShared>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ __align__(16) Shared sh;
  constexpr int N = Vec16<T>::N;
  const int r = blockIdx.x / cluster_size();
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const float t = __ldg(p.temperature + r), top_p = __ldg(p.top_p + r), u = __ldg(p.uniform + r);
  uint4* buf = slice_of<NT>(dyn, p);
  Slice<T, NT, kShared> sl = make_slice<T, NT, kShared>(row, p.vocab, p.slice, buf);
  const int begin = min((int)cluster_rank() * p.slice, p.vocab), end = min(begin + p.slice, p.vocab);
  float* probs = p.probs == nullptr ? nullptr : p.probs + (int64_t)r * p.probs_stride;
  const bool greedy = !(t > 0.f);
  Walk walk;
  int first = -1;
  if (greedy) first = greedy_walk(sl, buf, walk.top, sh);
  else walk = weight_walk(sl, buf, t, sh);
  if (greedy || walk.top == -INFINITY) {  // or a row without a token
    if (cluster_rank() == 0 && threadIdx.x == 0) p.tokens[r] = max(first, 0);
    if (probs != nullptr)
      for (int i = begin + threadIdx.x; i < end; i += NT) probs[i] = i == first ? 1.f : 0.f;
  } else {
    const float top = settle(sl, walk.top);
    Mass mass;
    mass.s = row_scale(top, sl.how == kQuartered ? t * 0.25f : t);
    mass.kept.value = -INFINITY;
    mass.kept.index = -1;
    double z;  // the kept weights' sum, in units of the top's
    if (!(top_p < 1.f) && !walk.far && draw_all(sl, walk, t, u, p.tokens + r, sh)) {
      z = in_fixed_units(walk, mass.s);
    } else {
      u64 mine;
      Near near = {reinterpret_cast<Entry*>(dyn), p.cap, 0, false};
      mass.kept = settled_border(sl, mass.s, top_p, top_p < 1.f ? in_fixed_units(walk, mass.s) : -1.0, near, sh, mine);
      mass.residual = false;
      mass.inv_z = 0.0; mass.minus = nullptr; mass.one_hot = -1;
      draw(sl, mass, near, u, !(top_p < 1.f), mine, 32, p.tokens + r, sh);
      z = (double)mass.kept.total;
    }
    if (probs != nullptr) {
      const float inv = (float)(top_weight(mass.s) / z);
      for (int v = threadIdx.x; v < sl.n_vec; v += NT) {
        float f[N];
        sl.get(v, f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int x = sl.first + v * N + i;
          if (x >= begin && x < end) probs[x] = mass.kept.holds(f[i], x) ? exp2f((f[i] - top) * mass.s.c32) * inv : 0.f;
        }
      }
    }
  }
  cluster_sync();  // the others may still read this CTA's slots
}

__device__ __forceinline__ int owner_of(const int32_t* __restrict__ indptr, int batch, int row) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(indptr + mid) <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// Does the draft x of a row pass, u q(x) < p(x)? The answer needs p(x) only to one side of u q(x): sums in fp32 from the first
// walk decide unless they come too close, or the nucleus' exact mass is needed (Z lies between top_p and 1 times the whole sum).
// Relative error of the sums: 2^-22 of ex2.approx, 2^-24 of an exponent below 2^14 (kept to 80 above the first entries, what lies far
// below does not count), 2^-24 of c for the same, 2^-24 for each of 128 additions: below 5e-5 up to exponents of 300; larger ones are
// left to the exact way. 1: yes, 0: no, -1: not known. Slots 0 and 1.
template <typename T, int NT>
__device__ int quick_walk(const Slice<T, NT, false>& sl, float temperature, float top_p, int x, float lx, double uq, QuickShared& sh) {
  constexpr int N = Vec16<T>::N;
  constexpr double kGuard = 1e-4;
  constexpr float kOctaves = 80.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float t = fminf(fmaxf(temperature, 1e-30f), 1e36f), c32 = 1.442695041f / t;
  const bool cut = top_p < 1.f;
  float m0 = -INFINITY, shift = 0.f, best = -INFINITY, all = 0.f, above = 0.f;
  const float below = lx == 0.f ? -1.4e-45f : __uint_as_float(__float_as_uint(lx) + (lx > 0.f ? -1 : 1));
  double sum_all = 0.0, sum_above = 0.0;
  int turn = 0;
  first_walk(sl, nullptr, [&](const float (&f)[N], int i0, int) {
    float m = largest(f);
    best = fmaxf(best, m);
    if (m0 == -INFINITY) {  // warp-uniform
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      m0 = m;
      shift = -m0 * c32;
    }
    if (m0 > -INFINITY) {
      // Entries of lower index rank ahead of x among equals: they are compared with the number just below lx.
      const float bar = i0 < x ? below : lx;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float w = ex2(fmaf(f[i], c32, shift));  // (NaN makes the sums NaN: not known)
        all += w;
        if (cut && f[i] > bar) above += w;
      }
      if (cut && i0 <= x && x < i0 + N) {  // the vector of x itself: what ranks behind it was counted
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i0 + i >= x && f[i] == lx) above -= i0 < x ? ex2(fmaf(f[i], c32, shift)) : 0.f;
      }
    }
    if (++turn == 16) {
      sum_all += (double)all;
      sum_above += (double)above;
      all = above = 0.f;
      turn = 0;
    }
  });
  sum_all += (double)all;
  sum_above += (double)above;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum_all += __shfl_xor_sync(0xffffffffu, sum_all, o);
    sum_above += __shfl_xor_sync(0xffffffffu, sum_above, o);
    best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  }
  const double c = 1.4426950408889634 / (double)t;
  bool far = best > -INFINITY && !((best - m0) * c32 < kOctaves && fabsf(shift) < 300.f);
  double e = m0 > -INFINITY && !far ? -(double)shift : -INFINITY;  // (shift as rounded: one factor for all)
  if (lane == 0) {
    sh.warp_a[warp] = as_bits(sum_all);
    sh.warp_b[warp] = as_bits(e);
    sh.warp_c[warp] = (u64)__float_as_uint(best) | (far ? 1ull << 32 : 0);
    sh.warp_d[warp] = as_bits(sum_above);
  }
  __syncthreads();
  double inc, own;
  if (warp == 0) {
    const bool in = lane < NT / 32;
    sum_all = in ? as_double(sh.warp_a[lane]) : 0.0;
    sum_above = in ? as_double(sh.warp_d[lane]) : 0.0;
    own = e = in ? as_double(sh.warp_b[lane]) : -INFINITY;
    best = in ? __uint_as_float((uint32_t)sh.warp_c[lane]) : -INFINITY;
    far = __any_sync(0xffffffffu, in && (sh.warp_c[lane] >> 32) != 0);
    join<true>(sum_all, e, inc, lane);
    const double whole = __shfl_sync(0xffffffffu, inc, 31);
    double g = own;
    join<true>(sum_above, g, inc, lane);
    const double ahead = __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) {
      sh.slot[0].a = as_bits(whole);
      sh.slot[0].b = as_bits(e);
      sh.slot[0].c = (u64)__float_as_uint(best) | (far ? 1ull << 32 : 0);
      sh.slot[1].a = as_bits(ahead);
    }
  }
  cluster_sync();
  const bool in = lane < (int)cluster_size();
  sum_all = in ? as_double(ld_remote64(remote(&sh.slot[0].a, lane))) : 0.0;
  own = e = in ? as_double(ld_remote64(remote(&sh.slot[0].b, lane))) : -INFINITY;
  const u64 z = in ? ld_remote64(remote(&sh.slot[0].c, lane)) : (u64)__float_as_uint(-INFINITY);
  sum_above = in ? as_double(ld_remote64(remote(&sh.slot[1].a, lane))) : 0.0;
  join<true>(sum_all, e, inc, lane);
  const double total = __shfl_sync(0xffffffffu, inc, 31);
  double g = own;
  join<true>(sum_above, g, inc, lane);
  const double ahead = __shfl_sync(0xffffffffu, inc, 31);
  best = __uint_as_float((uint32_t)z);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (__any_sync(0xffffffffu, (z >> 32) != 0) || best == INFINITY || best < -1e38f) return -1;
  if (((double)best - (double)lx) * c > 44.0) return -1;  // may be below what can be drawn: its fixed-point weight says
  const double wx = exp2(fmax((double)lx * c - e, -2000.0));
  double least = total, most = total;  // bounds of Z
  if (cut) {
    least = total * fmax((double)top_p, 0.0);
    if (ahead * (1 - kGuard) > least * (1 + kGuard)) return 0;      // not in the nucleus
    if (!(ahead * (1 + kGuard) <= least * (1 - kGuard))) return -1;
    most = fmin(total, least + wx);  // the border's weight is at most that of a kept token
  }
  if (uq * most * (1 + kGuard) < wx) return 1;
  if (uq * least * (1 - kGuard) >= wx) return 0;
  return -1;
}

// One cluster per row that has a draft behind it: is the draft accepted? Reads its row once and keeps nothing of it.
enum : uint8_t { kRejected = 0, kAccepted = 1, kUnknown = 2 };
constexpr int kQuickThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kQuickThreads, 4) verify_rows_kernel(const SampleParams p) {
  __shared__ QuickShared sh;
  const int r = blockIdx.x / cluster_size();
  const int req = owner_of(p.indptr, p.batch, r);
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (r < begin || r + 1 >= end || end > p.nnz) {  // a last row, or behind the last request (the whole cluster)
    // With an indptr that is not monotone the draw kernel may take it for another request's: nothing there is left undefined.
    if (cluster_rank() == 0 && threadIdx.x == 0) p.ok[r] = kRejected;
    return;
  }
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const int x = __ldg(p.draft + r + 1);
  const float t = __ldg(p.temperature + req), top_p = __ldg(p.top_p + req);
  const bool token = x >= 0 && x < p.vocab;
  const float lx = token ? to_f32(row[x]) : -INFINITY;
  const double q = p.draft_probs == nullptr || !token ? 1.0 : (double)__ldg(p.draft_probs + (int64_t)r * p.draft_stride + x);
  const double uq = (double)__ldg(p.uniform + r) * q;
  int ok = 0;
  if (lx > -INFINITY) {  // a token
    const Slice<T, kQuickThreads, false> sl = make_slice<T, kQuickThreads, false>(row, p.vocab, p.slice, nullptr);
    float top;
    if (!(t > 0.f)) ok = greedy_walk(sl, nullptr, top, sh) == x && uq < 1.0;
    else ok = quick_walk(sl, t, top_p, x, lx, uq, sh);
  }
  if (cluster_rank() == 0 && threadIdx.x == 0) p.ok[r] = ok < 0 ? kUnknown : ok ? kAccepted : kRejected;
  cluster_sync();
}

// One cluster per request: the accepted prefix (drafts that the sums of the rows kernel did not decide are tested exactly), then a
// draw from the residual of the first rejected row or from the last row.
template <typename T, int NT, bool kShared>
__global__ void __launch_bounds__(NT, 1024 / NT) verify_draw_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ __align__(16) Shared sh;
  const int req = blockIdx.x / cluster_size();
  const bool lead = cluster_rank() == 0 && threadIdx.x == 0;
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (begin < 0 || end <= begin || end > p.nnz) {
    if (lead) {
      if (begin != end) record_status(p.status, ST_BAD_REQUEST);
      p.accepted[req] = 0;
      p.tokens[req] = -1;
    }
    return;
  }
  const float t = __ldg(p.temperature + req), top_p = __ldg(p.top_p + req), u = __ldg(p.uniform + end - 1);
  const bool greedy = !(t > 0.f), cut = top_p < 1.f;
  uint4* buf = slice_of<NT>(dyn, p);
  for (int r = begin;; ++r) {
    const uint8_t said = r + 1 < end ? p.ok[r] : kRejected;
    if (said == kAccepted) continue;
    const bool last = r + 1 == end;
    const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
    const float* q_row = p.draft_probs == nullptr ? nullptr : p.draft_probs + (int64_t)r * p.draft_stride;
    const int x = last ? -1 : __ldg(p.draft + r + 1);
    Slice<T, NT, kShared> sl = make_slice<T, NT, kShared>(row, p.vocab, p.slice, buf);
    Walk walk;
    int first = -1;
    if (greedy) first = greedy_walk(sl, buf, walk.top, sh);
    else walk = weight_walk(sl, buf, t, sh);
    Mass mass;
    u64 mine = 0;
    Near near = {reinterpret_cast<Entry*>(dyn), p.cap, 0, false};
    const bool none = walk.top == -INFINITY;
    bool done = greedy || none;
    if (done) {
      if (lead) p.tokens[req] = max(first, 0);
    } else {
      const float top = settle(sl, walk.top);
      mass.s = row_scale(top, sl.how == kQuartered ? t * 0.25f : t);
      // Sums in double decide where they are far enough from a border, else the row goes the exact way.
      bool plain = !cut && !walk.far;
      const float l = said == kUnknown ? rewritten(to_f32(row[x]), sl.how) : 0.f;
      const double uq = said == kUnknown ? (double)__ldg(p.uniform + r) * (q_row == nullptr ? 1.0 : (double)__ldg(q_row + x)) : 0.0;
      if (plain && said == kUnknown) {
        const double w = weight(l, mass.s) * top_units(walk, t), bar = uq * walk.total;
        plain = fabs(w - bar) > sum_margin(walk, t, p.vocab);
        if (plain && bar < w) {
          cluster_sync();  // the others may still read this CTA's slots
          continue;
        }
      }
      if (plain) done = last ? draw_all(sl, walk, t, u, p.tokens + req, sh) : draw_rest(sl, walk, t, q_row, q_row == nullptr ? x : -1, u, p.tokens + req, sh);
      if (!done) {
        mass.kept = settled_border(sl, mass.s, top_p, cut ? in_fixed_units(walk, mass.s) : -1.0, near, sh, mine);
        if (said == kUnknown && !plain) {
          const u64 w = mass.kept.holds(l, x) ? raw_weight(l, mass.s, sh.table) - kRaw : 0;
          if (uq < (double)w / (double)mass.kept.total) {
            cluster_sync();
            continue;
          }
        }
        mass.inv_z = 1.0 / (double)mass.kept.total;
        mass.residual = !last;
        mass.minus = last ? nullptr : q_row;
        mass.one_hot = q_row == nullptr ? x : -1;
        if (!draw(sl, mass, near, u, last && !cut, mine, 31, p.tokens + req, sh) && mass.residual) {  // nothing is left above the draft's
          mass.residual = false;
          draw(sl, mass, near, u, false, 0, 34, p.tokens + req, sh);
        }
      }
    }
    if (lead) p.accepted[req] = r - begin;
    break;
  }
  cluster_sync();
}

// ---- host --------------------------------------------------------------------------------------------
constexpr size_t kMostSmem = 96 * 1024;  // of pick_shape: a slice of 72 KB and its alignment, 16 KB of lists
struct Shape {
  int ctas, slice, cap;
  bool shared;  // rows in shared memory, 512 threads; else in L2, 256 threads
  size_t smem;
};
// Few rows: as many CTAs (up to 8) per row as two per SM have room for, the row in shared memory. Many rows: CTAs of 256
// threads, four per SM, later walks from L2; up to 8 CTAs per row while there are not more than about four rounds of them.
// (128 rows of 128,256: 8 CTAs from L2 and 4 from shared memory the same within 5 %, 1 from L2 three times as long; 1024 rows: 1 or 2
// from L2 the same, 4 from shared memory twice as long, since the CTAs of a cluster wait for one another at every exchange.)
Shape pick_shape(int rows, int vocab, int es) {
  Shape s;
  s.ctas = 1;
  while (s.ctas < kMaxCtas && (int64_t)rows * s.ctas * 2 <= 296 && vocab / (s.ctas * 2) >= 2048) s.ctas *= 2;
  s.shared = (int64_t)rows * s.ctas <= 296 && (int64_t)(vocab / s.ctas + 64) * es <= 72 * 1024;
  if (!s.shared) {
    s.ctas = 1;
    while (s.ctas < kMaxCtas && (int64_t)rows * s.ctas * 2 <= 2400 && vocab / (s.ctas * 2) >= 2048) s.ctas *= 2;
  }
  s.slice = ((vocab + s.ctas - 1) / s.ctas + 63) & ~63;
  s.cap = s.shared ? 64 : 176;
  s.smem = (s.shared ? (size_t)s.slice * es + 32 : 0) + (size_t)s.cap * (s.shared ? 16 : 8) * sizeof(Entry);
  return s;
}

template <auto kKernel, int NT>
cudaError_t launch(int rows, const Shape& s, const SampleParams& p, cudaStream_t st) {
  if (s.smem > 0) {
    const cudaError_t e = allow_smem<kKernel>(kMostSmem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * s.ctas);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = s.ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kKernel, p);
}

}  // namespace
}  // namespace dsv

extern "C" {

int dsv_sample_top_p(const void* logits, int64_t row_stride, int rows, int vocab, const float* temperature,
                     const float* top_p, const float* uniform, int32_t* tokens, float* probs, int64_t probs_stride,
                     int dtype, void* stream) {
  using namespace dsv;
  DSV_REQUIRE(dtype_ok(dtype), "sample_top_p: unknown dtype %d", dtype);
  DSV_REQUIRE(rows >= 0 && vocab > 0, "sample_top_p: bad shape");
  if (vocab > kMaxVocab) return fail(DSV_E_UNSUPPORTED, "sample_top_p: vocabulary %d above %d", vocab, kMaxVocab);
  if (rows == 0) return DSV_OK;
  DSV_REQUIRE(logits && temperature && top_p && uniform && tokens, "sample_top_p: null pointer argument");
  DSV_REQUIRE(row_stride >= vocab && (probs == nullptr || probs_stride >= vocab), "sample_top_p: row stride smaller than a row");
  DSV_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (elem_size(dtype) - 1)) == 0, "sample_top_p: misaligned logits");
  // a warp may write probabilities while another still looks for the token
  DSV_REQUIRE(logits != (const void*)probs, "sample_top_p: probs must not be logits");
  SampleParams p = {};
  p.logits = logits; p.row_stride = row_stride; p.vocab = vocab; p.temperature = temperature; p.top_p = top_p;
  p.uniform = uniform; p.tokens = tokens; p.probs = probs; p.probs_stride = probs_stride;
  const Shape shape = pick_shape(rows, vocab, elem_size(dtype));
  p.slice = shape.slice; p.cap = shape.cap;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    return shape.shared ? launch<sample_kernel<T, 512, true>, 512>(rows, shape, p, st)
                        : launch<sample_kernel<T, 256, false>, 256>(rows, shape, p, st);
  };
  const cudaError_t e = dtype == DSV_F32 ? go(float{}) : dtype == DSV_F16 ? go(__half{}) : go(__nv_bfloat16{});
  if (e != cudaSuccess) return fail(DSV_E_CUDA, "sample_top_p launch failed: %s", cudaGetErrorString(e));
  return DSV_OK;
}

int dsv_verify_draft(const void* logits, int64_t row_stride, int nnz, int vocab, const int32_t* tokens,
                     const int32_t* indptr, int batch, const float* uniform, const float* temperature,
                     const float* top_p, const float* draft_probs, int64_t draft_stride, uint8_t* workspace,
                     int64_t workspace_bytes, int32_t* accepted, int32_t* next_tokens, int dtype, void* stream) {
  using namespace dsv;
  DSV_REQUIRE(dtype_ok(dtype), "verify_draft: unknown dtype %d", dtype);
  DSV_REQUIRE(nnz >= 0 && batch >= 0 && vocab > 0, "verify_draft: bad shape");
  if (vocab > kMaxVocab) return fail(DSV_E_UNSUPPORTED, "verify_draft: vocabulary %d above %d", vocab, kMaxVocab);
  if (batch == 0) return DSV_OK;
  DSV_REQUIRE(indptr && accepted && next_tokens, "verify_draft: null pointer argument");
  DSV_REQUIRE(nnz == 0 || (logits && tokens && uniform && temperature && top_p && workspace), "verify_draft: null pointer argument");
  DSV_REQUIRE(row_stride >= vocab && (draft_probs == nullptr || draft_stride >= vocab), "verify_draft: row stride smaller than a row");
  DSV_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (elem_size(dtype) - 1)) == 0, "verify_draft: misaligned logits");
  if (workspace_bytes < nnz)
    return fail(DSV_E_WORKSPACE, "verify_draft: workspace needs %d bytes, got %lld", nnz, (long long)workspace_bytes);
  SampleParams p = {};
  p.logits = logits; p.row_stride = row_stride; p.vocab = vocab; p.temperature = temperature; p.top_p = top_p;
  p.uniform = uniform; p.tokens = next_tokens; p.indptr = indptr; p.draft = tokens; p.draft_probs = draft_probs;
  p.draft_stride = draft_stride; p.ok = workspace; p.accepted = accepted; p.batch = batch; p.nnz = nnz;
  p.status = device_status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if (nnz > 0) {
      // one round of CTAs, four per SM, where there are enough rows for it
      Shape shape = {};
      shape.ctas = 1;
      while (shape.ctas < kMaxCtas && (int64_t)nnz * shape.ctas < 592 && vocab / (shape.ctas * 2) >= 2048) shape.ctas *= 2;
      p.slice = ((vocab + shape.ctas - 1) / shape.ctas + 63) & ~63;
      const cudaError_t er = launch<verify_rows_kernel<T>, kQuickThreads>(nnz, shape, p, st);
      if (er != cudaSuccess) return er;
    }
    const Shape shape = pick_shape(batch, vocab, elem_size(dtype));
    p.slice = shape.slice; p.cap = shape.cap;
    return shape.shared ? launch<verify_draw_kernel<T, 512, true>, 512>(batch, shape, p, st)
                      : launch<verify_draw_kernel<T, 256, false>, 256>(batch, shape, p, st);
  };
  const cudaError_t e = dtype == DSV_F32 ? go(float{}) : dtype == DSV_F16 ? go(__half{}) : go(__nv_bfloat16{});
  if (e != cudaSuccess) return fail(DSV_E_CUDA, "verify_draft launch failed: %s", cudaGetErrorString(e));
  return DSV_OK;
}

}  // extern "C"
