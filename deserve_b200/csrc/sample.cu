// Temperature / top-p sampling and the verification of drafted tokens.
//
// A row of logits gives weights w_v = exp((l_v - max l) / T). Tokens are ranked by value, lower index
// first among equals; token v is kept when the weights ranked before it sum to at most top_p times the
// whole sum. With Z the sum of the kept weights, p_v = w_v / Z for kept v and 0 otherwise. A draw with
// u in [0, 1) takes the first v in INDEX order whose running sum of p exceeds u times the whole.
//
// Which token a draw takes depends on ~1e5 borders per row: sums in fp32 would move some of them and the
// result would depend on how a row is cut among threads. Weights are therefore 64-bit fixed point
// (units of 2^-44 of the largest weight, evaluated in double): integer sums are exact and associative,
// so every cut of the row, and every order of the atomics, gives the same token. 2^18 entries of
// weight one still fit 63 bits, hence the bound on the vocabulary.
//
// A cluster of 1 to 8 CTAs owns a row and keeps it in shared memory (one pass over HBM): the largest
// logit, the weight sums, the top-p border and the draw each walk it again there. Sums and histograms
// of the CTAs meet through distributed shared memory.
//
// The top-p border is found without sorting: a histogram of weight over 2048 bins of (max - l) / T gives
// the bin of the border; the members of that bin are then split 2048 ways again by (value, index) until
// one token is left (two or three times).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dsv {
namespace {

constexpr int kBins = 2048;
constexpr int kMaxCtas = 8;   // of a cluster (the portable limit)
constexpr int kMaxWarps = 16;
constexpr int kList = 256;    // members of the border's bin that are ranked directly
constexpr int kMaxVocab = 1 << 18, kIndexBits = 18;
constexpr double kOne = 17592186044416.0;          // 2^44: the fixed-point weight of the largest logit
constexpr double kProbOne = 1152921504606846976.0;  // 2^60: fixed-point probabilities of the residual
constexpr float kWindow = 8.f;                      // nats below the top that the first histogram covers
constexpr int kTable = 64;
typedef unsigned long long u64;
constexpr u64 kRaw = 0x4330000000000000ull;  // 2^52 as a double: integers sit behind it

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
  int* status;
};

// What the CTAs of a cluster show one another. Every exchange uses a slot of its own, so one cluster
// barrier per exchange is enough.
struct Slot {
  u64 a, b;
};
struct Shared {
  uint32_t hist_lo[kBins], hist_hi[kBins];
  double table[kTable];  // 2^(j / 64 + 44)
  Slot slot[32];
  u64 warp_a[kMaxWarps], warp_b[kMaxWarps];
  u64 seg[kMaxWarps];    // mass of the warps' segments
  u64 list[kList];       // this CTA's members of the border's bin
  u64 all_key[kList], all_w[kList];
  int n_list;
  u64 border, kept;
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
  double one;    // the fixed-point weight of the top: 2^44 2^((top c - K) / 64)
};
__device__ __forceinline__ RowScale row_scale(float top, float temperature) {
  RowScale s;
  s.top = top;
  s.t = fminf(temperature, 1e36f);  // (so that the cutoff below stays finite)
  const double inv = 1.0 / (double)s.t;
  // A temperature so small that one unit in the last place of the top already gives weight 0 gives the same weights
  // as 2^37 / |top|, which keeps the exponents in range.
  s.c = fmin(92.332482616893657 * inv, 137438953472.0 / fabs((double)top));
  s.c32 = (float)fmin(1.4426950408889634 * inv, 3e38);
  const float ulp = __uint_as_float(__float_as_uint(fabsf(top)) + 1u) - fabsf(top);
  s.cutoff = top - fmaxf(64.f * s.t, 2.f * ulp);
  const double k = rint((double)top * s.c);
  s.magic = 6755399441055744.0 - k;
  s.one = kOne * exp2(fma((double)top, s.c, -k) * 0.015625);
  return s;
}
// Fixed-point weight behind kRaw (subtract it; sums may subtract it once per entry). With l c = N + r, |r| <= 1/2:
// 2^((N - K) / 64) from a table of 2^(j / 64) and an exponent, e^(r ln 2 / 64) to the fourth power (its argument is
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
  const double scaled = __hiloint2double(__double2hiint(t) + ((n >> 6) << 20), __double2loint(t));
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

// A CTA's slice of a row in shared memory: 16-byte vectors as in global memory, what lies before and behind
// the slice filled with -inf (no token). Vector v holds the entries first + v * N and on.
template <typename T, int NT>
struct Slice {
  static constexpr int N = Vec16<T>::N;
  uint4* v;
  int n_vec, first;
  int seg;  // vectors of a warp's contiguous segment
  __device__ __forceinline__ void get(int i, float (&f)[N]) const { Vec16<T>::unpack(v[i], f); }
  __device__ __forceinline__ int begin(int warp) const { return min(warp * seg, n_vec); }
  __device__ __forceinline__ int end(int warp) const { return min(warp * seg + seg, n_vec); }
};

// Load the slice; its largest entry that is a number (NaN ignored).
template <typename T, int NT>
__device__ __forceinline__ Slice<T, NT> load_slice(const T* row, int vocab, int slice, uint4* buf, float& best) {
  constexpr int N = Vec16<T>::N, W = NT / 32;
  const int begin = min((int)cluster_rank() * slice, vocab), end = min(begin + slice, vocab);
  const T* src = row + begin;
  const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T)), n = end - begin;
  Slice<T, NT> sl;
  sl.v = buf;
  sl.first = begin - lead;
  sl.n_vec = n > 0 ? (lead + n + N - 1) / N : 0;
  sl.seg = ((sl.n_vec + W * 32 - 1) / (W * 32)) * 32;
  best = -INFINITY;
  const uint4* g = reinterpret_cast<const uint4*>(src - lead);
  auto take = [&](int v, const uint4& u) {
    buf[v] = u;
    float f[N];
    Vec16<T>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < N; ++i) best = fmaxf(best, f[i]);
  };
  auto ragged = [&](int e) {  // a vector that reaches over an end of the slice
    __align__(16) T tmp[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = e * N + i - lead;
      tmp[i] = k >= 0 && k < n ? src[k] : from_f32<T>(-INFINITY);
    }
    take(e, *reinterpret_cast<const uint4*>(tmp));
  };
  const int v0 = lead > 0 ? 1 : 0, v1 = n > 0 ? (lead + n) / N : 0;  // whole vectors
  int v = v0 + threadIdx.x;
  for (; v + 7 * NT < v1; v += 8 * NT) {
    uint4 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = ld_stream16(g + v + k * NT);
#pragma unroll
    for (int k = 0; k < 8; ++k) take(v + k * NT, u[k]);
  }
  for (; v + 3 * NT < v1; v += 4 * NT) {
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = ld_stream16(g + v + k * NT);
#pragma unroll
    for (int k = 0; k < 4; ++k) take(v + k * NT, u[k]);
  }
  for (; v < v1; v += NT) take(v, ld_stream16(g + v));
  if (threadIdx.x == 0 && lead > 0 && n > 0) ragged(0);
  if (threadIdx.x == 1 && v1 < sl.n_vec && (sl.n_vec > 1 || lead == 0)) ragged(sl.n_vec - 1);
  return sl;
}

// The cluster's largest logit, -inf when it holds nothing but NaN and -inf. Rows at the ends of the number range are
// rewritten in place, without changing an order or a weight: +inf entries become 0 and all others -inf; a row below
// -1e38 is scaled by 1/4 (with its temperature). Also readies the table of the exponential.
enum : int { kAsIs = 0, kInfinite = 1, kQuartered = 2 };
__device__ __forceinline__ float rewritten(float l, int how) {
  return how == kInfinite ? (l == INFINITY ? 0.f : -INFINITY) : how == kQuartered ? l * 0.25f : l;
}
template <typename T, int NT>
__device__ float row_top(const Slice<T, NT>& sl, float best, int& how, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sh.warp_a[warp] = __float_as_uint(best);
  if (threadIdx.x < kTable) sh.table[threadIdx.x] = exp2((double)threadIdx.x / kTable) * kOne;
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  if (warp == 0) {
    best = __uint_as_float((uint32_t)sh.warp_a[min(lane, NT / 32 - 1)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.slot[0].a = __float_as_uint(best);
  }
  cluster_sync();
  float top = -INFINITY;
  for (int r = 0; r < (int)cluster_size(); ++r) top = fmaxf(top, __uint_as_float((uint32_t)ld_remote64(remote(&sh.slot[0].a, r))));
  how = top == INFINITY ? kInfinite : top < -1e38f && top > -INFINITY ? kQuartered : kAsIs;
  if (how != kAsIs) {
    for (int v = threadIdx.x; v < sl.n_vec; v += NT) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = rewritten(f[i], how);
      sl.v[v] = Vec16<T>::pack(f);
    }
    __syncthreads();
    top = rewritten(top, how);
  }
  return top;
}
// Lowest index of the largest logit (of a row that has one), through slot 1.
template <typename T, int NT>
__device__ int row_first(const Slice<T, NT>& sl, float top, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  int at = 0x7fffffff;
  for (int v = threadIdx.x; v < sl.n_vec; v += NT) {
    float f[N];
    sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f[i] == top) at = min(at, sl.first + v * N + i);
  }
  at = __reduce_min_sync(0xffffffffu, at);
  if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = (u64)at;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 m = sh.warp_a[0];
    for (int w = 1; w < NT / 32; ++w) m = min(m, sh.warp_a[w]);
    sh.slot[1].a = m;
  }
  cluster_sync();
  u64 m = ~0ull;
  for (int r = 0; r < (int)cluster_size(); ++r) m = min(m, ld_remote64(remote(&sh.slot[1].a, r)));
  return (int)m;
}

// Sums over the cluster of two integers per warp (in its lane 0), through slot `s`: the wholes, and what the CTAs before this
// one have of the first.
template <int NT>
__device__ Slot cluster_total(u64 a, u64 b, Shared& sh, int s, u64& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) { sh.warp_a[warp] = a; sh.warp_b[warp] = b; }
  __syncthreads();
  if (warp == 0) {
    const u64 va = warp_sum(lane < NT / 32 ? sh.warp_a[lane] : 0), vb = warp_sum(lane < NT / 32 ? sh.warp_b[lane] : 0);
    if (lane == 0) { sh.slot[s].a = va; sh.slot[s].b = vb; }
  }
  cluster_sync();
  const int c = cluster_size(), rank = cluster_rank();
  Slot all = {0, 0};
  before = 0;
  for (int r = 0; r < c; ++r) {
    const u64 v = ld_remote64(remote(&sh.slot[s].a, r));
    if (r < rank) before += v;
    all.a += v;
    all.b += ld_remote64(remote(&sh.slot[s].b, r));
  }
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
// mass; -1: none, `before` is the whole. `extra` (per warp, lane 0) is summed over the cluster along with it;
// limit_of(histogram's whole, extra's whole) gives the limit. Each CTA sums its share of the bins over the cluster. Slots
// s to s + 2.
template <int NT, typename F>
__device__ int hist_find(Shared& sh, int s, u64 extra, F limit_of, u64& limit, u64& before, u64& mass) {
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
      u64 lo = 0, hi = 0;
      for (int r = 0; r < c; ++r) {
        lo += ld_remote32(remote(&sh.hist_lo[b], r));
        hi += ld_remote32(remote(&sh.hist_hi[b], r));
      }
      v[i] = (hi << 32) + lo;
    }
    mine += v[i];
  }
  const u64 inc = warp_scan(mine, lane), warp_mass = __shfl_sync(0xffffffffu, inc, 31);
  if (threadIdx.x == 0) sh.slot[s + 1].a = ~0ull;
  u64 cta_before, base = 0;
  const Slot all = cluster_total<NT>(warp_mass, extra, sh, s, cta_before);
  limit = limit_of(all.a, all.b);
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
  int bin = -1;
  for (int r = 0; r < c; ++r) {
    const u64 x = ld_remote64(remote(&sh.slot[s + 1].a, r));
    if (x != ~0ull) {
      bin = (int)x;
      before = ld_remote64(remote(&sh.slot[s + 1].b, r));
      mass = ld_remote64(remote(&sh.slot[s + 2].a, r));
    }
  }
  return bin;
}

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

// Top-p border of the row. Without a cut the masses of the warps' segments are left in sh.seg. Slots 2 to 26.
template <typename T, int NT>
__device__ Kept find_kept(const Slice<T, NT>& sl, const RowScale& s, float top_p, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Kept k;
  k.value = -INFINITY;
  k.index = -1;
  const int w0 = sl.begin(warp), w1 = sl.end(warp);
  if (!(top_p < 1.f)) {  // NaN: no cut
    u64 sum = 0, before;
    for (int v = w0 + lane; v < w1; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += raw_weight(f[i], s, sh.table);
      sum -= N * kRaw;
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.seg[warp] = sum;
    k.total = cluster_total<NT>(sum, 0, sh, 2, before).a;
    return k;
  }
  // Histogram of the tokens within kWindow nats of the top; the others' weight is one sum. (The tail of a vocabulary is
  // most of its entries and seldom holds the border: their atomics would cost more than all the rest.)
  hist_clear<NT>(sh);
  __syncthreads();
  const float light = s.top - kWindow * s.t, near_scale = (float)kBins / (kWindow * s.t);
  auto near_bin = [&](float l) { return min((int)((s.top - l) * near_scale), kBins - 1); };
  u64 tail = 0;
  for (int v = w0 + lane; v < w1; v += 32) {
    float f[N];
    sl.get(v, f);
    u64 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = raw_weight(f[i], s, sh.table) - kRaw;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (f[i] >= light) hist_add(sh, near_bin(f[i]), w[i]);
      else tail += w[i];
    }
  }
  u64 limit, before, mass, lo = ~0ull, hi = 0;
  const double share = (double)fmaxf(top_p, 0.f);
  int bin = hist_find<NT>(sh, 3, warp_sum(tail), [&](u64 a, u64 b) { k.total = a + b; return (u64)(share * (double)(a + b)); }, limit,
                          before, mass);
  limit -= before;
  u64 kept = before;
  // The border lies in the tail: a histogram of it, over the 64 nats that hold any weight.
  const bool far = bin < 0;
  const float far_scale = (float)kBins / (56.f * s.t);
  auto far_bin = [&](float l) { return min((int)(fmaxf(light - l, 0.f) * far_scale), kBins - 1); };
  if (far) {
    hist_clear<NT>(sh);  // (every CTA has read it: the cluster barrier in cluster_total)
    __syncthreads();
    for (int v = w0 + lane; v < w1; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u64 w = raw_weight(f[i], s, sh.table) - kRaw;
        if (w && !(f[i] >= light)) hist_add(sh, far_bin(f[i]), w);
      }
    }
    u64 same;
    bin = hist_find<NT>(sh, 6, 0, [&](u64, u64) { return limit; }, same, before, mass);
    if (bin < 0) return k;  // cannot happen with top_p < 1: the whole exceeds the limit
    limit -= before;
    kept += before;
  }
  // Members of the border's bin: listed, and the range of their rank keys.
  for (int v = w0 + lane; v < w1; v += 32) {
    float f[N];
    sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float l = f[i];
      if (!(l > s.cutoff) || (l >= light) == far || (far ? far_bin(l) : near_bin(l)) != bin) continue;
      const u64 key = rank_key<T>(l, sl.first + v * N + i);
      lo = min(lo, key);
      hi = max(hi, key);
      const int at = atomicAdd(&sh.n_list, 1);
      if (at < kList) sh.list[at] = key;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lo = min(lo, shfl_xor64(lo, o)); hi = max(hi, shfl_xor64(hi, o)); }
  if (lane == 0) { sh.warp_a[warp] = lo; sh.warp_b[warp] = hi; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NT / 32; ++w) { lo = min(lo, sh.warp_a[w]); hi = max(hi, sh.warp_b[w]); }
    sh.slot[9].a = lo;
    sh.slot[9].b = hi;
    sh.slot[10].a = (u64)sh.n_list;
  }
  cluster_sync();  // also: every CTA has read the histogram that is cleared next
  int members = 0;
  for (int r = 0; r < (int)cluster_size(); ++r) {
    lo = min(lo, ld_remote64(remote(&sh.slot[9].a, r)));
    hi = max(hi, ld_remote64(remote(&sh.slot[9].b, r)));
    members += (int)min(ld_remote64(remote(&sh.slot[10].a, r)), (u64)1 << 20);
  }
  if (members <= kList) {  // few: every CTA ranks all of them
    int base = 0;
    for (int r = 0; r < (int)cluster_size(); ++r) {
      const int n = (int)ld_remote64(remote(&sh.slot[10].a, r));
      for (int i = threadIdx.x; i < n; i += NT) {
        const u64 key = ld_remote64(remote(&sh.list[i], r));
        sh.all_key[base + i] = key;
        sh.all_w[base + i] = raw_weight(key_value<T>((uint32_t)(key >> kIndexBits)), s, sh.table) - kRaw;
      }
      base += n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < members; i += NT) {
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
    return k;
  }
  for (int s0 = 11;; s0 += 3) {  // 50 bits of rank key, 11 a round: five rounds at most
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
    hist_clear<NT>(sh);
    __syncthreads();
    for (int v = w0 + lane; v < w1; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!(f[i] > s.cutoff)) continue;
        const u64 key = rank_key<T>(f[i], sl.first + v * N + i);
        if (key >= lo && key <= hi) hist_add(sh, (int)((hi - key) >> shift), raw_weight(f[i], s, sh.table) - kRaw);
      }
    }
    u64 same;
    bin = hist_find<NT>(sh, s0, 0, [&](u64, u64) { return limit; }, same, before, mass);
    if (bin < 0) return k;  // cannot happen: the members' mass exceeds the limit
    limit -= before;
    kept += before;
    hi -= (u64)bin << shift;
    const u64 width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    if (shift == 0) {
      set_border<T>(k, hi);
      k.total = kept + mass;
      return k;
    }
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
  __device__ __forceinline__ u64 operator()(float l, int i, const Shared& sh) const {
    if (!kept.holds(l, i)) return 0;  // NaN and -inf are never kept
    u64 w = raw_weight(l, s, sh.table) - kRaw;
    if (residual && w) {
      const double q = minus != nullptr ? (double)__ldg(minus + i) : i == one_hot ? 1.0 : 0.0;
      const double r = (double)w * inv_z - q;
      w = r > 0.0 ? (u64)__double2ull_rn(r * kProbOne) : 0;
    }
    return w;
  }
};

// First index whose running sum of mass exceeds u * (whole sum). The CTA that holds it writes it to *out; false when
// there is no mass. `ready`: sh.seg holds the masses of the warps' segments already.
template <typename T, int NT>
__device__ bool draw(const Slice<T, NT>& sl, const Mass& mass, float u, bool ready, int slot, int32_t* out, Shared& sh) {
  constexpr int N = Vec16<T>::N, W = NT / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto sum_of = [&](int a, int b) {
    u64 sum = 0;
    for (int v = a + lane; v < b; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += mass(f[i], sl.first + v * N + i, sh);
    }
    return warp_sum(sum);
  };
  if (!ready) {
    const u64 sum = sum_of(sl.begin(warp), sl.end(warp));
    if (lane == 0) sh.seg[warp] = sum;
  }
  __syncthreads();
  u64 before;
  const u64 all = cluster_total<NT>(sh.seg[warp], 0, sh, slot, before).a;
  if (all == 0) return false;
  const double x = u > 0.f ? (double)u * (double)all : 0.0;  // NaN: 0
  u64 target = x < (double)all ? min((u64)x, all - 1) : all - 1;
  u64 mine = 0;
  for (int w = 0; w < W; ++w) mine += sh.seg[w];
  if (target < before || target - before >= mine) return true;  // another CTA's
  target -= before;
  int w = 0;
  while (w < W - 1 && target >= sh.seg[w]) target -= sh.seg[w++];
  // the warps share that segment
  const int begin = sl.begin(w), end = sl.end(w);
  const int sub = (end - begin + W - 1) / W;
  const int a = min(begin + warp * sub, end), b = min(a + sub, end);
  const u64 sum = sum_of(a, b);
  __syncthreads();
  if (lane == 0) sh.warp_b[warp] = sum;
  __syncthreads();
  w = 0;
  while (w < W - 1 && target >= sh.warp_b[w]) target -= sh.warp_b[w++];
  if (warp != w) return true;
  for (int v0 = a; v0 < b; v0 += 32) {
    const int v = v0 + lane;
    u64 m[N], total = 0;
    float f[N];
    if (v < b) sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = v < b ? mass(f[i], sl.first + v * N + i, sh) : 0;
      total += m[i];
    }
    const u64 inc = warp_scan(total, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        u64 run = inc - total;
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
  return true;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ __align__(16) Shared sh;
  constexpr int N = Vec16<T>::N;
  const int r = blockIdx.x / cluster_size();
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const float t = __ldg(p.temperature + r), top_p = __ldg(p.top_p + r), u = __ldg(p.uniform + r);
  float best;
  int how;
  const Slice<T, NT> sl = load_slice<T, NT>(row, p.vocab, p.slice, reinterpret_cast<uint4*>(dyn), best);
  const float top = row_top(sl, best, how, sh);
  const int begin = min((int)cluster_rank() * p.slice, p.vocab), end = min(begin + p.slice, p.vocab);
  float* probs = p.probs == nullptr ? nullptr : p.probs + (int64_t)r * p.probs_stride;
  if (!(t > 0.f) || top == -INFINITY) {  // greedy, or a row without a token
    const int first = top == -INFINITY ? -1 : row_first(sl, top, sh);
    if (cluster_rank() == 0 && threadIdx.x == 0) p.tokens[r] = max(first, 0);
    if (probs != nullptr)
      for (int i = begin + threadIdx.x; i < end; i += NT) probs[i] = i == first ? 1.f : 0.f;
  } else {
    Mass mass;
    mass.s = row_scale(top, how == kQuartered ? t * 0.25f : t);
    mass.kept = find_kept(sl, mass.s, top_p, sh);
    mass.residual = false;
    mass.inv_z = 0.0; mass.minus = nullptr; mass.one_hot = -1;
    draw(sl, mass, u, !(top_p < 1.f), 27, p.tokens + r, sh);
    if (probs != nullptr) {
      const float inv = (float)(mass.s.one / (double)mass.kept.total);
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

// Does the draft x of a row pass, u q(x) < p(x)? The answer needs p(x) only to one side of u q(x): sums in fp32 decide
// unless they come too close (1e-5 bounds their error: 2^-22 of ex2.approx, 2^-23 of the exponent's size, which the
// weights average to at most log2 of the vocabulary, 128 additions), or the nucleus' exact mass is needed: Z lies
// between top_p and 1 times the whole sum. 1: yes, 0: no, -1: not known.
template <typename T, int NT>
__device__ int quick_test(const Slice<T, NT>& sl, const RowScale& s, float top_p, int x, float lx, double wx, double uq, Shared& sh) {
  constexpr int N = Vec16<T>::N;
  constexpr double kFix = 1099511627776.0, kGuard = 4e-5;  // 2^40
  float all = 0.f, above = 0.f;
  const bool cut = top_p < 1.f;
  u64 fall = 0, fabove = 0;
  int n = 0;
  for (int v = threadIdx.x; v < sl.n_vec; v += NT) {
    float f[N];
    sl.get(v, f);
    const int i0 = sl.first + v * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = ex2((fmaxf(f[i], s.cutoff) - s.top) * s.c32);
      all += w;
      if (cut) above += f[i] > lx || (f[i] == lx && i0 + i < x) ? w : 0.f;
    }
    if (++n * N >= 128) {
      fall += (u64)(all * (float)kFix);
      fabove += (u64)(above * (float)kFix);
      all = above = 0.f;
      n = 0;
    }
  }
  fall = warp_sum(fall + (u64)(all * (float)kFix));
  fabove = warp_sum(fabove + (u64)(above * (float)kFix));
  u64 before;
  const Slot sum = cluster_total<NT>(fall, fabove, sh, 28, before);
  const double total = (double)sum.a / kFix, ahead = (double)sum.b / kFix;
  double least = total;  // of Z
  if (cut) {
    least = total * fmax((double)top_p, 0.0);
    if (ahead * (1 - kGuard) > least * (1 + kGuard)) return 0;      // not in the nucleus
    if (!(ahead * (1 + kGuard) <= least * (1 - kGuard))) return -1;  // (and its first token when top_p is 0)
  }
  if (uq * total * (1 + kGuard) < wx) return 1;
  if (uq * least * (1 - kGuard) >= wx) return 0;
  return -1;
}

// One cluster per row that has a draft behind it: is the draft accepted?
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) verify_rows_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ __align__(16) Shared sh;
  const int r = blockIdx.x / cluster_size();
  const int req = owner_of(p.indptr, p.batch, r);
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (r < begin || r + 1 >= end || end > p.nnz) return;  // a last row, or behind the last request (the whole cluster)
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const int x = __ldg(p.draft + r + 1);
  const float t = __ldg(p.temperature + req), top_p = __ldg(p.top_p + req);
  const bool token = x >= 0 && x < p.vocab;
  const float lx = token ? to_f32(row[x]) : -INFINITY;
  const double q = p.draft_probs == nullptr || !token ? 1.0 : (double)__ldg(p.draft_probs + (int64_t)r * p.draft_stride + x);
  const double uq = (double)__ldg(p.uniform + r) * q;
  float best;
  int how, ok = 0;
  const Slice<T, NT> sl = load_slice<T, NT>(row, p.vocab, p.slice, reinterpret_cast<uint4*>(dyn), best);
  const float top = row_top(sl, best, how, sh), l = rewritten(lx, how);
  if (l > -INFINITY) {  // a token (and so the row has a top)
    if (!(t > 0.f)) {
      ok = l == top && row_first(sl, top, sh) == x && uq < 1.0;
    } else {
      const RowScale s = row_scale(top, how == kQuartered ? t * 0.25f : t);
      const double wx = weight(l, s);
      ok = quick_test(sl, s, top_p, x, l, wx, uq, sh);
      if (ok < 0) {
        const Kept k = find_kept(sl, s, top_p, sh);
        ok = k.holds(l, x) && uq < wx * (s.one / (double)k.total);
      }
    }
  }
  if (cluster_rank() == 0 && threadIdx.x == 0) p.ok[r] = (uint8_t)ok;
  cluster_sync();
}

// One cluster per request: the accepted prefix, then a draw from the residual of the first rejected row or
// from the last row.
template <typename T, int NT>
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
  int r = begin;
  while (r + 1 < end && p.ok[r]) ++r;
  const bool rejected = r + 1 < end;
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const float t = __ldg(p.temperature + req), top_p = __ldg(p.top_p + req), u = __ldg(p.uniform + end - 1);
  float best;
  int how;
  const Slice<T, NT> sl = load_slice<T, NT>(row, p.vocab, p.slice, reinterpret_cast<uint4*>(dyn), best);
  const float top = row_top(sl, best, how, sh);
  if (lead) p.accepted[req] = r - begin;
  if (!(t > 0.f) || top == -INFINITY) {
    const int first = top == -INFINITY ? 0 : row_first(sl, top, sh);
    if (lead) p.tokens[req] = first;
  } else {
    Mass mass;
    mass.s = row_scale(top, how == kQuartered ? t * 0.25f : t);
    mass.kept = find_kept(sl, mass.s, top_p, sh);
    mass.inv_z = 1.0 / (double)mass.kept.total;
    mass.residual = rejected;
    mass.minus = rejected && p.draft_probs != nullptr ? p.draft_probs + (int64_t)r * p.draft_stride : nullptr;
    mass.one_hot = rejected ? __ldg(p.draft + r + 1) : -1;
    if (!draw(sl, mass, u, !rejected && !(top_p < 1.f), 29, p.tokens + req, sh)) {
      mass.residual = false;  // nothing left above the draft's distribution: the target's own
      draw(sl, mass, u, false, 30, p.tokens + req, sh);
    }
  }
  cluster_sync();
}

// ---- host --------------------------------------------------------------------------------------------
struct Shape {
  int ctas, slice;
  bool wide;  // 512 threads, else 256
  size_t smem;
};
// CTAs of a row: as few as keep a slice within 32 KB, four CTAs of 256 threads per SM, so that some load while others
// compute; where all rows fit the SMs at once anyway, more CTAs (up to 8, slices of 2048 entries at least) of 512 threads.
Shape pick_shape(int rows, int vocab, int es) {
  Shape s;
  s.ctas = 1;
  while (s.ctas < kMaxCtas && (int64_t)vocab * es > (int64_t)s.ctas * 32768) s.ctas *= 2;
  while (s.ctas < kMaxCtas && (int64_t)rows * s.ctas * 2 <= 148 && vocab / (s.ctas * 2) >= 2048) s.ctas *= 2;
  s.wide = (int64_t)rows * s.ctas <= 148;
  s.slice = ((vocab + s.ctas - 1) / s.ctas + 63) & ~63;
  s.smem = (size_t)s.slice * es + 32;
  return s;
}

template <int NT, typename K>
cudaError_t launch(K kernel, int rows, const Shape& s, const SampleParams& p, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem);
  if (e != cudaSuccess) return e;
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
  return cudaLaunchKernelEx(&cfg, kernel, p);
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
  SampleParams p = {};
  p.logits = logits; p.row_stride = row_stride; p.vocab = vocab; p.temperature = temperature; p.top_p = top_p;
  p.uniform = uniform; p.tokens = tokens; p.probs = probs; p.probs_stride = probs_stride;
  const Shape shape = pick_shape(rows, vocab, elem_size(dtype));
  p.slice = shape.slice;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    return shape.wide ? launch<512>(sample_kernel<T, 512>, rows, shape, p, st) : launch<256>(sample_kernel<T, 256>, rows, shape, p, st);
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
      const Shape shape = pick_shape(nnz, vocab, elem_size(dtype));
      p.slice = shape.slice;
      const cudaError_t er = shape.wide ? launch<512>(verify_rows_kernel<T, 512>, nnz, shape, p, st)
                                        : launch<256>(verify_rows_kernel<T, 256>, nnz, shape, p, st);
      if (er != cudaSuccess) return er;
    }
    const Shape shape = pick_shape(batch, vocab, elem_size(dtype));
    p.slice = shape.slice;
    return shape.wide ? launch<512>(verify_draw_kernel<T, 512>, batch, shape, p, st)
                      : launch<256>(verify_draw_kernel<T, 256>, batch, shape, p, st);
  };
  const cudaError_t e = dtype == DSV_F32 ? go(float{}) : dtype == DSV_F16 ? go(__half{}) : go(__nv_bfloat16{});
  if (e != cudaSuccess) return fail(DSV_E_CUDA, "verify_draft launch failed: %s", cudaGetErrorString(e));
  return DSV_OK;
}

}  // extern "C"
