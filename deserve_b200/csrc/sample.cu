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

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCtas = 8;  // of a cluster (the portable limit)
constexpr int kMaxVocab = 1 << 18, kIndexBits = 18;
constexpr double kOne = 17592186044416.0;          // 2^44: the fixed-point weight of the largest logit
constexpr double kProbOne = 1152921504606846976.0;  // 2^60: fixed-point probabilities of the residual
constexpr double kLowest = -46.0 * 64.0;            // in 1/64 of a factor of two: weights below round to 0
constexpr int kTable = 64;
typedef unsigned long long u64;

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
  Slot slot[24];
  u64 warp_a[kWarps], warp_b[kWarps];
  u64 seg[kWarps];  // mass of the warps' segments
  u64 found;
  int found_i;
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

// What is known of a row: its largest logit and the scale of its exponent.
struct RowScale {
  float top;        // largest logit that is a number
  double c;         // 64 log2(e) / T
  float c32;        // log2(e) / T
  float bin_scale;  // bins per unit of (top - l)
};
__device__ __forceinline__ RowScale row_scale(float top, float temperature) {
  RowScale s;
  s.top = top;
  const double inv = 1.0 / (double)temperature;
  s.c = 92.332482616893657 * inv;  // 64 / ln 2
  s.c32 = (float)fmin(1.4426950408889634 * inv, 3e38);
  s.bin_scale = (float)fmin(64.0 * inv, 3e38);  // bins of 1/64: the 32 nats that a 2^-44 weight can lie below the top
  return s;
}
// Fixed-point weight: 2^(d / 64), d = 64 log2(e) (l - top) / T = n + r with |r| <= 1/2, from a table of 2^(j / 64)
// and e^(r ln 2 / 64) to the fourth power (|r ln 2 / 64| < 0.0055: the next term is below 2^-44). Ten FP64
// instructions; 128,256 entries keep one SM's FP64 units busy for about 11 us, twice what its share of HBM needs.
__device__ __forceinline__ u64 fixed_weight(float l, const RowScale& s, const Shared& sh) {
  const double d = ((double)l - (double)s.top) * s.c;
  const bool any = d >= kLowest;  // NaN and -inf: no weight
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it leaves the rounded integer in the low bits
  const double m = (any ? d : 0.0) + magic;
  const int n = __double2loint(m);
  const double r = (any ? d : 0.0) - (m - magic);
  constexpr double a = 0.010830424696249145;  // ln 2 / 64
  double e = fma(r, a * a * a * a / 24.0, a * a * a / 6.0);
  e = fma(r, e, a * a / 2.0);
  e = fma(r, e, a);
  e = fma(r, e, 1.0);
  const double t = sh.table[n & (kTable - 1)];
  const double scaled = __hiloint2double(__double2hiint(t) + ((n >> 6) << 20), __double2loint(t));
  const u64 bits = (u64)__double_as_longlong(fma(scaled, e, 4503599627370496.0));  // + 2^52: rounded to an integer
  return any ? bits - 0x4330000000000000ull : 0;
}
__device__ __forceinline__ double weight(float l, const RowScale& s) {  // in units of the largest, where one entry counts
  const double x = ((double)l - (double)s.top) * s.c;
  return x > -64000.0 ? exp2(x * 0.015625) : 0.0;
}
__device__ __forceinline__ int bin_of(float l, const RowScale& s) {
  return (int)fminf((s.top - l) * s.bin_scale, (float)(kBins - 1));
}

// A CTA's slice of a row in shared memory: 16-byte vectors as in global memory, what lies before and behind
// the slice filled with -inf (no token). Vector v holds the entries first + v * N and on.
template <typename T>
struct Slice {
  static constexpr int N = Vec16<T>::N;
  const uint4* v;
  int n_vec, first;
  int seg;  // vectors of a warp's contiguous segment
  __device__ __forceinline__ void get(int i, float (&f)[N]) const { Vec16<T>::unpack(v[i], f); }
};

template <typename T>
__device__ __forceinline__ T minus_inf() { return from_f32<T>(-INFINITY); }

// Load the slice; largest entry that is a number (NaN ignored) and its lowest index.
template <typename T>
__device__ Slice<T> load_slice(const T* row, int vocab, int slice, uint4* buf, float& best, int& at) {
  constexpr int N = Slice<T>::N;
  const int begin = min((int)cluster_rank() * slice, vocab), end = min(begin + slice, vocab);
  const T* src = row + begin;
  const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T)), n = end - begin;
  Slice<T> sl;
  sl.v = buf;
  sl.first = begin - lead;
  sl.n_vec = n > 0 ? (lead + n + N - 1) / N : 0;
  sl.seg = ((sl.n_vec + kWarps * 32 - 1) / (kWarps * 32)) * 32;
  best = -INFINITY;
  at = 0x7fffffff;
  const uint4* g = reinterpret_cast<const uint4*>(src - lead);
  auto take = [&](int v, const uint4& u) {
    buf[v] = u;
    float f[N];
    Vec16<T>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f[i] > best) { best = f[i]; at = sl.first + v * N + i; }
  };
  const int v0 = lead > 0 ? 1 : 0, v1 = n > 0 ? (lead + n) / N : 0;  // whole vectors
  auto ragged = [&](int e) {  // a vector that reaches over an end of the slice
    __align__(16) T tmp[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = e * N + i - lead;
      tmp[i] = k >= 0 && k < n ? src[k] : minus_inf<T>();
    }
    take(e, *reinterpret_cast<const uint4*>(tmp));
  };
  // (every thread meets its vectors in ascending order: the first of equal maxima stays)
  if (threadIdx.x == 0 && lead > 0 && n > 0) ragged(0);
  int v = v0 + threadIdx.x;
  for (; v + 3 * kThreads < v1; v += 4 * kThreads) {
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = ld_stream16(g + v + k * kThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k) take(v + k * kThreads, u[k]);
  }
  for (; v < v1; v += kThreads) take(v, ld_stream16(g + v));
  if (threadIdx.x == 1 && v1 < sl.n_vec && (sl.n_vec > 1 || lead == 0)) ragged(sl.n_vec - 1);
  return sl;
}

// The cluster's largest logit and its lowest index (index -1: nothing but NaN and -inf). A row with +inf becomes one
// of 0 (those) and -inf. Also readies the table of the exponential.
template <typename T>
__device__ float row_top(const Slice<T>& sl, float best, int at, int& index, Shared& sh, uint4* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // (value, lowest index) as one integer
  u64 k = at == 0x7fffffff ? 0 : ((u64)order_key<float>(best) << 32) | (u64)(0xffffffffu - (uint32_t)at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, shfl_xor64(k, o));
  if (lane == 0) sh.warp_a[warp] = k;
  if (threadIdx.x < kTable) sh.table[threadIdx.x] = exp2((double)threadIdx.x / kTable) * kOne;
  __syncthreads();
  if (warp == 0) {
    k = lane < kWarps ? sh.warp_a[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = max(k, shfl_xor64(k, o));
    if (lane == 0) sh.slot[0].a = k;
  }
  cluster_sync();
  const int c = cluster_size();
  k = 0;
  for (int r = 0; r < c; ++r) k = max(k, ld_remote64(remote(&sh.slot[0].a, r)));
  if (k == 0) {
    index = -1;
    return -INFINITY;
  }
  index = (int)(0xffffffffu - (uint32_t)k);
  const uint32_t key = (uint32_t)(k >> 32);
  float top = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
  if (top == INFINITY) {
    constexpr int N = Slice<T>::N;
    for (int v = threadIdx.x; v < sl.n_vec; v += kThreads) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = f[i] == INFINITY ? 0.f : -INFINITY;
      buf[v] = Vec16<T>::pack(f);
    }
    __syncthreads();
    top = 0.f;
  }
  return top;
}

// Sum over the cluster of one integer per warp, through slot `s`: the whole, and what the CTAs before this one have.
__device__ u64 cluster_total(u64 mine, Shared& sh, int s, u64& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) sh.warp_a[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const u64 v = warp_sum(lane < kWarps ? sh.warp_a[lane] : 0);
    if (lane == 0) sh.slot[s].a = v;
  }
  cluster_sync();
  const int c = cluster_size(), rank = cluster_rank();
  u64 all = 0;
  before = 0;
  for (int r = 0; r < c; ++r) {
    const u64 v = ld_remote64(remote(&sh.slot[s].a, r));
    if (r < rank) before += v;
    all += v;
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
__device__ __forceinline__ void hist_clear(Shared& sh) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist_lo[i] = sh.hist_hi[i] = 0;
}

// First bin of the cluster's summed histogram whose inclusive running sum exceeds a limit, the sum before it and its own
// mass; -1: none. limit_of(whole) gives the limit. Each CTA sums its share of the bins over the cluster; three slots.
template <typename F>
__device__ int hist_find(Shared& sh, int s, F limit_of, u64& limit, u64& before, u64& mass) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = cluster_size(), rank = cluster_rank();
  const int bins = kBins / c, per = max(1, bins / kThreads);  // bins of this CTA, of a thread
  cluster_sync();  // all histograms are complete
  u64 v[kBins / kThreads], mine = 0;
  const int b0 = threadIdx.x * per;
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) {
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
  if (lane == 0) sh.warp_b[warp] = warp_mass;
  if (threadIdx.x == 0) sh.slot[s + 1].a = ~0ull;
  u64 cta_before, base = 0;
  limit = limit_of(cluster_total(warp_mass, sh, s, cta_before));
  for (int w = 0; w < warp; ++w) base += sh.warp_b[w];
  u64 at = cta_before + base + inc - mine;
  if (at <= limit && at + mine > limit) {
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      if (at <= limit && at + v[i] > limit) {
        sh.slot[s + 1].a = (u64)(rank * bins + b0 + i);
        sh.slot[s + 1].b = at;
        sh.slot[s + 2].a = v[i];
      }
      at += v[i];
    }
  }
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

struct Kept {
  u64 border;  // rank key of the last kept token; 0: all
  u64 total;   // sum of the kept weights
};

// Top-p border of the row. Without a cut the masses of the warps' segments are left in sh.seg.
template <typename T>
__device__ Kept find_kept(const Slice<T>& sl, const RowScale& s, float top_p, Shared& sh) {
  constexpr int N = Slice<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Kept k;
  k.border = 0;
  const int w0 = min(warp * sl.seg, sl.n_vec), w1 = min(w0 + sl.seg, sl.n_vec);
  if (!(top_p < 1.f)) {  // NaN: no cut
    u64 sum = 0, before;
    for (int v = w0 + lane; v < w1; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += fixed_weight(f[i], s, sh);
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.seg[warp] = sum;
    k.total = cluster_total(sum, sh, 1, before);
    return k;
  }
  hist_clear(sh);
  __syncthreads();
  for (int v = w0 + lane; v < w1; v += 32) {
    float f[N];
    sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u64 w = fixed_weight(f[i], s, sh);
      if (w) hist_add(sh, bin_of(f[i], s), w);
    }
  }
  u64 limit, before, mass;
  const double share = (double)fmaxf(top_p, 0.f);
  int bin = hist_find(sh, 2, [&](u64 all) { k.total = all; return (u64)(share * (double)all); }, limit, before, mass);
  if (bin < 0) return k;  // cannot happen with top_p < 1
  limit -= before;
  u64 kept = before, lo = ~0ull, hi = 0;
  for (int v = w0 + lane; v < w1; v += 32) {
    float f[N];
    sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!(f[i] > -INFINITY) || bin_of(f[i], s) != bin) continue;
      const u64 key = rank_key<T>(f[i], sl.first + v * N + i);
      lo = min(lo, key);
      hi = max(hi, key);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lo = min(lo, shfl_xor64(lo, o)); hi = max(hi, shfl_xor64(hi, o)); }
  if (lane == 0) { sh.warp_a[warp] = lo; sh.warp_b[warp] = hi; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) { lo = min(lo, sh.warp_a[w]); hi = max(hi, sh.warp_b[w]); }
    sh.slot[5].a = lo;
    sh.slot[5].b = hi;
  }
  cluster_sync();  // also: every CTA has read the histogram that is cleared next
  for (int r = 0; r < (int)cluster_size(); ++r) {
    lo = min(lo, ld_remote64(remote(&sh.slot[5].a, r)));
    hi = max(hi, ld_remote64(remote(&sh.slot[5].b, r)));
  }
  for (int s0 = 6;; s0 += 3) {  // 50 bits of rank key, 11 a round: five rounds at most
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
    hist_clear(sh);
    __syncthreads();
    for (int v = w0 + lane; v < w1; v += 32) {
      float f[N];
      sl.get(v, f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!(f[i] > -INFINITY)) continue;
        const u64 key = rank_key<T>(f[i], sl.first + v * N + i);
        if (key < lo || key > hi) continue;
        const u64 w = fixed_weight(f[i], s, sh);
        if (w) hist_add(sh, (int)((hi - key) >> shift), w);
      }
    }
    u64 same;
    bin = hist_find(sh, s0, [&](u64) { return limit; }, same, before, mass);
    if (bin < 0) return k;  // cannot happen: the members' mass exceeds the limit
    limit -= before;
    kept += before;
    hi -= (u64)bin << shift;
    const u64 width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    if (shift == 0) {
      k.border = hi;
      k.total = kept + mass;
      return k;
    }
  }
}

// One entry's mass in a draw.
template <typename T>
struct Mass {
  RowScale s;
  u64 border;
  double inv_z;         // 1 / Z in units of 2^-44, residual only
  const float* minus;   // row of the draft distribution to subtract, or null
  int one_hot;          // or the token whose draft probability is 1, or -1
  bool residual;
  __device__ __forceinline__ u64 operator()(float l, int i, const Shared& sh) const {
    if (!(l > -INFINITY) || rank_key<T>(l, i) < border) return 0;
    u64 w = fixed_weight(l, s, sh);
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
template <typename T>
__device__ bool draw(const Slice<T>& sl, const Mass<T>& mass, float u, bool ready, int slot, int32_t* out, Shared& sh) {
  constexpr int N = Slice<T>::N;
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
    const int w0 = min(warp * sl.seg, sl.n_vec);
    const u64 sum = sum_of(w0, min(w0 + sl.seg, sl.n_vec));
    if (lane == 0) sh.seg[warp] = sum;
  }
  __syncthreads();
  u64 before;
  const u64 all = cluster_total(sh.seg[warp], sh, slot, before);
  if (all == 0) return false;
  const double x = u > 0.f ? (double)u * (double)all : 0.0;  // NaN: 0
  u64 target = x < (double)all ? min((u64)x, all - 1) : all - 1;
  u64 mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += sh.seg[w];
  if (target < before || target - before >= mine) return true;  // another CTA's
  target -= before;
  int w = 0;
  while (w < kWarps - 1 && target >= sh.seg[w]) target -= sh.seg[w++];
  // the warps share that segment
  const int begin = min(w * sl.seg, sl.n_vec), end = min(begin + sl.seg, sl.n_vec);
  const int sub = (end - begin + kWarps - 1) / kWarps;
  const int a = min(begin + warp * sub, end);
  const u64 sum = sum_of(a, min(a + sub, end));
  if (lane == 0) sh.warp_b[warp] = sum;
  __syncthreads();
  w = 0;
  while (w < kWarps - 1 && target >= sh.warp_b[w]) target -= sh.warp_b[w++];
  if (warp != w) return true;
  for (int v0 = a; v0 < min(a + sub, end); v0 += 32) {
    const int v = v0 + lane;
    u64 m[N], total = 0;
    const bool in = v < min(a + sub, end);
    float f[N];
    if (in) sl.get(v, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = in ? mass(f[i], sl.first + v * N + i, sh) : 0;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint4* buf = reinterpret_cast<uint4*>(dyn);
  const int r = blockIdx.x / cluster_size();
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const float t = __ldg(p.temperature + r);
  float best;
  int at, first;
  const Slice<T> sl = load_slice(row, p.vocab, p.slice, buf, best, at);
  const float top = row_top(sl, best, at, first, sh, buf);
  constexpr int N = Slice<T>::N;
  const int begin = min((int)cluster_rank() * p.slice, p.vocab), end = min(begin + p.slice, p.vocab);
  float* probs = p.probs == nullptr ? nullptr : p.probs + (int64_t)r * p.probs_stride;
  if (!(t > 0.f) || first < 0) {  // greedy, or a row without a token
    if (cluster_rank() == 0 && threadIdx.x == 0) p.tokens[r] = max(first, 0);
    if (probs != nullptr)
      for (int i = begin + threadIdx.x; i < end; i += kThreads) probs[i] = i == first ? 1.f : 0.f;
  } else {
    Mass<T> mass;
    mass.s = row_scale(top, t);
    const float top_p = __ldg(p.top_p + r);
    const Kept k = find_kept(sl, mass.s, top_p, sh);
    mass.border = k.border; mass.inv_z = 0.0; mass.minus = nullptr; mass.one_hot = -1; mass.residual = false;
    draw(sl, mass, __ldg(p.uniform + r), !(top_p < 1.f), 22, p.tokens + r, sh);
    if (probs != nullptr) {
      const float inv = (float)(kOne / (double)k.total);
      for (int v = threadIdx.x; v < sl.n_vec; v += kThreads) {
        float f[N];
        sl.get(v, f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int x = sl.first + v * N + i;
          if (x >= begin && x < end)
            probs[x] = f[i] > -INFINITY && rank_key<T>(f[i], x) >= k.border ? exp2f((f[i] - top) * mass.s.c32) * inv : 0.f;
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

// One cluster per row that has a draft behind it: is the draft accepted?
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint4* buf = reinterpret_cast<uint4*>(dyn);
  const int r = blockIdx.x / cluster_size();
  const int req = owner_of(p.indptr, p.batch, r);
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (r < begin || r + 1 >= end || end > p.nnz) return;  // a last row, or behind the last request (the whole cluster)
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const int x = __ldg(p.draft + r + 1);
  const float t = __ldg(p.temperature + req);
  float best;
  int at, first;
  const Slice<T> sl = load_slice(row, p.vocab, p.slice, buf, best, at);
  const float top = row_top(sl, best, at, first, sh, buf);
  double px = 0.0;
  if (first >= 0 && x >= 0 && x < p.vocab) {
    if (!(t > 0.f)) {
      px = x == first ? 1.0 : 0.0;
    } else {
      const RowScale s = row_scale(top, t);
      const Kept k = find_kept(sl, s, __ldg(p.top_p + req), sh);
      float l = to_f32(row[x]);
      if (l == INFINITY) l = 0.f;  // as row_top rewrote the row
      else if (top == 0.f && to_f32(row[first]) == INFINITY) l = -INFINITY;
      if (l > -INFINITY && rank_key<T>(l, x) >= k.border) px = weight(l, s) * (kOne / (double)k.total);
    }
  }
  if (cluster_rank() == 0 && threadIdx.x == 0) {
    const double q = p.draft_probs == nullptr || x < 0 || x >= p.vocab
                         ? 1.0 : (double)__ldg(p.draft_probs + (int64_t)r * p.draft_stride + x);
    p.ok[r] = (double)__ldg(p.uniform + r) * q < px ? 1 : 0;
  }
  cluster_sync();
}

// One cluster per request: the accepted prefix, then a draw from the residual of the first rejected row or
// from the last row.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draw_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint4* buf = reinterpret_cast<uint4*>(dyn);
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
  const float t = __ldg(p.temperature + req);
  float best;
  int at, first;
  const Slice<T> sl = load_slice(row, p.vocab, p.slice, buf, best, at);
  const float top = row_top(sl, best, at, first, sh, buf);
  if (lead) p.accepted[req] = r - begin;
  if (!(t > 0.f) || first < 0) {
    if (lead) p.tokens[req] = max(first, 0);
  } else {
    Mass<T> mass;
    mass.s = row_scale(top, t);
    const float top_p = __ldg(p.top_p + req), u = __ldg(p.uniform + end - 1);
    const Kept k = find_kept(sl, mass.s, top_p, sh);
    mass.border = k.border;
    mass.inv_z = 1.0 / (double)k.total;
    mass.residual = rejected;
    mass.minus = rejected && p.draft_probs != nullptr ? p.draft_probs + (int64_t)r * p.draft_stride : nullptr;
    mass.one_hot = rejected ? __ldg(p.draft + r + 1) : -1;
    if (!draw(sl, mass, u, !rejected && !(top_p < 1.f), 22, p.tokens + req, sh)) {
      mass.residual = false;  // nothing left above the draft's distribution: the target's own
      draw(sl, mass, u, false, 23, p.tokens + req, sh);
    }
  }
  cluster_sync();
}

// ---- host --------------------------------------------------------------------------------------------
struct Shape {
  int ctas, slice;
  size_t smem;
};
// CTAs of a row: as few as keep a slice within 64 KB (two CTAs per SM, so that one loads while the other
// computes); more, up to 8, while all of them still fit the machine at once and a slice keeps 2048 entries.
Shape pick_shape(int rows, int vocab, int es) {
  Shape s;
  s.ctas = 1;
  while (s.ctas < kMaxCtas && (int64_t)vocab * es > (int64_t)s.ctas * 65536) s.ctas *= 2;
  while (s.ctas < kMaxCtas && (int64_t)rows * s.ctas * 2 <= 296 && vocab / (s.ctas * 2) >= 2048) s.ctas *= 2;
  s.slice = ((vocab + s.ctas - 1) / s.ctas + 63) & ~63;
  s.smem = (size_t)s.slice * es + 32;
  return s;
}

template <typename K>
cudaError_t launch(K kernel, int rows, const Shape& s, const SampleParams& p, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * s.ctas);
  cfg.blockDim = dim3(kThreads);
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
  cudaError_t e;
  switch (dtype) {
    case DSV_F32: e = launch(sample_kernel<float>, rows, shape, p, st); break;
    case DSV_F16: e = launch(sample_kernel<__half>, rows, shape, p, st); break;
    default: e = launch(sample_kernel<__nv_bfloat16>, rows, shape, p, st);
  }
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
  auto go = [&](auto rows_kernel, auto draw_kernel) -> cudaError_t {
    if (nnz > 0) {
      const Shape shape = pick_shape(nnz, vocab, elem_size(dtype));
      p.slice = shape.slice;
      const cudaError_t er = launch(rows_kernel, nnz, shape, p, st);
      if (er != cudaSuccess) return er;
    }
    const Shape shape = pick_shape(batch, vocab, elem_size(dtype));
    p.slice = shape.slice;
    return launch(draw_kernel, batch, shape, p, st);
  };
  cudaError_t e;
  switch (dtype) {
    case DSV_F32: e = go(verify_rows_kernel<float>, verify_draw_kernel<float>); break;
    case DSV_F16: e = go(verify_rows_kernel<__half>, verify_draw_kernel<__half>); break;
    default: e = go(verify_rows_kernel<__nv_bfloat16>, verify_draw_kernel<__nv_bfloat16>);
  }
  if (e != cudaSuccess) return fail(DSV_E_CUDA, "verify_draft launch failed: %s", cudaGetErrorString(e));
  return DSV_OK;
}

}  // extern "C"
