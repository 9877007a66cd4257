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
// The top-p border is found without sorting: a histogram of weight over 2048 bins of (max - l) / T gives
// the bin of the border; the members of that bin are then split 2048 ways again by (value, index) until
// one token is left (two or three times).
#include <algorithm>

#include "common.cuh"

namespace dsv {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;
constexpr int kMaxVocab = 1 << 18;
constexpr double kOne = 17592186044416.0;          // 2^44: the fixed-point weight of the largest logit
constexpr double kProbOne = 1152921504606846976.0;  // 2^60: fixed-point probabilities of the residual
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
  int* status;
};

struct Shared {
  uint32_t hist_lo[kBins], hist_hi[kBins];
  u64 warp_a[32], warp_b[32];
  float warp_f[32];
  int warp_i[32];
  u64 out[4];
  int out_i[2];
};

// order-preserving integer of a float (NaN excluded by the callers)
__device__ __forceinline__ uint32_t order_key(float x) {
  x += 0.f;  // -0 ranks with +0
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// (value, index) as one integer, larger = ranked earlier; unique within a row
__device__ __forceinline__ u64 rank_key(float l, int index) {
  return ((u64)order_key(l) << 18) | (u64)(kMaxVocab - 1 - index);
}

__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

__device__ __forceinline__ u64 block_sum64(u64 v, Shared& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += shfl_xor64(v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.warp_a[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += shfl_xor64(v, o);
  return v;
}

// What is known of a row: its largest logit and the scale of its exponent.
struct RowScale {
  float top;        // largest logit that is a number
  double inv_t;
  float bin_scale;  // bins per unit of (top - l)
};

__device__ __forceinline__ RowScale row_scale(float top, float temperature) {
  RowScale s;
  s.top = top;
  s.inv_t = 1.0 / (double)temperature;
  // bins of 1/64: the 32 nats that a 2^-44 weight can lie below the top
  s.bin_scale = (float)fmin(64.0 * s.inv_t, 3e38);
  return s;
}
__device__ __forceinline__ double weight(float l, const RowScale& s) {
  if (l == s.top) return 1.0;
  const double x = ((double)l - (double)s.top) * s.inv_t;
  return x > -700.0 ? exp(x) : 0.0;  // NaN is no token: 0
}
__device__ __forceinline__ u64 fixed_weight(float l, const RowScale& s) { return (u64)__double2ull_rn(weight(l, s) * kOne); }
__device__ __forceinline__ int bin_of(float l, const RowScale& s) {
  if (l == s.top) return 0;
  return (int)fminf((s.top - l) * s.bin_scale, (float)(kBins - 1));
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
// First bin whose inclusive running sum exceeds `limit`, with the sum before it; -1: none. All threads get the answer.
__device__ __forceinline__ int hist_find(Shared& sh, u64 limit, u64& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int PER = kBins / kThreads;
  u64 v[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = threadIdx.x * PER + i;
    v[i] = ((u64)sh.hist_hi[b] << 32) + sh.hist_lo[b];
    mine += v[i];
  }
  u64 inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) sh.warp_b[warp] = inc;
  if (threadIdx.x == 0) sh.out_i[0] = -1;
  __syncthreads();
  u64 base = 0;
  for (int w = 0; w < warp; ++w) base += sh.warp_b[w];
  u64 at = base + inc - mine;
  if (at <= limit && at + mine > limit) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (at + v[i] > limit) {
        sh.out_i[0] = threadIdx.x * PER + i;
        sh.out[0] = at;
        break;
      }
      at += v[i];
    }
  }
  __syncthreads();
  before = sh.out[0];
  return sh.out_i[0];
}

// Largest logit and its lowest index (index -1: nothing but NaN and -inf).
template <typename T>
__device__ __forceinline__ float row_top(const T* row, int n, int& index, Shared& sh) {
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float l = to_f32(row[i]);
    if (l > best) { best = l; at = i; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (ob > best || (ob == best && oi < at)) { best = ob; at = oi; }
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { sh.warp_f[threadIdx.x >> 5] = best; sh.warp_i[threadIdx.x >> 5] = at; }
  __syncthreads();
  best = sh.warp_f[threadIdx.x & 31];
  at = sh.warp_i[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (ob > best || (ob == best && oi < at)) { best = ob; at = oi; }
  }
  index = at == 0x7fffffff ? -1 : at;
  return best;
}

struct Kept {
  u64 border;  // rank key of the last kept token; 0: all
  u64 total;   // sum of the kept weights
};

template <typename T>
__device__ Kept find_kept(const T* row, int n, const RowScale& s, float top_p, Shared& sh) {
  Kept k;
  k.border = 0;
  const bool cut = top_p < 1.f;  // NaN: no cut
  __syncthreads();
  if (cut) hist_clear(sh);
  __syncthreads();
  u64 sum = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float l = to_f32(row[i]);
    const u64 w = fixed_weight(l, s);
    sum += w;
    if (cut && w) hist_add(sh, bin_of(l, s), w);
  }
  k.total = block_sum64(sum, sh);
  if (!cut) return k;
  u64 limit = (u64)((double)fmaxf(top_p, 0.f) * (double)k.total), before;
  int bin = hist_find(sh, limit, before);
  if (bin < 0) return k;  // cannot happen with top_p < 1
  limit -= before;
  u64 kept = before, lo = ~0ull, hi = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float l = to_f32(row[i]);
    if (!(l > -INFINITY) || bin_of(l, s) != bin || !fixed_weight(l, s)) continue;
    const u64 key = rank_key(l, i);
    lo = min(lo, key);
    hi = max(hi, key);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lo = min(lo, shfl_xor64(lo, o)); hi = max(hi, shfl_xor64(hi, o)); }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { sh.warp_a[threadIdx.x >> 5] = lo; sh.warp_b[threadIdx.x >> 5] = hi; }
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) { lo = min(lo, sh.warp_a[w]); hi = max(hi, sh.warp_b[w]); }
  for (;;) {
    const u64 range = hi - lo;
    const int shift = max(0, 64 - __clzll((long long)range) - 11);
    __syncthreads();
    hist_clear(sh);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float l = to_f32(row[i]);
      if (!(l > -INFINITY)) continue;
      const u64 key = rank_key(l, i);
      if (key < lo || key > hi) continue;
      const u64 w = fixed_weight(l, s);
      if (w) hist_add(sh, (int)((hi - key) >> shift), w);
    }
    __syncthreads();
    bin = hist_find(sh, limit, before);
    if (bin < 0) return k;  // cannot happen: the members' weight exceeds the limit
    limit -= before;
    kept += before;
    hi -= (u64)bin << shift;
    const u64 width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    if (shift == 0) {
      k.border = hi;
      k.total = kept + (((u64)sh.hist_hi[bin] << 32) + sh.hist_lo[bin]);
      __syncthreads();
      return k;
    }
  }
}

// One entry's mass in a draw.
struct Mass {
  RowScale s;
  u64 border;
  double inv_z;         // 1 / Z in units of 2^-44, residual only
  const float* minus;   // row of the draft distribution to subtract, or null
  int one_hot;          // or the token whose draft probability is 1, or -1
  bool residual;
  __device__ __forceinline__ u64 operator()(float l, int i) const {
    if (!(l > -INFINITY)) return 0;
    u64 w = rank_key(l, i) >= border ? fixed_weight(l, s) : 0;
    if (residual && w) {
      const double q = minus != nullptr ? (double)__ldg(minus + i) : i == one_hot ? 1.0 : 0.0;
      const double r = (double)w * inv_z - q;
      w = r > 0.0 ? (u64)__double2ull_rn(r * kProbOne) : 0;
    }
    return w;
  }
};

// First index whose running sum of mass exceeds u * (whole sum); -1 when there is no mass.
template <typename T>
__device__ int draw(const T* row, int n, const Mass& mass, float u, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int begin = 0, end = n;
  u64 target = 0;
  for (int level = 0; level < 2; ++level) {  // 32 warps share [begin, end); then the warp segment that holds the target
    const int seg = (end - begin + 31) / 32;
    const int a = min(begin + warp * seg, end), b = min(a + seg, end);
    u64 sum = 0;
    for (int i = a + lane; i < b; i += 32) sum += mass(to_f32(row[i]), i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += shfl_xor64(sum, o);
    __syncthreads();
    if (lane == 0) sh.warp_a[warp] = sum;
    __syncthreads();
    if (level == 0) {
      u64 all = 0;
      for (int w = 0; w < 32; ++w) all += sh.warp_a[w];
      if (all == 0) return -1;
      const double x = u > 0.f ? (double)u * (double)all : 0.0;  // NaN: 0
      target = x < (double)all ? min((u64)x, all - 1) : all - 1;
    }
    int w = 0;
    while (w < 31 && target >= sh.warp_a[w]) target -= sh.warp_a[w++];
    begin = min(begin + w * seg, end);
    end = min(begin + seg, end);
  }
  // a few entries per lane are left: every warp walks them (the answer is needed by all)
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    const u64 m = i < end ? mass(to_f32(row[i]), i) : 0;
    u64 inc = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
    if (hit) return i0 + __ffs(hit) - 1;
    target -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return end - 1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Shared sh;
  const int r = blockIdx.x;
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  float* probs = p.probs == nullptr ? nullptr : p.probs + (int64_t)r * p.probs_stride;
  const float t = __ldg(p.temperature + r);
  int first;
  const float top = row_top(row, p.vocab, first, sh);
  if (!(t > 0.f) || first < 0) {  // greedy, or a row without a token
    if (threadIdx.x == 0) p.tokens[r] = max(first, 0);
    if (probs != nullptr)
      for (int i = threadIdx.x; i < p.vocab; i += kThreads) probs[i] = i == first ? 1.f : 0.f;
    return;
  }
  Mass mass;
  mass.s = row_scale(top, t);
  const Kept k = find_kept(row, p.vocab, mass.s, __ldg(p.top_p + r), sh);
  mass.border = k.border; mass.inv_z = 0.0; mass.minus = nullptr; mass.one_hot = -1; mass.residual = false;
  const int token = draw(row, p.vocab, mass, __ldg(p.uniform + r), sh);
  if (threadIdx.x == 0) p.tokens[r] = token;
  if (probs != nullptr) {
    const double inv = kOne / (double)k.total;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
      const float l = to_f32(row[i]);
      probs[i] = l > -INFINITY && rank_key(l, i) >= k.border ? (float)(weight(l, mass.s) * inv) : 0.f;
    }
  }
}

__device__ __forceinline__ int owner_of(const int32_t* __restrict__ indptr, int batch, int row) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(indptr + mid) <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// One CTA per row that has a draft behind it: is the draft accepted?
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const SampleParams p) {
  __shared__ Shared sh;
  const int r = blockIdx.x;
  const int req = owner_of(p.indptr, p.batch, r);
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (r < begin || r + 1 >= end || end > p.nnz) return;  // a last row, or behind the last request
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
  const int x = __ldg(p.draft + r + 1);
  const float t = __ldg(p.temperature + req);
  int first;
  const float top = row_top(row, p.vocab, first, sh);
  double px = 0.0;
  if (first >= 0 && x >= 0 && x < p.vocab) {
    if (!(t > 0.f)) {
      px = x == first ? 1.0 : 0.0;
    } else {
      const RowScale s = row_scale(top, t);
      const Kept k = find_kept(row, p.vocab, s, __ldg(p.top_p + req), sh);
      const float l = to_f32(row[x]);
      if (l > -INFINITY && rank_key(l, x) >= k.border) px = weight(l, s) * (kOne / (double)k.total);
    }
  }
  if (threadIdx.x == 0) {
    const double q = p.draft_probs == nullptr || x < 0 || x >= p.vocab
                         ? 1.0 : (double)__ldg(p.draft_probs + (int64_t)r * p.draft_stride + x);
    p.ok[r] = (double)__ldg(p.uniform + r) * q < px ? 1 : 0;
  }
}

// One CTA per request: the accepted prefix, then a draw from the residual of the first rejected row or
// from the last row.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draw_kernel(const SampleParams p) {
  __shared__ Shared sh;
  const int req = blockIdx.x;
  const int begin = __ldg(p.indptr + req), end = __ldg(p.indptr + req + 1);
  if (begin < 0 || end <= begin || end > p.nnz) {
    if (threadIdx.x == 0) {
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
  int first, token;
  const float top = row_top(row, p.vocab, first, sh);
  if (!(t > 0.f) || first < 0) {
    token = max(first, 0);
  } else {
    Mass mass;
    mass.s = row_scale(top, t);
    const Kept k = find_kept(row, p.vocab, mass.s, __ldg(p.top_p + req), sh);
    mass.border = k.border;
    mass.inv_z = 1.0 / (double)k.total;
    mass.residual = rejected;
    mass.minus = rejected && p.draft_probs != nullptr ? p.draft_probs + (int64_t)r * p.draft_stride : nullptr;
    mass.one_hot = rejected ? __ldg(p.draft + r + 1) : -1;
    const float u = __ldg(p.uniform + end - 1);
    token = draw(row, p.vocab, mass, u, sh);
    if (token < 0) {  // nothing left above the draft's distribution: the target's own
      mass.residual = false;
      token = draw(row, p.vocab, mass, u, sh);
    }
  }
  if (threadIdx.x == 0) {
    p.accepted[req] = r - begin;
    p.tokens[req] = token;
  }
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
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DSV_F32: sample_kernel<float><<<rows, kThreads, 0, st>>>(p); break;
    case DSV_F16: sample_kernel<__half><<<rows, kThreads, 0, st>>>(p); break;
    default: sample_kernel<__nv_bfloat16><<<rows, kThreads, 0, st>>>(p);
  }
  DSV_CUDA(cudaGetLastError());
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
    if (nnz > 0) rows_kernel<<<nnz, kThreads, 0, st>>>(p);
    draw_kernel<<<batch, kThreads, 0, st>>>(p);
    return cudaGetLastError();
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
