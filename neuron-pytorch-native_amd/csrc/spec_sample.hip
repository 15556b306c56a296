// Sampling of one token per row of logits with temperature, top-k, top-p and min-p from given
// uniforms, for gfx950.
//
// A row's tokens are ranked by logit, larger first, the lower index first among equals. With the
// row's maximum m, token i weighs w_i = exp((l_i - m) / T). Each filter keeps a prefix of the ranks:
//   top-k  the first k;
//   top-p  as many as it takes for their weight to reach p times the top-k prefix's;
//   min-p  those with w_i >= min_p.
// The shortest of the three is sampled by inversion: the first rank whose cumulative weight exceeds
// u times the prefix's. A prefix is known by its weight alone (the shorter weighs less), so all that
// has to be found in the row are three ranks, "the first with a cumulative count or weight of at
// least x", one after the other: the last of the k, the last of the top-p prefix, the sample.
//
// Weights are integers, W_i = round(w_i 2^42) from a 64-bit exponential (a row of 2^20 sums to at
// most 2^62), so sums are exact whatever their order and every run gives the same token; tokens that
// round to 0 (w < 2^-43) have no part in it. 32-bit exponentials would not do: the ranks' borders in
// a flat row of 150000 tokens lie 10^-5 of the sum apart or less.
#include "npn_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr double kOne = 4398046511104.0;  // 2^42
constexpr int kDigit = 11;                // bits of a key per level of the search
constexpr int kBins = 1 << kDigit;

struct SampleArgs {
  const uint8_t* logits;  // [R][V] f32 or bf16
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int64_t* ids;
  int R, V;
};

// A row's logits in 16-byte groups at 16-byte aligned addresses (rows of odd length start anywhere):
// group g holds elements [g * VE - lead, + VE) of the row, those outside it as -inf, read one by one
// where a group is not the row's alone. NaN counts as -inf and -0 as +0.
template <bool BF>
struct Row {
  static constexpr int ES = BF ? 2 : 4, VE = 16 / ES;
  const uint8_t* p;
  int V, lead, groups;

  __device__ __forceinline__ Row(const SampleArgs& a, int r) {
    p = a.logits + (size_t)r * a.V * ES;
    V = a.V;
    lead = (int)((reinterpret_cast<uintptr_t>(p) & 15) / ES);
    groups = (lead + V + VE - 1) / VE;
  }
  static __device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (BF) return clean(npn::bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[e]));
    else return clean(reinterpret_cast<const float*>(p)[e]);
  }
  __device__ __forceinline__ int first(int g) const { return g * VE - lead; }
  __device__ __forceinline__ void load(int g, float (&x)[VE]) const {
    const int e0 = first(g);
    if (e0 >= 0 && e0 + VE <= V) {
      const uint4 q = *reinterpret_cast<const uint4*>(p + (ptrdiff_t)e0 * ES);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < VE; ++j)
        x[j] = clean(BF ? ((j & 1) ? npn::bf16hi(w[j >> 1]) : npn::bf16lo(w[j >> 1]))
                        : __uint_as_float(w[j & 3]));
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = e0 + j >= 0 && e0 + j < V ? at(e0 + j) : -INFINITY;
    }
  }
};

// Order-preserving key of a clean logit (no NaN, no -0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ ((uint32_t)(~(int)key >> 31) | 0x80000000u));
}

// exp((x - m) / T), 0 for -inf; in a row with m = +inf those at +inf share it all.
struct Weigh {
  float m;
  double inv;
  __device__ __forceinline__ double real(float x) const {
    if (x == m) return 1.0;
    if (x == -INFINITY || m == INFINITY) return 0.0;
    return exp(((double)x - (double)m) * inv);
  }
  __device__ __forceinline__ uint64_t fixed(float x) const { return (uint64_t)rint(real(x) * kOne); }
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return ((uint64_t)(uint32_t)__shfl_up((int)(v >> 32), d, 64) << 32) |
         (uint32_t)__shfl_up((int)(uint32_t)v, d, 64);
}

// Inclusive scan over the workgroup's threads.
__device__ __forceinline__ uint64_t scan64(uint64_t v, uint64_t* s_wave, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t o = shfl_up64(v, off);
    if (lane >= off) v += o;
  }
  __syncthreads();  // s_wave of an earlier scan has been read
  if (lane == 63) s_wave[w] = v;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    before += k < w ? s_wave[k] : 0;
    total += s_wave[k];
  }
  return v + before;
}

// floor(f x) and ceil(f x) for 0 <= f < 1: f in 64 fractional bits (exact down to f = 2^-40).
__device__ __forceinline__ uint64_t fraction(float f) {
  return (uint64_t)((double)f * 18446744073709551616.0);
}
__device__ __forceinline__ uint64_t floor_mul(float f, uint64_t x) { return __umul64hi(fraction(f), x); }
__device__ __forceinline__ uint64_t ceil_mul(float f, uint64_t x) {
  const uint64_t q = fraction(f);
  return __umul64hi(q, x) + (q * x != 0);
}
__device__ __forceinline__ float clean_u(float u) {  // [0, 1), NaN as 0
  return fminf(fmaxf(u, 0.0f), 0.99999994039535522f);
}

struct RowSmem {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t wave[kWaves];
  uint64_t found[4];
  uint32_t red_key[kWaves];
  int red_idx[kWaves];
};

// One workgroup finds a row's ranks by digits of the key: a level's histogram of counts and weights
// (of the tokens that share the digits found so far) is summed from the top bin until the target
// falls into a bin, 11 + 11 + 10 bits. Each level reads the row once.
template <bool BF>
struct RowSearch {
  const Row<BF>& row;
  const Weigh& weigh;
  RowSmem& sm;

  __device__ __forceinline__ void histogram(int level, uint32_t prefix) const {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      sm.count[b] = 0;
      sm.mass[b] = 0;
    }
    __syncthreads();
    const int low = level == 0 ? 21 : level == 1 ? 10 : 0;          // lowest bit of the digit
    const int high = level == 0 ? 32 : level == 1 ? 21 : 10;        // lowest bit of the prefix
    const uint32_t mask = level == 2 ? 1023u : 2047u;
    for (int g = threadIdx.x; g < row.groups; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j) {
        const uint32_t k = key_of(x[j]);
        if (level > 0 && k >> high != prefix) continue;
        const uint64_t w = weigh.fixed(x[j]);
        if (w == 0) continue;
        const uint32_t bin = (k >> low) & mask;
        atomicAdd(&sm.count[bin], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&sm.mass[bin]), (unsigned long long)w);
      }
    }
    __syncthreads();
  }

  // The bin, from the top, in which the running count (or weight) reaches target; the counts and
  // weights before it are added to `count` and `mass`. target is at most the bins' sum.
  __device__ __forceinline__ uint32_t pick(bool by_count, uint64_t target, uint64_t& count,
                                           uint64_t& mass) const {
    const int b0 = kBins - 1 - 2 * threadIdx.x;  // this thread's bins b0, b0 - 1
    uint64_t total;
    const uint64_t c = (uint64_t)sm.count[b0] + sm.count[b0 - 1], cs = scan64(c, sm.wave, total);
    const uint64_t w = sm.mass[b0] + sm.mass[b0 - 1], ws = scan64(w, sm.wave, total);
    const uint64_t mine = by_count ? c : w, upto = by_count ? cs : ws;
    if (upto >= target && upto - mine < target) {
      const uint64_t first = by_count ? (uint64_t)sm.count[b0] : sm.mass[b0];
      const bool second = upto - mine + first < target;
      sm.found[0] = b0 - second;
      sm.found[1] = cs - c + (second ? sm.count[b0] : 0);
      sm.found[2] = ws - w + (second ? sm.mass[b0] : 0);
    }
    __syncthreads();
    const uint32_t bin = (uint32_t)sm.found[0];
    count += sm.found[1];
    mass += sm.found[2];
    __syncthreads();
    return bin;
  }

  struct Rank {
    uint32_t key;
    uint64_t count, mass;  // of the tokens with larger keys
  };

  // `level0`: the histogram of the first digit is in LDS already.
  __device__ Rank find(bool by_count, uint64_t target, bool level0) const {
    Rank r{0, 0, 0};
    for (int level = 0; level < 3; ++level) {
      if (level > 0 || !level0) histogram(level, r.key);
      const uint64_t left = target - (by_count ? r.count : r.mass);
      const uint32_t bin = pick(by_count, left, r.count, r.mass);
      r.key = (r.key << (level == 2 ? 10 : kDigit)) | bin;
    }
    return r;
  }

  // Index of the n-th token (from 1) with this key, in index order.
  __device__ int nth(uint32_t key, uint64_t n) const {
    uint64_t before = 0;
    for (int g0 = 0; g0 < row.groups; g0 += kThreads) {
      const int g = g0 + threadIdx.x;
      uint32_t is = 0;
      if (g < row.groups) {
        float x[Row<BF>::VE];
        row.load(g, x);
#pragma unroll
        for (int j = 0; j < Row<BF>::VE; ++j) {
          const int e = row.first(g) + j;
          is |= (e >= 0 && e < row.V && key_of(x[j]) == key ? 1u : 0u) << j;
        }
      }
      uint64_t total;
      const uint64_t upto = before + scan64(__popc(is), sm.wave, total);
      if (upto >= n && upto - __popc(is) < n) {
        int skip = (int)(n - (upto - __popc(is))) - 1;
        while (skip-- > 0) is &= is - 1;
        sm.found[3] = row.first(g) + __ffs(is) - 1;
      }
      before += total;
      if (before >= n) break;  // the same for all threads
    }
    __syncthreads();
    return (int)sm.found[3];
  }
};

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
  __shared__ RowSmem sm;
  const int r = blockIdx.x;
  const Row<BF> row(a, r);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;

  // the maximum and its first index
  uint32_t key = 0;
  int idx = 0x7FFFFFFF;
  for (int g = threadIdx.x; g < row.groups; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
#pragma unroll
    for (int j = 0; j < Row<BF>::VE; ++j) {
      const uint32_t k = key_of(x[j]);
      if (k > key) {
        key = k;
        idx = row.first(g) + j;
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t ok = (uint32_t)__shfl_xor((int)key, off, 64);
    const int oi = __shfl_xor(idx, off, 64);
    if (ok > key || (ok == key && oi < idx)) {
      key = ok;
      idx = oi;
    }
  }
  if (lane == 0) {
    sm.red_key[wv] = key;
    sm.red_idx[wv] = idx;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWaves; ++k)
    if (sm.red_key[k] > key || (sm.red_key[k] == key && sm.red_idx[k] < idx)) {
      key = sm.red_key[k];
      idx = sm.red_idx[k];
    }
  const float m = logit_of(key), T = a.temperature[r];
  if (m == -INFINITY || !(T > 0.0f)) {  // nothing to sample, or greedy
    if (threadIdx.x == 0) a.ids[r] = m == -INFINITY ? -1 : idx;
    return;
  }
  const Weigh weigh{m, 1.0 / (double)T};
  const RowSearch<BF> search{row, weigh, sm};

  search.histogram(0, 0);
  uint64_t count, mass;
  scan64((uint64_t)sm.count[2 * threadIdx.x] + sm.count[2 * threadIdx.x + 1], sm.wave, count);
  scan64(sm.mass[2 * threadIdx.x] + sm.mass[2 * threadIdx.x + 1], sm.wave, mass);
  bool level0 = true;
  const int k = a.top_k[r];
  if (k > 0 && (uint64_t)k < count) {
    const auto f = search.find(true, (uint64_t)k, level0);
    mass = f.mass + ((uint64_t)k - f.count) * weigh.fixed(logit_of(f.key));
    level0 = false;
  }
  uint64_t kept = mass;
  const float p = a.top_p[r];
  if (p < 1.0f) {
    const uint64_t target = p > 0.0f ? max(ceil_mul(p, mass), (uint64_t)1) : 1;
    const auto f = search.find(false, target, level0);
    const uint64_t w = weigh.fixed(logit_of(f.key));
    kept = min(kept, f.mass + (target - f.mass + w - 1) / w * w);
    level0 = false;
  }
  if (a.min_p[r] > 0.0f) {
    const float mp = fminf(a.min_p[r], 1.0f);
    uint64_t sum = 0;
    for (int g = threadIdx.x; g < row.groups; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if (weigh.real(x[j]) >= (double)mp) sum += weigh.fixed(x[j]);
    }
    uint64_t total;
    scan64(sum, sm.wave, total);
    kept = min(kept, total);
  }
  const uint64_t target = floor_mul(clean_u(a.u[r]), kept) + 1;
  const auto f = search.find(false, target, level0);
  const uint64_t w = weigh.fixed(logit_of(f.key));
  const int id = search.nth(f.key, (target - f.mass + w - 1) / w);
  if (threadIdx.x == 0) a.ids[r] = id;
}

}  // namespace

extern "C" int npn_sample(const void* logits, int bf16, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          const float* u, int64_t* ids, int R, int V, void* stream) {
  NPN_REQUIRE(logits && temperature && top_k && top_p && min_p && u && ids, NPN_ERR_NULL);
  NPN_REQUIRE(R >= 1 && V >= 1 && V <= 1 << 20 && (bf16 == 0 || bf16 == 1), NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(logits), NPN_ERR_ALIGN);
  const SampleArgs a{static_cast<const uint8_t*>(logits), temperature, top_k, top_p, min_p, u, ids, R, V};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (bf16) hipLaunchKernelGGL(sample_rows_kernel<true>, dim3(R), dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(sample_rows_kernel<false>, dim3(R), dim3(kThreads), 0, s, a);
  return npn_launch_status();
}
