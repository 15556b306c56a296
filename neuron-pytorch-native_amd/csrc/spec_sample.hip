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
//
// Four launches, C workgroups to a row in the first three:
//  1. max: the row's maximum (and its first index, for greedy rows) and least finite logit.
//  2. histogram over 2048 bins of equal width in (m - l) / T: counts where a top-k of at most kCap
//     applies (no exponentials are needed then), else weights, whose running sums say to within a bin
//     where the top-p prefix ends, where min-p cuts and between which bins the sample must lie.
//  3. collect: the tokens of the bins in question (all down to the k-th's bin, or the few bins of the
//     borders) go into a list of at most kCap.
//  4. finish: one workgroup sorts the list by rank, and with the bins' sums before each the three
//     ranks are exact. A row whose list is too long (thousands of equal logits), or a longer top-k, is
//     searched by the digits of its keys instead, which reads it some ten times.
#include "npn_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr double kOne = 4398046511104.0;  // 2^42
constexpr int kDigit = 11;                // bits of a key per level of the search by digits
constexpr int kBins = 1 << kDigit;
constexpr int kCap = 4096;                // list entries per row
constexpr float kMaxExp = 43.0f;          // weights below 2^-43 of the largest round to 0

struct RowState;
struct SampleArgs {
  const uint8_t* logits;  // [R][V] f32 or bf16
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int64_t* ids;
  int R, V, C;
  float* cmax;      // [R][C] each chunk's maximum, its first index and its least finite logit
  int32_t* cidx;
  float* cmin;
  uint64_t* hist;   // [R][kBins] counts or weights
  RowState* state;    // [R] settings
  RowState* decided;  // [R] and the deciding bins
  int32_t* listed;  // [R] tokens that go on the list
  uint64_t* list;   // [R][kCap] inverted key above index: ascending is rank order
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

// 2^(t/64) for t in [-60 * 64, 0], to 2^-51 relative: 2^(j/64) from the table by t's nearest whole
// number, times the series of e^r, |r| <= ln(2)/128, to r^5/120 (the next term is under 2^-54); the
// power's whole part goes into the exponent's bits.
__device__ __forceinline__ double exp2_64ths(double t, const double* table) {
  constexpr double L = 0.69314718055994530942 / 64;
  const double whole = rint(t), r = t - whole;
  const int n = (int)whole;
  double p = fma(r, L * L * L * L * L / 120, L * L * L * L / 24);
  p = fma(r, p, L * L * L / 6);
  p = fma(r, p, L * L / 2);
  p = fma(r, p, L);
  p = fma(r, p, 1.0);
  return __longlong_as_double(__double_as_longlong(p * table[n & 63]) + ((int64_t)(n >> 6) << 52));
}

// 2^((x - m) log2(e) / T), no less than 2^-60 (which weighs nothing). In a row with m = +inf those at
// +inf share it all: what lies below is infinitely far off.
struct Weigh {
  float m;
  double c64;           // 64 log2(e) / T
  const double* table;  // 2^(j/64)
  __device__ __forceinline__ double real(float x) const {
    const double d = x == m ? 0.0 : (double)x - (double)m;
    return exp2_64ths(fmax(d * c64, -60.0 * 64), table);
  }
  // round(w 2^42): the sum with 2^52 has the integer in its low bits.
  __device__ __forceinline__ uint64_t fixed(float x) const {
    return (uint64_t)__double_as_longlong(fma(real(x), kOne, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }
};

// The bin of a token x >= cut, `scale` bins per unit of m - x. Equal logits share a bin and larger ones
// never lie in a later one: that is all the bins have to be, so 32 bits do. The last bin has the rest,
// among it all that weighs nothing.
__device__ __forceinline__ int bin_of(float x, float m, float scale) {
  const float t = x == m ? 0.0f : fminf(m - x, 3.4e38f) * scale;
  return (int)fminf(t, (float)(kBins - 1));
}

__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x * 0.015625);
}

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

  // The row's token: top-k, top-p, min-p (as given) and a cleaned u.
  __device__ int sample(int k, float p, float min_p, float u) const {
    histogram(0, 0);
    uint64_t count, mass;
    scan64((uint64_t)sm.count[2 * threadIdx.x] + sm.count[2 * threadIdx.x + 1], sm.wave, count);
    scan64(sm.mass[2 * threadIdx.x] + sm.mass[2 * threadIdx.x + 1], sm.wave, mass);
    bool level0 = true;
    if (k > 0 && (uint64_t)k < count) {
      const auto f = find(true, (uint64_t)k, level0);
      mass = f.mass + ((uint64_t)k - f.count) * weigh.fixed(logit_of(f.key));
      level0 = false;
    }
    uint64_t kept = mass;
    if (p < 1.0f) {
      const uint64_t target = p > 0.0f ? max(ceil_mul(p, mass), (uint64_t)1) : 1;
      const auto f = find(false, target, level0);
      const uint64_t w = weigh.fixed(logit_of(f.key));
      kept = min(kept, f.mass + (target - f.mass + w - 1) / w * w);
      level0 = false;
    }
    if (min_p > 0.0f) {
      const float mp = fminf(min_p, 1.0f);
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
    const uint64_t target = floor_mul(u, kept) + 1;
    const auto f = find(false, target, level0);
    const uint64_t w = weigh.fixed(logit_of(f.key));
    return nth(f.key, (target - f.mass + w - 1) / w);
  }
};

// ---- 1. max -----------------------------------------------------------------------------------------
// The groups of chunk c of C.
template <bool BF>
__device__ __forceinline__ void chunk_of(const Row<BF>& row, int c, int C, int& g0, int& g1) {
  g0 = (int)((int64_t)row.groups * c / C);
  g1 = (int)((int64_t)row.groups * (c + 1) / C);
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ uint32_t s_key[kWaves];
  __shared__ int s_idx[kWaves];
  __shared__ float s_min[kWaves];
  const int c = blockIdx.x, r = blockIdx.y;
  const Row<BF> row(a, r);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  for (int b = c * kThreads + threadIdx.x; b < kBins; b += a.C * kThreads) a.hist[(size_t)r * kBins + b] = 0;
  if (c == 0 && threadIdx.x == 0) a.listed[r] = 0;
  uint32_t key = 0;
  int idx = 0x7FFFFFFF;
  float low = INFINITY;
  for (int g = g0 + threadIdx.x; g < g1; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
#pragma unroll
    for (int j = 0; j < Row<BF>::VE; ++j) {
      const uint32_t k = key_of(x[j]);
      if (k > key) {
        key = k;
        idx = row.first(g) + j;
      }
      low = fminf(low, x[j] == -INFINITY ? INFINITY : x[j]);
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
    low = fminf(low, __shfl_xor(low, off, 64));
  }
  if (lane == 0) {
    s_key[wv] = key;
    s_idx[wv] = idx;
    s_min[wv] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kWaves; ++k) {
      if (s_key[k] > key || (s_key[k] == key && s_idx[k] < idx)) {
        key = s_key[k];
        idx = s_idx[k];
      }
      low = fminf(low, s_min[k]);
    }
    a.cmax[(size_t)r * a.C + c] = key == 0 ? -INFINITY : logit_of(key);
    a.cidx[(size_t)r * a.C + c] = idx;
    a.cmin[(size_t)r * a.C + c] = low;
  }
}

// A row's settings, and the bins whose tokens decide, in up to three ranges, ascending and disjoint.
struct RowState {
  enum { kDone, kCounts, kWeights, kDigits };
  float m, cut, scale;
  int mode, ranges;
  int lo[3], hi[3];
  int k;
  float p, min_p, u;
  double c;
  uint64_t base[3];  // sum of the bins before each range
  uint64_t total;    // and of all
  uint64_t above;    // of those whose tokens are all past min_p
};

// The row's settings, from its chunks (every wave for itself, a lane per chunk); a row whose token is
// known by its maximum gets it.
__device__ __forceinline__ void row_settings(const SampleArgs& a, int r, RowState& o, int& id) {
  const float T = a.temperature[r];
  o.k = a.top_k[r];
  o.p = a.top_p[r];
  o.min_p = a.min_p[r];
  o.u = clean_u(a.u[r]);
  float m = -INFINITY, low = INFINITY;
  int idx = 0x7FFFFFFF;
  for (int c = threadIdx.x & 63; c < a.C; c += 64) {
    const size_t at = (size_t)r * a.C + c;
    const float v = a.cmax[at], w = a.cmin[at];
    const int i = a.cidx[at];
    if (v > m) {  // chunks ascend, so the first of equal maxima stays
      m = v;
      idx = i;
    }
    low = fminf(low, w);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float om = __shfl_xor(m, off, 64);
    const int oi = __shfl_xor(idx, off, 64);
    if (om > m || (om == m && oi < idx)) {
      m = om;
      idx = oi;
    }
    low = fminf(low, __shfl_xor(low, off, 64));
  }
  id = m == -INFINITY ? -1 : idx;
  o.m = m;
  o.cut = m == INFINITY ? INFINITY : -3.402823466e38f;
  o.ranges = 0;
  o.c = 1.4426950408889634074 / (double)T;
  // bins over what weighs something at all, or over the row's range where that is less
  const double range = fmin(((double)kMaxExp + 1.0) / o.c, (double)m - (double)low);
  o.scale = !(range > 0.0) || m == INFINITY ? 0.0f : (float)fmin(kBins / range, 3.4e38);
  const bool cut_k = o.k > 0 && o.k < a.V;
  o.mode = m == -INFINITY || !(T > 0.0f) ? RowState::kDone
           : !cut_k ? RowState::kWeights : o.k <= kCap ? RowState::kCounts : RowState::kDigits;
}

// ---- 2. histogram -------------------------------------------------------------------------------------
struct BinSmem {
  uint64_t before[kBins];  // sums of the bins before each
  uint64_t wave[kWaves];
  int at[4];
};

// First bin whose running sum (with it) reaches the target (at least 1, at most the total), by the
// thread that has it, into *out.
__device__ __forceinline__ void reach(const uint64_t (&h)[2], uint64_t first, uint64_t target, int* out) {
  if (first < target && first + h[0] >= target) *out = 2 * threadIdx.x;
  else if (first + h[0] < target && first + h[0] + h[1] >= target) *out = 2 * threadIdx.x + 1;
}

// The deciding bins into o (in LDS), from this thread's bins 2 tid and 2 tid + 1.
__device__ void decide(const uint64_t (&h)[2], RowState& o, BinSmem& sm) {
  const int tid = threadIdx.x;
  uint64_t total;
  const uint64_t first = scan64(h[0] + h[1], sm.wave, total) - h[0] - h[1];
  sm.before[2 * tid] = first;
  sm.before[2 * tid + 1] = first + h[0];
  if (tid < 4) sm.at[tid] = kBins - 1;
  __syncthreads();
  if (o.mode == RowState::kCounts) {  // everything down to the k-th token's bin (or all)
    if ((uint64_t)o.k <= total) reach(h, first, (uint64_t)o.k, &sm.at[0]);
    __syncthreads();
    if (tid == 0) {
      o.total = total;
      o.above = 0;
      o.ranges = 1;
      o.lo[0] = 0;
      o.hi[0] = sm.at[0];
      o.base[0] = 0;
    }
    __syncthreads();
    return;
  }
  // The kept prefix's weight, between its bounds where a border's bin is all that is known, and with
  // it the bins that the sample may lie in.
  auto sum_to = [&](int bin) { return bin + 1 < kBins ? sm.before[bin + 1] : total; };
  uint64_t least = total, most = total;
  const bool by_p = o.p < 1.0f, by_min = o.min_p > 0.0f;
  if (by_p) {
    reach(h, first, o.p > 0.0f ? max(ceil_mul(o.p, total), (uint64_t)1) : 1, &sm.at[0]);
    __syncthreads();
    least = sm.before[sm.at[0]];
    most = sum_to(sm.at[0]);
  }
  int m0 = 0, m1 = 0;
  if (by_min) {  // w = min_p at -y = log2(1 / min_p), give or take the roundings of y, w and bins
    const double per = (double)o.scale / o.c;  // bins per unit of y
    const double y = -log2((double)fminf(o.min_p, 1.0f));
    m0 = (int)fmin(fmax((y - 1e-14) * per * (1.0 - 1e-6) - 1e-6, 0.0), (double)(kBins - 1));
    m1 = (int)fmin((y + 1e-14) * per * (1.0 + 1e-6) + 1e-6, (double)(kBins - 1));
    least = min(least, sm.before[m0]);
    most = min(most, sum_to(m1));
  }
  reach(h, first, floor_mul(o.u, least) + 1, &sm.at[1]);
  reach(h, first, min(floor_mul(o.u, most) + 1, total), &sm.at[2]);
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    auto add = [&](int lo, int hi) {  // ascending by lo, touching ranges as one
      int k = n;
      for (; k > 0 && lo < o.lo[k - 1]; --k) {
        o.lo[k] = o.lo[k - 1];
        o.hi[k] = o.hi[k - 1];
      }
      o.lo[k] = lo;
      o.hi[k] = hi;
      ++n;
    };
    add(sm.at[1], sm.at[2]);
    if (by_p) add(sm.at[0], sm.at[0]);
    if (by_min) add(m0, m1);
    int k = 0;
    for (int i = 1; i < n; ++i) {
      if (o.lo[i] <= o.hi[k] + 1) {
        o.hi[k] = max(o.hi[k], o.hi[i]);
      } else {
        ++k;
        o.lo[k] = o.lo[i];
        o.hi[k] = o.hi[i];
      }
    }
    o.ranges = k + 1;
    for (int i = 0; i <= k; ++i) o.base[i] = sm.before[o.lo[i]];
    o.total = total;
    o.above = sm.before[m0];
  }
  __syncthreads();
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(SampleArgs a) {
  __shared__ double s_table[64];
  __shared__ uint64_t s_hist[kBins];
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  fill_table(s_table);
  RowState st;
  int id;
  row_settings(a, r, st, id);
  if (c == 0 && tid == 0) {
    a.state[r] = st;
    if (st.mode == RowState::kDone) a.ids[r] = id;
  }
  if (st.mode == RowState::kDone || st.mode == RowState::kDigits) return;
  const bool counts = st.mode == RowState::kCounts;
  for (int b = tid; b < kBins; b += kThreads) s_hist[b] = 0;
  __syncthreads();
  const Row<BF> row(a, r);
  const Weigh weigh{st.m, 64.0 * st.c, s_table};
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  for (int g = g0 + tid; g < g1; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
    if (counts) {
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if (x[j] >= st.cut)
          atomicAdd(reinterpret_cast<uint32_t*>(&s_hist[bin_of(x[j], st.m, st.scale)]), 1u);
    } else {
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j) {
        const uint64_t w = weigh.fixed(x[j]);
        if (w != 0)
          atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[bin_of(x[j], st.m, st.scale)]),
                    (unsigned long long)w);
      }
    }
  }
  __syncthreads();
  unsigned long long* hist = reinterpret_cast<unsigned long long*>(a.hist + (size_t)r * kBins);
  for (int b = tid; b < kBins; b += kThreads) {
    if (a.C == 1) hist[b] = s_hist[b];
    else if (s_hist[b] != 0) atomicAdd(&hist[b], (unsigned long long)s_hist[b]);
  }
}

// ---- 3. collect ---------------------------------------------------------------------------------------
template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_collect_kernel(SampleArgs a) {
  // The workgroup's finds meet in LDS and go out together: their order does not matter, they are
  // sorted. More than kCap of them make the row's list too long whatever the others find.
  __shared__ uint64_t s_list[kCap];
  __shared__ int s_count, s_at;
  const int c = blockIdx.x, r = blockIdx.y;
  __shared__ BinSmem bins;
  const uint64_t* hist = a.hist + (size_t)r * kBins + 2 * threadIdx.x;
  const uint64_t h[2] = {hist[0], hist[1]};
  const int mode = a.state[r].mode;
  if (mode != RowState::kCounts && mode != RowState::kWeights) return;
  __shared__ RowState st;
  if (threadIdx.x == 0) st = a.state[r];
  decide(h, st, bins);
  if (c == 0 && threadIdx.x == 0) a.decided[r] = st;
  const float m = st.m, cut = st.cut, scale = st.scale;
  uint32_t lo[3], width[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    lo[k] = k < st.ranges ? st.lo[k] : kBins;  // none: no bin is there
    width[k] = k < st.ranges ? st.hi[k] - st.lo[k] : 0;
  }
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  const Row<BF> row(a, r);
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  for (int g = g0 + threadIdx.x; g < g1; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < Row<BF>::VE; ++j) {
      const uint32_t b = (uint32_t)bin_of(x[j], m, scale);
      const bool on = x[j] >= cut && ((b - lo[0] <= width[0]) | (b - lo[1] <= width[1]) | (b - lo[2] <= width[2]));
      hits |= (on ? 1u : 0u) << j;
    }
    if (hits == 0) continue;
#pragma unroll
    for (int j = 0; j < Row<BF>::VE; ++j) {
      if (!(hits >> j & 1)) continue;
      const int at = atomicAdd(&s_count, 1);
      if (at < kCap) s_list[at] = ((uint64_t)~key_of(x[j]) << 32) | (uint32_t)(row.first(g) + j);
    }
  }
  __syncthreads();
  const int n = s_count;
  if (n == 0) return;
  if (threadIdx.x == 0) s_at = atomicAdd(&a.listed[r], n);
  __syncthreads();
  const int at = s_at;
  if (at + n > kCap) return;
  for (int k = threadIdx.x; k < n; k += kThreads) a.list[(size_t)r * kCap + at + k] = s_list[k];
}

// ---- 4. finish ----------------------------------------------------------------------------------------
struct FinishSmem {
  union {
    struct {
      uint64_t item[kCap];  // sorted: inverted key, index
      uint64_t upto[kCap];  // weights up to and including each
    } s;
    RowSmem row;
  };
  uint64_t wave[kWaves];
  uint64_t skipped[3], end;
  int at;
};

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a) {
  __shared__ double s_table[64];
  __shared__ FinishSmem sm;
  const int r = blockIdx.x, tid = threadIdx.x;
  __shared__ RowState st;
  const int n = a.listed[r], mode = a.state[r].mode;
  if (mode == RowState::kDone) return;
  if (tid == 0) st = mode == RowState::kDigits ? a.state[r] : a.decided[r];
  fill_table(s_table);
  __syncthreads();
  const Weigh weigh{st.m, 64.0 * st.c, s_table};
  if (n > kCap || mode == RowState::kDigits) {
    const Row<BF> row(a, r);
    const RowSearch<BF> search{row, weigh, sm.row};
    const int id = search.sample(st.k, st.p, st.min_p, st.u);
    if (tid == 0) a.ids[r] = id;
    return;
  }
  int size = 64;
  while (size < n) size *= 2;
  for (int k = tid; k < size; k += kThreads) sm.s.item[k] = k < n ? a.list[(size_t)r * kCap + k] : ~0ull;
  __syncthreads();
  // Bitonic; each wave keeps to its own share of the items wherever the step lies inside it, so only
  // the wide steps meet at a barrier.
  const int share = max(size / kWaves, 64), wv = tid >> 6, lane = tid & 63;
  for (int len = 2; len <= size; len *= 2)
    for (int step = len / 2; step > 0; step /= 2) {
      if (step >= share) __syncthreads();
      if (wv * share < size)
        for (int k = (wv * share >> 1) + lane; k < ((wv + 1) * share >> 1); k += 64) {
          const int lo = 2 * k - (k & (step - 1)), hi = lo + step;
          const uint64_t x = sm.s.item[lo], y = sm.s.item[hi];
          if ((x > y) == ((lo & len) == 0)) {
            sm.s.item[lo] = y;
            sm.s.item[hi] = x;
          }
        }
      if (step >= share) __syncthreads();
      else __builtin_amdgcn_wave_barrier();
    }
  __syncthreads();
  auto logit = [&](int k) { return logit_of(~(uint32_t)(sm.s.item[k] >> 32)); };
  // Running weights of the row: those of the list (kCap / kThreads tokens a thread), with what lies
  // before a token's range in place of the list's before it.
  auto range_of = [&](int k) {
    const int b = bin_of(logit(k), st.m, st.scale);
    return (st.ranges > 1 && b >= st.lo[1] ? 1 : 0) + (st.ranges > 2 && b >= st.lo[2] ? 1 : 0);
  };
  constexpr int PER = kCap / kThreads;
  uint64_t w[PER], sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int k = tid * PER + j;
    w[j] = k < n ? weigh.fixed(logit(k)) : 0;
    sum += w[j];
  }
  uint64_t total;
  uint64_t run = scan64(sum, sm.wave, total) - sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int k = tid * PER + j;
    if (k < n) {
      const int g = range_of(k);
      if (k == 0 || range_of(k - 1) != g) sm.skipped[g] = run;
      sm.s.upto[k] = run + w[j];
    }
    run += w[j];
  }
  if (tid == 0) sm.end = st.above;
  __syncthreads();
  for (int k = tid; k < n; k += kThreads) {
    const int g = range_of(k);
    sm.s.upto[k] += st.base[g] - sm.skipped[g];
  }
  __syncthreads();
  // First listed token whose running weight reaches x.
  auto rank_of = [&](uint64_t x) {
    if (tid == 0) sm.at = n - 1;
    __syncthreads();
    for (int k = tid; k < n; k += kThreads)
      if (sm.s.upto[k] >= x && (k == 0 || sm.s.upto[k - 1] < x)) sm.at = k;
    __syncthreads();
    const int k = sm.at;
    __syncthreads();
    return k;
  };
  const uint64_t mass = mode == RowState::kCounts ? sm.s.upto[min(st.k, n) - 1] : st.total;
  uint64_t kept = mass;
  if (st.p < 1.0f)
    kept = min(kept, sm.s.upto[rank_of(st.p > 0.0f ? max(ceil_mul(st.p, mass), (uint64_t)1) : 1)]);
  if (st.min_p > 0.0f) {  // the last listed token past min_p ends that prefix, or the bins before all that may
    const double least = (double)fminf(st.min_p, 1.0f);
    for (int k = tid; k < n; k += kThreads)
      if (weigh.real(logit(k)) >= least && (k + 1 == n || weigh.real(logit(k + 1)) < least))
        atomicMax(reinterpret_cast<unsigned long long*>(&sm.end), (unsigned long long)sm.s.upto[k]);
    __syncthreads();
    kept = min(kept, sm.end);
  }
  const int at = rank_of(floor_mul(st.u, kept) + 1);
  if (tid == 0) a.ids[r] = (int64_t)(uint32_t)sm.s.item[at];
}

struct SamplePlan {
  int C;
  size_t o_idx, o_min, o_hist, o_state, o_decided, o_listed, o_list, bytes;
};

constexpr int kRows = 2048;  // rows at a time: a row has 48 KB of workspace

SamplePlan sample_plan(int R, int V) {
  SamplePlan p{};
  if (R < 1 || V < 1 || V > 1 << 20 || R > 65535) return p;
  R = R < kRows ? R : kRows;
  // Workgroups per row: two per CU in all, and more of at most 32768 tokens each (rows differ in cost), chunks of 4096 tokens at least.
  p.C = max(1, max(min(512 / R, (V + 4095) / 4096), V / 32768));
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t chunks = up((size_t)R * p.C * 4);
  p.o_idx = chunks;
  p.o_min = 2 * chunks;
  p.o_hist = 3 * chunks;
  p.o_state = p.o_hist + (size_t)R * kBins * 8;
  p.o_decided = p.o_state + up((size_t)R * sizeof(RowState));
  p.o_listed = p.o_decided + up((size_t)R * sizeof(RowState));
  p.o_list = p.o_listed + up((size_t)R * 4);
  p.bytes = p.o_list + (size_t)R * kCap * 8;
  return p;
}

template <bool BF>
void sample_launch(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(a.C, a.R), block(kThreads);
  hipLaunchKernelGGL(sample_max_kernel<BF>, grid, block, 0, s, a);
  hipLaunchKernelGGL(sample_hist_kernel<BF>, grid, block, 0, s, a);
  hipLaunchKernelGGL(sample_collect_kernel<BF>, grid, block, 0, s, a);
  hipLaunchKernelGGL(sample_finish_kernel<BF>, dim3(a.R), block, 0, s, a);
}

}  // namespace

extern "C" size_t npn_sample_workspace_size(int R, int V) { return sample_plan(R, V).bytes; }

extern "C" int npn_sample(const void* logits, int bf16, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          const float* u, int64_t* ids, int R, int V, void* workspace,
                          size_t workspace_bytes, void* stream) {
  NPN_REQUIRE(logits && temperature && top_k && top_p && min_p && u && ids, NPN_ERR_NULL);
  const SamplePlan p = sample_plan(R, V);
  NPN_REQUIRE(p.bytes != 0 && (bf16 == 0 || bf16 == 1), NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(logits) && NPN_ALIGNED16(workspace), NPN_ERR_ALIGN);
  NPN_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes, NPN_ERR_WORKSPACE);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  for (int r0 = 0; r0 < R; r0 += kRows) {
    const int n = R - r0 < kRows ? R - r0 : kRows;
    const SampleArgs a{static_cast<const uint8_t*>(logits) + (size_t)r0 * V * (bf16 ? 2 : 4), temperature + r0,
                       top_k + r0, top_p + r0, min_p + r0, u + r0, ids + r0, n, V, p.C,
                       reinterpret_cast<float*>(ws), reinterpret_cast<int32_t*>(ws + p.o_idx),
                       reinterpret_cast<float*>(ws + p.o_min), reinterpret_cast<uint64_t*>(ws + p.o_hist),
                       reinterpret_cast<RowState*>(ws + p.o_state), reinterpret_cast<RowState*>(ws + p.o_decided),
                       reinterpret_cast<int32_t*>(ws + p.o_listed), reinterpret_cast<uint64_t*>(ws + p.o_list)};
    if (bf16) sample_launch<true>(a, static_cast<hipStream_t>(stream));
    else sample_launch<false>(a, static_cast<hipStream_t>(stream));
  }
  return npn_launch_status();
}
