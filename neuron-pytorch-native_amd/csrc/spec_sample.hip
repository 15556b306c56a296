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
//  1. max: the row's maximum (and its first index, for greedy rows), its least finite logit, and the
//     maxima of G groups of lanes.
//  2. histogram over 2048 bins of equal width in (m - l) / T. Without a top-k of weights, whose running
//     sums say to within a bin where the top-p prefix ends, where min-p cuts and between which bins
//     the sample must lie. With one no weights are needed yet: counts of the groups' maxima where
//     they are more than k (the k-th largest of them is no more than the row's k-th largest logit, and
//     close to it, so the row itself is not read here), of the row's tokens up to a k of kCap.
//  3. collect: the tokens of the bins in question (all down to the k-th's bin, or the few bins of the
//     borders) go into a list of at most kCap.
//  4. finish: one workgroup sorts the list by rank, and with the bins' sums before each the three
//     ranks are exact. Where the maxima let too many tokens pass (large logits side by side in few
//     groups) the workgroup counts the row's tokens itself. A row whose list is too long all the same
//     (thousands of equal logits), or a longer top-k, is searched by the digits of its keys instead,
//     which reads it some ten times.
//
// Measured on 256 rows of 248320 bf16 logits (127 MB), settings mixed: 25 + 38 + 35 + 12 us for the four
// launches, where one reading takes 21 from HBM at 6.15 TB/s; on 32 rows of 151936 in float 7 + 11 + 13 +
// 11 us, on one 4.4 + 5.4 + 7 + 4.3. The first pass runs at 5.1 TB/s. The others are bound by instructions:
// three loads in flight instead of one made them slower (all rows without top-k: histogram 66 -> 110 us),
// while loads without the cleaning of NaN and -0, maxima by groups of 16 bytes, and one t for both weight
// and bin made them 1.3 times faster. Weights are the longest, 66 us when no row has a top-k, next the
// start of collect, some 6 us for each of the rounds that its workgroups run in.
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
  int R, V, C, G, gl;  // gl: log2 of a group's lanes
  float* cmax;      // [R][C] each chunk's maximum, its first group and the least finite logit
  int32_t* cgroup;
  float* cmin;
  float* tops;      // [R][G] maxima of the groups of lanes
  uint64_t* hist;   // [R][kBins] counts or weights
  RowState* state;    // [R] settings
  RowState* decided;  // [R] and the deciding bins
  int32_t* listed;  // [R] tokens that go on the list
  uint64_t* list;   // [R][kCap] inverted key above index: ascending is rank order
};

// A row's logits in 16-byte groups at 16-byte aligned addresses (rows of odd length start anywhere):
// group g holds elements [g * VE - lead, + VE) of the row, those outside it as -inf, read one by one
// where a group is not the row's alone. NaN counts as -inf and -0 as +0: clean() makes them so where
// comparisons do not by themselves.
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }

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
  __device__ __forceinline__ float at(int e) const {
    if constexpr (BF) return npn::bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[e]);
    else return reinterpret_cast<const float*>(p)[e];
  }
  __device__ __forceinline__ int first(int g) const { return g * VE - lead; }
  __device__ __forceinline__ void load(int g, float (&x)[VE]) const {
    const int e0 = first(g);
    if (e0 >= 0 && e0 + VE <= V) {
      const uint4 q = *reinterpret_cast<const uint4*>(p + (ptrdiff_t)e0 * ES);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < VE; ++j)
        x[j] = BF ? ((j & 1) ? npn::bf16hi(w[j >> 1]) : npn::bf16lo(w[j >> 1])) : __uint_as_float(w[j & 3]);
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = e0 + j >= 0 && e0 + j < V ? at(e0 + j) : -INFINITY;
    }
  }
  __device__ __forceinline__ void load_clean(int g, float (&x)[VE]) const {
    load(g, x);
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] = clean(x[j]);
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

// A token's weight is 2^(t/256), t = (x - m) 256 log2(e) / T, to 2^-51 relative: 2^(j/256) from the
// table by t's nearest whole number, times the series of e^r, |r| <= ln(2)/512, to r^4/24 (the next
// term is under 2^-54); the power's whole part goes into the exponent's bits. t is cut off at 2^-60,
// which weighs nothing; so do NaN and -inf.
constexpr int kTable = 256;
constexpr double kCut = -60.0 * kTable;

struct Weigh {
  float m;
  double c;             // 256 log2(e) / T
  const double* table;  // 2^(j/256)
  __device__ __forceinline__ double power(double t) const {
    constexpr double L = 0.69314718055994530942 / kTable;
    const double whole = rint(t), r = t - whole;
    const int n = (int)whole;
    double p = fma(r, L * L * L * L / 24, L * L * L / 6);
    p = fma(r, p, L * L / 2);
    p = fma(r, p, L);
    p = fma(r, p, 1.0);
    p *= table[n & (kTable - 1)];
    return __hiloint2double(__double2hiint(p) + (n >> 8) * (1 << 20), __double2loint(p));
  }
  // round(w 2^42): the sum with 2^52 has the integer in its low bits.
  __device__ __forceinline__ uint64_t fixed_at(double t) const {
    const double s = fma(power(t), kOne, 4503599627370496.0);
    return (uint64_t)(__double2hiint(s) & 0xFFFFF) << 32 | (uint32_t)__double2loint(s);
  }
  __device__ __forceinline__ double at(float x) const { return fmax(((double)x - (double)m) * c, kCut); }
  // In a row with m = +inf those at +inf share it all: what lies below is infinitely far off.
  __device__ __forceinline__ double real(float x) const { return power(x == m ? 0.0 : at(x)); }
  __device__ __forceinline__ uint64_t fixed(float x) const { return fixed_at(x == m ? 0.0 : at(x)); }
};

// The bin of a token at t, `per` (at most 0) bins for each -1 of it. Equal logits share a bin and larger
// ones never lie in a later one. The last bin has the rest, among it all that weighs nothing.
__device__ __forceinline__ int bin_of(double t, double per) { return (int)fmin(t * per, (double)(kBins - 1)); }

__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < kTable) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / kTable));
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
      row.load_clean(g, x);
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
        row.load_clean(g, x);
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
        row.load_clean(g, x);
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
// The larger of the lane's and the lane ^ off's maximum, the first group among equals, and their minima.
__device__ __forceinline__ void best_of(float& best, int& group, float& low, int off) {
  const float ob = __shfl_xor(best, off, 64);
  const int og = __shfl_xor(group, off, 64);
  if (ob > best || (ob == best && og < group)) {
    best = ob;
    group = og;
  }
  low = fminf(low, __shfl_xor(low, off, 64));
}

// The groups of chunk c of C.
template <bool BF>
__device__ __forceinline__ void chunk_of(const Row<BF>& row, int c, int C, int& g0, int& g1) {
  g0 = (int)((int64_t)row.groups * c / C);
  g1 = (int)((int64_t)row.groups * (c + 1) / C);
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ float s_best[kWaves], s_low[kWaves];
  __shared__ int s_group[kWaves];
  const int c = blockIdx.x, r = blockIdx.y;
  const Row<BF> row(a, r);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  for (int b = c * kThreads + threadIdx.x; b < kBins; b += a.C * kThreads) a.hist[(size_t)r * kBins + b] = 0;
  if (c == 0 && threadIdx.x == 0) a.listed[r] = 0;
  float best = -INFINITY, low = INFINITY;
  int group = 0x7FFFFFFF;
  for (int g = g0 + threadIdx.x; g < g1; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
    float most = x[0], least = x[0];  // NaN only where all are
#pragma unroll
    for (int j = 1; j < Row<BF>::VE; ++j) {
      most = fmaxf(most, x[j]);
      least = fminf(least, x[j]);
    }
    if (least == -INFINITY) {
      least = INFINITY;
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j) least = fminf(least, x[j] == -INFINITY ? INFINITY : x[j]);
    }
    if (most > best) {
      best = most;
      group = g;
    }
    low = fminf(low, least);
  }
#pragma unroll
  for (int step = 0; step < 6; ++step) {
    if (step == a.gl && (lane & ((1 << step) - 1)) == 0)
      a.tops[(size_t)r * a.G + ((c * kThreads + threadIdx.x) >> step)] = best;
    best_of(best, group, low, 1 << step);
  }
  if (lane == 0) {
    if (a.gl == 6) a.tops[(size_t)r * a.G + c * kWaves + wv] = best;
    s_best[wv] = best;
    s_group[wv] = group;
    s_low[wv] = low;
  }
  __syncthreads();
  if (wv == 0) {
    best = s_best[lane % kWaves];
    group = s_group[lane % kWaves];
    low = s_low[lane % kWaves];
#pragma unroll
    for (int step = 1; step < kWaves; step *= 2) best_of(best, group, low, step);
  }
  if (threadIdx.x == 0) {
    a.cmax[(size_t)r * a.C + c] = best;
    a.cgroup[(size_t)r * a.C + c] = group;
    a.cmin[(size_t)r * a.C + c] = low;
  }
}

// A row's settings, and the bins whose tokens decide, in up to three ranges, ascending and disjoint.
struct RowState {
  enum { kDone, kCounts, kWeights, kDigits, kTops };
  float m;
  int mode, ranges;
  int lo[3], hi[3];
  float least[3], most[3];  // the logits of each range's bins
  int k;
  float p, min_p, u;
  double c, per;
  uint64_t base[3];  // sum of the bins before each range
  uint64_t total;    // and of all; 0 where they are counts
  uint64_t above;    // of those whose tokens are all past min_p

  __device__ __forceinline__ int range_of(float x) const {
    return (ranges > 1 && x < least[0] ? 1 : 0) + (ranges > 2 && x < least[1] ? 1 : 0);
  }
};

// The row's settings, from its chunks, a lane per chunk: one wave. `group`: the first that holds the
// maximum.
__device__ __forceinline__ void row_settings(const SampleArgs& a, int r, RowState& o, int& group) {
  const float T = a.temperature[r];
  o.k = a.top_k[r];
  o.p = a.top_p[r];
  o.min_p = a.min_p[r];
  o.u = clean_u(a.u[r]);
  float m = -INFINITY, low = INFINITY;
  group = 0x7FFFFFFF;
  for (int c = threadIdx.x & 63; c < a.C; c += 64) {  // chunks ascend, so the first of equal maxima stays
    const size_t at = (size_t)r * a.C + c;
    if (a.cmax[at] > m) {
      m = a.cmax[at];
      group = a.cgroup[at];
    }
    low = fminf(low, a.cmin[at]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) best_of(m, group, low, off);
  o.m = m + 0.0f;
  o.ranges = 0;
  o.c = kTable * 1.4426950408889634074 / (double)T;
  // bins over what weighs something at all, or over the row's range where that is less
  const double range = fmin(kTable * ((double)kMaxExp + 1.0), ((double)m - (double)low) * o.c);
  o.per = range > 0.0 ? -fmin(kBins / range, 1e300) : 0.0;
  // At k = 3/4 of the groups a quarter of them has no token past the k-th maximum, so that they have ln 4 on
  // average: a list of 1.85 k, within kCap for k up to its half.
  const bool cut_k = o.k > 0 && o.k < a.V;
  o.mode = m == -INFINITY || !(T > 0.0f) ? RowState::kDone
           : m == INFINITY ? RowState::kDigits
           : !cut_k ? RowState::kWeights
           : o.k <= a.G - a.G / 4 && o.k <= kCap / 2 ? RowState::kTops
           : o.k <= kCap ? RowState::kCounts : RowState::kDigits;
}

// ---- 2. histogram -------------------------------------------------------------------------------------
struct BinSmem {
  uint64_t before[kBins];  // sums of the bins before each
  uint64_t wave[kWaves];
  int at[3], min_p[2];
};

// First bin whose running sum (with it) reaches the target (at least 1, at most the total), by the
// thread that has it, into *out.
__device__ __forceinline__ void reach(const uint64_t (&h)[2], uint64_t first, uint64_t target, int* out) {
  if (first < target && first + h[0] >= target) *out = 2 * threadIdx.x;
  else if (first + h[0] < target && first + h[0] + h[1] >= target) *out = 2 * threadIdx.x + 1;
}

// The logits that lie in each range's bins: a wave for each end finds, in six steps of 64 keys, the
// least key with a bin <= hi, or with one < lo (bins fall as keys rise).
__device__ __forceinline__ void range_logits(RowState& o) {
  const int end = threadIdx.x >> 6, lane = threadIdx.x & 63, g = end >> 1;
  if (g >= o.ranges) return;
  const int want = (end & 1) ? o.lo[g] - 1 : o.hi[g];
  const Weigh weigh{o.m, o.c, nullptr};
  const double per = o.per;
  uint32_t lo = key_of(-3.402823466e38f), hi = key_of(o.m) + 1;  // it is in [lo, hi]
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) / 64, key = lo + lane * step;
    const uint64_t in = __ballot(key >= hi || bin_of(weigh.at(logit_of(key)), per) <= want);
    const int j = in == 0 ? 64 : __ffsll((unsigned long long)in) - 1;
    hi = min(hi, lo + j * step);
    lo += j == 0 ? 0 : (j - 1) * step + 1;
  }
  if (lane == 0) {
    if (end & 1) o.most[g] = logit_of(lo - 1);
    else o.least[g] = logit_of(lo);
  }
}

// In collect every workgroup of a row does this for itself: once a row, by the last of the histogram's
// workgroups to arrive, the fence that its sums need cost 20 times the histogram.
// The deciding bins into o (in LDS), from this thread's bins 2 tid and 2 tid + 1.
__device__ __forceinline__ void decide(const uint64_t (&h)[2], RowState& o, BinSmem& sm) {
  const int tid = threadIdx.x;
  uint64_t total;
  const uint64_t first = scan64(h[0] + h[1], sm.wave, total) - h[0] - h[1];
  sm.before[2 * tid] = first;
  sm.before[2 * tid + 1] = first + h[0];
  if (tid < 3) sm.at[tid] = kBins - 1;
  __syncthreads();
  if (o.mode != RowState::kWeights) {  // everything down to the k-th token's bin (or all)
    if ((uint64_t)o.k <= total) reach(h, first, (uint64_t)o.k, &sm.at[0]);
    __syncthreads();
    if (tid == 0) {
      o.total = 0;
      o.above = 0;
      o.ranges = 1;
      o.lo[0] = 0;
      o.hi[0] = sm.at[0];
      o.base[0] = 0;
    }
    __syncthreads();
    range_logits(o);
    __syncthreads();
    return;
  }
  // The kept prefix's weight, between its bounds where a border's bin is all that is known, and with
  // it the bins that the sample may lie in.
  auto sum_to = [&](int bin) { return bin + 1 < kBins ? sm.before[bin + 1] : total; };
  uint64_t least = total, most = total;
  const bool by_p = o.p < 1.0f, by_min = o.min_p > 0.0f;
  if (by_p) reach(h, first, o.p > 0.0f ? max(ceil_mul(o.p, total), (uint64_t)1) : 1, &sm.at[0]);
  if (by_min && tid < 64) {  // w = min_p at -t = 256 log2(1 / min_p), give or take the roundings of t, w and bins
    const double per = -o.per, t = -kTable * log2((double)fminf(o.min_p, 1.0f));
    sm.min_p[0] = (int)fmin(fmax((t - 1e-9) * per * (1.0 - 1e-9) - 1e-9, 0.0), (double)(kBins - 1));
    sm.min_p[1] = (int)fmin((t + 1e-9) * per * (1.0 + 1e-9) + 1e-9, (double)(kBins - 1));
  }
  __syncthreads();
  if (by_p) {
    least = sm.before[sm.at[0]];
    most = sum_to(sm.at[0]);
  }
  const int m0 = by_min ? sm.min_p[0] : 0, m1 = by_min ? sm.min_p[1] : 0;
  if (by_min) {
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
  range_logits(o);
  __syncthreads();
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(SampleArgs a) {
  __shared__ double s_table[kTable];
  __shared__ uint64_t s_hist[kBins];
  __shared__ RowState s_state;
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  const Row<BF> row(a, r);
  if (tid < 64) {
    RowState o;
    int group;
    row_settings(a, r, o, group);
    if (tid == 0) s_state = o;
    if (c == 0 && tid == 0) {
      a.state[r] = o;
      if (o.mode == RowState::kDone) {
        int64_t id = -1;
        if (o.m != -INFINITY) {
          float x[Row<BF>::VE];
          row.load(group, x);
#pragma unroll
          for (int j = Row<BF>::VE - 1; j >= 0; --j)
            if (x[j] == o.m) id = row.first(group) + j;
        }
        a.ids[r] = id;
      }
    }
  }
  for (int b = tid; b < kBins; b += kThreads) s_hist[b] = 0;
  fill_table(s_table);
  __syncthreads();
  RowState& st = s_state;
  if (st.mode == RowState::kDone || st.mode == RowState::kDigits) return;
  const bool tops = st.mode == RowState::kTops, counts = st.mode == RowState::kCounts;
  if (tops && c != 0) return;
  const Weigh weigh{st.m, st.c, s_table};
  const double per = st.per;
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  if (tops) {
    for (int g = tid; g < a.G; g += kThreads) {
      const float x = a.tops[(size_t)r * a.G + g];
      if (x > -INFINITY) atomicAdd(reinterpret_cast<uint32_t*>(&s_hist[bin_of(weigh.at(x), per)]), 1u);
    }
  } else if (counts) {
    for (int g = g0 + tid; g < g1; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if (x[j] > -INFINITY) atomicAdd(reinterpret_cast<uint32_t*>(&s_hist[bin_of(weigh.at(x[j]), per)]), 1u);
    }
  } else {
    for (int g = g0 + tid; g < g1; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j0 = 0; j0 < Row<BF>::VE; j0 += 4) {
        double t[4];
        uint64_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t[j] = weigh.at(x[j0 + j]);
          w[j] = weigh.fixed_at(t[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (w[j] != 0)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[bin_of(t[j], per)]), (unsigned long long)w[j]);
      }
    }
  }
  __syncthreads();
  if (tops) {  // all of the row's counts are here
    __shared__ BinSmem s_bins;
    const uint64_t h[2] = {s_hist[2 * tid], s_hist[2 * tid + 1]};
    decide(h, st, s_bins);
    if (tid == 0) a.decided[r] = st;
    return;
  }
  unsigned long long* hist = reinterpret_cast<unsigned long long*>(a.hist + (size_t)r * kBins);
  for (int b = tid; b < kBins; b += kThreads) {
    if (a.C == 1) hist[b] = s_hist[b];
    else if (s_hist[b] != 0) atomicAdd(&hist[b], (unsigned long long)s_hist[b]);
  }
}

// ---- 3. collect ---------------------------------------------------------------------------------------
template <bool BF>
__global__ __launch_bounds__(kThreads, 8) void sample_collect_kernel(SampleArgs a) {
  // The workgroup's finds meet in LDS and go out together: their order does not matter, they are
  // sorted. More than kCap of them make the row's list too long whatever the others find.
  __shared__ uint64_t s_list[kCap];
  __shared__ int s_count, s_at;
  const int c = blockIdx.x, r = blockIdx.y;
  __shared__ BinSmem bins;
  __shared__ RowState st;
  const int mode = a.state[r].mode;
  if (mode == RowState::kDone || mode == RowState::kDigits) return;
  const bool tops = mode == RowState::kTops;
  const uint64_t* hist = a.hist + (size_t)r * kBins + 2 * threadIdx.x;
  const uint64_t h[2] = {tops ? 0 : hist[0], tops ? 0 : hist[1]};
  constexpr int kWords = sizeof(RowState) / 4;
  if (threadIdx.x < kWords)
    reinterpret_cast<uint32_t*>(&st)[threadIdx.x] =
        reinterpret_cast<const uint32_t*>(tops ? &a.decided[r] : &a.state[r])[threadIdx.x];
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  if (!tops) {
    decide(h, st, bins);
    if (c == 0 && threadIdx.x < kWords)
      reinterpret_cast<uint32_t*>(&a.decided[r])[threadIdx.x] = reinterpret_cast<const uint32_t*>(&st)[threadIdx.x];
  }
  float least[3], most[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    least[k] = k < st.ranges ? st.least[k] : INFINITY;  // none: empty
    most[k] = k < st.ranges ? st.most[k] : -INFINITY;
  }
  const bool one = st.ranges == 1;
  const Row<BF> row(a, r);
  int g0, g1;
  chunk_of(row, c, a.C, g0, g1);
  auto list = [&](float x, int e) {
    const int at = atomicAdd(&s_count, 1);
    if (at < kCap) s_list[at] = ((uint64_t)~key_of(x + 0.0f) << 32) | (uint32_t)e;
  };
  // Lanes whose group's maximum is too small have nothing to list.
  if (tops && !(a.tops[(size_t)r * a.G + ((c * kThreads + threadIdx.x) >> a.gl)] >= least[0]))
    g1 = g0;
  for (int g = g0 + threadIdx.x; g < g1; g += kThreads) {
    float x[Row<BF>::VE];
    row.load(g, x);
    if (one) {
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if (x[j] >= least[0] && x[j] <= most[0]) list(x[j], row.first(g) + j);
    } else {
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if ((x[j] >= least[0] && x[j] <= most[0]) || (x[j] >= least[1] && x[j] <= most[1]) ||
            (x[j] >= least[2] && x[j] <= most[2]))
          list(x[j], row.first(g) + j);
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
      union {
        uint64_t upto[kCap];  // weights up to and including each
        uint64_t other[kCap]; // items on their way
      };
      union {
        uint32_t start[kBins];
        uint64_t hist[kBins];  // a second look at a row
      };
      BinSmem bins;
    } s;
    RowSmem row;
  };
  uint64_t wave[kWaves];
  uint64_t skipped[3], end;
  int at, n, sub[3];
};

// The n items of `item` in ascending order (they differ), in place; all threads.
template <bool BF>
__device__ __forceinline__ void sort_items(FinishSmem& sm, const RowState& st, int V, int n) {
  uint64_t* item = sm.s.item;
  uint64_t* other = sm.s.other;
  const int tid = threadIdx.x;
  if (n <= 256) {  // each finds its rank
    uint64_t mine = 0;
    int rank = 0;
    if (tid < n) {
      mine = item[tid];
      for (int k = 0; k < n; ++k) rank += item[k] < mine;
    }
    __syncthreads();
    if (tid < n) item[rank] = mine;
    __syncthreads();
    return;
  }
  // By bins, as many over each of the listed ranges, then each finds its rank in its bin.
  const int bins = kBins / st.ranges;
  if (tid == 0) sm.at = 0;
  if (tid < st.ranges) {  // bins to a value where a range has few (a bf16 row's often have), by index
    const uint32_t values = (key_of(st.most[tid]) - key_of(st.least[tid])) / (BF ? 65536u : 1u) + 1;
    sm.sub[tid] = values != 0 && values <= (uint32_t)bins / 2 ? bins / (int)values : 0;  // 0: an empty range
  }
  for (int b = tid; b < kBins; b += kThreads) sm.s.start[b] = 0;
  __syncthreads();
  auto bin = [&](uint64_t item) {
    const float x = logit_of(~(uint32_t)(item >> 32));
    const int g = st.range_of(x);
    if (const int sub = sm.sub[g])
      return g * bins + (int)((key_of(st.most[g]) - key_of(x)) / (BF ? 65536u : 1u)) * sub +
             min(sub - 1, (int)((float)(uint32_t)item * ((float)sub / (float)V)));
    const float most = st.most[g], width = most - st.least[g];
    const float t = x == most ? 0.0f : fminf(most - x, 3.4e38f) * ((float)bins / fminf(width, 3.4e38f));
    return g * bins + (int)fminf(t, (float)(bins - 1));
  };
  constexpr int PER = kCap / kThreads;
  uint64_t mine[PER];
  int place[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int k = tid + j * kThreads;
    if (k < n) {
      mine[j] = item[k];
      place[j] = atomicAdd(&sm.s.start[bin(mine[j])], 1u);
      // A bin too full to be searched item by item (96 of 4096): as many compares as the steps below.
      if (place[j] * n > 400000) sm.at = 1;
    }
  }
  __syncthreads();
  const bool full = sm.at != 0;
  if (!full) {
    const uint32_t c0 = sm.s.start[2 * tid], c1 = sm.s.start[2 * tid + 1];
    uint64_t total;
    const uint32_t first = (uint32_t)scan64(c0 + c1, sm.wave, total) - c0 - c1;
    sm.s.start[2 * tid] = first;
    sm.s.start[2 * tid + 1] = first + c0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (tid + j * kThreads < n) other[sm.s.start[bin(mine[j])] + place[j]] = mine[j];
    __syncthreads();
    for (int k = tid; k < n; k += kThreads) {
      const uint64_t x = other[k];
      const int b = bin(x), from = sm.s.start[b], to = b + 1 < kBins ? (int)sm.s.start[b + 1] : n;
      int rank = from;
      for (int i = from; i < to; ++i) rank += other[i] < x;
      item[rank] = x;
    }
    __syncthreads();
    return;
  }
  // Bitonic; each wave keeps to its own share of the items wherever the step lies inside it, so only
  // the wide steps meet at a barrier.
  int size = 256;
  while (size < n) size *= 2;
  for (int k = n + tid; k < size; k += kThreads) item[k] = ~0ull;
  __syncthreads();
  const int share = max(size / kWaves, 64), wv = tid >> 6, lane = tid & 63;
  for (int len = 2; len <= size; len *= 2)
    for (int step = len / 2; step > 0; step /= 2) {
      if (step >= share) __syncthreads();
      if (wv * share < size)
        for (int k = (wv * share >> 1) + lane; k < ((wv + 1) * share >> 1); k += 64) {
          const int lo = 2 * k - (k & (step - 1)), hi = lo + step;
          const uint64_t x = item[lo], y = item[hi];
          if ((x > y) == ((lo & len) == 0)) {
            item[lo] = y;
            item[hi] = x;
          }
        }
      if (step >= share) __syncthreads();
      else __builtin_amdgcn_wave_barrier();
    }
  __syncthreads();
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a) {
  __shared__ double s_table[kTable];
  __shared__ FinishSmem sm;
  __shared__ RowState st;
  const int r = blockIdx.x, tid = threadIdx.x;
  int n = a.listed[r];
  const int mode = a.state[r].mode;
  if (mode == RowState::kDone) return;
  constexpr int kWords = sizeof(RowState) / 4;
  if (tid < kWords)
    reinterpret_cast<uint32_t*>(&st)[tid] =
        reinterpret_cast<const uint32_t*>(mode == RowState::kDigits ? &a.state[r] : &a.decided[r])[tid];
  fill_table(s_table);
  for (int k = tid; k < n && n <= kCap; k += kThreads) sm.s.item[k] = a.list[(size_t)r * kCap + k];
  __syncthreads();
  const Row<BF> row(a, r);
  const Weigh weigh{st.m, st.c, s_table};
  if (mode == RowState::kTops && n > kCap) {
    // The row's largest logits lie in few groups, so that the k-th of the maxima is too low: the tokens
    // down to the k-th's own bin, by this workgroup alone.
    for (int b = tid; b < kBins; b += kThreads) sm.s.hist[b] = 0;
    if (tid == 0) {
      st.mode = RowState::kCounts;
      sm.n = 0;
    }
    __syncthreads();
    for (int g = tid; g < row.groups; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j)
        if (x[j] > -INFINITY)
          atomicAdd(reinterpret_cast<uint32_t*>(&sm.s.hist[bin_of(weigh.at(x[j]), st.per)]), 1u);
    }
    __syncthreads();
    const uint64_t h[2] = {sm.s.hist[2 * tid], sm.s.hist[2 * tid + 1]};
    decide(h, st, sm.s.bins);
    for (int g = tid; g < row.groups; g += kThreads) {
      float x[Row<BF>::VE];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < Row<BF>::VE; ++j) {
        if (!(x[j] >= st.least[0])) continue;
        const int at = atomicAdd(&sm.n, 1);
        if (at < kCap) sm.s.item[at] = ((uint64_t)~key_of(x[j] + 0.0f) << 32) | (uint32_t)(row.first(g) + j);
      }
    }
    __syncthreads();
    n = sm.n;
  }
  if (n > kCap || mode == RowState::kDigits) {
    __syncthreads();
    const RowSearch<BF> search{row, weigh, sm.row};
    const int id = search.sample(st.k, st.p, st.min_p, st.u);
    if (tid == 0) a.ids[r] = id;
    return;
  }
  sort_items<BF>(sm, st, a.V, n);
  auto logit = [&](int k) { return logit_of(~(uint32_t)(sm.s.item[k] >> 32)); };
  // Running weights of the row: those of the list (kCap / kThreads tokens a thread), with what lies
  // before a token's range in place of the list's before it.
  auto range_of = [&](int k) { return st.range_of(logit(k)); };
  constexpr int PER = kCap / kThreads;
  uint64_t w[PER], sum = 0;
  const int own = n <= kThreads ? 1 : PER;  // tokens a thread
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int k = tid * own + j;
    w[j] = j < own && k < n ? weigh.fixed(logit(k)) : 0;
    sum += w[j];
  }
  uint64_t total;
  uint64_t run = scan64(sum, sm.wave, total) - sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int k = tid * own + j;
    if (j < own && k < n) {
      const int g = range_of(k);
      if (k == 0 || range_of(k - 1) != g) sm.skipped[g] = run;
      sm.s.upto[k] = run + w[j];
    }
    run += w[j];
  }
  if (tid == 0) sm.end = st.above;
  __syncthreads();
  if (st.total != 0) {  // bins of weights
    for (int k = tid; k < n; k += kThreads) {
      const int g = range_of(k);
      sm.s.upto[k] += st.base[g] - sm.skipped[g];
    }
    __syncthreads();
  }
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
  const uint64_t mass = mode == RowState::kWeights ? st.total : sm.s.upto[min(st.k, n) - 1];
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
  int C, G, gl;
  size_t o_idx, o_min, o_tops, o_hist, o_state, o_decided, o_listed, o_list, bytes;
};

constexpr int kRows = 2048;  // rows at a time: a row has 50 to 65 KB of workspace

SamplePlan sample_plan(int R, int V) {
  SamplePlan p{};
  if (R < 1 || V < 1 || V > 1 << 20 || R > 65535) return p;
  R = R < kRows ? R : kRows;
  // Workgroups per row: two per CU in all (what their registers let run at once), chunks of 4096 tokens at
  // least, a load or two a thread; and of many long rows chunks of 32768 at most, since greedy rows are
  // done at once: 256 rows of 248320 take 107 us so, 146 with 65536, 171 with 131072.
  p.C = max(1, max(min(512 / R, (V + 4095) / 4096), V / 32768));
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t chunks = up((size_t)R * p.C * 4);
  p.o_idx = chunks;
  p.o_min = 2 * chunks;
  p.gl = p.C <= 16 ? 2 : p.C <= 64 ? 4 : 6;  // at most 4096 groups
  p.G = p.C * (kThreads >> p.gl);
  p.o_tops = 3 * chunks;
  p.o_hist = p.o_tops + up((size_t)R * p.G * 4);
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
                       top_k + r0, top_p + r0, min_p + r0, u + r0, ids + r0, n, V, p.C, p.G, p.gl,
                       reinterpret_cast<float*>(ws), reinterpret_cast<int32_t*>(ws + p.o_idx),
                       reinterpret_cast<float*>(ws + p.o_min), reinterpret_cast<float*>(ws + p.o_tops),
                       reinterpret_cast<uint64_t*>(ws + p.o_hist),
                       reinterpret_cast<RowState*>(ws + p.o_state), reinterpret_cast<RowState*>(ws + p.o_decided),
                       reinterpret_cast<int32_t*>(ws + p.o_listed), reinterpret_cast<uint64_t*>(ws + p.o_list)};
    if (bf16) sample_launch<true>(a, static_cast<hipStream_t>(stream));
    else sample_launch<false>(a, static_cast<hipStream_t>(stream));
  }
  return npn_launch_status();
}
