// Paged 8-bit KV cache for gfx950: the block tables' plan on the device, and the append of new
// K/V rows into e4m3 pages. (The attention over the pages is in paged_gqa.hip.)
//
// The cache: cache_k [N][Hkv][bs][256] and cache_v [N][Hkv][256][bs] OCP e4m3fn bytes -- V pages
// hold dims as rows, so that the attention's V^T operand is 16 contiguous keys per lane -- and one
// fp32 scale per (block, kv head) for each, always a power of two: value = e4m3 * scale, an exact
// bf16 number, and a page's older rows move to a larger scale by a shift of their exponent, exact
// except where e4m3 runs into its subnormals.
#include "npn_common.h"

namespace {

constexpr int DH = 256;
constexpr int ROPE = 64;
constexpr float kEps = 1e-6f;
constexpr int kMinScaleExp = -100;  // the least scale is 2^-100: an all-zero page's

// ---- the block tables ---------------------------------------------------------------------------
//
// Request b holds blocks table[b][0, num_blocks[b]); the free blocks are a stack. One call moves
// every request to want_b = ceil((kv_len_b + n_b) / bs) blocks, n_b = new_len_b clamped to [0, T]:
//   give back   a request with more drops its blocks from want_b on (table entries become -1). The
//               stack grows by them with the last request's last block lowest, so giving back what
//               the previous call granted leaves the stack as it was before that call.
//   grant       then, in request order, a request with fewer takes its missing blocks off the top,
//               as long as the requests up to and including it need no more than there is (a
//               request that finds too few ends the granting for all after it that need any; one
//               that cannot fit its table row is refused and not counted). A refused request's
//               row and count stay, its slots are -1 and granted[b] is 0.
//   slots       slot[b][t] = block * bs + offset of position kv_len_b + t for t < granted[b], else -1.
// One workgroup: the prefix sums over the requests are its scans, and the block moves are dealt to
// its threads one block each by a search in those sums, so one long prompt does not hold up a
// thread. The slots go with it when there are few, else to a second launch over the whole chip.
struct PlanArgs {
  const int32_t* kv_len;
  const int32_t* new_len;
  int32_t* table;       // [B][P]
  int32_t* num_blocks;  // [B]
  int32_t* stack;       // [N]
  int32_t* free_count;  // [1]
  int64_t* slots;       // [B][T]
  int32_t* granted;     // [B]
  int B, P, N, T, sh;
  int slots_here;       // write the slots in the plan's launch
};

constexpr int kPlanThreads = 1024;

// Inclusive scan over the workgroup's kPlanThreads threads; s_wave holds one sum per wave.
__device__ __forceinline__ int plan_scan(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  __syncthreads();  // s_wave of an earlier scan has been read
  if (lane == 63) s_wave[w] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < kPlanThreads / 64; ++k) {
    before += k < w ? s_wave[k] : 0;
    total += s_wave[k];
  }
  return v + before;
}

struct Req {
  int kv, n, want, held;
};

__device__ __forceinline__ Req load_req(const PlanArgs& a, int b) {
  Req r{0, 0, 0, 0};
  if (b < a.B) {
    r.kv = max(a.kv_len[b], 0);
    r.n = min(max(a.new_len[b], 0), a.T);
    r.want = (int)(((int64_t)r.kv + r.n + (1 << a.sh) - 1) >> a.sh);
    r.held = min(max(a.num_blocks[b], 0), a.P);
  }
  return r;
}

// The request (index in this group of kPlanThreads) whose moves hold item i: the first with
// upto > i, upto the inclusive prefix sums.
__device__ __forceinline__ int find_req(const int* upto, int i) {
  int lo = 0, n = kPlanThreads;
  while (n > 1) {
    const int half = n >> 1;
    if (upto[lo + half - 1] <= i) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return lo;
}

__device__ __forceinline__ int64_t slot_of(const PlanArgs& a, int b, int t, int kv, int granted) {
  if (t >= granted) return -1;
  const int64_t pos = (int64_t)kv + t;
  return ((int64_t)a.table[(size_t)b * a.P + (pos >> a.sh)] << a.sh) + (pos & ((1 << a.sh) - 1));
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int s_wave[kPlanThreads / 64];
  __shared__ int s_upto[kPlanThreads];
  __shared__ int s_at[kPlanThreads];  // first entry of the request's row to move
  const int tid = threadIdx.x;
  const int count0 = min(max(a.free_count[0], 0), a.N);

  // blocks given back by all requests
  int given = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const Req r = load_req(a, b0 + tid);
    int total;
    plan_scan(max(r.held - r.want, 0), s_wave, total);
    given += total;
  }
  if (given > 0) {
    int run = 0;  // given back by earlier groups of requests
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
      const Req r = load_req(a, b0 + tid);
      const int mine = max(r.held - r.want, 0);
      int total;
      const int upto = plan_scan(mine, s_wave, total);
      s_upto[tid] = upto;
      s_at[tid] = r.want;
      __syncthreads();
      for (int i = tid; i < total; i += kPlanThreads) {
        const int q = find_req(s_upto, i);
        const int first = q > 0 ? s_upto[q - 1] : 0;
        int32_t* e = a.table + (size_t)(b0 + q) * a.P + s_at[q] + (i - first);
        const int64_t at = (int64_t)count0 + (given - 1 - (run + i));
        if (at < a.N) a.stack[at] = *e;
        *e = -1;
      }
      run += total;
      __syncthreads();
    }
  }
  const int count = (int)min((int64_t)count0 + given, (int64_t)a.N);

  // grants in request order
  int64_t asked = 0;  // needed by earlier groups of requests
  int taken = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const Req r = load_req(a, b);
    const bool room = r.want <= a.P;
    const int need = room ? max(r.want - r.held, 0) : 0;
    int total;
    const int upto = plan_scan(need, s_wave, total);
    const bool fits = room && (need == 0 || asked + upto <= count);
    int took;
    const int moved = plan_scan(fits ? need : 0, s_wave, took);
    s_upto[tid] = moved;
    s_at[tid] = r.held;
    __syncthreads();
    for (int i = tid; i < took; i += kPlanThreads) {
      const int q = find_req(s_upto, i);
      const int first = q > 0 ? s_upto[q - 1] : 0;
      a.table[(size_t)(b0 + q) * a.P + s_at[q] + (i - first)] = a.stack[count - 1 - (taken + i)];
    }
    taken += took;
    asked += total;
    if (b < a.B) {
      a.granted[b] = fits ? r.n : 0;
      a.num_blocks[b] = fits ? r.want : r.held;
    }
    __syncthreads();
  }
  if (tid == 0) a.free_count[0] = count - taken;
  if (a.slots_here) {  // the table and granted are this workgroup's own writes: visible after the barrier
    const int n = a.B * a.T;
    for (int i = tid; i < n; i += kPlanThreads) {
      const int b = i / a.T, t = i - b * a.T;
      a.slots[i] = slot_of(a, b, t, max(a.kv_len[b], 0), a.granted[b]);
    }
  }
}

// The slots of many tokens: grid (ceil(T / 512), B), two slots per thread and store.
__global__ __launch_bounds__(256) void paged_slots_kernel(PlanArgs a) {
  const int b = blockIdx.y;
  const int t = (blockIdx.x * 256 + threadIdx.x) * 2;
  if (t >= a.T) return;
  const int kv = max(a.kv_len[b], 0), granted = a.granted[b];
  const int64_t s0 = slot_of(a, b, t, kv, granted);
  int64_t* dst = a.slots + (size_t)b * a.T + t;
  if (t + 1 < a.T) {
    const int64_t s1 = slot_of(a, b, t + 1, kv, granted);
    if (NPN_ALIGNED16(dst)) {
      typedef long long i64x2 __attribute__((ext_vector_type(2)));
      *reinterpret_cast<i64x2*>(dst) = i64x2{s0, s1};
    } else {
      dst[0] = s0;
      dst[1] = s1;
    }
  } else {
    dst[0] = s0;
  }
}

// ---- the append -----------------------------------------------------------------------------------
//
// k = rope((1 + w) * key * rsqrt(mean key^2 + 1e-6)) in fp32 (no rounding before the page's own),
// v = value. For each (block, head) that gets rows: need = the least power of two with
// amax <= 448 * need over the new rows' finite values (at least 2^-100); the scale becomes need where
// the block's first row is new, else max(old, need), and older rows move to it; new rows are
// round-to-nearest-even e4m3(x / scale). NaN and infinities are stored as NaN and leave the scale.
//
// One workgroup of four waves per (request, block touched, head, K or V): it owns the page, so the
// scale and the older rows need no atomics. Lane l of a wave holds dims 4l..4l+3 of its rows in
// registers from the first load to the rounding (RPW rows per wave), so each input is read once.
struct PagedAppendArgs {
  const uint16_t* key;    // [B][T][Hkv][256]
  const uint16_t* value;
  const float* k_norm;
  const float* cos;       // [positions][64]
  const float* sin;
  const int32_t* kv_len;
  const int64_t* slots;   // [B][T]
  uint8_t* cache_k;
  uint8_t* cache_v;
  float* k_scale;         // [N][Hkv]
  float* v_scale;
  int B, T, Hkv, N, sh, positions;
};

__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7FFFFFu) <= 0x600000u ? 8 : 7);  // 448 = 1.75 * 2^8
  return __uint_as_float((uint32_t)(max(e, kMinScaleExp) + 127) << 23);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Four values / scale -> e4m3 bytes (|x| <= 448 scale where finite; the rest become NaN, 0x7F).
__device__ __forceinline__ uint32_t to_e4m3(const float* x, float inv) {
  float y[4];
  uint32_t nan = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool ok = finite(x[j]);
    y[j] = ok ? x[j] * inv : 0.f;
    nan |= ok ? 0u : 0x7Fu << (8 * j);
  }
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
  return (uint32_t)p | nan;
}

// e4m3 bytes times a power of two <= 1.
__device__ __forceinline__ uint32_t rescale_e4m3(uint32_t w, float by) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  const float x[4] = {lo[0], lo[1], hi[0], hi[1]};
  return to_e4m3(x, by);
}

template <int RPW>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
  const int b = blockIdx.z, h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int bs = 1 << a.sh;
  const int64_t* slots = a.slots + (size_t)b * a.T;

  // The rows [t0, t1) of this block: the request's first slot says where its blocks end.
  const int64_t first = slots[0];
  if (first < 0) return;
  const int off0 = (int)(first & (bs - 1));
  const int t0 = blockIdx.x == 0 ? 0 : bs - off0 + ((int)blockIdx.x - 1) * bs;
  if (t0 >= a.T) return;
  const int64_t slot = slots[t0];
  if (slot < 0 || slot >= (int64_t)a.N << a.sh) return;
  const int64_t block = slot >> a.sh;
  const int off = (int)(slot & (bs - 1));
  __shared__ int s_rows;
  if (threadIdx.x == 0) s_rows = min(bs - off, a.T - t0);
  __syncthreads();
  if ((int)threadIdx.x < min(bs - off, a.T - t0) && slots[t0 + threadIdx.x] != slot + threadIdx.x)
    atomicMin(&s_rows, (int)threadIdx.x);  // padding (or another block) begins here
  __syncthreads();
  const int rows = s_rows;

  // This wave's rows w, w + 4, ... of them.
  float x[RPW][4];
  const uint16_t* src = (is_v ? a.value : a.key) + (((size_t)b * a.T + t0) * a.Hkv + h) * DH + 4 * lane;
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = w + 4 * i;
    uint2 u = make_uint2(0u, 0u);
    if (r < rows) u = *reinterpret_cast<const uint2*>(src + (size_t)r * a.Hkv * DH);
    x[i][0] = npn::bf16lo(u.x);
    x[i][1] = npn::bf16hi(u.x);
    x[i][2] = npn::bf16lo(u.y);
    x[i][3] = npn::bf16hi(u.y);
  }
  float amax = 0.f;
  if (!is_v) {
    const float4 nw = *reinterpret_cast<const float4*>(a.k_norm + 4 * lane);
    const float wt[4] = {1.0f + nw.x, 1.0f + nw.y, 1.0f + nw.z, 1.0f + nw.w};
    const int64_t pos0 = (int64_t)a.kv_len[b] + t0;
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + 4 * i;
      if (r >= rows) break;  // wave-uniform
      const float ss = npn::wave_sum(x[i][0] * x[i][0] + x[i][1] * x[i][1] + x[i][2] * x[i][2] +
                                     x[i][3] * x[i][3]);
      const float rn = rsqrtf(ss * (1.0f / DH) + kEps);
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i][j] = wt[j] * (x[i][j] * rn);
        y[j] = __shfl_xor(x[i][j], 8, 64);  // dim d ^ 32
      }
      if (lane < ROPE / 4) {
        int64_t pos = pos0 + r;
        pos = pos < 0 ? 0 : (pos >= a.positions ? a.positions - 1 : pos);
        const float4 c = *reinterpret_cast<const float4*>(a.cos + pos * ROPE + 4 * lane);
        const float4 s = *reinterpret_cast<const float4*>(a.sin + pos * ROPE + 4 * lane);
        const float sg = lane < ROPE / 8 ? -1.0f : 1.0f;
        x[i][0] = x[i][0] * c.x + sg * y[0] * s.x;
        x[i][1] = x[i][1] * c.y + sg * y[1] * s.y;
        x[i][2] = x[i][2] * c.z + sg * y[2] * s.z;
        x[i][3] = x[i][3] * c.w + sg * y[3] * s.w;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) amax = fmaxf(amax, finite(x[i][j]) ? fabsf(x[i][j]) : 0.f);
  __shared__ float s_amax[4];
  amax = npn::wave_max(amax);
  if (lane == 0) s_amax[w] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(s_amax[0], s_amax[1]), fmaxf(s_amax[2], s_amax[3]));
  float* scale = (is_v ? a.v_scale : a.k_scale) + block * a.Hkv + h;
  const float need = scale_of(amax);
  const float old = off > 0 ? *scale : need;
  const float now = fmaxf(old, need);
  const bool grew = now > old;  // only where off > 0
  const float inv = 1.0f / now, by = old / now;
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0 && (off == 0 || grew)) *scale = now;

  if (!is_v) {
    uint8_t* page = a.cache_k + ((size_t)block * a.Hkv + h) * ((size_t)DH << a.sh) + 4 * lane;
    if (grew)
      for (int r = w; r < off; r += 4) {
        uint32_t* p = reinterpret_cast<uint32_t*>(page + (size_t)r * DH);
        *p = rescale_e4m3(*p, by);
      }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + 4 * i;
      if (r >= rows) break;
      *reinterpret_cast<uint32_t*>(page + (size_t)(off + r) * DH) = to_e4m3(x[i], inv);
    }
    return;
  }
  // V: the rows become columns. Bytes go through LDS as [dim][row] (16 bytes of padding per dim
  // keep the four-dim writes of a row off one bank), then thread d reads, changes and writes the
  // 16-row groups of dim d that hold new rows (or older ones, if the scale grew); the page is this
  // workgroup's alone, and bytes of rows that it does not touch go back as they were.
  constexpr int kStride = RPW * 4 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t s_v[DH * kStride];
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = w + 4 * i;
    if (r >= rows) break;
    const uint32_t q = to_e4m3(x[i], inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) s_v[(4 * lane + j) * kStride + r] = (uint8_t)(q >> (8 * j));
  }
  __syncthreads();
  const int d = threadIdx.x;
  uint8_t* page = a.cache_v + ((size_t)block * a.Hkv + h) * ((size_t)DH << a.sh) + ((size_t)d << a.sh);
  const uint8_t* sv = s_v + d * kStride;
  const int end = off + rows;
  for (int g = grew ? 0 : off & ~15; g < end; g += 16) {
    uint4 v = *reinterpret_cast<const uint4*>(page + g);
    uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r0 = g + 4 * k;
      const uint32_t moved = grew && r0 < off ? rescale_e4m3(word[k], by) : word[k];
      uint32_t out = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + j;
        uint32_t byte = ((r < off ? moved : word[k]) >> (8 * j)) & 0xFFu;
        if (r >= off && r < end) byte = sv[r - off];
        out |= byte << (8 * j);
      }
      word[k] = out;
    }
    *reinterpret_cast<uint4*>(page + g) = make_uint4(word[0], word[1], word[2], word[3]);
  }
}

}  // namespace

static int block_shift(int block_size) {
  switch (block_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

extern "C" int npn_paged_update_blocks(const int32_t* kv_len, const int32_t* new_len,
                                       int32_t* block_table, int32_t* num_blocks,
                                       int32_t* free_blocks, int32_t* free_count, int64_t* slots,
                                       int32_t* granted, int B, int max_blocks, int n_blocks,
                                       int block_size, int T, void* stream) {
  NPN_REQUIRE(kv_len && new_len && block_table && num_blocks && free_blocks && free_count &&
                  slots && granted, NPN_ERR_NULL);
  const int sh = block_shift(block_size);
  NPN_REQUIRE(sh >= 0 && B >= 1 && B <= 65535 && max_blocks >= 1 && n_blocks >= 1 && T >= 1,
              NPN_ERR_SHAPE);
  NPN_REQUIRE((int64_t)B * max_blocks <= (int64_t)1 << 30 && (int64_t)B * T <= (int64_t)1 << 30,
              NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(slots), NPN_ERR_ALIGN);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int here = (int64_t)B * T <= 4 * kPlanThreads;
  const PlanArgs a{kv_len, new_len, block_table, num_blocks, free_blocks, free_count, slots, granted,
                   B, max_blocks, n_blocks, T, sh, here};
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
  if (!here)
    hipLaunchKernelGGL(paged_slots_kernel, dim3((T + 511) / 512, B), dim3(256), 0, s, a);
  return npn_launch_status();
}

extern "C" int npn_gqa_kv_append_paged(const uint16_t* key, const uint16_t* value,
                                       const float* k_norm, const float* cos_table,
                                       const float* sin_table, int positions,
                                       const int32_t* kv_len, const int64_t* slots,
                                       int8_t* cache_k, int8_t* cache_v, float* k_scale,
                                       float* v_scale, int B, int T, int kv_heads, int n_blocks,
                                       int block_size, void* stream) {
  NPN_REQUIRE(key && value && k_norm && cos_table && sin_table && kv_len && slots && cache_k &&
                  cache_v && k_scale && v_scale, NPN_ERR_NULL);
  const int sh = block_shift(block_size);
  NPN_REQUIRE(sh >= 0 && B >= 1 && B <= 65535 && T >= 1 && T <= 1 << 24 && kv_heads >= 1 &&
                  kv_heads <= 1024 && n_blocks >= 1 && positions >= 1, NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(key) && NPN_ALIGNED16(value) && NPN_ALIGNED16(k_norm) &&
                  NPN_ALIGNED16(cos_table) && NPN_ALIGNED16(sin_table) && NPN_ALIGNED16(cache_k) &&
                  NPN_ALIGNED16(cache_v), NPN_ERR_ALIGN);
  const PagedAppendArgs a{key, value, k_norm, cos_table, sin_table, kv_len, slots,
                          reinterpret_cast<uint8_t*>(cache_k), reinterpret_cast<uint8_t*>(cache_v),
                          k_scale, v_scale, B, T, kv_heads, n_blocks, sh, positions};
  // A request's rows touch at most 1 + ceil((T - 1) / bs) blocks.
  const dim3 grid(1 + (T - 1 + block_size - 1) / block_size, 2 * kv_heads, B);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rpw = ((T < block_size ? T : block_size) + 3) / 4;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
  if (rpw <= 1) launch(paged_append_kernel<1>);
  else if (rpw <= 2) launch(paged_append_kernel<2>);
  else if (rpw <= 4) launch(paged_append_kernel<4>);
  else if (rpw <= 8) launch(paged_append_kernel<8>);
  else if (rpw <= 16) launch(paged_append_kernel<16>);
  else launch(paged_append_kernel<32>);
  return npn_launch_status();
}
