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
// thread. The slots go with it when there are few (up to four to a thread), else to a second launch over
// the whole chip, which takes 4 us for 512 K slots. Bound by one workgroup's dependent loads, scans and
// searches: 5 us for a step of 64 requests, 13 for 256 prompts of up to 2048 tokens in blocks of 16.
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

// Moves i = 0 .. n - 1 of a group of requests, one a thread and four at a time in flight: a move's
// request is the first whose inclusive prefix sum `upto` passes i, its table entry counts from there.
// from(i, entry) is where the block's id lies, to(i, entry, id) takes it. (One at a time, 16384 blocks'
// searches and round trips to memory took 18 us.)
template <class From, class To>
__device__ __forceinline__ void move_blocks(const PlanArgs& a, const int* upto, const int* at, int b0, int n,
                                            From from, To to) {
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * kPlanThreads) {
    int i[4], q[4] = {0, 0, 0, 0};
    int32_t* entry[4];
    int32_t id[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) i[k] = min(i0 + k * kPlanThreads, n - 1);
#pragma unroll
    for (int half = kPlanThreads / 2; half > 0; half /= 2)
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] += upto[q[k] + half - 1] <= i[k] ? half : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int before = q[k] > 0 ? upto[q[k] - 1] : 0;
      entry[k] = a.table + (size_t)(b0 + q[k]) * a.P + at[q[k]] + (i[k] - before);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) id[k] = *from(i[k], entry[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + k * kPlanThreads < n) to(i[k], entry[k], id[k]);
  }
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
  const Req r0 = load_req(a, tid);  // kept: most batches have no request past these

  // blocks given back by all requests
  int given = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const Req r = b0 == 0 ? r0 : load_req(a, b0 + tid);
    int total;
    plan_scan(max(r.held - r.want, 0), s_wave, total);
    given += total;
  }
  if (given > 0) {
    int run = 0;  // given back by earlier groups of requests
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
      const Req r = b0 == 0 ? r0 : load_req(a, b0 + tid);
      const int mine = max(r.held - r.want, 0);
      int total;
      const int upto = plan_scan(mine, s_wave, total);
      s_upto[tid] = upto;
      s_at[tid] = r.want;
      __syncthreads();
      move_blocks(a, s_upto, s_at, b0, total, [&](int, int32_t* entry) { return entry; },
                  [&](int i, int32_t* entry, int32_t id) {
                    const int64_t at = (int64_t)count0 + (given - 1 - (run + i));
                    if (at < a.N) a.stack[at] = id;
                    *entry = -1;
                  });
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
    const Req r = b0 == 0 ? r0 : load_req(a, b);
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
    move_blocks(a, s_upto, s_at, b0, took, [&](int i, int32_t*) { return a.stack + (count - 1 - (taken + i)); },
                [&](int, int32_t* entry, int32_t id) { *entry = id; });
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
// One workgroup per (request, block touched, head, K or V): it owns the page, so the
// scale and the older rows need no atomics. Lane l of a wave holds dims 4l..4l+3 of its rows in
// registers from the first load to the rounding (RPW rows per wave), so each input is read once.
// 32 requests of one to eight rows take 5 us (a launch and one chain of loads), whether their pages' scales
// hold already or all grow, older rows moved with them; 4 x 4096 rows of 4 heads
// in blocks of 64 (101 MB read and written) 30 us, 3.4 TB/s, bound by instructions to a row and by a
// workgroup's rows all having to arrive before its scale is known: only then can it write. (Checks for
// infinities at each conversion: 36 us. Four waves a workgroup of 16 rows each: 62, and 16 of 4 rows,
// more of which fit a CU: 32. Blocks of 128 with 8 waves of 16 rows 43, with 16 of 8 rows 35.)
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

// Four values / scale -> e4m3 bytes (|x| <= 448 scale where finite; the rest become NaN, 0x7F). Where all
// of a wave's are finite, the checks, most of the instructions, are left out.
__device__ __forceinline__ uint32_t to_e4m3(const float* x, float inv, bool all_finite = false) {
  if (all_finite) {
    const int q = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, q, true);
  }
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

// Sum over the wave: inside 16-lane rows by DPP, then across them by gfx950's row swaps.
__device__ __forceinline__ float wave_sum_valu(float v) {
  v += __uint_as_float(npn::dpp32<npn::kDppStep[0]>(__float_as_uint(v)));
  v += __uint_as_float(npn::dpp32<npn::kDppStep[1]>(__float_as_uint(v)));
  v += __uint_as_float(npn::dpp32<npn::kDppStep[2]>(__float_as_uint(v)));
  v += __uint_as_float(npn::dpp32<npn::kDppStep[3]>(__float_as_uint(v)));
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// NW waves, RPW rows each: below 4 rows w, w + NW, ..; from 4 on blocks of four rows w, w + NW, .., whose 4 x 4
// bytes a lane turns from rows into dims in registers.
template <int RPW, int NW>
__global__ __launch_bounds__(NW * 64, 4) void paged_append_kernel(PagedAppendArgs a) {
  const int b = blockIdx.z, h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int bs = 1 << a.sh;
  const int64_t* slots = a.slots + (size_t)b * a.T;

  // The rows [t0, t1) of this block: the request's first slot says where its blocks end, also where
  // its block is none (id -1: a slot of -bs + its row). A request without rows has -1 throughout.
  const int64_t first = slots[0];
  const int off0 = (int)(first & (bs - 1));
  const int t0 = blockIdx.x == 0 ? 0 : bs - off0 + ((int)blockIdx.x - 1) * bs;
  if (t0 >= a.T || (first < 0 && slots[t0] < 0)) return;
  const int room = min(blockIdx.x == 0 ? bs - off0 : bs, a.T - t0);
  auto row_of = [&](int i) { return RPW < 4 ? w + NW * i : 4 * (w + NW * (i >> 2)) + (i & 3); };

  // This wave's rows, from the input once (those past the last one repeat it and go nowhere).
  uint2 in[RPW];
  const uint16_t* src = (is_v ? a.value : a.key) + (((size_t)b * a.T + t0) * a.Hkv + h) * DH + 4 * lane;
#pragma unroll
  for (int i = 0; i < RPW; ++i)
    in[i] = *reinterpret_cast<const uint2*>(src + (size_t)min(row_of(i), room - 1) * a.Hkv * DH);
  const int64_t slot = slots[t0];
  if (slot < 0 || slot >= (int64_t)a.N << a.sh) return;
  const int64_t block = slot >> a.sh;
  const int off = (int)(slot & (bs - 1));
  const int most = min(bs - off, room);
  float x[RPW][4];
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    x[i][0] = npn::bf16lo(in[i].x);
    x[i][1] = npn::bf16hi(in[i].x);
    x[i][2] = npn::bf16lo(in[i].y);
    x[i][3] = npn::bf16hi(in[i].y);
  }
  // Padding, or another block, may begin before the block ends.
  __shared__ int s_rows;
  __shared__ float s_amax[NW];
  if (threadIdx.x == 0) s_rows = most;
  __syncthreads();
  if ((int)threadIdx.x < most && slots[t0 + threadIdx.x] != slot + threadIdx.x)
    atomicMin(&s_rows, (int)threadIdx.x);
  __syncthreads();
  const int rows = s_rows;

  if (!is_v) {
    const float4 nw = *reinterpret_cast<const float4*>(a.k_norm + 4 * lane);
    const float wt[4] = {1.0f + nw.x, 1.0f + nw.y, 1.0f + nw.z, 1.0f + nw.w};
    const int64_t pos0 = (int64_t)max(a.kv_len[b], 0) + t0;
    constexpr int BATCH = RPW < 4 ? RPW : 4;  // rows whose RoPE rows are loaded at a time, without branches
#pragma unroll
    for (int i0 = 0; i0 < RPW; i0 += BATCH) {
      float4 c[BATCH], s[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        int64_t pos = pos0 + min(row_of(i0 + k), most - 1);
        pos = pos >= a.positions ? a.positions - 1 : pos;
        c[k] = *reinterpret_cast<const float4*>(a.cos + pos * ROPE + 4 * (lane & 15));
        s[k] = *reinterpret_cast<const float4*>(a.sin + pos * ROPE + 4 * (lane & 15));
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        float* v = x[i0 + k];
        const float ss = wave_sum_valu(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]);
        const float rn = rsqrtf(ss * (1.0f / DH) + kEps);
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = wt[j] * (v[j] * rn);
          y[j] = __uint_as_float(npn::dpp32<0x128>(__float_as_uint(v[j])));  // dim d ^ 32: 8 lanes round the 16
        }
        const float sg = lane < ROPE / 8 ? -1.0f : 1.0f;
        const float t[4] = {v[0] * c[k].x + sg * y[0] * s[k].x, v[1] * c[k].y + sg * y[1] * s[k].y,
                            v[2] * c[k].z + sg * y[2] * s[k].z, v[3] * c[k].w + sg * y[3] * s[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lane < ROPE / 4 ? t[j] : v[j];
      }
    }
  }
  float amax = 0.f, none = 0.f;
#pragma unroll
  for (int i = 0; i < RPW; ++i)
    if (row_of(i) < rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        amax = fmaxf(amax, fabsf(x[i][j]));
        none = fmaf(x[i][j], 0.0f, none);  // NaN from the first that is not finite
      }
    }
  const bool all_finite = __builtin_amdgcn_ballot_w64(none != none) == 0;
  if (!all_finite) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < RPW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        amax = fmaxf(amax, row_of(i) < rows && finite(x[i][j]) ? fabsf(x[i][j]) : 0.f);
  }
  amax = npn::wave_max(amax);
  if (lane == 0) s_amax[w] = amax;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NW; ++k) amax = fmaxf(amax, s_amax[k]);
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
      for (int r = w; r < off; r += NW) {
        uint32_t* p = reinterpret_cast<uint32_t*>(page + (size_t)r * DH);
        *p = rescale_e4m3(*p, by);
      }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = row_of(i);
      if (r < rows) *reinterpret_cast<uint32_t*>(page + (size_t)(off + r) * DH) = to_e4m3(x[i], inv, all_finite);
    }
    return;
  }
  // V: the rows become columns, through LDS as [dim][row]. Dim d lies in line 64 (d % 4) + d / 4, of an
  // odd number of words, so that a wave's writes of four rows (or one) of a dim a lane meet no bank
  // twice (or four times).
  constexpr int kLine = RPW < 4 ? (RPW * NW + 3) / 4 | 1 : RPW * NW / 4 + 1;  // words
  __shared__ uint32_t s_v[DH * kLine];
  uint8_t* bytes = reinterpret_cast<uint8_t*>(s_v);
  if constexpr (RPW < 4) {
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const uint32_t q = to_e4m3(x[i], inv, all_finite);
#pragma unroll
      for (int j = 0; j < 4; ++j) bytes[(64 * j + lane) * kLine * 4 + w + NW * i] = (uint8_t)(q >> (8 * j));
    }
  } else {
#pragma unroll
    for (int i = 0; i < RPW; i += 4) {
      const uint32_t q0 = to_e4m3(x[i], inv, all_finite), q1 = to_e4m3(x[i + 1], inv, all_finite);
      const uint32_t q2 = to_e4m3(x[i + 2], inv, all_finite), q3 = to_e4m3(x[i + 3], inv, all_finite);
      const uint32_t a0 = __builtin_amdgcn_perm(q1, q0, 0x05010400u);  // rows 0, 1 of dims 0, 1
      const uint32_t a1 = __builtin_amdgcn_perm(q1, q0, 0x07030602u);  // and of dims 2, 3
      const uint32_t b0 = __builtin_amdgcn_perm(q3, q2, 0x05010400u);
      const uint32_t b1 = __builtin_amdgcn_perm(q3, q2, 0x07030602u);
      const uint32_t d[4] = {__builtin_amdgcn_perm(b0, a0, 0x05040100u), __builtin_amdgcn_perm(b0, a0, 0x07060302u),
                             __builtin_amdgcn_perm(b1, a1, 0x05040100u), __builtin_amdgcn_perm(b1, a1, 0x07060302u)};
#pragma unroll
      for (int j = 0; j < 4; ++j) s_v[(64 * j + lane) * kLine + w + NW * (i >> 2)] = d[j];
    }
  }
  __syncthreads();
  // 16 rows of a dim at a time, all that hold new rows (or older ones, if the scale grew); neighbours
  // write neighbouring 16 bytes. The page is this workgroup's alone, and bytes of rows that it does
  // not touch go back as they were.
  uint8_t* page = a.cache_v + ((size_t)block * a.Hkv + h) * ((size_t)DH << a.sh);
  const int end = off + rows, g0 = grew ? 0 : off >> 4, groups = ((end + 15) >> 4) - g0;
  for (int k = threadIdx.x; k < DH * groups; k += NW * 64) {
    const int d = k / groups, g = (g0 + k - d * groups) * 16;
    const uint32_t* line = s_v + (64 * (d & 3) + (d >> 2)) * kLine;
    uint4* dst = reinterpret_cast<uint4*>(page + ((size_t)d << a.sh) + g);
    if (RPW >= 4 && g >= off && g + 16 <= end && (off & 3) == 0) {
      const uint32_t* v = line + ((g - off) >> 2);
      *dst = make_uint4(v[0], v[1], v[2], v[3]);
      continue;
    }
    const uint4 v = *dst;
    uint32_t word[4] = {v.x, v.y, v.z, v.w};
    const uint8_t* sv = reinterpret_cast<const uint8_t*>(line);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r0 = g + 4 * q;
      const uint32_t moved = grew && r0 < off ? rescale_e4m3(word[q], by) : word[q];
      uint32_t out = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + j;
        uint32_t byte = ((r < off ? moved : word[q]) >> (8 * j)) & 0xFFu;
        if (r >= off && r < end) byte = sv[r - off];
        out |= byte << (8 * j);
      }
      word[q] = out;
    }
    *dst = make_uint4(word[0], word[1], word[2], word[3]);
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
  // In a graph, without moves: 4.2 us for 512 slots in the plan's launch, 4.9 for 2048, 5.9 for 4096 and 7.8
  // for 8192; with a launch for them 5.8 for any of these.
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
  const int rows = T < block_size ? T : block_size;
  auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, s, a); };
  if (rows <= 4) launch(paged_append_kernel<1, 4>, 4);
  else if (rows <= 8) launch(paged_append_kernel<2, 4>, 4);
  else if (rows <= 16) launch(paged_append_kernel<4, 4>, 4);
  else if (rows <= 32) launch(paged_append_kernel<4, 8>, 8);
  else if (rows <= 64) launch(paged_append_kernel<8, 8>, 8);
  else launch(paged_append_kernel<8, 16>, 16);
  return npn_launch_status();
}
