// Paged 8-bit KV cache for gfx950: the block tables' plan on the device, and the append of new
// K/V rows into e4m3 pages. (The attention over the pages is in paged_gqa.hip.)
//
// The cache: cache_k [N][Hkv][bs][256] and cache_v [N][Hkv][256][bs] OCP e4m3fn bytes -- V pages
// hold dims as rows, so that the attention's V^T operand is 16 contiguous keys per lane -- and one
// fp32 scale per (block, kv head) for each, always a power of two: value = e4m3 * scale, an exact
// bf16 number, and a page's older rows move to a larger scale by a shift of their exponent, exact
// except where e4m3 runs into its subnormals.
#include "npn_common.h"
#include "paged_append.h"

namespace {

using append::PagedAppendArgs;

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

// ---- the append (paged_append.h) --------------------------------------------------------------------
template <int RPW, int NW>
__global__ __launch_bounds__(NW * 64, 4) void paged_append_kernel(PagedAppendArgs a) {
  const int64_t kv = max(a.kv_len[blockIdx.z], 0);
  append::append_block<RPW, NW>(a, (int)blockIdx.x, (int)blockIdx.z, (int)blockIdx.y >> 1, blockIdx.y & 1,
                                [&](int t) { return kv + t; });
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
