// After a tree's walk: the accepted path's K/V rows to the front of the tree's rows in the e4m3 pages
// (paged_kv.hip has their layout), in all layers at once. Node t's row lies at slots[b][t]; row path[b][d]
// goes to slots[b][d]. path[d] >= d, so rows only move forward, over rejected nodes' rows or others that move.
//
// A page's scale is the page's own: a row that comes from a page of another scale is rounded to its new
// page's, which grows first where the row needs it (as an append's does), the page's older rows with it.
//
// One workgroup per (layer, request, head, K or V): all rows that move go through its LDS before the first
// is written, since one row's place is another's source. Bound by a chain of loads: path and slots, scales
// and rows.
#include "paged_append.h"
#include "tree.h"

namespace {

using append::DH;

constexpr int kCompactLayers = 32;
constexpr int kCompactThreads = 256;
static_assert(kCompactThreads == DH, "a thread for each dim of V");

struct CompactArgs {
  uint8_t* cache_k[kCompactLayers];
  uint8_t* cache_v[kCompactLayers];
  float* k_scale[kCompactLayers];
  float* v_scale[kCompactLayers];
  const int32_t* path;   // [B][T]
  const int64_t* slots;  // [B][T]
  int T, Hkv, N, sh;
};

__global__ __launch_bounds__(kCompactThreads) void paged_compact_kernel(CompactArgs a) {
  constexpr int kRows = npn::kMaxNodes, kWaves = kCompactThreads / 64;
  __shared__ uint32_t s_row[kRows][DH / 4];  // the rows that move
  __shared__ int64_t s_src[kRows], s_dst[kRows];
  __shared__ float s_by[kRows];
  __shared__ int s_max[kRows];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int h = blockIdx.x >> 1, b = blockIdx.y, layer = blockIdx.z;
  const bool is_v = blockIdx.x & 1;
  const int bs = 1 << a.sh;

  // Every wave has the whole path, lane d its row d.
  const int64_t end = (int64_t)a.N << a.sh;
  const size_t at = (size_t)b * a.T + lane;
  const int node = lane < a.T ? a.path[at] : -1;
  const int64_t dst = lane < a.T ? a.slots[at] : -1;
  const int64_t src = (int64_t)npn::shfl64(dst, min(max(node, 0), a.T - 1));
  const int n = npn::path_length(node, a.T, lane, dst >= 0 && dst < end && src >= 0 && src < end);
  const bool row = lane < n, moves = row && src != dst;
  const uint64_t moving = __builtin_amdgcn_ballot_w64(moves);
  if (moving == 0) return;  // the same in all waves
  const int m = __popcll(moving), mine = __popcll(moving & ((1ull << lane) - 1));  // of those that move
  float* scale = is_v ? a.v_scale[layer] : a.k_scale[layer];
  uint8_t* cache = is_v ? a.cache_v[layer] : a.cache_k[layer];
  const int64_t dst_page = dst >> a.sh;
  const float s_old = row ? scale[(src >> a.sh) * a.Hkv + h] : 0.f;  // of the row where it lies
  const float d_old = row ? scale[dst_page * a.Hkv + h] : 0.f;       // and of the page that it goes to
  // Byte offset of a slot's row (K), of its place in the first dim's line (V).
  auto place = [&](int64_t slot) {
    return ((slot >> a.sh) * a.Hkv + h) * ((int64_t)DH << a.sh) +
           (is_v ? (slot & (bs - 1)) : (slot & (bs - 1)) * DH);
  };
  if (w == 0 && moves) {
    s_src[mine] = place(src);
    s_dst[mine] = place(dst);
  }
  __syncthreads();
  uint8_t* bytes = reinterpret_cast<uint8_t*>(s_row);
  constexpr int kBatch = 8;  // loads in flight
  if (!is_v) {
    for (int i0 = w; i0 < m; i0 += kBatch * kWaves) {
      uint32_t x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        x[j] = *reinterpret_cast<const uint32_t*>(cache + s_src[min(i0 + j * kWaves, m - 1)] + 4 * lane);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kWaves < m) s_row[i0 + j * kWaves][lane] = x[j];
    }
  } else {
    for (int i0 = 0; i0 < m; i0 += kBatch) {
      uint8_t x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) x[j] = cache[s_src[min(i0 + j, m - 1)] + ((int64_t)tid << a.sh)];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j < m) bytes[(i0 + j) * DH + tid] = x[j];
    }
  }
  __syncthreads();

  // The pages' new scales. Where no row comes from a larger one they stay.
  float now = d_old;
  if (__builtin_amdgcn_ballot_w64(moves && s_old > d_old) != 0) {
    for (int i = w; i < m; i += kWaves) {
      const uint32_t x = s_row[i][lane];
      int big = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int mag = (int)(x >> (8 * j)) & 0x7F;
        big = max(big, mag == 0x7F ? 0 : mag);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) big = max(big, __shfl_xor(big, off, 64));
      if (lane == 0) s_max[i] = big;
    }
    __syncthreads();
    float need = 0.f;
    if (moves) {
      const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(s_max[mine], false);
      need = v[0] > 0.f ? append::scale_of(v[0] * s_old) : 0.f;
    }
    uint64_t left = __builtin_amdgcn_ballot_w64(row);
    while (left != 0) {  // page by page
      const bool here = row && dst_page == (int64_t)npn::shfl64(dst_page, __builtin_ctzll(left));
      const float top = npn::wave_max(here ? fmaxf(d_old, need) : 0.f);
      if (here) now = top;
      left &= ~__builtin_amdgcn_ballot_w64(here);
    }
  }
  if (w == 0 && moves) s_by[mine] = s_old / now;
  uint64_t grown = __builtin_amdgcn_ballot_w64(row && now > d_old);
  __syncthreads();  // rows, factors and old scales have been read
  while (grown != 0) {  // a grown page's rows up to the path's last in it move to the new scale
    const int first = __builtin_ctzll(grown);
    const int64_t page = (int64_t)npn::shfl64(dst_page, first);
    const bool here = row && dst_page == page;
    const uint64_t in = __builtin_amdgcn_ballot_w64(here);
    const int last = 63 - __builtin_clzll(in);
    const int upto = (int)(npn::shfl64(dst, last) & (bs - 1));
    const float by = __shfl(d_old, first, 64) / __shfl(now, first, 64);
    uint8_t* p = cache + (page * a.Hkv + h) * ((int64_t)DH << a.sh);
    if (!is_v) {
      for (int r = w; r <= upto; r += kWaves) {
        uint32_t* word = reinterpret_cast<uint32_t*>(p + (size_t)r * DH) + lane;
        *word = append::rescale_e4m3(*word, by);
      }
    } else {
      for (int r = 0; r <= upto; r += 4) {
        uint32_t* word = reinterpret_cast<uint32_t*>(p + ((size_t)tid << a.sh) + r);
        const uint32_t keep = upto - r >= 3 ? 0u : ~0u << (8 * (upto - r + 1));
        *word = (*word & keep) | (append::rescale_e4m3(*word, by) & ~keep);
      }
    }
    if (tid == first) scale[page * a.Hkv + h] = now;
    grown &= ~in;
  }
  __syncthreads();  // the rows that move are written over those
  if (!is_v) {
    for (int i = w; i < m; i += kWaves) {
      const uint32_t x = s_row[i][lane];
      const float by = s_by[i];
      *reinterpret_cast<uint32_t*>(cache + s_dst[i] + 4 * lane) = by == 1.0f ? x : append::rescale_e4m3(x, by);
    }
  } else {
    for (int i = 0; i < m; ++i) {
      const uint32_t x = bytes[i * DH + tid];
      const float by = s_by[i];
      cache[s_dst[i] + ((int64_t)tid << a.sh)] = (uint8_t)(by == 1.0f ? x : append::rescale_e4m3(x, by));
    }
  }
}

}  // namespace

extern "C" int npn_gqa_compact_paged(const int32_t* path, const int64_t* slots, int8_t* const* cache_k,
                                     int8_t* const* cache_v, float* const* k_scale, float* const* v_scale,
                                     int layers, int B, int T, int kv_heads, int n_blocks, int block_size,
                                     void* stream) {
  NPN_REQUIRE(path && slots && (layers == 0 || (cache_k && cache_v && k_scale && v_scale)), NPN_ERR_NULL);
  const int sh = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : block_size == 128 ? 7 : -1;
  NPN_REQUIRE(sh >= 0 && layers >= 0 && B >= 1 && B <= 65535 && T >= 1 && T <= npn::kMaxNodes &&
                  kv_heads >= 1 && kv_heads <= 1024 && n_blocks >= 1,
              NPN_ERR_SHAPE);
  for (int l = 0; l < layers; ++l) {
    NPN_REQUIRE(cache_k[l] && cache_v[l] && k_scale[l] && v_scale[l], NPN_ERR_NULL);
    NPN_REQUIRE(NPN_ALIGNED16(cache_k[l]) && NPN_ALIGNED16(cache_v[l]), NPN_ERR_ALIGN);
    for (int k = 0; k < l; ++k) NPN_REQUIRE(cache_k[k] != cache_k[l] && cache_v[k] != cache_v[l], NPN_ERR_VALUE);
  }
  for (int l0 = 0; l0 < layers; l0 += kCompactLayers) {
    CompactArgs a{};
    const int n = layers - l0 < kCompactLayers ? layers - l0 : kCompactLayers;
    for (int l = 0; l < n; ++l) {
      a.cache_k[l] = reinterpret_cast<uint8_t*>(cache_k[l0 + l]);
      a.cache_v[l] = reinterpret_cast<uint8_t*>(cache_v[l0 + l]);
      a.k_scale[l] = k_scale[l0 + l];
      a.v_scale[l] = v_scale[l0 + l];
    }
    a.path = path;
    a.slots = slots;
    a.T = T;
    a.Hkv = kv_heads;
    a.N = n_blocks;
    a.sh = sh;
    hipLaunchKernelGGL(paged_compact_kernel, dim3(2 * kv_heads, B, n), dim3(kCompactThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    const int st = npn_launch_status();
    if (st != NPN_OK) return st;
  }
  return NPN_OK;
}
