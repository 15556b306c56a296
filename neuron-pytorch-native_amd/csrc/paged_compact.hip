// After a tree's walk: the accepted path's K/V rows to the front of the tree's rows in the e4m3 pages
// (paged_kv.hip has their layout), in all layers at once. Node t's row lies at slots[b][t]; row path[b][d]
// goes to slots[b][d]. path[d] >= d, so rows only move forward, over rejected nodes' rows or others that move.
//
// A page's scale is the page's own: a row that comes from a page of another scale is rounded to its new
// page's, which grows first where the row needs it (as an append's does), the page's older rows with it.
//
// K: a wave has the rows of one (layer, request, head), 256 bytes each. It takes them in order, a batch into registers and
// then to their places: a row's place is no later row's source, so nothing waits for other waves.
// V: rows are columns of their page, bytes a line apart. A thread of a workgroup has one dim: it loads the 16 rows of each
// piece of the tree that has a part in it, up to five, at once, moves bytes between them in LDS of its own and
// stores the pieces that rows went to.
// Bound by a chain of loads (path and slots, scales and rows) where there is little to move, one layer of one request
// 4.2 us, and by lines of the pages, which V's bytes take whole, where there is much: 16 layers of 64 requests of 64
// nodes over blocks of 16, whose paths touch four pieces of five, 39 us for 120 MB read and 97 written, 5.5 TB/s. (There V's
// bytes moved one by one: 51 us by a wave for all dims, 39 by a workgroup with all rows in LDS, which took 5.2 for the one
// request.)
#include "paged_append.h"
#include "tree.h"

namespace {

using append::DH;

constexpr int kCompactLayers = 32;
constexpr int kCompactWaves = 4;  // of a workgroup; for K they share nothing
constexpr int kBatch = 8;         // K's rows in registers
constexpr int kPieces = 5;        // 64 rows from any place on lie in at most so many pieces of 16
static_assert(64 * kCompactWaves == DH, "a thread for each dim of V");

struct CompactArgs {
  uint8_t* cache_k[kCompactLayers];
  uint8_t* cache_v[kCompactLayers];
  float* k_scale[kCompactLayers];
  float* v_scale[kCompactLayers];
  const int32_t* path;   // [B][T]
  const int64_t* slots;  // [B][T]
  int T, Hkv, N, sh;
};

// A path as a wave has it: lane d row d.
struct Path {
  int node, off;       // and where the first row lies in its piece of 16 positions
  int64_t src, dst, dst_page;
  bool row, moves;
  uint64_t moving;     // bits of the rows that move
  float s_old, d_old;  // the scales of the row where it lies and of the page that it goes to
};

__device__ __forceinline__ Path path_of(const CompactArgs& a, const float* scale, int b, int h) {
  const int lane = threadIdx.x & 63;
  const int64_t end = (int64_t)a.N << a.sh;
  const size_t at = (size_t)b * a.T + lane;
  Path p;
  p.node = lane < a.T ? a.path[at] : -1;
  p.dst = lane < a.T ? a.slots[at] : -1;
  p.src = (int64_t)npn::shfl64((uint64_t)p.dst, min(max(p.node, 0), a.T - 1));
  // Rows lie one behind the other, in a block to its end and from the next one's begin: then a row's place counted from
  // the beginning of the first one's piece of 16 positions tells where its own piece begins, and a block's rows among the
  // path's are a run of them. The first row that does not ends what can move.
  p.off = (int)(npn::tree_bits((uint64_t)p.dst, 0) & 15);
  const int64_t mask = (1 << a.sh) - 1, next = (int64_t)npn::shfl64((uint64_t)p.dst, max(lane - 1, 0)) + 1;
  const bool behind = lane == 0 || ((p.dst & mask) == 0 ? (next & mask) == 0 : p.dst == next);
  const uint64_t breaks = __builtin_amdgcn_ballot_w64(!behind);
  const int rows = breaks ? __builtin_ctzll(breaks) : npn::kMaxNodes;
  const bool in = p.dst >= 0 && p.dst < end && p.src >= 0 && p.src < end;
  const int n = npn::path_length(p.node, a.T, lane, in && p.node < rows);
  p.dst_page = p.dst >> a.sh;
  p.row = lane < n;
  p.moves = p.row && p.src != p.dst;
  p.moving = __builtin_amdgcn_ballot_w64(p.moves);
  p.s_old = p.moves ? scale[(p.src >> a.sh) * a.Hkv + h] : 0.f;
  p.d_old = p.row && p.moving ? scale[p.dst_page * a.Hkv + h] : 0.f;
  return p;
}

// The largest magnitude among a word's bytes that is not NaN.
__device__ __forceinline__ int largest_byte(uint32_t x) {
  int big = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int mag = (int)(x >> (8 * j)) & 0x7F;
    big = max(big, mag == 0x7F ? 0 : mag);
  }
  return big;
}
__device__ __forceinline__ int wave_max_int(int x) {
  x = max(x, (int)npn::dpp32<npn::kDppStep[0]>((uint32_t)x));
  x = max(x, (int)npn::dpp32<npn::kDppStep[1]>((uint32_t)x));
  x = max(x, (int)npn::dpp32<npn::kDppStep[2]>((uint32_t)x));
  x = max(x, (int)npn::dpp32<npn::kDppStep[3]>((uint32_t)x));
  const auto a = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  x = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
  return max((int)b[0], (int)b[1]);
}
// The scale that a row needs whose largest byte this is.
__device__ __forceinline__ float need_of(int big, float scale) {
  const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(big, false);
  return v[0] > 0.f ? append::scale_of(v[0] * scale) : 0.f;
}
// The factor from a row's scale to its new page's: infinite only for a row without a finite number but 0, as any
// other has made its page's scale grow. Such a row's bytes stay, as do those of a row whose scale is its new page's.
__device__ __forceinline__ float factor_of(float from, float to) {
  const float by = from / to;
  return from == to || (by == INFINITY && from < INFINITY) ? 1.0f : by;
}
// The new scale of each row's page, from what its rows need.
__device__ __forceinline__ float grown_scale(const Path& p, float need) {
  float now = p.d_old;
  uint64_t left = __builtin_amdgcn_ballot_w64(p.row);
  while (left != 0) {  // page by page
    const bool here = p.row && p.dst_page == (int64_t)npn::tree_bits((uint64_t)p.dst_page, __builtin_ctzll(left));
    const float top = npn::wave_max(here ? fmaxf(p.d_old, need) : 0.f);
    if (here) now = top;
    left &= ~__builtin_amdgcn_ballot_w64(here);
  }
  return now;
}
// For each grown page: f(page, its first row of the path, its last one's place in it, factor, new scale). Of its rows up
// to that place those move to the new scale that the path does not overwrite. No source is among them: where its
// place is one of the path's, another row moves there.
template <class F>
__device__ __forceinline__ void each_grown(const CompactArgs& a, const Path& p, float now, F&& f) {
  uint64_t grown = __builtin_amdgcn_ballot_w64(p.row && now > p.d_old);
  while (grown != 0) {
    const int first = __builtin_ctzll(grown);
    const int64_t page = (int64_t)npn::tree_bits((uint64_t)p.dst_page, first);
    const uint64_t in = __builtin_amdgcn_ballot_w64(p.row && p.dst_page == page);
    const int upto = (int)(npn::tree_bits((uint64_t)p.dst, 63 - __builtin_clzll(in)) & ((1 << a.sh) - 1));
    const float old = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p.d_old), first));
    const float to = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(now), first));
    f(page, first, upto, old / to, to);
    grown &= ~in;
  }
}
// Whether the path moves a row to this slot (wave-uniform).
__device__ __forceinline__ bool moved_to(const Path& p, int64_t slot) {
  return __builtin_amdgcn_ballot_w64(p.moves && p.dst == slot) != 0;
}

__device__ __forceinline__ void compact_k(const CompactArgs& a, uint8_t* cache, float* scale, int b, int h) {
  const int lane = threadIdx.x & 63;
  const Path p = path_of(a, scale, b, h);
  if (p.moving == 0) return;
  auto place = [&](int64_t slot) {  // a slot's row
    return ((slot >> a.sh) * a.Hkv + h) * ((int64_t)DH << a.sh) + (slot & ((1 << a.sh) - 1)) * DH;
  };
  const int64_t from = place(p.src), to = place(p.dst);  // of lanes that have no row: not used
  // The rows that move, kBatch at a time from `left` on: which, and the lane's bytes of them.
  auto take = [&](uint64_t& left, int (&d)[kBatch], uint32_t (&x)[kBatch]) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      d[k] = left ? __builtin_ctzll(left) : -1;
      left &= left - 1;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (d[k] >= 0)
        x[k] = *reinterpret_cast<const uint32_t*>(cache + (int64_t)npn::tree_bits((uint64_t)from, d[k]) + 4 * lane);
  };
  // The pages' new scales. Where no row comes from a larger one they stay.
  float now = p.d_old;
  if (__builtin_amdgcn_ballot_w64(p.moves && p.s_old > p.d_old) != 0) {
    float need = 0.f;
    uint64_t left = p.moving;
    while (left != 0) {
      int d[kBatch];
      uint32_t x[kBatch];
      take(left, d, x);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (d[k] < 0) continue;
        const int big = wave_max_int(largest_byte(x[k]));
        if (lane == d[k]) need = need_of(big, p.s_old);
      }
    }
    now = grown_scale(p, need);
    each_grown(a, p, now, [&](int64_t page, int, int upto, float by, float to_scale) {
      uint32_t* rows = reinterpret_cast<uint32_t*>(cache + (page * a.Hkv + h) * ((int64_t)DH << a.sh)) + lane;
      for (int r0 = 0; r0 <= upto; r0 += kBatch) {
        uint32_t x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = rows[min(r0 + k, upto) * (DH / 4)];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (r0 + k <= upto && !moved_to(p, (page << a.sh) + r0 + k))
            rows[(r0 + k) * (DH / 4)] = append::rescale_e4m3(x[k], by);
      }
      if (lane == 0) scale[page * a.Hkv + h] = to_scale;
    });
  }
  const float by = factor_of(p.s_old, now);
  uint64_t left = p.moving;
  while (left != 0) {
    int d[kBatch];
    uint32_t x[kBatch];
    take(left, d, x);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (d[k] < 0) continue;
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), d[k]));
      *reinterpret_cast<uint32_t*>(cache + (int64_t)npn::tree_bits((uint64_t)to, d[k]) + 4 * lane) =
          f == 1.0f ? x[k] : append::rescale_e4m3(x[k], f);
    }
  }
}

__device__ __forceinline__ void compact_v(const CompactArgs& a, uint8_t* cache, float* scale, int b, int h) {
  __shared__ uint4 s_piece[kPieces][DH];
  __shared__ int s_big[kCompactWaves][npn::kMaxNodes];
  const int dim = threadIdx.x, lane = dim & 63, w = __builtin_amdgcn_readfirstlane(dim >> 6);
  const Path p = path_of(a, scale, b, h);  // the same in every wave
  if (p.moving == 0) return;
  uint8_t* line = cache + (size_t)h * ((size_t)DH << a.sh) + ((size_t)dim << a.sh);  // of this dim in block 0
  const int64_t block = (int64_t)a.Hkv * DH << a.sh;
  const int mask = (1 << a.sh) - 1;
  const int src_at = p.off + p.node, dst_at = p.off + lane;

  // The pieces up to the last row's and those of the sources, all in flight.
  const bool grows = __builtin_amdgcn_ballot_w64(p.moves && p.s_old > p.d_old) != 0;  // some may
  unsigned load = 0, store = 0;
  uint4 x[kPieces];
  uint8_t* at[kPieces];
#pragma unroll
  for (int c = kPieces - 1; c >= 0; --c) {
    const bool to = __builtin_amdgcn_ballot_w64(p.moves && dst_at >> 4 == c) != 0;
    if (to || (grows && store != 0)) store |= 1u << c;
    if (__builtin_amdgcn_ballot_w64(p.moves && src_at >> 4 == c) != 0) load |= 1u << c;
    load |= store;
    if (!(load >> c & 1)) continue;
    const int64_t slot = (int64_t)npn::tree_bits((uint64_t)p.dst, max(16 * c - p.off, 0)) & ~15ll;
    at[c] = line + (slot >> a.sh) * block + (slot & mask);
    x[c] = *reinterpret_cast<const uint4*>(at[c]);
  }
#pragma unroll
  for (int c = 0; c < kPieces; ++c)
    if (load >> c & 1) s_piece[c][dim] = x[c];
  auto byte_of = [&](int place) {
    return reinterpret_cast<uint8_t*>(s_piece) + ((place >> 4) * DH + dim) * 16 + (place & 15);
  };

  float now = p.d_old;
  if (grows) {
    for (uint64_t left = p.moving; left != 0; left &= left - 1) {
      const int d = __builtin_ctzll(left);
      const int big = wave_max_int(largest_byte(*byte_of(__builtin_amdgcn_readlane(src_at, d))));
      if (lane == 0) s_big[w][d] = big;
    }
    __syncthreads();
    int big = 0;
#pragma unroll
    for (int k = 0; k < kCompactWaves; ++k) big = max(big, p.moves ? s_big[k][lane] : 0);
    now = grown_scale(p, need_of(big, p.s_old));
    each_grown(a, p, now, [&](int64_t page, int first, int upto, float by, float to_scale) {
      const int first_at = (int)(npn::tree_bits((uint64_t)p.dst, first) & mask);
      for (int r = 0; r <= upto; r += 4) {
        uint32_t change = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r + j <= upto && !moved_to(p, (page << a.sh) + r + j)) change |= 0xFFu << (8 * j);
        const int place = p.off + first + r - first_at;  // below 0: before the pieces
        uint32_t* word = place >= 0 ? reinterpret_cast<uint32_t*>(byte_of(place))
                                    : reinterpret_cast<uint32_t*>(line + page * block + r);
        const uint32_t old = *word;
        *word = (old & ~change) | (append::rescale_e4m3(old, by) & change);
      }
      if (dim == 0) scale[page * a.Hkv + h] = to_scale;  // every wave has read the old one
    });
  }

  const float by = factor_of(p.s_old, now);
  uint64_t left = p.moving;
  while (left != 0) {
    int d[kBatch];
    uint32_t y[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      d[k] = left ? __builtin_ctzll(left) : -1;
      left &= left - 1;
      if (d[k] >= 0) y[k] = *byte_of(__builtin_amdgcn_readlane(src_at, d[k]));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (d[k] < 0) continue;
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), d[k]));
      *byte_of(p.off + d[k]) = (uint8_t)(f == 1.0f ? y[k] : append::rescale_e4m3(y[k], f));
    }
  }
#pragma unroll
  for (int c = 0; c < kPieces; ++c)
    if (store >> c & 1) *reinterpret_cast<uint4*>(at[c]) = s_piece[c][dim];
}

__global__ __launch_bounds__(64 * kCompactWaves) void paged_compact_kernel(CompactArgs a) {
  const int b = blockIdx.y, layer = blockIdx.z, x = blockIdx.x;
  if (x < a.Hkv) {
    compact_v(a, a.cache_v[layer], a.v_scale[layer], b, x);
    return;
  }
  const int h = __builtin_amdgcn_readfirstlane((x - a.Hkv) * kCompactWaves + ((int)threadIdx.x >> 6));
  if (h < a.Hkv) compact_k(a, a.cache_k[layer], a.k_scale[layer], b, h);
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
  const size_t blocks = (size_t)n_blocks * kv_heads, pages = blocks * block_size * 256, scales = 4 * blocks;
  for (int l = 0; l < layers; ++l) {
    NPN_REQUIRE(cache_k[l] && cache_v[l] && k_scale[l] && v_scale[l], NPN_ERR_NULL);
    NPN_REQUIRE(NPN_ALIGNED16(cache_k[l]) && NPN_ALIGNED16(cache_v[l]), NPN_ERR_ALIGN);
    for (int k = 0; k <= l; ++k)
      NPN_REQUIRE((k == l || (npn_apart(cache_k[k], pages, cache_k[l], pages) &&
                              npn_apart(cache_v[k], pages, cache_v[l], pages) &&
                              npn_apart(k_scale[k], scales, k_scale[l], scales) &&
                              npn_apart(v_scale[k], scales, v_scale[l], scales))) &&
                      npn_apart(cache_k[k], pages, cache_v[l], pages) && npn_apart(cache_v[k], pages, cache_k[l], pages) &&
                      npn_apart(k_scale[k], scales, v_scale[l], scales) &&
                      npn_apart(v_scale[k], scales, k_scale[l], scales),
                  NPN_ERR_VALUE);
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
    hipLaunchKernelGGL(paged_compact_kernel, dim3(kv_heads + (kv_heads + kCompactWaves - 1) / kCompactWaves, B, n),
                       dim3(64 * kCompactWaves), 0,
                       static_cast<hipStream_t>(stream), a);
    const int st = npn_launch_status();
    if (st != NPN_OK) return st;
  }
  return NPN_OK;
}
