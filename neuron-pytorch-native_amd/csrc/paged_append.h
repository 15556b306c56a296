// The append of K/V rows into the pages of an e4m3 cache (paged_kv.hip has the cache's layout): one
// workgroup's part of it, for the kernels that append.
#pragma once

#include "npn_common.h"

namespace {
namespace append {

constexpr int DH = 256;
constexpr int ROPE = 64;
constexpr float kEps = 1e-6f;
constexpr int kMinScaleExp = -100;  // the least scale is 2^-100: an all-zero page's

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

// e4m3 bytes times a power of two, finite, with which none passes 448; NaN stays.
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
// Workgroup `part` of request b's blocks, for head h's K or V; row t's position is pos(t), t wave-uniform.
template <int RPW, int NW, class Pos>
__device__ __forceinline__ void append_block(const PagedAppendArgs& a, int part, int b, int h, bool is_v,
                                                   Pos&& pos) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int bs = 1 << a.sh;
  const int64_t* slots = a.slots + (size_t)b * a.T;

  // The rows [t0, t1) of this block: the request's first slot says where its blocks end, also where
  // its block is none (id -1: a slot of -bs + its row). A request without rows has -1 throughout.
  const int64_t first = slots[0];
  const int off0 = (int)(first & (bs - 1));
  const int t0 = part == 0 ? 0 : bs - off0 + (part - 1) * bs;
  if (t0 >= a.T || (first < 0 && slots[t0] < 0)) return;
  const int room = min(part == 0 ? bs - off0 : bs, a.T - t0);
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
    constexpr int BATCH = RPW < 4 ? RPW : 4;  // rows whose RoPE rows are loaded at a time, without branches
#pragma unroll
    for (int i0 = 0; i0 < RPW; i0 += BATCH) {
      float4 c[BATCH], s[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        int64_t at = pos(t0 + min(row_of(i0 + k), most - 1));
        at = at >= a.positions ? a.positions - 1 : at;
        c[k] = *reinterpret_cast<const float4*>(a.cos + at * ROPE + 4 * (lane & 15));
        s[k] = *reinterpret_cast<const float4*>(a.sin + at * ROPE + 4 * (lane & 15));
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


}  // namespace append
}  // namespace
