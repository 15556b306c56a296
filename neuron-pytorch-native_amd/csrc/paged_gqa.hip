// GQA attention over the paged e4m3 KV cache for gfx950: T new tokens per request (1: plain
// decode, a few: a verify step, many: a prompt's chunk).
//
// Math per query row (b, t, head), t < q_len[b]:
//   q' = (1 + w) * q * rsqrt(mean(q^2) + 1e-6), partial RoPE on q'[:64] (rotate_half inside the
//   64); s_j = q'.K_j / 16 over the keys j <= kv_len[b] + t; out = (softmax(s) V) * sigmoid(gate),
//   K and V the e4m3 bytes times their (block, head) scale. Rows t >= q_len[b] are 0.
//
// The rows of a kv head (token-major, grp heads per token) are cut into groups of R = 16, 32 or 48 rows,
// as they need, or of 128 where they are more (of a tree also two of 32, or several of 48: paged_plan has
// the rule); a (request, row group) is a unit, a (unit, kv head) a pair of its rows and its keys, taken in
// steps of 64 keys (128 with R = 128 but for trees). Three launches:
//  1. prep: q' of every pair as MFMA B operands, and, in its first block, the plan: the host does not
//     know the lengths. A pair of n steps gets ceil(n / Q) workgroups, Q the least number of steps
//     (a multiple of what the waves take at a time) with which all pairs' workgroups are at most `most`.
//     (Equal cuts through the pairs laid end to end balanced better and cost most workgroups a second
//     segment, with its own start and end: 20 us of 80 for 64 sequences of one token.)
//  2. attn, up to 48 rows: a workgroup takes an equal part of its pair's steps; its NW waves (eight for
//     up to 16 rows; four, with all of a SIMD's registers, for more) take those in turn, each alone:
//       S^T[64 keys x 16 rows] = K Q'^T   A = K, 16 bytes per lane as they lie in the page: lane (i, G)
//         of tile j holds key 16 (i / 4) + 4 j + i % 4, dims 64 c + 16 G + [0, 16) for column c; the
//         product's k order follows (Q' is laid out in the same order). In f16: every e4m3 value is
//         an f16 number, q' over a power of two per row has 11 bits, and both scales go into the
//         fp32 scores;
//       online softmax per row in fp32, base 2; that key order puts keys 16 G + [0, 16) of a row
//         into one lane, in order, so
//       O^T[256 x 16 rows] += V^T P^T     takes P straight from the score registers as B, and A = V^T
//         is 16 bytes of a page's dim row. In f16 again: V's bytes as they are, and P times its page's
//         scale, over a running power of two per row that keeps the largest of these products between
//         2^11 and 2^15 (a second running maximum, of log2 of P times the scale): 11 bits of those down
//         to 2^-25 of it, and steps of 2^-35 below, where the cache's own are 2^-10 of a page's scale.
//         (P in bf16 with the scale in V: the output's error was 0.0029 against its own rounding's
//         0.0017. P in two bf16 parts: as exact as f16, with twice these products; 16 requests of 8 x 6
//         rows over up to 32768 keys took 142 us instead of 134.)
//     The bytes go from the pages by DMA to a part of LDS that is the wave's own, in groups of 8 KB
//     in the order of their use (two K tiles, or eight V tiles of 16 dims); a wave takes a group into
//     registers, sends its place for a later one and works on it, with one (NW = 8) to three groups
//     in flight. (A group's eight DMAs in one or two statements, which set M0 once: one by one all of these take 2 to 4 %
//     longer, by the instructions alone.) Nothing else may touch memory in that loop: a reload of a spilled register waits,
//     in order, for every DMA before it.
//     The waves' (m, l, O) meet in LDS; a pair with one workgroup is written out at once. Bound by
//     the cache's bytes: one row group over 32768 keys of 4 heads (67 MB) 18 us, 3.7 TB/s with the start
//     and end in it; 64 sequences of up to 16384 (271 MB) 57 us, 4.7 TB/s; the 16 requests above (607 MB)
//     134 us, 4.5 TB/s; a large read reaches 6.15.
//  2b. rows, R = 128: eight waves of 16 rows share the steps, which pass once through LDS, two steps in
//     all there. Half of the instructions above made f16 of K's and V's bytes, for 16 to 48 rows at
//     a time, and the matrix units were busy for a quarter of the time. Here the bytes go into
//     the 16x16x128 products as they are, and q' as three e4m3 parts of four bits each, 2^-4
//     and 2^-8 in the product's scale operand: 12 bits, for 1.5 times the f16 products' time. P goes in
//     parts too, two of e4m3 and one of e5m2, over a power of two of its own for each 32 keys of a row,
//     which is what that operand holds one number for: 13 bits of the weights down to 2^-13 of the 32's
//     largest, and some of those down to 2^-40 of it. (With three e4m3 parts over one power of two a
//     row, 2^-17 was the least step: a row's other weights were off by 6 % at 2^-20 of its largest and
//     gone at 2^-22, which is all there is where the largest one's value is near 0. 1 us less.) 2 chunks of
//     256 x 6 rows over up to 8192 keys: 130 us (157 with groups of 48 rows; 142 with 128 rows in f16),
//     608 TFLOP/s by the formula's operations. Matrix units 48 %, vector units 54 % busy, which
//     overlap little: without the softmax 100 us would remain, without V's products 100, without the DMAs
//     123. Priorities for one wave of each SIMD, its V products half a step behind the other's, or LDS
//     reads ahead of the products before them changed nothing.
//  2c. the same of a tree: four waves of 32 rows, one to a SIMD, share steps of 64 keys in f16, K's and V's bytes made f16 for
//     32 rows at a time in 32x32x16 products. A lane (i, G) has 16 keys of row i in a tile of 32, in order, so that P is
//     again the next product's operand where it is, over powers of two as in 2. The next step's scores are computed
//     between this step's weights. Of a step's 4700 cycles the matrix unit is busy for 2050 and the vector unit for 2900, the
//     bytes' conversion and the softmax, in the same issue slots as the products; start and end 13000 each: the plan,
//     the first bytes' way, and the parts' 128 KB. 16 requests of 64 x 6 rows over up to 8192 keys 187 us, 620 TFLOP/s
//     by the formula's operations (2b with a tree's masks 224); 8 of 32 x 6 rows 60 (groups of 48: 73).
//     In f16, q' over its row's power of two and the weights over a running one have 11 bits, where 2b's parts have 12
//     and 13: outputs are off by 0.00168 of their norm, their own rounding to bf16 alone and 2b by 0.00166.
//     Tried: DMAs between the products, whose branches had registers spilled (283 us for 232 in all); two chains of
//     products at once, as fast as one; the longest workgroups first, as fast.
//  3. merge: the log-sum-exp merge of the other pairs' workgroups, times sigmoid(gate), to bf16.
// prep takes 4 to 9 us and merge 5 to 10 for 2's and 2b's cases; for trees prep, with their append, 6 (96 rows) to 18
// (24576), and merge 5 to 21.
#include "npn_common.h"
#include "paged_append.h"
#include "tree.h"

namespace {

constexpr int DH = 256;
constexpr int ROPE = 64;
constexpr float kEps = 1e-6f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1.0e30f;   // finite "no key yet" running max (avoids inf - inf)
constexpr float kRescaleLog2 = 4.0f;  // a row's exponents' bases move only when its maxima grow by > 2^4
constexpr float kPLog2 = 11.0f;       // P in f16 is at most 2^(4 + 11), under its 65504
constexpr int KS = 64;                // keys per step
constexpr int kChunk = 64;            // steps whose page ids and scales are in LDS at a time
constexpr int kPages = kChunk * KS / 16 + 1;
constexpr int kRows = 128;            // rows of a group of many

typedef __bf16 bf16x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
typedef __bf16 bf16x2 __attribute__((__vector_size__(2 * sizeof(__bf16))));
typedef _Float16 f16x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));
typedef _Float16 f16x2 __attribute__((__vector_size__(2 * sizeof(_Float16))));
typedef float f32x4 __attribute__((__vector_size__(4 * sizeof(float))));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((__vector_size__(16 * sizeof(float))));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct PagedArgs {
  const uint16_t* query;  // [B][T][Hq][256]
  const uint16_t* gate;
  const float* q_norm;
  const float* cos;       // [positions][64]
  const float* sin;
  const uint8_t* cache_k;  // [N][Hkv][bs][256]
  const uint8_t* cache_v;  // [N][Hkv][256][bs]
  const float* k_scale;    // [N][Hkv]
  const float* v_scale;
  const int32_t* table;    // [B][P]
  const int32_t* kv_len;
  const int32_t* q_len;
  uint16_t* out;
  u32x4* q;                // q' as B operands: [pairs][8][NRT][64], or [pairs][8][2][3 parts][2][64] for R = 128
  float* q_scale;          // [pairs][R]
  float* part_o;           // [slots][R][256] O of the workgroups of split pairs
  float* part_ml;          // [slots][R][2]
  uint64_t* anc;           // trees: [B][T] each node and its ancestors as bits
  int32_t* wstart;         // [U + 1] first workgroup of each unit
  int32_t* sstart;         // [U] first slot of each unit
  int positions, B, T, Hq, Hkv, grp, R, RG, P, N, sh, nw, ks;  // ks: keys of a step
  uint64_t by_grp;         // 2^32 / grp + 1: rows are below 2^21

  __device__ __forceinline__ int token_of(int row) const { return (int)((row * by_grp) >> 32); }
  __device__ __forceinline__ int units() const { return B * RG; }
};

// Unit u = (request, row group): its keys [0, kend) and the tokens it covers.
struct Unit {
  int b, t0, kv, kend, steps;
};

__device__ __forceinline__ Unit unit_of(const PagedArgs& a, int u) {
  Unit r;
  r.b = u / a.RG;
  const int rg = u - r.b * a.RG;
  r.t0 = a.token_of(rg * a.R);  // the group's first token
  const int t1 = min(a.token_of((rg + 1) * a.R - 1), a.T - 1);
  const int n = min(min(a.q_len[r.b], a.T), t1 + 1);  // tokens up to the group's last live one
  const int cap = a.P << a.sh;  // <= 2^30
  r.kv = min(max(a.kv_len[r.b], 0), cap);
  r.kend = n > r.t0 ? min(r.kv + n, cap) : 0;
  r.steps = (r.kend + a.ks - 1) / a.ks;
  return r;
}

// The last of n ascending starts that is at most x (wave-uniform; the first is), 64 at a time.
__device__ __forceinline__ int last_start(const int32_t* start, int n, int x) {
  const int lane = threadIdx.x & 63;
  int u = 0;
  while (n > 1) {
    const int stride = (n + 63) / 64, at = lane * stride;
    const bool le = at < n && start[u + at] <= x;
    const int last = __popcll(__builtin_amdgcn_ballot_w64(le)) - 1;
    n = min(stride, n - last * stride);
    u = __builtin_amdgcn_readfirstlane(u + last * stride);
  }
  return u;
}

// Scores' factor: at least 2^-126, so that -inf times it is -inf; NaN stays. (A row that sees none of a
// lane's 16 keys takes 1, and 0 as their values' logarithm: their page's scales are not its business.)
__device__ __forceinline__ float not_zero(float x) { return x < 0x1p-126f ? 0x1p-126f : x; }
// 2^x for x up to 120, and 2^120 above; NaN stays.
__device__ __forceinline__ float exp2_bounded(float x) { return __builtin_amdgcn_exp2f(x > 120.0f ? 120.0f : x); }

// Maxima over the lanes (i, G) of a column: of G and G ^ 2, of G and G ^ 1, of all.
__device__ __forceinline__ float max_over_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float max_over_pair(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
// Sum and maximum over the wave by lane permutes of the VALU: lane ^ 32, 16, 8, 4, 2, 1 in this order. (Shuffles through
// LDS, 16 a row with its rotation: prep of 24576 rows 21 us instead of 19.5.)
__device__ __forceinline__ float lane_xor4(float x) {
  const int v = (int)__float_as_uint(x);
  const int up = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xF, 0x5, false);  // from 4 lanes on where bit 2 is 0
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(up, v, 0x114, 0xF, 0xA, false));
}
__device__ __forceinline__ float lane_xor8(float x) { return __uint_as_float(npn::dpp32<0x128>(__float_as_uint(x))); }
__device__ __forceinline__ float lane_xor2(float x) { return __uint_as_float(npn::dpp32<0x4E>(__float_as_uint(x))); }
__device__ __forceinline__ float lane_xor1(float x) { return __uint_as_float(npn::dpp32<0xB1>(__float_as_uint(x))); }
__device__ __forceinline__ float max_over_groups(float x) { return max_over_pair(max_over_halves(x)); }
__device__ __forceinline__ float sum_over_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x = sum_over_halves(x);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float wave_sum(float x) {
  x = sum_over_groups(x);
  x += lane_xor8(x);
  x += lane_xor4(x);
  x += lane_xor2(x);
  return x + lane_xor1(x);
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_over_groups(x);
  x = fmaxf(x, lane_xor8(x));
  x = fmaxf(x, lane_xor4(x));
  x = fmaxf(x, lane_xor2(x));
  return fmaxf(x, lane_xor1(x));
}

__device__ __forceinline__ bf16x8 dequant8(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  const u32x4 v = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                   __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
  return __builtin_bit_cast(bf16x8, v);
}

__device__ __forceinline__ f16x8 to_f16x8(uint32_t w0, uint32_t w1) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
  const u32x4 v = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                   __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
  return __builtin_bit_cast(f16x8, v);
}

// A word's bytes of keys [0, n) kept, n <= 0: none, n >= 4: all.
__device__ __forceinline__ uint32_t keep_bytes(int n) {
  return n >= 4 ? ~0u : (n <= 0 ? 0u : (1u << (8 * n)) - 1);
}
// 0xFF in each byte that is an e4m3 NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t t = (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
  return t * 0xFFu;
}

// 16 bytes per lane into LDS at a wave-uniform address, from a per-lane address or an offset. The
// caller waits with vmcnt.
using npn::lds_dma16_soff_uniform;
using npn::lds_dma16_uniform;

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
// D = A B 16^-part + C over 128 e4m3 of k (lane (i, G): 32 of row or column i).
__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 a, i32x8 b, f32x4 c, int part) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127 - 4 * part);
}
// The same with a part of P as B: e5m2 for the last, and byte `part` of `scales`, the biased exponents of
// the powers of two that a block of 32 k is times. Of a lane's 32 bytes the first 16 are k 16 G + [0, 16),
// the others 64 more; block n of k, [32 n, + 32), takes its exponent from the lanes with G = n.
template <int PART>
__device__ __forceinline__ f32x4 mfma_p(i32x8 a, i32x8 b, f32x4 c, int scales) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, PART == 2 ? 1 : 0, 0, 127, PART, scales);
}

// LDS by address, element k of 16 bytes (1 KB apart: one per lane) from a per-lane base. The bases are
// hidden from the optimiser (opaque): left to itself it kept some hundred of base + offset sums,
// past the 16-bit offset of an LDS instruction, in registers and spilled them.
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
__device__ __forceinline__ u32x4 lds_read(unsigned base, int k) {
  return reinterpret_cast<lds_u32x4*>(base)[64 * k];
}
__device__ __forceinline__ void lds_write(unsigned base, int k, u32x4 v) {
  reinterpret_cast<lds_u32x4*>(base)[64 * k] = v;
}
// With a SIMD to itself a wave's accumulators stay in AGPRs: without a word at the places where VALU
// work touches them, the compiler carried them in VGPRs and copied all of them twice a step.
__device__ __forceinline__ void pin(f32x4& x) { asm volatile("" : "+a"(x)); }
__device__ __forceinline__ void pin(f32x16& x) { asm volatile("" : "+a"(x)); }
__device__ __forceinline__ unsigned opaque(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Four DMAs of 1 KB each: from a uniform base + o0, o1, o0 and o1, the later ones 1, 2 and 3 KB behind, as are their places.
__device__ __forceinline__ void lds_dma16x4_soff(const void* sbase, unsigned o0, unsigned o1, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %4\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %3\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:0x400\n\t"
      "global_load_lds_dwordx4 %1, %3 offset:0x800\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:0xc00\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(o0), "v"(o1), "s"(sbase), "s"(lds)
      : "memory");
}
// The same from per-lane addresses, `step` bytes apart.
__device__ __forceinline__ void lds_dma16x4(const uint8_t* g, size_t step, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %5\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %4, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(g), "v"(g + step), "v"(g + 2 * step), "v"(g + 3 * step), "s"(lds)
      : "memory", "scc");
}

// Eight DMAs of 1 KB each from four uniform bases + o ^ 0, 64, 128 and 192, two 1 KB apart from each; their places follow
// one another.
__device__ __forceinline__ void lds_dma16x8_soff(const uint8_t* const (&base)[4], unsigned o, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %9\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %5\n\t"
      "global_load_lds_dwordx4 %1, %5 offset:0x400\n\t"
      "s_add_u32 m0, m0, 0x800\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %6\n\t"
      "global_load_lds_dwordx4 %2, %6 offset:0x400\n\t"
      "s_add_u32 m0, m0, 0x800\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %7\n\t"
      "global_load_lds_dwordx4 %3, %7 offset:0x400\n\t"
      "s_add_u32 m0, m0, 0x800\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %8\n\t"
      "global_load_lds_dwordx4 %4, %8 offset:0x400\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(o), "v"(o ^ 64u), "v"(o ^ 128u), "v"(o ^ 192u), "s"(base[0]), "s"(base[1]), "s"(base[2]), "s"(base[3]), "s"(lds)
      : "memory", "scc");
}

// Four dims of a row's output: o / l * sigmoid(gate); 0 for a row without keys (inv = 0), whatever its
// gate, and for tokens past q_len.
__device__ __forceinline__ void write_out(const PagedArgs& a, int b, int row, int h, int dim, f32x4 o, float inv) {
  const int t = a.token_of(row), qh = h * a.grp + row - t * a.grp;
  const size_t at = (((size_t)b * a.T + t) * a.Hq + qh) * DH + dim;
  const uint2 g = *reinterpret_cast<const uint2*>(a.gate + at);
  const uint32_t gw[2] = {g.x, g.y};
  const bool live = inv != 0.f && t < a.q_len[b];
  uint32_t y[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float v0 = o[2 * j] * inv * npn::sigmoid(npn::bf16lo(gw[j]));
    const float v1 = o[2 * j + 1] * inv * npn::sigmoid(npn::bf16hi(gw[j]));
    y[j] = live ? npn::f32_to_bf16(v0) | ((uint32_t)npn::f32_to_bf16(v1) << 16) : 0u;
  }
  *reinterpret_cast<uint2*>(a.out + at) = make_uint2(y[0], y[1]);
}

// Four numbers of at most 448 as a word each of three e4m3 parts, x = p0 + p1 / 16 + p2 / 256: each part
// takes 4 bits of what the ones before leave, 12 in all, down to steps of 2^-17. For q', whose small
// elements count by what they add to the row's large ones.
__device__ __forceinline__ void split3(float x0, float x1, float x2, float x3, uint32_t (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    part[k] = (uint32_t)w;
    if (k == 2) break;
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x0 = (x0 - lo[0]) * 16.0f;
    x1 = (x1 - lo[1]) * 16.0f;
    x2 = (x2 - hi[0]) * 16.0f;
    x3 = (x3 - hi[1]) * 16.0f;
  }
}

// Four weights of at most 2^8, x = p0 + 2^-5 p1 + 2^-17 p2, p0 and p1 in e4m3 and p2 in e5m2, which has 3 bits
// instead of 4 but reaches 2^-16 instead of 2^-9. What p0 and p1 leave is at most 2^-9 of x's power of two, or
// half of p1's least step, 2^-15; p2 has it to 2^-4 of its own: x to 2^-13 down to 2^-6, to 2^-19 below that,
// and where it is p2 alone, to 2^-3 of itself down to 2^-31, with steps of 2^-33 to the end.
__device__ __forceinline__ void split_p(float x0, float x1, float x2, float x3, uint32_t (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    part[k] = (uint32_t)w;
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    const float by = k == 0 ? 0x1p5f : 0x1p12f;
    x0 = (x0 - lo[0]) * by;
    x1 = (x1 - lo[1]) * by;
    x2 = (x2 - hi[0]) * by;
    x3 = (x3 - hi[1]) * by;
  }
  int w = __builtin_amdgcn_cvt_pk_bf8_f32(x0, x1, 0, false);
  w = __builtin_amdgcn_cvt_pk_bf8_f32(x2, x3, w, true);
  part[2] = (uint32_t)w;
}
constexpr int kPartExp[3] = {0, 5, 17};

// ---- 1. prep ----------------------------------------------------------------------------------------
constexpr int kPrepWaves = 8;
constexpr int kPlanUnits = 4096;  // units whose steps the plan keeps in LDS

// One workgroup per CU where the pairs with steps are few enough to be cut so; else one each and 512
// more for the longest. Requests of 100 to 16384 keys, 4 kv heads: 128 pairs 119 us in 256 workgroups and
// 129 in 640, 180 pairs of 48 rows 214 and 201, 240 pairs 232 and 209. Groups of 128 rows are few and long,
// so that a second round of workgroups may pay where the first leaves many CUs idle: 512 x 6 rows over
// 16384 keys, 96 pairs, take 330 us in 192 workgroups and 290 in 480. The plan takes the cheaper by the
// steps of 128 keys that the rounds last, with 1.5 for a workgroup's start and end and 2.5 for writing
// and merging the parts of 256. (Of trees the steps have 64 keys, and start and end take as long as five of them.)
__host__ __device__ constexpr int most_workgroups(int R, int pairs, int rounds) {
  return R == kRows && rounds == 2 && pairs > 64 && pairs <= 448 ? 512 : pairs <= 160 ? 256 : pairs + 512;
}
// Split pairs' workgroups: all of 256 or 512, or, as a pair of c >= 2 has c - 1 of the 512 more, twice
// those.
constexpr int kSlots = 1024;

// Workgroups of each unit's pairs: the least Q = nw k with sum ceil(n / Q) <= most lies between
// k = S / (most nw) and S / ((most - pairs) nw); the eight waves test eight k of what is left at a time.
__device__ void plan_block(const PagedArgs& a) {
  __shared__ int s_n[kPlanUnits];
  __shared__ int s_wave[kPrepWaves][2];
  __shared__ int s_sum[kPrepWaves * 64][2];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int U = a.units();
  auto steps_of = [&](int u) { return u < kPlanUnits ? s_n[u] : unit_of(a, u).steps; };
  int sum = 0, some = 0;
  for (int u = tid; u < U; u += kPrepWaves * 64) {
    const int n = unit_of(a, u).steps;
    if (u < kPlanUnits) s_n[u] = n;
    sum += n;
    some += n > 0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, 64);
    some += __shfl_xor(some, off, 64);
  }
  if (lane == 0) {
    s_wave[w][0] = sum;
    s_wave[w][1] = some;
  }
  __syncthreads();
  sum = some = 0;
  for (int k = 0; k < kPrepWaves; ++k) {
    sum += s_wave[k][0];
    some += s_wave[k][1];
  }
  const int S = sum * a.Hkv, pairs = some * a.Hkv;  // S < 2^30
  auto up = [](int n, int d) { return (n + d - 1) / d; };
  // The least Q that `most` workgroups allow, and the workgroups that it makes.
  auto least = [&](int most, int& made) {
    int lo = max(1, up(up(S, most), a.nw)), hi = max(lo, up(up(S, max(most - pairs, 1)), a.nw));
    made = most;
    while (lo < hi) {
      const int Q = (lo + (int)((int64_t)(hi - lo) * w / kPrepWaves)) * a.nw;
      int g = 0;
      for (int u = lane; u < U; u += 64) g += up(steps_of(u), Q);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) g += __shfl_xor(g, off, 64);
      __syncthreads();  // s_wave has been read
      if (lane == 0) s_wave[w][0] = g;
      __syncthreads();
      int nlo = lo, nhi = hi;
      for (int k = kPrepWaves - 1; k >= 0; --k) {
        const int t = lo + (int)((int64_t)(hi - lo) * k / kPrepWaves);
        if ((int64_t)s_wave[k][0] * a.Hkv <= most) {
          nhi = t;
          made = s_wave[k][0] * a.Hkv;
        } else {
          nlo = max(nlo, t + 1);
        }
      }
      lo = min(nlo, nhi);
      hi = nhi;
    }
    return hi * a.nw;
  };
  int made;
  int Q = least(most_workgroups(a.R, pairs, 1), made);
  if (a.R == kRows && most_workgroups(a.R, pairs, 2) > most_workgroups(a.R, pairs, 1)) {
    const float part = a.ks == KS ? 5.0f : 1.5f, join = a.ks == KS ? 0.02f : 0.01f;
    auto cost = [&](int q, int g) { return up(g, 256) * (q + part) + g * join; };
    const float one = cost(Q, made);
    const int Q2 = least(most_workgroups(a.R, pairs, 2), made);
    if (cost(Q2, made) < one) Q = Q2;
  }
  // First workgroup and first slot of each unit: scans over threads' slices of the units.
  const int per = up(U, kPrepWaves * 64);
  const int u0 = min(U, tid * per), u1 = min(U, u0 + per);
  int wg = 0, slot = 0;
  for (int u = u0; u < u1; ++u) {
    const int c = up(steps_of(u), Q) * a.Hkv;
    wg += c;
    slot += c > a.Hkv ? c : 0;
  }
  const int wg_mine = wg, slot_mine = slot;
  for (int off = 1; off < kPrepWaves * 64; off <<= 1) {
    s_sum[tid][0] = wg;
    s_sum[tid][1] = slot;
    __syncthreads();
    if (tid >= off) {
      wg += s_sum[tid - off][0];
      slot += s_sum[tid - off][1];
    }
    __syncthreads();
  }
  if (tid == kPrepWaves * 64 - 1) a.wstart[U] = wg;
  wg -= wg_mine;
  slot -= slot_mine;
  for (int u = u0; u < u1; ++u) {
    const int c = up(steps_of(u), Q) * a.Hkv;
    a.wstart[u] = wg;
    a.sstart[u] = slot;
    wg += c;
    slot += c > a.Hkv ? c : 0;
  }
}

// q' of one padded row per wave (rows that are none repeat the pair's last), over the least power of
// two above the row's largest element. In f16 dim d = 64 c + 16 g + 8 h + e is element e of lane group
// g in k step 2 c + h; in e4m3 parts d = 128 m + 64 x + 16 g + e is byte 16 x + e of group g in step m.
// A wave has RW rows in turn, whose loads go out together. TREE: a row's position is its node's depth behind the
// committed ones.
template <bool TREE, int RW>
__device__ __forceinline__ void prep_rows(const PagedArgs& a, const int32_t* parent, int64_t wave) {
  const int lane = threadIdx.x & 63;
  const int64_t first = wave * RW;
  const int pair = (int)(first / a.R), r0 = (int)(first - (int64_t)pair * a.R);
  if (pair >= a.units() * a.Hkv) return;
  const int u = pair / a.Hkv, h = pair - u * a.Hkv;
  const int b = u / a.RG;
  const int parent_of = TREE ? npn::tree_parent(parent + (size_t)b * a.T, a.T, lane) : 0;
  const float4 nw = *reinterpret_cast<const float4*>(a.q_norm + 4 * lane);
  uint2 q[RW];
  float4 cs[RW], sn[RW];
  int t[RW];
#pragma unroll
  for (int k = 0; k < RW; ++k) {
    const int row = min((u - b * a.RG) * a.R + r0 + k, a.T * a.grp - 1);
    t[k] = a.token_of(row);
    const int qh = h * a.grp + row - t[k] * a.grp;
    q[k] = *reinterpret_cast<const uint2*>(a.query + (((size_t)b * a.T + t[k]) * a.Hq + qh) * DH + 4 * lane);
  }
  const int64_t kv = max(a.kv_len[b], 0);
  __builtin_amdgcn_sched_barrier(0);
  uint64_t anc = 0;
  if constexpr (TREE) anc = npn::tree_ancestors(parent_of, a.T, lane);
#pragma unroll
  for (int k = 0; k < RW; ++k) {
    int behind = t[k];
    if constexpr (TREE) {
      behind = __popcll(npn::tree_bits(anc, __builtin_amdgcn_readfirstlane(t[k]))) - 1;
      // (rows that repeat the last write the same)
      if (h == 0 && lane == t[k]) a.anc[(size_t)b * a.T + t[k]] = anc;
    }
    // The row's own position, also where the table ends before it.
    const int64_t at = min(kv + behind, (int64_t)a.positions - 1);
    const size_t pos = (size_t)at * ROPE + 4 * (lane & 15);
    cs[k] = *reinterpret_cast<const float4*>(a.cos + pos);
    sn[k] = *reinterpret_cast<const float4*>(a.sin + pos);
  }
#pragma unroll
  for (int k = 0; k < RW; ++k) {
    const int r = r0 + k;
    const float4 c = cs[k], s = sn[k];
    float v[4] = {npn::bf16lo(q[k].x), npn::bf16hi(q[k].x), npn::bf16lo(q[k].y), npn::bf16hi(q[k].y)};
    const float ss = wave_sum(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]);
    const float rn = rsqrtf(ss * (1.0f / DH) + kEps);
    v[0] = (1.0f + nw.x) * (v[0] * rn);
    v[1] = (1.0f + nw.y) * (v[1] * rn);
    v[2] = (1.0f + nw.z) * (v[2] * rn);
    v[3] = (1.0f + nw.w) * (v[3] * rn);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = lane_xor8(v[j]);  // dim d ^ 32
    if (lane < ROPE / 4) {
      const float sg = lane < ROPE / 8 ? -1.0f : 1.0f;
      v[0] = v[0] * c.x + sg * y[0] * s.x;
      v[1] = v[1] * c.y + sg * y[1] * s.y;
      v[2] = v[2] * c.z + sg * y[2] * s.z;
      v[3] = v[3] * c.w + sg * y[3] * s.w;
    }
    const float big = wave_max(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
    const uint32_t e = min(max(__float_as_uint(big) >> 23, 64u), 190u);  // 2^-63 to 2^63
    float inv = __uint_as_float((253u - e) << 23);                      // 2^-(e - 126)
    float q_scale = __uint_as_float((e + 1) << 23) * (kLog2e / 16.0f);
    const int d = 4 * lane;
    if (!TREE && a.R == kRows) {  // three e4m3 parts of 256 times as much
      inv *= 256.0f;
      q_scale *= 1.0f / 256;
      if (lane == 0) a.q_scale[(size_t)pair * a.R + r] = q_scale;
      uint32_t part[3];
      split3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, part);
      const size_t at = ((((size_t)pair * 8 + (r >> 4)) * 2 + (d >> 7)) * 3 * 2 + ((d >> 6) & 1)) * 64;
      uint32_t* dst = reinterpret_cast<uint32_t*>(a.q + at + 16 * ((d >> 4) & 3) + (r & 15));
#pragma unroll
      for (int k = 0; k < 3; ++k) dst[k * 512 + ((d >> 2) & 3)] = part[k];
      continue;
    }
    if (lane == 0) a.q_scale[(size_t)pair * a.R + r] = q_scale;
    uint32_t two[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f16x2 x = {(_Float16)(v[2 * j] * inv), (_Float16)(v[2 * j + 1] * inv)};
      two[j] = __builtin_bit_cast(uint32_t, x);
    }
    u32x4* dst;
    if (TREE && a.R == kRows) {  // d = 32 c + 16 g + 8 h + e, k step 2 c + h of 16, rows 32 to a product
      const int step = 2 * (d >> 5) + ((d >> 3) & 1), g = (d >> 4) & 1;
      dst = a.q + (((size_t)pair * 4 + (r >> 5)) * 16 + step) * 64 + 32 * g + (r & 31);
    } else {
      const int step = 2 * (d >> 6) + ((d >> 3) & 1), g = (d >> 4) & 3;
      dst = a.q + (((size_t)pair * 8 + step) * (a.R / 16) + (r >> 4)) * 64 + 16 * g + (r & 15);
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint32_t*>(dst) + ((d & 4) >> 1)) = make_uint2(two[0], two[1]);
  }
}

__global__ __launch_bounds__(kPrepWaves * 64) void paged_prep_kernel(PagedArgs a) {
  if (blockIdx.x == 0) plan_block(a);
  else prep_rows<false, 1>(a, nullptr, (int64_t)(blockIdx.x - 1) * kPrepWaves + (threadIdx.x >> 6));
}

// The same for a tree, and before it, in `appends` workgroups, the append of its nodes' rows, which the attention's
// launch reads: none of the three parts reads what another writes.
template <int RPW, int QR>
__global__ __launch_bounds__(kPrepWaves * 64) void tree_prep_kernel(PagedArgs a, append::PagedAppendArgs ap,
                                                                    const int32_t* parent, int appends, int per) {
  const int x = (int)blockIdx.x - 1;
  if (x < 0) {
    plan_block(a);
  } else if (x >= appends) {
    prep_rows<true, QR>(a, parent, (int64_t)(x - appends) * kPrepWaves + (threadIdx.x >> 6));
  } else {
    const int bh = x / per, b = bh / (2 * ap.Hkv), hv = bh - b * 2 * ap.Hkv, lane = threadIdx.x & 63;
    const uint64_t anc =
        npn::tree_ancestors(npn::tree_parent(parent + (size_t)b * ap.T, ap.T, lane), ap.T, lane);
    const int64_t kv = max(ap.kv_len[b], 0);
    append::append_block<RPW, kPrepWaves>(ap, x - bh * per, b, hv >> 1, hv & 1, [&](int t) {
      return kv + __popcll(npn::tree_bits(anc, __builtin_amdgcn_readfirstlane(t))) - 1;
    });
  }
}

// ---- 2. attn ----------------------------------------------------------------------------------------
// Trees: which of a lane's 16 keys a row sees, as bits: of those up to its last one, `left` from the lane's first
// on, the committed ones and the nodes `anc`. The first is `at` places behind the committed ones.
__device__ __forceinline__ uint32_t seen16(uint64_t anc, int at, int left) {
  // bits [at + 32, at + 48) of 32 committed keys, the nodes and nothing
  const int s = min(max(at + 32, 0), 96), k = s >> 5;
  const uint32_t lo = (uint32_t)anc, hi = (uint32_t)(anc >> 32);
  const uint32_t a = k == 0 ? ~0u : k == 1 ? lo : k == 2 ? hi : 0u, b = k == 0 ? lo : k == 1 ? hi : 0u;
  return __builtin_amdgcn_alignbit(b, a, s & 31) & (0xFFFFu >> (16 - min(max(left, 0), 16)));
}
// x where bit k of `bits` is set, else -inf.
__device__ __forceinline__ float if_seen(uint32_t bits, int k, float x) {
  const int keep = (int)(bits << (31 - k)) >> 31;
  return __uint_as_float((__float_as_uint(x) & keep) | (0xFF800000u & ~keep));
}

template <int NRT, int NW, bool TREE>
struct PagedSmem {
  static constexpr int DR = NRT == 3 ? 8 : 16;  // 16-dim tiles of O that all waves have in LDS at once
  union {
    uint8_t ring[NW][16 / NW][8192];            // each wave's groups
    f32x4 o[NW][NRT][DR][64];
  };
  u32x4 q[8][NW == 4 ? NRT : 1][64];            // q' as B operands: [k step][row tile][lane]
  float m[NW][NRT * 16], l[NW][NRT * 16], inv[NRT * 16];
  int page[kPages];                             // -1: none
  float ks[kPages], vs[kPages];                 // the keys' scales, the logarithms of the values'
  uint64_t anc[TREE ? NRT * 16 : 1];            // what a row sees of the nodes
  int lim[TREE ? NRT * 16 : 1];
};

template <int NRT, int NW, bool TREE>
__global__ __launch_bounds__(NW * 64, NW / 4) void paged_attn_kernel(PagedArgs a) {
  constexpr int R = NRT * 16;
  constexpr int NR = 16 / NW;  // groups in a wave's ring
  constexpr int kThreads = NW * 64;
  using Smem = PagedSmem<NRT, NW, TREE>;
  __shared__ __attribute__((aligned(1024))) Smem sm;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int i = lane & 15, G = lane >> 4;
  const int bs = 1 << a.sh;
  const int U = a.units();

  // This workgroup's unit, kv head and steps [s_lo, s_lo + steps).
  if ((int)blockIdx.x >= a.wstart[U]) return;
  const int u = last_start(a.wstart, U, (int)blockIdx.x);
  const Unit un = unit_of(a, u);
  const int w0 = a.wstart[u], parts = (a.wstart[u + 1] - w0) / a.Hkv;
  const int h = ((int)blockIdx.x - w0) / parts, part = (int)blockIdx.x - w0 - h * parts;
  const int s_lo = (int)((int64_t)part * un.steps / parts);
  const int steps = (int)((int64_t)(part + 1) * un.steps / parts) - s_lo;
  const int pair = u * a.Hkv + h;
  const int row0 = (u - un.b * a.RG) * R;  // the group's first row
  const int rows = min(R, a.T * a.grp - row0);

  // The last key of each of this lane's rows (one per tile); -1 for rows that are none.
  int lim[NRT];
  float q_scale[NRT], m_run[NRT], l_run[NRT], w_run[NRT];
#pragma unroll
  for (int nt = 0; nt < NRT; ++nt) {
    const int r = 16 * nt + i, t = a.token_of(row0 + r);
    lim[nt] = r < rows && t < a.q_len[un.b] ? min(un.kv + t, un.kend - 1) : -1;
    if constexpr (TREE) {
      if (w == 0 && G == 0) {
        sm.anc[r] = a.anc[(size_t)un.b * a.T + min(t, a.T - 1)];
        sm.lim[r] = lim[nt];
      }
    }
    q_scale[nt] = a.q_scale[(size_t)pair * R + r];
    m_run[nt] = kNegBig;
    w_run[nt] = kNegBig;
    l_run[nt] = 0.f;
  }
  const int lim0 = TREE ? un.kv - 1 : un.kv + un.t0;  // every row of the group sees the keys up to here
  const unsigned ring_lds = __builtin_amdgcn_readfirstlane(npn::lds_addr(&sm.ring[w][0][0]));
  const u32x4* qsrc = a.q + (size_t)pair * 8 * NRT * 64 + lane;
  u32x4 qreg[NW == 8 ? 8 : 1];
  if constexpr (NW == 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) qreg[k] = qsrc[64 * k];
  } else {
#pragma unroll
    for (int k = 0; k < 2 * NRT; ++k)
      lds_dma16_uniform(qsrc + 64 * (w * 2 * NRT + k),
            __builtin_amdgcn_readfirstlane(npn::lds_addr(&sm.q[0][0][0])) + (w * 2 * NRT + k) * 1024u);
  }

  // K goes four whole rows (1 KB) to a DMA, column c of row r (of the step's 64) to place c ^ f(r) of
  // the row's 256 bytes, f(r) = 4 (r / 16) + r % 4: lane (i, G)'s row of a tile has f = i, so the 16
  // rows that a tile reads at one column lie in 16 different places. A group holds rows 16 k + 8 n
  // .. + 7 for k = 0..3 as its rows 8 k .. + 7. Sources and places of the k (or c) differ in bits 6
  // and 7 alone.
  const unsigned ksrc = (unsigned)(G * DH + ((i ^ G) << 4));
  const unsigned k_at = ring_lds + (unsigned)((8 * (i >> 2) + (i & 3)) * DH + ((i ^ G) << 4));
  const unsigned v_at = ring_lds + lane * 16u;
  const unsigned q_at = npn::lds_addr(&sm.q[0][0][lane]);

  // Steps are taken kChunk at a time, [c0, c0 + cn) of this workgroup's, with their pages in LDS.
  int cn, key0, page0;
  // The pages of a step's keys: 16 k .. + 15 (k < 4), and the lane's 16.
  auto pages_of = [&](int s, int (&id)[5]) {
    const int k0 = key0 + s * KS;
#pragma unroll
    for (int k = 0; k < 4; ++k) id[k] = sm.page[((k0 + 16 * k) >> a.sh) - page0];
    id[4] = sm.page[((k0 + 16 * G) >> a.sh) - page0];
  };
  auto load_k = [&](int s, const int (&id)[5], int n, int at) {  // tiles 2 n, 2 n + 1
    const uint8_t* pg[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = key0 + s * KS + 16 * k, page = __builtin_amdgcn_readfirstlane(max(id[k], 0));
      pg[k] = a.cache_k + ((((size_t)page * a.Hkv + h) << a.sh) + (key & (bs - 1)) + 8 * n) * DH;
    }
    lds_dma16x8_soff(pg, opaque(ksrc), ring_lds + (unsigned)(at * 8192));
  };
  auto load_v = [&](int s, const int (&id)[5], int n, int at) {  // dims 128 n .. + 127
    const int key = key0 + s * KS + 16 * G;
    const uint8_t* pg = a.cache_v + ((((size_t)max(id[4], 0) * a.Hkv + h) * DH + 128 * n + i) << a.sh) + (key & (bs - 1));
    const size_t step = (size_t)16 << a.sh;
    lds_dma16x4(pg, step, ring_lds + (unsigned)(at * 8192));
    lds_dma16x4(pg + 4 * step, step, ring_lds + (unsigned)(at * 8192 + 4096));
  };
  auto begin_chunk = [&](int c0) {
    cn = min(kChunk, steps - c0);
    key0 = (s_lo + c0) * KS;
    page0 = key0 >> a.sh;
    const int pages = ((min(key0 + cn * KS, un.kend) - 1) >> a.sh) - page0 + 1;
    __syncthreads();  // the last chunk's pages have been used
    for (int p = tid; p < kPages; p += kThreads) {
      int id = -1;
      if (p < pages) id = a.table[(size_t)un.b * a.P + page0 + p];
      const bool ok = id >= 0 && id < a.N;
      sm.page[p] = ok ? id : -1;
      sm.ks[p] = ok ? a.k_scale[(size_t)id * a.Hkv + h] : 1.0f;
      sm.vs[p] = ok ? log2f(a.v_scale[(size_t)id * a.Hkv + h]) : 0.0f;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // and q' is in LDS
    __syncthreads();
  };
  auto first_sends = [&]() {
    if (w < cn) {
      int id[5];
      pages_of(w, id);
      load_k(w, id, 0, 0);
      load_k(w, id, 1, 1);
      if constexpr (NR == 4) {
        load_v(w, id, 0, 2);
        load_v(w, id, 1, 3);
      }
    }
  };
  begin_chunk(0);
  // What was loaded so far is waited for here: a wait behind the first DMAs would drain them.
#pragma unroll
  for (int nt = 0; nt < NRT; ++nt) asm volatile("" : "+v"(lim[nt]), "+v"(q_scale[nt]));
#pragma unroll
  for (int k = 0; k < (NW == 8 ? 8 : 1); ++k) asm volatile("" : "+v"(qreg[k]));
  first_sends();

  f32x4 acc[NRT][16];
#pragma unroll
  for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
    for (int d = 0; d < 16; ++d) acc[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int c0 = 0; c0 < steps; c0 += kChunk) {
    if (c0 > 0) {
      begin_chunk(c0);
      first_sends();
    }
    for (int s = w; s < cn; s += NW) {
      if constexpr (NW == 4) {
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
          for (int d = 0; d < 16; ++d) pin(acc[nt][d]);
      }
      const int k0 = key0 + s * KS;
      const int page = ((k0 + 16 * G) >> a.sh) - page0;  // of this lane's 16 keys
      const float ks = sm.ks[page], vs = sm.vs[page];
      const bool held = sm.page[page] >= 0;  // they exist
      const bool next = s + NW < cn;
      const int sn = next ? s + NW : s;
      int id[5];
      pages_of(sn, id);
      if constexpr (NR != 4) id[4] = sm.page[page];

      f32x4 st[NRT][4];
#pragma unroll
      for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) st[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      // Groups K 0, K 1, V 0, V 1 (0 to 3) in places 0 .. NR - 1 in turn. A group has landed when at
      // most the DMAs of the NR - 1 after it are in flight (fewer at the end); once it is in
      // registers its place is sent for the group NR further on.
      auto landed = [&](int g) {
        if (next || 3 - g >= NR - 1)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(8 * (NR - 1)) : "memory");
        else if (g == 1)
          asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        else if (g == 2)
          asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      };
      auto send = [&](int g) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (NR == 4) {
          if (next) {
            if (g < 2) load_k(sn, id, g, g);
            else load_v(sn, id, g - 2, g);
          }
        } else {
          if (g < 2) load_v(s, id, g, g);
          else if (next) load_k(sn, id, g - 2, g - 2);
        }
      };
      const unsigned kat = opaque(k_at), vat = opaque(v_at);
      if constexpr (NW == 8) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          landed(n);
          u32x4 kw[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) kw[j][c] = lds_read(kat ^ (c << 6), 8 * n + j);
          send(n);
#pragma unroll
          for (int step = 0; step < 8; ++step)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const u32x4 k4 = kw[j][step >> 1];
              const f16x8 kf = (step & 1) ? to_f16x8(k4[2], k4[3]) : to_f16x8(k4[0], k4[1]);
              st[0][2 * n + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  kf, __builtin_bit_cast(f16x8, qreg[step]), st[0][2 * n + j], 0, 0, 0);
            }
        }
      } else {  // both K groups together, so that q' is read from LDS once
        asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        const unsigned qat = opaque(q_at);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4 kw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) kw[j] = lds_read(kat ^ (c << 6), 8 * (j >> 1) + (j & 1));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            f16x8 q[NRT];
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
              q[nt] = __builtin_bit_cast(f16x8, lds_read(qat, (2 * c + half) * NRT + nt));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f16x8 kf = to_f16x8(kw[j][2 * half], kw[j][2 * half + 1]);
#pragma unroll
              for (int nt = 0; nt < NRT; ++nt)
                st[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[nt], st[nt][j], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        send(0);
        send(1);
      }

      // A step with keys past the group's first limit, or past a page that is none, is masked.
      const bool tail = k0 + KS - 1 > lim0 || __builtin_amdgcn_ballot_w64(!held) != 0;
      auto seen = [&](int nt) {
        const int r = TREE ? 16 * nt + i : 0, kb = k0 + 16 * G;
        return seen16(sm.anc[r], kb - un.kv, sm.lim[r] + 1 - kb);
      };
      uint32_t bits[TREE ? NRT : 1];
      if constexpr (TREE) {
        // In every step: computed where it is needed, in the branch below, it had thirty registers spilled.
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) bits[nt] = held ? seen(nt) : 0u;
      }
      if (tail) {
        const int kb = k0 + 16 * G;
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if constexpr (TREE) st[nt][j][r] = if_seen(bits[nt], 4 * j + r, st[nt][j][r]);
              else if (!held || kb + 4 * j + r > lim[nt]) st[nt][j][r] = -INFINITY;
            }
        }
      }

      f16x8 pw[NRT][2];
#pragma unroll
      for (int nt = 0; nt < NRT; ++nt) {
        float mx = st[nt][0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[nt][j][r]);
        // All 16 keys of the lane. (Scores are not infinite; masked ones beside a NaN do no harm: it stays.)
        const bool hidden = TREE ? mx == -INFINITY : tail && k0 + 16 * G > lim[nt];
        const float c = hidden ? 1.0f : not_zero(ks * q_scale[nt]), vsn = hidden ? 0.0f : vs;
        mx *= c;
        const float wx = max_over_groups(mx + vsn);
        mx = max_over_groups(mx);
        const bool grow = mx > m_run[nt] + kRescaleLog2, wgrow = wx > w_run[nt] + kRescaleLog2;
        if (__builtin_amdgcn_ballot_w64(grow || wgrow) != 0) {
          const float mnew = grow ? mx : m_run[nt], wnew = wgrow ? wx : w_run[nt];
          const float corr = exp2f(w_run[nt] - wnew);
          l_run[nt] *= exp2f(m_run[nt] - mnew);
          m_run[nt] = mnew;
          w_run[nt] = wnew;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            acc[nt][d] *= corr;
            if constexpr (NW == 4) pin(acc[nt][d]);
          }
        }
        const float f = exp2_bounded(m_run[nt] + vsn - w_run[nt] + kPLog2);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float pv = __builtin_amdgcn_exp2f(fmaf(st[nt][j][r], c, -m_run[nt]));
            sum += pv;
            pw[nt][j >> 1][(j & 1) * 4 + r] = (_Float16)(pv * f);
          }
        l_run[nt] += sum;
      }

#pragma unroll
      for (int n = 0; n < 2; ++n) {
        landed(2 + n);
        u32x4 v[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) v[d] = lds_read(vat, 8 * ((2 + n) % NR) + d);
        send(2 + n);
        if (tail) {
          // V bytes of keys that no row sees are cleared (0 times NaN is NaN). A NaN at a key that
          // some rows see reaches those and no others: it is cleared too, and the product of "is
          // NaN" and "sees it", 2^100 each, makes the outputs that it belongs in infinite, which
          // the segment's end makes NaN (as it would a sum past the largest float).
          const int live = held ? un.kend - (k0 + 16 * G) : 0;
          uint32_t nan_seen = 0;
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[d][k] &= keep_bytes(live - 4 * k);
              nan_seen |= nan_bytes(v[d][k]);
            }
          if (__builtin_amdgcn_ballot_w64(nan_seen != 0) != 0) {
            bf16x8 see[NRT][2];
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                see[nt][e >> 3][e & 7] =
                    (__bf16)((TREE ? seen(nt) >> e & 1 : k0 + 16 * G + e <= lim[nt]) ? 0x1p100f : 0.0f);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              u32x4 is;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                is[k] = nan_bytes(v[d][k]) & 0x38383838u;  // e4m3 1.0
                v[d][k] &= ~nan_bytes(v[d][k]);
              }
#pragma unroll
              for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  acc[nt][8 * n + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      dequant8(is[2 * k], is[2 * k + 1], 0x1p100f), see[nt][k], acc[nt][8 * n + d], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const f16x8 vf = to_f16x8(v[d][2 * k], v[d][2 * k + 1]);
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
              acc[nt][8 * n + d] =
                  __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pw[nt][k], acc[nt][8 * n + d], 0, 0, 0);
          }
          if (d % 2) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // The waves' rows meet: all scaled to the common maximum, DR dim tiles of every wave's O into LDS,
  // where each wave sums its share over the waves and writes it: the partial of a split pair, else
  // the output.
#pragma unroll
  for (int nt = 0; nt < NRT; ++nt) {
    l_run[nt] = sum_over_groups(l_run[nt]);
    if (G == 0) {
      sm.m[w][16 * nt + i] = m_run[nt];
      sm.l[w][16 * nt + i] = l_run[nt];
    }
  }
  __syncthreads();  // every wave is done with its ring, which O takes over
  const size_t slot = (size_t)a.sstart[u] + h * parts + part;
#pragma unroll
  for (int nt = 0; nt < NRT; ++nt) {
    float m = kNegBig, l = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) m = fmaxf(m, sm.m[k][16 * nt + i]);
#pragma unroll
    for (int k = 0; k < NW; ++k) l += exp2f(sm.m[k][16 * nt + i] - m) * sm.l[k][16 * nt + i];
    const float f = exp2f(w_run[nt] - m - kPLog2);
#pragma unroll
    for (int d = 0; d < 16; ++d) acc[nt][d] *= f;
    if (w == 0 && G == 0) {
      const int r = 16 * nt + i;
      sm.inv[r] = l != 0.f ? 1.0f / l : 0.f;
      if (parts > 1) {
        a.part_ml[(slot * R + r) * 2] = m;
        a.part_ml[(slot * R + r) * 2 + 1] = l;
      }
    }
  }
  const unsigned o_at = npn::lds_addr(&sm.o[w][0][0][lane]), o_all = npn::lds_addr(&sm.o[0][0][0][lane]);
#pragma unroll
  for (int d0 = 0; d0 < 16; d0 += Smem::DR) {
    if (d0 > 0) __syncthreads();  // the tiles before have been summed
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
      for (int d = 0; d < Smem::DR; ++d)
        lds_write(o_at, nt * Smem::DR + d, __builtin_bit_cast(u32x4, acc[nt][d0 + d]));
    __syncthreads();
    for (int k = w; k < NRT * Smem::DR; k += NW) {
      const int nt = k / Smem::DR, d = d0 + k % Smem::DR;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < NW; ++v)
        o += __builtin_bit_cast(f32x4, lds_read(o_all + k * 1024, v * NRT * Smem::DR));
      o += o * 0.0f;  // infinite: NaN
      const int r = 16 * nt + i;
      if (parts > 1)
        *reinterpret_cast<f32x4*>(a.part_o + (slot * R + r) * DH + 16 * d + 4 * G) = o;
      else if (r < rows)
        write_out(a, un.b, row0 + r, h, 16 * d + 4 * G, o, sm.inv[r]);
    }
  }
}

// ---- 2b. attn of many rows ----------------------------------------------------------------------------
struct RowsSmem {
  union {
    uint8_t ring[2][65536];  // two steps of 128 keys: for each half two groups of K and two of V, as above
    f32x4 o[8][16][64];      // 16 rows of 256 to a wave
  };
  float inv[kRows];
  int lim[kRows];
  int nan_key[DH];         // the first key past lim0 whose value at a dim is NaN
  int page[kPages];
  float ks[kPages], vs[kPages];
};

__global__ __launch_bounds__(512, 2) void paged_rows_kernel(PagedArgs a) {
  constexpr int R = kRows, KR = 128, kSteps = kChunk * KS / KR;
  constexpr int kTop = 7;  // a block's largest weight is taken to [2^kTop, 2^(kTop + 1))
  __shared__ __attribute__((aligned(1024))) RowsSmem sm;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int i = lane & 15, G = lane >> 4;
  const int bs = 1 << a.sh;
  const int U = a.units();

  if ((int)blockIdx.x >= a.wstart[U]) return;
  const int u = last_start(a.wstart, U, (int)blockIdx.x);
  const Unit un = unit_of(a, u);
  const int w0 = a.wstart[u], parts = (a.wstart[u + 1] - w0) / a.Hkv;
  const int h = ((int)blockIdx.x - w0) / parts, part = (int)blockIdx.x - w0 - h * parts;
  const int s_lo = (int)((int64_t)part * un.steps / parts);
  const int steps = (int)((int64_t)(part + 1) * un.steps / parts) - s_lo;
  const int pair = u * a.Hkv + h;
  const int row0 = (u - un.b * a.RG) * R;
  const int rows = min(R, a.T * a.grp - row0);

  const int r = 16 * w + i, t = a.token_of(row0 + r);  // this lane's row and its last key, or -1
  int lim = r < rows && t < a.q_len[un.b] ? min(un.kv + t, un.kend - 1) : -1;
  float q_scale = a.q_scale[(size_t)pair * R + r];
  float m_run = kNegBig, w_run = kNegBig, l_run = 0.f;
  const int lim0 = un.kv + un.t0;
  i32x8 q[2][3];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const u32x4* src = a.q + ((((size_t)pair * 8 + w) * 2 + m) * 3 + k) * 128 + lane;
      q[m][k] = join(src[0], src[64]);
    }

  const unsigned ring_lds = __builtin_amdgcn_readfirstlane(npn::lds_addr(&sm.ring[0][0]));
  const unsigned ksrc = (unsigned)(G * DH + ((i ^ G) << 4)) ^ ((w >> 1) << 6);
  const unsigned k_at = ring_lds + (unsigned)((8 * (i >> 2) + (i & 3)) * DH + ((i ^ G) << 4));
  const unsigned v_at = ring_lds + lane * 16u;

  int cn, key0, page0;
  // A wave's eight of a step's 64 DMAs: one to each group.
  auto load_step = [&](int s) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const unsigned at = ring_lds + (unsigned)((s & 1) * 65536 + half * 32768 + w * 1024);
      const int k0 = key0 + s * KR + half * KS;
      const int kk = k0 + 16 * (w >> 1), kv = k0 + 16 * G;
      const int kid = __builtin_amdgcn_readfirstlane(max(sm.page[(kk >> a.sh) - page0], 0));
      const uint8_t* const kp =
          a.cache_k + ((((size_t)kid * a.Hkv + h) << a.sh) + (kk & (bs - 1))) * DH + (w & 1) * 4 * DH;
      lds_dma16_soff_uniform(kp, ksrc, at);
      lds_dma16_soff_uniform(kp + 8 * DH, ksrc, at + 8192);
      const int vid = max(sm.page[(kv >> a.sh) - page0], 0);
      const uint8_t* const vp =
          a.cache_v + ((((size_t)vid * a.Hkv + h) * DH + 16 * w + i) << a.sh) + (kv & (bs - 1));
      lds_dma16_uniform(vp, at + 2 * 8192);
      lds_dma16_uniform(vp + ((size_t)128 << a.sh), at + 3 * 8192);
    }
  };
  // V bytes of keys that no row sees are cleared (0 times NaN is NaN), each wave those that it sent for. So
  // is a NaN at a key that some rows see, and the first such key of its dim noted: the rows that see it
  // get the NaN at the end.
  auto clean = [&](int k0, unsigned place) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k1 = k0 + KS * half + 16 * G;
      const int live = sm.page[(k1 >> a.sh) - page0] >= 0 ? un.kend - k1 : 0;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const unsigned at = opaque(v_at + place + half * 32768u + (2 + n) * 8192u + w * 1024u);
        u32x4 v = lds_read(at, 0);
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          v[k] &= keep_bytes(live - 4 * k);
          const uint32_t nan = nan_bytes(v[k]);
          if (nan != 0) {
            atomicMin(&sm.nan_key[16 * (w + 8 * n) + i], k1 + 4 * k + (__ffs(nan) - 1) / 8);
            v[k] &= ~nan;
          }
        }
        lds_write(at, 0, v);
      }
    }
  };
  auto missing = [&](int k0) {  // a page of the step is none
    return __builtin_amdgcn_ballot_w64(sm.page[((k0 + 16 * G) >> a.sh) - page0] < 0 ||
                                       sm.page[((k0 + KS + 16 * G) >> a.sh) - page0] < 0) != 0;
  };
  auto begin_chunk = [&](int c0) {
    cn = min(kSteps, steps - c0);
    key0 = (s_lo + c0) * KR;
    page0 = key0 >> a.sh;
    const int pages = ((min(key0 + cn * KR, un.kend) - 1) >> a.sh) - page0 + 1;
    __syncthreads();  // the last chunk's pages and steps have been used
    for (int p = tid; p < kPages; p += 512) {
      int id = -1;
      if (p < pages) id = a.table[(size_t)un.b * a.P + page0 + p];
      const bool ok = id >= 0 && id < a.N;
      sm.page[p] = ok ? id : -1;
      sm.ks[p] = ok ? a.k_scale[(size_t)id * a.Hkv + h] : 1.0f;
      sm.vs[p] = ok ? log2f(a.v_scale[(size_t)id * a.Hkv + h]) : 0.0f;
    }
    __syncthreads();
  };
  if (tid < DH) sm.nan_key[tid] = 0x7FFFFFFF;
  begin_chunk(0);
  // What was loaded so far is waited for before the first DMAs.
  asm volatile("" : "+v"(lim), "+v"(q_scale));
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int k = 0; k < 3; ++k) asm volatile("" : "+v"(q[m][k]));
  load_step(0);

  f32x4 acc[16];
#pragma unroll
  for (int d = 0; d < 16; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int c0 = 0; c0 < steps; c0 += kSteps) {
    if (c0 > 0) {
      begin_chunk(c0);
      load_step(0);
    }
    for (int s = 0; s < cn; ++s) {
      // The step has landed for every wave past the barrier, and all are done with the step before,
      // whose place the next takes.
      const int k0 = key0 + s * KR;
      const bool tail = k0 + KR - 1 > lim0 || missing(k0);
      if (tail) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        clean(k0, (unsigned)(s & 1) * 65536u);
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (s + 1 < cn) load_step(s + 1);
      if (__builtin_amdgcn_ballot_w64(lim >= k0) == 0) continue;  // none of the wave's rows sees it
      const unsigned place = (unsigned)(s & 1) * 65536u;
      float ks[2], vs[2];
      bool held[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int page = ((k0 + KS * half + 16 * G) >> a.sh) - page0;
        ks[half] = sm.ks[page];
        vs[half] = sm.vs[page];
        held[half] = sm.page[page] >= 0;
      }

      f32x4 st[2][4];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const unsigned kat = opaque(k_at + place + half * 32768u);
          u32x4 kw[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) kw[j][c] = lds_read(kat ^ (c << 6), 8 * n + j);
          f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
              for (int j = 0; j < 2; ++j) x[j] = mfma_e4m3(join(kw[j][2 * m], kw[j][2 * m + 1]), q[m][k], x[j], k);
          st[half][2 * n] = x[0];
          st[half][2 * n + 1] = x[1];
          asm volatile("" : "+v"(st[half][2 * n]), "+v"(st[half][2 * n + 1])::"memory");
          __builtin_amdgcn_sched_barrier(0);
        }

      if (tail) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!held[half] || k0 + KS * half + 16 * G + 4 * j + e > lim) st[half][j][e] = -INFINITY;
      }

      // Beside the row's maxima, `top` of each block of 32 keys that its products take as one: those of
      // the lanes G and G ^ 1 in a half.
      float c[2], mx = -INFINITY, top[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bool hidden = tail && k0 + KS * half + 16 * G > lim;
        c[half] = hidden ? 1.0f : not_zero(ks[half] * q_scale);
        vs[half] = hidden ? 0.0f : vs[half];
        float x = st[half][0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) x = fmaxf(x, st[half][j][e]);
        mx = fmaxf(mx, x * c[half]);
        top[half] = max_over_pair(x * c[half] + vs[half]);
      }
      const float wx = max_over_halves(fmaxf(top[0], top[1]));
      mx = max_over_groups(mx);
      const bool grow = mx > m_run + kRescaleLog2, wgrow = wx > w_run + kRescaleLog2;
      if (__builtin_amdgcn_ballot_w64(grow || wgrow) != 0) {
        const float mnew = grow ? mx : m_run, wnew = wgrow ? wx : w_run;
        const float corr = exp2f(w_run - wnew);
        l_run *= exp2f(m_run - mnew);
        m_run = mnew;
        w_run = wnew;
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[d] *= corr;
      }
      // Each block's weights over a power of two of their own: whole, 2^-100 of the row's at least.
      i32x8 p[3];
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, block[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        block[half] = fminf(fmaxf(floorf(top[half] - w_run), -100.0f), kRescaleLog2);
        const float f = exp2_bounded(m_run + vs[half] - w_run + (kTop - block[half]));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pv[e] = __builtin_amdgcn_exp2f(fmaf(st[half][j][e], c[half], -m_run));
            sum[e] += pv[e];
          }
          uint32_t word[3];
          split_p(pv[0] * f, pv[1] * f, pv[2] * f, pv[3] * f, word);
#pragma unroll
          for (int k = 0; k < 3; ++k) p[k][4 * half + j] = (int)word[k];
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      // Lanes G = 0, 1, 2, 3 hand over the exponents of half 0's first and second block and half 1's.
      const auto lo_hi = __builtin_amdgcn_permlane32_swap((int)block[0], (int)block[1], false, false);
      int scales = (127 - kTop + (int)((G & 1) ? lo_hi[1] : lo_hi[0])) * 0x010101;
      scales -= kPartExp[1] << 8 | kPartExp[2] << 16;

#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const unsigned vat = opaque(v_at + place);
        u32x4 v[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int d = 0; d < 4; ++d) v[half][d] = lds_read(vat, 32 * half + 16 + 4 * n + d);
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[4 * n + d] = mfma_p<0>(join(v[0][d], v[1][d]), p[0], acc[4 * n + d], scales);
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[4 * n + d] = mfma_p<1>(join(v[0][d], v[1][d]), p[1], acc[4 * n + d], scales);
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[4 * n + d] = mfma_p<2>(join(v[0][d], v[1][d]), p[2], acc[4 * n + d], scales);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // A wave has its rows whole: through LDS, for stores of whole rows, 16 bytes at f of dim 4 f to place
  // f ^ i of row i.
  const float l = sum_over_groups(l_run), scale = exp2f(w_run - m_run);
  const size_t slot = (size_t)a.sstart[u] + h * parts + part;
  __syncthreads();  // every wave is done with the ring
  f32x4* const o = &sm.o[w][0][0];
#pragma unroll
  for (int d = 0; d < 16; ++d) o[64 * i + ((4 * d + G) ^ i)] = acc[d] * scale;
  if (G == 0) {
    sm.inv[r] = l != 0.f ? 1.0f / l : 0.f;
    sm.lim[r] = lim;
    if (parts > 1) {
      a.part_ml[(slot * R + r) * 2] = m_run;
      a.part_ml[(slot * R + r) * 2 + 1] = l;
    }
  }
  __syncthreads();
  for (int k = 0; k < 16; ++k) {
    const int rk = 16 * w + k;
    f32x4 x = o[64 * k + (lane ^ k)];
    x += x * 0.0f;  // infinite: NaN
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (sm.lim[rk] >= sm.nan_key[4 * lane + e]) x[e] = NAN;
    if (parts > 1)
      *reinterpret_cast<f32x4*>(a.part_o + (slot * R + rk) * DH + 4 * lane) = x;
    else if (rk < rows)
      write_out(a, un.b, row0 + rk, h, 4 * lane, x, sm.inv[rk]);
  }
}

// ---- 2c. attn of many rows of a tree -------------------------------------------------------------------
struct TreeRowsSmem {
  union {
    uint8_t ring[4][32768];  // four steps of 64 keys: K, 64 rows of 256 bytes, and V, 16 groups of 16 dims
    f32x4 o[4][32][64];      // 32 rows of 256 to a wave
  };
  float inv[kRows];
  uint64_t anc[kRows];   // what a row sees of the nodes; 0: not even the committed keys
  uint64_t nan_node[DH]; // the nodes whose value at a dim is NaN; all where a committed key's is
  int page[kPages];
  float ks[kPages], vs[kPages];
};

__global__ __launch_bounds__(256, 1) void paged_tree_rows_kernel(PagedArgs a) {
  constexpr int R = kRows;
  constexpr int NS = 4;  // steps in LDS
  __shared__ __attribute__((aligned(1024))) TreeRowsSmem sm;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int i = lane & 31, G = lane >> 5;
  const int bs = 1 << a.sh;
  const int U = a.units();

  if ((int)blockIdx.x >= a.wstart[U]) return;
  const int u = last_start(a.wstart, U, (int)blockIdx.x);
  const Unit un = unit_of(a, u);
  const int w0 = a.wstart[u], parts = (a.wstart[u + 1] - w0) / a.Hkv;
  const int h = ((int)blockIdx.x - w0) / parts, part = (int)blockIdx.x - w0 - h * parts;
  const int s_lo = (int)((int64_t)part * un.steps / parts);
  const int steps = (int)((int64_t)(part + 1) * un.steps / parts) - s_lo;
  const int pair = u * a.Hkv + h;
  const int row0 = (u - un.b * a.RG) * R;
  const int rows = min(R, a.T * a.grp - row0);

  const int r = 32 * w + i, t = a.token_of(row0 + r);  // this lane's row and its last key, or -1
  int lim = r < rows && t < a.q_len[un.b] ? min(un.kv + t, un.kend - 1) : -1;
  uint64_t anc = a.anc[(size_t)un.b * a.T + min(t, a.T - 1)];
  float q_scale = a.q_scale[(size_t)pair * R + r];
  float m_run = kNegBig, w_run = kNegBig, l_run = 0.f;
  u32x4 q[16];
  {
    const u32x4* src = a.q + ((size_t)pair * 4 + w) * 16 * 64 + lane;
#pragma unroll
    for (int k = 0; k < 16; ++k) q[k] = src[64 * k];
  }

  // K goes four whole rows to a DMA, column c of row r to place c ^ f(r) of the row's 256 bytes, f(r) = bits 0, 1, 4 and 2 of
  // r: lane (i, G)'s row of a tile, bits 0, 1, 3, 4 and 2 of i, has f = i % 16. V's groups of 16 dims lie as they come.
  const unsigned ring_lds = __builtin_amdgcn_readfirstlane(npn::lds_addr(&sm.ring[0][0]));
  const int i16 = lane & 15, G16 = lane >> 4;
  const unsigned ksrc = (unsigned)(G16 * DH + ((i16 ^ G16) << 4)) ^ ((w & 1) << 6);
  const unsigned k_at = ring_lds + (unsigned)((16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3)) * DH + ((G ^ i16) << 4));
  const unsigned v_at = ring_lds + 16384u + (unsigned)((i >> 4) * 1024 + G * 256 + i16 * 16);

  int cn, key0, page0;
  bool missing;  // a page of the chunk is none
  // A wave's eight of a step's 32 DMAs: rows 16 k + 4 w .. + 3 of K, dims 16 (w + 4 k) .. + 15 of V.
  // Pages of a wave's part of a step: keys 16 w .. + 15 of K, and of V the lane's 16 keys of dims 64 w .. + 63.
  int k_id, v_id;
  auto pages_of = [&](int s) __attribute__((always_inline)) {
    const int k0 = key0 + min(s, cn - 1) * KS;
    k_id = sm.page[((k0 + 16 * w) >> a.sh) - page0];
    v_id = sm.page[((k0 + 16 * G16) >> a.sh) - page0];
  };
  auto load_step = [&](int s) __attribute__((always_inline)) {
    const unsigned at = ring_lds + (unsigned)((s & (NS - 1)) * 32768 + w * 4096);
    const int kk = key0 + s * KS + 16 * w, kv = key0 + s * KS + 16 * G16;
    const int id = __builtin_amdgcn_readfirstlane(max(k_id, 0));
    lds_dma16x4_soff(a.cache_k + ((((size_t)id * a.Hkv + h) << a.sh) + (kk & (bs - 1))) * DH, ksrc, ksrc ^ 128u, at);
    const uint8_t* const vp =
        a.cache_v + ((((size_t)max(v_id, 0) * a.Hkv + h) * DH + 64 * w + i16) << a.sh) + (kv & (bs - 1));
    lds_dma16x4(vp, (size_t)16 << a.sh, at + 16384);
  };
  // V bytes of keys that no row sees are cleared (0 times NaN is NaN), each wave those that it sent for. So
  // is a NaN at a key that some rows see, and the key's node noted at its dim: the rows that see it get the NaN
  // at the end.
  auto clean = [&](int k0, unsigned place) __attribute__((always_inline)) {
    const int k1 = k0 + 16 * G16;
    const int live = sm.page[(k1 >> a.sh) - page0] >= 0 ? un.kend - k1 : 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const unsigned at = opaque(ring_lds + place + 16384u + (unsigned)((4 * w + n) * 1024 + lane * 16));
      u32x4 v = lds_read(at, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] &= keep_bytes(live - 4 * k);
        const uint32_t nan = nan_bytes(v[k]);
        if (nan != 0) {
          uint64_t nodes = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int node = k1 + 4 * k + e - un.kv;  // below 64: behind kend they have been cleared
            if ((nan >> (8 * e)) & 1) nodes |= node < 0 ? ~0ull : 1ull << node;
          }
          atomicOr(reinterpret_cast<unsigned long long*>(&sm.nan_node[16 * (4 * w + n) + i16]), (unsigned long long)nodes);
          v[k] &= ~nan;
        }
      }
      lds_write(at, 0, v);
    }
  };
  auto begin_chunk = [&](int c0) __attribute__((always_inline)) {
    cn = min(kChunk, steps - c0);
    key0 = (s_lo + c0) * KS;
    page0 = key0 >> a.sh;
    const int pages = ((min(key0 + cn * KS, un.kend) - 1) >> a.sh) - page0 + 1;
    __syncthreads();  // the last chunk's pages and steps have been used
    int none = 0;
    for (int p = tid; p < kPages; p += 256) {
      int id = -1;
      if (p < pages) id = a.table[(size_t)un.b * a.P + page0 + p];
      const bool ok = id >= 0 && id < a.N;
      sm.page[p] = ok ? id : -1;
      none |= p < pages && !ok;
      sm.ks[p] = ok ? a.k_scale[(size_t)id * a.Hkv + h] : 1.0f;
      sm.vs[p] = ok ? log2f(a.v_scale[(size_t)id * a.Hkv + h]) : 0.0f;
    }
    missing = __syncthreads_or(none) != 0;
  };
  auto first_sends = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NS - 2; ++s)
      if (s < cn) {
        pages_of(s);
        load_step(s);
      }
    pages_of(NS - 2);
  };
  for (int d = tid; d < DH; d += 256) sm.nan_node[d] = 0;
  begin_chunk(0);
  // What was loaded so far is waited for before the first DMAs.
  asm volatile("" : "+v"(lim), "+v"(q_scale), "+v"(anc));
#pragma unroll
  for (int k = 0; k < 16; ++k) asm volatile("" : "+v"(q[k]));
  first_sends();

  // The step has landed for every wave past the barrier, and all are done with the step before, whose place the next
  // one to be sent takes. Whether the step is masked.
  auto begin_step = [&](int s, int k0, unsigned place) __attribute__((always_inline)) {
    const bool tail = k0 + KS > un.kv || missing;
    if (tail) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      clean(k0, place);
    } else if (s + 1 < cn) {
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + NS - 2 < cn) load_step(s + NS - 2);
    return tail;
  };
  const bool idle = __builtin_amdgcn_ballot_w64(lim >= 0) == 0;  // a wave without a row: only its part of the DMAs
  f32x16 acc[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) acc[d] = f32x16{};

  for (int c0 = 0; idle && c0 < steps; c0 += kChunk) {
    if (c0 > 0) {
      begin_chunk(c0);
      first_sends();
    }
    for (int s = 0; s < cn; ++s) {
      begin_step(s, key0 + s * KS, (unsigned)(s & (NS - 1)) * 32768u);
      pages_of(s + NS - 1);
    }
  }
  u32x4 kw[3][2];
  unsigned kat;
  auto read_k = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) kw[c % 3][j] = lds_read(kat ^ (c << 5), 8 * j);
  };
  auto score = [&](f32x16 (&st)[2], int c) __attribute__((always_inline)) {  // dims 32 c .. + 31
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        st[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(to_f16x8(kw[c % 3][j][2 * b], kw[c % 3][j][2 * b + 1]),
                                                       __builtin_bit_cast(f16x8, q[2 * c + b]), st[j], 0, 0, 0);
  };
  for (int c0 = 0; !idle && c0 < steps; c0 += kChunk) {
    if (c0 > 0) {
      begin_chunk(c0);
      first_sends();
    }
    bool tail = begin_step(0, key0, 0);
    f32x16 sn[2] = {f32x16{}, f32x16{}};
    kat = opaque(k_at);
    read_k(0);
    read_k(1);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c + 2 < 8) read_k(c + 2);
      __builtin_amdgcn_sched_barrier(0);
      score(sn, c);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int s = 0; s < cn; ++s) {
#pragma unroll
      for (int d = 0; d < 8; ++d) pin(acc[d]);
#pragma unroll
      for (int k = 0; k < 16; ++k) asm volatile("" : "+v"(q[k]));
      const int k0 = key0 + s * KS;
      f32x16 st[2] = {sn[0], sn[1]};
      asm volatile("" : "+v"(st[0]), "+v"(st[1]));
      pages_of(s + NS - 1);
      float ks[2], vs[2];
      bool hidden[2] = {false, false};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int page = ((k0 + 32 * j + 16 * G) >> a.sh) - page0;
        ks[j] = sm.ks[page];
        vs[j] = sm.vs[page];
        if (tail) {
          const int kb = k0 + 32 * j + 16 * G;
          const uint32_t bits = sm.page[page] >= 0 ? seen16(anc, kb - un.kv, lim + 1 - kb) : 0u;
          hidden[j] = bits == 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) st[j][e] = if_seen(bits, e, st[j][e]);
        }
      }

      float c[2], mx = -INFINITY, wx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c[j] = hidden[j] ? 1.0f : not_zero(ks[j] * q_scale);
        vs[j] = hidden[j] ? 0.0f : vs[j];
        float x = st[j][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) x = fmaxf(x, st[j][e]);
        mx = fmaxf(mx, x * c[j]);
        wx = fmaxf(wx, x * c[j] + vs[j]);
      }
      mx = max_over_halves(mx);
      wx = max_over_halves(wx);
      const bool grow = mx > m_run + kRescaleLog2, wgrow = wx > w_run + kRescaleLog2;
      if (__builtin_amdgcn_ballot_w64(grow || wgrow) != 0) {
        const float mnew = grow ? mx : m_run, wnew = wgrow ? wx : w_run;
        const float corr = exp2f(w_run - wnew);
        l_run *= exp2f(m_run - mnew);
        m_run = mnew;
        w_run = wnew;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          pin(acc[d]);  // (else it is read in every step)
          acc[d] *= corr;
          pin(acc[d]);
        }
      }
      const unsigned place = (unsigned)(s & (NS - 1)) * 32768u, after = (unsigned)((s + 1) & (NS - 1)) * 32768u;
      if (s + 1 < cn) tail = begin_step(s + 1, k0 + KS, after);
      // The next step's scores between this one's weights (behind the last step they are no step's).
      kat = opaque(k_at + after);
      const unsigned vat = opaque(v_at + place);
      read_k(0);
      read_k(1);
      float f[2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 2; ++j) f[j] = exp2_bounded(m_run + vs[j] - w_run + kPLog2);
      f16x8 pw[2][2];
      u32x4 v[3][2];
      sn[0] = sn[1] = f32x16{};
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (n + 2 < 8) {
          read_k(n + 2);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) v[n - 6][j] = reinterpret_cast<lds_u32x4*>(vat)[128 * (n - 6) + 32 * j];
        }
        __builtin_amdgcn_sched_barrier(0);
        score(sn, n);
        const int j = n >> 2;
#pragma unroll
        for (int e = 4 * (n & 3); e < 4 * (n & 3) + 4; ++e) {
          const float pv = __builtin_amdgcn_exp2f(fmaf(st[j][e], c[j], -m_run));
          sum[j] += pv;
          pw[j][e >> 3][e & 7] = (_Float16)(pv * f[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      l_run += sum[0] + sum[1];
#pragma unroll
      for (int d = 0; d < 8; ++d) pin(acc[d]);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        if (d + 2 < 8) {
#pragma unroll
          for (int j = 0; j < 2; ++j) v[(d + 2) % 3][j] = reinterpret_cast<lds_u32x4*>(vat)[128 * (d + 2) + 32 * j];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(to_f16x8(v[d % 3][j][2 * b], v[d % 3][j][2 * b + 1]), pw[j][b],
                                                            acc[d], 0, 0, 0);
        pin(acc[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // A wave has its rows whole: through LDS, for stores of whole rows, 16 bytes at f of dim 4 f to place
  // f ^ i of row i.
  const float l = sum_over_halves(l_run), scale = exp2f(w_run - m_run - kPLog2);
  const size_t slot = (size_t)a.sstart[u] + h * parts + part;
  __syncthreads();  // every wave is done with the ring
  f32x4* const o = &sm.o[w][0][0];
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 x = {acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]};
      o[64 * i + ((8 * d + 2 * k + G) ^ i16)] = x * scale;
    }
  if (G == 0) {
    sm.inv[r] = l != 0.f ? 1.0f / l : 0.f;
    sm.anc[r] = lim >= 0 ? anc : 0;
    if (parts > 1) {
      a.part_ml[(slot * R + r) * 2] = m_run;
      a.part_ml[(slot * R + r) * 2 + 1] = l;
    }
  }
  __syncthreads();
  uint64_t nan[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) nan[e] = sm.nan_node[4 * lane + e];
#pragma unroll 4
  for (int k = 0; k < 32; ++k) {
    const int rk = 32 * w + k;
    if (rk >= rows) break;
    f32x4 x = o[64 * k + (lane ^ (k & 15))];
    x += x * 0.0f;  // infinite: NaN
    const uint64_t sees = sm.anc[rk];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((sees & nan[e]) != 0) x[e] = NAN;
    if (parts > 1)
      *reinterpret_cast<f32x4*>(a.part_o + (slot * R + rk) * DH + 4 * lane) = x;
    else
      write_out(a, un.b, row0 + rk, h, 4 * lane, x, sm.inv[rk]);
  }
}

// ---- 3. merge ---------------------------------------------------------------------------------------
// The workgroups' (m, l, O) of a row of a pair, WPR waves to a row: wave q takes parts q, q + WPR, ...,
// four loads of each at a time, and the first wave merges the waves'. Four waves where rows are few and so
// have many parts, else one. With both launches before it, four waves and one: 4 pairs of 16 rows with
// 64 parts each 27.5 and 37.2 us, 32 pairs 62.6 and 66.2, 64 pairs 57.9 and 59.0, 96 pairs 91.1 and 90.8,
// 96 pairs of 48 rows 115.3 and 113.4.
template <int WPR>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int q = wv % WPR;
  const int r = blockIdx.x * (4 / WPR) + wv / WPR;
  const int pair = blockIdx.y;
  const int u = pair / a.Hkv, h = pair - u * a.Hkv;
  const int parts = (a.wstart[u + 1] - a.wstart[u]) / a.Hkv;
  if (parts == 1) return;  // written by its workgroup
  const int b = u / a.RG;
  const int row = (u - b * a.RG) * a.R + r;
  if (row >= a.T * a.grp) return;  // the whole workgroup where WPR = 4; no barrier where WPR = 1
  const size_t slot = (size_t)a.sstart[u] + h * parts;
  float m = kNegBig, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k = q; k < parts; k += 4 * WPR) {
    float mv[4], lv[4];
    f32x4 ov[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = k + j * WPR < parts;
      const size_t at = (slot + k + j * WPR) * a.R + r;
      mv[j] = ok ? a.part_ml[2 * at] : kNegBig;
      lv[j] = ok ? a.part_ml[2 * at + 1] : 0.f;
      ov[j] = ok ? *reinterpret_cast<const f32x4*>(a.part_o + at * DH + 4 * lane)
                 : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float mn = fmaxf(fmaxf(fmaxf(m, mv[0]), fmaxf(mv[1], mv[2])), mv[3]);
    const float f = exp2f(m - mn);
    l *= f;
    o *= f;
    m = mn;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float fj = exp2f(mv[j] - mn);
      l += lv[j] * fj;
      o += ov[j] * fj;
    }
  }
  if constexpr (WPR > 1) {
    __shared__ float s_m[WPR], s_l[WPR];
    __shared__ f32x4 s_o[WPR][64];
    if (lane == 0) {
      s_m[q] = m;
      s_l[q] = l;
    }
    s_o[q][lane] = o;
    __syncthreads();
    if (q != 0) return;
#pragma unroll
    for (int k = 1; k < WPR; ++k) {
      const float mn = fmaxf(m, s_m[k]);
      const float f0 = exp2f(m - mn), f1 = exp2f(s_m[k] - mn);
      m = mn;
      l = l * f0 + s_l[k] * f1;
      o = o * f0 + s_o[k][lane] * f1;
    }
  }
  write_out(a, b, row, h, 4 * lane, o, l != 0.f ? 1.0f / l : 0.f);
}

struct PagedPlan {
  bool ok;
  int grp, R, RG, pairs, grid, nw, ks;
  size_t o_qs, o_po, o_ml, o_an, o_ws, o_ss, bytes;  // q first
};

PagedPlan paged_plan(int B, int T, int q_heads, int kv_heads, int max_blocks, int block_size, bool tree) {
  PagedPlan p{};
  if (tree && T > npn::kMaxNodes) return p;
  if (B < 1 || T < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || max_blocks < 1) return p;
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return p;
  p.grp = q_heads / kv_heads;
  const int64_t rows = (int64_t)T * p.grp;
  if (p.grp > 48 || rows > 1 << 20 || (int64_t)max_blocks * block_size > (int64_t)1 << 30) return p;
  // Groups of 128 against groups of 48: 32 requests of 54 rows 46 and 53 us, one of 54 27 and 31, 8 of 384 75
  // and 98, 2 of 1536 128 and 165; 16 of 96 146 and 148; but 4 of 192 59 and 54, one of 1536 over an empty
  // cache 35 and 30.
  p.R = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 48 ? 48 : kRows;
  // Trees have groups of 128 too, but where there are few pairs, and groups of 48 nearly full, those: one request of 96 rows
  // over 16384 keys of one head 30 us and 36 with groups of 128, two of 144 rows over 4 heads 49 and 54; 4 of 96 rows over
  // up to 16384 keys 53 and 52, 16 of them 158 and 126, 8 of 192 rows over up to 8192 91 and 77.
  const int64_t by48 = (rows + 47) / 48, by128 = (rows + kRows - 1) / kRows;
  if (tree && rows > 48 && by48 * 48 * 4 <= by128 * kRows * 3 && rows * 8 >= by48 * 48 * 7 && B * by48 * kv_heads < 32)
    p.R = 48;
  // And up to 64 rows two groups of 32, as of 128 half would be empty: one request of 60 rows over 32768 keys 39 us and 45
  // with a group of 128, 32 of them over up to 16384 186 and 193, 8 of 54 rows over up to 8192 49 and 51.5, 4 over up to
  // 2000 25 and 31. (72 rows as 48 and 24: 8 requests 59 us and 53 with a group of 128, 32 of them 220 and 197.)
  if (tree && rows > 48 && rows <= 64) p.R = 32;
  p.RG = (int)((rows + p.R - 1) / p.R);
  const int64_t pairs = (int64_t)B * p.RG * kv_heads;
  const int64_t keys = (int64_t)max_blocks * block_size;
  if (pairs > 65535 || pairs * ((keys + KS - 1) / KS) >= (int64_t)1 << 30) return p;
  p.pairs = (int)pairs;
  p.nw = p.R == 16 ? 8 : p.R == kRows ? 1 : 4;
  p.ks = p.R == kRows && !tree ? 2 * KS : KS;
  p.grid = max(most_workgroups(p.R, p.pairs, 1), most_workgroups(p.R, p.pairs, 2));
  const size_t slots = p.grid == 256 ? 256 : kSlots;
  const size_t units = (size_t)B * p.RG;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.o_qs = up((size_t)pairs * p.R * DH * (p.R == kRows && !tree ? 3 : 2));
  p.o_po = p.o_qs + up((size_t)pairs * p.R * sizeof(float));
  p.o_ml = p.o_po + up(slots * p.R * DH * sizeof(float));
  p.o_an = p.o_ml + up(slots * p.R * 2 * sizeof(float));
  p.o_ws = p.o_an + (tree ? up((size_t)B * T * sizeof(uint64_t)) : 0);
  p.o_ss = p.o_ws + up((units + 1) * sizeof(int32_t));
  p.bytes = p.o_ss + up(units * sizeof(int32_t));
  p.ok = true;
  return p;
}

int block_shift(int block_size) { return block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7; }

PagedArgs paged_args(const PagedPlan& p, const uint16_t* query, const uint16_t* gate, const float* q_norm,
                     const float* cos_table, const float* sin_table, int positions, const int8_t* cache_k,
                     const int8_t* cache_v, const float* k_scale, const float* v_scale,
                     const int32_t* block_table, const int32_t* kv_len, const int32_t* q_len, uint16_t* out,
                     int B, int T, int q_heads, int kv_heads, int n_blocks, int max_blocks, int block_size,
                     void* workspace) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return PagedArgs{query, gate, q_norm, cos_table, sin_table,
                   reinterpret_cast<const uint8_t*>(cache_k),
                   reinterpret_cast<const uint8_t*>(cache_v), k_scale, v_scale, block_table,
                   kv_len, q_len, out, reinterpret_cast<u32x4*>(ws),
                   reinterpret_cast<float*>(ws + p.o_qs), reinterpret_cast<float*>(ws + p.o_po),
                   reinterpret_cast<float*>(ws + p.o_ml), reinterpret_cast<uint64_t*>(ws + p.o_an),
                   reinterpret_cast<int32_t*>(ws + p.o_ws), reinterpret_cast<int32_t*>(ws + p.o_ss), positions,
                   B, T, q_heads, kv_heads, p.grp, p.R, p.RG, max_blocks, n_blocks, block_shift(block_size),
                   p.nw, p.ks, (1ull << 32) / p.grp + 1};
}

// The launches after the prep's.
template <bool TREE>
void launch_attn(const PagedPlan& p, const PagedArgs& a, hipStream_t s) {
  if (p.R == 16)
    hipLaunchKernelGGL((paged_attn_kernel<1, 8, TREE>), dim3(p.grid), dim3(512), 0, s, a);
  else if (p.R == 32)
    hipLaunchKernelGGL((paged_attn_kernel<2, 4, TREE>), dim3(p.grid), dim3(256), 0, s, a);
  else if (p.R == 48)
    hipLaunchKernelGGL((paged_attn_kernel<3, 4, TREE>), dim3(p.grid), dim3(256), 0, s, a);
  else if (TREE)
    hipLaunchKernelGGL(paged_tree_rows_kernel, dim3(p.grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(paged_rows_kernel, dim3(p.grid), dim3(512), 0, s, a);
  if (p.pairs < 32 || p.pairs * p.R < 96 * 16)
    hipLaunchKernelGGL(paged_merge_kernel<4>, dim3(p.R, p.pairs), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(paged_merge_kernel<1>, dim3(p.R / 4, p.pairs), dim3(256), 0, s, a);
}

}  // namespace

extern "C" size_t npn_gqa_tail_verify_paged_workspace_size(int B, int T, int q_heads, int kv_heads,
                                                           int max_blocks, int block_size) {
  return paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size, false).bytes;
}

extern "C" int npn_gqa_tail_verify_paged(
    const uint16_t* query, const uint16_t* gate, const float* q_norm, const float* cos_table,
    const float* sin_table, int positions, const int8_t* cache_k, const int8_t* cache_v,
    const float* k_scale, const float* v_scale, const int32_t* block_table, const int32_t* kv_len,
    const int32_t* q_len, uint16_t* out, int B, int T, int q_heads, int kv_heads, int n_blocks,
    int max_blocks, int block_size, void* workspace, size_t workspace_bytes, void* stream) {
  NPN_REQUIRE(query && gate && q_norm && cos_table && sin_table && cache_k && cache_v && k_scale &&
                  v_scale && block_table && kv_len && q_len && out, NPN_ERR_NULL);
  const PagedPlan p = paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size, false);
  NPN_REQUIRE(p.ok && n_blocks >= 1 && positions >= 1, NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(query) && NPN_ALIGNED16(gate) && NPN_ALIGNED16(q_norm) &&
                  NPN_ALIGNED16(cos_table) && NPN_ALIGNED16(sin_table) && NPN_ALIGNED16(cache_k) &&
                  NPN_ALIGNED16(cache_v) && NPN_ALIGNED16(out) && NPN_ALIGNED16(workspace),
              NPN_ERR_ALIGN);
  NPN_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes, NPN_ERR_WORKSPACE);
  const PagedArgs a = paged_args(p, query, gate, q_norm, cos_table, sin_table, positions, cache_k, cache_v,
                                 k_scale, v_scale, block_table, kv_len, q_len, out, B, T, q_heads, kv_heads,
                                 n_blocks, max_blocks, block_size, workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(paged_prep_kernel, dim3(1 + p.pairs * p.R / kPrepWaves), dim3(kPrepWaves * 64), 0, s, a);
  launch_attn<false>(p, a, s);
  return npn_launch_status();
}

extern "C" size_t npn_gqa_tree_verify_paged_workspace_size(int B, int T, int q_heads, int kv_heads,
                                                           int max_blocks, int block_size) {
  return paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size, true).bytes;
}

extern "C" int npn_gqa_tree_verify_paged(
    const uint16_t* query, const uint16_t* gate, const uint16_t* key, const uint16_t* value,
    const float* q_norm, const float* k_norm, const float* cos_table, const float* sin_table, int positions,
    int8_t* cache_k, int8_t* cache_v, float* k_scale, float* v_scale, const int32_t* block_table,
    const int32_t* kv_len, const int64_t* slots, const int32_t* q_len, const int32_t* parent, uint16_t* out,
    int B, int T, int q_heads, int kv_heads, int n_blocks, int max_blocks, int block_size, void* workspace,
    size_t workspace_bytes, void* stream) {
  NPN_REQUIRE(query && gate && key && value && q_norm && k_norm && cos_table && sin_table && cache_k &&
                  cache_v && k_scale && v_scale && block_table && kv_len && slots && q_len && parent && out,
              NPN_ERR_NULL);
  const PagedPlan p = paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size, true);
  NPN_REQUIRE(p.ok && n_blocks >= 1 && positions >= 1 && kv_heads <= 1024, NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(query) && NPN_ALIGNED16(gate) && NPN_ALIGNED16(key) && NPN_ALIGNED16(value) &&
                  NPN_ALIGNED16(q_norm) && NPN_ALIGNED16(k_norm) && NPN_ALIGNED16(cos_table) &&
                  NPN_ALIGNED16(sin_table) && NPN_ALIGNED16(cache_k) && NPN_ALIGNED16(cache_v) &&
                  NPN_ALIGNED16(out) && NPN_ALIGNED16(workspace),
              NPN_ERR_ALIGN);
  NPN_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes, NPN_ERR_WORKSPACE);
  const PagedArgs a = paged_args(p, query, gate, q_norm, cos_table, sin_table, positions, cache_k, cache_v,
                                 k_scale, v_scale, block_table, kv_len, q_len, out, B, T, q_heads, kv_heads,
                                 n_blocks, max_blocks, block_size, workspace);
  const append::PagedAppendArgs ap{key, value, k_norm, cos_table, sin_table, kv_len, slots,
                                   reinterpret_cast<uint8_t*>(cache_k), reinterpret_cast<uint8_t*>(cache_v),
                                   k_scale, v_scale, B, T, kv_heads, n_blocks, a.sh, positions};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int per = 1 + (T - 1 + block_size - 1) / block_size;  // a request's rows touch at most so many blocks
  const int appends = per * 2 * kv_heads * B;
  const int at_once = T < block_size ? T : block_size;
  // Four rows of q' to a wave where one each would be more waves than run at once: 24576 rows with their append 18 us
  // instead of 32, 6144 8.3 instead of 10.5; 512 rows with four to a wave 6.0 instead of 5.0.
  const int qr = p.pairs * p.R > 4096 ? 4 : 1;
  const int rows = p.pairs * p.R / (kPrepWaves * qr) + (p.pairs * p.R % (kPrepWaves * qr) != 0);  // workgroups of q'
  auto prep = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(1 + appends + rows), dim3(kPrepWaves * 64), 0, s, a, ap, parent, appends, per);
  };
  auto by_rows = [&](auto one, auto four) { qr == 4 ? prep(four) : prep(one); };
  if (at_once <= 8) by_rows(tree_prep_kernel<1, 1>, tree_prep_kernel<1, 4>);
  else if (at_once <= 16) by_rows(tree_prep_kernel<2, 1>, tree_prep_kernel<2, 4>);
  else if (at_once <= 32) by_rows(tree_prep_kernel<4, 1>, tree_prep_kernel<4, 4>);
  else by_rows(tree_prep_kernel<8, 1>, tree_prep_kernel<8, 4>);
  launch_attn<true>(p, a, s);
  return npn_launch_status();
}
