// GQA attention over the paged e4m3 KV cache for gfx950: T new tokens per request (1: plain
// decode, a few: a verify step, many: a prompt's chunk).
//
// Math per query row (b, t, head), t < q_len[b]:
//   q' = (1 + w) * q * rsqrt(mean(q^2) + 1e-6), partial RoPE on q'[:64] (rotate_half inside the
//   64); s_j = q'.K_j / 16 over the keys j <= kv_len[b] + t; out = (softmax(s) V) * sigmoid(gate),
//   K and V the e4m3 bytes times their (block, head) scale. Rows t >= q_len[b] are 0.
//
// The rows of a kv head (token-major, grp heads per token) are cut into groups of R = 16 NRT rows;
// a (request, row group, kv head) is a "pair" of its rows and its keys. Two launches:
//  1. attn: the pairs' 64-key steps are laid end to end and cut into W equal ranges, one per
//     workgroup of four waves; every workgroup finds its range from the lengths itself (the host
//     does not know them). Wave w takes every fourth step of a segment, on its own: no barrier and
//     no LDS between the loads and the products.
//       S^T[64 keys x 16 rows] = K Q'^T   A = K, 16 bytes per lane straight from the page: lane
//         (i, G) of tile j holds key 16 (i / 4) + 4 j + i % 4, dims 64 c + 16 G + [0, 16) for load
//         c; the product's k order follows (Q' lies in LDS in the same order), so the page row is
//         read as it is;
//       online softmax per row in fp32, base 2; that key order puts keys 16 G + [0, 16) of a row
//         into one lane, in order, so
//       O^T[256 x 16 rows] += V^T P^T     takes P straight from the score registers as B, and A = V^T
//         is 16 bytes of a page's dim row [dim][16 G + [0, 16)].
//     The bytes go from the pages to a part of LDS that is the wave's own by DMA (a lane reads back
//     the 16 bytes that it sent, so nothing but the wave's own vmcnt wait stands between), and
//     become bf16 with the page's scale in v_cvt_scalef32_pk_bf16_fp8, exactly (an e4m3 value times
//     a power of two is a bf16 number). The next step's K is sent for when this step's is used up,
//     V likewise, so a wave has 16 to 32 KB in flight and no register holds them (held in
//     registers, 128 a lane beside the accumulators, they spilled).
//     The four waves' (m, l, O) meet in LDS at the segment's end.
//  2. merge: the log-sum-exp merge of a pair's segments, times sigmoid(gate), to bf16.
#include "npn_common.h"

namespace {

constexpr int DH = 256;
constexpr int ROPE = 64;
constexpr float kEps = 1e-6f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1.0e30f;   // finite "no key yet" running max (avoids inf - inf)
constexpr float kRescaleLog2 = 8.0f;  // the exponent base moves only when a row max grows > 2^8
constexpr int KS = 64;                // keys per step
constexpr int kWaves = 4;
constexpr int kMaxWG = 256;           // one workgroup per CU: its rings fill the LDS
constexpr int kChunk = 64;            // steps whose page ids and scales are in LDS at a time
constexpr int kPages = kChunk * KS / 16 + 1;

typedef __bf16 bf16x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
typedef __bf16 bf16x2 __attribute__((__vector_size__(2 * sizeof(__bf16))));
typedef float f32x4 __attribute__((__vector_size__(4 * sizeof(float))));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

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
  float* part_o;           // [kMaxWG + pairs][R][256]
  float* part_ml;          // [kMaxWG + pairs][R][2]
  int32_t* ustart;         // [U + 2]: first step of each unit, all steps, workgroups
  int positions, B, T, Hq, Hkv, grp, R, RG, P, N, sh, min_steps;
};

// Unit u = (request, row group): its keys [0, kend) and the tokens it covers.
struct Unit {
  int b, t0, kv, kend, steps;
};

__device__ __forceinline__ Unit unit_of(const PagedArgs& a, int u) {
  Unit r;
  r.b = u / a.RG;
  const int rg = u - r.b * a.RG;
  r.t0 = rg * a.R / a.grp;  // the group's first token
  const int t1 = min(((rg + 1) * a.R - 1) / a.grp, a.T - 1);
  const int n = min(min(a.q_len[r.b], a.T), t1 + 1);  // tokens up to the group's last live one
  const int cap = a.P << a.sh;  // <= 2^30
  r.kv = min(max(a.kv_len[r.b], 0), cap);
  r.kend = n > r.t0 ? min(r.kv + n, cap) : 0;
  r.steps = (r.kend + KS - 1) / KS;
  return r;
}

// Workgroups that take part for S steps.
__device__ __forceinline__ int paged_wgs(int S, int min_steps, int most) {
  return max(1, min(most, S / min_steps));
}

__device__ __forceinline__ int wg_first_step(int w, int S, int W) {
  return (int)((int64_t)w * S / W);
}

__device__ __forceinline__ float max_over_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
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

// A word's bytes of keys [0, n) kept, n <= 0: none, n >= 4: all.
__device__ __forceinline__ uint32_t keep_bytes(int n) {
  return n >= 4 ? ~0u : (n <= 0 ? 0u : (1u << (8 * n)) - 1);
}
// 0xFF in each byte that is an e4m3 NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t t = (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
  return t * 0xFFu;
}

// 16 bytes per lane from g into LDS at lds + 16 * lane (global_load_lds_dwordx4, its LDS base in m0:
// see npn::lds_dma16); lds is wave-uniform. The caller waits with vmcnt.
__device__ __forceinline__ void dma16(const void* g, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(g), "s"(lds)
      : "memory");
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
__device__ __forceinline__ unsigned opaque(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int NRT>
struct PagedSmem {
  union {
    struct {
      u32x4 k[4][4][64];                  // a step's K as sent: [key tile][64-dim column][lane]
      u32x4 v[16][64];                    // and V: [dim tile][lane]
    } ring[kWaves];
    f32x4 o[2][NRT][16][64];              // two waves' O on their way to the other two
  };
  u32x4 q[8][NRT][64];                    // q' as B operands: [k step][row tile][lane]
  float m[kWaves][NRT * 16], l[kWaves][NRT * 16];
  int page[kPages];                       // -1: none
  float ks[kPages], vs[kPages];
  int scan[256];
};

template <int NRT>
__global__ __launch_bounds__(256, 1) void paged_attn_kernel(PagedArgs a) {
  constexpr int R = NRT * 16;
  __shared__ __attribute__((aligned(16))) PagedSmem<NRT> sm;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int i = lane & 15, G = lane >> 4;
  const int bs = 1 << a.sh;
  const int U = a.B * a.RG;
  const unsigned ring_lds = __builtin_amdgcn_readfirstlane(npn::lds_addr(&sm.ring[w]));
  const unsigned k_at = opaque(npn::lds_addr(&sm.ring[w].k[0][0][lane]));
  const unsigned v_at = opaque(npn::lds_addr(&sm.ring[w].v[0][lane]));
  const unsigned q_at = opaque(npn::lds_addr(&sm.q[0][0][lane]));
  const unsigned o_at = opaque(npn::lds_addr(&sm.o[0][0][0][lane]));

  // The steps of all units: thread t sums its slice of them, and a scan over the slices.
  const int per = (U + 255) / 256;
  const int u0 = min(U, tid * per), u1 = min(U, u0 + per);
  int mine = 0;
  for (int u = u0; u < u1; ++u) mine += unit_of(a, u).steps;
  sm.scan[tid] = mine * a.Hkv;
  __syncthreads();
  for (int off = 1; off < 256; off <<= 1) {
    const int v = tid >= off ? sm.scan[tid - off] : 0;
    __syncthreads();
    sm.scan[tid] += v;
    __syncthreads();
  }
  const int S = sm.scan[255];
  const int W = paged_wgs(S, a.min_steps, (int)gridDim.x);
  if (blockIdx.x == 0) {  // the merge finds the segments by these
    int run = sm.scan[tid] - mine * a.Hkv;
    for (int u = u0; u < u1; ++u) {
      a.ustart[u] = run;
      run += unit_of(a, u).steps * a.Hkv;
    }
    if (tid == 0) {
      a.ustart[U] = S;
      a.ustart[U + 1] = W;
    }
  }
  if ((int)blockIdx.x >= W) return;
  int x = wg_first_step(blockIdx.x, S, W);
  const int x_end = wg_first_step(blockIdx.x + 1, S, W);
  if (x >= x_end) return;

  // The unit of step x: the slice with it, then the unit inside the slice.
  int slice = 0;
  for (int n = 256; n > 1;) {
    const int half = n >> 1;
    if (sm.scan[slice + half - 1] <= x) {
      slice += half;
      n -= half;
    } else {
      n = half;
    }
  }
  int u = __builtin_amdgcn_readfirstlane(slice * per);
  int ubeg = __builtin_amdgcn_readfirstlane(slice > 0 ? sm.scan[slice - 1] : 0);
  Unit un = unit_of(a, u);
  while (ubeg + un.steps * a.Hkv <= x) {
    ubeg += un.steps * a.Hkv;
    un = unit_of(a, ++u);
  }

  while (x < x_end) {
    const int h = (x - ubeg) / un.steps;
    const int s_lo = (x - ubeg) - h * un.steps;
    const int steps = min(x_end - x, un.steps - s_lo);
    const int pair = u * a.Hkv + h;
    const int row0 = (u - un.b * a.RG) * R;  // the group's first row
    const int rows = min(R, a.T * a.grp - row0);

    // q' of the group's rows, as B operands in LDS: wave w prepares rows w, w + 4, ...
    __syncthreads();  // the previous segment is done with LDS
    {
      const float4 nw = *reinterpret_cast<const float4*>(a.q_norm + 4 * lane);
      for (int r = w; r < R; r += kWaves) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
          const int t = (row0 + r) / a.grp, qh = h * a.grp + (row0 + r) - t * a.grp;
          const uint2 p = *reinterpret_cast<const uint2*>(
              a.query + (((size_t)un.b * a.T + t) * a.Hq + qh) * DH + 4 * lane);
          v[0] = npn::bf16lo(p.x);
          v[1] = npn::bf16hi(p.x);
          v[2] = npn::bf16lo(p.y);
          v[3] = npn::bf16hi(p.y);
          const float ss = npn::wave_sum(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]);
          const float rn = rsqrtf(ss * (1.0f / DH) + kEps);
          v[0] = (1.0f + nw.x) * (v[0] * rn);
          v[1] = (1.0f + nw.y) * (v[1] * rn);
          v[2] = (1.0f + nw.z) * (v[2] * rn);
          v[3] = (1.0f + nw.w) * (v[3] * rn);
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = __shfl_xor(v[j], 8, 64);  // dim d ^ 32
          if (lane < ROPE / 4) {
            const int64_t pos = min((int64_t)un.kv + t, (int64_t)a.positions - 1);
            const float4 c = *reinterpret_cast<const float4*>(a.cos + pos * ROPE + 4 * lane);
            const float4 s = *reinterpret_cast<const float4*>(a.sin + pos * ROPE + 4 * lane);
            const float sg = lane < ROPE / 8 ? -1.0f : 1.0f;
            v[0] = v[0] * c.x + sg * y[0] * s.x;
            v[1] = v[1] * c.y + sg * y[1] * s.y;
            v[2] = v[2] * c.z + sg * y[2] * s.z;
            v[3] = v[3] * c.w + sg * y[3] * s.w;
          }
        }
        uint32_t b[2];
        constexpr float scale = kLog2e / 16.0f;  // softmax scale 1/sqrt(256), in base 2
#pragma unroll
        for (int j = 0; j < 2; ++j)
          b[j] = npn::f32_to_bf16(v[2 * j] * scale) |
                 ((uint32_t)npn::f32_to_bf16(v[2 * j + 1] * scale) << 16);
        // dim d = 64 c + 16 g + 8 h + e sits in k step 2 c + h, lane group g, element e
        const int d = 4 * lane;
        const int step = 2 * (d >> 6) + ((d >> 3) & 1), g = (d >> 4) & 3;
        uint32_t* dst = reinterpret_cast<uint32_t*>(&sm.q[step][r >> 4][16 * g + (r & 15)]) +
                        ((d & 4) >> 1);
        dst[0] = b[0];
        dst[1] = b[1];
      }
    }

    // The last key of each of this lane's rows (one per tile); -1 for rows that are none.
    int lim[NRT];
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
      const int r = 16 * nt + i, t = (row0 + r) / a.grp;
      lim[nt] = r < rows && t < a.q_len[un.b] ? min(un.kv + t, un.kend - 1) : -1;
    }
    const int lim0 = un.kv + un.t0;  // no row of the group sees less

    float m_run[NRT], l_run[NRT];
    f32x4 acc[NRT][16];
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
      m_run[nt] = kNegBig;
      l_run[nt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) acc[nt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    for (int c0 = 0; c0 < steps; c0 += kChunk) {
      const int cn = min(kChunk, steps - c0);
      const int key0 = (s_lo + c0) * KS;
      const int page0 = key0 >> a.sh;
      const int pages = ((min(key0 + cn * KS, un.kend) - 1) >> a.sh) - page0 + 1;
      __syncthreads();  // the last chunk's pages have been used; q' is in LDS
      for (int p = tid; p < kPages; p += 256) {
        int id = -1;
        if (p < pages) id = a.table[(size_t)un.b * a.P + page0 + p];
        const bool ok = id >= 0 && id < a.N;
        sm.page[p] = ok ? id : -1;
        sm.ks[p] = ok ? a.k_scale[(size_t)id * a.Hkv + h] : 1.0f;
        sm.vs[p] = ok ? a.v_scale[(size_t)id * a.Hkv + h] : 1.0f;
      }
      __syncthreads();

      auto load_k = [&](int s) {
        const int key = key0 + s * KS + 16 * (i >> 2);
        const int id = max(sm.page[(key >> a.sh) - page0], 0);
        const uint8_t* p = a.cache_k +
            ((((size_t)id * a.Hkv + h) << a.sh) + (key & (bs - 1)) + (i & 3)) * DH + 16 * G;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) dma16(p + j * 4 * DH + c * 64, ring_lds + (j * 4 + c) * 1024);
      };
      auto load_v = [&](int s) {
        const int key = key0 + s * KS + 16 * G;
        const int id = max(sm.page[(key >> a.sh) - page0], 0);
        const uint8_t* p = a.cache_v + ((((size_t)id * a.Hkv + h) * DH + i) << a.sh) + (key & (bs - 1));
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
          dma16(p + ((size_t)dt << (a.sh + 4)), ring_lds + 16384 + dt * 1024);
      };
      if (w < cn) {
        load_k(w);
        load_v(w);
      }
      for (int s = w; s < cn; s += kWaves) {
        const int k0 = key0 + s * KS;
        const float ks = sm.ks[((k0 + 16 * (i >> 2)) >> a.sh) - page0];
        const int vpage = ((k0 + 16 * G) >> a.sh) - page0;
        const float vs = sm.vs[vpage];
        const bool held = sm.page[vpage] >= 0;  // this lane's 16 keys exist
        const bool next = s + kWaves < cn;

        // The 16 DMAs of this step's K are older than the 16 of its V.
        asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        f32x4 st[NRT][4];
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) st[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4 kw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) kw[j] = lds_read(k_at, 4 * j + c);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            bf16x8 q[NRT];
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
              q[nt] = __builtin_bit_cast(bf16x8, lds_read(q_at, (2 * c + half) * NRT + nt));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bf16x8 kf = dequant8(kw[j][2 * half], kw[j][2 * half + 1], ks);
#pragma unroll
              for (int nt = 0; nt < NRT; ++nt)
                st[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[nt], st[nt][j], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (next) {  // this step's K has been read into registers
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          load_k(s + kWaves);
        }

        // A step with keys past the group's first limit, or past a page that is none, is masked.
        const bool tail = k0 + KS - 1 > lim0 || __builtin_amdgcn_ballot_w64(!held) != 0;
        if (tail) {
          const int kb = k0 + 16 * G;
#pragma unroll
          for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (!held || kb + 4 * j + r > lim[nt]) st[nt][j][r] = -INFINITY;
        }

        bf16x8 p[NRT][2];
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
          float mx = st[nt][0][0];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[nt][j][r]);
          mx = max_over_groups(mx);
          const bool grow = mx > m_run[nt] + kRescaleLog2;
          if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float mnew = grow ? mx : m_run[nt];
            const float corr = exp2f(m_run[nt] - mnew);
            m_run[nt] = mnew;
            l_run[nt] *= corr;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) acc[nt][dt] *= corr;
          }
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float pv = __builtin_amdgcn_exp2f(st[nt][j][r] - m_run[nt]);
              sum += pv;
              p[nt][j >> 1][(j & 1) * 4 + r] = (__bf16)pv;
            }
          l_run[nt] += sum;
        }

        if (next)
          asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (tail) {
          // V bytes of keys that no row sees are cleared (0 times NaN is NaN). A NaN at a key that
          // some rows see reaches those and no others: the rows' products with "is NaN" say which
          // outputs become NaN, and the byte is then cleared too.
          const int live = held ? un.kend - (k0 + 16 * G) : 0;
          uint32_t nan_seen = 0;
#pragma unroll 1
          for (int dt = 0; dt < 16; ++dt) {
            u32x4 v = lds_read(v_at, dt);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[k] &= keep_bytes(live - 4 * k);
              nan_seen |= nan_bytes(v[k]);
            }
            lds_write(v_at, dt, v);
          }
          if (__builtin_amdgcn_ballot_w64(nan_seen != 0) != 0) {
            bf16x8 see[NRT][2];
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                see[nt][e >> 3][e & 7] = (__bf16)(k0 + 16 * G + e <= lim[nt] ? 1.0f : 0.0f);
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) {
              u32x4 v = lds_read(v_at, dt), is;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                is[k] = nan_bytes(v[k]) & 0x38383838u;  // e4m3 1.0
                v[k] &= ~nan_bytes(v[k]);
              }
              lds_write(v_at, dt, v);
#pragma unroll
              for (int nt = 0; nt < NRT; ++nt) {
                f32x4 hit = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      dequant8(is[2 * k], is[2 * k + 1], 1.0f), see[nt][k], hit, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (hit[r] > 0.f) acc[nt][dt][r] = NAN;
              }
            }
          }
        }
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
          const u32x4 v = lds_read(v_at, dt);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const bf16x8 vf = dequant8(v[2 * k], v[2 * k + 1], vs);
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt)
              acc[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, p[nt][k], acc[nt][dt], 0, 0, 0);
          }
          if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        if (next) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          load_v(s + kWaves);
        }
      }
    }

    // The four waves' rows meet: all scaled to the common maximum, then waves 2 and 3 hand theirs
    // to 0 and 1, and 1 to 0.
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
      l_run[nt] = sum_over_groups(l_run[nt]);
      if (G == 0) {
        sm.m[w][16 * nt + i] = m_run[nt];
        sm.l[w][16 * nt + i] = l_run[nt];
      }
    }
    __syncthreads();
    float m_all[NRT], l_all[NRT];
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
      float m = kNegBig, l = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = fmaxf(m, sm.m[k][16 * nt + i]);
#pragma unroll
      for (int k = 0; k < kWaves; ++k) l += exp2f(sm.m[k][16 * nt + i] - m) * sm.l[k][16 * nt + i];
      m_all[nt] = m;
      l_all[nt] = l;
      const float f = exp2f(m_run[nt] - m);
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) acc[nt][dt] *= f;
    }
    __syncthreads();  // every wave is done with its ring, which O takes over
    auto put = [&](int k) {
      const unsigned at = o_at + (unsigned)(k * sizeof(sm.o[0]));
#pragma unroll
      for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
          lds_write(at, nt * 16 + dt, __builtin_bit_cast(u32x4, acc[nt][dt]));
    };
    auto add = [&](int k) {
      const unsigned at = o_at + (unsigned)(k * sizeof(sm.o[0]));
#pragma unroll
      for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
          acc[nt][dt] += __builtin_bit_cast(f32x4, lds_read(at, nt * 16 + dt));
          if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (w >= 2) put(w - 2);
    __syncthreads();
    if (w < 2) add(w);
    if (w == 1) put(1);  // its own buffer, read by itself alone
    __syncthreads();
    if (w == 0) {
      add(1);
      const size_t slot = (size_t)blockIdx.x + pair;  // unique: a workgroup's pairs are consecutive
#pragma unroll
      for (int nt = 0; nt < NRT; ++nt) {
        const int r = 16 * nt + i;
        float* po = a.part_o + (slot * R + r) * DH;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt + 4 * G) = acc[nt][dt];
        if (G == 0) {
          a.part_ml[(slot * R + r) * 2] = m_all[nt];
          a.part_ml[(slot * R + r) * 2 + 1] = l_all[nt];
        }
      }
    }

    x += steps;
    if (x - ubeg >= un.steps * a.Hkv && x < x_end) {
      do {
        ubeg += un.steps * a.Hkv;
        un = unit_of(a, ++u);
      } while (un.steps == 0);  // ends: a step of a later unit is in this range
    }
  }
}

// One wave per (row of a pair): the segments' (m, l, O) merged in segment order.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  const int q = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + q;
  const int pair = blockIdx.y;
  const int u = pair / a.Hkv, h = pair - u * a.Hkv;
  const int b = u / a.RG;
  const int row = (u - b * a.RG) * a.R + r;
  if (r >= a.R || row >= a.T * a.grp) return;
  const int t = row / a.grp, qh = h * a.grp + row - t * a.grp;
  const size_t oi = (((size_t)b * a.T + t) * a.Hq + qh) * DH + 4 * lane;
  const int U = a.B * a.RG;
  const int S = a.ustart[U], W = a.ustart[U + 1];
  const int ub = a.ustart[u], steps = (a.ustart[u + 1] - ub) / a.Hkv;
  float m = kNegBig, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (steps > 0 && t < a.q_len[b]) {
    const int x0 = ub + h * steps, x1 = x0 + steps - 1;
    const int w0 = (int)(((int64_t)(x0 + 1) * W - 1) / S);
    const int w1 = (int)(((int64_t)(x1 + 1) * W - 1) / S);
    for (int w = w0; w <= w1; ++w) {
      const size_t at = ((size_t)w + pair) * a.R + r;
      const float mv = a.part_ml[2 * at], lv = a.part_ml[2 * at + 1];
      const f32x4 ov = *reinterpret_cast<const f32x4*>(a.part_o + at * DH + 4 * lane);
      const float mn = fmaxf(m, mv);
      const float f0 = exp2f(m - mn), f1 = exp2f(mv - mn);
      m = mn;
      l = l * f0 + lv * f1;
      o = o * f0 + ov * f1;
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;  // a row without keys (pages that are none) is 0
  const uint2 g = *reinterpret_cast<const uint2*>(a.gate + oi);
  const uint32_t gw[2] = {g.x, g.y};
  uint32_t y[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float v0 = o[2 * j] * inv * npn::sigmoid(npn::bf16lo(gw[j]));
    float v1 = o[2 * j + 1] * inv * npn::sigmoid(npn::bf16hi(gw[j]));
    if (l == 0.f) v0 = v1 = 0.f;  // whatever the gate
    y[j] = npn::f32_to_bf16(v0) | ((uint32_t)npn::f32_to_bf16(v1) << 16);
  }
  *reinterpret_cast<uint2*>(a.out + oi) = make_uint2(y[0], y[1]);
}

struct PagedPlan {
  bool ok;
  int grp, R, RG, pairs;
  size_t o_ml, o_us, bytes;  // part_o first
};

PagedPlan paged_plan(int B, int T, int q_heads, int kv_heads, int max_blocks, int block_size) {
  PagedPlan p{};
  if (B < 1 || T < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || max_blocks < 1) return p;
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return p;
  p.grp = q_heads / kv_heads;
  const int64_t rows = (int64_t)T * p.grp;
  if (p.grp > 48 || rows > 1 << 20 || (int64_t)max_blocks * block_size > (int64_t)1 << 30) return p;
  p.R = rows <= 16 ? 16 : (rows <= 32 ? 32 : 48);
  p.RG = (int)((rows + p.R - 1) / p.R);
  const int64_t pairs = (int64_t)B * p.RG * kv_heads;
  const int64_t keys = (int64_t)max_blocks * block_size;
  if (pairs > 65535 || pairs * ((keys + KS - 1) / KS) >= (int64_t)1 << 31) return p;
  p.pairs = (int)pairs;
  const size_t slots = (size_t)kMaxWG + p.pairs;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.o_ml = up(slots * p.R * DH * sizeof(float));
  p.o_us = p.o_ml + up(slots * p.R * 2 * sizeof(float));
  p.bytes = p.o_us + up(((size_t)B * p.RG + 2) * sizeof(int32_t));
  p.ok = true;
  return p;
}

}  // namespace

extern "C" size_t npn_gqa_tail_verify_paged_workspace_size(int B, int T, int q_heads, int kv_heads,
                                                           int max_blocks, int block_size) {
  return paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size).bytes;
}

extern "C" int npn_gqa_tail_verify_paged(
    const uint16_t* query, const uint16_t* gate, const float* q_norm, const float* cos_table,
    const float* sin_table, int positions, const int8_t* cache_k, const int8_t* cache_v,
    const float* k_scale, const float* v_scale, const int32_t* block_table, const int32_t* kv_len,
    const int32_t* q_len, uint16_t* out, int B, int T, int q_heads, int kv_heads, int n_blocks,
    int max_blocks, int block_size, void* workspace, size_t workspace_bytes, void* stream) {
  NPN_REQUIRE(query && gate && q_norm && cos_table && sin_table && cache_k && cache_v && k_scale &&
                  v_scale && block_table && kv_len && q_len && out, NPN_ERR_NULL);
  const PagedPlan p = paged_plan(B, T, q_heads, kv_heads, max_blocks, block_size);
  NPN_REQUIRE(p.ok && n_blocks >= 1 && positions >= 1, NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(query) && NPN_ALIGNED16(gate) && NPN_ALIGNED16(q_norm) &&
                  NPN_ALIGNED16(cos_table) && NPN_ALIGNED16(sin_table) && NPN_ALIGNED16(cache_k) &&
                  NPN_ALIGNED16(cache_v) && NPN_ALIGNED16(out) && NPN_ALIGNED16(workspace),
              NPN_ERR_ALIGN);
  NPN_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes, NPN_ERR_WORKSPACE);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int sh = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  const PagedArgs a{query, gate, q_norm, cos_table, sin_table,
                    reinterpret_cast<const uint8_t*>(cache_k),
                    reinterpret_cast<const uint8_t*>(cache_v), k_scale, v_scale, block_table,
                    kv_len, q_len, out, reinterpret_cast<float*>(ws),
                    reinterpret_cast<float*>(ws + p.o_ml), reinterpret_cast<int32_t*>(ws + p.o_us),
                    positions, B, T, q_heads, kv_heads, p.grp, p.R, p.RG, max_blocks, n_blocks, sh, 4};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int nrt = p.R / 16;
  if (nrt == 1)
    hipLaunchKernelGGL(paged_attn_kernel<1>, dim3(kMaxWG), dim3(256), 0, s, a);
  else if (nrt == 2)
    hipLaunchKernelGGL(paged_attn_kernel<2>, dim3(kMaxWG), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(paged_attn_kernel<3>, dim3(kMaxWG), dim3(256), 0, s, a);
  hipLaunchKernelGGL(paged_merge_kernel, dim3(p.R / 4, p.pairs), dim3(256), 0, s, a);
  return npn_launch_status();
}
