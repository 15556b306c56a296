// Gated DeltaNet over a tree of drafted tokens for gfx950: every node's output from the committed state
// (verify), and the state moved along the accepted path (commit). The token step is deltanet.hip's.
//
// Math (request b, v-head h, node t with parent p, k-head h / (Hv/Hk)): conv window = the last three inputs of
// t's ancestors (before the first: conv_state) and x_t; y = silu(w . window + bias); q, k L2-normalised (q
// also / sqrt(128)); g = -exp(A_log) softplus(a + dt_bias); beta = sigmoid(b);
//   S_t = e^g_t S_p;  u_t = beta_t (v_t - S_t^T k_t);  S_t += k_t u_t^T;  o_t = S_t^T q_t
//   out_t = o_t rsqrt(mean o_t^2 + 1e-6) norm_w silu(z_t)
// A state per node would be 64 KB for each node and head. None is formed: with G_t the sum of g over t and its
// ancestors, D(t, s) = e^(G_t - G_s) and sums over t's ancestors s (for o also t itself),
//   u_t = beta_t (v_t - e^G_t S0^T k_t - sum_s D(t, s) (k_s . k_t) u_s)
//   o_t = e^G_t S0^T q_t + sum_s D(t, s) (k_s . q_t) u_s
// so that S0 is read once, whatever the tree, and what the commit needs is two rows a node:
//   S_n = (prod decay) S0 + sum_s (prod of the later decays) k_s u_s^T over the path.
// The sums of g are in 64 bits (each g at least -256, which is a decay of 0): the difference of two far from 0 is
// exact to more than fp32's rounding.
#include "tree.h"

namespace {

constexpr int D = 128;
constexpr float kEps = 1e-6f;

struct TreeArgs {
  const float* state;           // [B][Hv][128][128]
  const int32_t* parent;        // [B][T]
  const uint16_t* mixed_qkv;    // [B][T][QKV]
  const uint16_t* conv_state;   // [B][QKV][3]
  const float* conv_weight;     // [QKV][4]
  const float* conv_bias;
  const float* a_out;           // [B][T][Hv]
  const float* b_out;
  const uint16_t* z;            // [B][T][Hv][128]
  const float* A_log;
  const float* dt_bias;
  const float* norm_weight;
  uint16_t* out;                // [B][T][Hv][128]
  float* rec_k;                 // [B][T][Hk][128]
  float* rec_u;                 // [B][T][Hv][128]
  float* rec_decay;             // [B][T][Hv]
  int B, T, Hk, Hv;
};

typedef _Float16 f16x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));
typedef _Float16 f16x2 __attribute__((__vector_size__(2 * sizeof(_Float16))));
typedef __bf16 bf16x2 __attribute__((__vector_size__(2 * sizeof(__bf16))));
typedef float f32x4 __attribute__((__vector_size__(4 * sizeof(float))));

// One workgroup of NW waves a (b, h); NT tiles of 16 nodes; wave w has columns CT (16 w + i) + [0, CT), CT = 8 / NW, of
// everything that has the state's columns (lane (i, G): i = lane % 16, G = lane / 16), so that the products' results are the
// next ones' operands where they are. Steps, with a barrier between them:
//   1. conv, SiLU and norms, a row of 128 channels to a wave at a time, two channels a lane, into LDS;
//   2. K S0, Q S0 and, tile by tile of the lower triangle, K K^T and Q K^T. In f16 MFMAs: a number is the sum of two
//      f16 (x 2^12, the state's columns over a power of two of their own), of whose four products the
//      smallest is left out: 22 bits each, accumulated in fp32, a fifth of fp32 MFMAs' time;
//   3. the inverses of the NT diagonal 16 x 16 blocks of 1 - low, low(t, s) = -beta_t D(t, s) (k_s . k_t) at t's
//      ancestors s, by forward substitution (low's powers may grow where its inverse does not);
//   4. block by block u = inverse (beta (v - e^G K S0) + low u of the blocks before), then o = e^G Q S0 + (D Q K^T) u,
//      in fp32 MFMAs;
//   5. the norm over the workgroup's columns, z and the output.
// A node whose input is not finite has zeros in these sums, which reach all nodes of a tile, and is noted: NaN
// goes to its own and its descendants' rows at the end.
// APART: q's rows take k's place once those have been used, and v's after them, so that two workgroups of 64 nodes fit a CU.
//
// Bound by the state and the rows' bytes where heads are many and trees small: 1536 heads of 16 nodes 37.5 us (141 MB, 27.4
// at a copy's rate); by the length of the steps above, one behind the other with a barrier between, where a CU has a head
// or two: 48 heads of 16 nodes 9.2 us, of 64 nodes 21.7, 384 heads of 64 nodes 37.5 (65 MB, 13 us; its products take 5);
// calls one behind the other, traced alone 9.8 and 40 for the first and the last.
template <int NT, int NW, bool APART>
struct TreeSmem {
  static constexpr int TM = 16 * NT, kTiles = NT * (NT + 1) / 2;
  union {
    struct {
      union {
        _Float16 x[2][APART ? TM : 2 * TM][D + 8];  // high and low parts of k's rows, then q's
        float v_apart[APART ? TM : 1][D + 4];
      };
      float low[kTiles][16][20], mix[kTiles][16][20];  // tile (a, s), s <= a, at a (a + 1) / 2 + s
    };
    uint32_t raw[3][3 + TM][64];  // the inputs of q, k, v: conv_state's, then the nodes'
  };
  float v[APART ? 1 : TM][D + 4];
  float inv[NT][16][20];
  float begun[TM], beta[TM], ss[NW][TM];
  double g[TM];  // sums of g along a node's line, base 2
  uint64_t anc[TM];
  uint64_t bad_kv[NW], bad_q[NW];  // by wave
  unsigned long long bad_u;
};
constexpr int tile_at(int a, int s) { return a * (a + 1) / 2 + s; }

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
// x sigmoid(x) to 2 ulp: the reciprocal's one and the product's. (0 where e^-x overflows.)
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

// Maximum over the lanes (i, G) of a column i.
__device__ __forceinline__ float max_over_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Sum over a row of 16 lanes.
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float(npn::dpp32<npn::kDppStep[0]>(__float_as_uint(x)));
  x += __uint_as_float(npn::dpp32<npn::kDppStep[1]>(__float_as_uint(x)));
  x += __uint_as_float(npn::dpp32<npn::kDppStep[2]>(__float_as_uint(x)));
  return x + __uint_as_float(npn::dpp32<npn::kDppStep[3]>(__float_as_uint(x)));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = row_sum(x);
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Four products over k = 16: lane (i, G) has the row's (a) or column's (b) k 4 G + [0, 4), b as a result has its rows.
__device__ __forceinline__ f32x4 mfma_f32(const float4 a, const f32x4 b, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b[2], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b[3], c, 0, 0, 0);
}

// N neighbouring floats.
template <int N>
struct Floats {
  float x[N];
};

template <int NT, int NW, bool APART>
__global__ __launch_bounds__(64 * NW, NW == 4 && (NT == 1 || APART) ? 2 : NW / 4) void dn_tree_verify_kernel(TreeArgs a) {
  constexpr int TM = 16 * NT;
  constexpr int CT = 8 / NW;              // column tiles of a wave
  constexpr int RW = TM / NW;             // rows of a wave in step 1
  constexpr float kUnit = 4096.0f;        // the rows' scale in f16
  __shared__ __attribute__((aligned(16))) TreeSmem<NT, NW, APART> sm;
  const int T = a.T, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, G = lane >> 4;
  const int b = blockIdx.x / a.Hv, h = blockIdx.x - b * a.Hv, kh = h / (a.Hv / a.Hk);
  const int QKV = (2 * a.Hk + a.Hv) * D;
  const int col = CT * (16 * w + i);      // this lane's first column

  // Loads return in order: what is needed first goes first, the state last.
  const int parent = npn::tree_parent(a.parent + (size_t)b * T, T, lane);
  constexpr int kGates = NW - 1;          // the wave that has the gates
  float in_a = 0.f, in_b = 0.f, in_log = 0.f, in_dt = 0.f;
  if (w == kGates) {
    const size_t gi = ((size_t)b * T + min(lane, T - 1)) * a.Hv + h;
    in_a = a.a_out[gi];
    in_b = a.b_out[gi];
    in_log = a.A_log[h];
    in_dt = a.dt_bias[h];
  }
  uint32_t raw[3][RW];                    // node w + NW k's inputs of two channels, q, k, v
  float4 wt[3][2];
  float2 bias[3];
  uint32_t old[3][3];                     // conv_state's
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    const int c = (which == 0 ? kh : which == 1 ? a.Hk + kh : 2 * a.Hk + h) * D + 2 * lane;
    const uint16_t* xb = a.mixed_qkv + (size_t)b * T * QKV + c;
#pragma unroll
    for (int k = 0; k < RW; ++k)
      raw[which][k] = *reinterpret_cast<const uint32_t*>(xb + (size_t)min(w + NW * k, T - 1) * QKV);
    wt[which][0] = *reinterpret_cast<const float4*>(a.conv_weight + 4 * c);
    wt[which][1] = *reinterpret_cast<const float4*>(a.conv_weight + 4 * c + 4);
    bias[which] = make_float2(a.conv_bias[c], a.conv_bias[c + 1]);
    const uint32_t* cs = reinterpret_cast<const uint32_t*>(a.conv_state + ((size_t)b * QKV + c) * 3);
#pragma unroll
    for (int j = 0; j < 3; ++j) old[which][j] = cs[j];
  }
  __builtin_amdgcn_sched_barrier(0);
  // The state, lane (i, G): rows 32 s + 8 G + e of its columns.
  const float* S0 = a.state + ((size_t)b * a.Hv + h) * D * D;
  const unsigned s_at = 8 * G * D + col;
  Floats<CT> s0[4][8];
  auto load_state = [&]() {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) s0[s][e] = *reinterpret_cast<const Floats<CT>*>(S0 + 32 * s * D + (s_at + e * D));
    __builtin_amdgcn_sched_barrier(0);
  };
  if constexpr (!APART) load_state();

  // Lane t: the rows below of node t's inputs one to three back.
  int tap[3];
  {
    int at = lane;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int up = __shfl(parent, max(at, 0), 64);
      at = at < 0 ? at - 1 : up;
      tap[j] = 3 + at;
    }
  }
  // 1. The inputs wait in LDS, a node t's in row 3 + t, those before the first node's in rows 0 to 2.
  if (w == 0) {
#pragma unroll
    for (int which = 0; which < 3; ++which) {  // [c0 c0][c0 c1][c1 c1], oldest first, to a word a step
      const uint32_t x = old[which][0], y = old[which][1], v = old[which][2];
      sm.raw[which][0][lane] = (x & 0xFFFFu) | (y & 0xFFFF0000u);
      sm.raw[which][1][lane] = (x >> 16) | (v << 16);
      sm.raw[which][2][lane] = (y & 0xFFFFu) | (v & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int which = 0; which < 3; ++which)
#pragma unroll
    for (int k = 0; k < RW; ++k) sm.raw[which][3 + w + NW * k][lane] = raw[which][k];
  uint64_t bad_kv = 0, bad_q = 0;  // wave-uniform
  if (w == kGates) {
    const float gf = -__expf(in_log) * npn::softplus(in_a + in_dt);
    float beta = npn::sigmoid(in_b);
    if (lane < T) a.rec_decay[((size_t)b * T + lane) * a.Hv + h] = __expf(gf);
    const bool bad = gf != gf || beta != beta;
    bad_kv = __builtin_amdgcn_ballot_w64(bad && lane < T);
    beta = bad || lane >= T ? 0.f : beta;
    double total = bad || lane >= T ? 0.0 : (double)fmaxf(gf, -256.0f) * 1.4426950408889634;
    const uint64_t anc = npn::tree_ancestors(parent, T, lane, total);
    if (lane < TM) {
      sm.anc[lane] = anc;
      sm.beta[lane] = beta;
      sm.g[lane] = total;
      sm.begun[lane] = __builtin_amdgcn_exp2f((float)total);
    }
    if (lane == 0) sm.bad_u = 0;
  }
  __syncthreads();
  float y[3][RW][2], none = 0.f;  // NaN from the first number that is not finite
#pragma unroll
  for (int k = 0; k < RW; ++k) {
    uint32_t x[3][3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint32_t* row = &sm.raw[0][0][lane] + 64 * __builtin_amdgcn_readlane(tap[j], w + NW * k);
#pragma unroll
      for (int which = 0; which < 3; ++which) x[which][j] = row[which * (3 + TM) * 64];
    }
#pragma unroll
    for (int which = 0; which < 3; ++which) {
      const float4 w0 = wt[which][0], w1 = wt[which][1];
      const float y0 = bias[which].x + w0.x * npn::bf16lo(x[which][2]) + w0.y * npn::bf16lo(x[which][1]) +
                       w0.z * npn::bf16lo(x[which][0]) + w0.w * npn::bf16lo(raw[which][k]);
      const float y1 = bias[which].y + w1.x * npn::bf16hi(x[which][2]) + w1.y * npn::bf16hi(x[which][1]) +
                       w1.z * npn::bf16hi(x[which][0]) + w1.w * npn::bf16hi(raw[which][k]);
      y[which][k][0] = silu(y0);
      y[which][k][1] = silu(y1);
      none = fmaf(y[which][k][0], 0.f, none);
      none = fmaf(y[which][k][1], 0.f, none);
    }
  }
  const bool some = __builtin_amdgcn_ballot_w64(none != none) != 0;
  if (some) {
#pragma unroll
    for (int k = 0; k < RW; ++k)
#pragma unroll
      for (int which = 0; which < 3; ++which) {
        const bool bad = w + NW * k < T &&
                         __builtin_amdgcn_ballot_w64(!finite(y[which][k][0]) || !finite(y[which][k][1])) != 0;
        (which == 0 ? bad_q : bad_kv) |= bad ? 1ull << (w + NW * k) : 0ull;
      }
  }
#pragma unroll
  for (int k = 0; k < RW; ++k)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float &y0 = y[which][k][0], &y1 = y[which][k][1];
      const float n = __builtin_amdgcn_rsqf(wave_sum(y0 * y0 + y1 * y1) + kEps) *
                      (which == 0 ? 0.08838834764831845f * kUnit : kUnit);  // q: / sqrt(128)
      y0 *= n;
      y1 *= n;
    }
  if (h == kh * (a.Hv / a.Hk)) {
#pragma unroll
    for (int k = 0; k < RW; ++k)
      if (w + NW * k < T)
        *reinterpret_cast<float2*>(a.rec_k + (((size_t)b * T + w + NW * k) * a.Hk + kh) * D + 2 * lane) =
            make_float2(y[1][k][0] * (1.0f / kUnit), y[1][k][1] * (1.0f / kUnit));
  }
  if (lane == 0) {
    sm.bad_kv[w] = bad_kv;
    sm.bad_q[w] = bad_q;
  }
  if (some) {  // zeros in the sums
#pragma unroll
    for (int k = 0; k < RW; ++k)
#pragma unroll
      for (int which = 0; which < 3; ++which)
        if ((which == 0 ? bad_q : bad_kv) >> (w + NW * k) & 1) y[which][k][0] = y[which][k][1] = 0.f;
  }
  if constexpr (APART) load_state();
  __syncthreads();  // the inputs have been read
  auto write_rows = [&](int which) {
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      const int t = w + NW * k;
      const float y0 = t < T ? y[which][k][0] : 0.f, y1 = t < T ? y[which][k][1] : 0.f;
      if (which < 2) {
        const f16x2 hi = {(_Float16)y0, (_Float16)y1};
        const f16x2 lo = {(_Float16)(y0 - (float)hi[0]), (_Float16)(y1 - (float)hi[1])};
        const int row = which == 0 && !APART ? TM + t : t;
        *reinterpret_cast<f16x2*>(&sm.x[0][row][2 * lane]) = hi;
        *reinterpret_cast<f16x2*>(&sm.x[1][row][2 * lane]) = lo;
      } else {
        *reinterpret_cast<float2*>(APART ? &sm.v_apart[APART ? t : 0][2 * lane] : &sm.v[APART ? 0 : t][2 * lane]) =
            make_float2(y0, y1);
      }
    }
  };
  write_rows(1);
  if constexpr (!APART) {
    write_rows(0);
    write_rows(2);
  }
  __syncthreads();

  // 2. the pairs' products, tile (a, s) with s <= a of k's rows and of q's, k's rows of tile s by `keys`
  auto rows_of = [&](int part, int tile, int step) {
    return *reinterpret_cast<const f16x8*>(&sm.x[part][16 * tile + i][32 * step + 8 * G]);
  };
  auto pair_tile = [&](int q, int ta, int ts, auto&& keys) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const int rows = q && !APART ? NT + ta : ta;
      const f16x8 xh = rows_of(0, rows, step), xl = rows_of(1, rows, step);
      const f16x8 kh8 = keys(0, step), kl8 = keys(1, step);
      p = mfma_f16(xl, kh8, p);
      p = mfma_f16(xh, kl8, p);
      p = mfma_f16(xh, kh8, p);
    }
    const int s = 16 * ts + i;
    const double gs = sm.g[s];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * ta + 4 * G + r;
      const bool sees = (sm.anc[t] >> s & 1) && (q || s != t);
      const float f = __builtin_amdgcn_exp2f((float)(sm.g[t] - gs)) * (1.0f / (kUnit * kUnit));
      (q ? sm.mix : sm.low)[tile_at(ta, ts)][4 * G + r][i] = sees ? p[r] * f * (q ? 1.0f : -sm.beta[t]) : 0.f;
    }
  };
  int turn = 0;
#pragma unroll
  for (int ta = 0; ta < NT; ++ta)
#pragma unroll
    for (int ts = 0; ts <= ta; ++ts)
#pragma unroll
      for (int q = 0; q < (APART ? 1 : 2); ++q)
        if ((turn++ & (NW - 1)) == w) pair_tile(q, ta, ts, [&](int part, int step) { return rows_of(part, ts, step); });
  // and the state's
  float scale[CT], inv_scale[CT];
  f32x4 ks[NT][CT], qs[NT][CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float big = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(s0[s][e].x[c]));
    // to [2^11, 2^12); of a column that is not finite some product is not either
    const uint32_t e = min(max(__float_as_uint(max_over_groups(big)) >> 23, 12u), 254u);
    scale[c] = __uint_as_float((265u - e) << 23);
    inv_scale[c] = __uint_as_float((e - 11u) << 23) * (1.0f / kUnit);
#pragma unroll
    for (int n = 0; n < NT; ++n) ks[n][c] = qs[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto state_parts = [&](int s, f16x8 (&hi)[CT], f16x8 (&lo)[CT]) {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = s0[s][e].x[c] * scale[c];
        hi[c][e] = (_Float16)x;
        lo[c][e] = (_Float16)(x - (float)hi[c][e]);
      }
  };
  auto state_tile = [&](int rows, int s, const f16x8 (&hi)[CT], const f16x8 (&lo)[CT], f32x4 (&p)[CT]) {
    const f16x8 xh = rows_of(0, rows, s), xl = rows_of(1, rows, s);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      p[c] = mfma_f16(xl, hi[c], p[c]);
      p[c] = mfma_f16(xh, lo[c], p[c]);
      p[c] = mfma_f16(xh, hi[c], p[c]);
    }
  };
  if constexpr (APART) {
    f16x8 hi[4][CT], lo[4][CT], key[2][4];  // wave w has tile w of k's rows when q's come
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      state_parts(s, hi[s], lo[s]);
#pragma unroll
      for (int n = 0; n < NT; ++n) state_tile(n, s, hi[s], lo[s], ks[n]);
    }
    const int mine = min(w, NT - 1);
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int s = 0; s < 4; ++s) key[part][s] = rows_of(part, mine, s);
    __syncthreads();
    write_rows(0);
    __syncthreads();
#pragma unroll
    for (int ta = 0; ta < NT; ++ta)
      if (ta >= w) pair_tile(1, ta, w, [&](int part, int step) { return key[part][step]; });
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) state_tile(n, s, hi[s], lo[s], qs[n]);
    __syncthreads();
    write_rows(2);
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      f16x8 hi[CT], lo[CT];
      state_parts(s, hi, lo);
#pragma unroll
      for (int n = 0; n < NT; ++n) state_tile(n, s, hi, lo, ks[n]);
#pragma unroll
      for (int n = 0; n < NT; ++n) state_tile(NT + n, s, hi, lo, qs[n]);
    }
  }
  // z is on its way by the time it is needed.
  const size_t node0 = (size_t)b * T * a.Hv * D;
  const unsigned node_at = h * D + col, node_step = a.Hv * D;  // node t: t steps behind
  uint32_t z[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint16_t* p = a.z + node0 + (node_at + min(16 * n + 4 * G + r, T - 1) * node_step);
      z[n][r] = CT == 2 ? *reinterpret_cast<const uint32_t*>(p) : *p;
    }
  const Floats<CT> nw = *reinterpret_cast<const Floats<CT>*>(a.norm_weight + col);
  auto right_sides = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const f32x4 begun = *reinterpret_cast<const f32x4*>(&sm.begun[16 * n + 4 * G]);
      const f32x4 beta = *reinterpret_cast<const f32x4*>(&sm.beta[16 * n + 4 * G]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * n + 4 * G + r;
        const Floats<CT> v =
            *reinterpret_cast<const Floats<CT>*>(APART ? &sm.v_apart[APART ? t : 0][col] : &sm.v[APART ? 0 : t][col]);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          ks[n][c][r] = beta[r] * (v.x[c] - begun[r] * (ks[n][c][r] * inv_scale[c]));
          qs[n][c][r] *= begun[r] * inv_scale[c];
        }
      }
    }
  };
  if constexpr (!APART) {
    right_sides();
    __syncthreads();
  }

  // 3. column i of the inverse of block w
  if (w < NT) {
    const float (*low)[20] = sm.low[tile_at(w, w)];
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float y = r == i ? 1.0f : 0.f;
#pragma unroll
      for (int q = 0; q < r; ++q) y = fmaf(low[r][q], x[q], y);
      x[r] = y;
      if (G == 0) sm.inv[w][r][i] = y;
    }
  }
  __syncthreads();
  if constexpr (APART) right_sides();

  // 4.
  // Rows' entries that are not finite count as 0 from here on, and their nodes as bad.
  auto clear = [&](f32x4 (&x)[CT], int tile) {
    float none = 0.f;  // NaN from the first that is not finite
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) none = fmaf(x[c][r], 0.f, none);
    if (__builtin_amdgcn_ballot_w64(none != none) == 0) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      bool bad = false;
#pragma unroll
      for (int c = 0; c < CT; ++c) bad |= !finite(x[c][r]);
      if (bad) {
#pragma unroll
        for (int c = 0; c < CT; ++c) x[c][r] = 0.f;
        atomicOr(&sm.bad_u, 1ull << (16 * tile + 4 * G + r));
      }
    }
  };
  f32x4 u[NT][CT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int s = 0; s < n; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(&sm.low[tile_at(n, s)][i][4 * G]);
#pragma unroll
      for (int c = 0; c < CT; ++c) ks[n][c] = mfma_f32(f, u[s][c], ks[n][c]);
    }
    clear(ks[n], n);
    const float4 f = *reinterpret_cast<const float4*>(&sm.inv[n][i][4 * G]);
#pragma unroll
    for (int c = 0; c < CT; ++c) u[n][c] = mfma_f32(f, ks[n][c], f32x4{0.f, 0.f, 0.f, 0.f});
    clear(u[n], n);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int s = 0; s <= n; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(&sm.mix[tile_at(n, s)][i][4 * G]);
#pragma unroll
      for (int c = 0; c < CT; ++c) qs[n][c] = mfma_f32(f, u[s][c], qs[n][c]);
    }
    f32x4 ss = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int c = 0; c < CT; ++c) ss[r] += qs[n][c][r] * qs[n][c][r];
      ss[r] = row_sum(ss[r]);
    }
    if (i == 0) *reinterpret_cast<f32x4*>(&sm.ss[w][16 * n + 4 * G]) = ss;
  }
  __syncthreads();

  // 5. A row's factor: NaN where the node or one before it is bad; of its record 0 or NaN.
  if (tid < TM) {
    uint64_t kv = sm.bad_u, bq = 0;
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      kv |= sm.bad_kv[k];
      bq |= sm.bad_q[k];
      ss += sm.ss[k][tid];
    }
    const bool nan = (sm.anc[tid] & kv) != 0;
    sm.begun[tid] = nan || (bq >> tid & 1) ? NAN : __builtin_amdgcn_rsqf(ss * (1.0f / D) + kEps);
    sm.beta[tid] = nan ? NAN : 0.f;
  }
  float gate[NT][4][CT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < CT; ++c)
        gate[n][r][c] = nw.x[c] * silu(c == 0 ? npn::bf16lo(z[n][r]) : npn::bf16hi(z[n][r]));
  __syncthreads();

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const f32x4 f = *reinterpret_cast<const f32x4*>(&sm.begun[16 * n + 4 * G]);
    const f32x4 none = *reinterpret_cast<const f32x4*>(&sm.beta[16 * n + 4 * G]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * n + 4 * G + r;
      if (t >= T) continue;
      const unsigned at = node_at + t * node_step;
      Floats<CT> rec;
      __bf16 o[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        o[c] = (__bf16)(qs[n][c][r] * f[r] * gate[n][r][c]);
        rec.x[c] = u[n][c][r] + none[r];
      }
      if constexpr (CT == 2) {
        const bf16x2 both = {o[0], o[1]};
        *reinterpret_cast<bf16x2*>(a.out + node0 + at) = both;
      } else {
        *reinterpret_cast<__bf16*>(a.out + node0 + at) = o[0];
      }
      *reinterpret_cast<Floats<CT>*>(a.rec_u + node0 + at) = rec;
    }
  }
}

// ---- commit -----------------------------------------------------------------------------------------
constexpr int kCommitLayers = 64;

struct CommitArgs {
  float* state[kCommitLayers];          // [B][Hv][128][128]
  uint16_t* conv[kCommitLayers];        // [B][QKV][3]
  const uint16_t* mixed[kCommitLayers]; // [B][T][QKV]
  const float* rec[kCommitLayers];      // k [B][T][Hk][128], u [B][T][Hv][128], decay [B][T][Hv]
  const int32_t* path;                  // [B][T]
  int layers, B, T, Hk, Hv;
  unsigned heads;                       // layers * B * Hv, then the windows' workgroups
};

// One workgroup a (layer, b, h), its 128 x 128 floats in registers: thread (r, c4) has rows r + 8 i of columns
// 4 c4 .. + 3. The workgroups behind move the conv windows, a thread a channel. Bound by the states' bytes, read and
// written once: 48 layers of 48 heads 65 us for 316 MB, 3 layers of 32 requests 131 us for 632 MB.
__global__ __launch_bounds__(256) void dn_tree_commit_kernel(CommitArgs a) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int QKV = (2 * a.Hk + a.Hv) * D;
  if (blockIdx.x >= a.heads) {
    const int per = (QKV + 255) / 256;  // workgroups a (layer, b)
    const int x = blockIdx.x - a.heads, lb = x / per, c = (x - lb * per) * 256 + tid;
    const int l = lb / a.B, b = lb - l * a.B;
    const int node = lane < a.T ? a.path[(size_t)b * a.T + lane] : -1;
    const int n = npn::path_length(node, a.T, lane);
    int last[3];
    for (int j = 0; j < 3; ++j) last[j] = __shfl(node, max(n - 3 + j, 0), 64);
    if (c >= QKV || n == 0) return;
    uint16_t* cs = a.conv[l] + ((size_t)b * QKV + c) * 3;
    uint16_t v[3];
    for (int j = 0; j < 3; ++j)
      v[j] = n + j < 3 ? cs[n + j] : a.mixed[l][((size_t)b * a.T + last[j]) * QKV + c];
    for (int j = 0; j < 3; ++j) cs[j] = v[j];
    return;
  }
  const int l = blockIdx.x / (a.B * a.Hv), bh = blockIdx.x - l * a.B * a.Hv;
  const int b = bh / a.Hv, h = bh - b * a.Hv, kh = h / (a.Hv / a.Hk);
  const int T = a.T;
  const int node = lane < T ? a.path[(size_t)b * T + lane] : -1;
  const int n = npn::path_length(node, T, lane);
  if (n == 0) return;
  const float* rec_k = a.rec[l];
  const float* rec_u = rec_k + (size_t)a.B * T * a.Hk * D;
  const float* rec_decay = rec_u + (size_t)a.B * T * a.Hv * D;
  float4* S = reinterpret_cast<float4*>(a.state[l] + ((size_t)b * a.Hv + h) * D * D) + tid;
  float4 s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = S[256 * i];
  __shared__ float s_k[D];
  __shared__ float4 s_u[D / 4];
  for (int d = 0; d < n; ++d) {
    const size_t at = (size_t)b * T + __builtin_amdgcn_readlane(node, d);
    const float decay = rec_decay[at * a.Hv + h];
    __syncthreads();
    if (tid < D) s_k[tid] = rec_k[(at * a.Hk + kh) * D + tid];
    else reinterpret_cast<float*>(s_u)[tid - D] = rec_u[(at * a.Hv + h) * D + tid - D];
    __syncthreads();
    const float4 u = s_u[tid & 31];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float k = s_k[8 * i + (tid >> 5)];
      s[i].x = s[i].x * decay + k * u.x;
      s[i].y = s[i].y * decay + k * u.y;
      s[i].z = s[i].z * decay + k * u.z;
      s[i].w = s[i].w * decay + k * u.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) S[256 * i] = s[i];
}

bool heads_ok(int B, int T, int k_heads, int v_heads) {
  return B >= 1 && B <= 65536 && T >= 1 && T <= npn::kMaxNodes && k_heads >= 1 && v_heads >= 1 &&
         v_heads % k_heads == 0 && v_heads <= 4096 && (int64_t)B * v_heads <= 1 << 22;
}

}  // namespace

extern "C" int npn_deltanet_verify_tree(const float* state, const int32_t* parent, const uint16_t* mixed_qkv,
                                        const uint16_t* conv_state, const float* conv_weight,
                                        const float* conv_bias, const float* a_out, const float* b_out,
                                        const uint16_t* z, const float* A_log, const float* dt_bias,
                                        const float* norm_weight, uint16_t* out, float* records, int B, int T,
                                        int k_heads, int v_heads, void* stream) {
  NPN_REQUIRE(state && parent && mixed_qkv && conv_state && conv_weight && conv_bias && a_out && b_out && z &&
                  A_log && dt_bias && norm_weight && out && records,
              NPN_ERR_NULL);
  NPN_REQUIRE(heads_ok(B, T, k_heads, v_heads), NPN_ERR_SHAPE);
  NPN_REQUIRE(NPN_ALIGNED16(state) && NPN_ALIGNED16(mixed_qkv) && NPN_ALIGNED16(conv_state) &&
                  NPN_ALIGNED16(conv_weight) && NPN_ALIGNED16(conv_bias) && NPN_ALIGNED16(norm_weight) &&
                  NPN_ALIGNED16(z) && NPN_ALIGNED16(out) && NPN_ALIGNED16(records),
              NPN_ERR_ALIGN);
  float* rec_u = records + (size_t)B * T * k_heads * D;
  float* rec_decay = rec_u + (size_t)B * T * v_heads * D;
  const TreeArgs a{state, parent, mixed_qkv, conv_state, conv_weight, conv_bias, a_out, b_out, z, A_log,
                   dt_bias, norm_weight, out, records, rec_u, rec_decay, B, T, k_heads, v_heads};
  const dim3 grid(B * v_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // Up to a head for each of the 256 CUs, eight waves: the steps are shorter. Above, two workgroups of four share a CU and
  // each fills the other's waits. us with four waves (APART above 32 nodes) and with eight, at 48, 240, 288 and 768 heads:
  //   16 nodes 10.1, 11.8, 15.5, 20.7 and 9.2, 11.3, 15.2, 22.6; 48 nodes 20, 23.0, 28.4, 46 and 17, 20.6, 35.4, 57;
  //   64 nodes 25.8, 29.0, 36.9, 61 and 21.6, 25.4, 43.9, 72.
  // 32 nodes have eight waves at all of them: 15, 21 at 288, 34 at 768 heads with four APART and 13, 21.4, 32 with eight.
  const bool many = B * v_heads > 256;
  auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, s, a); };
  if (T <= 16) many ? launch(dn_tree_verify_kernel<1, 4, false>, 4) : launch(dn_tree_verify_kernel<1, 8, false>, 8);
  else if (T <= 32) launch(dn_tree_verify_kernel<2, 8, false>, 8);
  else if (T <= 48) many ? launch(dn_tree_verify_kernel<3, 4, true>, 4) : launch(dn_tree_verify_kernel<3, 8, false>, 8);
  else many ? launch(dn_tree_verify_kernel<4, 4, true>, 4) : launch(dn_tree_verify_kernel<4, 8, false>, 8);
  return npn_launch_status();
}

extern "C" int npn_deltanet_commit_tree(float* const* state, uint16_t* const* conv_state,
                                        const uint16_t* const* mixed_qkv, const float* const* records,
                                        int layers, const int32_t* path, int B, int T, int k_heads,
                                        int v_heads, void* stream) {
  NPN_REQUIRE(path && (layers == 0 || (state && conv_state && mixed_qkv && records)), NPN_ERR_NULL);
  NPN_REQUIRE(layers >= 0 && heads_ok(B, T, k_heads, v_heads), NPN_ERR_SHAPE);
  const size_t states = sizeof(float) * B * v_heads * D * D;
  const size_t windows = sizeof(uint16_t) * 3 * B * (2 * k_heads + v_heads) * D;
  for (int l = 0; l < layers; ++l) {
    NPN_REQUIRE(state[l] && conv_state[l] && mixed_qkv[l] && records[l], NPN_ERR_NULL);
    NPN_REQUIRE(NPN_ALIGNED16(state[l]), NPN_ERR_ALIGN);
    for (int k = 0; k < l; ++k)
      NPN_REQUIRE(npn_apart(state[k], states, state[l], states) && npn_apart(conv_state[k], windows, conv_state[l], windows),
                  NPN_ERR_VALUE);
  }
  const int per = ((2 * k_heads + v_heads) * D + 255) / 256;
  const int64_t blocks = (int64_t)B * (v_heads + per);  // a layer's workgroups
  const int most = (int)max((int64_t)1, min((int64_t)kCommitLayers, ((int64_t)1 << 23) / blocks));  // a launch
  for (int l0 = 0; l0 < layers; l0 += most) {
    CommitArgs a{};
    a.layers = layers - l0 < most ? layers - l0 : most;
    for (int l = 0; l < a.layers; ++l) {
      a.state[l] = state[l0 + l];
      a.conv[l] = conv_state[l0 + l];
      a.mixed[l] = mixed_qkv[l0 + l];
      a.rec[l] = records[l0 + l];
    }
    a.path = path;
    a.B = B;
    a.T = T;
    a.Hk = k_heads;
    a.Hv = v_heads;
    a.heads = (unsigned)(a.layers * B * v_heads);
    hipLaunchKernelGGL(dn_tree_commit_kernel, dim3((unsigned)(a.layers * blocks)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
    const int st = npn_launch_status();
    if (st != NPN_OK) return st;
  }
  return NPN_OK;
}
