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

// One workgroup a (b, h), thread (c, p) for column c of the state: p = 0 the rows of k, p = 1 those of q.
template <int TMAX>
__global__ __launch_bounds__(256) void dn_tree_verify_kernel(TreeArgs a) {
  __shared__ float s_q[TMAX][D], s_k[TMAX][D], s_u[TMAX][D];
  __shared__ float s_kk[TMAX][TMAX + 1], s_qk[TMAX][TMAX + 1];
  __shared__ double s_g[TMAX];
  __shared__ float s_begun[TMAX], s_beta[TMAX], s_sum[TMAX][2];
  __shared__ uint64_t s_anc[TMAX];
  __shared__ int s_tap[TMAX][3];
  const int T = a.T, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = blockIdx.x / a.Hv, h = blockIdx.x - b * a.Hv, kh = h / (a.Hv / a.Hk);
  const int QKV = (2 * a.Hk + a.Hv) * D;

  const int parent = npn::tree_parent(a.parent + (size_t)b * T, T, lane);
  const uint64_t anc = npn::tree_ancestors(parent, T, lane);
  if (w == 0) {
    // The window's inputs one to three back: a node, or -1 .. -3 for the last to the first of conv_state.
    int at = lane;
    for (int j = 0; j < 3; ++j) {
      const int up = __shfl(parent, max(at, 0), 64);
      at = at < 0 ? at - 1 : up;
      if (lane < T) s_tap[lane][j] = at;
    }
    double g = 0.0;
    if (lane < T) {
      const size_t gi = ((size_t)b * T + lane) * a.Hv + h;
      const float gf = -__expf(a.A_log[h]) * npn::softplus(a.a_out[gi] + a.dt_bias[h]);
      a.rec_decay[gi] = __expf(gf);
      s_beta[lane] = npn::sigmoid(a.b_out[gi]);
      g = gf < -256.0f ? -256.0 : (double)gf;
      s_anc[lane] = anc;
    }
    double total = 0.0;
    for (int t = 0; t < T; ++t) {
      const double x = __longlong_as_double(npn::tree_bits(__double_as_longlong(g), t));
      total += (anc >> t) & 1 ? x : 0.0;
    }
    if (lane < T) {
      s_g[lane] = total;
      s_begun[lane] = __expf((float)total);
    }
  }
  __syncthreads();

  const uint16_t* xb = a.mixed_qkv + (size_t)b * T * QKV;
  const uint16_t* csb = a.conv_state + (size_t)b * QKV * 3;
  for (int idx = tid; idx < T * 3 * D; idx += 256) {
    const int t = idx / (3 * D), ch = idx - t * 3 * D, which = ch / D, i = ch - which * D;
    const int c = which == 0 ? kh * D + i : which == 1 ? (a.Hk + kh) * D + i : (2 * a.Hk + h) * D + i;
    float y = a.conv_bias[c];
    for (int j = 2; j >= 0; --j) {
      const int at = s_tap[t][j];
      const uint16_t x = at >= 0 ? xb[(size_t)at * QKV + c] : csb[(size_t)c * 3 + 3 + at];
      y += a.conv_weight[c * 4 + 2 - j] * npn::bf16_to_f32(x);
    }
    y += a.conv_weight[c * 4 + 3] * npn::bf16_to_f32(xb[(size_t)t * QKV + c]);
    (which == 0 ? s_q : which == 1 ? s_k : s_u)[t][i] = npn::silu(y);
  }
  __syncthreads();
  for (int r = w; r < 2 * T; r += 4) {
    float* x = r < T ? s_q[r] : s_k[r - T];
    const float x0 = x[lane], x1 = x[lane + 64];
    const float n = rsqrtf(npn::wave_sum(x0 * x0 + x1 * x1) + kEps) * (r < T ? 0.08838834764831845f : 1.0f);
    x[lane] = x0 * n;
    x[lane + 64] = x1 * n;
    if (r >= T && h == kh * (a.Hv / a.Hk)) {
      float* k = a.rec_k + (((size_t)b * T + r - T) * a.Hk + kh) * D;
      k[lane] = x0 * n;
      k[lane + 64] = x1 * n;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < 2 * T * T; idx += 256) {
    const int which = idx / (T * T), t = (idx - which * T * T) / T, s = idx % T;
    if (!((s_anc[t] >> s) & 1)) continue;
    const float* x = which ? s_q[t] : s_k[t];
    float dot = 0.f;
    for (int i = 0; i < D; ++i) dot += x[i] * s_k[s][i];
    (which ? s_qk : s_kk)[t][s] = dot * __expf((float)(s_g[t] - s_g[s]));
  }
  __syncthreads();

  const int c = tid & (D - 1), p = tid >> 7;
  const float* S0 = a.state + ((size_t)b * a.Hv + h) * D * D + c;
  const float (*x)[D] = p ? s_q : s_k;
  float acc[TMAX];
#pragma unroll
  for (int t = 0; t < TMAX; ++t) acc[t] = 0.f;
  for (int i = 0; i < D; ++i) {
    const float s = S0[(size_t)i * D];
#pragma unroll
    for (int t = 0; t < TMAX; ++t)
      if (t < T) acc[t] += x[t][i] * s;
  }
  if (p == 0) {
#pragma unroll
    for (int t = 0; t < TMAX; ++t)
      if (t < T) {
        float r = s_u[t][c] - s_begun[t] * acc[t];
        for (uint64_t m = s_anc[t] & ~(1ull << t); m; m &= m - 1) {
          const int s = __builtin_ctzll(m);
          r -= s_kk[t][s] * s_u[s][c];
        }
        s_u[t][c] = r * s_beta[t];
        a.rec_u[(((size_t)b * T + t) * a.Hv + h) * D + c] = r * s_beta[t];
      }
  }
  __syncthreads();
  if (p == 1) {
#pragma unroll
    for (int t = 0; t < TMAX; ++t)
      if (t < T) {
        float o = s_begun[t] * acc[t];
        for (uint64_t m = s_anc[t]; m; m &= m - 1) {
          const int s = __builtin_ctzll(m);
          o += s_qk[t][s] * s_u[s][c];
        }
        acc[t] = o;
        const float sum = npn::wave_sum(o * o);
        if (lane == 0) s_sum[t][w & 1] = sum;
      }
  }
  __syncthreads();
  if (p == 1) {
    const float nw = a.norm_weight[c];
#pragma unroll
    for (int t = 0; t < TMAX; ++t)
      if (t < T) {
        const size_t oi = (((size_t)b * T + t) * a.Hv + h) * D + c;
        const float r = rsqrtf((s_sum[t][0] + s_sum[t][1]) * (1.0f / D) + kEps);
        a.out[oi] = npn::f32_to_bf16(acc[t] * r * nw * npn::silu(npn::bf16_to_f32(a.z[oi])));
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
// 4 c4 .. + 3. The workgroups behind move the conv windows, a thread a channel.
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
  NPN_REQUIRE(NPN_ALIGNED16(state) && NPN_ALIGNED16(mixed_qkv) && NPN_ALIGNED16(conv_weight) &&
                  NPN_ALIGNED16(z) && NPN_ALIGNED16(out) && NPN_ALIGNED16(records),
              NPN_ERR_ALIGN);
  float* rec_u = records + (size_t)B * T * k_heads * D;
  float* rec_decay = rec_u + (size_t)B * T * v_heads * D;
  const TreeArgs a{state, parent, mixed_qkv, conv_state, conv_weight, conv_bias, a_out, b_out, z, A_log,
                   dt_bias, norm_weight, out, records, rec_u, rec_decay, B, T, k_heads, v_heads};
  const dim3 grid(B * v_heads), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (T <= 16) hipLaunchKernelGGL(dn_tree_verify_kernel<16>, grid, block, 0, s, a);
  else if (T <= 32) hipLaunchKernelGGL(dn_tree_verify_kernel<32>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(dn_tree_verify_kernel<64>, grid, block, 0, s, a);
  return npn_launch_status();
}

extern "C" int npn_deltanet_commit_tree(float* const* state, uint16_t* const* conv_state,
                                        const uint16_t* const* mixed_qkv, const float* const* records,
                                        int layers, const int32_t* path, int B, int T, int k_heads,
                                        int v_heads, void* stream) {
  NPN_REQUIRE(path && (layers == 0 || (state && conv_state && mixed_qkv && records)), NPN_ERR_NULL);
  NPN_REQUIRE(layers >= 0 && heads_ok(B, T, k_heads, v_heads), NPN_ERR_SHAPE);
  for (int l = 0; l < layers; ++l) {
    NPN_REQUIRE(state[l] && conv_state[l] && mixed_qkv[l] && records[l], NPN_ERR_NULL);
    NPN_REQUIRE(NPN_ALIGNED16(state[l]) && NPN_ALIGNED16(records[l]), NPN_ERR_ALIGN);
    for (int k = 0; k < l; ++k) NPN_REQUIRE(state[k] != state[l] && conv_state[k] != conv_state[l], NPN_ERR_VALUE);
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
