// Sliding-window attention for a few queries behind many keys (one new token a row), forward only, for sm_100a (rule: window.cuh).
// With so few rows the work is reading K and V once, and what counts is how much of that is in flight: the tiles of the
// tensor-memory kernel would have 128 rows for 8. A cluster of CTAs shares the keys of one (row, key/value head); a warp takes 16
// keys at a time into registers, 16-byte loads throughout, for up to 8 rows (queries x query heads of the group) at once, with an
// online softmax of its own. The products run as warp-wide m16n8k16 MMAs, whose operands come straight from those loads: the
// head dimension may be permuted in S = Q K^T as long as Q and K agree, and the rows of O^T = V^T P^T may be any 16 dimensions,
// so no value changes its lane (on the FMA pipe the same loop took 75 us for the case below, 1.4 times the tile kernel). The
// parts are joined in shared memory, then across the cluster, in one launch and in a fixed order.
// Bound by HBM: 8 rows x 2052 visible keys x 8 key/value heads of 128 are 67 MB, 10 us at the copy rate; it takes 25 us (31 us
// with a cold L2): a single wave of clusters, whose first loads and last join nothing hides.
#include "host.h"
#include "ptx.cuh"
#include "window.cuh"

namespace mb {

constexpr int kWtThreads = 128, kWtWarps = kWtThreads / 32;
constexpr int kWtRows = 8;          // rows a CTA handles
constexpr int kWtKeys = 16;         // keys a warp takes at a time
constexpr int kWtMaxCluster = 8;

struct WindowTokenArgs {
  const __nv_bfloat16 *q, *k, *v;
  long long q_t, q_b, k_t, k_b, v_t, v_b;   // strides in elements, heads contiguous inside a token
  __nv_bfloat16* out;       // [B, Sq, Hq, D]
  float* lse;               // [B, Hq, Sq] or null
  WindowRule rule;
  int B, Sq, Sk, Hq, Hkv, row_groups;
  float scale_log2;
};

__device__ __forceinline__ float wt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float wt_ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// c += a b, a [16 x 16] row-major, b [16 x 8] column-major, bf16, in the registers of a warp.
__device__ __forceinline__ void wt_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t wt_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Grid (cluster, key/value heads x row groups, B). In a warp: g = lane / 4, t = lane % 4.
template <int D>
__global__ void __launch_bounds__(kWtThreads, 4) window_token_kernel(const WindowTokenArgs p) {
  constexpr int QC = D / 32, VC = D / 64;           // 16-byte chunks of a K row, and of a V row, that a lane loads
  __shared__ float s_o[kWtWarps][kWtRows][D], s_m[kWtWarps][kWtRows], s_l[kWtWarps][kWtRows], s_x[kWtWarps][kWtRows];
  __shared__ float c_o[kWtRows][D], c_m[kWtRows], c_l[kWtRows], c_x[kWtRows];   // of this CTA, read by the others of the cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ctas = gridDim.x, rank = blockIdx.x;    // the cluster spans the grid's first dimension
  const int kv_head = blockIdx.y / p.row_groups, first_row = blockIdx.y % p.row_groups * kWtRows, batch = blockIdx.z;
  const int group = p.Hq / p.Hkv, rows = p.Sq * group;

  // row g: its keys, and its query in the order of the K chunks
  const int row = first_row + g, qi = row / group;
  const bool valid = row < rows;
  const WindowRow w = window_row(p.rule, batch, p.Sk, qi + p.Sk - p.Sq, valid);
  uint4 q[QC];
#pragma unroll
  for (int s = 0; s < QC; ++s) {
    q[s] = make_uint4(0u, 0u, 0u, 0u);
    if (valid) q[s] = __ldg(reinterpret_cast<const uint4*>(p.q + batch * p.q_b + qi * p.q_t + static_cast<long long>(kv_head * group + row % group) * D + (4 * s + t) * 8));
  }
  // keys in order: first tokens before the window of all rows, then that window
  const int lo = __reduce_min_sync(0xffffffffu, w.lo), hi = __reduce_max_sync(0xffffffffu, w.hi), far = __reduce_min_sync(0xffffffffu, w.sink_begin);
  const int n_far = hi < 0 ? 0 : max(0, min(far + p.rule.sinks, lo) - far), n_keys = hi < 0 ? 0 : n_far + hi - lo + 1;

  float m = -INFINITY, l = 0.f, x = 0.f;            // of row g: maximum, sum of the rounded weights, of the weights
  float o[4 * VC][4];                               // O^T: [0], [1] dimension 2j of chunk g for rows 2t, 2t + 1; [2], [3] dimension 2j + 1
#pragma unroll
  for (int j = 0; j < 4 * VC; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
  const __nv_bfloat16* kb = p.k + batch * p.k_b + static_cast<long long>(kv_head) * D;
  const __nv_bfloat16* vb = p.v + batch * p.v_b + static_cast<long long>(kv_head) * D;
  for (int at = (rank * kWtWarps + warp) * kWtKeys; at < n_keys; at += ctas * kWtWarps * kWtKeys) {
    auto key_of = [&](int i) {                      // the batch's key i, -1 past the end
      const int n = at + i;
      return n >= n_keys ? -1 : n < n_far ? far + n : lo + n - n_far;
    };
    uint4 kx[2][QC], vx[4][VC];
    int key[4];                                     // 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = key_of(g + 8 * h);
#pragma unroll
      for (int s = 0; s < QC; ++s) {
        kx[h][s] = make_uint4(0u, 0u, 0u, 0u);
        if (k >= 0) kx[h][s] = __ldg(reinterpret_cast<const uint4*>(kb + k * p.k_t + (4 * s + t) * 8));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      key[i] = key_of(2 * t + (i & 1) + (i >> 1) * 8);
#pragma unroll
      for (int s = 0; s < VC; ++s) {
        vx[i][s] = make_uint4(0u, 0u, 0u, 0u);
        if (key[i] >= 0) vx[i][s] = __ldg(reinterpret_cast<const uint4*>(vb + key[i] * p.v_t + (8 * s + g) * 8));
      }
    }
    float s4[4];                                    // scores of row g for those four keys
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < QC; ++s) {
        wt_mma(c, q[s].x, 0u, q[s].y, 0u, kx[h][s].x, kx[h][s].y);
        wt_mma(c, q[s].z, 0u, q[s].w, 0u, kx[h][s].z, kx[h][s].w);
      }
      s4[2 * h] = c[0], s4[2 * h + 1] = c[1];
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool seen = key[i] >= 0 && ((key[i] >= w.lo && key[i] <= w.hi) || (key[i] >= w.sink_begin && key[i] < w.sink_end));
      s4[i] = seen ? s4[i] * p.scale_log2 : -INFINITY;
      top = fmaxf(top, s4[i]);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float safe = top == -INFINITY ? 0.f : top, alpha = wt_exp2(m - safe);   // m -inf: 0
    m = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) s4[i] = wt_exp2(s4[i] - safe);
    // rounded to bf16 for the product (V's type; error 0.0018 relative to 64 bits, 0.0017 of it the output's own rounding), and
    // divided by the sum of what was rounded
    const uint32_t p0 = pack_bf16x2(s4[0], s4[1]), p1 = pack_bf16x2(s4[2], s4[3]);
    x = x * alpha + (s4[0] + s4[1]) + (s4[2] + s4[3]);
    l = l * alpha + (__uint_as_float(p0 << 16) + __uint_as_float(p0 & 0xffff0000u)) + (__uint_as_float(p1 << 16) + __uint_as_float(p1 & 0xffff0000u));
    const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);   // of rows 2t, 2t + 1
#pragma unroll
    for (int s = 0; s < VC; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float(&c)[4] = o[4 * s + j];
        c[0] *= a0, c[1] *= a1, c[2] *= a0, c[3] *= a1;
        const uint32_t v0 = wt_word(vx[0][s], j), v1 = wt_word(vx[1][s], j), v2 = wt_word(vx[2][s], j), v3 = wt_word(vx[3][s], j);
        wt_mma(c, __byte_perm(v0, v1, 0x5410), __byte_perm(v0, v1, 0x7632), __byte_perm(v2, v3, 0x5410), __byte_perm(v2, v3, 0x7632), p0, p1);
      }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d), x += __shfl_xor_sync(0xffffffffu, x, d);
#pragma unroll
  for (int s = 0; s < VC; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = (8 * s + g) * 8 + 2 * j;
      *reinterpret_cast<float2*>(&s_o[warp][2 * t][d]) = make_float2(o[4 * s + j][0], o[4 * s + j][2]);
      *reinterpret_cast<float2*>(&s_o[warp][2 * t + 1][d]) = make_float2(o[4 * s + j][1], o[4 * s + j][3]);
    }
  if (t == 0) s_m[warp][g] = m, s_l[warp][g] = l, s_x[warp][g] = x;
  __syncthreads();
  // the warps of the CTA
  for (int e = threadIdx.x; e < kWtRows * D; e += kWtThreads) {
    const int r = e / D, d = e % D;
    float top = -INFINITY, sum = 0.f, sum_x = 0.f, val = 0.f;
#pragma unroll
    for (int i = 0; i < kWtWarps; ++i) top = fmaxf(top, s_m[i][r]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < kWtWarps; ++i) {
      const float a = wt_exp2(s_m[i][r] - safe);
      sum += a * s_l[i][r], sum_x += a * s_x[i][r], val += a * s_o[i][r][d];
    }
    c_o[r][d] = val;
    if (d == 0) c_m[r] = top, c_l[r] = sum, c_x[r] = sum_x;
  }
  cluster_arrive();
  cluster_wait();
  // the CTAs of the cluster: every one finishes a share of the values
  for (int e = rank * kWtThreads + threadIdx.x; e < kWtRows * D; e += ctas * kWtThreads) {
    const int r = e / D, d = e % D, out_row = first_row + r, oq = out_row / group, head = kv_head * group + out_row % group;
    float cm[kWtMaxCluster], cl[kWtMaxCluster], cx[kWtMaxCluster], co[kWtMaxCluster];
#pragma unroll
    for (int i = 0; i < kWtMaxCluster; ++i) {
      cm[i] = -INFINITY, cl[i] = cx[i] = co[i] = 0.f;
      if (i < ctas) {
        cm[i] = wt_ld_cluster(mapa_u32(&c_m[r], i)), cl[i] = wt_ld_cluster(mapa_u32(&c_l[r], i));
        cx[i] = wt_ld_cluster(mapa_u32(&c_x[r], i)), co[i] = wt_ld_cluster(mapa_u32(&c_o[r][d], i));
      }
    }
    float top = -INFINITY, sum = 0.f, sum_x = 0.f, val = 0.f;
#pragma unroll
    for (int i = 0; i < kWtMaxCluster; ++i) top = fmaxf(top, cm[i]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < kWtMaxCluster; ++i) {
      const float a = wt_exp2(cm[i] - safe);
      sum += a * cl[i], sum_x += a * cx[i], val += a * co[i];
    }
    if (out_row < rows) {
      // told by the row's visibility, not by its sum: a query that is no number has to stay one
      const bool sees = window_row(p.rule, batch, p.Sk, oq + p.Sk - p.Sq, true).hi >= 0;
      p.out[((static_cast<long long>(batch) * p.Sq + oq) * p.Hq + head) * D + d] = __float2bfloat16(sees ? val / sum : 0.f);
      if (d == 0 && p.lse)
        p.lse[(static_cast<long long>(batch) * p.Hq + head) * p.Sq + oq] = sees ? (top + log2f(sum_x)) * 0.6931471805599453f : -INFINITY;
    }
  }
  cluster_arrive();                                 // nobody leaves while its shared memory is read
  cluster_wait();
}

template <int D>
static int launch_window_token(const WindowTokenArgs& a, int ctas, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, a.Hkv * a.row_groups, a.B);
  cfg.blockDim = dim3(kWtThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  MB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, window_token_kernel<D>, a));
  count_launch();
  return 0;
}

}  // namespace mb

// As mb_window_attn_fwd without what the backward needs; for few queries: B, key/value heads x row groups up to 65535.
MB_API int mb_window_attn_token(const void* q, long long q_tstride, long long q_bstride, const void* k, long long k_tstride,
                                long long k_bstride, const void* v, long long v_tstride, long long v_bstride, void* out, float* lse,
                                const int* starts, int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, float scale,
                                cudaStream_t stream) {
  using namespace mb;
  const long long strides[] = {q_tstride, q_bstride, k_tstride, k_bstride, v_tstride, v_bstride};
  const void* pointers[] = {q, k, v, out};
  if (const char* what = window_attn_problem(B, Sq, Sk, Hq, Hkv, D, window, sinks, strides, 6, pointers, 4)) {
    set_last_error(what);
    return -1;
  }
  WindowTokenArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q), a.k = static_cast<const __nv_bfloat16*>(k), a.v = static_cast<const __nv_bfloat16*>(v);
  a.q_t = q_tstride, a.q_b = q_bstride, a.k_t = k_tstride, a.k_b = k_bstride, a.v_t = v_tstride, a.v_b = v_bstride;
  a.out = static_cast<__nv_bfloat16*>(out), a.lse = lse;
  a.rule = {starts, nullptr, window < Sk ? window : Sk, sinks < Sk ? sinks : Sk};
  a.B = B, a.Sq = Sq, a.Sk = Sk, a.Hq = Hq, a.Hkv = Hkv;
  a.scale_log2 = scale * 1.4426950408889634f;
  const long long rows = static_cast<long long>(Sq) * (Hq / Hkv);
  const long long groups = (rows + kWtRows - 1) / kWtRows;
  if (groups * Hkv > 65535) {
    set_last_error("mb_window_attn_token: too many query rows for this path");
    return -1;
  }
  a.row_groups = static_cast<int>(groups);
  // CTAs of a cluster: so many that each warp has a batch of keys or two
  const long long keys = static_cast<long long>(a.rule.window) + a.rule.sinks + Sq;
  int ctas = 1;
  while (ctas < kWtMaxCluster && static_cast<long long>(ctas) * kWtWarps * kWtKeys < keys) ctas *= 2;
  return D == 128 ? launch_window_token<128>(a, ctas, stream) : launch_window_token<64>(a, ctas, stream);
}
