// The seam between two blocks of a decoder in one pass, forward and backward (bf16, fp16, fp32, math in fp32):
//   u = w1 * x * r1,  r1 = rsqrt(mean(x^2) + eps)      (u = x without w1)         norm after the block
//   h = residual + scale * gate * u                     (gate: none, [H], or [rows, H])
//   y = w2 * h * r2,  r2 = rsqrt(mean(h^2) + eps)       (not without w2)           norm before the next block
// The forward keeps r1 and r2, the backward needs x, h and the two of them:
//   dn2 = dy * w2, hn = h * r2, c2 = mean(dn2 * hn);  dt = dh + r2 * (dn2 - hn * c2)      = dresidual
//   dg = scale * dt * u;  dn1 = scale * gate * dt * w1, xn = x * r1, c1 = mean(dn1 * xn);  dx = r1 * (dn1 - xn * c1)
// c1 is linear in dt: with e = scale * gate * w1 * xn it is mean(e * (dh + r2 * dn2)) - c2 * mean(e * r2 * hn), so ONE round of
// sums (c2 and the two means) serves both norms. For a gate a channel, dw1 and dgate are gate and w1 times the same column
// sum of scale * dt * xn, so two column sums cover three gradients.
// Everything is bound by memory: rows stay in registers between the sums and the write-back.
#include "host.h"
#include "ptx.cuh"
#include "vec.cuh"

namespace mb {

constexpr int kBnVec = 8;                          // elements a thread handles at a time
constexpr int kBnMaxH = 16384;
constexpr int kBnMaxThreads = 512;

struct BlockNormFwdArgs {
  const void *x, *residual, *w1, *w2, *gate;
  void *h, *y;
  float *r1, *r2;
  long long rows;
  int H, gate_mode;         // 0 none, 1 a channel, 2 an element
  float scale, eps;
};

struct BlockNormBwdArgs {
  const void *dy, *dh, *x, *h, *w1, *w2, *gate;    // dy, dh: null where the output was not used
  const float *r1, *r2;
  void *dx, *dres, *dgate;  // dgate: the [rows, H] one
  float *part1, *part2;     // [CTAs, H] column sums of scale * dt * gate' * xn (gate' = gate an element, else 1) and of dy * hn
  long long rows;
  int H, gate_mode;
  float scale;
};

// Sums over the `threads` of one row (a multiple of 32), the same for all of them. A row that has a warp to
// itself needs no barrier.
template <int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*red)[K], int threads) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (threads == 32) return;
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  if (l == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[w][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = l < (threads >> 5) ? red[l][k] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

// blockDim = (threads of a row, rows of the block); V vectors a thread.
template <typename T, int V>
__global__ void __launch_bounds__(kBnMaxThreads) block_norm_fwd_kernel(const BlockNormFwdArgs p) {
  __shared__ float red1[32][1], red2[32][1];
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;                       // whole warps; several rows to a block only where a row is one warp
  const long long base = row * p.H;
  const T* x = static_cast<const T*>(p.x) + base;
  const T* res = static_cast<const T*>(p.residual) + base;
  const T *w1 = static_cast<const T*>(p.w1), *w2 = static_cast<const T*>(p.w2);
  const T* gate = p.gate_mode == 0 ? nullptr : static_cast<const T*>(p.gate) + (p.gate_mode == 2 ? base : 0);
  Vec<T, kBnVec> a[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    a[j].zero(), b[j].zero();
    if (c < p.H) {
      a[j].load_once(x + c);
      b[j].load_once(res + c);
    }
  }
  float r1 = 1.f;
  if (w1) {
    float ss[1] = {0.f};
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < kBnVec; ++i) ss[0] += a[j].get(i) * a[j].get(i);
    row_sums(ss, red1, blockDim.x);
    r1 = rsqrtf(ss[0] / static_cast<float>(p.H) + p.eps);
    if (threadIdx.x == 0 && p.r1) p.r1[row] = r1;
  }
  float h[V][kBnVec], ss[1] = {0.f};
  T* ho = static_cast<T*>(p.h) + base;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      Vec<T, kBnVec> w, g, o;
      if (w1) w.load(w1 + c);
      if (gate) g.load(gate + c);
#pragma unroll
      for (int i = 0; i < kBnVec; ++i) {
        float u = a[j].get(i);
        if (w1) u = u * r1 * w.get(i);
        if (gate) u *= g.get(i);
        // the norm below sees the sum before its rounding to the stream's type: one rounding less in y
        h[j][i] = fmaf(p.scale, u, b[j].get(i));
        o.set(i, h[j][i]);
        ss[0] += h[j][i] * h[j][i];
      }
      o.store(ho + c);
    }
  }
  if (!w2) return;
  row_sums(ss, red2, blockDim.x);
  const float r2 = rsqrtf(ss[0] / static_cast<float>(p.H) + p.eps);
  if (threadIdx.x == 0 && p.r2) p.r2[row] = r2;
  T* y = static_cast<T*>(p.y) + base;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      Vec<T, kBnVec> w, o;
      w.load(w2 + c);
#pragma unroll
      for (int i = 0; i < kBnVec; ++i) o.set(i, h[j][i] * r2 * w.get(i));
      o.store(y + c);
    }
  }
}

// What the backward reads of one row.
template <typename T, int V, bool PRE, int GATE>
struct BlockNormRow {
  Vec<T, kBnVec> x[V], dh[V], h[PRE ? V : 1], dy[PRE ? V : 1], g[GATE == 2 ? V : 1];
  float r1, r2;
  __device__ __forceinline__ void load(const BlockNormBwdArgs& p, long long row) {
    const long long base = row * p.H;
    r1 = p.w1 ? p.r1[row] : 1.f, r2 = PRE ? p.r2[row] : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
      x[j].zero(), dh[j].zero();
      if (PRE) h[j].zero(), dy[j].zero();
      if (GATE == 2) g[j].zero();
      if (c < p.H) {
        if (p.x) x[j].load_once(static_cast<const T*>(p.x) + base + c);
        if (p.dh) dh[j].load_once(static_cast<const T*>(p.dh) + base + c);
        if (PRE) h[j].load_once(static_cast<const T*>(p.h) + base + c);
        if (PRE && p.dy) dy[j].load_once(static_cast<const T*>(p.dy) + base + c);
        if (GATE == 2) g[j].load_once(static_cast<const T*>(p.gate) + base + c);
      }
    }
  }
};

// Rows blockIdx.x, + gridDim.x, ...; a thread keeps the column sums of its V vectors and, one row ahead, its loads in registers.
// Without the loads ahead the barrier in the middle of a row leaves memory idle: 8192 rows of 4096 in bf16 took 149 us.
template <typename T, int V, bool PRE, int GATE>
__global__ void __launch_bounds__(kBnMaxThreads, 1) block_norm_bwd_kernel(const BlockNormBwdArgs p) {
  __shared__ float red[2][32][3];                  // two, so that one barrier a row is enough
  const T *w1 = static_cast<const T*>(p.w1), *w2 = static_cast<const T*>(p.w2);
  Vec<T, kBnVec> v1[V], v2[PRE ? V : 1], vg[GATE == 1 ? V : 1];
  float s1[V][kBnVec], s2[PRE ? V : 1][kBnVec];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      if (w1) v1[j].load(w1 + c);
      if (PRE) v2[j].load(w2 + c);
      if (GATE == 1) vg[j].load(static_cast<const T*>(p.gate) + c);
    }
#pragma unroll
    for (int i = 0; i < kBnVec; ++i) {
      s1[j][i] = 0.f;
      if (PRE) s2[j][i] = 0.f;
    }
  }
  const float inv = 1.f / static_cast<float>(p.H);
  int parity = 0;
  BlockNormRow<T, V, PRE, GATE> cur, next;
  if (static_cast<long long>(blockIdx.x) < p.rows) cur.load(p, blockIdx.x);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, parity ^= 1) {
    if (row + gridDim.x < p.rows) next.load(p, row + gridDim.x);
    const float r1 = cur.r1, r2 = cur.r2;
    float sums[3] = {0.f, 0.f, 0.f};               // dn2 * hn, e * (dh + r2 * dn2), e * r2 * hn
    auto gate = [&](int j, int i) { return GATE == 1 ? vg[GATE == 1 ? j : 0].get(i) : GATE == 2 ? cur.g[GATE == 2 ? j : 0].get(i) : 1.f; };
    if (PRE || w1) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
        if (c < p.H) {
#pragma unroll
          for (int i = 0; i < kBnVec; ++i) {
            const float hn = PRE ? cur.h[PRE ? j : 0].get(i) * r2 : 0.f, dyi = PRE ? cur.dy[PRE ? j : 0].get(i) : 0.f;
            const float dn2 = PRE ? dyi * v2[PRE ? j : 0].get(i) : 0.f;
            if (PRE) {
              sums[0] += dn2 * hn;
              s2[PRE ? j : 0][i] += dyi * hn;
            }
            if (w1) {
              const float e = cur.x[j].get(i) * r1 * v1[j].get(i) * p.scale * gate(j, i);
              sums[1] += e * (cur.dh[j].get(i) + r2 * dn2);
              if (PRE) sums[2] += e * r2 * hn;
            }
          }
        }
      }
      row_sums(sums, red[parity], blockDim.x);
    }
    const float c2 = sums[0] * inv, c1 = (sums[1] - c2 * sums[2]) * inv;
    const long long base = row * p.H;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
      if (c < p.H) {
        Vec<T, kBnVec> ox, or_, og;
#pragma unroll
        for (int i = 0; i < kBnVec; ++i) {
          const float gi = gate(j, i);
          float dt = cur.dh[j].get(i);
          if (PRE) dt += r2 * (cur.dy[PRE ? j : 0].get(i) * v2[PRE ? j : 0].get(i) - cur.h[PRE ? j : 0].get(i) * r2 * c2);
          const float sd = p.scale * dt, xn = cur.x[j].get(i) * r1;
          or_.set(i, dt);
          if (GATE == 2) og.set(i, sd * xn * (w1 ? v1[j].get(i) : 1.f));
          s1[j][i] += sd * xn * (GATE == 2 ? gi : 1.f);
          float du = sd * gi;
          if (w1) du = r1 * (du * v1[j].get(i) - xn * c1);
          ox.set(i, du);
        }
        or_.store(static_cast<T*>(p.dres) + base + c);
        ox.store(static_cast<T*>(p.dx) + base + c);
        if (GATE == 2) og.store(static_cast<T*>(p.dgate) + base + c);
      }
    }
    cur = next;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      const long long at = static_cast<long long>(blockIdx.x) * p.H + c;
#pragma unroll
      for (int i = 0; i < kBnVec; i += 4) {
        if (p.part1) *reinterpret_cast<float4*>(p.part1 + at + i) = make_float4(s1[j][i], s1[j][i + 1], s1[j][i + 2], s1[j][i + 3]);
        if (PRE) *reinterpret_cast<float4*>(p.part2 + at + i) = make_float4(s2[PRE ? j : 0][i], s2[PRE ? j : 0][i + 1], s2[PRE ? j : 0][i + 2], s2[PRE ? j : 0][i + 3]);
      }
    }
  }
}

// dw1 = gate_c * S1, dgate = w1 * S1, dw2 = S2 (S: sums of the CTAs' column sums, in their order). 32 columns a block, the
// partial rows divided over 16 warps.
constexpr int kBnColWarps = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kBnColWarps) block_norm_columns_kernel(const float* __restrict__ part1, const float* __restrict__ part2,
                                                                              int parts, int H, const T* __restrict__ w1,
                                                                              const T* __restrict__ gate, T* __restrict__ dw1,
                                                                              T* __restrict__ dgate, T* __restrict__ dw2) {
  __shared__ float red[kBnColWarps][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* part = blockIdx.y ? part2 : part1;
  float a = 0.f;
  if (c < H) {
    part += c;
#pragma unroll 10
    for (int r = threadIdx.y; r < parts; r += kBnColWarps) a += part[static_cast<long long>(r) * H];
  }
  red[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y != 0 || c >= H) return;
  a = 0.f;
#pragma unroll
  for (int r = 0; r < kBnColWarps; ++r) a += red[r][threadIdx.x];
  if (blockIdx.y) {
    dw2[c] = from_float<T>(a);
    return;
  }
  if (dw1) dw1[c] = from_float<T>(gate ? a * to_float(gate[c]) : a);
  if (dgate) dgate[c] = from_float<T>(w1 ? a * to_float(w1[c]) : a);
}

// Threads of a row for V vectors each: whole warps that cover the row.
static int bn_threads(int H, int V) { return ((H / kBnVec + V - 1) / V + 31) / 32 * 32; }

template <typename T>
static int launch_block_norm_fwd(const BlockNormFwdArgs& a, cudaStream_t stream) {
  const int V = a.H <= 128 * kBnVec ? 1 : a.H <= 1024 * kBnVec ? 2 : 4;
  const int x = bn_threads(a.H, V), y = x == 32 ? 4 : 1;
  const long long grid = (a.rows + y - 1) / y;
  const dim3 block(x, y);
  if (V == 1) block_norm_fwd_kernel<T, 1><<<static_cast<unsigned>(grid), block, 0, stream>>>(a);
  else if (V == 2) block_norm_fwd_kernel<T, 2><<<static_cast<unsigned>(grid), block, 0, stream>>>(a);
  else block_norm_fwd_kernel<T, 4><<<static_cast<unsigned>(grid), block, 0, stream>>>(a);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

static int bn_bwd_vectors(int H) { return H <= 512 * kBnVec ? 1 : H <= 1024 * kBnVec ? 2 : 4; }

// CTAs of the backward, each of which leaves a row of column sums: as many as fit the SMs at once, by their threads.
static int bn_bwd_ctas(long long rows, int H) {
  const int x = bn_threads(H, bn_bwd_vectors(H));
  const long long n = static_cast<long long>(sm_count()) * (x > 256 ? 1 : x > 128 ? 2 : 4);
  return static_cast<int>(rows < n ? rows : n);
}

template <typename T, int V, bool PRE>
static void bn_bwd_gate(const BlockNormBwdArgs& a, int ctas, int x, cudaStream_t stream) {
  if (a.gate_mode == 0) block_norm_bwd_kernel<T, V, PRE, 0><<<ctas, x, 0, stream>>>(a);
  else if (a.gate_mode == 1) block_norm_bwd_kernel<T, V, PRE, 1><<<ctas, x, 0, stream>>>(a);
  else block_norm_bwd_kernel<T, V, PRE, 2><<<ctas, x, 0, stream>>>(a);
}

template <typename T>
static int launch_block_norm_bwd(const BlockNormBwdArgs& a, void* dw1, void* dgate, void* dw2, cudaStream_t stream) {
  const int V = bn_bwd_vectors(a.H), ctas = bn_bwd_ctas(a.rows, a.H), x = bn_threads(a.H, V);
  if (a.w2) {
    if (V == 1) bn_bwd_gate<T, 1, true>(a, ctas, x, stream);
    else if (V == 2) bn_bwd_gate<T, 2, true>(a, ctas, x, stream);
    else bn_bwd_gate<T, 4, true>(a, ctas, x, stream);
  } else {
    if (V == 1) bn_bwd_gate<T, 1, false>(a, ctas, x, stream);
    else if (V == 2) bn_bwd_gate<T, 2, false>(a, ctas, x, stream);
    else bn_bwd_gate<T, 4, false>(a, ctas, x, stream);
  }
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  if (a.part1 || a.part2) {
    // part1 in the grid's first row, part2 in its second; without part1 the first row has nothing to write
    block_norm_columns_kernel<T><<<dim3((a.H + 31) / 32, a.part2 ? 2 : 1), dim3(32, kBnColWarps), 0, stream>>>(
        a.part1 ? a.part1 : a.part2, a.part2, ctas, a.H, static_cast<const T*>(a.w1),
        a.gate_mode == 1 ? static_cast<const T*>(a.gate) : nullptr, static_cast<T*>(dw1), static_cast<T*>(dgate), static_cast<T*>(dw2));
    count_launch();
    MB_CHECK_CUDA(cudaGetLastError());
  }
  return 0;
}

static const char* block_norm_problem(int dtype, long long rows, int H, int gate_mode, const void* gate, const void* const* pointers, int n) {
  if (dtype < 0 || dtype > 2) return "block_norm: bf16, fp16 or fp32";
  if (H < kBnVec || H % kBnVec != 0 || H > kBnMaxH) return "block_norm: hidden size must be a multiple of 8, at most 16384";
  if (rows < 1 || rows >= (1ll << 31)) return "block_norm: rows must be positive and below 2^31";
  if (gate_mode < 0 || gate_mode > 2 || (gate_mode != 0) != (gate != nullptr)) return "block_norm: gate and its kind do not agree";
  for (int i = 0; i < n; ++i)
    if (reinterpret_cast<uintptr_t>(pointers[i]) & 15) return "block_norm: tensors must be 16-byte aligned";
  return nullptr;
}

}  // namespace mb

// x, residual, h, y [rows, H], w1, w2 [H] or null, gate by gate_mode; r1, r2 [rows] fp32 (or null); dtype 0 bf16, 1 fp16, 2 fp32.
// y and r2 go with w2, r1 with w1.
MB_API int mb_block_norm_fwd(const void* x, const void* residual, const void* w1, const void* w2, const void* gate, int gate_mode, void* h,
                             void* y, float* r1, float* r2, int dtype, long long rows, int H, float scale, float eps, cudaStream_t stream) {
  using namespace mb;
  const void* pointers[] = {x, residual, w1, w2, gate, h, y};
  const char* what = block_norm_problem(dtype, rows, H, gate_mode, gate, pointers, 7);
  if (!what && (w2 != nullptr) != (y != nullptr)) what = "block_norm: y goes with the second weight";
  if (what) {
    set_last_error(what);
    return -1;
  }
  const BlockNormFwdArgs a = {x, residual, w1, w2, gate, h, y, r1, r2, rows, H, gate_mode, scale, eps};
  if (dtype == 2) return launch_block_norm_fwd<float>(a, stream);
  if (dtype == 1) return launch_block_norm_fwd<__half>(a, stream);
  return launch_block_norm_fwd<__nv_bfloat16>(a, stream);
}

// Rows of fp32 column sums that the backward needs as scratch (H floats each, for each of the two sums that are asked for).
MB_API int mb_block_norm_bwd_parts(long long rows, int H) {
  return H < mb::kBnVec || H > mb::kBnMaxH ? 0 : mb::bn_bwd_ctas(rows, H);
}

// Gradients of mb_block_norm_fwd. dy / dh null: that output has no gradient. dgate: [H] or [rows, H] by gate_mode. part1 goes with
// dw1 or a [H] dgate, part2 with dw2; x null where neither w1 nor a gate needs it.
MB_API int mb_block_norm_bwd(const void* dy, const void* dh, const void* x, const void* h, const void* w1, const void* w2, const void* gate,
                             int gate_mode, const float* r1, const float* r2, void* dx, void* dresidual, void* dw1, void* dw2, void* dgate,
                             float* part1, float* part2, int dtype, long long rows, int H, float scale, cudaStream_t stream) {
  using namespace mb;
  const void* pointers[] = {dy, dh, x, h, w1, w2, gate, dx, dresidual, dgate, part1, part2};
  const char* what = block_norm_problem(dtype, rows, H, gate_mode, gate, pointers, 12);
  if (!what && ((w1 && (!r1 || !x || !dw1)) || (w2 && (!r2 || !h || !dw2 || !part2)) || (gate && (!x || !dgate)) || !dx || !dresidual ||
                ((w1 || gate_mode == 1) && !part1)))
    what = "mb_block_norm_bwd: a tensor that these arguments need is missing";
  if (what) {
    set_last_error(what);
    return -1;
  }
  const BlockNormBwdArgs a = {dy, dh, x, h, w1, w2, gate, r1, r2, dx, dresidual, gate_mode == 2 ? dgate : nullptr,
                              w1 || gate_mode == 1 ? part1 : nullptr, w2 ? part2 : nullptr, rows, H, gate_mode, scale};
  void* dgate_c = gate_mode == 1 ? dgate : nullptr;
  if (dtype == 2) return launch_block_norm_bwd<float>(a, dw1, dgate_c, dw2, stream);
  if (dtype == 1) return launch_block_norm_bwd<__half>(a, dw1, dgate_c, dw2, stream);
  return launch_block_norm_bwd<__nv_bfloat16>(a, dw1, dgate_c, dw2, stream);
}
