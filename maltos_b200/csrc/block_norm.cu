// The seam between two blocks of a decoder in one pass, forward and backward (bf16, fp16, fp32, math in fp32):
//   u = w1 * x * r1,  r1 = rsqrt(mean(x^2) + eps)      (u = x without w1)         norm after the block
//   h = residual + scale * gate * u                     (gate: none, [H], or [rows, H])
//   y = w2 * h * r2,  r2 = rsqrt(mean(h^2) + eps)       (not without w2)           norm before the next block
// The forward keeps r1 and r2, the backward needs x, h and the two of them:
//   dn2 = dy * w2, hn = h * r2, c2 = mean(dn2 * hn);  dt = dh + r2 * (dn2 - hn * c2)      = dresidual
//   dg = scale * dt * u;  dn1 = scale * gate * dt * w1, xn = x * r1, c1 = mean(dn1 * xn);  dx = r1 * (dn1 - xn * c1)
// c1 is linear in dt: with a = gate * w1 * xn it is scale * (mean(a * (dh + r2 * dn2)) - r2 * c2 * mean(a * hn)), so ONE round of
// sums (c2 and the two means) serves both norms. Products are formed around xn and hn, which are of order one: with r1 * r1 or
// r2 * r2 taken out of the sums, rows of 1e15 and more (or 1e-13 and less, with a small eps) left the range of fp32 on the way,
// and dx lost its second term or was infinite although the gradient itself is well inside. For a gate a channel, dw1 and dgate are
// gate and w1 times the same column sum of scale * dt * xn, so two column sums cover three gradients.
// The backward reads h as it was stored, rounded to the stream's type, while r2 is of the sum before: forming h again would hold x's
// residual for the backward too. It puts half a step of h, at random, into the terms of dnext_weight and of dt's mean (relative
// error against 64 bits 0.0024 in bf16, 0.0017 with h in fp32).
// The forward is bound by memory, rows in registers between the sums and the write-back: 8192 rows of 4096 in bf16 take 51 us (5.2
// TB/s; launches in a graph, L2 flushed between), forward and backward 139 to 141 us, of which 8 us are the column sums; 4093 rows of
// 5120 with a gate a channel 127 us. The backward (90 us by itself) waits: at 0.66 instructions a cycle and scheduler and 50 % of the DRAM
// rate neither is at its limit, and every row has a barrier in its middle.
#include "host.h"
#include "ptx.cuh"
#include "vec.cuh"

namespace mb {

constexpr int kBnVec = 8;                          // elements a thread handles at a time
constexpr int kBnMaxH = 16384;
constexpr int kBnMaxThreads = 512;
template <typename T> constexpr bool bn_is_half = false;
template <> constexpr bool bn_is_half<__half> = true;

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
  int* status;
};

// The sum over the `threads` of one row (a multiple of 32), the same for all of them. A row that has a warp to itself needs no
// barrier.
__device__ __forceinline__ float row_sum(float v, float* red, int threads) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threads == 32) return v;
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  if (l == 0) red[w] = v;
  __syncthreads();
  v = l < (threads >> 5) ? red[l] : 0.f;
#pragma unroll
  for (int o = kBnMaxThreads / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}

// Three of them at once: lane l of four takes on value l, so that the three cost 12 shuffles and not 27.
__device__ __forceinline__ void row_sums(float (&v)[3], float (*red)[4], int threads) {
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  float a = (l & 1) ? v[1] : v[0];
  a += __shfl_xor_sync(0xffffffffu, (l & 1) ? v[0] : v[1], 1);
  const float b = v[2] + __shfl_xor_sync(0xffffffffu, v[2], 1);
  float c = (l & 2) ? b : a;
  c += __shfl_xor_sync(0xffffffffu, (l & 2) ? a : b, 2);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  if (threads > 32) {
    if (l < 4) red[w][l] = c;
    __syncthreads();
    const int warps = threads >> 5;
    c = 0.f;
    for (int from = l >> 2; from < warps; from += 8) c += red[from][l & 3];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = __shfl_sync(0xffffffffu, c, k);
}

// Elements 2i and 2i + 1 of a vector as a pair of fp32, for the two-wide multiply-adds: between load and store these kernels are
// held up by their instructions as much as by memory (8192 rows of 4096, one element at a time: forward 52 us for 46).
template <typename T>
__device__ __forceinline__ uint64_t pair_of(const Vec<T, kBnVec>& v, int i) {
  if constexpr (sizeof(T) == 4) return f32x2(v.at[2 * i], v.at[2 * i + 1]);
  else if constexpr (sizeof(T) == 2 && !bn_is_half<T>) return bf16x2_as_f32x2(v.word[i]);
  else return f32x2(to_float(v.at[2 * i]), to_float(v.at[2 * i + 1]));
}
template <typename T>
__device__ __forceinline__ void set_pair(Vec<T, kBnVec>& v, int i, uint64_t x) {
  float lo, hi;
  f32x2_split(x, lo, hi);
  if constexpr (sizeof(T) == 2 && !bn_is_half<T>) v.word[i] = pack_bf16x2(lo, hi);
  else v.set(2 * i, lo), v.set(2 * i + 1, hi);
}
__device__ __forceinline__ float both(uint64_t x) {
  float lo, hi;
  f32x2_split(x, lo, hi);
  return lo + hi;
}
constexpr int kBnPairs = kBnVec / 2;

// blockDim = (threads of a row, rows of the block); V vectors a thread. Memory is kept busy by the rows that an SM has at once, so the
// registers are held to what three of the largest blocks (two of four vectors, or in fp32) leave to each, for a few spilled bytes:
// 4096 rows of 8192 in bf16 53 us for 63, 2048 of 16384 53 for 72.
constexpr int bn_fwd_blocks(int size, int V) { return size == 4 ? (V == 4 ? 1 : 2) : V == 4 ? 2 : 3; }
template <typename T, int V>
__global__ void __launch_bounds__(kBnMaxThreads, bn_fwd_blocks(sizeof(T), V)) block_norm_fwd_kernel(const BlockNormFwdArgs p) {
  __shared__ float red1[kBnMaxThreads / 32], red2[kBnMaxThreads / 32];
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
    uint64_t squares = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < kBnPairs; ++i) squares = fma_f32x2(pair_of(a[j], i), pair_of(a[j], i), squares);
    r1 = rsqrtf(row_sum(both(squares), red1, blockDim.x) / static_cast<float>(p.H) + p.eps);
    if (threadIdx.x == 0 && p.r1) p.r1[row] = r1;
  }
  uint64_t h[V][kBnPairs], squares = 0;
  const uint64_t r1_2 = f32x2(r1, r1), scale_2 = f32x2(p.scale, p.scale);
  T* ho = static_cast<T*>(p.h) + base;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      Vec<T, kBnVec> w, g, o;
      if (w1) w.load(w1 + c);
      if (gate) g.load(gate + c);
#pragma unroll
      for (int i = 0; i < kBnPairs; ++i) {
        uint64_t u = pair_of(a[j], i);
        if (w1) u = mul_f32x2(mul_f32x2(u, r1_2), pair_of(w, i));
        if (gate) u = mul_f32x2(u, pair_of(g, i));
        // the norm below sees the sum before its rounding to the stream's type: one rounding less in y
        h[j][i] = fma_f32x2(scale_2, u, pair_of(b[j], i));
        set_pair(o, i, h[j][i]);
        squares = fma_f32x2(h[j][i], h[j][i], squares);
      }
      o.store(ho + c);
    }
  }
  if (!w2) return;
  const float r2 = rsqrtf(row_sum(both(squares), red2, blockDim.x) / static_cast<float>(p.H) + p.eps);
  if (threadIdx.x == 0 && p.r2) p.r2[row] = r2;
  const uint64_t r2_2 = f32x2(r2, r2);
  T* y = static_cast<T*>(p.y) + base;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * kBnVec;
    if (c < p.H) {
      Vec<T, kBnVec> w, o;
      w.load(w2 + c);
#pragma unroll
      for (int i = 0; i < kBnPairs; ++i) set_pair(o, i, mul_f32x2(mul_f32x2(h[j][i], r2_2), pair_of(w, i)));
      o.store(y + c);
    }
  }
}

// The backward's ring of row pieces in shared memory: piece j of a row is its columns [j * 8 * blockDim.x, ...), one vector a thread.
struct BlockNormRing {
  int slots;                // 0: no ring, the row is read from memory twice
  int slot_bytes;
  int at[5];                // of x, dh, h, dy and the gate in a slot; -1 where absent
};
constexpr int kBnMaxSlots = 16;

// Threads of an SM, at most of a row, in the backward. One vector a thread of a 16-bit type fits 64 registers (with a few spilled):
// 1024 threads hide more than 512 with two vectors each (8192 rows of 4096: 87 us against 94; 4093 of 5120, where 320 threads
// would have an SM to themselves: 86 against 129). In fp32 that would spill 150 bytes a thread (4096 rows of 4096: 106 against 75).
constexpr int bn_bwd_threads(int size, int V) { return size == 2 && V == 1 ? 1024 : 512; }
constexpr int bn_bwd_vectors(int size, int H) { return H <= bn_bwd_threads(size, 1) * kBnVec ? 1 : H <= 1024 * kBnVec ? 2 : 4; }

// Rows blockIdx.x, + gridDim.x, ...; a thread keeps the column sums of its V vectors. What a row needs is brought by bulk copies
// into a ring that is as deep as shared memory allows, so that memory is busy through the barrier in the middle of a row.
template <typename T, int V, bool PRE, int GATE>
__global__ void __launch_bounds__(bn_bwd_threads(sizeof(T), V), 1) block_norm_bwd_kernel(const BlockNormBwdArgs p, const BlockNormRing ring) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][bn_bwd_threads(sizeof(T), V) / 32][4];  // two, so that one barrier a row is enough
  __shared__ __align__(8) uint64_t full[kBnMaxSlots];
  __shared__ int control[2];                       // abort flag, wait limit
  volatile int* abort_flag = control;
  constexpr bool KEEP = V == 1;                    // the weights, and b below from pass to pass, stay in registers
  const T *w1 = static_cast<const T*>(p.w1), *w2 = static_cast<const T*>(p.w2), *wg = static_cast<const T*>(p.gate);
  const void* const source[5] = {p.x, p.dh, p.h, p.dy, GATE == 2 ? p.gate : nullptr};
  const int tid = threadIdx.x, width = blockDim.x * kBnVec;
  const int n = static_cast<int>((p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);   // rows of this CTA: the grid is at most p.rows
  if (tid == 0) {
    abort_flag[0] = 0;
    abort_flag[1] = p.status[3];
    for (int i = 0; i < ring.slots; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncthreads();
  // by thread 0: piece j of the CTA's row `it` into a slot
  auto issue = [&](int slot, int it, int j) {
    const long long at = (blockIdx.x + static_cast<long long>(it) * gridDim.x) * p.H + j * width;
    const uint32_t bytes = static_cast<uint32_t>(min(p.H - j * width, width)) * sizeof(T);
    uint32_t all = 0;
#pragma unroll
    for (int k = 0; k < 5; ++k) all += ring.at[k] >= 0 ? bytes : 0u;
    mbar_arrive_expect_tx(&full[slot], all);
#pragma unroll
    for (int k = 0; k < 5; ++k)
      if (ring.at[k] >= 0) bulk_load(smem + slot * ring.slot_bytes + ring.at[k], static_cast<const T*>(source[k]) + at, bytes, &full[slot]);
  };
  if (tid == 0)
    for (int q = 0; q < min(ring.slots, n * V); ++q) issue(q, q / V, q % V);
  // when everyone is done with row `it`, whose first piece is in `first`: what comes next into its slots
  auto refill = [&](int first, int it) {
    for (int q = it * V + ring.slots; q < min((it + 1) * V + ring.slots, n * V); ++q) {
      issue(first, q / V, q % V);
      if (++first == ring.slots) first = 0;
    }
  };

  Vec<T, kBnVec> v1[KEEP ? V : 1], v2[KEEP && PRE ? V : 1], vg[KEEP && GATE == 1 ? V : 1];
  auto load_weights = [&](int j) {
    const int m = KEEP ? j : 0, c = tid * kBnVec + j * width;
    if (w1) v1[m].load(w1 + c);
    if (PRE) v2[PRE ? m : 0].load(w2 + c);
    if (GATE == 1) vg[GATE == 1 ? m : 0].load(wg + c);
  };
  uint64_t s1[V][kBnPairs], s2[PRE ? V : 1][kBnPairs];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (KEEP && tid * kBnVec + j * width < p.H) load_weights(j);
#pragma unroll
    for (int i = 0; i < kBnPairs; ++i) s1[j][i] = s2[PRE ? j : 0][i] = 0;
  }
  const float inv = 1.f / static_cast<float>(p.H);
  int slot0 = 0, phase0 = 0;                       // of the row's first piece
  float next_r1 = p.w1 ? p.r1[blockIdx.x] : 1.f, next_r2 = PRE ? p.r2[blockIdx.x] : 0.f;
  for (int it = 0; it < n; ++it) {
    const long long row = blockIdx.x + static_cast<long long>(it) * gridDim.x, base = row * p.H;
    const float r1 = next_r1, r2 = next_r2;
    if (it + 1 < n) {
      if (p.w1) next_r1 = p.r1[row + gridDim.x];
      if (PRE) next_r2 = p.r2[row + gridDim.x];
    }
    const uint64_t r1_2 = f32x2(r1, r1), r2_2 = f32x2(r2, r2);
    // of a piece: x, h, the gate and b = dh + r2 * dn2
    Vec<T, kBnVec> x, h, g;
    uint64_t b[KEEP ? V : 1][kBnPairs], acc[3] = {0, 0, 0};
    auto gated = [&](uint64_t v, int j, int i) {
      return GATE == 0 ? v : mul_f32x2(v, GATE == 2 ? pair_of(g, i) : pair_of(vg[KEEP && GATE == 1 ? j : 0], i));
    };
    auto values = [&](int j, bool first_pass) {
      const int m = KEEP ? j : 0, c = tid * kBnVec + j * width;
      const int s = slot0 + j >= ring.slots ? slot0 + j - ring.slots : slot0 + j;
      auto fetch = [&](int k) {
        Vec<T, kBnVec> v;
        v.zero();
        if (ring.slots) {
          if (ring.at[k] >= 0) v.load_shared(reinterpret_cast<const T*>(smem + s * ring.slot_bytes + ring.at[k]) + tid * kBnVec);
        } else if (source[k]) {
          v.load(static_cast<const T*>(source[k]) + base + c);
        }
        return v;
      };
      x = fetch(0);
      if (PRE) h = fetch(2);
      if (GATE == 2) g = fetch(4);
      if (KEEP && !first_pass) return;             // b and the weights are there
      if (!KEEP) load_weights(j);
      const Vec<T, kBnVec> dh = fetch(1);
#pragma unroll
      for (int i = 0; i < kBnPairs; ++i) b[m][i] = pair_of(dh, i);
      if (PRE) {
        const Vec<T, kBnVec> dy = fetch(3);
#pragma unroll
        for (int i = 0; i < kBnPairs; ++i) {
          const uint64_t dyr = mul_f32x2(pair_of(dy, i), r2_2), w = pair_of(v2[KEEP && PRE ? j : 0], i);
          if (first_pass) {
            const uint64_t dn2 = mul_f32x2(dyr, w);
            b[m][i] = add_f32x2(b[m][i], dn2);
            acc[0] = fma_f32x2(dn2, pair_of(h, i), acc[0]);
            s2[PRE ? j : 0][i] = fma_f32x2(dyr, pair_of(h, i), s2[PRE ? j : 0][i]);
          } else {
            b[m][i] = fma_f32x2(dyr, w, b[m][i]);
          }
        }
      }
    };
    // sums over the row of r2 * dn2 * h, a * b and a * h with a = gate * w1 * xn; what is the same for the whole row comes in later
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int s = slot0 + j, m = KEEP ? j : 0, c = tid * kBnVec + j * width;
      // (a wait that runs out: the sums are wrong, and the status says so)
      if (ring.slots) mbar_wait(&full[s >= ring.slots ? s - ring.slots : s], s >= ring.slots ? phase0 ^ 1 : phase0, abort_flag);
      if (c < p.H && (PRE || w1 || KEEP)) {
        values(j, true);
        if (w1) {
#pragma unroll
          for (int i = 0; i < kBnPairs; ++i) {
            const uint64_t a = gated(mul_f32x2(mul_f32x2(pair_of(x, i), r1_2), pair_of(v1[KEEP ? j : 0], i)), j, i);
            acc[1] = fma_f32x2(a, b[m][i], acc[1]);
            if (PRE) acc[2] = fma_f32x2(a, pair_of(h, i), acc[2]);
          }
        }
      }
    }
    float sums[3] = {both(acc[0]), both(acc[1]), both(acc[2])};
    if (PRE || w1) row_sums(sums, red[it & 1], blockDim.x);
    else __syncthreads();
    __syncwarp();                                  // a row of one warp has no barrier
    const bool beside = ring.slots >= 2 * V;       // the next row fits beside this one
    if (tid == 0 && beside && it > 0) refill(slot0 >= V ? slot0 - V : slot0 - V + ring.slots, it - 1);   // everyone is done with the row before
    // with c2 = mean(dn2 * hn) and c1 = mean(scale * a * (b - r2 * hn * c2)): k2 = r2 * c2, k1 = r1 * c1
    const float k2 = r2 * (sums[0] * inv), sr1 = p.scale * r1;
    const float k1 = sr1 * ((sums[1] - k2 * (r2 * sums[2])) * inv);
    const uint64_t minus_k2 = f32x2(-k2, -k2), minus_k1 = f32x2(-k1, -k1), sr1_2 = f32x2(sr1, sr1);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = tid * kBnVec + j * width, m = KEEP ? j : 0, wm = KEEP ? j : 0;
      if (c < p.H) {
        values(j, false);
        Vec<T, kBnVec> ox, or_, og;
#pragma unroll
        for (int i = 0; i < kBnPairs; ++i) {
          const uint64_t dt = PRE ? fma_f32x2(mul_f32x2(pair_of(h, i), r2_2), minus_k2, b[m][i]) : b[m][i];
          set_pair(or_, i, dt);
          const uint64_t sdt = mul_f32x2(dt, sr1_2), xi = pair_of(x, i);   // scale * dt * r1; r1 is 1 without w1
          uint64_t du = w1 ? mul_f32x2(sdt, pair_of(v1[wm], i)) : sdt;
          if (GATE == 2) set_pair(og, i, mul_f32x2(du, xi));
          s1[j][i] = fma_f32x2(GATE == 2 ? gated(sdt, j, i) : sdt, xi, s1[j][i]);
          du = gated(du, j, i);
          if (w1) du = fma_f32x2(mul_f32x2(xi, r1_2), minus_k1, du);
          set_pair(ox, i, du);
        }
        or_.store(static_cast<T*>(p.dres) + base + c);
        ox.store(static_cast<T*>(p.dx) + base + c);
        if (GATE == 2) og.store(static_cast<T*>(p.dgate) + base + c);
      }
    }
    if (ring.slots && !beside) {
      __syncthreads();
      if (tid == 0) refill(slot0, it);
    }
    slot0 += V;
    if (ring.slots && slot0 >= ring.slots) slot0 -= ring.slots, phase0 ^= 1;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = tid * kBnVec + j * width;
    if (c < p.H) {
      const long long at = static_cast<long long>(blockIdx.x) * p.H + c;
#pragma unroll
      for (int i = 0; i < kBnPairs; i += 2) {
        if (p.part1) *reinterpret_cast<ulonglong2*>(p.part1 + at + 2 * i) = make_ulonglong2(s1[j][i], s1[j][i + 1]);
        if (PRE) *reinterpret_cast<ulonglong2*>(p.part2 + at + 2 * i) = make_ulonglong2(s2[PRE ? j : 0][i], s2[PRE ? j : 0][i + 1]);
      }
    }
  }
  if (*abort_flag) {
    __nanosleep(50000);
    if (tid == 0) {
      atomicOr(&p.status[0], MB_ERR_MBAR_TIMEOUT);
      p.status[1] = static_cast<int>(blockIdx.x);
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

// CTAs of the backward on an SM, and in all; each leaves a row of column sums.
static int bn_bwd_per_sm(int size, int V, int threads) { return bn_bwd_threads(size, V) / threads; }
static int bn_bwd_ctas(int size, long long rows, int H) {
  const int V = bn_bwd_vectors(size, H);
  const long long n = static_cast<long long>(sm_count()) * bn_bwd_per_sm(size, V, bn_threads(H, V));
  return static_cast<int>(rows < n ? rows : n);
}

// As many slots as fit beside the other CTAs of the SM and as a CTA has pieces. A row has to fit; where it does not (8192 < H in
// fp32, by the number of tensors) it is read from memory twice, the second time from L2.
template <typename T>
static BlockNormRing bn_bwd_ring(const BlockNormBwdArgs& a, int ctas, int threads, int V) {
  BlockNormRing r;
  const void* const source[5] = {a.x, a.dh, a.w2 ? a.h : nullptr, a.w2 ? a.dy : nullptr, a.gate_mode == 2 ? a.gate : nullptr};
  const int piece = threads * kBnVec * static_cast<int>(sizeof(T));
  r.slot_bytes = 0;
  for (int k = 0; k < 5; ++k) {
    r.at[k] = source[k] ? r.slot_bytes : -1;
    if (source[k]) r.slot_bytes += piece;
  }
  r.slots = 0;
  if (r.slot_bytes == 0) return r;
  const long long fit = (226 * 1024 / bn_bwd_per_sm(sizeof(T), V, threads) - 2560) / r.slot_bytes, pieces = (a.rows + ctas - 1) / ctas * V;
  r.slots = static_cast<int>(fit < kBnMaxSlots ? fit : kBnMaxSlots);
  if (r.slots < V) r.slots = 0;
  else if (pieces < r.slots) r.slots = static_cast<int>(pieces);
  return r;
}

template <typename T, int V, bool PRE, int GATE>
static int bn_bwd_launch(const BlockNormBwdArgs& a, int ctas, int threads, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  MB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    MB_CHECK_CUDA(cudaFuncSetAttribute(block_norm_bwd_kernel<T, V, PRE, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024 - 2560));
    configured[dev & 63] = true;
  }
  const BlockNormRing ring = bn_bwd_ring<T>(a, ctas, threads, V);
  block_norm_bwd_kernel<T, V, PRE, GATE><<<ctas, threads, ring.slots * ring.slot_bytes, stream>>>(a, ring);
  return 0;
}

template <typename T, int V, bool PRE>
static int bn_bwd_gate(const BlockNormBwdArgs& a, int ctas, int x, cudaStream_t stream) {
  if (a.gate_mode == 0) return bn_bwd_launch<T, V, PRE, 0>(a, ctas, x, stream);
  if (a.gate_mode == 1) return bn_bwd_launch<T, V, PRE, 1>(a, ctas, x, stream);
  return bn_bwd_launch<T, V, PRE, 2>(a, ctas, x, stream);
}

template <typename T>
static int launch_block_norm_bwd(const BlockNormBwdArgs& a, void* dw1, void* dgate, void* dw2, cudaStream_t stream) {
  const int V = bn_bwd_vectors(sizeof(T), a.H), ctas = bn_bwd_ctas(sizeof(T), a.rows, a.H), x = bn_threads(a.H, V);
  const bool pre = a.w2 != nullptr;
  int rc;
  if (V == 1) rc = pre ? bn_bwd_gate<T, 1, true>(a, ctas, x, stream) : bn_bwd_gate<T, 1, false>(a, ctas, x, stream);
  else if (V == 4) rc = pre ? bn_bwd_gate<T, 4, true>(a, ctas, x, stream) : bn_bwd_gate<T, 4, false>(a, ctas, x, stream);
  else if constexpr (sizeof(T) == 4) rc = pre ? bn_bwd_gate<T, 2, true>(a, ctas, x, stream) : bn_bwd_gate<T, 2, false>(a, ctas, x, stream);
  else rc = -1;                                    // (two vectors: fp32 only)
  if (rc) return rc;
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
MB_API int mb_block_norm_bwd_parts(int dtype, long long rows, int H) {
  return H < mb::kBnVec || H > mb::kBnMaxH ? 0 : mb::bn_bwd_ctas(dtype == 2 ? 4 : 2, rows, H);
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
  int* status = status_ptr();
  if (!status) return -4;
  const BlockNormBwdArgs a = {dy, dh, x, h, w1, w2, gate, r1, r2, dx, dresidual, gate_mode == 2 ? dgate : nullptr,
                              w1 || gate_mode == 1 ? part1 : nullptr, w2 ? part2 : nullptr, rows, H, gate_mode, scale, status};
  void* dgate_c = gate_mode == 1 ? dgate : nullptr;
  if (dtype == 2) return launch_block_norm_bwd<float>(a, dw1, dgate_c, dw2, stream);
  if (dtype == 1) return launch_block_norm_bwd<__half>(a, dw1, dgate_c, dw2, stream);
  return launch_block_norm_bwd<__nv_bfloat16>(a, dw1, dgate_c, dw2, stream);
}
