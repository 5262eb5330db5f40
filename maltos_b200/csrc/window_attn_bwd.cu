// Backward of sliding-window attention for sm_100a (rule: window.cuh, forward: window_attn.cu):
//   P = 2^(c S - lse2),  dP = dO V^T,  dS = P * (dP - delta),  delta = rowsum(dO * (out + out_lo)),
//   dV = P^T dO,  dK = scale * dS^T Q,  dQ = scale * dS K.
// Launches:
//   window_bwd_prep_kernel    delta and lse2, padded to whole tiles (padding rows get lse2 = +inf, so their P is zero); its first CTA
//                             writes the list of work for dK / dV;
//   window_bwd_dkdv_kernel    persistent; an item is 128 keys of one key/value head and a piece of the (query head, 128 query rows)
//                             that see them. Transposed products S^T = K Q^T and dP^T = V dO^T (TMEM lane = key) leave P^T and dS^T
//                             in tensor memory as the A operands of dV += P^T dO and dK += dS^T Q;
//   window_bwd_dq_kernel      persistent; an item is 128 query rows of one head, S double-buffered, dS written over S. At its end the
//                             CTAs add up key blocks whose work was cut into pieces, in the pieces' order (in a launch of its own,
//                             where a few blocks have all the pieces, that took 23 us of the layer's 570).
// The keys of first tokens are seen by every later query, so a block that holds some has many times the work of the others; and
// with few heads there are fewer blocks than SMs. Both are met by cutting a block's work into pieces. No atomics: the same bits
// every time.
// P and dS enter their products in bf16, since the operands of a UMMA have one type and Q, K and dO are bf16; sums are fp32. Each
// rounding is up to half a step of one term, at random over a sum's terms: dQ, dK and dV are 0.0030 to 0.0035 off relative to 64 bits,
// where their own rounding alone is 0.0017. delta is known to some 17 bits, from out and out_lo.
// What bounds it: the UMMAs (7 products of 128 x 128 x D a tile pair, against 5 that the mathematics needs) and the waits
// between them; see the notes at the two loops. Measured with the forward (launches in a graph, L2 flushed between): 8192 rows, 32 / 8
// heads of 128, window 1024 746 to 760 us, 606 to 596 TFLOP/s of the seven products counted (two boxes; preparation 42, dK / dV 328, dQ
// 236 each by itself under a profiler); 16384 rows, 8 / 2 heads, window 4096 1165 us, 725 TFLOP/s.
#include "host.h"
#include "ptx.cuh"
#include "window.cuh"

namespace mb {

constexpr int kWbArithWarps = 16;
constexpr int kWbThreads = 32 * (4 + kWbArithWarps);   // warp 0 TMA producer, warps 1..3 UMMA issuers, warps 4..19 arithmetic
constexpr float kWbLog2e = 1.4426950408889634f;

struct WindowBwdArgs {
  __nv_bfloat16 *dq, *dk, *dv;   // contiguous [B, S, H, D]
  const float *lse2, *delta;     // [B * Hq, Sq_pad]
  const int* list;               // [0]: entries, [1]: cut blocks; from 4 on: int4 {block, first, one past the last iteration, slot or -1}
  const int4* cuts;              // [list[1]] {block, first slot, pieces, -}: blocks of more than one piece
  float* parts;                  // [slots, Hkv, 2 (dK, dV), 128, D]
  WindowRule rule;
  int B, Sq, Sk, Hq, Hkv, Sq_pad;
  int key_blocks;                // of one row
  int row_tiles;                 // of 128 query rows
  float scale, scale_log2;
  int* status;
};

struct WindowBwdPrepArgs {
  const __nv_bfloat16 *out, *out_lo, *dout;
  long long do_tstride, do_bstride;
  const float* lse2_in;          // [B, Hq, Sq]
  float *lse2, *delta;
  int* list;
  int4* cuts;
  WindowRule rule;
  int B, Sq, Sk, Hq, Hkv, Sq_pad, key_blocks;
  int piece;                     // iterations of a piece
  int max_slots;
};

__device__ __forceinline__ float wb_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x for a pair, x <= 120, on the multiply-add pipe: x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves n in the low
// bits), 2^f by a polynomial on [-1/2, 1/2], n added to the exponent. The coefficients are the minimax fit of degree 4 to the
// relative error with p(0) = 1 (solved as a linear programme on a grid): 2.8e-6, far below the bf16 rounding that follows.
// x below -127 gives exactly 0: there n = -127, f = 0, and the exponent of 1 becomes that of zero.
__device__ __forceinline__ void wb_exp2_poly(uint64_t x, float& a, float& b) {
  float lo, hi;
  f32x2_split(x, lo, hi);
  x = f32x2(fmaxf(lo, -127.f), fmaxf(hi, -127.f));
  const uint64_t magic = f32x2(12582912.f, 12582912.f), minus_magic = f32x2(-12582912.f, -12582912.f), minus_one = f32x2(-1.f, -1.f);
  const uint64_t t = add_f32x2(x, magic);
  const uint64_t f = fma_f32x2(add_f32x2(t, minus_magic), minus_one, x);
  uint64_t r = fma_f32x2(f32x2(0.009582576341927052f, 0.009582576341927052f), f, f32x2(0.05590682849287987f, 0.05590682849287987f));
  r = fma_f32x2(r, f, f32x2(0.24024106562137604f, 0.24024106562137604f));
  r = fma_f32x2(r, f, f32x2(0.6931241154670715f, 0.6931241154670715f));
  r = fma_f32x2(r, f, f32x2(1.f, 1.f));
  float ta, tb, ra, rb;
  f32x2_split(t, ta, tb);
  f32x2_split(r, ra, rb);
  a = __uint_as_float(__float_as_uint(ra) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(rb) + (__float_as_uint(tb) << 23));
}

// Pair i of a thread's 16. Four warps share a scheduler here, and the special-function unit alone would take 1024 cycles a tile:
// one pair in kWbPolyOf goes to the multiply-add pipe.
constexpr int kWbPolyOf = 4;
__device__ __forceinline__ uint32_t wb_exp2_pair(uint64_t x, int i) {
  float a, b;
  if (i % kWbPolyOf == 0) {
    wb_exp2_poly(x, a, b);
  } else {
    f32x2_split(x, a, b);
    a = wb_exp2(a), b = wb_exp2(b);
  }
  return pack_bf16x2(a, b);
}

// ---------------------------------------------------------------------------------------------- preparation
constexpr int kWbPrepThreads = 1024;

// The list of work: every key block's iterations, (query heads of the group) x (query tiles that see it), cut into pieces.
__device__ void window_bwd_list(const WindowBwdPrepArgs& p) {
  __shared__ int warp_entries[32], warp_slots[32];
  __shared__ int total_entries, total_slots, total_cuts;
  __shared__ int found[kWbPrepThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int blocks = p.B * p.key_blocks, group = p.Hq / p.Hkv;
  int4* entry = reinterpret_cast<int4*>(p.list + 4);
  if (tid == 0) total_entries = total_slots = total_cuts = 0;
  __syncthreads();
  for (int base = 0; base < blocks; base += kWbPrepThreads) {
    // a block per thread; with documents a block's range is a warp's work, the blocks dealt out to the warps
    const int mine = base + tid;
    auto iterations = [&](int b) {
      const WindowKeys k = window_keys(p.rule, b / p.key_blocks, p.Sq, p.Sk, (b % p.key_blocks) * kWinBlock);
      return k.q_hi > k.q_lo ? ((k.q_hi + kWinBlock - 1) / kWinBlock - k.q_lo / kWinBlock) * group : 0;
    };
    if (p.rule.starts == nullptr) {
      found[tid] = mine < blocks ? iterations(mine) : 0;
    } else {
      for (int i = warp; i < kWbPrepThreads && base + i < blocks; i += 32) {
        const int n = iterations(base + i);
        if (lane == 0) found[i] = n;
      }
    }
    __syncthreads();
    const int n_iter = mine < blocks ? found[tid] : 0;
    int n = mine < blocks ? max(1, (n_iter + p.piece - 1) / p.piece) : 0;   // a block that nobody sees still has zeros to write
    // positions by a scan over the block
    auto scan = [&](int v, int* warps, int& total, int& before) {
      int inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      if (lane == 31) warps[warp] = inc;
      __syncthreads();
      int w = lane < warp ? warps[lane] : 0, all = warps[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o), all += __shfl_xor_sync(0xffffffffu, all, o);
      before = total + w + inc - v;
      __syncthreads();
      if (tid == 0) total += all;
      __syncthreads();
    };
    int slot = 0, at = 0, cut = 0;
    scan(n > 1 ? n : 0, warp_slots, total_slots, slot);
    if (n > 1 && slot + n > p.max_slots) n = 1;    // the caller's bound says that this does not happen
    scan(n, warp_entries, total_entries, at);
    scan(n > 1 ? 1 : 0, warp_slots, total_cuts, cut);
    if (mine < blocks) {
      if (n > 1) p.cuts[cut] = make_int4(mine, slot, n, 0);
      const int per = n > 1 ? p.piece : n_iter;
      for (int i = 0; i < n; ++i) entry[at + i] = make_int4(mine, i * per, min(n_iter, (i + 1) * per), n > 1 ? slot + i : -1);
    }
  }
  if (tid == 0) p.list[0] = total_entries, p.list[1] = total_cuts;
}

// CTA 0: the list. Others: delta and lse2, D / 8 lanes a row, rows in memory order.
template <int D>
__global__ void __launch_bounds__(kWbPrepThreads) window_bwd_prep_kernel(const WindowBwdPrepArgs p) {
  if (blockIdx.x == 0) {
    window_bwd_list(p);
    return;
  }
  constexpr int LANES = D / 8;
  const long long row = (static_cast<long long>(blockIdx.x - 1) * kWbPrepThreads + threadIdx.x) / LANES;   // (b, q, h), q to Sq_pad
  const int lane = threadIdx.x % LANES;
  if (row >= static_cast<long long>(p.B) * p.Sq_pad * p.Hq) return;   // whole warps: the product is a multiple of 128
  const int h = static_cast<int>(row % p.Hq);
  const long long bq = row / p.Hq;
  const int q = static_cast<int>(bq % p.Sq_pad), b = static_cast<int>(bq / p.Sq_pad);
  float acc = 0.f, l2 = INFINITY;
  if (q < p.Sq) {
    const long long o_at = ((static_cast<long long>(b) * p.Sq + q) * p.Hq + h) * D + lane * 8;
    const uint4 o = *reinterpret_cast<const uint4*>(p.out + o_at), r = *reinterpret_cast<const uint4*>(p.out_lo + o_at);
    const uint4 d = *reinterpret_cast<const uint4*>(p.dout + b * p.do_bstride + q * p.do_tstride + static_cast<long long>(h) * D + lane * 8);
    const uint32_t ov[4] = {o.x, o.y, o.z, o.w}, rv[4] = {r.x, r.y, r.z, r.w}, dv[4] = {d.x, d.y, d.z, d.w};
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fma_f32x2(add_f32x2(bf16x2_as_f32x2(ov[i]), bf16x2_as_f32x2(rv[i])), bf16x2_as_f32x2(dv[i]), sum);
    float lo, hi;
    f32x2_split(sum, lo, hi);
    acc = lo + hi;
    if (lane == 0) {
      l2 = p.lse2_in[(static_cast<long long>(b) * p.Hq + h) * p.Sq + q];
      if (l2 == -INFINITY) l2 = INFINITY;
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) {
    const long long at = (static_cast<long long>(b) * p.Hq + h) * p.Sq_pad + q;
    p.lse2[at] = l2;
    p.delta[at] = acc;
  }
}

// ---------------------------------------------------------------------------------------------- dK / dV
// One iteration is 128 keys x 128 queries of one head; S^T and dP^T have one TMEM buffer each. The tensor cores go
//     dV(i) | S(i+1) | dK(i) | dP(i+1)
// and the arithmetic warps alternate between the exponentials of S(i+1) (under dK(i), dP(i+1)) and dS(i) (under dV(i), S(i+1)).
// S(i+1) is what the arithmetic waits for, so dK and dP are issued behind it: left to themselves they share the tensor cores
// with it (4100 cycles an iteration, of 2048 of UMMAs). Each pair has an issuer of its own all the same, because a wait that is
// satisfied already costs 50 to 250 cycles, more the busier shared memory is, and so one pair's waits run under the other's
// products (3590 cycles with one issuer for all). A third Q tile lets its load start a whole iteration ahead. Blocks of 64
// queries, which would leave room for two buffers, are bound by shared memory: a UMMA with 64 columns reads its operands at 192
// bytes a cycle, of 128 that there are.
template <int D>
__global__ void __launch_bounds__(kWbThreads, 1)
window_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                       const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const WindowBwdArgs p) {
  constexpr int ATOMS = D / 64;
  constexpr int TILE_BYTES = kWinBlock * D * 2, ATOM_BYTES = kWinBlock * 128;
  constexpr int Q_STAGES = 3, STAGES = 2;           // tiles of Q; of dO, and of the statistics
  constexpr int AUX_BYTES = 2 * kWinBlock * 4;      // lse2, delta of one query tile
  constexpr uint32_t TMEM_COLS = 512, S_COL = 0, DP_COL = 128, DV_COL = 256, DK_COL = 256 + D;

  extern __shared__ __align__(1024) uint8_t smem_raw[];   // with head_dim 128 the tiles fill it: its start has to be aligned
  uint8_t* smem = smem_raw;
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE_BYTES;
  uint8_t* sQ = sV + TILE_BYTES;                    // Q_STAGES
  uint8_t* sDO = sQ + Q_STAGES * TILE_BYTES;        // STAGES
  uint8_t* sAux = sDO + STAGES * TILE_BYTES;        // STAGES x AUX_BYTES
  uint64_t* bars = reinterpret_cast<uint64_t*>(sAux + STAGES * AUX_BYTES);
  uint64_t* kv_full = bars;                 // 1
  uint64_t* kv_empty = bars + 1;            // 1 (both issuers)
  uint64_t* q_full = bars + 2;              // Q_STAGES
  uint64_t* q_empty = bars + 5;             // Q_STAGES
  uint64_t* do_full = bars + 8;             // STAGES
  uint64_t* do_empty = bars + 10;           // STAGES (both issuers: dV, dP)
  uint64_t* aux_full = bars + 12;           // STAGES
  uint64_t* aux_empty = bars + 14;          // STAGES
  uint64_t* s_full = bars + 16;             // 1
  uint64_t* p_full = bars + 17;             // 1
  uint64_t* dp_full = bars + 18;            // 1
  uint64_t* ds_full = bars + 19;            // 1
  uint64_t* acc_full = bars + 20;           // 1 (both issuers)
  uint64_t* s_issued = bars + 21;           // 2: S(i+1) is on its way, dK(i) may follow (two, so that none is lost)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {   // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_BAD_INDEX);
      p.status[2] = 1014;
    }
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 2);
    for (int i = 0; i < Q_STAGES; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 2);
      mbar_init(&s_issued[i], 1);
      mbar_init(&aux_full[i], 1);
      mbar_init(&aux_empty[i], kWbArithWarps);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, kWbArithWarps);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kWbArithWarps);
    mbar_init(acc_full, 2);
    abort_flag[0] = 0;
    abort_flag[1] = p.status[3];
    fence_barrier_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmDO);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int group = p.Hq / p.Hkv, off = p.Sk - p.Sq;
  const int items = p.list[0] * p.Hkv;
  const int4* entry = reinterpret_cast<const int4*>(p.list + 4);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t kv_phase = 0;
    int n = 0;                                      // query tiles loaded so far
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int4 e = entry[item / p.Hkv];
      const int kv_head = item % p.Hkv, batch = e.x / p.key_blocks, k0 = (e.x % p.key_blocks) * kWinBlock;
      const WindowKeys wk = window_keys(p.rule, batch, p.Sq, p.Sk, k0);
      const int qb = wk.q_lo / kWinBlock, n_q = (wk.q_hi + kWinBlock - 1) / kWinBlock - qb;
      if (lane == 0 && e.z > e.y) {
        ok = mbar_wait(kv_empty, (kv_phase & 1) ^ 1, abort_flag);
        ++kv_phase;
        if (ok) {
          mbar_arrive_expect_tx(kv_full, 2 * TILE_BYTES);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a) {
            tma_load_4d(sK + a * ATOM_BYTES, &tmK, kv_full, a * 64, kv_head, k0, batch);
            tma_load_4d(sV + a * ATOM_BYTES, &tmV, kv_full, a * 64, kv_head, k0, batch);
          }
        }
        for (int it = e.y; ok && it < e.z; ++it, ++n) {
          const int qs = n % Q_STAGES, st = n % STAGES, head = kv_head * group + it / n_q, q0 = (qb + it % n_q) * kWinBlock;
          const uint32_t parity = ((n / STAGES) & 1) ^ 1;
          ok = mbar_wait(&q_empty[qs], ((n / Q_STAGES) & 1) ^ 1, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&q_full[qs], TILE_BYTES);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a) tma_load_4d(sQ + qs * TILE_BYTES + a * ATOM_BYTES, &tmQ, &q_full[qs], a * 64, head, q0, batch);
          ok = mbar_wait(&do_empty[st], parity, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&do_full[st], TILE_BYTES);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a) tma_load_4d(sDO + st * TILE_BYTES + a * ATOM_BYTES, &tmDO, &do_full[st], a * 64, head, q0, batch);
          ok = mbar_wait(&aux_empty[st], parity, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&aux_full[st], AUX_BYTES);
          const long long row = (static_cast<long long>(batch) * p.Hq + head) * p.Sq_pad + q0;
          bulk_load(sAux + st * AUX_BYTES, p.lse2 + row, kWinBlock * 4, &aux_full[st]);
          bulk_load(sAux + st * AUX_BYTES + kWinBlock * 4, p.delta + row, kWinBlock * 4, &aux_full[st]);
        }
      }
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      if (!ok) break;
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ UMMA issuers: warp 1 dV and S, warp 2 dK and dP
    if (warp < 3 && lane == 0) {
      const uint32_t idesc_s = make_idesc_bf16(kWinBlock, kWinBlock, 0, 0);   // [128 keys, 128 queries]
      const uint32_t idesc_acc = make_idesc_bf16(kWinBlock, D, 0, 1);         // [128 keys, D] = A(TMEM) x B(MN-major)
      constexpr uint32_t hi = smem_desc_hi_sw128(1024);
      const uint32_t k_lo = smem_desc_lo(smem_u32(sK), 16), v_lo = smem_desc_lo(smem_u32(sV), 16);
      auto scores = [&](uint32_t d_tmem, uint32_t a_lo, const uint8_t* b_tile) {
        const uint32_t b_lo = smem_desc_lo(smem_u32(b_tile), 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t o = static_cast<uint32_t>(((kk >> 2) * ATOM_BYTES + (kk & 3) * 32) >> 4);
          umma_bf16_ss_lh(d_tmem, a_lo + o, hi, b_lo + o, hi, idesc_s, kk != 0 ? 1u : 0u);
        }
      };
      auto accumulate = [&](uint32_t d_tmem, uint32_t a_tmem, const uint8_t* b_tile, bool begin) {
        const uint32_t b_lo = smem_desc_lo(smem_u32(b_tile), ATOM_BYTES);
#pragma unroll
        for (int kk = 0; kk < kWinBlock / 16; ++kk)   // the 32 queries of a warp group sit packed in the first 16 of their 32 columns
          umma_bf16_ts_lh(d_tmem, a_tmem + static_cast<uint32_t>((kk >> 1) * 32 + (kk & 1) * 8), b_lo + static_cast<uint32_t>(kk * 128), hi,
                          idesc_acc, kk != 0 ? 1u : begin ? 0u : 1u);
      };
      auto wait_q = [&](int n) { return mbar_wait(&q_full[n % Q_STAGES], (n / Q_STAGES) & 1, abort_flag); };
      auto wait_do = [&](int n) { return mbar_wait(&do_full[n % STAGES], (n / STAGES) & 1, abort_flag); };
      auto q_tile = [&](int n) { return sQ + (n % Q_STAGES) * TILE_BYTES; };
      auto do_tile = [&](int n) { return sDO + (n % STAGES) * TILE_BYTES; };
      uint32_t kv_phase = 0, turn[2] = {0, 0};      // turn: of s_issued, which the last iteration of an item does not use
      int n = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const int4 e = entry[item / p.Hkv];
        const int len = e.z - e.y;
        if (len <= 0) continue;
        ok = mbar_wait(kv_full, kv_phase & 1, abort_flag) && (warp == 1 ? wait_q(n) : wait_do(n));
        ++kv_phase;
        if (!ok) break;
        tc_fence_after();
        if (warp == 1) {
          scores(tmem_base + S_COL, k_lo, q_tile(n));
          umma_commit(s_full);
          if (len == 1) umma_commit(kv_empty);
          for (int i = 0; i < len; ++i, ++n) {
            const bool more = i + 1 < len;
            ok = (!more || wait_q(n + 1)) && wait_do(n) && mbar_wait(p_full, n & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            accumulate(tmem_base + DV_COL, tmem_base + S_COL, do_tile(n), i == 0);
            if (more) {
              scores(tmem_base + S_COL, k_lo, q_tile(n + 1));
              mbar_arrive(&s_issued[n & 1]);
              umma_commit(s_full);
              if (i + 2 == len) umma_commit(kv_empty);   // K is not read again: the next item's may come
            }
            umma_commit(&do_empty[n % STAGES]);
          }
        } else {
          scores(tmem_base + DP_COL, v_lo, do_tile(n));
          umma_commit(dp_full);
          umma_commit(&do_empty[n % STAGES]);
          if (len == 1) umma_commit(kv_empty);
          for (int i = 0; i < len; ++i, ++n) {
            const bool more = i + 1 < len;
            ok = wait_q(n) && (!more || (wait_do(n + 1) && mbar_wait(&s_issued[n & 1], turn[n & 1]++ & 1, abort_flag))) &&
                 mbar_wait(ds_full, n & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            accumulate(tmem_base + DK_COL, tmem_base + DP_COL, q_tile(n), i == 0);
            if (more) {
              scores(tmem_base + DP_COL, v_lo, do_tile(n + 1));
              umma_commit(dp_full);
              umma_commit(&do_empty[(n + 1) % STAGES]);
              if (i + 2 == len) umma_commit(kv_empty);
            }
            umma_commit(&q_empty[n % Q_STAGES]);
          }
        }
        if (ok) umma_commit(acc_full);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ arithmetic: lane = key, 32 query columns per thread
    const int qw = warp & 3;                        // TMEM lane quarter this warp may touch
    const int grp = (warp - 4) >> 2;                // which 32 of the 128 queries
    const int row = qw * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(qw * 32) << 16;
    const uint32_t t_s = tmem_base + S_COL + static_cast<uint32_t>(grp * 32) + t_lane;
    const uint32_t t_dp = tmem_base + DP_COL + static_cast<uint32_t>(grp * 32) + t_lane;
    const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2), minus = f32x2(-1.f, -1.f);
    uint32_t acc_phase = 0;
    int n = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int4 e = entry[item / p.Hkv];
      const int kv_head = item % p.Hkv, batch = e.x / p.key_blocks, k0 = (e.x % p.key_blocks) * kWinBlock;
      const WindowKeys wk = window_keys(p.rule, batch, p.Sq, p.Sk, k0);
      const int qb = wk.q_lo / kWinBlock, n_q = (wk.q_hi + kWinBlock - 1) / kWinBlock - qb;
      const int kj = k0 + row;
      int upper = 0;                                // queries at positions [kj, upper) see this key
      if (kj < p.Sk) {
        const long long at = static_cast<long long>(batch) * p.Sk + kj;
        const int start = p.rule.starts ? p.rule.starts[at] : 0;
        if (start != kWinNone) upper = window_upper(p.rule, start, p.rule.starts ? p.rule.ends[at] : p.Sk, kj);
      }
      for (int it = e.y; it < e.z; ++it, ++n) {
        const int st = n % STAGES;
        const float* aux = reinterpret_cast<const float*>(sAux + st * AUX_BYTES) + grp * 32;
        const int pos0 = (qb + it % n_q) * kWinBlock + off;     // position of the tile's first query
        ok = mbar_wait(&aux_full[st], (n / STAGES) & 1, abort_flag) && mbar_wait(s_full, n & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t t[32], wt[16];                     // scores (later dP); P in bf16, two a register
        tmem_ld_32x32b_x32(t_s, t);
        uint32_t seen = 0xffffffffu;
        if (pos0 < k0 + kWinBlock - 1 || pos0 + kWinBlock > wk.full_hi) seen = interval_bits(pos0 + grp * 32, kj, upper);
        tmem_ld_wait();
        const bool some = __any_sync(0xffffffffu, seen != 0u);
        if (some) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 v = reinterpret_cast<const float4*>(aux)[i];
            wt[2 * i] = wb_exp2_pair(fma_f32x2(f32x2(__uint_as_float(t[4 * i]), __uint_as_float(t[4 * i + 1])), scale2, f32x2(-v.x, -v.y)), 2 * i);
            wt[2 * i + 1] = wb_exp2_pair(fma_f32x2(f32x2(__uint_as_float(t[4 * i + 2]), __uint_as_float(t[4 * i + 3])), scale2, f32x2(-v.z, -v.w)), 2 * i + 1);
          }
          if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (!((seen >> (2 * i)) & 1u)) wt[i] &= 0xffff0000u;
              if (!((seen >> (2 * i + 1)) & 1u)) wt[i] &= 0x0000ffffu;
            }
          }
        } else {                                    // far queries of a block with a few first tokens: most keys are not theirs
#pragma unroll
          for (int i = 0; i < 16; ++i) wt[i] = 0u;
        }
        tmem_st_32x32b_x16(t_s, wt);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
        // ---------------------------------------------------------------- dS
        ok = mbar_wait(dp_full, n & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (some) {
          tmem_ld_32x32b_x32(t_dp, t);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 v = reinterpret_cast<const float4*>(aux + kWinBlock)[i];
            float a, b, c, d;
            f32x2_split(mul_f32x2(bf16x2_as_f32x2(wt[2 * i]), fma_f32x2(f32x2(v.x, v.y), minus, f32x2(__uint_as_float(t[4 * i]), __uint_as_float(t[4 * i + 1])))), a, b);
            f32x2_split(mul_f32x2(bf16x2_as_f32x2(wt[2 * i + 1]), fma_f32x2(f32x2(v.z, v.w), minus, f32x2(__uint_as_float(t[4 * i + 2]), __uint_as_float(t[4 * i + 3])))), c, d);
            wt[2 * i] = pack_bf16x2(a, b), wt[2 * i + 1] = pack_bf16x2(c, d);
          }
        }
        tmem_st_32x32b_x16(t_dp, wt);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&aux_empty[st]);
          mbar_arrive(ds_full);
        }
      }
      if (!ok) break;
      // ---------------------------------------------------------------- this piece's dK, dV rows
      const bool any = e.z > e.y;
      if (any) {
        ok = mbar_wait(acc_full, acc_phase & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++acc_phase;
        tc_fence_after();
      }
      constexpr int QUART_D = D / 4;                // columns of the head dimension per thread
      const long long to = ((static_cast<long long>(batch) * p.Sk + kj) * p.Hkv + kv_head) * D + grp * QUART_D;
      float* part = e.w < 0 ? nullptr : p.parts + ((static_cast<long long>(e.w) * p.Hkv + kv_head) * 2 * kWinBlock + row) * D + grp * QUART_D;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t col = (which ? DV_COL : DK_COL) + static_cast<uint32_t>(grp * QUART_D);
        const float mul = which ? 1.f : p.scale;
        __nv_bfloat16* dst = which ? p.dv : p.dk;
#pragma unroll
        for (int c = 0; c < QUART_D; c += 16) {
          uint32_t r[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = 0u;
          if (any) {
            tmem_ld_32x32b_x16(tmem_base + col + static_cast<uint32_t>(c) + t_lane, r);
            tmem_ld_wait();
          }
          if (part) {                               // rows past the end hold zeros there
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              uint32_t v[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(__uint_as_float(r[i + k]) * mul);
              store_32_bytes(part + which * kWinBlock * D + c + i, v);
            }
          } else if (kj < p.Sk) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = pack_bf16x2(__uint_as_float(r[2 * k]) * mul, __uint_as_float(r[2 * k + 1]) * mul);
            store_32_bytes(dst + to + c, v);
          }
        }
      }
      tc_fence_before();                            // before the next item's first products (via p_full)
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    __nanosleep(50000);
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_MBAR_TIMEOUT);
      p.status[1] = static_cast<int>(blockIdx.x);
      p.status[2] = 1011;
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Key blocks of several pieces: their sums, the work dealt out to all threads of the grid.
template <int D>
__device__ __forceinline__ void window_bwd_join(const WindowBwdArgs& p) {
  constexpr long long kQuads = 2 * kWinBlock * D / 4;      // of a block and head: dK, then dV
  const long long all = p.list[1] * static_cast<long long>(p.Hkv) * kQuads, step = static_cast<long long>(gridDim.x) * kWbThreads;
  for (long long i = blockIdx.x * static_cast<long long>(kWbThreads) + threadIdx.x; i < all; i += step) {
    const int e = static_cast<int>(i % kQuads), unit = static_cast<int>(i / kQuads), kv_head = unit % p.Hkv;
    const int4 cut = p.cuts[unit / p.Hkv];
    const int which = e / (kWinBlock * D / 4), row = e % (kWinBlock * D / 4) / (D / 4), c = e % (D / 4) * 4;
    const int batch = cut.x / p.key_blocks, key = cut.x % p.key_blocks * kWinBlock + row;
    if (key >= p.Sk) continue;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* part = p.parts + (static_cast<long long>(cut.y) * p.Hkv + kv_head) * 2 * kWinBlock * D + 4ll * e;
#pragma unroll 4
    for (int s = 0; s < cut.z; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(part + s * (static_cast<long long>(p.Hkv) * 2 * kWinBlock * D));
      a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    }
    uint2 v;
    v.x = pack_bf16x2(a.x, a.y), v.y = pack_bf16x2(a.z, a.w);
    *reinterpret_cast<uint2*>((which ? p.dv : p.dk) + ((static_cast<long long>(batch) * p.Sk + key) * p.Hkv + kv_head) * D + c) = v;
  }
}

// ---------------------------------------------------------------------------------------------- dQ
// The items' key blocks form one stream; element g has its scores in TMEM buffer g & 1. S, dP and dQ have an issuer each, which
// issues as soon as its buffers allow it, so that nobody's wait (50 to 250 cycles even when satisfied) delays another's product;
// the arithmetic warps work on element g while S and dP of g + 1 are formed. dQ(g-1) frees the buffer of S(g+1); dP has one
// buffer, free as soon as the arithmetic has it in registers. With one issuer for the three an element took 3450 cycles, with two
// 2470, of 1536 of UMMAs.
template <int D>
__global__ void __launch_bounds__(kWbThreads, 1)
window_bwd_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                     const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const WindowBwdArgs p) {
  constexpr int ATOMS = D / 64;
  constexpr int TILE_BYTES = kWinBlock * D * 2, ATOM_BYTES = kWinBlock * 128;
  constexpr uint32_t TMEM_COLS = 512, DP_COL = 256, DQ_COL = 384;
  constexpr int K_STAGES = 3, V_STAGES = 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];   // with head_dim 128 the tiles fill it: its start has to be aligned
  uint8_t* smem = smem_raw;
  uint8_t* sQ = smem;
  uint8_t* sDO = sQ + TILE_BYTES;
  uint8_t* sK = sDO + TILE_BYTES;                   // K_STAGES
  uint8_t* sV = sK + K_STAGES * TILE_BYTES;         // V_STAGES
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + V_STAGES * TILE_BYTES);
  uint64_t* q_full = bars;            // 1
  uint64_t* q_empty = bars + 1;       // 1 (two issuers: S, dP)
  uint64_t* k_full = bars + 2;        // K_STAGES
  uint64_t* k_empty = bars + 5;       // K_STAGES
  uint64_t* v_full = bars + 8;        // V_STAGES
  uint64_t* v_empty = bars + 10;      // V_STAGES
  uint64_t* s_full = bars + 12;       // 2
  uint64_t* dp_full = bars + 14;      // 1
  uint64_t* dp_free = bars + 15;      // 1
  uint64_t* ds_full = bars + 16;      // 2: the arithmetic may finish element g + 1 before the issuer asks for element g
  uint64_t* dq_full = bars + 18;      // 1
  uint64_t* s_empty = bars + 19;      // 2: dQ has read the buffer
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {   // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_BAD_INDEX);
      p.status[2] = 1013;
    }
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int i = 0; i < K_STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < V_STAGES; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, kWbArithWarps);
    mbar_init(&ds_full[0], kWbArithWarps);
    mbar_init(&ds_full[1], kWbArithWarps);
    mbar_init(dq_full, 1);
    mbar_init(&s_empty[0], 1);
    mbar_init(&s_empty[1], 1);
    abort_flag[0] = 0;
    abort_flag[1] = p.status[3];
    fence_barrier_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmDO);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int items = p.row_tiles * p.Hq * p.B, group = p.Hq / p.Hkv;
  // late rows (long lists) first, the heads of one row tile next to one another
  auto where = [&](int item, int& batch, int& head, int& q0) {
    head = item % p.Hq;
    const int rest = item / p.Hq;
    q0 = (p.row_tiles - 1 - rest % p.row_tiles) * kWinBlock;
    batch = rest / p.row_tiles;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t q_uses = 0;
    int g = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      int batch, head, q0;
      where(item, batch, head, q0);
      const WindowTile t = window_tile(p.rule, batch, p.Sq, p.Sk, q0);
      const int n = t.count(), kv_head = head / group;
      if (lane == 0 && n > 0) {
        if (item + static_cast<int>(gridDim.x) < items) {   // the next item's rows on their way to L2
          int nb, nh, nq;
          where(item + gridDim.x, nb, nh, nq);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a) {
            tma_prefetch_4d(&tmQ, a * 64, nh, nq, nb);
            tma_prefetch_4d(&tmDO, a * 64, nh, nq, nb);
          }
        }
        for (int j = 0; ok && j < n; ++j, ++g) {
          const int ks = g % K_STAGES, vs = g % V_STAGES, key0 = t.block(j) * kWinBlock;
          ok = mbar_wait(&k_empty[ks], ((g / K_STAGES) & 1) ^ 1, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[ks], TILE_BYTES);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a)
            tma_load_4d(sK + ks * TILE_BYTES + a * ATOM_BYTES, &tmK, &k_full[ks], a * 64, kv_head, key0, batch);
          ok = mbar_wait(&v_empty[vs], ((g / V_STAGES) & 1) ^ 1, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[vs], TILE_BYTES);
#pragma unroll
          for (int a = 0; a < ATOMS; ++a)
            tma_load_4d(sV + vs * TILE_BYTES + a * ATOM_BYTES, &tmV, &v_full[vs], a * 64, kv_head, key0, batch);
          if (j == 0) {
            ok = mbar_wait(q_empty, (q_uses & 1) ^ 1, abort_flag);
            if (!ok) break;
            ++q_uses;
            mbar_arrive_expect_tx(q_full, 2 * TILE_BYTES);
#pragma unroll
            for (int a = 0; a < ATOMS; ++a) {
              tma_load_4d(sQ + a * ATOM_BYTES, &tmQ, q_full, a * 64, head, q0, batch);
              tma_load_4d(sDO + a * ATOM_BYTES, &tmDO, q_full, a * 64, head, q0, batch);
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      if (!ok) break;
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ UMMA issuers: warp 1 S, warp 2 dP, warp 3 dQ
    const uint32_t idesc_s = make_idesc_bf16(kWinBlock, kWinBlock, 0, 0);   // [128 q, 128 keys]
    const uint32_t idesc_dq = make_idesc_bf16(kWinBlock, D, 0, 1);          // [128 q, D] = A(TMEM) x B(K tile, MN-major)
    constexpr uint32_t hi = smem_desc_hi_sw128(1024);
    const uint32_t q_lo = smem_desc_lo(smem_u32(sQ), 16), do_lo = smem_desc_lo(smem_u32(sDO), 16);
    auto scores = [&](uint32_t d_tmem, uint32_t a_lo, const uint8_t* b_tile) {
      const uint32_t b_lo = smem_desc_lo(smem_u32(b_tile), 16);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o = static_cast<uint32_t>(((kk >> 2) * ATOM_BYTES + (kk & 3) * 32) >> 4);
        umma_bf16_ss_lh(d_tmem, a_lo + o, hi, b_lo + o, hi, idesc_s, kk != 0 ? 1u : 0u);
      }
    };
    int g = 0;
    uint32_t q_phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      int batch, head, q0;
      where(item, batch, head, q0);
      const int n = window_tile(p.rule, batch, p.Sq, p.Sk, q0).count();
      if (lane == 0) {
        for (int j = 0; j < n; ++j, ++g) {
          const int ks = g % K_STAGES, vs = g % V_STAGES;
          const uint32_t k_phase = (g / K_STAGES) & 1;
          if (warp == 1) {
            ok = mbar_wait(&k_full[ks], k_phase, abort_flag) && (j > 0 || mbar_wait(q_full, q_phase & 1, abort_flag)) &&
                 mbar_wait(&s_empty[g & 1], ((g >> 1) & 1) ^ 1, abort_flag);
            if (!ok) break;
            if (j == 0) ++q_phase;
            tc_fence_after();
            scores(tmem_base + static_cast<uint32_t>(g & 1) * 128u, q_lo, sK + ks * TILE_BYTES);
            umma_commit(&s_full[g & 1]);
            if (j + 1 == n) umma_commit(q_empty);
          } else if (warp == 2) {
            ok = (j > 0 || mbar_wait(q_full, q_phase & 1, abort_flag)) && mbar_wait(&v_full[vs], (g / V_STAGES) & 1, abort_flag) &&
                 mbar_wait(dp_free, (g & 1) ^ 1, abort_flag);
            if (!ok) break;
            if (j == 0) ++q_phase;
            tc_fence_after();
            scores(tmem_base + DP_COL, do_lo, sV + vs * TILE_BYTES);
            umma_commit(dp_full);
            umma_commit(&v_empty[vs]);
            if (j + 1 == n) umma_commit(q_empty);
          } else {
            ok = mbar_wait(&k_full[ks], k_phase, abort_flag) && mbar_wait(&ds_full[g & 1], (g >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t k_lo = smem_desc_lo(smem_u32(sK + ks * TILE_BYTES), ATOM_BYTES);
            const uint32_t s_col = tmem_base + static_cast<uint32_t>(g & 1) * 128u;
#pragma unroll
            for (int kk = 0; kk < kWinBlock / 16; ++kk)   // the 32 keys of a warp group sit packed in the first 16 of their 32 columns
              umma_bf16_ts_lh(tmem_base + DQ_COL, s_col + static_cast<uint32_t>((kk >> 1) * 32 + (kk & 1) * 8), k_lo + static_cast<uint32_t>(kk * 128),
                              hi, idesc_dq, kk != 0 || j != 0 ? 1u : 0u);
            umma_commit(&s_empty[g & 1]);
            umma_commit(&k_empty[ks]);
            if (j + 1 == n) umma_commit(dq_full);
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      if (!ok) break;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ arithmetic: lane = query row, 32 key columns per thread
    const int qw = warp & 3;
    const int grp = (warp - 4) >> 2;                // which 32 of the 128 keys
    const int row = qw * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(qw * 32) << 16;
    const uint32_t t_dp = tmem_base + DP_COL + static_cast<uint32_t>(grp * 32) + t_lane;
    const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2);
    uint32_t dq_phase = 0;
    int g = 0;
    bool ok = true;
    // what an item's rows need from memory, fetched while the item before is finished
    int batch = 0, head = 0, q0 = 0;
    WindowTile t{};
    WindowRow w{};
    float my_lse = 0.f, my_delta = 0.f;
    auto fetch = [&](int item) {
      where(item, batch, head, q0);
      const long long stat = (static_cast<long long>(batch) * p.Hq + head) * p.Sq_pad + q0 + row;   // padded: always in range
      my_lse = p.lse2[stat], my_delta = p.delta[stat];
      t = window_tile(p.rule, batch, p.Sq, p.Sk, q0);
      w = window_row(p.rule, batch, p.Sk, q0 + row + p.Sk - p.Sq, q0 + row < p.Sq);
    };
    if (static_cast<int>(blockIdx.x) < items) fetch(blockIdx.x);
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int n = t.count(), qi = q0 + row;
      // Weights rounded on the forward's grid, so that the terms of dS cancel nearly as exactly as there: relative to a whole power of
      // two (the forward's differ from it by another such factor), rounded to bf16, times what is left of 2^-lse2. They are the
      // forward's but for a neighbouring bf16 value now and then, since a quarter comes from the polynomial.
      const float shift = floorf(my_lse);
      const float factor = my_lse != INFINITY ? wb_exp2(shift - my_lse) : 0.f;
      const uint64_t shift2 = f32x2(-shift, -shift), factor2 = f32x2(factor, factor), offset2 = f32x2(-my_delta * factor, -my_delta * factor);
      for (int j = 0; j < n; ++j, ++g) {
        ok = mbar_wait(&s_full[g & 1], (g >> 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = tmem_base + static_cast<uint32_t>((g & 1) * 128 + grp * 32) + t_lane;
        uint32_t sc[32];
        tmem_ld_32x32b_x32(t_s, sc);
        tmem_ld_wait();
        const int key0 = t.block(j) * kWinBlock;
        uint32_t wt[16];                            // rounded weights, two a register
#pragma unroll
        for (int i = 0; i < 16; ++i)
          wt[i] = wb_exp2_pair(fma_f32x2(f32x2(__uint_as_float(sc[2 * i]), __uint_as_float(sc[2 * i + 1])), scale2, shift2), i);
        if (key0 < t.full_lo || key0 + kWinBlock - 1 > t.full_hi) {
          const uint32_t seen = window_bits(w, key0 + grp * 32);
          if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (!((seen >> (2 * i)) & 1u)) wt[i] &= 0xffff0000u;
              if (!((seen >> (2 * i + 1)) & 1u)) wt[i] &= 0x0000ffffu;
            }
          }
        }
        ok = mbar_wait(dp_full, g & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t dp[32];
        tmem_ld_32x32b_x32(t_dp, dp);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dp_free);        // the next element's dP may be issued
        uint32_t ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a, b;
          const uint64_t d = fma_f32x2(f32x2(__uint_as_float(dp[2 * i]), __uint_as_float(dp[2 * i + 1])), factor2, offset2);
          f32x2_split(mul_f32x2(bf16x2_as_f32x2(wt[i]), d), a, b);
          ds[i] = pack_bf16x2(a, b);
        }
        tmem_st_32x32b_x16(t_s, ds);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[g & 1]);
      }
      if (!ok) break;
      constexpr int QUART_D = D / 4;
      __nv_bfloat16* dst = p.dq + ((static_cast<long long>(batch) * p.Sq + qi) * p.Hq + head) * D + grp * QUART_D;
      if (item + static_cast<int>(gridDim.x) < items) fetch(item + gridDim.x);
      if (n > 0) {
        ok = mbar_wait(dq_full, dq_phase & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++dq_phase;
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < QUART_D; c += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
        if (n > 0) {
          tmem_ld_32x32b_x16(tmem_base + DQ_COL + static_cast<uint32_t>(grp * QUART_D + c) + t_lane, r);
          tmem_ld_wait();
        }
        if (qi < p.Sq) {
          uint32_t v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = pack_bf16x2(__uint_as_float(r[2 * k]) * p.scale, __uint_as_float(r[2 * k + 1]) * p.scale);
          store_32_bytes(dst + c, v);
        }
      }
      tc_fence_before();                            // before the next item's first dQ (via ds_full)
    }
  }

  tc_fence_before();
  __syncthreads();
  window_bwd_join<D>(p);
  if (*abort_flag) {
    __nanosleep(50000);
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_MBAR_TIMEOUT);
      p.status[1] = static_cast<int>(blockIdx.x);
      p.status[2] = 1012;
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------- host
// How a key block's work is cut, and what that needs of scratch memory.
struct WindowBwdPlan {
  int sq_pad, key_blocks, row_tiles, piece;
  long long blocks, max_slots, rows;
  long long at_delta, at_list, at_cuts, at_parts, words;   // in 4-byte words
};

// Pieces that packed rows can need at most, beside those of blocks that the window alone makes too long. A block is cut for its
// first tokens only if the queries behind them fill more tiles than a piece takes, so their document is long, and a row has few
// such documents: with m tiles to exceed, T queries fill at most (T - 1) / 128 + 2 tiles, and up to 127 of them come from before the
// document. Each of its blocks (of first tokens) takes at most its iterations over the piece, and one more.
// (4 rows of 8192 tokens, 32 heads of 128, window 512, 4 first tokens: 112 pieces of up to 11 iterations, 448 MiB beside 512 MiB of
// gradients. A bound by iterations alone, without the documents' lengths, asked for 2.2 GiB.)
static long long window_bwd_packed_slots(long long B, long long Sq, long long sinks, long long group, long long near, long long piece) {
  const long long row_tiles = (Sq + kWinBlock - 1) / kWinBlock, m = (piece > near ? piece : near) / group + 1;
  const long long shortest = (m - 2) * kWinBlock - 126, documents = shortest < 1 ? Sq : Sq / shortest;
  const long long blocks = (sinks + kWinBlock - 2) / kWinBlock + 1;
  return B * blocks * ((row_tiles + 3 * documents) * group / piece + documents);
}

static WindowBwdPlan window_bwd_plan(int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, bool packed) {
  WindowBwdPlan w{};
  const long long group = Hq / Hkv;
  w.row_tiles = (Sq + kWinBlock - 1) / kWinBlock;
  w.key_blocks = (Sk + kWinBlock - 1) / kWinBlock;
  w.sq_pad = w.row_tiles * kWinBlock;
  w.blocks = static_cast<long long>(B) * w.key_blocks;
  // iterations of a block whose keys are seen through the window only, and of one that every query of its row sees
  const long long tiles = (static_cast<long long>(window < Sk ? window : Sk) + kWinBlock - 1) / kWinBlock + 2;
  const long long near = (tiles < w.row_tiles ? tiles : w.row_tiles) * group, all = w.row_tiles * group;
  const long long items = w.blocks * Hkv;
  // Pieces a quarter longer than an ordinary block's work: only blocks with first tokens are cut. With fewer blocks than SMs
  // ordinary blocks are cut too, into as many pieces as there are SMs for.
  long long piece = sinks > 0 ? near + near / 4 + 1 : near;
  if (items < sm_count()) {
    const long long share = sm_count() / items;
    piece = (near + share - 1) / share;
    if (piece < 2) piece = 2;
  }
  // Pieces of blocks that hold first tokens. Their parts may take as much as dK and dV themselves (half a slot a block), or two pieces
  // an SM if that is more; where they would take more, pieces get longer, which costs nothing when every SM has several.
  const long long sink_blocks = (sinks + kWinBlock - 1) / kWinBlock;
  const long long limit = w.blocks / 2 > 2 * sm_count() / Hkv ? w.blocks / 2 : 2 * sm_count() / Hkv;
  long long sink_slots = 0;
  while (sinks > 0 && all > piece) {
    sink_slots = packed ? window_bwd_packed_slots(B, Sq, sinks, group, near, piece)
                        : B * (sink_blocks < w.key_blocks ? sink_blocks : w.key_blocks) * ((all + piece - 1) / piece);
    if (sink_slots <= limit) break;
    sink_slots = 0;
    piece += piece / 4 + 1;
  }
  const long long ordinary = (near + piece - 1) / piece;
  const long long slots = sink_slots + (ordinary > 1 ? w.blocks * ordinary : 0);
  w.piece = static_cast<int>(piece < (1 << 30) ? piece : (1 << 30));
  w.max_slots = slots;
  w.rows = static_cast<long long>(B) * Hq * w.sq_pad;
  w.at_delta = w.rows;
  w.at_list = 2 * w.rows;
  w.at_cuts = w.at_list + 4 + 4 * (w.blocks + slots);       // int4 entries: at_list is a multiple of 128 words
  w.at_parts = (w.at_cuts + 4 * w.blocks + 7) / 8 * 8;     // stored 32 bytes at a time
  w.words = w.at_parts + slots * Hkv * 2 * kWinBlock * D;
  return w;
}

struct WindowBwdMaps {
  CUtensorMap q, dout, k, v;
};

template <int D>
static int launch_window_bwd(const WindowBwdMaps& m, const WindowBwdPrepArgs& prep, const WindowBwdArgs& a, const WindowBwdPlan& plan,
                             cudaStream_t stream) {
  constexpr size_t tile = kWinBlock * D * 2;
  constexpr size_t smem_dkdv = 7 * tile + 2 * (2 * kWinBlock * 4) + 256, smem_dq = 7 * tile + 256;
  static bool configured[64] = {false};
  int dev = 0;
  MB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    MB_CHECK_CUDA(cudaFuncSetAttribute(window_bwd_dkdv_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_dkdv)));
    MB_CHECK_CUDA(cudaFuncSetAttribute(window_bwd_dq_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_dq)));
    configured[dev & 63] = true;
  }
  const long long prep_blocks = 1 + (plan.rows * (D / 8) + kWbPrepThreads - 1) / kWbPrepThreads;
  window_bwd_prep_kernel<D><<<static_cast<unsigned>(prep_blocks), kWbPrepThreads, 0, stream>>>(prep);
  const long long most = (plan.blocks + plan.max_slots) * a.Hkv;
  const int grid_kv = static_cast<int>(most < sm_count() ? most : sm_count());
  window_bwd_dkdv_kernel<D><<<grid_kv, kWbThreads, smem_dkdv, stream>>>(m.q, m.dout, m.k, m.v, a);
  count_launch(2);
  const long long tiles = static_cast<long long>(plan.row_tiles) * a.Hq * a.B;
  window_bwd_dq_kernel<D><<<static_cast<int>(tiles < sm_count() ? tiles : sm_count()), kWbThreads, smem_dq, stream>>>(m.q, m.dout, m.k, m.v, a);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace mb

// 4-byte words of scratch memory mb_window_attn_bwd needs; `packed`: it is given documents.
MB_API long long mb_window_attn_bwd_scratch_words(int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, int packed) {
  if (B < 1 || Sq < 1 || Sk < 1 || Hkv < 1 || Hq % Hkv != 0) return 0;
  return mb::window_bwd_plan(B, Sq, Sk, Hq, Hkv, D, window, sinks, packed != 0).words;
}

// Backward of mb_window_attn_fwd. q, k, v, out, out_lo, lse2 as there, dout with strides of its own, dq / dk / dv bf16 contiguous.
// starts, ends: mb_document_bounds of the key rows, or both null. scratch: mb_window_attn_bwd_scratch_words() words.
MB_API int mb_window_attn_bwd(const void* q, long long q_tstride, long long q_bstride, const void* k, long long k_tstride,
                              long long k_bstride, const void* v, long long v_tstride, long long v_bstride, const void* out,
                              const void* out_lo, const void* dout, long long do_tstride, long long do_bstride, const float* lse2, void* dq,
                              void* dk, void* dv, const int* starts, const int* ends, int* scratch, int B, int Sq, int Sk, int Hq, int Hkv,
                              int D, int window, int sinks, float scale, cudaStream_t stream) {
  using namespace mb;
  const long long strides[] = {q_tstride, q_bstride, k_tstride, k_bstride, v_tstride, v_bstride, do_tstride, do_bstride};
  const void* pointers[] = {q, k, v, out, out_lo, dout, dq, dk, dv, scratch};
  if (const char* what = window_attn_problem(B, Sq, Sk, Hq, Hkv, D, window, sinks, strides, 8, pointers, 10)) {
    set_last_error(what);
    return -1;
  }
  if ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
       reinterpret_cast<uintptr_t>(scratch)) & 31) {
    set_last_error("mb_window_attn_bwd: gradients and scratch must be 32-byte aligned");
    return -3;
  }
  if ((starts == nullptr) != (ends == nullptr)) {
    set_last_error("mb_window_attn_bwd: starts and ends come together");
    return -2;
  }
  int* status = status_ptr();
  if (!status) return -4;
  const WindowBwdPlan plan = window_bwd_plan(B, Sq, Sk, Hq, Hkv, D, window, sinks, starts != nullptr);
  if (plan.blocks * Hkv >= (1ll << 31) - 65536 || static_cast<long long>(plan.row_tiles) * Hq * B >= (1ll << 31) - 65536 ||
      plan.rows * (D / 8) / kWbPrepThreads >= (1ll << 31) - 65536 || (plan.blocks + plan.max_slots) * Hkv >= (1ll << 31) - 65536) {
    set_last_error("mb_window_attn_bwd: too many tiles");
    return -1;
  }
  const WindowRule rule = {starts, ends, window < Sk ? window : Sk, sinks < Sk ? sinks : Sk};
  float* lse2_pad = reinterpret_cast<float*>(scratch);
  float* delta = lse2_pad + plan.at_delta;
  int* list = scratch + plan.at_list;
  int4* cuts = reinterpret_cast<int4*>(scratch + plan.at_cuts);
  WindowBwdPrepArgs prep;
  prep.out = static_cast<const __nv_bfloat16*>(out), prep.out_lo = static_cast<const __nv_bfloat16*>(out_lo);
  prep.dout = static_cast<const __nv_bfloat16*>(dout);
  prep.do_tstride = do_tstride, prep.do_bstride = do_bstride;
  prep.lse2_in = lse2, prep.lse2 = lse2_pad, prep.delta = delta, prep.list = list, prep.cuts = cuts, prep.rule = rule;
  prep.B = B, prep.Sq = Sq, prep.Sk = Sk, prep.Hq = Hq, prep.Hkv = Hkv, prep.Sq_pad = plan.sq_pad, prep.key_blocks = plan.key_blocks;
  prep.piece = plan.piece, prep.max_slots = static_cast<int>(plan.max_slots);
  WindowBwdArgs a;
  a.dq = static_cast<__nv_bfloat16*>(dq), a.dk = static_cast<__nv_bfloat16*>(dk), a.dv = static_cast<__nv_bfloat16*>(dv);
  a.lse2 = lse2_pad, a.delta = delta, a.list = list, a.cuts = cuts, a.parts = reinterpret_cast<float*>(scratch + plan.at_parts);
  a.rule = rule;
  a.B = B, a.Sq = Sq, a.Sk = Sk, a.Hq = Hq, a.Hkv = Hkv, a.Sq_pad = plan.sq_pad;
  a.key_blocks = plan.key_blocks, a.row_tiles = plan.row_tiles;
  a.scale = scale, a.scale_log2 = scale * kWbLog2e;
  a.status = status;
  WindowBwdMaps m;
  const uint32_t box[4] = {64, 1, static_cast<uint32_t>(kWinBlock), 1};
  auto encode = [&](CUtensorMap* t, const void* x, int heads, int S, long long tstride, long long bstride) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)S, (uint64_t)B};
    const uint64_t bytes[3] = {(uint64_t)D * 2, (uint64_t)tstride * 2, (uint64_t)bstride * 2};
    return encode_tmap_4d(t, x, dims, bytes, box, 2, true);
  };
  if (!encode(&m.q, q, Hq, Sq, q_tstride, q_bstride) || !encode(&m.dout, dout, Hq, Sq, do_tstride, do_bstride) ||
      !encode(&m.k, k, Hkv, Sk, k_tstride, k_bstride) || !encode(&m.v, v, Hkv, Sk, v_tstride, v_bstride))
    return -5;
  return D == 128 ? launch_window_bwd<128>(m, prep, a, plan, stream) : launch_window_bwd<64>(m, prep, a, plan, stream);
}
