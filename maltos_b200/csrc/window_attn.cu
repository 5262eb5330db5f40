// Sliding-window attention, forward, for sm_100a (visibility rule: window.cuh). Persistent CTAs; an item of work is one or two
// tiles of 128 query rows that walk the same list of key blocks, so a K / V block fetched once serves both tiles and the
// softmax of one tile runs under the matrix products of the other:
//   warp 0       TMA producer: the tiles' queries and a ring of K and V blocks,
//   warps 1, 2   one per tile: issue S = Q K^T and O += P V as UMMAs; S, P and O stay in tensor memory (P overwrites the scores it
//                came from),
//   warps 3-18   eight per tile, two threads per query row with 32 keys each: running maximum and sum, P in bf16, output.
// A block's keys are worked on in two halves of 64 with buffers of their own, so that a tile hides its products itself: while the
// arithmetic is at one half, O += P V of the other and the other's next scores are formed. (With whole blocks a tile alternates
// between 2600 cycles of arithmetic and 1800 of products and their waits, and the two tiles hide only part of that from one
// another: 4400 cycles for the pair, of 2048 of UMMAs.) Halves of which no row sees a key are left out.
// Measured (launches recorded into a graph, L2 flushed between them, median; TFLOP/s of the visible pairs): 8192 rows, 32 / 8 heads of
// 128, window 1024 191 to 197 us / 679 to 658 (two boxes); 16384 rows, 8 / 2 heads, window 4096 297 us / 813; the whole causal triangle
// of 8192 rows 610 us / 901; 32 / 8 heads of 64 176 us / 367, since a product of half the work leaves the same arithmetic. What takes
// the time is the tile's arithmetic between two products, its instructions more than the exponentials (a quarter of them by
// polynomial on the multiply-add pipe costs 7 per cent here, where the backward gains): a state of this code, not a limit of the GPU.
// The two tiles are two query heads of one key/value head on the same rows where the group is even, else neighbouring rows of
// one head. O is rescaled only when a row's maximum has grown by more than 2^8 since the last rescale: P then stays below 2^8
// and its bf16 rounding is relative, so nothing is lost, and after the first blocks the rescale hardly ever happens.
//
// Roundings. P is bf16 because the operands of a UMMA have one type, and V is bf16: a weight is off by up to half a step, at random
// over the keys, which adds to the output less than its own rounding (relative error against 64 bits 0.0022 where fp32 weights give
// 0.0017). P is relative to a whole power of two and O is divided by the sum of the ROUNDED P, so that the dQ kernel can round its
// weights on the same grid (they differ by a step now and then: part of its exponentials come from a polynomial) and the terms of dS
// cancel nearly as in the exact softmax. For the same reason the forward of a training step keeps what the rounding of O left
// (out_lo): where nearly all weight is on one key, as trained models' is on the first, dS is a small difference, and with delta
// from the rounded output alone dQ of such rows was 8 to 23 times as far off. dK and dV round the normalised weights on a grid of their
// own: a key's sum over queries has no such cancellation.
#include "host.h"
#include "ptx.cuh"
#include "window.cuh"

namespace mb {

constexpr int kWfSoftmaxWarps = 16;
constexpr int kWfThreads = 32 * (3 + kWfSoftmaxWarps);
constexpr int kWfStages = 5;                       // K and V blocks in flight
constexpr float kWfLog2e = 1.4426950408889634f, kWfLn2 = 0.6931471805599453f;
constexpr float kWfGrowth = 8.f;                   // log2 of how far P may exceed 1 before O is rescaled

struct WindowFwdArgs {
  __nv_bfloat16* out;       // [B, Sq, Hq, D]
  __nv_bfloat16* out_lo;    // the same shape: O - out, for the backward; or null
  float* lse2;              // [B, Hq, Sq] log2 of the sum of the rounded weights, for the backward; or null
  float* lse;               // [B, Hq, Sq] log-sum-exp of the scores; or null (then its sum is not formed)
  WindowRule rule;
  int B, Sq, Sk, Hq, Hkv;
  int pair;                 // tiles of an item: 0 one tile, 1 two heads of a group, 2 two neighbouring row tiles
  int row_units, head_units, items;
  float scale_log2;
  int* status;
};

__device__ __forceinline__ float wf_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct WindowItem {
  int batch, kv_head;
  int head[2], q0[2];
  WindowTile tile[2];
  int a0, na, w0, n;        // union list: blocks a0 .. a0 + na, then w0 ..; n in all
  __device__ __forceinline__ int block(int u) const { return u < na ? a0 + u : w0 + u - na; }
};

// Where the tiles of an item lie; late rows (long lists) first. `with_tiles`: also what they visit (warp-collective).
__device__ __forceinline__ void window_item(const WindowFwdArgs& p, int item, WindowItem& it) {
  const int hu = item % p.head_units;
  const int rest = item / p.head_units;
  const int ru = p.row_units - 1 - rest % p.row_units;
  it.batch = rest / p.row_units;
  const int head = p.pair == 1 ? 2 * hu : hu;
  it.kv_head = head / (p.Hq / p.Hkv);
  it.head[0] = head, it.head[1] = p.pair == 1 ? head + 1 : head;
  it.q0[0] = ru * (p.pair == 2 ? 2 : 1) * kWinBlock;
  it.q0[1] = p.pair == 0 ? p.Sq : p.pair == 1 ? it.q0[0] : it.q0[0] + kWinBlock;   // a tile from row Sq on is empty
}

__device__ __forceinline__ void window_item_blocks(const WindowFwdArgs& p, WindowItem& it) {
  it.tile[0] = window_tile(p.rule, it.batch, p.Sq, p.Sk, it.q0[0]);
  it.tile[1] = p.pair == 1 ? it.tile[0] : window_tile(p.rule, it.batch, p.Sq, p.Sk, it.q0[1]);
  const WindowTile &x = it.tile[0], &y = it.tile[1];
  it.a0 = it.na = it.w0 = it.n = 0;
  const bool hx = x.b1 > x.b0, hy = y.b1 > y.b0;
  if (!hx && !hy) return;
  it.w0 = !hx ? y.b0 : !hy ? x.b0 : min(x.b0, y.b0);
  const int w1 = max(x.b1, y.b1);
  // first tokens before the union's window; a tile whose document starts later has its own inside it
  int lo = kWinNone, hi = 0;
  if (x.ea > x.sa) lo = x.sa, hi = x.ea;
  if (y.ea > y.sa) lo = min(lo, y.sa), hi = max(hi, y.ea);
  hi = min(hi, it.w0);
  if (lo < hi) it.a0 = lo, it.na = hi - lo;
  it.n = it.na + w1 - it.w0;
}

template <int D, bool LSE>
__global__ void __launch_bounds__(kWfThreads, 1)
window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const WindowFwdArgs p) {
  constexpr int ATOMS = D / 64;                    // 64-wide swizzle atoms along head_dim
  constexpr int TILE_BYTES = kWinBlock * D * 2;
  constexpr int ATOM_BYTES = kWinBlock * 128;
  constexpr uint32_t TMEM_COLS = 512, O_COL = 0, S_COL = 256;   // O of tile t at t * 128, its scores at 256 + t * 128

  extern __shared__ __align__(1024) uint8_t smem_raw[];   // with head_dim 128 the tiles fill it: its start has to be aligned
  uint8_t* smem = smem_raw;
  uint8_t* sQ = smem;                              // 2 tiles
  uint8_t* sKV = sQ + 2 * TILE_BYTES;              // kWfStages blocks
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kWfStages * TILE_BYTES);
  uint64_t* q_full = bars;                         // 2
  uint64_t* q_empty = bars + 2;                    // 2
  uint64_t* s_full = bars + 4;                     // 2 tiles x 2 halves
  uint64_t* p_full = bars + 8;                     // 2 x 2
  uint64_t* o_done = bars + 12;                    // 2 x 2: the tile's product k (odd, even) is in O; two may be on their way
  uint64_t* kv_full = bars + 16;                   // kWfStages
  uint64_t* kv_empty = kv_full + kWfStages;        // kWfStages
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kWfStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* exchange = reinterpret_cast<float*>(smem + (2 + kWfStages) * TILE_BYTES + 256);   // [tile][half][row]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {   // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_BAD_INDEX);
      p.status[2] = 1015;
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s_full[2 * t + h], 1);
        mbar_init(&p_full[2 * t + h], 8);
        mbar_init(&o_done[2 * t + h], 1);
      }
    }
    for (int i = 0; i < kWfStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);
    }
    abort_flag[0] = 0;
    abort_flag[1] = p.status[3];
    fence_barrier_init();
    prefetch_tmap(&tmQ);
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

  if (warp < 3) {
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer
      int slot = 0, round = 0;                     // ring position and how often it has gone round
      int q_uses[2] = {0, 0};
      bool ok = true;
      for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
        WindowItem it;
        window_item(p, item, it);
        window_item_blocks(p, it);
        if (lane == 0) {
          // The next item's queries and first blocks on their way to L2, so that its start does not wait for HBM.
          if (item + static_cast<int>(gridDim.x) < p.items) {
            WindowItem next;
            window_item(p, item + gridDim.x, next);
            for (int t = 0; t < 2; ++t)
              if (next.q0[t] < p.Sq)
#pragma unroll
                for (int a = 0; a < ATOMS; ++a) tma_prefetch_4d(&tmQ, a * 64, next.head[t], next.q0[t], next.batch);
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || it.tile[t].count() == 0) continue;
            ok = mbar_wait(&q_empty[t], (q_uses[t] & 1) ^ 1, abort_flag);
            if (!ok) continue;
            ++q_uses[t];
            mbar_arrive_expect_tx(&q_full[t], TILE_BYTES);
#pragma unroll
            for (int a = 0; a < ATOMS; ++a)
              tma_load_4d(sQ + t * TILE_BYTES + a * ATOM_BYTES, &tmQ, &q_full[t], a * 64, it.head[t], it.q0[t], it.batch);
          }
          for (int u = 0; ok && u < it.n; ++u) {
            const int key0 = it.block(u) * kWinBlock;
            for (int kv = 0; kv < 2; ++kv) {
              ok = mbar_wait(&kv_empty[slot], (round & 1) ^ 1, abort_flag);
              if (!ok) break;
              mbar_arrive_expect_tx(&kv_full[slot], TILE_BYTES);
#pragma unroll
              for (int a = 0; a < ATOMS; ++a)
                tma_load_4d(sKV + slot * TILE_BYTES + a * ATOM_BYTES, kv ? &tmV : &tmK, &kv_full[slot], a * 64, it.kv_head, key0, it.batch);
              if (++slot == kWfStages) slot = 0, ++round;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
        if (!ok) break;
      }
    } else {
      // ---------------------------------------------------------------- UMMA issuer of tile t
      // Step (u, h): O += P V of what half h holds from block u - 1, then the scores of half h of block u in its place. The products
      // thus come in the order of the arithmetic, none later than one block after its scores.
      const int t = warp - 1;
      const uint32_t idesc_qk = make_idesc_bf16(kWinBlock, 64, 0, 0);
      const uint32_t idesc_pv = make_idesc_bf16(kWinBlock, D, 0, 1);
      constexpr uint32_t hi = smem_desc_hi_sw128(1024);
      const uint32_t s_tmem = tmem_base + S_COL + static_cast<uint32_t>(t) * 128u, o_tmem = tmem_base + O_COL + static_cast<uint32_t>(t) * 128u;
      const uint32_t q_lo = smem_desc_lo(smem_u32(sQ + t * TILE_BYTES), 16);
      int ring = 0, ring_round = 0;                // position of the block's K in the ring
      uint32_t p_phase[2] = {0, 0}, q_phase = 0, products = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
        WindowItem it;
        window_item(p, item, it);
        window_item_blocks(p, it);
        if (lane == 0) {
          const WindowTile tile = t ? it.tile[1] : it.tile[0];
          int left = tile.count();                 // blocks whose scores are not issued yet
          bool pending[2] = {false, false}, begun = false, has_o = false;
          int vs = 0, v_round = 0;                 // ring position of V of the block before
          for (int u = 0; u <= it.n; ++u) {
            const int ks = ring, blk = u < it.n ? it.block(u) : 0;
            const bool mine = u < it.n && tile.has(blk), used = pending[0] || pending[1];
            // what was loaded long ago is waited for first, the waits that matter (for P) come last
            ok = (u == 0 || mbar_wait(&kv_full[vs], v_round & 1, abort_flag)) && (u == it.n || mbar_wait(&kv_full[ks], ring_round & 1, abort_flag));
            if (!ok) break;
            if (mine && !begun) {
              ok = mbar_wait(&q_full[t], q_phase & 1, abort_flag);
              if (!ok) break;
              ++q_phase;
              begun = true;
            }
            const uint32_t v_lo = smem_desc_lo(smem_u32(sKV + vs * TILE_BYTES), ATOM_BYTES), k_lo = smem_desc_lo(smem_u32(sKV + ks * TILE_BYTES), 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (pending[h]) {
                ok = ok && mbar_wait(&p_full[2 * t + h], p_phase[h] & 1, abort_flag);
                if (!ok) continue;
                ++p_phase[h];
                tc_fence_after();
                const uint32_t acc0 = has_o ? 1u : 0u;
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2)     // the 32 keys of a thread sit packed in the first 16 of their 32 columns
                  umma_bf16_ts_lh(o_tmem, s_tmem + static_cast<uint32_t>(h * 64 + (k2 >> 1) * 32 + (k2 & 1) * 8),
                                  v_lo + static_cast<uint32_t>((h * 4 + k2) * 128), hi, idesc_pv, k2 != 0 ? 1u : acc0);
                umma_commit(&o_done[2 * t + (products++ & 1)]);
                has_o = true;
                pending[h] = false;
              }
              if (mine && tile.sees64(blk * kWinBlock + h * 64)) {
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint32_t off = static_cast<uint32_t>(((kk >> 2) * ATOM_BYTES + (kk & 3) * 32) >> 4);
                  umma_bf16_ss_lh(s_tmem + static_cast<uint32_t>(h * 64), q_lo + off, hi, k_lo + off + static_cast<uint32_t>(h * (64 * 128 >> 4)), hi,
                                  idesc_qk, kk != 0 ? 1u : 0u);
                }
                umma_commit(&s_full[2 * t + h]);
                pending[h] = true;
              }
            }
            if (!ok) break;
            if (mine) {
              umma_commit(&kv_empty[ks]);
              if (--left == 0) umma_commit(&q_empty[t]);
            } else if (u < it.n) {
              mbar_arrive(&kv_empty[ks]);          // the other tile's block
            }
            if (u > 0) {
              if (used) umma_commit(&kv_empty[vs]);
              else mbar_arrive(&kv_empty[vs]);
            }
            if (u < it.n) {
              if (++ring == kWfStages) ring = 0, ++ring_round;
              vs = ring, v_round = ring_round;
              if (++ring == kWfStages) ring = 0, ++ring_round;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
        if (!ok) break;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output: two threads per query row
    const int t = (warp - 3) >> 3, half = ((warp - 3) >> 2) & 1;   // half: which 32 of a buffer's 64 keys, which half of O's columns
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem_base + S_COL + static_cast<uint32_t>(t * 128 + half * 32) + t_lane;
    constexpr int HALF_D = D / 2;                  // columns of O that this thread rescales and stores
    const uint32_t o_tmem = tmem_base + O_COL + static_cast<uint32_t>(t * 128 + half * HALF_D) + t_lane;
    // The two threads of a row exchange a value through shared memory and barriers of their two warps; maxima only when one of the
    // 64 threads has to rescale, which one barrier tells them all. NaN says that a wait of
    // one of them ran out: both then leave at the same place, so that neither is left behind at the barrier (a maximum is never
    // NaN, and a sum that is NaN stops nothing but the output loop of its own rows, for which `stop` is not looked at).
    float* slot = exchange + (t * 2 + half) * kWinBlock + row;
    const volatile float* partner = exchange + (t * 2 + (half ^ 1)) * kWinBlock + row;
    auto pair_barrier = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + (warp & 3)) : "memory"); };
    auto pair_any = [&](bool mine) {               // of the 64 threads
      int any;
      asm volatile(
          "{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.or.pred q, %2, 64, p;\nselp.s32 %0, 1, 0, q;\n}"
          : "=r"(any) : "r"(static_cast<int>(mine)), "r"(1 + t * 4 + (warp & 3)) : "memory");
      return any != 0;
    };
    auto swap = [&](float mine) {
      *slot = mine;
      pair_barrier();
      const float theirs = *partner;
      pair_barrier();                              // both have read: the slot may be written again
      return theirs;
    };
    uint32_t s_phase[2] = {0, 0}, products = 0;    // products: of this tile so far, its halves in all items
    auto product_done = [&] {                      // the last one
      const bool there = mbar_wait(&o_done[2 * t + ((products - 1) & 1)], ((products - 1) >> 1) & 1, abort_flag);
      return __all_sync(0xffffffffu, there) != 0;
    };
    bool ok = true, stop = false;
    for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
      WindowItem it;
      window_item(p, item, it);
      const int q0 = it.q0[t], head = it.head[t];
      if (q0 >= p.Sq) continue;                    // the missing second tile
      const WindowTile tile = window_tile(p.rule, it.batch, p.Sq, p.Sk, q0);
      const int n = tile.count();
      const int qi = q0 + row;
      const WindowRow w = window_row(p.rule, it.batch, p.Sk, qi + p.Sk - p.Sq, qi < p.Sq);
      // m_run: the power of two that P is relative to; l_run: this thread's sum of the rounded P; x_run: of P as it was before
      float m_run = -INFINITY, l_run = 0.f, x_run = 0.f;
      bool first = true;
      for (int j = 0; j < n; ++j) {
        const int blk0 = tile.block(j) * kWinBlock;
        const bool edge = blk0 < tile.full_lo || blk0 + kWinBlock - 1 > tile.full_hi;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (stop || !tile.sees64(blk0 + h * 64)) continue;
          ok = ok && mbar_wait(&s_full[2 * t + h], s_phase[h] & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          ++s_phase[h];
          tc_fence_after();
          uint32_t s[32], seen = 0xffffffffu;
          float m_blk = -INFINITY;
          if (ok) {
            tmem_ld_32x32b_x32(s_tmem + h * 64, s);
            if (edge) seen = window_bits(w, blk0 + h * 64 + half * 32);
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, seen != 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((seen >> i) & 1u)) s[i] = __float_as_uint(-INFINITY);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], __uint_as_float(s[i + 2 * k])), __uint_as_float(s[i + 2 * k + 1]));
            m_blk = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
          }
          if (pair_any(!ok || m_blk > m_run + kWfGrowth)) {   // seldom, after the first blocks; the same for the two warps of these rows
            const float m_other = swap(ok ? m_blk : NAN);
            stop = __any_sync(0xffffffffu, !ok || m_other != m_other);
            if (stop) continue;
            m_blk = fmaxf(m_blk, m_other);
            const float m_new = fmaxf(m_run, ceilf(m_blk));
            const float alpha = m_run == -INFINITY ? 0.f : wf_exp2(m_run - m_new);   // a power of two
            m_run = m_new;
            l_run *= alpha;
            if (LSE) x_run *= alpha;
            if (!first) {                          // once the product before is in O (a wait that runs out is acted on at the next exchange)
              ok = product_done();
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HALF_D; c += 16) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(o_tmem + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                tmem_st_32x32b_x16(o_tmem + c, r);
              }
            }
          }
          first = false;
          ++products;
          const float m_safe = m_run == -INFINITY ? 0.f : m_run;
          const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2), shift2 = f32x2(-m_safe, -m_safe);
          uint64_t sum[2] = {0, 0}, sum_x[2] = {0, 0};
          uint32_t pk[16];
          if (__any_sync(0xffffffffu, seen != 0u)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float a, b;
              f32x2_split(fma_f32x2(f32x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, shift2), a, b);
              a = wf_exp2(a), b = wf_exp2(b);
              pk[i] = pack_bf16x2(a, b);
              sum[i & 1] = add_f32x2(sum[i & 1], bf16x2_as_f32x2(pk[i]));
              if (LSE) sum_x[i & 1] = add_f32x2(sum_x[i & 1], f32x2(a, b));
            }
          } else {                                 // no row of the warp sees one of its keys
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = 0u;
          }
          tmem_st_32x32b_x16(s_tmem + h * 64, pk);
          float lo, hi;
          f32x2_split(add_f32x2(sum[0], sum[1]), lo, hi);
          l_run += lo + hi;
          if (LSE) {
            f32x2_split(add_f32x2(sum_x[0], sum_x[1]), lo, hi);
            x_run += lo + hi;
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + h]);
        }
        if (stop) break;
      }
      if (stop) break;
      // ---------------------------------------------------------------- output
      if (n > 0) {
        ok = ok && product_done();
        tc_fence_after();
      }
      l_run += swap(l_run);
      if (LSE) x_run += swap(x_run);
      // A row that sees nothing is told by its visibility, not by its sum: a query that is no number has to stay one.
      const bool sees = w.hi >= 0;
      const float inv = sees ? 1.f / l_run : 0.f;
      const long long at = ((static_cast<long long>(it.batch) * p.Sq + qi) * p.Hq + head) * D + half * HALF_D;
#pragma unroll 1
      for (int c = 0; c < HALF_D; c += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
        if (n > 0 && ok) {                         // warp-collective: every lane takes part, rows inside the sequence are stored
          tmem_ld_32x32b_x16(o_tmem + c, r);
          tmem_ld_wait();
        }
        if (qi < p.Sq) {
          uint32_t v[8], lo[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float a = __uint_as_float(r[2 * k]) * inv, b = __uint_as_float(r[2 * k + 1]) * inv;
            v[k] = pack_bf16x2(a, b);
            lo[k] = pack_bf16x2(a - __uint_as_float(v[k] << 16), b - __uint_as_float(v[k] & 0xffff0000u));
          }
          store_32_bytes(p.out + at + c, v);
          if (p.out_lo) store_32_bytes(p.out_lo + at + c, lo);
        }
      }
      tc_fence_before();                           // these reads of O come before the next item's first product (via p_full)
      if (qi < p.Sq && half == 0) {
        const long long stat = (static_cast<long long>(it.batch) * p.Hq + head) * p.Sq + qi;
        if (p.lse2) p.lse2[stat] = sees ? m_run + log2f(l_run) : -INFINITY;
        if (LSE) p.lse[stat] = sees ? (m_run + log2f(x_run)) * kWfLn2 : -INFINITY;
      }
    }
  }

  // -------------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    __nanosleep(50000);
    if (threadIdx.x == 0) {
      atomicOr(&p.status[0], MB_ERR_MBAR_TIMEOUT);
      p.status[1] = static_cast<int>(blockIdx.x);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int D, bool LSE>
static int launch_window_fwd(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const WindowFwdArgs& args,
                             cudaStream_t stream) {
  constexpr size_t smem = (2 + kWfStages) * (kWinBlock * D * 2) + 256 + 4 * kWinBlock * sizeof(float);
  static bool configured[64] = {false};
  int dev = 0;
  MB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    MB_CHECK_CUDA(cudaFuncSetAttribute(window_fwd_kernel<D, LSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    configured[dev & 63] = true;
  }
  const int grid = args.items < sm_count() ? args.items : sm_count();
  window_fwd_kernel<D, LSE><<<grid, kWfThreads, smem, stream>>>(tmQ, tmK, tmV, args);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

// ---------------------------------------------------------------------------------------------- documents
// First and one-past-last index of every token's document, one block per row: a thread owns a contiguous piece of the row,
// the pieces are joined by a scan over the block (the last boundary to the left, the first to the right).
constexpr int kDocThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kDocThreads) document_bounds_kernel(const T* __restrict__ ids_all, int* __restrict__ starts_all,
                                                                      int* __restrict__ ends_all, int S) {
  __shared__ int left[kDocThreads], right[kDocThreads];
  const T* ids = ids_all + static_cast<long long>(blockIdx.x) * S;
  int* starts = starts_all + static_cast<long long>(blockIdx.x) * S;
  int* ends = ends_all + static_cast<long long>(blockIdx.x) * S;
  const int per = (S + kDocThreads - 1) / kDocThreads;
  const int tid = threadIdx.x;
  const int a = min(tid * per, S), b = min(a + per, S);
  int first = S, last = 0;                         // first and last index of the piece at which a run begins
  for (int j = a; j < b; ++j)
    if (j == 0 || ids[j] != ids[j - 1]) {
      first = min(first, j);
      last = j;
    }
  left[tid] = last, right[tid] = first;
  __syncthreads();
  for (int o = 1; o < kDocThreads; o <<= 1) {
    const int l = tid >= o ? left[tid - o] : 0, r = tid + o < kDocThreads ? right[tid + o] : S;
    __syncthreads();
    left[tid] = max(left[tid], l), right[tid] = min(right[tid], r);
    __syncthreads();
  }
  int s = tid ? left[tid - 1] : 0;                 // the run that the piece's first token may continue
  const int after = tid + 1 < kDocThreads ? right[tid + 1] : S;
  for (int j = a; j < b; ++j) {
    if (j == 0 || ids[j] != ids[j - 1]) s = j;
    starts[j] = ids[j] == static_cast<T>(-1) ? kWinNone : s;
  }
  int e = after;
  for (int j = b - 1; j >= a; --j) {
    ends[j] = ids[j] == static_cast<T>(-1) ? 0 : e;
    if (j == 0 || ids[j] != ids[j - 1]) e = j;
  }
}

// Sizes, strides and addresses that both directions ask for; nullptr or what is wrong.
const char* window_attn_problem(int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, const long long* strides,
                                int n_strides, const void* const* pointers, int n_pointers) {
  if ((D != 64 && D != 128) || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || B < 1 || Sq < 1 || Sk < 1)
    return "head_dim must be 64 or 128, query heads a multiple of key/value heads, lengths positive";
  if (window < 1 || sinks < 0) return "window must be positive and sinks not negative";
  if (Sq >= (1 << 30) || Sk >= (1 << 30) || B > 65535 || Hq > 65535) return "lengths of 2^30 and more, or over 65535 rows or heads";
  for (int i = 0; i < n_strides; ++i)
    if (strides[i] & 7) return "strides must be multiples of 8 elements";
  for (int i = 0; i < n_pointers; ++i)
    if (reinterpret_cast<uintptr_t>(pointers[i]) & 15) return "tensors must be 16-byte aligned";
  return nullptr;
}

}  // namespace mb

// ids [B, S] (int64 when `wide`, else int32; runs of one id are documents, -1 is padding) -> starts, ends [B, S] as in window.cuh.
MB_API int mb_document_bounds(const void* ids, int wide, int* starts, int* ends, int B, int S, cudaStream_t stream) {
  using namespace mb;
  if (B < 1 || S < 1 || S >= (1 << 30)) {
    set_last_error("mb_document_bounds: rows and lengths must be positive, lengths below 2^30");
    return -1;
  }
  if (wide) document_bounds_kernel<long long><<<B, kDocThreads, 0, stream>>>(static_cast<const long long*>(ids), starts, ends, S);
  else document_bounds_kernel<int><<<B, kDocThreads, 0, stream>>>(static_cast<const int*>(ids), starts, ends, S);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

// q [B, Sq, Hq, D], k / v [B, Sk, Hkv, D] bf16 with element strides between tokens and batches (heads contiguous inside a
// token), out [B, Sq, Hq, D] bf16 contiguous. For the backward: out_lo like out and lse2 [B, Hq, Sq] fp32, or both null. lse
// [B, Hq, Sq] fp32 or null: log-sum-exp, -inf where nothing is visible. starts: mb_document_bounds of the key rows, or null for
// one document a row.
MB_API int mb_window_attn_fwd(const void* q, long long q_tstride, long long q_bstride, const void* k, long long k_tstride,
                              long long k_bstride, const void* v, long long v_tstride, long long v_bstride, void* out, void* out_lo,
                              float* lse2, float* lse, const int* starts, int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, float scale,
                              cudaStream_t stream) {
  using namespace mb;
  const long long strides[] = {q_tstride, q_bstride, k_tstride, k_bstride, v_tstride, v_bstride};
  const void* pointers[] = {q, k, v, out, out_lo};
  if (const char* what = window_attn_problem(B, Sq, Sk, Hq, Hkv, D, window, sinks, strides, 6, pointers, 5)) {
    set_last_error(what);
    return -1;
  }
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_lo)) & 31) {
    set_last_error("mb_window_attn_fwd: outputs must be 32-byte aligned");
    return -3;
  }
  int* status = status_ptr();
  if (!status) return -4;
  WindowFwdArgs a;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_lo = static_cast<__nv_bfloat16*>(out_lo);
  a.lse2 = lse2, a.lse = lse;
  a.rule = {starts, nullptr, window < Sk ? window : Sk, sinks < Sk ? sinks : Sk};
  a.B = B, a.Sq = Sq, a.Sk = Sk, a.Hq = Hq, a.Hkv = Hkv;
  a.scale_log2 = scale * kWfLog2e;
  a.status = status;
  // Two tiles to an item once there are more tiles than SMs; below that every tile gets an SM of its own.
  const long long row_tiles = (Sq + kWinBlock - 1) / kWinBlock;
  a.pair = row_tiles * Hq * B <= sm_count() ? 0 : (Hq / Hkv) % 2 == 0 ? 1 : 2;
  a.row_units = static_cast<int>(a.pair == 2 ? (row_tiles + 1) / 2 : row_tiles);
  a.head_units = a.pair == 1 ? Hq / 2 : Hq;
  const long long items = static_cast<long long>(a.row_units) * a.head_units * B;
  if (items >= (1ll << 31) - 65536) {
    set_last_error("mb_window_attn_fwd: too many query tiles");
    return -1;
  }
  a.items = static_cast<int>(items);
  CUtensorMap tmQ, tmK, tmV;
  const uint32_t box[4] = {64, 1, static_cast<uint32_t>(kWinBlock), 1};
  auto encode = [&](CUtensorMap* m, const void* x, int heads, int S, long long tstride, long long bstride) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)S, (uint64_t)B};
    const uint64_t bytes[3] = {(uint64_t)D * 2, (uint64_t)tstride * 2, (uint64_t)bstride * 2};
    return encode_tmap_4d(m, x, dims, bytes, box, 2, true);
  };
  if (!encode(&tmQ, q, Hq, Sq, q_tstride, q_bstride) || !encode(&tmK, k, Hkv, Sk, k_tstride, k_bstride) ||
      !encode(&tmV, v, Hkv, Sk, v_tstride, v_bstride))
    return -5;
  if (D == 128) return lse ? launch_window_fwd<128, true>(tmQ, tmK, tmV, a, stream) : launch_window_fwd<128, false>(tmQ, tmK, tmV, a, stream);
  return lse ? launch_window_fwd<64, true>(tmQ, tmK, tmV, a, stream) : launch_window_fwd<64, false>(tmQ, tmK, tmV, a, stream);
}
