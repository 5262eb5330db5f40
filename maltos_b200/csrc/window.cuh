// The visibility rule of sliding-window attention, shared by its forward and backward kernels. Query i of Sq stands at key
// index p = i + Sk - Sq; s(p) is the first index of p's document (0 without documents). Key j is visible to p iff
//     s(p) <= j <= p  and  (p - j < window  or  j - s(p) < sinks).
// For a query that is the union of two intervals, [lo, p] and [s, sink_end); for a key it is ONE interval of queries,
// [j, upper). Documents enter only through two arrays, starts and ends, so no sequence ids are compared in the loops.
#pragma once
#include "ptx.cuh"

namespace mb {

// Sizes, strides and addresses that both directions ask for; nullptr or what is wrong (window_attn.cu).
const char* window_attn_problem(int B, int Sq, int Sk, int Hq, int Hkv, int D, int window, int sinks, const long long* strides,
                                int n_strides, const void* const* pointers, int n_pointers);

constexpr int kWinNone = 0x7fffffff;   // start of a padding token: sees nothing
constexpr int kWinBlock = 128;         // keys per block, query rows per tile

struct WindowRule {
  const int* starts;   // [B, Sk] first index of the token's document, kWinNone for padding; nullptr: one document a row
  const int* ends;     // [B, Sk] one past the last index of the token's document, 0 for padding (with starts)
  int window, sinks;   // both at most Sk
};

// Key intervals of one query.
struct WindowRow {
  int lo, hi;                 // [lo, hi]
  int sink_begin, sink_end;   // [sink_begin, sink_end), before lo
};

__device__ __forceinline__ WindowRow window_row(const WindowRule& r, int batch, int Sk, int p, bool valid) {
  WindowRow w;
  w.lo = w.sink_begin = w.sink_end = kWinNone, w.hi = -1;
  if (!valid || p < 0) return w;
  const int s = r.starts ? r.starts[static_cast<long long>(batch) * Sk + p] : 0;
  if (s == kWinNone) return w;
  w.lo = max(s, p - r.window + 1);
  w.hi = p;
  w.sink_begin = s;
  w.sink_end = min(s + r.sinks, w.lo);
  return w;
}

// Bits of the 32 keys from key0 that lie in [begin, end).
__device__ __forceinline__ uint32_t interval_bits(int key0, int begin, int end) {
  const int a = min(max(begin - key0, 0), 32), b = min(max(end - key0, 0), 32);
  uint32_t m;
  asm("bmsk.clamp.b32 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(max(b - a, 0)));
  return m;
}
__device__ __forceinline__ uint32_t window_bits(const WindowRow& w, int key0) {
  return interval_bits(key0, w.lo, w.hi + 1) | interval_bits(key0, w.sink_begin, w.sink_end);
}

// Key blocks that the 128 query rows from q0 have to visit: first tokens [sa, ea), then the window [b0, b1), ea <= b0. Every
// row sees every key of a block that lies inside [full_lo, full_hi]. Called by a whole warp, the same for all lanes: lo and the
// document's start never fall with p, so with documents the first real row decides where the window and the first tokens begin
// (a document that starts inside the tile has its first tokens in the window's blocks).
struct WindowTile {
  int sa, ea, b0, b1;
  int full_lo, full_hi;
  int lo, last, far, far_end;   // keys that some row sees: [lo, last] and [far, far_end)
  // whether some row sees a key of the 64 from `key0`
  __device__ __forceinline__ bool sees64(int key0) const { return (key0 <= last && key0 + 63 >= lo) || (key0 < far_end && key0 + 63 >= far); }
  __device__ __forceinline__ int count() const { return (ea - sa) + (b1 - b0); }
  __device__ __forceinline__ bool has(int blk) const { return (blk >= sa && blk < ea) || (blk >= b0 && blk < b1); }
  __device__ __forceinline__ int block(int n) const { return n < ea - sa ? sa + n : b0 + n - (ea - sa); }
};

__device__ __forceinline__ WindowTile window_tile(const WindowRule& r, int batch, int Sq, int Sk, int q0) {
  WindowTile t;
  t.sa = t.ea = t.b0 = t.b1 = 0;
  t.full_lo = kWinNone, t.full_hi = -1;
  t.lo = t.far = kWinNone, t.last = t.far_end = -1;
  const int off = Sk - Sq;
  const int first = q0 + off, p1 = min(q0 + kWinBlock, Sq) - 1 + off;
  if (q0 >= Sq || p1 < 0) return t;
  const int p0 = max(first, 0);
  int start, lo, last, lo_max;
  bool whole = first >= 0;
  if (r.starts == nullptr) {
    start = 0, lo = max(0, p0 - r.window + 1), last = p1, lo_max = max(0, p1 - r.window + 1);
  } else {
    start = kWinNone, lo = kWinNone, last = -1, lo_max = -1;
    int pad = 0;
    const int* s = r.starts + static_cast<long long>(batch) * Sk;
    for (int p = p0 + static_cast<int>(lane_id()); p <= p1; p += 32) {
      const int sp = s[p];
      if (sp == kWinNone) {
        pad = 1;
        continue;
      }
      const int l = max(sp, p - r.window + 1);
      start = min(start, sp), lo = min(lo, l), last = max(last, p), lo_max = max(lo_max, l);
    }
    start = __reduce_min_sync(0xffffffffu, start);
    lo = __reduce_min_sync(0xffffffffu, lo);
    last = __reduce_max_sync(0xffffffffu, last);
    lo_max = __reduce_max_sync(0xffffffffu, lo_max);
    if (__any_sync(0xffffffffu, pad)) whole = false;
    if (last < 0) return t;
  }
  t.b0 = lo / kWinBlock, t.b1 = last / kWinBlock + 1;
  t.lo = lo, t.last = last;
  const int far_end = min(start + r.sinks, lo);
  if (far_end > start) {                           // else nothing lies before the window (no first tokens, or all inside it)
    t.far = start, t.far_end = far_end;
    t.sa = start / kWinBlock, t.ea = min((far_end + kWinBlock - 1) / kWinBlock, t.b0);
    if (t.ea <= t.sa) t.sa = t.ea = 0;
  }
  if (whole) t.full_lo = lo_max, t.full_hi = p0;
  return t;
}

// One past the last query position that sees key j of the document [start, end).
__device__ __forceinline__ int window_upper(const WindowRule& r, int start, int end, int j) {
  return j - start < r.sinks ? end : min(end, j + r.window);
}


// Query rows [q_lo, q_hi) that see some of the 128 keys from k0. Every query at a position in [k0 + 127, full_hi) sees all of them
// (full_hi 0: no such query). Called by a whole warp, the same for all lanes.
struct WindowKeys {
  int q_lo, q_hi, full_hi;
};

__device__ __forceinline__ WindowKeys window_keys(const WindowRule& r, int batch, int Sq, int Sk, int k0) {
  WindowKeys t;
  const int off = Sk - Sq, k1 = min(k0 + kWinBlock, Sk) - 1;
  int first, up_min, up_max;
  bool whole = k0 + kWinBlock <= Sk;
  if (r.starts == nullptr) {
    first = k0;
    up_max = k0 < r.sinks ? Sk : min(Sk, k1 + r.window);
    up_min = k1 < r.sinks ? Sk : min(Sk, max(k0, r.sinks) + r.window);
  } else {
    first = kWinNone, up_min = kWinNone, up_max = 0;
    int pad = 0;
    const long long base = static_cast<long long>(batch) * Sk;
    for (int j = k0 + static_cast<int>(lane_id()); j <= k1; j += 32) {
      const int s = r.starts[base + j];
      if (s == kWinNone) {
        pad = 1;
        continue;
      }
      const int up = window_upper(r, s, r.ends[base + j], j);
      first = min(first, j), up_min = min(up_min, up), up_max = max(up_max, up);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    up_min = __reduce_min_sync(0xffffffffu, up_min);
    up_max = __reduce_max_sync(0xffffffffu, up_max);
    if (__any_sync(0xffffffffu, pad)) whole = false;
    if (up_max == 0) {                             // padding only
      t.q_lo = t.q_hi = t.full_hi = 0;
      return t;
    }
  }
  t.q_lo = max(0, first - off);
  t.q_hi = min(Sq, up_max - off);
  t.full_hi = whole ? up_min : 0;
  return t;
}

}  // namespace mb
