// Embedding lookup with a scale, and its gradient by sorted tokens (bf16, fp16, fp32 tables).
//   forward   out[t] = scale * weight[ids[t]]
//   gradient  dweight[r] = scale * sum of dout[t] over the tokens t of row r, in the order of t and in fp32, rounded once
// Three launches make the gradient, without atomics on floating-point values, so its bits do not depend on the schedule:
//   embedding_sort_kernel   one cluster sorts the pairs (row, t) by row, stably, with digits of up to 9 bits (two passes
//                           up to 2^18 rows; of 8 bits three from 2^16 on: 33 us for 32768 tokens, where two take 28);
//   embedding_chunk_kernel  one CTA per 32 sorted tokens (and slice of columns): runs that lie inside go straight to their row,
//                           the parts of runs that cross a chunk's border go to fp32 buffers. A frequent token is thereby
//                           spread over as many CTAs as it has chunks. The CTAs behind them write the zeros, of which most of
//                           dweight consists: each looks its rows up among the sorted ones;
//   embedding_join_kernel   adds the parts of the crossing runs, in order.
// Bound by memory: 32768 tokens into a bf16 table of 128256 x 4096 take 70 us forward and 250 us backward: sort 28, runs and zeros
// 198 (1.3 GB at 6.7 TB/s), join 23. (Zeros of the whole table, written under the sort by the other CTAs of its grid, took 217 us:
// a grid of clusters does not keep the SMs full.) With few tokens the launches are what counts: 1024 tokens of a 32000 x 512 table
// 4 + 27 us.
// Ids outside the table set the status word (index out of bounds), read as zero rows and get no gradient.
#include "host.h"
#include "ptx.cuh"
#include "vec.cuh"

namespace mb {

constexpr int kEmbThreads = 256;
constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBins = 512;
constexpr int kEmbChunk = 32;
constexpr int kZeroBytes = 128 * 1024;   // of a CTA of zeros, which looks up 32 rows (wide tables) to 256 (narrow ones)
constexpr int kEmbJoinThreads = 64;   // narrow blocks: a frequent token's parts are added by several SMs

template <typename I>
__device__ __forceinline__ long long emb_row(const I* ids, long long t, long long rows) {
  const long long r = static_cast<long long>(ids[t]);
  return r >= 0 && r < rows ? r : -1;
}

// threadIdx.x walks the columns of a row, threadIdx.y picks the token.
template <typename T, int N, typename I>
__global__ void __launch_bounds__(kEmbThreads) embedding_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ weight, T* __restrict__ out,
                                                                    long long tokens, int H, long long rows, float scale, int* status) {
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= tokens) return;
  const long long r = emb_row(ids, t, rows);
  if (r < 0 && threadIdx.x == 0) {
    atomicOr(&status[0], MB_ERR_BAD_INDEX);
    status[2] = static_cast<int>(ids[t]);
  }
  const T* src = weight + r * H;
  T* dst = out + t * H;
  const int step = blockDim.x * N;
#pragma unroll 4
  for (int c = threadIdx.x * N; c < H; c += step) {
    Vec<T, N> v;
    if (r >= 0) {
      v.load(src + c);
#pragma unroll
      for (int k = 0; k < N; ++k) v.set(k, v.get(k) * scale);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) v.set(k, 0.f);
    }
    v.store(dst + c);
  }
}

// ---------------------------------------------------------------------------------------------- sort
struct EmbSortArgs {
  const void* ids;
  int* key[2];        // ping-pong pairs; the sorted ones end in [passes & 1 ? 0 : 1]
  int* pos[2];
  int tokens, rows;   // rows: also the key of tokens that get no gradient (outside the table, or padding_idx)
  int pad;            // padding_idx, or -1
  int passes, bits;
};

// shared memory of another CTA of the cluster
__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename I>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads) embedding_sort_kernel(const EmbSortArgs p) {
  extern __shared__ int hist_all[];             // per warp: counts, then where the warp's next element of a digit goes
  int(*hist)[kSortBins] = reinterpret_cast<int(*)[kSortBins]>(hist_all);
  __shared__ int total[kSortBins];              // of this CTA, read by the others
  __shared__ int scan[kSortBins / 32];
  const int cta = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const I* ids = static_cast<const I*>(p.ids);
  // A CTA owns a contiguous piece, a warp a contiguous part of it, multiples of 32 long: elements are in the order of (CTA, warp,
  // step, lane). Few tokens are few warps' work, since the counts of all warps are added up one after the other.
  const long long cta_per = (static_cast<long long>(p.tokens + kSortCtas - 1) / kSortCtas + 31) / 32 * 32;
  const int warps = static_cast<int>(cta_per / 32 < kSortWarps ? cta_per / 32 : kSortWarps);
  const long long per = (cta_per / 32 + warps - 1) / warps * 32;
  const long long cta_end = min((cta + 1) * cta_per, static_cast<long long>(p.tokens));
  const int a = static_cast<int>(min(cta * cta_per + warp * per, cta_end)), b = warp < warps ? static_cast<int>(min(a + per, cta_end)) : a;
  const int bins = 1 << p.bits;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const int* key_in = p.key[(pass + 1) & 1];
    const int* pos_in = p.pos[(pass + 1) & 1];
    int* key_out = p.key[pass & 1];
    int* pos_out = p.pos[pass & 1];
    // the pairs were written by other SMs of the cluster: read past L1
    auto fetch = [&](int i) -> int {
      if (pass) return __ldcg(key_in + i);
      const long long r = emb_row(ids, i, p.rows);
      return r < 0 || r == p.pad ? p.rows : static_cast<int>(r);
    };
    for (int d = lane; d < bins; d += 32) hist[warp][d] = 0;
    __syncwarp();
    for (int i0 = a; i0 < b; i0 += 32) {
      const int i = i0 + lane;
      const int d = i < b ? (fetch(i) >> shift) & (bins - 1) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (d >= 0 && (same & ((1u << lane) - 1)) == 0) hist[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    int sum = 0;                                // of digit `tid` in this CTA
    if (tid < bins) {
      for (int w = 0; w < warps; ++w) {
        const int n = hist[w][tid];
        hist[w][tid] = sum;
        sum += n;
      }
      total[tid] = sum;
    }
    cluster_arrive();
    cluster_wait();
    int before = 0, all = 0;                    // this digit in earlier CTAs, and everywhere
    if (tid < bins)
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        const int n = ld_cluster_s32(mapa_u32(&total[tid], c));
        all += n;
        if (c < cta) before += n;
      }
    // digits in order: a scan of each warp's 32, then of the warps
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    if (lane == 31 && warp < kSortBins / 32) scan[warp] = inc;
    __syncthreads();
    if (tid < bins) {
      int base = inc - all + before;
      for (int w = 0; w < warp; ++w) base += scan[w];
      for (int w = 0; w < warps; ++w) hist[w][tid] += base;
    }
    __syncthreads();
    for (int i0 = a; i0 < b; i0 += 32) {
      const int i = i0 + lane;
      const int key = i < b ? fetch(i) : 0;
      const int d = i < b ? (key >> shift) & (bins - 1) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      const unsigned lower = same & ((1u << lane) - 1);
      if (d >= 0) {
        const int at = hist[warp][d] + __popc(lower);
        key_out[at] = key;
        pos_out[at] = pass ? __ldcg(pos_in + i) : i;
      }
      __syncwarp();
      if (d >= 0 && lower == 0) hist[warp][d] += __popc(same);
      __syncwarp();
    }
    cluster_arrive();                           // the pairs of this pass are written, and nobody reads `total` any more
    cluster_wait();
  }
}

// ---------------------------------------------------------------------------------------------- runs
// N consecutive fp32 values, 16 bytes at a time where they fill that.
template <int N>
__device__ __forceinline__ void add_row(float (&acc)[N], const float* p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + k);
      acc[k] += v.x, acc[k + 1] += v.y, acc[k + 2] += v.z, acc[k + 3] += v.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += p[k];
  }
}
template <int N>
__device__ __forceinline__ void put_row(float* p, const float (&acc)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(p + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) p[k] = acc[k];
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kEmbThreads) embedding_chunk_kernel(const int* __restrict__ key, const int* __restrict__ pos,
                                                                      const T* __restrict__ dout, T* __restrict__ dweight,
                                                                      float* __restrict__ head, float* __restrict__ tail, int tokens, int H,
                                                                      int rows, int chunks, int zero_rows, float scale) {
  __shared__ int s_key[kEmbChunk + 2], s_pos[kEmbChunk];
  __shared__ bool s_used[kEmbThreads];
  const int c = (blockIdx.y * kEmbThreads + threadIdx.x) * N;
  if (static_cast<int>(blockIdx.x) >= chunks) {    // zeros of the rows that no token has
    const long long row0 = static_cast<long long>(blockIdx.x - chunks) * zero_rows;
    const int n = static_cast<int>(rows - row0 < zero_rows ? rows - row0 : zero_rows);
    if (threadIdx.x < n) {
      const int r = static_cast<int>(row0) + threadIdx.x;
      int lo = 0, hi = tokens;                     // the first token whose row is r or a later one
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (key[mid] < r) lo = mid + 1;
        else hi = mid;
      }
      s_used[threadIdx.x] = lo < tokens && key[lo] == r;
    }
    __syncthreads();
    // vector by vector of this slice of columns, row after row, so that narrow rows keep all threads busy
    const int c0 = blockIdx.y * kEmbThreads * N, width = min(kEmbThreads, (H - c0) / N);
    Vec<T, N> none;
#pragma unroll
    for (int k = 0; k < N; ++k) none.set(k, 0.f);
    int i = threadIdx.x / width, v = threadIdx.x % width;
    const int down = kEmbThreads / width, right = kEmbThreads % width;
    while (i < n) {
      if (!s_used[i]) none.store(dweight + (row0 + i) * H + c0 + v * N);
      i += down, v += right;
      if (v >= width) v -= width, ++i;
    }
    return;
  }
  const long long first = static_cast<long long>(blockIdx.x) * kEmbChunk;
  const int n = static_cast<int>(tokens - first < kEmbChunk ? tokens - first : kEmbChunk);
  if (threadIdx.x < kEmbChunk + 2) {               // the chunk's rows with one neighbour on either side, -1 beyond the ends
    const long long i = first + threadIdx.x - 1;
    s_key[threadIdx.x] = i >= 0 && i < tokens ? key[i] : -1;
    if (threadIdx.x < n) s_pos[threadIdx.x] = pos[first + threadIdx.x];
  }
  __syncthreads();
  if (c >= H) return;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  constexpr int AHEAD = 8;
  bool from_left = s_key[0] == s_key[1];           // the run that is being summed began in an earlier chunk
  for (int i0 = 0; i0 < n; i0 += AHEAD) {
    Vec<T, N> v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i0 + j < n && s_key[i0 + j + 1] != rows) v[j].load(dout + static_cast<long long>(s_pos[i0 + j]) * H + c);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j;
      if (i >= n) break;
      const int r = s_key[i + 1];
      if (r == rows) break;                        // sorted: only tokens without a gradient from here on
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += v[j].get(k);
      const bool run_ends = s_key[i + 2] != r;
      if (!run_ends && i + 1 < n) continue;
      if (run_ends && !from_left) {
        Vec<T, N> o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.set(k, acc[k] * scale);
        o.store(dweight + static_cast<long long>(r) * H + c);
      } else {                                     // `head` where the run came in from the left, `tail` where it began here
        put_row(((from_left ? head : tail) + static_cast<long long>(blockIdx.x) * H + c), acc);
      }
      from_left = false;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.f;
    }
  }
}

// One CTA per chunk in which a run begins that crosses the chunk's right border.
template <typename T, int N>
__global__ void __launch_bounds__(kEmbJoinThreads) embedding_join_kernel(const int* __restrict__ key, T* __restrict__ dweight,
                                                                     const float* __restrict__ head, const float* __restrict__ tail,
                                                                     int tokens, int H, int rows, float scale) {
  const int chunk = blockIdx.x;
  const long long first = static_cast<long long>(chunk) * kEmbChunk, next = first + kEmbChunk;
  if (next >= tokens) return;
  const int r = key[next - 1];
  if (r == rows || key[next] != r) return;                                  // nothing crosses
  if (key[first] == r && first > 0 && key[first - 1] == r) return;          // it began earlier: that chunk's CTA adds it up
  // the chunks that the run goes on in: sorted, so the number of chunks that begin with r; looked for by the whole block at once
  int more = 0;
  for (int base = 0;; base += kEmbJoinThreads) {
    const long long at = next + static_cast<long long>(base + threadIdx.x) * kEmbChunk;
    const int hit = __syncthreads_count(at < tokens && key[at] == r);
    more += hit;
    if (hit < kEmbJoinThreads) break;
  }
  const int c = (blockIdx.y * kEmbJoinThreads + threadIdx.x) * N;
  if (c >= H) return;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  add_row(acc, tail + static_cast<long long>(chunk) * H + c);
#pragma unroll 8
  for (int i = 1; i <= more; ++i) add_row(acc, head + static_cast<long long>(chunk + i) * H + c);
  Vec<T, N> o;
#pragma unroll
  for (int k = 0; k < N; ++k) o.set(k, acc[k] * scale);
  o.store(dweight + static_cast<long long>(r) * H + c);
}

template <typename T, int N, typename I>
static int launch_embedding_fwd(const void* ids, const void* weight, void* out, long long tokens, int H, long long rows, float scale,
                                int* status, cudaStream_t stream) {
  int x = 32;                                      // threads along a row: enough to cover it, at most the block
  while (x < kEmbThreads && x * N < H) x *= 2;
  const int y = kEmbThreads / x;
  embedding_fwd_kernel<T, N, I><<<static_cast<unsigned>((tokens + y - 1) / y), dim3(x, y), 0, stream>>>(
      static_cast<const I*>(ids), static_cast<const T*>(weight), static_cast<T*>(out), tokens, H, rows, scale, status);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <typename T, int N>
static int launch_embedding_runs(const EmbSortArgs& s, const void* dout, void* dweight, float* parts, int H, float scale, cudaStream_t stream) {
  const int* key = s.key[(s.passes - 1) & 1];
  const int* pos = s.pos[(s.passes - 1) & 1];
  const int chunks = (s.tokens + kEmbChunk - 1) / kEmbChunk;
  float* tail = parts + static_cast<long long>(chunks) * H;
  const int slice = (H / N < kEmbThreads ? H / N : kEmbThreads) * N * static_cast<int>(sizeof(T));   // bytes of a row in a CTA of zeros
  const int zero_rows = kZeroBytes / slice < 32 ? 32 : kZeroBytes / slice < kEmbThreads ? kZeroBytes / slice : kEmbThreads;
  const long long zeros = (static_cast<long long>(s.rows) + zero_rows - 1) / zero_rows;
  const dim3 grid(static_cast<unsigned>(chunks + zeros), (H / N + kEmbThreads - 1) / kEmbThreads);
  embedding_chunk_kernel<T, N><<<grid, kEmbThreads, 0, stream>>>(key, pos, static_cast<const T*>(dout), static_cast<T*>(dweight), parts,
                                                               tail, s.tokens, H, s.rows, chunks, zero_rows, scale);
  embedding_join_kernel<T, N><<<dim3(chunks, (H / N + kEmbJoinThreads - 1) / kEmbJoinThreads), kEmbJoinThreads, 0, stream>>>(key, static_cast<T*>(dweight), parts, tail, s.tokens, H, s.rows, scale);
  count_launch(2);
  MB_CHECK_CUDA(cudaGetLastError());
  return 0;
}

static const char* embedding_problem(int dtype, long long tokens, long long rows, int H) {
  if (dtype < 0 || dtype > 2) return "embedding: the table is bf16, fp16 or fp32";
  if (tokens < 1 || tokens >= (1ll << 31) - 65536 || rows < 1 || rows >= (1ll << 31) - 1 || H < 1 || H > (1 << 21))
    return "embedding: tokens and rows below 2^31, hidden size up to 2^21, all positive";
  return nullptr;
}

}  // namespace mb

// ids [tokens] int64 (`wide`) or int32, weight [rows, H] contiguous, out [tokens, H]; dtype 0 bf16, 1 fp16, 2 fp32.
MB_API int mb_embedding_fwd(const void* ids, int wide, const void* weight, void* out, int dtype, long long tokens, int H, long long rows,
                            float scale, cudaStream_t stream) {
  using namespace mb;
  if (const char* what = embedding_problem(dtype, tokens, rows, H)) {
    set_last_error(what);
    return -1;
  }
  int* status = status_ptr();
  if (!status) return -4;
  const bool aligned = ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
#define MB_EMB(T, N)                                                                                                     \
  (wide ? launch_embedding_fwd<T, N, long long>(ids, weight, out, tokens, H, rows, scale, status, stream)                \
        : launch_embedding_fwd<T, N, int>(ids, weight, out, tokens, H, rows, scale, status, stream))
  if (dtype == 2) return aligned && H % 4 == 0 ? MB_EMB(float, 4) : MB_EMB(float, 1);
  if (dtype == 1) return aligned && H % 8 == 0 ? MB_EMB(__half, 8) : MB_EMB(__half, 1);
  return aligned && H % 8 == 0 ? MB_EMB(__nv_bfloat16, 8) : MB_EMB(__nv_bfloat16, 1);
#undef MB_EMB
}

// 4-byte words of scratch for mb_embedding_bwd: the pairs twice, and two fp32 rows per chunk of sorted tokens.
MB_API long long mb_embedding_bwd_scratch_words(long long tokens, int H) {
  const long long chunks = (tokens + mb::kEmbChunk - 1) / mb::kEmbChunk;
  return (4 * tokens + 3) / 4 * 4 + 2 * chunks * H;
}

// dout [tokens, H] contiguous -> dweight [rows, H], every element written. padding_idx -1: none.
MB_API int mb_embedding_bwd(const void* ids, int wide, const void* dout, void* dweight, int* scratch, int dtype, long long tokens, int H,
                            long long rows, long long padding_idx, float scale, cudaStream_t stream) {
  using namespace mb;
  if (const char* what = embedding_problem(dtype, tokens, rows, H)) {
    set_last_error(what);
    return -1;
  }
  if ((reinterpret_cast<uintptr_t>(dweight) | reinterpret_cast<uintptr_t>(scratch)) & 15) {
    set_last_error("mb_embedding_bwd: dweight and scratch must be 16-byte aligned");
    return -3;
  }
  EmbSortArgs s;
  s.ids = ids;
  s.key[0] = scratch, s.key[1] = scratch + tokens, s.pos[0] = scratch + 2 * tokens, s.pos[1] = scratch + 3 * tokens;
  float* parts = reinterpret_cast<float*>(scratch + (4 * tokens + 3) / 4 * 4);
  s.tokens = static_cast<int>(tokens), s.rows = static_cast<int>(rows), s.pad = static_cast<int>(padding_idx);
  int width = 1;
  while ((rows >> width) != 0) ++width;            // bits of the largest key, `rows`
  s.passes = (width + 8) / 9;
  s.bits = (width + s.passes - 1) / s.passes;
  constexpr int kSortBytes = kSortWarps * kSortBins * static_cast<int>(sizeof(int));
  static bool configured[64] = {false};
  int dev = 0;
  MB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    MB_CHECK_CUDA(cudaFuncSetAttribute(embedding_sort_kernel<long long>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortBytes));
    MB_CHECK_CUDA(cudaFuncSetAttribute(embedding_sort_kernel<int>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortBytes));
    configured[dev & 63] = true;
  }
  if (wide) embedding_sort_kernel<long long><<<kSortCtas, kSortThreads, kSortBytes, stream>>>(s);
  else embedding_sort_kernel<int><<<kSortCtas, kSortThreads, kSortBytes, stream>>>(s);
  count_launch();
  MB_CHECK_CUDA(cudaGetLastError());
  const bool aligned = (reinterpret_cast<uintptr_t>(dout) & 15) == 0;
  if (dtype == 2) return aligned && H % 4 == 0 ? launch_embedding_runs<float, 4>(s, dout, dweight, parts, H, scale, stream)
                                               : launch_embedding_runs<float, 1>(s, dout, dweight, parts, H, scale, stream);
  if (dtype == 1) return aligned && H % 8 == 0 ? launch_embedding_runs<__half, 8>(s, dout, dweight, parts, H, scale, stream)
                                               : launch_embedding_runs<__half, 1>(s, dout, dweight, parts, H, scale, stream);
  return aligned && H % 8 == 0 ? launch_embedding_runs<__nv_bfloat16, 8>(s, dout, dweight, parts, H, scale, stream)
                               : launch_embedding_runs<__nv_bfloat16, 1>(s, dout, dweight, parts, H, scale, stream);
}
