// Embedding lookup with scaling and its gradient by sorted tokens.
//
// For token ids t (n of them), a table W (vocab x dim, fp32 or bf16) and a scale s:
//   lookup     y_i = s W[t_i]
//   gradient   dW[v] = s sum_{i : t_i = v} dy_i   (0 where no token is v or v is the padding id)
// The lookup is linear in W and the gradient in dy, so each is the other's derivative:
// the backward's backward is the lookup of the cotangent of dW, and so on for any order.
//
// The lookup reads and writes one row a token: bound by memory, or by launch latency for
// a few tokens.
//
// The gradient has to write the whole table, most of it zeros when there are fewer tokens
// than rows, and to add up the rows of equal tokens in an order that does not depend on
// the run (no floating-point atomics). Three launches:
//   1. One cluster of CTAs sorts (token, position) stably: a radix sort, least significant
//      digit first, over one to four digits of at most 10 bits. The digit counts of its
//      CTAs meet in distributed shared memory, so a pass needs cluster barriers only. The
//      other clusters of the same launch fill dW with zeros meanwhile: that is most of the
//      gradient's bytes at the sizes of a training step, and it hides the sort.
//   2. The sorted list is cut into chunks. A CTA adds up the runs of equal tokens of its
//      chunk in fp32, in the order of the positions, and writes the sums of the runs that
//      lie inside the chunk; of a run that crosses the chunk's ends it keeps partial sums.
//   3. The runs that cross chunk borders: their partial sums are added in chunk order.
// One rounding to the table's type, at the end.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "vec_io.cuh"

namespace fh {
namespace {

// ------------------------------------------------------------------------------------
// Lookup
// ------------------------------------------------------------------------------------

constexpr int kLookupThreads = 256;

// `lanes` (a power of two up to kLookupThreads) threads per token, each block kLookupRows
// times as many tokens as it has such groups: their ids are loaded together, then their
// rows, so that a group has several rows in flight. A token outside [0, vocab) gives `oob`
// in every element; token `skip` gives zeros (-1: none).
constexpr int kLookupRows = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kLookupThreads)
    embed_lookup_kernel(long long n, long long vocab, int dim, int lanes_log2, const long long* __restrict__ tokens,
                        const T* __restrict__ w, float scale, long long skip, float oob, T* __restrict__ y) {
  constexpr int E = VEC ? 16 / sizeof(T) : 1;
  const int lane = threadIdx.x & ((1 << lanes_log2) - 1);
  const int groups = kLookupThreads >> lanes_log2, nv = dim / E;
  const long long i0 = static_cast<long long>(blockIdx.x) * groups * kLookupRows + (threadIdx.x >> lanes_log2);
  long long t[kLookupRows];
  bool plain = i0 + (kLookupRows - 1) * groups < n;  // whole group of rows, every token in the table
#pragma unroll
  for (int r = 0; r < kLookupRows; ++r) {
    const long long i = i0 + r * groups;
    t[r] = i < n ? tokens[i] : -1;
    plain = plain && t[r] >= 0 && t[r] < vocab && t[r] != skip;
  }
  if (plain) {
    for (int c = lane; c < nv; c += 1 << lanes_log2) {
      float v[kLookupRows][E];
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r) load_vec<T, E>(w + t[r] * dim + c * E, v[r]);
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r) {
#pragma unroll
        for (int k = 0; k < E; ++k) v[r][k] *= scale;
        store_vec<T, E>(y + (i0 + r * groups) * dim + c * E, v[r]);
      }
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < kLookupRows; ++r) {
    const long long i = i0 + r * groups;
    if (i >= n) return;
    const bool outside = t[r] < 0 || t[r] >= vocab, none = outside || t[r] == skip;
    const T* row = w + (none ? 0 : t[r]) * dim;
    for (int c = lane; c < nv; c += 1 << lanes_log2) {
      float v[E];
      load_vec<T, E>(row + c * E, v);
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = none ? (outside ? oob : 0.f) : v[k] * scale;
      store_vec<T, E>(y + i * dim + c * E, v);
    }
  }
}

// ------------------------------------------------------------------------------------
// Gradient, 1: sort and zero fill
// ------------------------------------------------------------------------------------

constexpr int kSortCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 10;

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Every thread of the cluster; orders global and (distributed) shared memory accesses.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ unsigned ld_dsmem(const unsigned* p, unsigned rank) {
  unsigned a = static_cast<unsigned>(__cvta_generic_to_shared(p)), ra, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ra) : "memory");
  return v;
}

struct SortArgs {
  int n;
  int vocab;          // keys are tokens, or `vocab` for those without a gradient (sorted last)
  long long padding;  // token without a gradient, -1: none
  const long long* tokens;
  unsigned *key[2], *pos[2];  // ping-pong buffers of n entries; the sorted list ends in [passes & 1]
  int bits, passes;           // bits per digit
  uint4* fill;                // the gradient, zero-filled by the clusters after the first
  long long fill_vecs;        // 16-byte vectors, then
  unsigned short* fill_tail;  // tail_halves 2-byte units
  int tail_halves;
};

__global__ void __cluster_dims__(kSortCluster, 1, 1) __launch_bounds__(kSortThreads)
    embed_sort_kernel(const SortArgs a) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (blockIdx.x >= kSortCluster) {
    // ------------------------------ zero fill ------------------------------
    const long long stride = static_cast<long long>(gridDim.x - kSortCluster) * kSortThreads;
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (long long i = static_cast<long long>(blockIdx.x - kSortCluster) * kSortThreads + tid; i < a.fill_vecs;
         i += stride)
      a.fill[i] = z;
    if (blockIdx.x == kSortCluster && tid < a.tail_halves) a.fill_tail[tid] = 0;
    return;
  }
  // -------------------------------- radix sort --------------------------------
  extern __shared__ unsigned sm[];
  const int bins = 1 << a.bits;
  unsigned* hist = sm;                        // [kSortWarps][bins]: counts, then each warp's next index
  unsigned* total = sm + kSortWarps * bins;   // [bins]: this CTA's counts, read by the cluster
  __shared__ unsigned warp_sum[kSortWarps];
  const unsigned rank = cluster_rank();
  // Each warp owns a run of consecutive elements (whole groups of 32), CTAs and warps in order.
  const long long groups = (a.n + 31) / 32;
  const long long per_warp = (groups + kSortCluster * kSortWarps - 1) / (kSortCluster * kSortWarps) * 32;
  const long long first = (static_cast<long long>(rank) * kSortWarps + warp) * per_warp;
  const long long last = min(first + per_warp, static_cast<long long>(a.n));
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    const unsigned* ksrc = a.key[pass & 1];
    const unsigned* psrc = a.pos[pass & 1];
    unsigned* kdst = a.key[(pass + 1) & 1];
    unsigned* pdst = a.pos[(pass + 1) & 1];
    auto load_key = [&](long long i) -> unsigned {
      if (pass > 0) return __ldcg(ksrc + i);
      const long long t = a.tokens[i];
      return (t < 0 || t >= a.vocab || t == a.padding) ? static_cast<unsigned>(a.vocab) : static_cast<unsigned>(t);
    };
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0u;
    __syncthreads();
    unsigned* mine = hist + warp * bins;
    for (long long i = first + lane; i < last; i += 32) atomicAdd(&mine[(load_key(i) >> shift) & (bins - 1)], 1u);
    __syncthreads();
    // Exclusive sums over this CTA's warps, per bin.
    for (int b = tid; b < bins; b += kSortThreads) {
      unsigned s = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = hist[w * bins + b];
        hist[w * bins + b] = s;
        s += c;
      }
      total[b] = s;
    }
    cluster_sync();  // every CTA's totals are there
    // Where this CTA's elements of bin `tid` go: all smaller bins, then the CTAs before it.
    unsigned all = 0, before = 0;
    if (tid < bins) {
#pragma unroll
      for (unsigned r = 0; r < kSortCluster; ++r) {
        const unsigned c = ld_dsmem(total + tid, r);
        before += r < rank ? c : 0u;
        all += c;
      }
    }
    unsigned incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    unsigned base = incl - all + before;
    for (int w = 0; w < warp; ++w) base += warp_sum[w];
    if (tid < bins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) hist[w * bins + tid] += base;
    }
    __syncthreads();
    // Stable scatter: 32 consecutive elements at a time, equal digits in lane order.
    for (long long g = first; g < last; g += 32) {
      const long long i = g + lane;
      const bool ok = i < last;
      const unsigned key = ok ? load_key(i) : 0u;
      const unsigned p = ok ? (pass > 0 ? __ldcg(psrc + i) : static_cast<unsigned>(i)) : 0u;
      const unsigned d = ok ? (key >> shift) & (bins - 1) : static_cast<unsigned>(bins);  // no element: its own class
      const unsigned peers = __match_any_sync(0xffffffffu, d);
      const unsigned rank_in = __popc(peers & ((1u << lane) - 1u));
      unsigned at = 0;
      if (ok) at = mine[d] + rank_in;
      __syncwarp();
      if (ok && rank_in == 0) mine[d] += __popc(peers);
      __syncwarp();
      if (ok) {
        __stcg(kdst + at, key);
        __stcg(pdst + at, p);
      }
    }
    cluster_sync();  // the sorted list of this pass is written; `total` may be overwritten
  }
}

// ------------------------------------------------------------------------------------
// Gradient, 2 and 3: sums over runs of equal tokens
// ------------------------------------------------------------------------------------

constexpr int kSumThreads = 128;
constexpr int kAhead = 8;  // rows whose loads are in flight at once

struct SumArgs {
  int n, vocab, dim, chunk, chunks;
  const unsigned *key, *pos;  // sorted
  float scale;
  float* head;  // [chunks][dim]: sum of the chunk's first run, if that began in an earlier chunk
  float* tail;  // [chunks][dim]: sum of the run that began in the chunk and goes on after it
};

// 16 bytes, or one element, as loaded: converted only when it is used, so that all loads
// of a batch of rows are issued before the first wait.
template <typename T, bool VEC>
struct Raw {
  static constexpr int E = VEC ? 16 / sizeof(T) : 1;
  alignas(VEC ? 16 : sizeof(T)) T v[E];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    else v[0] = *p;
  }
  __device__ __forceinline__ void add_to(float (&acc)[E]) const {
    float x[E];
    load_vec<T, E>(v, x);
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] += x[k];
  }
};

// One chunk (blockIdx.x) x one tile of kSumThreads * E columns (blockIdx.y).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumThreads) embed_sum_kernel(const SumArgs a, const T* __restrict__ dy,
                                                                T* __restrict__ dw) {
  constexpr int E = VEC ? 16 / sizeof(T) : 1;
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * E;
  const int j0 = blockIdx.x * a.chunk, j1 = min(j0 + a.chunk, a.n);
  const unsigned vocab = static_cast<unsigned>(a.vocab);
  if (col >= a.dim || a.key[j0] == vocab) return;
  bool from_before = j0 > 0 && a.key[j0 - 1] == a.key[j0];
  float acc[E];
#pragma unroll
  for (int k = 0; k < E; ++k) acc[k] = 0.f;
  for (int j = j0; j < j1; j += kAhead) {
    unsigned key[kAhead + 1];
    Raw<T, VEC> v[kAhead];
#pragma unroll
    for (int u = 0; u <= kAhead; ++u) key[u] = j + u < a.n ? a.key[j + u] : vocab;
    // Entries past the chunk or without a gradient load some row of dy all the same: a
    // load under a condition would wait for the one before it.
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u].load(dy + static_cast<long long>(a.pos[min(j + u, a.n - 1)]) * a.dim + col);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u >= j1 || key[u] == vocab) continue;
      v[u].add_to(acc);
      const bool ends = key[u + 1] != key[u];  // the list's end counts as another key
      if (!ends && j + u + 1 < j1) continue;
      if (from_before) {
        store_vec<float, E>(a.head + static_cast<long long>(blockIdx.x) * a.dim + col, acc);
      } else if (!ends) {
        store_vec<float, E>(a.tail + static_cast<long long>(blockIdx.x) * a.dim + col, acc);
      } else {
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] *= a.scale;
        store_vec<T, E>(dw + static_cast<long long>(key[u]) * a.dim + col, acc);
      }
      from_before = false;
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] = 0.f;
    }
  }
}

// Partial sums [p0, p1) of the run that begins in chunk c0, in order: number 0 is c0's
// tail, number q > 0 the head of chunk c0 + q.
template <int E>
__device__ __forceinline__ void add_parts(const SumArgs& a, int c0, int p0, int p1, int col, float (&acc)[E]) {
  for (int p = p0; p < p1; p += 4) {
    alignas(16) float x[4][E];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int q = min(p + u, p1 - 1);
      const float* src = (q == 0 ? a.tail : a.head) + static_cast<long long>(c0 + q) * a.dim + col;
      load_vec<float, E>(src, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (p + u < p1)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += x[u][k];
  }
}

// The runs that begin in one of the kJoinWarps chunks of blockIdx.x and go on after it, one
// tile of 32 * E columns (blockIdx.y). Each warp looks at its chunk's run and adds it up if
// it spans a few chunks; the block adds up the longer ones together, each warp a stretch of
// the run, the warps' sums in order.
constexpr int kJoinWarps = 8;
constexpr int kJoinAlone = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kJoinWarps) embed_join_kernel(const SumArgs a, T* __restrict__ dw) {
  constexpr int E = VEC ? 16 / sizeof(T) : 1;
  __shared__ float parts[kJoinWarps][32 * E];
  __shared__ int spans[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * E;
  const bool ok = col < a.dim;
  auto finish = [&](unsigned key, float (&acc)[E]) {
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] *= a.scale;
    store_vec<T, E>(dw + static_cast<long long>(key) * a.dim + col, acc);
  };
  // Chunks that the run of this warp's chunk spans; 0 where none begins here and goes on.
  const int c = blockIdx.x * kJoinWarps + warp;
  int span = 0;
  if (c + 1 < a.chunks) {
    const int j0 = c * a.chunk, next = j0 + a.chunk;
    const unsigned key = a.key[next - 1];
    if (key != static_cast<unsigned>(a.vocab) && a.key[next] == key && (j0 == 0 || a.key[j0 - 1] != key)) {
      // Whether the run fills chunk c + 1 + l and reaches the next, 32 chunks at a time.
      for (span = 1;; span += 32) {
        const long long after = static_cast<long long>(c + span + lane + 1) * a.chunk;
        const unsigned on = __ballot_sync(0xffffffffu, after < a.n && a.key[after] == key);
        if (on != 0xffffffffu) {
          span += __ffs(~on);
          break;
        }
      }
    }
  }
  if (lane == 0) spans[warp] = span;
  if (span > 0 && span <= kJoinAlone && ok) {
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    add_parts<E>(a, c, 0, span, col, acc);
    finish(a.key[c * a.chunk + a.chunk - 1], acc);
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    const int n = spans[w], c0 = blockIdx.x * kJoinWarps + w;
    if (n <= kJoinAlone) continue;
    const int per = (n + kJoinWarps - 1) / kJoinWarps, p0 = min(warp * per, n), p1 = min(p0 + per, n);
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    if (ok) add_parts<E>(a, c0, p0, p1, col, acc);
#pragma unroll
    for (int k = 0; k < E; ++k) parts[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    if (warp == 0 && ok) {
#pragma unroll
      for (int g = 1; g < kJoinWarps; ++g)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += parts[g][k * 32 + lane];
      finish(a.key[c0 * a.chunk + a.chunk - 1], acc);
    }
    __syncthreads();
  }
}

// Sorted entries per chunk: small enough that the chunks of a short list still fill the
// GPU, and from 32 on larger only for long lists: long runs leave at most two fp32 rows of
// partial sums a chunk, a small part of the chunk's own 32 rows, and the join of a run
// reads them all (500000 tokens with a run of 52800, dim 64: sums and join 85 us in chunks
// of 32, 66 us of 128).
int embed_chunk(int n) {
  int c = 8;
  while (c < 32 && n / c > 4 * 148) c *= 2;
  while (c >= 32 && c < 128 && n / c > 32 * 148) c *= 2;
  return c;
}

long long round16(long long v) { return (v + 15) / 16 * 16; }

}  // namespace

long long embed_scratch_bytes(int n, int dim) {
  const long long chunks = (n + embed_chunk(n) - 1) / embed_chunk(n);
  return 4 * round16(4ll * n) + 2 * round16(4 * chunks * dim);
}

int launch_embed_lookup(bool bf16, long long n, int vocab, int dim, const long long* tokens, const void* w,
                        float scale, long long skip, float oob, void* y, cudaStream_t stream) {
  const int e = bf16 ? 8 : 4;
  const bool vec = dim % e == 0 && vec_aligned(w) && vec_aligned(y);
  const int per_row = vec ? dim / e : dim;
  // Threads per token: enough for one 16-byte access each, or the whole block.
  int lg = 0;
  while ((1 << lg) < per_row && (1 << lg) < kLookupThreads) ++lg;
  const int rows = (kLookupThreads >> lg) * kLookupRows;
  const unsigned grid = static_cast<unsigned>((n + rows - 1) / rows);
#define FH_LOOKUP(T, V)                                                                                           \
  embed_lookup_kernel<T, V><<<grid, kLookupThreads, 0, stream>>>(n, vocab, dim, lg, tokens, static_cast<const T*>(w), \
                                                                 scale, skip, oob, static_cast<T*>(y))
  if (bf16 && vec) FH_LOOKUP(__nv_bfloat16, true);
  else if (bf16) FH_LOOKUP(__nv_bfloat16, false);
  else if (vec) FH_LOOKUP(float, true);
  else FH_LOOKUP(float, false);
#undef FH_LOOKUP
  return after_launch();
}

int launch_embed_grad(bool bf16, int n, int vocab, int dim, const long long* tokens, const void* dy, float scale,
                      long long padding, void* dw, void* scratch, cudaStream_t stream) {
  const int size = bf16 ? 2 : 4;
  uint8_t* s = static_cast<uint8_t*>(scratch);
  SortArgs so{};
  so.n = n;
  so.vocab = vocab;
  so.padding = padding;
  so.tokens = tokens;
  for (int i = 0; i < 2; ++i) {
    so.key[i] = reinterpret_cast<unsigned*>(s);
    so.pos[i] = reinterpret_cast<unsigned*>(s + round16(4ll * n));
    s += 2 * round16(4ll * n);
  }
  int bits = 1;
  while (bits < 31 && (vocab >> bits) != 0) ++bits;  // keys are 0 .. vocab
  so.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  so.bits = (bits + so.passes - 1) / so.passes;
  const long long bytes = static_cast<long long>(vocab) * dim * size;
  so.fill = static_cast<uint4*>(dw);
  so.fill_vecs = bytes / 16;
  so.fill_tail = reinterpret_cast<unsigned short*>(static_cast<uint8_t*>(dw) + so.fill_vecs * 16);
  so.tail_halves = static_cast<int>((bytes - so.fill_vecs * 16) / 2);
  const int smem = (kSortWarps + 1) * (1 << so.bits) * 4;
  if (ensure_smem_limit(reinterpret_cast<const void*>(&embed_sort_kernel),
                        (kSortWarps + 1) * (1 << kMaxDigitBits) * 4) != kOk)
    return kLaunchFailed;
  // CTAs that fill: two per SM, or fewer when there is little to fill. (With one per SM
  // the clusters of a GPC share its SMs unevenly: 98 MB took 26 us.) At digits of 10 bits
  // (tables of 512 to 1023 rows and of 2^18 to 2^20, say) the launch's shared memory, 135 KB
  // for the filling CTAs too, leaves room for one on an SM: they run one after the other.
  const long long want = (so.fill_vecs + 8ll * kSortThreads - 1) / (8ll * kSortThreads) + 1;
  const long long most = 2 * sm_count() - kSortCluster;
  const long long ctas = want < most ? want : most;
  const unsigned grid = static_cast<unsigned>(kSortCluster * (1 + (ctas + kSortCluster - 1) / kSortCluster));
  embed_sort_kernel<<<grid, kSortThreads, smem, stream>>>(so);
  if (after_launch() != kOk) return kLaunchFailed;
  if (n == 0) return kOk;  // the zeros are the gradient
  SumArgs su{};
  su.n = n;
  su.vocab = vocab;
  su.dim = dim;
  su.chunk = embed_chunk(n);
  su.chunks = (n + su.chunk - 1) / su.chunk;
  su.key = so.key[so.passes & 1];
  su.pos = so.pos[so.passes & 1];
  su.scale = scale;
  su.head = reinterpret_cast<float*>(s);
  su.tail = reinterpret_cast<float*>(s + round16(4ll * su.chunks * dim));
  const int e = 16 / size;
  const bool vec = dim % e == 0 && vec_aligned(dy) && vec_aligned(dw);
  const int cols = kSumThreads * (vec ? e : 1);
  const dim3 g(su.chunks, (dim + cols - 1) / cols);
  const int join_cols = 32 * (vec ? e : 1);
  const dim3 gj((su.chunks + kJoinWarps - 1) / kJoinWarps, (dim + join_cols - 1) / join_cols);
#define FH_SUM(T, V)                                                                                              \
  do {                                                                                                            \
    embed_sum_kernel<T, V><<<g, kSumThreads, 0, stream>>>(su, static_cast<const T*>(dy), static_cast<T*>(dw));    \
    if (after_launch() != kOk) return kLaunchFailed;                                                              \
    if (su.chunks > 1) {                                                                                          \
      embed_join_kernel<T, V><<<gj, 32 * kJoinWarps, 0, stream>>>(su, static_cast<T*>(dw));                            \
      return after_launch();                                                                                      \
    }                                                                                                             \
    return kOk;                                                                                                   \
  } while (0)
  if (bf16 && vec) FH_SUM(__nv_bfloat16, true);
  else if (bf16) FH_SUM(__nv_bfloat16, false);
  else if (vec) FH_SUM(float, true);
  else FH_SUM(float, false);
#undef FH_SUM
}

}  // namespace fh
