// Attention forward of a few query rows over a window with sinks: single tokens on long
// key/value tensors.
//
//   O = softmax(scale Q K^T + mask) V,  L = log-sum-exp
//
// The tile kernel (fwd.cu) gives a CTA 128 query rows of one head; with one row, 127 of its
// rows are idle, and a CTA walks all key tiles of its head by itself. Here a CTA takes the
// rows of all query heads of one key head (grouped heads read their keys once), up to 16,
// and a cluster of CTAs shares the visible keys: a few hundred KB per key head, bound by
// memory and, at these sizes, by latency. (16 sequences x 16 heads, 4 key heads, head_dim 64,
// window 1024 of 8192 keys, 4 sinks: 22 us in the tile kernel, 8.4 us here, 2.6 us at the
// copy rate; 64 sequences: 74, 17 and 10 us.)
//
// The visible keys of the CTA's rows are one list: the sinks, then the window's. Each CTA
// takes a stretch of it, each warp 16 keys at a time with its own running maximum, sum and
// output (online softmax), so the loop over the keys has no barrier: a warp copies its own
// keys ahead (cp.async) and waits for them alone. Sixteen rows are one m16n8k16 product
// (mma.sync: a 128-row tcgen05 tile would be an eighth full at best, and the time is the
// keys' way here). P enters the second product as two bf16 parts, hi + lo, so that its
// rounding (2^-17) does not count. The warps and the cluster's CTAs are joined once at the
// end, in a fixed order.

#include <cuda_runtime.h>

#include <cmath>

#include "kernels.h"

namespace fh {
namespace {

constexpr int kFewThreads = 128;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewCluster = 8;    // CTAs that share a key head's keys, at most
constexpr int kFewKeys = 16;      // keys a warp takes at once
constexpr int kFewStep = kFewWarps * kFewKeys;

template <int HD>
constexpr int kFewStages = HD == 64 ? 4 : 3;  // batches of keys in shared memory: 64 or 96 KB, two CTAs per SM
template <int HD>
constexpr int kFewSmem = kFewStages<HD> * 2 * kFewStep * HD * 2;

struct FewArgs {
  SinkShape sh;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  float* lse;
  int splits;  // CTAs per (batch, key head): the cluster
};

__device__ __forceinline__ void few_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float few_remote(const float* p, unsigned rank) {
  unsigned a = static_cast<unsigned>(__cvta_generic_to_shared(p)), ra;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra) : "memory");
  return v;
}

// 16 bytes to shared memory; zeros where `ok` is false.
__device__ __forceinline__ void few_copy(uint32_t dst, const __nv_bfloat16* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// c (16 x 8) += a (16 x 16) b (16 x 8)
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^(a - b) for running maxima in the log2 domain: 0 from -inf, whatever b.
__device__ __forceinline__ float few_scale(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

// Grid (splits, key heads, batch), clusters of (splits, 1, 1).
template <int HD, bool VL>
__global__ void __launch_bounds__(kFewThreads, 2) fwd_few_kernel(const FewArgs a) {
  constexpr int ST = kFewStages<HD>, CH = HD / 8, KS = HD / 16;  // 16-byte chunks and k-steps of a row
  constexpr int TILE = kFewKeys * HD * 2;                        // a warp's keys: K, then V
  extern __shared__ __align__(128) uint8_t s_stage[];            // [stage][warp][K | V]
  __shared__ float s_m[kFewWarps][kFewRows], s_l[kFewWarps][kFewRows];
  __shared__ float s_out[kFewRows][HD], s_outm[kFewRows], s_outl[kFewRows];  // this CTA's share, read by the cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hk = blockIdx.y, b = blockIdx.z, split = blockIdx.x;
  SeqRange sr;
  const SinkShape sh = seq_shape<VL>(a.sh, b, &sr);
  const int rows = sh.Tq * sh.G;  // row r: token r / G, head hk G + r % G
  const float sc2 = sh.scale * kLog2e;
  // The list of visible keys: `front` sinks, then keys lo, lo + 1, ..., hi.
  int lo = 0, hi = -1, front = 0;
  if (rows > 0) {
    lo = key_lo(sh, 0);
    hi = key_hi(sh, sh.Tq - 1);
    front = max(0, min(min(sh.sinks, lo), hi + 1));
    if (sh.sinks >= lo) lo = front = 0;  // one run
  }
  const int total = front + max(0, hi - lo + 1);
  const int p0 = static_cast<int>(static_cast<long long>(total) * split / a.splits);
  const int p1 = static_cast<int>(static_cast<long long>(total) * (split + 1) / a.splits);
  auto key_of = [&](int p) { return p < front ? p : lo + p - front; };
  const int batches = (p1 - p0 + kFewStep - 1) / kFewStep;
  const uint32_t mine = smem_u32(s_stage) + warp * 2 * TILE;
  constexpr uint32_t kStage = kFewWarps * 2 * TILE;
  auto first_of = [&](int it) { return p0 + (it * kFewWarps + warp) * kFewKeys; };  // list position of the warp's batch
  auto chunk_at = [](int key, int c) { return static_cast<uint32_t>(key * (HD * 2) + ((c ^ (key & 7)) << 4)); };
  auto fetch = [&](int it) {
    if (it < batches) {
      const uint32_t to = mine + (it % ST) * kStage;
#pragma unroll
      for (int u = 0; u < kFewKeys * CH / 32; ++u) {
        const int i = u * 32 + lane, key = i / CH, c = i % CH, at = first_of(it) + key;
        const bool ok = at < p1;
        const size_t off = k_row(sh, sr, ok ? key_of(at) : 0, hk) + c * 8;
        few_copy(to + chunk_at(key, c), a.k + off, ok);
        few_copy(to + TILE + chunk_at(key, c), a.v + off, ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // an empty group keeps the count
  };
#pragma unroll
  for (int it = 0; it < ST - 1; ++it) fetch(it);
  // Q as the left operand: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) and 8 further.
  const int r0 = lane >> 2, pair = (lane & 3) * 2;
  uint32_t qf[KS][4];
  int khi[2], klo[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = r0 + 8 * half;
    const bool ok = r < rows;
    const int t = ok ? r / sh.G : 0;
    khi[half] = ok ? key_hi(sh, t) : -1;
    klo[half] = ok ? key_lo(sh, t) : 0;
    const __nv_bfloat16* src = a.q + (ok ? q_row(sh, sr, t, hk * sh.G + r % sh.G) : 0) + pair;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks][half] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
      qf[ks][half + 2] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
    }
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[CH][4];
#pragma unroll
  for (int n = 0; n < CH; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  for (int it = 0; it < batches; ++it) {
    fetch(it + ST - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
    __syncwarp();  // the other lanes' copies of this batch
    const uint32_t kb = mine + (it % ST) * kStage, vb = kb + TILE;
    const int first = first_of(it);
    float s[2][4] = {};  // keys 0-7 and 8-15
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t bk[4];
      ldmatrix4(bk, kb + chunk_at((lane >> 4) * 8 + (lane & 7), 2 * ks + ((lane >> 3) & 1)));
      mma16816(s[0], qf[ks], bk[0], bk[1]);
      mma16816(s[1], qf[ks], bk[2], bk[3]);
    }
    uint32_t hi_part[4], lo_part[4];  // P as the left operand of P V
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float top = m[half];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = first + j * 8 + pair + e, key = key_of(at);
          float& x = s[j][half * 2 + e];
          x = at < p1 && key <= khi[half] && (key >= klo[half] || key < sh.sinks) ? x * sc2 : -INFINITY;
          top = fmaxf(top, x);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float f = few_scale(m[half], top), base = top == -INFINITY ? 0.f : top;
      m[half] = top;
      l[half] *= f;
#pragma unroll
      for (int n = 0; n < CH; ++n) {
        o[n][half * 2] *= f;
        o[n][half * 2 + 1] *= f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = ex2(s[j][half * 2] - base), y = ex2(s[j][half * 2 + 1] - base);
        l[half] += x + y;
        const uint32_t h = pack_bf16(x, y);
        hi_part[half + 2 * j] = h;
        lo_part[half + 2 * j] = pack_bf16(x - __uint_as_float(h << 16), y - __uint_as_float(h & 0xffff0000u));
      }
    }
#pragma unroll
    for (int n = 0; n < CH; n += 2) {
      uint32_t bv[4];
      ldmatrix4_trans(bv, vb + chunk_at(((lane >> 3) & 1) * 8 + (lane & 7), n + (lane >> 4)));
      mma16816(o[n], hi_part, bv[0], bv[1]);
      mma16816(o[n], lo_part, bv[0], bv[1]);
      mma16816(o[n + 1], hi_part, bv[2], bv[3]);
      mma16816(o[n + 1], lo_part, bv[2], bv[3]);
    }
    __syncwarp();  // every lane has read the batch that the next fetch overwrites
  }
  // The warps, then the CTAs of the cluster. The warps' outputs take the place of the keys.
  float(*s_part)[kFewRows][HD + 2] = reinterpret_cast<float(*)[kFewRows][HD + 2]>(s_stage);
  static_assert(kFewWarps * kFewRows * (HD + 2) * 4 <= kFewSmem<HD>, "the warps' outputs fit");
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = r0 + 8 * half;
    float sum = l[half];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if ((lane & 3) == 0) {
      s_m[warp][r] = m[half];
      s_l[warp][r] = sum;
    }
#pragma unroll
    for (int n = 0; n < CH; ++n)
      *reinterpret_cast<float2*>(&s_part[warp][r][n * 8 + pair]) = make_float2(o[n][half * 2], o[n][half * 2 + 1]);
  }
  __syncthreads();
  for (int i = tid; i < rows * HD; i += kFewThreads) {
    const int r = i / HD, d = i - r * HD;
    float to = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kFewWarps; ++w) to = fmaxf(to, s_m[w][r]);
    float x = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float f = few_scale(s_m[w][r], to);
      x += s_part[w][r][d] * f;
      sum += s_l[w][r] * f;
    }
    s_out[r][d] = x;
    if (d == 0) {
      s_outm[r] = to;
      s_outl[r] = sum;
    }
  }
  if (a.splits > 1) few_cluster_sync();
  else __syncthreads();
  // The CTAs of the cluster share the outputs.
  for (int i = split * kFewThreads + tid; i < rows * HD; i += a.splits * kFewThreads) {
    const int r = i / HD, d = i - r * HD;
    float cm[kFewCluster], cl[kFewCluster], cx[kFewCluster];  // all loads before the first use
#pragma unroll
    for (int c = 0; c < kFewCluster; ++c) {
      cm[c] = -INFINITY;
      cl[c] = cx[c] = 0.f;
      if (c >= a.splits) continue;
      cm[c] = a.splits > 1 ? few_remote(&s_outm[r], c) : s_outm[r];
      cl[c] = a.splits > 1 ? few_remote(&s_outl[r], c) : s_outl[r];
      cx[c] = a.splits > 1 ? few_remote(&s_out[r][d], c) : s_out[r][d];
    }
    float to = cm[0];
#pragma unroll
    for (int c = 1; c < kFewCluster; ++c) to = fmaxf(to, cm[c]);
    float x = 0.f, sum = 0.f;
#pragma unroll
    for (int c = 0; c < kFewCluster; ++c) {
      const float f = few_scale(cm[c], to);
      x += cx[c] * f;
      sum += cl[c] * f;
    }
    const int t = r / sh.G, h = hk * sh.G + r % sh.G;
    a.o[q_row(sh, sr, t, h) + d] = __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);  // no visible key: 0
    if (d == 0) a.lse[q_stat(sh, sr, t, h)] = (to + log2f(sum)) * kLn2;
  }
  if (a.splits > 1) few_cluster_sync();  // the others have read this CTA's share
}

template <int HD, bool VL>
int launch_few(const FewArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.splits, a.sh.Hk, a.sh.B);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = kFewSmem<HD>;
  if (ensure_smem_limit(reinterpret_cast<const void*>(&fwd_few_kernel<HD, VL>), kFewSmem<HD>) != kOk)
    return kLaunchFailed;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.splits > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, fwd_few_kernel<HD, VL>, a) != cudaSuccess) {
    cudaGetLastError();
    return kLaunchFailed;
  }
  return after_launch();
}

}  // namespace

// With sinks only: a token under a plain window would have the same list of keys and the same
// gain, but keeps the tile kernel, whose results such calls have always had bit for bit.
bool fwd_few_applies(const SinkShape& s) {
  return s.sinks > 0 && static_cast<long long>(s.Tq) * s.G <= kFewRows && s.Hk <= 65535 && s.B <= 65535;
}

int launch_fwd_few(const SinkShape& s, int hd, const FwdPtrs& p, cudaStream_t stream) {
  // As many CTAs per key head as are resident at once, each with 64 keys at least: a CTA is
  // mostly latency, and a second wave doubles it.
  const long long pairs = static_cast<long long>(s.Hk) * s.B;
  const long long keys = static_cast<long long>(s.sinks < s.Tk ? s.sinks : s.Tk) + (s.window < s.Tk ? s.window : s.Tk);
  int splits = 1;
  while (splits < kFewCluster && 2 * splits * pairs <= 2 * 148 && keys / (2 * splits) >= kFewStep) splits *= 2;
  const FewArgs a{s,
                  static_cast<const __nv_bfloat16*>(p.q),
                  static_cast<const __nv_bfloat16*>(p.k),
                  static_cast<const __nv_bfloat16*>(p.v),
                  static_cast<__nv_bfloat16*>(p.o),
                  p.lse,
                  splits};
  if (hd == 64) return s.cu_q ? launch_few<64, true>(a, stream) : launch_few<64, false>(a, stream);
  return s.cu_q ? launch_few<128, true>(a, stream) : launch_few<128, false>(a, stream);
}

}  // namespace fh
