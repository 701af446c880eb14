// Attention forward of a few query rows over a window with sinks: single tokens on long
// key/value tensors.
//
//   O = softmax(scale Q K^T + mask) V,  L = log-sum-exp
//
// The tile kernel (fwd.cu) gives a CTA 128 query rows of one head; with one row, 127 of its
// rows are idle, and a CTA walks all key tiles of its head by itself. Here a CTA takes the
// rows of all query heads of one key head (grouped heads read their keys once), the products
// run on the CUDA cores in fp32, and a cluster of CTAs shares the visible keys: a few
// hundred KB per key head, bound by memory and, at these sizes, by latency. (16 sequences x
// 16 heads x 8192 keys, 4 key heads, head_dim 64, window 1024, 4 sinks: 22 us in the tile
// kernel, 7.5 us here.)
//
// The visible keys of the CTA's rows are one list: the sinks, then the window's. Each CTA
// takes a stretch of it; in a CTA, HD / 8 lanes form a group that takes every 256 / (HD / 8)-th
// key, 16 bytes of its row a lane. A group keeps its own running maximum, sum and output
// (online softmax), so the loop over the keys has no barrier; the groups, the warps and the
// cluster's CTAs are joined once at the end, in a fixed order.

#include <cuda_runtime.h>

#include <cmath>

#include "kernels.h"
#include "vec_io.cuh"

namespace fh {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewRows = 8;       // query rows (tokens x heads of a group) a CTA can take
constexpr int kFewCluster = 8;    // CTAs that share a key head's keys, at most
constexpr int kFewAhead = 4;      // keys a group takes at once
constexpr int kFewStages = 3;     // batches of them in shared memory
constexpr int kFewSmem = kFewStages * 2 * kFewAhead * kFewThreads * 16;

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

__device__ __forceinline__ void few_copy(uint4* dst, const __nv_bfloat16* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// 2^(a - b) for running maxima in the log2 domain: 0 from -inf, whatever b.
__device__ __forceinline__ float few_scale(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

// RM: the rows, rounded up to 1, 4 or 8. Grid (splits, key heads, batch), clusters of
// (splits, 1, 1).
template <int HD, int RM, bool VL>
__global__ void __launch_bounds__(kFewThreads, RM == 8 ? 1 : 2) fwd_few_kernel(const FewArgs a) {
  constexpr int LPR = HD / 8;                  // lanes per key row
  constexpr int GROUPS = kFewThreads / LPR;    // keys in flight per step of the CTA
  __shared__ alignas(16) float s_q[RM][HD];
  __shared__ float s_part[kFewWarps][RM][HD], s_m[kFewWarps][RM], s_l[kFewWarps][RM];
  __shared__ float s_out[RM][HD], s_outm[RM], s_outl[RM];  // this CTA's share, read by the cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hk = blockIdx.y, b = blockIdx.z, split = blockIdx.x;
  SeqRange sr;
  const SinkShape sh = seq_shape<VL>(a.sh, b, &sr);
  const int rows = sh.Tq * sh.G;  // row r: token r / G, head hk G + r % G
  const float sc2 = sh.scale * kLog2e;
  for (int i = tid; i < RM * HD; i += kFewThreads) {
    const int r = i / HD, d = i - r * HD;
    s_q[r][d] = r < rows ? __bfloat162float(a.q[q_row(sh, sr, r / sh.G, hk * sh.G + r % sh.G) + d]) * sc2 : 0.f;
  }
  // The list of visible keys: `front` sinks, then keys lo, lo + 1, ..., hi.
  int lo = 0, hi = -1, front = 0;
  if (rows > 0) {
    lo = key_lo(sh, 0);
    hi = key_hi(sh, sh.Tq - 1);
    front = min(min(sh.sinks, lo), hi + 1);
    if (front < 0) front = 0;
    if (sh.sinks >= lo) lo = front = 0;  // one run
  }
  const int total = front + max(0, hi - lo + 1);
  const int p0 = static_cast<int>(static_cast<long long>(total) * split / a.splits);
  const int p1 = static_cast<int>(static_cast<long long>(total) * (split + 1) / a.splits);
  auto key_of = [&](int p) { return p < front ? p : lo + p - front; };
  int khi[RM], klo[RM];  // visible keys of each row
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int t = r / sh.G;
    khi[r] = r < rows ? key_hi(sh, t) : -1;
    klo[r] = r < rows ? key_lo(sh, t) : 0;
  }
  __syncthreads();
  const int group = tid / LPR, part = tid % LPR;
  float m[RM], l[RM], acc[RM][8];
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[r][e] = 0.f;
  }
  // Batches of kFewAhead keys a group, kFewStages - 1 of them on their way at once. A lane
  // stages its own 16 bytes of each key in shared memory and reads them back itself, so the
  // copies need no barrier, only its own wait.
  extern __shared__ uint4 s_stage[];  // [stage][K | V][kFewAhead][thread]
  const int batches = (p1 - p0 + GROUPS * kFewAhead - 1) / (GROUPS * kFewAhead);
  auto stage = [&](int it, int matrix, int u) {
    return s_stage + (((it % kFewStages) * 2 + matrix) * kFewAhead + u) * kFewThreads + tid;
  };
  auto key_at = [&](int it, int u) {  // -1 past this CTA's keys
    const int at = p0 + (it * kFewAhead + u) * GROUPS + group;
    return at < p1 ? key_of(at) : -1;
  };
  auto fetch = [&](int it) {
    if (it < batches) {
#pragma unroll
      for (int u = 0; u < kFewAhead; ++u) {
        const int key = key_at(it, u);
        const size_t off = k_row(sh, sr, key < 0 ? key_of(p0) : key, hk) + part * 8;
        few_copy(stage(it, 0, u), a.k + off);
        few_copy(stage(it, 1, u), a.v + off);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // an empty group keeps the count
  };
#pragma unroll
  for (int it = 0; it < kFewStages - 1; ++it) fetch(it);
  for (int it = 0; it < batches; ++it) {
    fetch(it + kFewStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 1) : "memory");
    int key[kFewAhead];
    uint4 kr[kFewAhead];
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      key[u] = key_at(it, u);
      kr[u] = *stage(it, 0, u);
    }
    float s[RM][kFewAhead];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const float4 q0 = *reinterpret_cast<const float4*>(&s_q[r][part * 8]);
      const float4 q1 = *reinterpret_cast<const float4*>(&s_q[r][part * 8 + 4]);
#pragma unroll
      for (int u = 0; u < kFewAhead; ++u) {
        float x[8];
        load_vec<__nv_bfloat16, 8>(reinterpret_cast<const __nv_bfloat16*>(&kr[u]), x);
        s[r][u] = fmaf(x[0], q0.x, fmaf(x[1], q0.y, fmaf(x[2], q0.z, x[3] * q0.w))) +
                  fmaf(x[4], q1.x, fmaf(x[5], q1.y, fmaf(x[6], q1.z, x[7] * q1.w)));
      }
    }
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1)
#pragma unroll
      for (int r = 0; r < RM; ++r)
#pragma unroll
        for (int u = 0; u < kFewAhead; ++u) s[r][u] += __shfl_xor_sync(0xffffffffu, s[r][u], o);
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      float top = m[r];
#pragma unroll
      for (int u = 0; u < kFewAhead; ++u) {
        const bool seen = key[u] >= 0 && key[u] <= khi[r] && (key[u] >= klo[r] || key[u] < sh.sinks);
        if (!seen) s[r][u] = -INFINITY;
        top = fmaxf(top, s[r][u]);
      }
      const float f = few_scale(m[r], top), base = top == -INFINITY ? 0.f : top;
      m[r] = top;
      l[r] *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] *= f;
#pragma unroll
      for (int u = 0; u < kFewAhead; ++u) {
        s[r][u] = ex2(s[r][u] - base);
        l[r] += s[r][u];
      }
    }
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      float x[8];
      load_vec<__nv_bfloat16, 8>(reinterpret_cast<const __nv_bfloat16*>(stage(it, 1, u)), x);
      // A key that is not there was loaded from another place and may be anything: 0 x NaN.
      if (key[u] < 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll
      for (int r = 0; r < RM; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(s[r][u], x[e], acc[r][e]);
    }
  }
  // The groups of a warp, then the warps, then the CTAs of the cluster.
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const float om = __shfl_xor_sync(0xffffffffu, m[r], o), ol = __shfl_xor_sync(0xffffffffu, l[r], o);
      const float to = fmaxf(m[r], om), f = few_scale(m[r], to), of = few_scale(om, to);
      l[r] = l[r] * f + ol * of;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        acc[r][e] = acc[r][e] * f + __shfl_xor_sync(0xffffffffu, acc[r][e], o) * of;
      m[r] = to;
    }
  if (lane < LPR)
#pragma unroll
    for (int r = 0; r < RM; ++r) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s_part[warp][r][part * 8 + e] = acc[r][e];
      if (lane == 0) {
        s_m[warp][r] = m[r];
        s_l[warp][r] = l[r];
      }
    }
  __syncthreads();
  for (int i = tid; i < RM * HD; i += kFewThreads) {
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
    a.o[q_row(sh, sr, t, h) + d] = __float2bfloat16_rn(sum > 0.f ? x / sum : 0.f);  // no visible key: 0
    if (d == 0) a.lse[q_stat(sh, sr, t, h)] = (to + log2f(sum)) * kLn2;
  }
  if (a.splits > 1) few_cluster_sync();  // the others have read this CTA's share
}

template <int HD, int RM, bool VL>
int launch_few(const FewArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.splits, a.sh.Hk, a.sh.B);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = kFewSmem;
  if (ensure_smem_limit(reinterpret_cast<const void*>(&fwd_few_kernel<HD, RM, VL>), kFewSmem) != kOk)
    return kLaunchFailed;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.splits > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, fwd_few_kernel<HD, RM, VL>, a) != cudaSuccess) {
    cudaGetLastError();
    return kLaunchFailed;
  }
  return after_launch();
}

}  // namespace

bool fwd_few_applies(const SinkShape& s) {
  return s.sinks > 0 && static_cast<long long>(s.Tq) * s.G <= kFewRows && s.Hk <= 65535 && s.B <= 65535;
}

int launch_fwd_few(const SinkShape& s, int hd, const FwdPtrs& p, cudaStream_t stream) {
  // As many CTAs per key head as are resident at once, each with 64 keys at least: a CTA is
  // mostly latency, and a second wave doubles it.
  const long long pairs = static_cast<long long>(s.Hk) * s.B;
  const long long keys = static_cast<long long>(s.sinks < s.Tk ? s.sinks : s.Tk) + (s.window < s.Tk ? s.window : s.Tk);
  const int rows = s.Tq * s.G;
  const long long resident = (rows > 4 ? 1 : 2) * 148;
  int splits = 1;
  while (splits < kFewCluster && 2 * splits * pairs <= resident && keys / (2 * splits) >= 64) splits *= 2;
  const FewArgs a{s,
                  static_cast<const __nv_bfloat16*>(p.q),
                  static_cast<const __nv_bfloat16*>(p.k),
                  static_cast<const __nv_bfloat16*>(p.v),
                  static_cast<__nv_bfloat16*>(p.o),
                  p.lse,
                  splits};
  auto run = [&](auto hd_tag, auto vl_tag) {
    constexpr int HD = decltype(hd_tag)::value;
    constexpr bool VL = decltype(vl_tag)::value;
    return rows == 1 ? launch_few<HD, 1, VL>(a, stream)
                     : rows <= 4 ? launch_few<HD, 4, VL>(a, stream) : launch_few<HD, 8, VL>(a, stream);
  };
  using I64 = std::integral_constant<int, 64>;
  using I128 = std::integral_constant<int, 128>;
  if (hd == 64) return s.cu_q ? run(I64{}, std::true_type{}) : run(I64{}, std::false_type{});
  return s.cu_q ? run(I128{}, std::true_type{}) : run(I128{}, std::false_type{});
}

}  // namespace fh
