// The gradients of key tiles that hold a sink, from the fp32 partial sums of their parts
// (sink_splits): dK and dV = the sum of the parts in order, plus the addends if there are
// any, rounded once to bf16. A few hundred KB to some MB: a launch's latency, hardly more.

#include <cuda_runtime.h>

#include "kernels.h"

namespace fh {
namespace {

constexpr int kJoinThreads = 256;

// One thread per 8 columns of a row of dK or dV. Grid (blocks of rows, key heads, batch).
template <int HD, bool VL>
__global__ void __launch_bounds__(kJoinThreads)
    sink_join_kernel(const SinkShape s, __nv_bfloat16* __restrict__ dk, __nv_bfloat16* __restrict__ dv,
                     const __nv_bfloat16* dk_acc, const __nv_bfloat16* dv_acc) {
  constexpr int CH = HD / 8;
  const int i = blockIdx.x * kJoinThreads + threadIdx.x;
  const int chunk = i % CH, matrix = (i / CH) & 1, key = i / (2 * CH);
  const int hk = blockIdx.y, b = blockIdx.z;
  SeqRange sr;
  const SinkShape l = seq_shape<VL>(s, b, &sr);
  if (key >= l.Tk) return;
  float v[8] = {};
#pragma unroll 4
  for (int p = 0; p < s.splits; ++p) {
    const float4* src = reinterpret_cast<const float4*>(
        sink_part_row(s, HD, key / kBM, b * s.Hk + hk, p, matrix, key % kBM) + chunk * 8);
    const float4 x = src[0], y = src[1];
    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
    v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
  }
  const size_t off = k_row(l, sr, key, hk) + chunk * 8;
  const __nv_bfloat16* add = matrix == 0 ? dk_acc : dv_acc;
  if (add)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += __bfloat162float(add[off + k]);  // may be the output: read before it is written
  __nv_bfloat16* dst = (matrix == 0 ? dk : dv) + off;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                              pack_bf16(v[6], v[7]));
}

}  // namespace

int launch_sink_join(const SinkShape& s, int hd, void* dk, void* dv, const void* dk_acc, const void* dv_acc,
                     cudaStream_t stream) {
  const int rows = sink_tiles(s) * kBM;
  const dim3 grid((rows * 2 * (hd / 8) + kJoinThreads - 1) / kJoinThreads, s.Hk, s.B);
  auto launch = [&](auto* kernel) {
    kernel<<<grid, kJoinThreads, 0, stream>>>(s, static_cast<__nv_bfloat16*>(dk), static_cast<__nv_bfloat16*>(dv),
                                              static_cast<const __nv_bfloat16*>(dk_acc),
                                              static_cast<const __nv_bfloat16*>(dv_acc));
    return after_launch();
  };
  if (hd == 64) return s.cu_q ? launch(&sink_join_kernel<64, true>) : launch(&sink_join_kernel<64, false>);
  return s.cu_q ? launch(&sink_join_kernel<128, true>) : launch(&sink_join_kernel<128, false>);
}

}  // namespace fh
