// Clipped policy loss with a KL term over language-model logits: forward, backward and the
// backward's backward.
//
// For logits z (rows x vocab, fp32 or bf16), per row an action a, the log probability the
// sampling policy gave it (old), an advantage A, a weight w and, with beta > 0, a reference
// policy's log probability (ref):
//   lp   = z_a - log sum_v exp z_v,   rho = exp(lp - old)
//   l    = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   loss = sum_r w l / N,  N = sum_r w or the caller's; 0 where N is 0
// The derivatives by lp: the clipped side of the minimum has none, so with
// open = not (A > 0 and rho > 1 + hi) and not (A < 0 and rho < 1 - lo)
//   c = dl/dlp = -open A rho + beta (1 - exp(ref - lp)),   c' = -open A rho + beta exp(ref - lp)
// and with p = softmax(z), e = onehot(a), g the upstream scalar and k = g w / N
//   backward             dz = k c (e - p)
//   backward's backward  given u: s = u_a - <p, u>:
//                        gz = k (c' s (e - p) - c p (u - <p, u>)),  gg = sum_r c s w / N
// A row of weight 0 is not read: its loss, log probability and gradients are 0 whatever its
// logits hold. An action outside [0, vocab) in another row gives NaN.
//
// Every pass reads the logits once (the backward's backward twice, the second time from
// L2) and is bound by memory. The exponentials are ex2((z - m) log2e) with the row maximum
// m; the forward keeps m and 1 / sum, so the passes after it form the same p. The per-row
// scalars (lp, rho, c, c') are formed in 64 bits: a ratio next to a clip border falls on
// the side that it has.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "kernels.h"
#include "vec_io.cuh"

namespace fh {
namespace {

constexpr int kPolThreads = 256;
constexpr int kPolWarps = kPolThreads / 32;
constexpr float kPLog2e = 1.4426950408889634f;

__device__ __forceinline__ float pol_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Block-wide sum of doubles (all threads receive it), warps in order.
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // `red` may still be read by a previous call
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) t = fmaxf(t, red[w]);
  return t;
}

// What the forward leaves for the backward passes: six fp32 vectors of `rows` -- m,
// 1 / sum, c, c', w l and w -- and 1 / N.
struct PolicyStats {
  float *m, *rsum, *c, *dc, *wl, *w, *inv_n;
};

__host__ __device__ inline PolicyStats policy_stats(float* s, int rows) {
  const size_t n = static_cast<size_t>(rows);
  return PolicyStats{s, s + n, s + 2 * n, s + 3 * n, s + 4 * n, s + 5 * n, s + 6 * n};
}

// A row's columns: `head` scalars up to the first 16-byte boundary, `nvec` vectors, then
// scalars again. All scalars where the row's tensors (`diff`: the bits in which their
// addresses differ) do not reach a boundary at the same column.
template <typename T>
struct RowSpan {
  static constexpr int E = 16 / sizeof(T);
  int head, nvec;
  __device__ __forceinline__ RowSpan(const T* row, int vocab, uintptr_t diff) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15u);
    head = (diff & 15u) ? vocab : min(vocab, static_cast<int>(((16 - off) & 15) / sizeof(T)));
    nvec = (vocab - head) / E;
  }
  __device__ __forceinline__ int vec(int i) const { return head + i * E; }  // first column of vector i
  __device__ __forceinline__ int scalars(int vocab) const { return vocab - nvec * E; }
  __device__ __forceinline__ int scalar(int i) const { return i < head ? i : i + nvec * E; }  // column of scalar i
};

__device__ __forceinline__ uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// exp(z - m). The difference first: z and m may both be the type's lowest value.
__device__ __forceinline__ float exp_of(float z, float m) { return pol_ex2((z - m) * kPLog2e); }

// The sum s of exp(z - m) over the values seen, m their running maximum.
struct RunningSum {
  float m = -INFINITY, s = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float x = v[0];
#pragma unroll
    for (int k = 1; k < N; ++k) x = fmaxf(x, v[k]);
    if (x > m) {
      s *= exp_of(m, x);  // s = 0 while m = -inf
      m = x;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) t += exp_of(v[k], base);
    s += t;
  }
};

template <typename T>
__global__ void __launch_bounds__(kPolThreads) policy_fwd_kernel(PolicyArgs a) {
  __shared__ double red[kPolWarps];
  __shared__ float redf[kPolWarps];
  const int r = blockIdx.x;
  const PolicyStats st = policy_stats(a.stats, a.rows);
  const float w = a.weights ? a.weights[r] : 1.f;
  if (w == 0.f) {
    if (threadIdx.x == 0) {
      a.lp[r] = 0.f;
      st.m[r] = st.rsum[r] = st.c[r] = st.dc[r] = st.wl[r] = st.w[r] = 0.f;
    }
    return;
  }
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld;
  using Span = RowSpan<T>;
  const Span sp(row, a.vocab, 0);
  RunningSum rs;
#pragma unroll 4
  for (int i = threadIdx.x; i < sp.nvec; i += kPolThreads) {
    float v[Span::E];
    load_vec<T, Span::E>(row + sp.vec(i), v);
    rs.add(v);
  }
  for (int i = threadIdx.x; i < sp.scalars(a.vocab); i += kPolThreads) {
    float v[1];
    load_vec<T, 1>(row + sp.scalar(i), v);
    rs.add(v);
  }
  // The threads' sums brought to the row's maximum. A thread without a finite value has
  // the sum 0, or NaN from a NaN logit.
  const float m = block_max(rs.m, redf);
  const float up = rs.m == -INFINITY ? 1.f : exp_of(rs.m, m);
  const double sum = block_sum_f64(static_cast<double>(rs.s) * up, red);
  if (threadIdx.x != 0) return;
  const long long act = a.actions[r];
  double lp = __longlong_as_double(0x7ff8000000000000ll);
  if (act >= 0 && act < a.vocab) lp = static_cast<double>(to_f32(row[act])) - static_cast<double>(m) - log(sum);
  const double adv = a.adv[r], rho = exp(lp - static_cast<double>(a.old[r]));
  const double clipped = fmin(fmax(rho, 1.0 - static_cast<double>(a.clip_low)), 1.0 + static_cast<double>(a.clip_high));
  const bool open = !((adv > 0.0 && rho > 1.0 + static_cast<double>(a.clip_high)) ||
                      (adv < 0.0 && rho < 1.0 - static_cast<double>(a.clip_low)));
  double l = -(open ? rho * adv : clipped * adv), dl = open ? -adv * rho : 0.0, ddl = dl;
  if (a.beta != 0.f) {
    const double beta = a.beta, d = static_cast<double>(a.ref[r]) - lp, e = exp(d);
    l += beta * (e - d - 1.0);
    dl += beta * (1.0 - e);
    ddl += beta * e;
  }
  a.lp[r] = static_cast<float>(lp);
  st.m[r] = m;
  st.rsum[r] = static_cast<float>(1.0 / sum);
  st.c[r] = static_cast<float>(dl);
  st.dc[r] = static_cast<float>(ddl);
  st.wl[r] = static_cast<float>(l * w);
  st.w[r] = w;
}

// loss = sum_r w l / N and 1 / N, one block, rows in a fixed order.
constexpr int kPolSumThreads = 1024;
__global__ void __launch_bounds__(kPolSumThreads) policy_sum_kernel(PolicyArgs a) {
  __shared__ double red[kPolSumThreads / 32];
  const PolicyStats st = policy_stats(a.stats, a.rows);
  double wl = 0.0, w = 0.0;
  for (int r = threadIdx.x; r < a.rows; r += kPolSumThreads) {
    wl += st.wl[r];
    w += st.w[r];
  }
  wl = block_sum_f64(wl, red);
  w = block_sum_f64(w, red);
  if (threadIdx.x == 0) {
    const double n = a.normalizer > 0.f ? static_cast<double>(a.normalizer) : w;
    a.loss[0] = n != 0.0 ? static_cast<float>(wl / n) : 0.f;
    st.inv_n[0] = n != 0.0 ? static_cast<float>(1.0 / n) : 0.f;
  }
}

// Zeros into a row's columns.
template <typename T>
__device__ __forceinline__ void zero_cols(T* out, int vocab) {
  const RowSpan<T> sp(out, vocab, 0);
  for (int i = threadIdx.x; i < sp.nvec; i += kPolThreads)
    *reinterpret_cast<uint4*>(out + sp.vec(i)) = make_uint4(0u, 0u, 0u, 0u);
  for (int i = threadIdx.x; i < sp.scalars(vocab); i += kPolThreads) out[sp.scalar(i)] = from_f32<T>(0.f);
}

template <typename T>
__global__ void __launch_bounds__(kPolThreads) policy_bwd_kernel(PolicyArgs a, const float* __restrict__ g,
                                                                 T* __restrict__ dz) {
  const int r = blockIdx.x;
  const PolicyStats st = policy_stats(a.stats, a.rows);
  T* out = dz + static_cast<long long>(r) * a.vocab;
  const float w = st.w[r];
  if (w == 0.f) return zero_cols(out, a.vocab);
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld;
  const float k = g[0] * w * st.inv_n[0] * st.c[r], m = st.m[r], kp = -k * st.rsum[r];
  const long long act = a.actions[r];
  using Span = RowSpan<T>;
  const Span sp(row, a.vocab, addr(row) ^ addr(out));
#pragma unroll 4
  for (int i = threadIdx.x; i < sp.nvec; i += kPolThreads) {
    const int col = sp.vec(i);
    float v[Span::E];
    load_vec<T, Span::E>(row + col, v);
#pragma unroll
    for (int e = 0; e < Span::E; ++e) v[e] = exp_of(v[e], m) * kp + (col + e == act ? k : 0.f);
    store_vec<T, Span::E>(out + col, v);
  }
  for (int i = threadIdx.x; i < sp.scalars(a.vocab); i += kPolThreads) {
    const int col = sp.scalar(i);
    out[col] = from_f32<T>(exp_of(to_f32(row[col]), m) * kp + (col == act ? k : 0.f));
  }
}

template <typename T>
__global__ void __launch_bounds__(kPolThreads) policy_bwd_bwd_kernel(PolicyArgs a, const float* __restrict__ g,
                                                                     const T* __restrict__ u, T* __restrict__ gz,
                                                                     float* __restrict__ gg) {
  __shared__ double red[kPolWarps];
  const int r = blockIdx.x;
  const PolicyStats st = policy_stats(a.stats, a.rows);
  T* out = gz + static_cast<long long>(r) * a.vocab;
  const float w = st.w[r];
  if (w == 0.f) {
    if (threadIdx.x == 0) gg[r] = 0.f;
    return zero_cols(out, a.vocab);
  }
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld;
  const T* urow = u + static_cast<long long>(r) * a.vocab;
  const float m = st.m[r], rsum = st.rsum[r];
  const long long act = a.actions[r];
  using Span = RowSpan<T>;
  const Span sp(row, a.vocab, (addr(row) ^ addr(out)) | (addr(row) ^ addr(urow)));
  float dot = 0.f;
  for (int i = threadIdx.x; i < sp.nvec; i += kPolThreads) {
    float v[Span::E], x[Span::E];
    load_vec<T, Span::E>(row + sp.vec(i), v);
    load_vec<T, Span::E>(urow + sp.vec(i), x);
#pragma unroll
    for (int e = 0; e < Span::E; ++e) dot = fmaf(exp_of(v[e], m), x[e], dot);
  }
  for (int i = threadIdx.x; i < sp.scalars(a.vocab); i += kPolThreads) {
    const int col = sp.scalar(i);
    dot = fmaf(exp_of(to_f32(row[col]), m), to_f32(urow[col]), dot);
  }
  const float pu = static_cast<float>(block_sum_f64(dot, red) * rsum);
  const bool inside = act >= 0 && act < a.vocab;
  const float s = inside ? to_f32(urow[act]) - pu : __int_as_float(0x7fc00000);
  const float wn = w * st.inv_n[0], k = g[0] * wn;
  // gz = k c' s (e - p) - k c p (u - <p, u>) = k c' s e + p (k c <p, u> - k c' s - k c u)
  const float ks = k * st.dc[r] * s, kc = k * st.c[r];
  const float b0 = (kc * pu - ks) * rsum, b1 = -kc * rsum;
  for (int i = threadIdx.x; i < sp.nvec; i += kPolThreads) {
    const int col = sp.vec(i);
    float v[Span::E], x[Span::E];
    load_vec<T, Span::E>(row + col, v);
    load_vec<T, Span::E>(urow + col, x);
#pragma unroll
    for (int e = 0; e < Span::E; ++e)
      v[e] = exp_of(v[e], m) * fmaf(b1, x[e], b0) + (col + e == act ? ks : 0.f);
    store_vec<T, Span::E>(out + col, v);
  }
  for (int i = threadIdx.x; i < sp.scalars(a.vocab); i += kPolThreads) {
    const int col = sp.scalar(i);
    out[col] = from_f32<T>(exp_of(to_f32(row[col]), m) * fmaf(b1, to_f32(urow[col]), b0) +
                           (col == act ? ks : 0.f));
  }
  if (threadIdx.x == 0) gg[r] = wn * st.c[r] * s;
}

}  // namespace

int launch_policy(int op, const PolicyArgs& a, const float* g, const void* u, void* out, float* gg,
                  cudaStream_t stream) {
  if (a.rows == 0 && op != 0) return kOk;
#define FH_POLICY(T)                                                                                             \
  do {                                                                                                           \
    if (op == 0) policy_fwd_kernel<T><<<a.rows, kPolThreads, 0, stream>>>(a);                                    \
    else if (op == 1) policy_bwd_kernel<T><<<a.rows, kPolThreads, 0, stream>>>(a, g, static_cast<T*>(out));      \
    else policy_bwd_bwd_kernel<T><<<a.rows, kPolThreads, 0, stream>>>(a, g, static_cast<const T*>(u),            \
                                                                      static_cast<T*>(out), gg);                 \
  } while (0)
  if (a.rows > 0) {
    if (a.bf16) FH_POLICY(__nv_bfloat16);
    else FH_POLICY(float);
    if (after_launch() != kOk) return kLaunchFailed;
  }
#undef FH_POLICY
  if (op != 0) return kOk;
  policy_sum_kernel<<<1, kPolSumThreads, 0, stream>>>(a);
  return after_launch();
}

}  // namespace fh
