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
// scalars (lp, rho, c, c') are formed in 64 bits from that sum, whose exponentials and
// additions are fp32: lp is off by some 1e-6 (1.6e-5 is the bound that the tests derive), and a
// ratio that close to a clip border may fall on its other side.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "vec_io.cuh"

namespace fh {
namespace {

constexpr int kPolThreads = 256;
// Columns up to which a row is one warp's (eight rows a block) instead of a block's: the
// threads of a block would have less than two 16-byte loads each (100000 rows of 1000 bf16:
// the sums take 299 us a block each, 61 us a warp each).
constexpr int kWarpRowBytes = 8192;
constexpr float kPLog2e = 1.4426950408889634f;

__device__ __forceinline__ float pol_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sum of doubles over a group of NT threads (a warp, or a block of NT), all of which receive
// it; warps in order.
template <int NT>
__device__ __forceinline__ double group_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (NT == 32) {
    return v;
  } else {
    __shared__ double red[NT / 32];
    __syncthreads();  // `red` may still be read by a previous call
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t += red[w];
    return t;
  }
}

// What the forward leaves for the backward passes -- four fp32 vectors of `rows`: m, 1 / sum,
// c and c'; the weights; 1 / N -- and, for the forward alone, the rows' partial sums, the
// blocks' partial losses and the count of finished blocks.
struct PolicyStats {
  float *m, *rsum, *c, *dc, *w, *inv_n;
  unsigned* done;
  float2* part;     // [rows][splits]: maximum and sum of exp(z - maximum) of a stretch of columns
  double2* blocks;  // [finish blocks]: sum of w l, sum of w
};

constexpr int kFinishThreads = 128;

__host__ __device__ inline int finish_blocks(int rows) {
  return rows > 0 ? (rows + kFinishThreads - 1) / kFinishThreads : 1;
}

// Stretches that a row's columns are cut into: with few rows, as many as it takes to give
// every SM four CTAs, but none shorter than 4096 columns (7 x 131072 fp32: the sums take
// 3 us in 32 stretches, 17 us whole).
__host__ __device__ inline int policy_splits(int rows, int vocab) {
  const int want = (4 * 148 + rows - 1) / (rows > 0 ? rows : 1), most = vocab / 4096;
  const int k = want < most ? want : most;
  return k < 1 ? 1 : k;
}

// Offsets in floats, the 8- and 16-byte members aligned.
struct PolicyLayout {
  long long part, blocks, total;
  __host__ __device__ PolicyLayout(int rows, int vocab) {
    const long long n = rows;
    blocks = (5 * n + 2 + 3) / 4 * 4;
    part = blocks + 4ll * finish_blocks(rows);
    total = part + 2 * n * policy_splits(rows, vocab);
  }
};

__host__ __device__ inline PolicyStats policy_stats(const PolicyArgs& a) {
  const size_t n = static_cast<size_t>(a.rows);
  const PolicyLayout l(a.rows, a.vocab);
  float* s = a.stats;
  return PolicyStats{s,
                     s + n,
                     s + 2 * n,
                     s + 3 * n,
                     s + 4 * n,
                     s + 5 * n,
                     reinterpret_cast<unsigned*>(s + 5 * n + 1),
                     reinterpret_cast<float2*>(s + l.part),
                     reinterpret_cast<double2*>(s + l.blocks)};
}

// Stretch k of `splits` of a row's columns.
struct Stretch {
  int first, count;
  __device__ __forceinline__ Stretch(int vocab, int splits, int k) {
    const int per = vocab / splits, rest = vocab - per * splits;  // the first `rest` are one longer
    first = k * per + min(k, rest);
    count = per + (k < rest ? 1 : 0);
  }
};

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

// exp(z - m) of two neighbouring columns, the arithmetic on fp32x2.
__device__ __forceinline__ float2 exp_of2(float a, float b, float2 neg_m) {
  const float2 x = __fmul2_rn(__fadd2_rn(make_float2(a, b), neg_m), make_float2(kPLog2e, kPLog2e));
  return make_float2(pol_ex2(x.x), pol_ex2(x.y));
}

// The largest of a 16-byte vector's elements (NaN passed over); bf16 pairs in one instruction.
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& x) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
  } else {
    auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(x.x), h(x.y)), __hmax2(h(x.z), h(x.w))));
    return fmaxf(f.x, f.y);
  }
}

// The sum s of exp(z - m) over the values seen, m their running maximum.
struct RunningSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void raise(float x) {
    if (x > m) {
      s *= exp_of(m, x);  // s = 0 while m = -inf
      m = x;
    }
  }
  template <typename T, int N>
  __device__ __forceinline__ void add(const uint4 (&x)[N]) {
    constexpr int E = 16 / sizeof(T);
    float top = vec_max<T>(x[0]);
#pragma unroll
    for (int u = 1; u < N; ++u) top = fmaxf(top, vec_max<T>(x[u]));
    raise(top);
    const float base = m == -INFINITY ? 0.f : m;
    const float2 nm = make_float2(-base, -base);
    float2 t[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float v[E];
      load_vec<T, E>(reinterpret_cast<const T*>(&x[u]), v);
#pragma unroll
      for (int k = 0; k < E; k += 2) t[u & 1] = __fadd2_rn(t[u & 1], exp_of2(v[k], v[k + 1], nm));
    }
    s += (t[0].x + t[0].y) + (t[1].x + t[1].y);
  }
  __device__ __forceinline__ void add(float v) {
    raise(v);
    s += exp_of(v, m == -INFINITY ? 0.f : m);
  }
};

// The running sums of a group of NT threads brought to their common maximum; every thread
// gets (m, s).
template <int NT>
__device__ __forceinline__ float2 group_join(const RunningSum& rs) {
  float m = rs.m, s = rs.s;
  // A thread without a finite value has the sum 0, or NaN from a NaN logit.
  auto bring = [](float m_from, float m_to) { return m_from == -INFINITY ? 1.f : exp_of(m_from, m_to); };
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    const float to = fmaxf(m, om);
    s = s * bring(m, to) + os * bring(om, to);
    m = to;
  }
  if constexpr (NT > 32) {
    __shared__ float redm[NT / 32], reds[NT / 32];
    if ((threadIdx.x & 31) == 0) {
      redm[threadIdx.x >> 5] = m;
      reds[threadIdx.x >> 5] = s;
    }
    __syncthreads();
    m = redm[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) m = fmaxf(m, redm[w]);
    s = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) s += reds[w] * bring(redm[w], m);
  }
  return make_float2(m, s);
}

// The stretch of a row that a group of NT threads works on: `splits` stretches a row, the
// groups in order over blocks of kPolThreads.
template <int NT>
struct Work {
  int row, stretch, t;  // t: this thread's number in its group
  bool any;             // false past the last stretch
  __device__ __forceinline__ Work(int rows, int splits) {
    const unsigned g = blockIdx.x * (kPolThreads / NT) + threadIdx.x / NT;  // below 2^31 + 8: few rows where splits > 1
    row = static_cast<int>(min(splits == 1 ? g : g / splits, 0x7fffffffu));
    stretch = splits == 1 ? 0 : static_cast<int>(g % splits);
    t = threadIdx.x % NT;
    any = row < rows;
  }
};

// Maximum and sum of exponentials of a stretch, a batch of vectors at a time: the maximum is
// compared and the sum rescaled once a batch.

template <typename T, int NT>
__global__ void __launch_bounds__(kPolThreads, NT == 32 ? 8 : 5) policy_sums_kernel(PolicyArgs a, int splits) {
  constexpr int kPolBatch = NT == 32 ? 2 : 4;
  const Work<NT> wk(a.rows, splits);
  const PolicyStats st = policy_stats(a);
  if (blockIdx.x == 0 && threadIdx.x == 0) *st.done = 0u;
  if (!wk.any || (a.weights && a.weights[wk.row] == 0.f)) return;
  const Stretch cols(a.vocab, splits, wk.stretch);
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(wk.row) * a.ld + cols.first;
  using Span = RowSpan<T>;
  const Span sp(row, cols.count, 0);
  const T* first = row + sp.head;
  RunningSum rs;
  int i = wk.t;
  for (; i + (kPolBatch - 1) * NT < sp.nvec; i += kPolBatch * NT) {
    uint4 x[kPolBatch];
#pragma unroll
    for (int u = 0; u < kPolBatch; ++u) x[u] = reinterpret_cast<const uint4*>(first)[i + u * NT];
    rs.add<T>(x);
  }
  if (i < sp.nvec) {  // the last, partial batch: -inf in the place of what is not there
    const uint32_t low = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    uint4 x[kPolBatch];
#pragma unroll
    for (int u = 0; u < kPolBatch; ++u)
      x[u] = i + u * NT < sp.nvec ? reinterpret_cast<const uint4*>(first)[i + u * NT] : make_uint4(low, low, low, low);
    rs.add<T>(x);
  }
  for (int j = wk.t; j < sp.scalars(cols.count); j += NT) rs.add(to_f32(row[sp.scalar(j)]));
  const float2 ms = group_join<NT>(rs);
  if (wk.t == 0) st.part[static_cast<size_t>(wk.row) * splits + wk.stretch] = ms;
}

// One thread per row: the row's scalars, in 64 bits; then the loss. The last block to finish
// adds up the blocks' sums, in the order of the blocks.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads) policy_finish_kernel(PolicyArgs a, int splits) {
  __shared__ bool last;
  const PolicyStats st = policy_stats(a);
  const int r = blockIdx.x * kFinishThreads + threadIdx.x;
  double wl = 0.0, weight = 0.0;
  if (r < a.rows) {
    // All that does not depend on another load first: the kernel's time is latency. (What
    // `part` holds in a row of weight 0 is not used.)
    const float w = a.weights ? a.weights[r] : 1.f;
    const float2* part = st.part + static_cast<size_t>(r) * splits;
    const float2 part0 = part[0];
    const long long act = a.actions[r];
    const double adv = a.adv[r], old = a.old[r], ref = a.beta != 0.f ? a.ref[r] : 0.f;
    st.w[r] = w;
    if (w == 0.f) {
      a.lp[r] = 0.f;
      st.m[r] = st.rsum[r] = st.c[r] = st.dc[r] = 0.f;
    } else {
      const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld;
      const bool inside = act >= 0 && act < a.vocab;
      const double za = inside ? to_f32(row[act]) : __int_as_float(0x7fc00000);
      float m = part0.x;
      for (int k = 1; k < splits; ++k) m = fmaxf(m, part[k].x);
      double sum = splits == 1 ? part0.y : 0.0;
      for (int k = 0; splits > 1 && k < splits; ++k) {
        const float2 p = part[k];
        sum += static_cast<double>(p.y) * (p.x == -INFINITY ? 1.f : exp_of(p.x, m));
      }
      const double lp = za - static_cast<double>(m) - log(sum);  // NaN for an action outside
      const double rho = exp(lp - old);
      const double low = 1.0 - static_cast<double>(a.clip_low), high = 1.0 + static_cast<double>(a.clip_high);
      const bool open = !((adv > 0.0 && rho > high) || (adv < 0.0 && rho < low));
      double l = -adv * (open ? rho : adv > 0.0 ? high : low), dl = open ? -adv * rho : 0.0, ddl = dl;
      if (a.beta != 0.f) {
        const double beta = a.beta, d = ref - lp, e = exp(d);
        l += beta * (e - d - 1.0);
        dl += beta * (1.0 - e);
        ddl += beta * e;
      }
      a.lp[r] = static_cast<float>(lp);
      st.m[r] = m;
      st.rsum[r] = static_cast<float>(1.0 / sum);
      st.c[r] = static_cast<float>(dl);
      st.dc[r] = static_cast<float>(ddl);
      wl = l * w;
      weight = w;
    }
  }
  wl = group_sum_f64<kFinishThreads>(wl);
  weight = group_sum_f64<kFinishThreads>(weight);
  if (threadIdx.x == 0) {
    st.blocks[blockIdx.x] = make_double2(wl, weight);
    __threadfence();  // before the count that tells the last block of it
    last = atomicAdd(st.done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double2 sum = make_double2(0.0, 0.0);
  for (int b = threadIdx.x; b < static_cast<int>(gridDim.x); b += kFinishThreads) {
    const double2 x = __ldcg(st.blocks + b);
    sum.x += x.x;
    sum.y += x.y;
  }
  sum.x = group_sum_f64<kFinishThreads>(sum.x);
  sum.y = group_sum_f64<kFinishThreads>(sum.y);
  if (threadIdx.x == 0) {
    const double n = a.normalizer > 0.f ? static_cast<double>(a.normalizer) : sum.y;
    a.loss[0] = n != 0.0 ? static_cast<float>(sum.x / n) : 0.f;
    st.inv_n[0] = n != 0.0 ? static_cast<float>(1.0 / n) : 0.f;
  }
}

// Zeros into `count` columns.
template <typename T, int NT>
__device__ __forceinline__ void zero_cols(T* out, int count, int t) {
  const RowSpan<T> sp(out, count, 0);
  for (int i = t; i < sp.nvec; i += NT)
    *reinterpret_cast<uint4*>(out + sp.vec(i)) = make_uint4(0u, 0u, 0u, 0u);
  for (int i = t; i < sp.scalars(count); i += NT) out[sp.scalar(i)] = from_f32<T>(0.f);
}

// Adds x to the element of v (columns col, col + 1, ...) that is column `act`, if one is.
template <int N>
__device__ __forceinline__ void add_at(float (&v)[N], long long act, int col, float x) {
  const long long at = act - col;
  if (at < 0 || at >= N) return;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] += e == at ? x : 0.f;
}

template <typename T, int NT>
__global__ void __launch_bounds__(kPolThreads, NT == 32 ? 8 : 1)
    policy_bwd_kernel(PolicyArgs a, int splits, const float* __restrict__ g, T* __restrict__ dz) {
  const Work<NT> wk(a.rows, splits);
  if (!wk.any) return;
  const int r = wk.row;
  const Stretch cols(a.vocab, splits, wk.stretch);
  const PolicyStats st = policy_stats(a);
  T* out = dz + static_cast<long long>(r) * a.vocab + cols.first;
  const float w = st.w[r];
  if (w == 0.f) return zero_cols<T, NT>(out, cols.count, wk.t);
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld + cols.first;
  const float k = g[0] * w * st.inv_n[0] * st.c[r], m = st.m[r], kp = -k * st.rsum[r];
  const long long act = a.actions[r] - cols.first;
  using Span = RowSpan<T>;
  const Span sp(row, cols.count, addr(row) ^ addr(out));
  const uint4* in4 = reinterpret_cast<const uint4*>(row + sp.head);
  uint4* out4 = reinterpret_cast<uint4*>(out + sp.head);
  // A block's row: four vectors' loads at once (4096 x 32000 bf16: 72 us, 82 us one by one);
  // a warp's: as many warps as an SM holds (100000 x 1000: 72 us, 113 us with four at once).
  constexpr int kUnroll = NT == 32 ? 1 : 4;
#pragma unroll kUnroll
  for (int i = wk.t; i < sp.nvec; i += NT) {
    const uint4 raw = in4[i];
    float v[Span::E];
    load_vec<T, Span::E>(reinterpret_cast<const T*>(&raw), v);
#pragma unroll
    for (int e = 0; e < Span::E; e += 2) {
      const float2 p = __fmul2_rn(exp_of2(v[e], v[e + 1], make_float2(-m, -m)), make_float2(kp, kp));
      v[e] = p.x;
      v[e + 1] = p.y;
    }
    add_at(v, act, sp.vec(i), k);
    uint4 o;
    store_vec<T, Span::E>(reinterpret_cast<T*>(&o), v);
    out4[i] = o;
  }
  for (int i = wk.t; i < sp.scalars(cols.count); i += NT) {
    const int col = sp.scalar(i);
    out[col] = from_f32<T>(exp_of(to_f32(row[col]), m) * kp + (col == act ? k : 0.f));
  }
}

// sum exp(z - m) u over a stretch of columns, this thread's share.
template <typename T, int NT>
__device__ __forceinline__ float dot_share(const T* row, const T* urow, const RowSpan<T>& sp, int count, float m,
                                           int t) {
  using Span = RowSpan<T>;
  const uint4* z4 = reinterpret_cast<const uint4*>(row + sp.head);
  const uint4* u4 = reinterpret_cast<const uint4*>(urow + sp.head);
  float2 dots = make_float2(0.f, 0.f);
  constexpr int kUnroll = NT == 32 ? 1 : 2;
#pragma unroll kUnroll
  for (int i = t; i < sp.nvec; i += NT) {
    const uint4 rz = z4[i], ru = u4[i];
    float v[Span::E], x[Span::E];
    load_vec<T, Span::E>(reinterpret_cast<const T*>(&rz), v);
    load_vec<T, Span::E>(reinterpret_cast<const T*>(&ru), x);
#pragma unroll
    for (int e = 0; e < Span::E; e += 2)
      dots = __ffma2_rn(exp_of2(v[e], v[e + 1], make_float2(-m, -m)), make_float2(x[e], x[e + 1]), dots);
  }
  float dot = dots.x + dots.y;
  for (int i = t; i < sp.scalars(count); i += NT) {
    const int col = sp.scalar(i);
    dot = fmaf(exp_of(to_f32(row[col]), m), to_f32(urow[col]), dot);
  }
  return dot;
}

// With splits > 1, first: the stretches' shares of sum <p, u>.
template <typename T, int NT>
__global__ void __launch_bounds__(kPolThreads) policy_dots_kernel(PolicyArgs a, int splits, const T* __restrict__ u,
                                                                  float* __restrict__ part) {
  const Work<NT> wk(a.rows, splits);
  if (!wk.any) return;
  const int r = wk.row;
  const Stretch cols(a.vocab, splits, wk.stretch);
  const PolicyStats st = policy_stats(a);
  if (st.w[r] == 0.f) return;
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld + cols.first;
  const T* urow = u + static_cast<long long>(r) * a.vocab + cols.first;
  const RowSpan<T> sp(row, cols.count, addr(row) ^ addr(urow));
  const double dot = group_sum_f64<NT>(dot_share<T, NT>(row, urow, sp, cols.count, st.m[r], wk.t));
  if (wk.t == 0) part[static_cast<size_t>(r) * splits + wk.stretch] = static_cast<float>(dot);
}

// The dot product <p, u> of the row comes from `part` (policy_dots_kernel) or, for whole rows,
// is formed here: the second reading of z and u then comes from L2, as far as the rows in
// flight fit there. So four blocks an SM, and the second reading and gz, which this
// kernel does not read again, marked as first to be evicted (4096 x 32000 bf16, all rows: 158 us; 206 with six
// blocks, 169 with three, 120 at the copy rate). Holding the row in a cluster's shared memory
// took 178 us: loading, joining and writing a row in turn leaves the memory idle, and clusters
// that stay and load the next row meanwhile took 250 us or more.
template <typename T, int NT>
__global__ void __launch_bounds__(kPolThreads, NT == 32 ? 6 : 4)
    policy_bwd_bwd_kernel(PolicyArgs a, int splits, const float* __restrict__ part, const float* __restrict__ g,
                          const T* __restrict__ u, T* __restrict__ gz, float* __restrict__ gg) {
  const Work<NT> wk(a.rows, splits);
  if (!wk.any) return;
  const int r = wk.row;
  const Stretch cols(a.vocab, splits, wk.stretch);
  const PolicyStats st = policy_stats(a);
  T* out = gz + static_cast<long long>(r) * a.vocab + cols.first;
  const float w = st.w[r];
  if (w == 0.f) {
    if (wk.t == 0 && wk.stretch == 0) gg[r] = 0.f;
    return zero_cols<T, NT>(out, cols.count, wk.t);
  }
  const T* row = static_cast<const T*>(a.z) + static_cast<long long>(r) * a.ld + cols.first;
  const T* urow = u + static_cast<long long>(r) * a.vocab + cols.first;
  const float m = st.m[r], rsum = st.rsum[r];
  const long long act = a.actions[r], here = act - cols.first;
  using Span = RowSpan<T>;
  const Span sp(row, cols.count, (addr(row) ^ addr(out)) | (addr(row) ^ addr(urow)));
  double dot = 0.0;
  if (splits > 1) {
    for (int k = 0; k < splits; ++k) dot += part[static_cast<size_t>(r) * splits + k];
  } else {
    dot = group_sum_f64<NT>(dot_share<T, NT>(row, urow, sp, cols.count, m, wk.t));
  }
  const float pu = static_cast<float>(dot * rsum);
  const bool inside = act >= 0 && act < a.vocab;
  const float s = inside ? to_f32(u[static_cast<long long>(r) * a.vocab + act]) - pu : __int_as_float(0x7fc00000);
  const float wn = w * st.inv_n[0], k = g[0] * wn;
  // gz = k c' s (e - p) - k c p (u - <p, u>) = k c' s e + p (k c <p, u> - k c' s - k c u)
  const float ks = k * st.dc[r] * s, kc = k * st.c[r];
  const float b0 = (kc * pu - ks) * rsum, b1 = -kc * rsum;
  const uint4* z4 = reinterpret_cast<const uint4*>(row + sp.head);
  const uint4* u4 = reinterpret_cast<const uint4*>(urow + sp.head);
  uint4* out4 = reinterpret_cast<uint4*>(out + sp.head);
  constexpr int kUnroll = NT == 32 ? 1 : 2;
#pragma unroll kUnroll
  for (int i = wk.t; i < sp.nvec; i += NT) {
    const uint4 rz = __ldcs(z4 + i), ru = __ldcs(u4 + i);
    float v[Span::E], x[Span::E];
    load_vec<T, Span::E>(reinterpret_cast<const T*>(&rz), v);
    load_vec<T, Span::E>(reinterpret_cast<const T*>(&ru), x);
#pragma unroll
    for (int e = 0; e < Span::E; e += 2) {
      const float2 q = __ffma2_rn(make_float2(b1, b1), make_float2(x[e], x[e + 1]), make_float2(b0, b0));
      const float2 p = __fmul2_rn(exp_of2(v[e], v[e + 1], make_float2(-m, -m)), q);
      v[e] = p.x;
      v[e + 1] = p.y;
    }
    add_at(v, here, sp.vec(i), ks);
    uint4 o;
    store_vec<T, Span::E>(reinterpret_cast<T*>(&o), v);
    __stcs(out4 + i, o);
  }
  for (int i = wk.t; i < sp.scalars(cols.count); i += NT) {
    const int col = sp.scalar(i);
    out[col] = from_f32<T>(exp_of(to_f32(row[col]), m) * fmaf(b1, to_f32(urow[col]), b0) + (col == here ? ks : 0.f));
  }
  if (wk.t == 0 && wk.stretch == 0) gg[r] = wn * st.c[r] * s;
}

}  // namespace

long long policy_stats_floats(int rows, int vocab) { return PolicyLayout(rows, vocab).total; }

long long policy_scratch_floats(int rows, int vocab) {
  const int splits = policy_splits(rows, vocab);
  return splits > 1 ? static_cast<long long>(rows) * splits : 0;
}

int launch_policy(int op, const PolicyArgs& a, const float* g, const void* u, void* out, float* gg, float* scratch,
                  cudaStream_t stream) {
  if (a.rows == 0 && op != 0) return kOk;
  const int splits = policy_splits(a.rows, a.vocab);
  auto run = [&](auto tag, auto group) -> int {
    using T = decltype(tag);
    constexpr int NT = decltype(group)::value;
    constexpr int kGroups = kPolThreads / NT;
    const unsigned grid = static_cast<unsigned>((static_cast<long long>(a.rows) * splits + kGroups - 1) / kGroups);
    T* o = static_cast<T*>(out);
    const T* uu = static_cast<const T*>(u);
    if (op == 0) {
      if (a.rows == 0) {  // the loss of nothing
        if (cudaMemsetAsync(policy_stats(a).done, 0, sizeof(unsigned), stream) != cudaSuccess) return kLaunchFailed;
      } else {
        policy_sums_kernel<T, NT><<<grid, kPolThreads, 0, stream>>>(a, splits);
        if (after_launch() != kOk) return kLaunchFailed;
      }
      policy_finish_kernel<T><<<finish_blocks(a.rows), kFinishThreads, 0, stream>>>(a, splits);
      return after_launch();
    }
    if (op == 1) {
      policy_bwd_kernel<T, NT><<<grid, kPolThreads, 0, stream>>>(a, splits, g, o);
      return after_launch();
    }
    if (splits > 1) {
      policy_dots_kernel<T, NT><<<grid, kPolThreads, 0, stream>>>(a, splits, uu, scratch);
      if (after_launch() != kOk) return kLaunchFailed;
    }
    policy_bwd_bwd_kernel<T, NT><<<grid, kPolThreads, 0, stream>>>(a, splits, scratch, g, uu, o, gg);
    return after_launch();
  };
  using Warp = std::integral_constant<int, 32>;
  using Block = std::integral_constant<int, kPolThreads>;
  const bool narrow = static_cast<long long>(a.vocab) * (a.bf16 ? 2 : 4) <= kWarpRowBytes;
  if (a.bf16) return narrow ? run(__nv_bfloat16{}, Warp{}) : run(__nv_bfloat16{}, Block{});
  return narrow ? run(0.f, Warp{}) : run(0.f, Block{});
}

}  // namespace fh
