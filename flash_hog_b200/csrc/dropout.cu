// Dropout from a counter-based generator, with the residual addition.
//
//   y_i = r_i + keep_i x_i / (1 - L / 65536),   keep_i = (u_i >= L),  L = round(65536 p)
//
// u_i is a 16-bit draw of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) with the 64-bit seed as key and the counter
// (i / 8, subsequence): a block of four 32-bit words gives eight draws, low half first. So
// the mask is a function of (seed, subsequence, i) alone: it is never stored, and the
// backward pass -- the same map applied to dy -- draws it again. The map is linear in x;
// its derivatives of any order are itself.
//
// Bound by memory (read x and r, write y). Sixteen bits a draw instead of thirty-two halve
// the generator's work, which at 2-byte elements is of the order of the memory's time:
// ten rounds are 20 wide multiplications a block.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "vec_io.cuh"

namespace fh {
namespace {

constexpr int kDropThreads = 256;
constexpr int kDraws = 8;  // draws, and elements, per Philox block

// Philox4x32-10 of counter (block, sub, 0) under key.
__device__ __forceinline__ uint4 philox(unsigned long long block, unsigned sub, unsigned long long key) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = sub, c3 = 0u;
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = 0xD2511F53ull * c0, p1 = 0xCD9E8D57ull * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// keep(k) of a Philox block's eight draws: draw k is the low (even k) or high half of word
// k / 2. Compared in the upper half of a word, where the other draw's bits do not count.
struct Keep {
  uint32_t words[4];
  uint32_t limit16;  // limit << 16; all dropped (limit 65536) is the caller's case
  __device__ __forceinline__ bool operator()(int k) const {
    return (k & 1 ? words[k >> 1] : words[k >> 1] << 16) >= limit16;
  }
};

// N elements' values as loaded, converted when used.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) v[q] = reinterpret_cast<const uint4*>(p)[q];
  }
  __device__ __forceinline__ void get(float (&x)[kDraws]) const {
    load_vec<T, kDraws>(reinterpret_cast<const T*>(v), x);
  }
};
template <>
struct Eight<void> {};

// TR = void: no residual. Each thread takes kDropBlocks whole Philox blocks of eight
// elements, whose loads are issued before the draws are computed. The last blocks, and all
// when a pointer is not 16-byte aligned (VEC false), go element by element.
constexpr int kDropBlocks = 2;

template <typename TI, typename TR, typename TO, bool VEC>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(long long n, const TI* __restrict__ x,
                                                               const TR* __restrict__ res, TO* __restrict__ y,
                                                               const long long* __restrict__ seed, unsigned sub,
                                                               unsigned limit, float factor) {
  constexpr bool RES = !std::is_same<TR, void>::value;
  const unsigned long long key = static_cast<unsigned long long>(*seed);
  const long long b0 = static_cast<long long>(blockIdx.x) * (kDropThreads * kDropBlocks) + threadIdx.x;
  auto draw = [&](long long b) {
    const uint4 w = philox(static_cast<unsigned long long>(b), sub, key);
    return Keep{{w.x, w.y, w.z, w.w}, limit << 16};
  };
  if (VEC && limit < 65536u && (b0 + (kDropBlocks - 1) * kDropThreads + 1) * kDraws <= n) {
    Eight<TI> xv[kDropBlocks];
    [[maybe_unused]] Eight<TR> rv[kDropBlocks];
#pragma unroll
    for (int q = 0; q < kDropBlocks; ++q) {
      const long long i0 = (b0 + q * kDropThreads) * kDraws;
      xv[q].load(x + i0);
      if constexpr (RES) rv[q].load(res + i0);
    }
#pragma unroll
    for (int q = 0; q < kDropBlocks; ++q) {
      const long long b = b0 + q * kDropThreads;
      const Keep keep = draw(b);
      float v[kDraws], o[kDraws];
      xv[q].get(v);
      if constexpr (RES) {
        float r[kDraws];
        rv[q].get(r);
#pragma unroll
        for (int k = 0; k < kDraws; ++k) o[k] = keep(k) ? fmaf(v[k], factor, r[k]) : r[k];
      } else {
#pragma unroll
        for (int k = 0; k < kDraws; ++k) o[k] = keep(k) ? v[k] * factor : 0.f;
      }
      store_vec<TO, kDraws>(y + b * kDraws, o);
    }
    return;
  }
  for (int q = 0; q < kDropBlocks; ++q) {
    const long long b = b0 + q * kDropThreads, i0 = b * kDraws;
    if (i0 >= n) return;
    const Keep keep = draw(b);
#pragma unroll
    for (int k = 0; k < kDraws; ++k) {
      if (i0 + k >= n) continue;
      float o = 0.f;
      if constexpr (RES) o = to_f32(res[i0 + k]);
      if (limit < 65536u && keep(k)) o = fmaf(to_f32(x[i0 + k]), factor, o);
      y[i0 + k] = from_f32<TO>(o);
    }
  }
}

template <typename TI, typename TR, typename TO>
int launch_typed(long long n, const void* x, const void* res, void* y, const long long* seed, unsigned sub,
                 unsigned limit, float factor, cudaStream_t stream) {
  const bool vec = vec_aligned(x) && vec_aligned(res) && vec_aligned(y);
  constexpr long long kPerBlock = static_cast<long long>(kDropThreads) * kDropBlocks * kDraws;
  const unsigned grid = static_cast<unsigned>((n + kPerBlock - 1) / kPerBlock);
  if (vec)
    dropout_kernel<TI, TR, TO, true><<<grid, kDropThreads, 0, stream>>>(
        n, static_cast<const TI*>(x), static_cast<const TR*>(res), static_cast<TO*>(y), seed, sub, limit, factor);
  else
    dropout_kernel<TI, TR, TO, false><<<grid, kDropThreads, 0, stream>>>(
        n, static_cast<const TI*>(x), static_cast<const TR*>(res), static_cast<TO*>(y), seed, sub, limit, factor);
  return after_launch();
}

}  // namespace

int launch_dropout(bool x_bf16, bool res_bf16, bool y_bf16, long long n, const void* x, const void* res, void* y,
                   const long long* seed, unsigned sub, unsigned limit, float factor, cudaStream_t stream) {
  using B = __nv_bfloat16;
#define FH_DROP(TI, TR, TO) return launch_typed<TI, TR, TO>(n, x, res, y, seed, sub, limit, factor, stream)
  if (!res) {
    if (!x_bf16 && !y_bf16) FH_DROP(float, void, float);
    if (x_bf16 && y_bf16) FH_DROP(B, void, B);
    if (!x_bf16 && y_bf16) FH_DROP(float, void, B);
    FH_DROP(B, void, float);
  }
  if (y_bf16) {  // only where both inputs are
    if (x_bf16 && res_bf16) FH_DROP(B, B, B);
    return kUnsupported;
  }
  if (!x_bf16 && !res_bf16) FH_DROP(float, float, float);
  if (x_bf16 && !res_bf16) FH_DROP(B, float, float);
  if (!x_bf16 && res_bf16) FH_DROP(float, B, float);
  return kUnsupported;
#undef FH_DROP
}

}  // namespace fh
