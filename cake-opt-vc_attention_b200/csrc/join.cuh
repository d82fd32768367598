// Partial attention results of a row whose keys were split over CTAs, and the
// kernel that joins them.
//
// Split s of a row leaves an unnormalised output O_s [D], the maximum m_s that
// its exponents were taken against (in powers of two; -inf: saw nothing) and
// its sum l_s.  The row is sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s with
// m = max m_s, summed in the order of s.
#pragma once
#include <atomic>
#include "common.cuh"

namespace vcb {

// Allows ``bytes`` of dynamic shared memory for a kernel, once a device (the
// attribute call costs about as much as a launch).  ``ready``: devices done.
inline bool allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit && (ready.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  ready.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

struct JoinParams {
  const float* part_o;    // [rows of all heads, splits, D]
  const float2* part_ml;  // [rows of all heads, splits]
  void* out;
  int64_t osb, osh, oss;
  int64_t heads;          // K/V heads
  int rows, G, splits;    // rows a K/V head: token r / G, query head hk * G + r % G
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One warp a row, D/32 channels a lane.
template <int D, typename T>
__global__ void __launch_bounds__(128) join_splits_kernel(JoinParams p, int64_t total) {
  const int64_t i = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= total) return;
  const float2* ml = p.part_ml + i * p.splits;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr int C = D / 32;
  float v[C], sum = 0.f;
#pragma unroll
  for (int k = 0; k < C; ++k) v[k] = 0.f;
  const float* src = p.part_o + i * p.splits * D + lane * C;
  for (int s = 0; s < p.splits; ++s) {
    const float2 a = ml[s];
    const float f = a.x == -INFINITY ? 0.f : exp2_fast(a.x - top);
    sum += a.x == -INFINITY ? a.y : a.y * f;   // without a maximum: 0, or NaN where every logit is
#pragma unroll
    for (int k = 0; k < C; ++k) v[k] += src[s * D + k] * f;
  }
  const int row = static_cast<int>(i % p.rows);
  const int64_t bh = i / p.rows, b = bh / p.heads, hk = bh % p.heads;
  T h[C];
#pragma unroll
  for (int k = 0; k < C; ++k) h[k] = from_f32<T>(sum == 0.f ? 0.f : v[k] / sum);
  T* dst = static_cast<T*>(p.out) + b * p.osb + (hk * p.G + row % p.G) * p.osh + int64_t(row / p.G) * p.oss + lane * C;
  if constexpr (C == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(h);
  else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(h);
}

template <int D, typename T>
inline void launch_join(const JoinParams& p, int64_t total, cudaStream_t st) {
  join_splits_kernel<D, T><<<static_cast<unsigned>((total + 3) / 4), 128, 0, st>>>(p, total);
}

}  // namespace vcb
