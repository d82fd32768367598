// Attention over 16-bit K/V with a sliding window and sinks: one warp a query
// row, lanes across the channels, keys one after the other.
#include "kernels.h"
#include "visible.cuh"

namespace vcb {
namespace {

constexpr int kThreads = 256;

struct RowParams {
  const void *q, *k, *v;
  void* out;
  int64_t qsb, qsh, qss, ksb, ksh, kss, vsb, vsh, vss, osb, osh, oss;
  const int32_t* kv_lengths;
  int64_t B, Hq, Hkv, Sq, Sk;
  Visibility vis;
  float scale;
};

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <int D, typename T>
__global__ void __launch_bounds__(kThreads) row_attention_kernel(RowParams p) {
  constexpr int C = D / 32;   // channels a lane
  const int64_t row = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.B * p.Hq * p.Sq) return;
  const int64_t t = row % p.Sq, h = row / p.Sq % p.Hq, b = row / p.Sq / p.Hq, hk = h / (p.Hq / p.Hkv);
  int64_t len = p.Sk;
  if (p.kv_lengths) len = max(int64_t(0), min64(__ldg(p.kv_lengths + b), p.Sk));
  const int64_t pos = p.Sk - p.Sq + t;
  const T* q = static_cast<const T*>(p.q) + b * p.qsb + h * p.qsh + t * p.qss + lane * C;
  float qv[C], o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    qv[c] = to_f32(q[c]) * p.scale;
    o[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const KeyRanges r = visible_keys(p.vis, pos, len);
  auto take = [&](int64_t j) {
    float kv[C], vv[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      kv[c] = to_f32((static_cast<const T*>(p.k) + b * p.ksb + hk * p.ksh + j * p.kss)[lane * C + c]);
      vv[c] = to_f32((static_cast<const T*>(p.v) + b * p.vsb + hk * p.vsh + j * p.vss)[lane * C + c]);
    }
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += qv[c] * kv[c];
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    const float mn = s > m || s != s ? s : m;
    const float a = m == mn ? 1.f : expf(m - mn), e = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * a + e;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = o[c] * a + e * vv[c];
    m = mn;
  };
  for (int64_t j = 0; j < r.sink_end; ++j) take(j);
  for (int64_t j = r.lo; j < r.hi; ++j) take(j);
  T* out = static_cast<T*>(p.out) + b * p.osb + h * p.osh + t * p.oss + lane * C;
#pragma unroll
  for (int c = 0; c < C; ++c) out[c] = from_f32<T>(l == 0.f ? 0.f : o[c] / l);
}

int launch_rows(const RowParams& p, int dtype, int64_t D, cudaStream_t st) {
  const int64_t rows = p.B * p.Hq * p.Sq;
  const unsigned blocks = static_cast<unsigned>((rows + kThreads / 32 - 1) / (kThreads / 32));
  if (dtype == VC_DTYPE_BF16) {
    if (D == 128) row_attention_kernel<128, __nv_bfloat16><<<blocks, kThreads, 0, st>>>(p);
    else row_attention_kernel<64, __nv_bfloat16><<<blocks, kThreads, 0, st>>>(p);
  } else {
    if (D == 128) row_attention_kernel<128, __half><<<blocks, kThreads, 0, st>>>(p);
    else row_attention_kernel<64, __half><<<blocks, kThreads, 0, st>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? VC_OK : VC_ERR_LAUNCH;
}

}  // namespace

int64_t window_attention_workspace(const WindowAttnArgs&) { return 0; }

int window_attention(const WindowAttnArgs& a, cudaStream_t st) {
  RowParams p{};
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out;
  p.qsb = a.qsb; p.qsh = a.qsh; p.qss = a.qss; p.ksb = a.ksb; p.ksh = a.ksh; p.kss = a.kss;
  p.vsb = a.vsb; p.vsh = a.vsh; p.vss = a.vss; p.osb = a.osb; p.osh = a.osh; p.oss = a.oss;
  p.kv_lengths = a.kv_lengths;
  p.B = a.B; p.Hq = a.Hq; p.Hkv = a.Hkv; p.Sq = a.Sq; p.Sk = a.Sk;
  p.vis = Visibility{a.window, a.sinks, a.causal};
  p.scale = a.sm_scale;
  return launch_rows(p, a.dtype, a.D, st);
}

}  // namespace vcb
