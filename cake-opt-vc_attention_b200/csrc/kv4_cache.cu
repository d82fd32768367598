// Writing to and reading from the paged 4-bit K/V cache.
//
// append: K (and the call's Q) rotated by position, K and V quantised, K/V
//   codes and (scale, minimum) pairs written to their pages, Q written out.
//     rotation   y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin (FP32; each product and sum rounded)
//     64 channels of a token and head: s = bf16((max - min) * (1/15)), m = bf16(min),
//     code = clamp(rint((x - m) * (1 / s)), 0, 15), 0 where s is 0 or not finite
//   A group that holds a NaN or an infinity reads back as NaN: its (s, m) are.
//   The minimum and maximum propagate NaN for that reason.
// read: the values the cache holds, s * code + m (product and sum rounded), in
//   the caller's type.
//
// Eight channels (one 16-byte word) a thread, D/8 threads a head: a group is
// eight neighbouring lanes (three shuffles for minimum and maximum), the
// half-style rotation partner of a lane is R/16 lanes away (one shuffle a
// channel), the eight codes of a lane are one 32-bit store.
#include <type_traits>
#include "kernels.h"
#include "kv4.cuh"

namespace vcb {
namespace {

constexpr int kThreads = 256;
constexpr float kLeastNormal = 1.1754943508222875e-38f;
constexpr float kFifteenth = 1.f / 15.f;

struct AppendParams {
  const void *k, *v, *q;
  void* q_out;
  int64_t ksb, ksh, kss, vsb, vsh, vss, qsb, qsh, qss, osb, osh, oss;
  const float *cos, *sin;
  int64_t rot_rows;
  int rot_dim, interleaved;
  const int32_t *positions, *lengths, *counts;
  Kv4Pages pages;
  int64_t B, S, Hq;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// One chunk of heads a blockIdx.y: HEADS heads of Q, K, V counted through, the
// same ones in the whole block, D/8 threads a token.  The HEADS loads of a
// thread are in flight together, and cos and sin are read once for them.
template <int D, typename T, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS > 1 ? 4 : 1) kv4_append_kernel(AppendParams p) {
  constexpr int L = D / 8;   // threads a token
  const int64_t token = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / L;
  const int l = threadIdx.x % L, Hkv = static_cast<int>(p.pages.heads), Hq = static_cast<int>(p.Hq);
  const bool live = token < p.B * p.S;
  const int b = live ? static_cast<int>(token / p.S) : 0;
  const int64_t t = live ? token - b * p.S : 0;
  const bool write = live && (!p.counts || t < __ldg(p.counts + b));
  const int c0 = l * 8, first = blockIdx.y * HEADS;
  uint4 u[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int head = first + i;
    u[i] = make_uint4(0, 0, 0, 0);
    if (live && head < Hq + 2 * Hkv) {
      const T* src = head < Hq         ? static_cast<const T*>(p.q) + b * p.qsb + head * p.qsh + t * p.qss
                     : head < Hq + Hkv ? static_cast<const T*>(p.k) + b * p.ksb + (head - Hq) * p.ksh + t * p.kss
                                       : static_cast<const T*>(p.v) + b * p.vsb + (head - Hq - Hkv) * p.vsh + t * p.vss;
      u[i] = __ldg(reinterpret_cast<const uint4*>(src + c0));
    }
  }
  const int64_t at = int64_t(__ldg(p.lengths + b)) + t;   // index in the sequence
  // cos and sin of this lane's channels (half style: pair index = channel mod R/2)
  const int R = p.rot_dim, half = R / 2;
  float cs[8], sn[8];
  const bool rotated = c0 < R && first < Hq + Hkv;
  if (rotated) {
    int64_t pos = p.positions ? int64_t(__ldg(p.positions + b * p.S + t)) : at;
    if (pos < 0 || pos >= p.rot_rows) {
      if (write) raise_error(kErrBadIndex);
      pos = 0;
    }
    const float *cr = p.cos + pos * half, *sr = p.sin + pos * half;
    if (p.interleaved) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(cr + c0 / 2)), d = __ldg(reinterpret_cast<const float4*>(sr + c0 / 2));
      cs[0] = cs[1] = a.x; cs[2] = cs[3] = a.y; cs[4] = cs[5] = a.z; cs[6] = cs[7] = a.w;
      sn[0] = sn[1] = d.x; sn[2] = sn[3] = d.y; sn[4] = sn[5] = d.z; sn[6] = sn[7] = d.w;
    } else {
      const int i0 = c0 < half ? c0 : c0 - half;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(cr + i0 + i)), d = __ldg(reinterpret_cast<const float4*>(sr + i0 + i));
        cs[i] = a.x; cs[i + 1] = a.y; cs[i + 2] = a.z; cs[i + 3] = a.w;
        sn[i] = d.x; sn[i + 1] = d.y; sn[i + 2] = d.z; sn[i + 3] = d.w;
      }
    }
  }
  const int lane = threadIdx.x & 31;
  const int partner = (lane & ~(L - 1)) | (rotated ? (c0 < half ? l + half / 8 : l - half / 8) : l);
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int head = first + i;
    if (head >= Hq + 2 * Hkv) break;   // (the same in every thread: the shuffles below are warp-wide)
    float x[8];
    unpack8<T>(u[i], x);
    if (R > 0 && head < Hq + Hkv) {
      if (p.interleaved) {
        if (rotated) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float a = x[j], c = x[j + 1];
            x[j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(c, sn[j]));
            x[j + 1] = __fadd_rn(__fmul_rn(c, cs[j]), __fmul_rn(a, sn[j]));
          }
        }
      } else {
        // the partner's sixteen bytes in the input type: four shuffles
        uint4 w;
        w.x = __shfl_sync(0xffffffffu, u[i].x, partner);
        w.y = __shfl_sync(0xffffffffu, u[i].y, partner);
        w.z = __shfl_sync(0xffffffffu, u[i].z, partner);
        w.w = __shfl_sync(0xffffffffu, u[i].w, partner);
        if (rotated) {
          float y[8];
          unpack8<T>(w, y);
          if (c0 < half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __fsub_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y[j], sn[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y[j], sn[j]));
          }
        }
      }
    }
    if (head < Hq) {
      if (live) {
        T* dst = static_cast<T*>(p.q_out) + b * p.osb + head * p.osh + t * p.oss + c0;
        *reinterpret_cast<uint4*>(dst) =
            make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
      }
      continue;
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      lo = min_nan(lo, x[j]);
      hi = max_nan(hi, x[j]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (write) {
      const bool is_v = head >= Hq + Hkv;
      const int64_t rec = at < 0 ? -1 : p.pages.record<D>(b, head - Hq - (is_v ? Hkv : 0), at >> 4);
      if (rec < 0) {
        raise_error(kErrBadIndex);
        continue;
      }
      const __nv_bfloat16 m16 = __float2bfloat16_rn(lo);
      __nv_bfloat16 s16 = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), kFifteenth));
      const float m = __bfloat162float(m16);
      float s = __bfloat162float(s16);
      if (s < kLeastNormal) {
        s = 0.f;
        s16 = __float2bfloat16_rn(0.f);
      }
      const float inv = s == 0.f ? 0.f : __fdiv_rn(1.f, s);
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = rintf(__fmul_rn(__fsub_rn(x[j], m), inv));
        w |= static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) << (4 * j);   // NaN -> 0
      }
      const int slot = static_cast<int>(at & 15);
      uint8_t* r = p.pages.pool + rec;
      *reinterpret_cast<uint32_t*>(r + (is_v ? Kv4Rec<D>::kV : Kv4Rec<D>::kK) + slot * Kv4Rec<D>::kCodeRow + l * 4) = w;
      if ((l & 7) == 0) {
        const uint32_t sm = uint32_t(__bfloat16_as_ushort(s16)) | (uint32_t(__bfloat16_as_ushort(m16)) << 16);
        *reinterpret_cast<uint32_t*>(r + (is_v ? Kv4Rec<D>::kVp : Kv4Rec<D>::kKp) + slot * Kv4Rec<D>::kParRow + (l >> 3) * 4) = sm;
      }
    }
  }
}

struct ReadParams {
  void *k, *v;
  int64_t ksb, ksh, kss, vsb, vsh, vss;
  const int32_t* start;
  Kv4Pages pages;
  int64_t B, N;
};

// One thread reads 16 bytes of codes (32 channels) of one token and head, of K
// (z = 0) or V (z = 1), and writes their values.
template <int D, typename T>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(ReadParams p) {
  constexpr int L = D / 32;
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int l = static_cast<int>(i % L), which = blockIdx.z;
  const int h = blockIdx.y, n = static_cast<int>(p.N);
  const int64_t row = i / L;
  if (row >= p.B * p.N) return;
  const int b = static_cast<int>(row / n), t = static_cast<int>(row - int64_t(b) * n);
  const int64_t at = (p.start ? int64_t(__ldg(p.start + b)) : 0) + t;
  const int64_t rec = at < 0 ? -1 : p.pages.record<D>(b, h, at >> 4);
  uint4 codes = make_uint4(0, 0, 0, 0);
  uint32_t sm = 0;   // without a page: zeros
  if (rec < 0) {
    raise_error(kErrBadIndex);
  } else {
    const int slot = static_cast<int>(at & 15);
    const uint8_t* r = p.pages.pool + rec;
    codes = __ldg(reinterpret_cast<const uint4*>(r + (which ? Kv4Rec<D>::kV : Kv4Rec<D>::kK) + slot * Kv4Rec<D>::kCodeRow + l * 16));
    sm = __ldg(reinterpret_cast<const uint32_t*>(r + (which ? Kv4Rec<D>::kVp : Kv4Rec<D>::kKp) + slot * Kv4Rec<D>::kParRow + (l >> 1) * 4));
  }
  const float s = bf16_lo(sm), m = bf16_hi(sm);
  T* dst = (which ? static_cast<T*>(p.v) + b * p.vsb + h * p.vsh + t * p.vss : static_cast<T*>(p.k) + b * p.ksb + h * p.ksh + t * p.kss) + l * 32;
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(static_cast<float>((w[k] >> (4 * j)) & 15u), s), m);
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(dst)[2 * k] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(dst)[2 * k + 1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      reinterpret_cast<uint4*>(dst)[k] =
          make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
    }
  }
}

int launched() { return cudaGetLastError() == cudaSuccess ? VC_OK : VC_ERR_LAUNCH; }

}  // namespace

int kv4_append(const Kv4AppendArgs& a, cudaStream_t st) {
  AppendParams p{a.k, a.v, a.q, a.q_out, a.ksb, a.ksh, a.kss, a.vsb, a.vsh, a.vss, a.qsb, a.qsh, a.qss, a.osb, a.osh,
                 a.oss, a.cos, a.sin, a.rot_rows, static_cast<int>(a.rot_dim), a.interleaved, a.positions, a.lengths,
                 a.counts, kv4_pages(a.cache), a.cache.B, a.S, a.q ? a.Hq : 0};
  const int64_t heads = p.Hq + 2 * a.cache.Hkv, threads = a.cache.B * a.S * (a.D / 8);
  const unsigned blocks = static_cast<unsigned>((threads + kThreads - 1) / kThreads);
  // four heads a thread where that still fills the GPU several times, else one (few tokens: latency)
  const bool many = blocks * ((heads + 3) / 4) >= 4 * 148;
  const dim3 grid(blocks, static_cast<unsigned>(many ? (heads + 3) / 4 : heads));
  auto go = [&](auto tag, auto dim) {
    using T = decltype(tag);
    constexpr int D = decltype(dim)::value;
    if (many) kv4_append_kernel<D, T, 4><<<grid, kThreads, 0, st>>>(p);
    else kv4_append_kernel<D, T, 1><<<grid, kThreads, 0, st>>>(p);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (a.dtype == VC_DTYPE_BF16) a.D == 128 ? go(__nv_bfloat16(), D128()) : go(__nv_bfloat16(), D64());
  else a.D == 128 ? go(__half(), D128()) : go(__half(), D64());
  return launched();
}

int kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
  ReadParams p{a.k, a.v, a.ksb, a.ksh, a.kss, a.vsb, a.vsh, a.vss, a.start, kv4_pages(a.cache), a.cache.B, a.N};
  const int64_t threads = a.cache.B * a.N * (a.D / 32);
  const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads), static_cast<unsigned>(a.cache.Hkv), 2);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (a.D == 128) kv4_read_kernel<128, T><<<grid, kThreads, 0, st>>>(p);
    else kv4_read_kernel<64, T><<<grid, kThreads, 0, st>>>(p);
  };
  if (a.dtype == VC_DTYPE_BF16) go(__nv_bfloat16());
  else if (a.dtype == VC_DTYPE_F16) go(__half());
  else go(float());
  return launched();
}

cudaError_t kv4_cache_error_word(uint32_t* code, bool clear) { return read_tu_error_word(code, clear); }

}  // namespace vcb
