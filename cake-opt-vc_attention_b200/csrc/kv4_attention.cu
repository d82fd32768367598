// Attention of a few rows per K/V head over the paged 4-bit cache: decoding
// (one token a sequence) and drafts.
//
// One CTA takes up to 8*NT rows (query tokens x the query heads that share a
// K/V head) of one sequence and K/V head, and a share of its keys; each of its
// eight warps streams tiles of 32 keys on its own, with its own running
// maximum, and the warps (then the splits, in a second kernel) are joined at
// the end.
//
// Memory-bound by design: a tile is two records of 18*D bytes (K and V codes
// with their scales), each brought by one bulk copy into the warp's ring of
// shared-memory stages, so page sizes and alignment do not matter and
// 8 warps x 3 tiles a CTA keep about 200 KB an SM in flight.
//
// The codes go to the tensor core as integers; no value is dequantised:
//   S^T = K Q^T   A = K codes (m = key), B = Q (n = row).  x = s u + m gives
//     q.k = sum_g s_g (q.u)_g + m_g (sum q)_g over the groups of 64 channels.
//     A nibble in the low byte of a 16-bit lane is the FP16 denormal u 2^-24
//     (or 16 u 2^-24 in the high nibble: that Q operand is divided by 16), so
//     one AND makes an operand register, exactly.  Q is scaled by a power of
//     two per row so that it fits FP16 whatever its range (BF16 has fewer
//     significant bits, so this too is exact except for channels 2^-28 below
//     the row's largest).  FP32 accumulation of exact products.
//   O^T = V^T P^T  A = V codes (m = channel) as BF16 128 + u (exact), B = p s_g
//     split into BF16 hi + lo (17 bits), so O is as good as FP32 arithmetic for
//     both input types; sum_j p_j (m - 128 s)_jg is accumulated in FP32 beside
//     it.  BF16 and not FP16 because p s has the range of the data.
//   S^T's accumulator layout becomes P^T's operand layout by one 8x8 transpose
//   (movmatrix) a register.
// The maximum that the exponents are taken against moves only when a logit
// exceeds it by more than 8 (in powers of two): until then p <= 2^8, which
// costs no precision, and the 32*NT accumulators are not rescaled.
#include <type_traits>
#include "join.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "visible.cuh"

namespace vcb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;        // keys of a warp's tile: two records
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;

struct DecodeParams {
  const void* q;
  void* out;
  int64_t qsb, qsh, qss, osb, osh, oss;
  const int32_t *lengths, *q_lengths;
  Kv4Pages pages;
  int64_t Hq, Sq;
  int G;               // query heads a K/V head
  int rows;            // Sq * G
  int splits;
  Visibility vis;
  float scale_log2;    // sm_scale * log2(e)
  float* part_o;       // [B*Hkv*rows, splits, D] (splits > 1)
  float2* part_ml;     // [B*Hkv*rows, splits]: running maximum (log2 units), sum
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf162_bits(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}

// Eight consecutive 16-bit values as FP32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}


template <int D, int NT>
struct DecodeSmem {
  static constexpr int kStages = 3;
  static constexpr int kTileBytes = 2 * Kv4Rec<D>::kBytes;
  static constexpr int kRing = kWarps * kStages * kTileBytes;
  static constexpr int kMerge = kWarps * 8 * (D + 4) * 4;         // one n-tile's O of every warp (row stride D + 4)
  static constexpr int kOffBar = kRing > kMerge ? kRing : kMerge;
  static constexpr int kOffStat = kOffBar + kWarps * kStages * 8; // float2 [warps][8 NT]
  static constexpr int kBytes = kOffStat + kWarps * 8 * NT * 8;
};

template <int D, typename T, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) kv4_decode_kernel(DecodeParams p) {
  using R = Kv4Rec<D>;
  using L = DecodeSmem<D, NT>;
  constexpr int NG = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int split = blockIdx.x;
  const int64_t bh = blockIdx.y, b = bh / p.pages.heads, hk = bh % p.pages.heads;
  const int row0 = blockIdx.z * 8 * NT;
  int len, nq;
  kv4_sequence(p.pages, p.lengths, p.q_lengths, static_cast<int>(p.Sq), b, len, nq);
  const int live_rows = nq * p.G;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + warp * L::kStages;
  if (lane == 0)
    for (int s = 0; s < L::kStages; ++s) mbar_init(&bars[s], 1);
  fence_barrier_init();
  __syncwarp();

  // keys that some row of this CTA sees, in tiles of 32: sinks [0, nsink) and [main0, main0 + nmain)
  int nsink = 0, main0 = 0, ntiles = 0;
  const int last_row = min(row0 + 8 * NT, live_rows) - 1;
  int pos_first = 0, pos_last = 0;
  if (last_row >= row0) {
    pos_first = len - nq + row0 / p.G;
    pos_last = len - nq + last_row / p.G;
    const KeyRanges a = visible_keys(p.vis, pos_first, len), z = visible_keys(p.vis, pos_last, len);
    const int lo = p.vis.window ? a.lo : 0, hi = z.hi;   // the last row reaches furthest, the first starts first
    const int sink_end = p.vis.window ? min(p.vis.sinks, hi) : 0;
    main0 = lo / kTile;
    const int end = (hi + kTile - 1) / kTile;
    nsink = min((sink_end + kTile - 1) / kTile, main0);
    ntiles = nsink + (end > main0 ? end - main0 : 0);
  }
  const int t_begin = static_cast<int>(int64_t(ntiles) * split / p.splits);
  const int t_end = static_cast<int>(int64_t(ntiles) * (split + 1) / p.splits);
  const int i0 = t_begin + warp;
  const int mine = i0 < t_end ? (t_end - i0 + kWarps - 1) / kWarps : 0;

  // ring: lanes 0 and 1 bring a record each; okbits: which of the lane's stages hold one
  uint8_t* ring = smem + warp * L::kStages * L::kTileBytes;
  uint32_t okbits = 0;
  auto tile_of = [&](int i) -> int {
    const int t = i0 + i * kWarps;
    return t < nsink ? t : main0 + (t - nsink);
  };
  auto locate = [&](int i) -> int64_t {   // lanes 0 and 1: the record's offset, -1 past the end, -2 without a page
    if (lane > 1 || i >= mine) return -1;
    const int blk = tile_of(i) * 2 + lane;
    if (blk * kKv4Block >= len) return -1;
    const int64_t rec = p.pages.record<D>(b, hk, blk);
    return rec < 0 ? -2 : rec;
  };
  auto issue = [&](int i, int64_t rec) {
    const int s = i % L::kStages;
    if (rec == -2) raise_error(kErrBadIndex);
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, rec >= 0));
    okbits = (okbits & ~(1u << s)) | (rec >= 0 ? 1u << s : 0u);
    if (lane == 0) mbar_expect_tx(&bars[s], n * R::kBytes);
    __syncwarp();
    if (rec >= 0) bulk_load(ring + s * L::kTileBytes + lane * R::kBytes, p.pages.pool + rec, R::kBytes, &bars[s]);
  };
  int64_t next = locate(0);
  for (int i = 0; i < L::kStages - 1 && i < mine; ++i) {
    const int64_t rec = next;
    next = locate(i + 1);
    issue(i, rec);
  }

  // Q operands of this warp's (all) rows; row n = r of each n-tile
  uint32_t qf[NT][NG][2][4];   // [word of 8 channels][b0 step 0, b1 step 0, b0 step 1, b1 step 1]
  float acol[NT][2], qsum[NT][NG][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + nt * 8 + r;
    float x[NG][16];
    float big = 0.f, sum[NG];
    const bool have = row < p.rows;
    const T* src = static_cast<const T*>(p.q) + b * p.qsb + (hk * p.G + (have ? row % p.G : 0)) * p.qsh + (have ? row / p.G : 0) * p.qss;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      load8(src + 64 * g + 16 * c, x[g]);
      load8(src + 64 * g + 16 * c + 8, x[g] + 8);
      sum[g] = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        big = fmaxf(big, fabsf(x[g][j]));
        sum[g] += x[g][j];
      }
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // a power of two that brings the row's largest value to [2^14, 2^15)
    int e = big > 0.f ? 14 + 127 - static_cast<int>(__float_as_uint(big) >> 23) : 0;
    e = max(-100, min(126, e));
    const float up = __uint_as_float(uint32_t(127 + e) << 23), up16 = up * 0.0625f;
    const float ac = __uint_as_float(uint32_t(127 - e) << 23) * 16777216.f * p.scale_log2;   // 2^(24 - e) scale
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float* y = x[g] + 8 * w;
        qf[nt][g][w][0] = half2_bits(y[0] * up, y[4] * up);
        qf[nt][g][w][1] = half2_bits(y[1] * up16, y[5] * up16);
        qf[nt][g][w][2] = half2_bits(y[2] * up, y[6] * up);
        qf[nt][g][w][3] = half2_bits(y[3] * up16, y[7] * up16);
      }
#pragma unroll
    for (int k = 0; k < 2; ++k) {   // this thread's accumulator columns are rows 2c and 2c + 1
      acol[nt][k] = __shfl_sync(0xffffffffu, ac, (2 * c + k) * 4);
#pragma unroll
      for (int g = 0; g < NG; ++g) qsum[nt][g][k] = __shfl_sync(0xffffffffu, sum[g], (2 * c + k) * 4) * p.scale_log2;
    }
  }

  float o[NT][NG][4][4];
  float m[NT][2], l[NT][2], vm[NT][NG][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[nt][k] = -INFINITY;
      l[nt][k] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        vm[nt][g][k] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][g][i][2 * k] = o[nt][g][i][2 * k + 1] = 0.f;
      }
    }

  // logical key row r of a record's m-tile is token pi(r) = r/2 + 4 (r%2) (and 8 + that for r + 8), so that
  // the V loads of the four c lanes, keys {c, c+4, c+8, c+12}, spread over the banks
  const int tok = (r >> 1) + 4 * (r & 1);
  // rows see all of a tile iff it ends before every row's last key and starts after every row's first
  const KeyRanges first = visible_keys(p.vis, pos_first, len);
  const int last_lo = visible_keys(p.vis, pos_last, len).lo;
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    {
      const int64_t rec = next;
      next = locate(i + L::kStages);
      if (i + L::kStages - 1 < mine) issue(i + L::kStages - 1, rec);
    }
    const int s = i % L::kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[s], (i / L::kStages) & 1, kErrTimeoutTma));
    if (!ok) break;
    const uint32_t have = __ballot_sync(0xffffffffu, (okbits >> s) & 1u) & 3u;
    const int key0 = tile_of(i) * kTile;
    const bool whole = have == 3u && key0 + kTile <= first.hi &&
                       (p.vis.window == 0 || key0 >= last_lo || key0 + kTile <= p.vis.sinks);
    const uint32_t base = smem_u32(ring + s * L::kTileBytes);
    float x[2][NT][4];
    uint2 vpar[2][2];   // V (scale, minimum) of token rows r and r + 8; .y the second group
#pragma unroll
    for (int k = 0; k < 2; ++k) {   // the two records
      const uint32_t rec = base + k * R::kBytes;
      float acc[NT][NG][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[nt][g][j] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 ca = lds64(rec + R::kK + tok * R::kCodeRow + g * 32 + c * 8);
        const uint2 cb = lds64(rec + R::kK + (tok + 8) * R::kCodeRow + g * 32 + c * 8);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t a = w ? ca.y : ca.x, bq = w ? cb.y : cb.x;
          const uint32_t a8 = a >> 8, b8 = bq >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][g], a & 0x000F000Fu, bq & 0x000F000Fu, a & 0x00F000F0u, bq & 0x00F000F0u, qf[nt][g][w][0], qf[nt][g][w][1]);
            mma_f16(acc[nt][g], a8 & 0x000F000Fu, b8 & 0x000F000Fu, a8 & 0x00F000F0u, b8 & 0x00F000F0u, qf[nt][g][w][2], qf[nt][g][w][3]);
          }
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = tok + 8 * half;
        uint2 kp;
        if constexpr (NG == 2) {
          kp = lds64(rec + R::kKp + t * R::kParRow);
          vpar[k][half] = lds64(rec + R::kVp + t * R::kParRow);
        } else {
          kp = make_uint2(lds32(rec + R::kKp + t * R::kParRow), 0u);
          vpar[k][half] = make_uint2(lds32(rec + R::kVp + t * R::kParRow), 0u);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float u = acc[nt][0][2 * half + j] * bf16_lo(kp.x), y = bf16_hi(kp.x) * qsum[nt][0][j];
            if constexpr (NG == 2) {
              u = fmaf(acc[nt][NG - 1][2 * half + j], bf16_lo(kp.y), u);
              y = fmaf(bf16_hi(kp.y), qsum[nt][NG - 1][j], y);
            }
            x[k][nt][2 * half + j] = fmaf(u, acol[nt][j], y);
          }
      }
    }
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = row0 + nt * 8 + 2 * c + j;
          const KeyRanges v = visible_keys(p.vis, len - nq + row / p.G, len);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int key = key0 + 16 * k + tok + 8 * half;
              const bool see = ((have >> k) & 1u) && key < v.hi && (key >= v.lo || key < v.sink_end);
              if (!see) x[k][nt][2 * half + j] = -INFINITY;
            }
        }
    }
    // move the maxima only if some logit is far above its own
    bool far = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float top = fmaxf(fmaxf(x[0][nt][j], x[0][nt][2 + j]), fmaxf(x[1][nt][j], x[1][nt][2 + j]));
        far |= top > m[nt][j] + kLazy;
      }
    if (__any_sync(0xffffffffu, far)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(fmaxf(x[0][nt][j], x[0][nt][2 + j]), fmaxf(x[1][nt][j], x[1][nt][2 + j]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float mn = fmaxf(m[nt][j], top);
          const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m[nt][j] - mn);
          m[nt][j] = mn;
          l[nt][j] *= alpha;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            vm[nt][g][j] *= alpha;
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
              o[nt][g][i4][j] *= alpha;
              o[nt][g][i4][2 + j] *= alpha;
            }
          }
        }
    }
    // probabilities, then O^T += V^T P^T
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t rec = base + k * R::kBytes;
      uint32_t bh_[NT][NG][2], bl_[NT][NG][2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float s0 = bf16_lo(vpar[k][half].x), s1 = bf16_lo(vpar[k][half].y);
        const float m0 = fmaf(-128.f, s0, bf16_hi(vpar[k][half].x)), m1 = fmaf(-128.f, s1, bf16_hi(vpar[k][half].y));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float e[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float v = x[k][nt][2 * half + j];
            e[j] = v == -INFINITY ? 0.f : exp2_fast(v - m[nt][j]);
            l[nt][j] += e[j];
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float sg = g ? s1 : s0, mg = g ? m1 : m0;
            float w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // a hidden key's scale may be anything: its weight is zero, not 0 * scale
              const bool hid = x[k][nt][2 * half + j] == -INFINITY;
              w[j] = hid ? 0.f : e[j] * sg;
              vm[nt][g][j] += hid ? 0.f : e[j] * mg;
            }
            const uint32_t hi = bf162_bits(w[0], w[1]);
            const uint32_t lo = bf162_bits(w[0] - bf16_lo(hi), w[1] - bf16_hi(hi));
            bh_[nt][g][half] = transpose8x8(hi);
            bl_[nt][g][half] = transpose8x8(lo);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t at = rec + R::kV + g * 32 + r * 4;
        const uint32_t w0 = lds32(at + c * R::kCodeRow), w1 = lds32(at + (c + 4) * R::kCodeRow);
        const uint32_t w2 = lds32(at + (c + 8) * R::kCodeRow), w3 = lds32(at + (c + 12) * R::kCodeRow);
        const uint32_t la = __byte_perm(w0, w1, 0x5410), ha = __byte_perm(w0, w1, 0x7632);
        const uint32_t lb = __byte_perm(w2, w3, 0x5410), hb = __byte_perm(w2, w3, 0x7632);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const uint32_t a0 = ((la >> (4 * i4)) & 0x000F000Fu) | 0x43004300u, a1 = ((ha >> (4 * i4)) & 0x000F000Fu) | 0x43004300u;
          const uint32_t a2 = ((lb >> (4 * i4)) & 0x000F000Fu) | 0x43004300u, a3 = ((hb >> (4 * i4)) & 0x000F000Fu) | 0x43004300u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16(o[nt][g][i4], a0, a1, a2, a3, bh_[nt][g][0], bh_[nt][g][1]);
            mma_bf16(o[nt][g][i4], a0, a1, a2, a3, bl_[nt][g][0], bl_[nt][g][1]);
          }
        }
      }
    }
    __syncwarp();   // every lane has read the stage that the next issue overwrites
  }

  // join the warps: sums over the lanes of a column, then maxima and sums over the warps
  float2* stat = reinterpret_cast<float2*>(smem + L::kOffStat);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], sh);
#pragma unroll
        for (int g = 0; g < NG; ++g) vm[nt][g][j] += __shfl_xor_sync(0xffffffffu, vm[nt][g][j], sh);
      }
      if (r == 0) stat[warp * 8 * NT + nt * 8 + 2 * c + j] = make_float2(m[nt][j], l[nt][j]);
    }
  __syncthreads();
  float* merge = reinterpret_cast<float*>(smem);
  constexpr int kRow = D + 4;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat[w * 8 * NT + nt * 8 + 2 * c + j].x);
      const float f = m[nt][j] == -INFINITY ? 0.f : exp2_fast(m[nt][j] - top);
      float* row = merge + (warp * 8 + 2 * c + j) * kRow;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float v[8];
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          v[i4] = (o[nt][g][i4][j] + vm[nt][g][j]) * f;
          v[4 + i4] = (o[nt][g][i4][2 + j] + vm[nt][g][j]) * f;
        }
        *reinterpret_cast<float4*>(row + 64 * g + 8 * r) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + 64 * g + 8 * r + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
    __syncthreads();
    // warp w joins row w of this n-tile; lane: D/32 channels
    const int row = row0 + nt * 8 + warp;
    if (row < p.rows) {
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat[w * 8 * NT + nt * 8 + warp].x);
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = stat[w * 8 * NT + nt * 8 + warp];
        sum += ml.x == -INFINITY ? ml.y : ml.y * exp2_fast(ml.x - top);   // no maximum: 0, or NaN if all logits are
      }
      constexpr int C = D / 32;
      float v[C];
#pragma unroll
      for (int k = 0; k < C; ++k) v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
#pragma unroll
        for (int k = 0; k < C; ++k) v[k] += merge[(w * 8 + warp) * kRow + lane * C + k];
      const bool dead = row >= live_rows || sum == 0.f;   // nothing seen
      if (p.splits == 1) {
        T h[C];
#pragma unroll
        for (int k = 0; k < C; ++k) h[k] = from_f32<T>(dead ? 0.f : v[k] / sum);
        T* dst = static_cast<T*>(p.out) + b * p.osb + (hk * p.G + row % p.G) * p.osh + int64_t(row / p.G) * p.oss + lane * C;
        if constexpr (C == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(h);
        else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(h);
      } else {
        const int64_t at = (bh * p.rows + row) * p.splits + split;
        float* dst = p.part_o + at * D + lane * C;
#pragma unroll
        for (int k = 0; k < C; ++k) dst[k] = dead ? 0.f : v[k];
        if (lane == 0) p.part_ml[at] = dead ? make_float2(-INFINITY, 0.f) : make_float2(top, sum);
      }
    }
    __syncthreads();
  }
}

struct Plan {
  int nt, blocks, splits;
};

// Rows a CTA (8, 16 or 32) and splits of the keys: enough CTAs to fill the
// GPU twice over, at least one tile a warp each.
Plan plan_of(const Kv4AttnArgs& a) {
  const int64_t rows = a.Sq * (a.Hq / a.cache.Hkv);
  Plan r;
  r.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  r.blocks = static_cast<int>((rows + 8 * r.nt - 1) / (8 * r.nt));
  int64_t keys = kv4_most(a.cache, a.max_length);
  if (a.window > 0) keys = min64(keys, a.window + a.Sq + a.sinks + 2 * kTile);
  const int64_t tiles = (keys + kTile - 1) / kTile, items = a.cache.B * a.cache.Hkv * r.blocks;
  int64_t s = (4 * 148 + items - 1) / items;
  s = min64(s, (tiles + kWarps - 1) / kWarps);
  r.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
  return r;
}

// From this many rows a K/V head on, the tile kernel.
constexpr int64_t kTileRows = 64;
bool use_tiles(const Kv4AttnArgs& a) { return a.Sq * (a.Hq / a.cache.Hkv) >= kTileRows; }

int launched() { return cudaGetLastError() == cudaSuccess ? VC_OK : VC_ERR_LAUNCH; }

template <int D, typename T, int NT>
int launch_decode(const DecodeParams& p, const Plan& plan, int64_t BH, cudaStream_t st) {
  auto* k = kv4_decode_kernel<D, T, NT>;
  constexpr int bytes = DecodeSmem<D, NT>::kBytes;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(reinterpret_cast<const void*>(k), bytes, ready)) return VC_ERR_LAUNCH;
  k<<<dim3(plan.splits, static_cast<unsigned>(BH), plan.blocks), kThreads, bytes, st>>>(p);
  if (plan.splits > 1) {
    const JoinParams j{p.part_o, p.part_ml, p.out, p.osb, p.osh, p.oss, p.pages.heads, p.rows, p.G, p.splits};
    launch_join<D, T>(j, BH * p.rows, st);
  }
  return launched();
}

template <int D, typename T>
int launch(const DecodeParams& p, const Plan& plan, int64_t BH, cudaStream_t st) {
  if (plan.nt == 1) return launch_decode<D, T, 1>(p, plan, BH, st);
  if (plan.nt == 2) return launch_decode<D, T, 2>(p, plan, BH, st);
  return launch_decode<D, T, 4>(p, plan, BH, st);
}

}  // namespace

int64_t kv4_attention_workspace(const Kv4AttnArgs& a) {
  if (use_tiles(a)) return kv4_chunk_workspace(a);
  const Plan plan = plan_of(a);
  if (plan.splits == 1) return 0;
  return a.cache.B * a.Hq * a.Sq * plan.splits * (a.D + 2) * 4;
}

int kv4_attention(const Kv4AttnArgs& a, cudaStream_t st) {
  if (use_tiles(a)) return kv4_chunk_attention(a, st);
  const Plan plan = plan_of(a);
  const int64_t BH = a.cache.B * a.cache.Hkv;
  DecodeParams p;
  p.q = a.q;
  p.out = a.out;
  p.qsb = a.qsb; p.qsh = a.qsh; p.qss = a.qss;
  p.osb = a.osb; p.osh = a.osh; p.oss = a.oss;
  p.lengths = a.lengths;
  p.q_lengths = a.q_lengths;
  p.pages = kv4_pages(a.cache, a.max_length);
  p.Hq = a.Hq;
  p.Sq = a.Sq;
  p.G = static_cast<int>(a.Hq / a.cache.Hkv);
  p.rows = static_cast<int>(a.Sq * p.G);
  p.splits = plan.splits;
  p.vis = visibility(a.window, a.sinks, a.causal);
  p.scale_log2 = a.sm_scale * kLog2e;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + BH * p.rows * plan.splits * a.D);
  if (a.dtype == VC_DTYPE_BF16) return a.D == 128 ? launch<128, __nv_bfloat16>(p, plan, BH, st) : launch<64, __nv_bfloat16>(p, plan, BH, st);
  return a.D == 128 ? launch<128, __half>(p, plan, BH, st) : launch<64, __half>(p, plan, BH, st);
}

cudaError_t kv4_attention_error_word(uint32_t* code, bool clear) { return read_tu_error_word(code, clear); }

}  // namespace vcb
