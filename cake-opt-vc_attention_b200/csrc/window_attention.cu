// Attention over 16-bit K/V with a sliding window and sinks: tensor maps and
// dispatch of the tile kernel (tile_attention.cuh).
#include "tile_attention.cuh"

namespace vcb {
namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn get_encode() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeFn>(ptr) : nullptr;
  }();
  return fn;
}

// [B, H, S, D] 16-bit tensor through its strides; boxes of 64 channels x 128 tokens.
bool make_map(CUtensorMap* m, const void* base, int dtype, int64_t B, int64_t H, int64_t S, int64_t D, int64_t sb,
              int64_t sh, int64_t ss) {
  EncodeFn enc = get_encode();
  if (!enc) return false;
  const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(S), cuuint64_t(H), cuuint64_t(B)};
  const cuuint64_t strides[3] = {cuuint64_t(ss) * 2, cuuint64_t(sh) * 2, cuuint64_t(sb) * 2};
  const cuuint32_t box[4] = {64, 128, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(m, dtype == VC_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

TilePlan plan_of(const WindowAttnArgs& a) {
  const int64_t G = a.Hq / a.Hkv;
  return tile_plan(a.B * a.Hkv, a.Sq * G, G, a.Sk, visibility(a.window, a.sinks, a.causal));
}

}  // namespace

int64_t window_attention_workspace(const WindowAttnArgs& a) {
  const TilePlan t = plan_of(a);
  return t.splits == 1 ? 0 : a.B * a.Hq * a.Sq * t.splits * (a.D + 2) * 4;
}

int window_attention(const WindowAttnArgs& a, cudaStream_t st) {
  const TilePlan t = plan_of(a);
  CUtensorMap mk, mv;
  // without keys nothing is loaded: the maps then describe q, which is there
  const bool none = a.Sk == 0;
  const int64_t H = none ? a.Hq : a.Hkv, S = none ? a.Sq : a.Sk;
  if (!make_map(&mk, none ? a.q : a.k, a.dtype, a.B, H, S, a.D, none ? a.qsb : a.ksb, none ? a.qsh : a.ksh, none ? a.qss : a.kss) ||
      !make_map(&mv, none ? a.q : a.v, a.dtype, a.B, H, S, a.D, none ? a.qsb : a.vsb, none ? a.qsh : a.vsh, none ? a.qss : a.vss)) {
    set_last_error("vc_window_attention_fwd: cuTensorMapEncodeTiled failed");
    return VC_ERR_LAUNCH;
  }
  TileParams p{};
  p.q = a.q;
  p.out = a.out;
  p.qsb = a.qsb; p.qsh = a.qsh; p.qss = a.qss;
  p.osb = a.osb; p.osh = a.osh; p.oss = a.oss;
  p.Hkv = static_cast<int>(a.Hkv);
  p.BH = static_cast<int>(a.B * a.Hkv);
  p.Sq = a.Sq;
  p.Sk = a.Sk;
  p.G = static_cast<int>(a.Hq / a.Hkv);
  p.rows = static_cast<int>(a.Sq * p.G);
  p.pairs = static_cast<int>(t.pairs);
  p.splits = static_cast<int>(t.splits);
  p.vis = visibility(a.window, a.sinks, a.causal);
  p.scale_log2 = a.sm_scale * kLog2e;
  p.lengths = a.kv_lengths;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + int64_t(p.BH) * p.rows * t.splits * a.D);
  if (a.dtype == VC_DTYPE_BF16)
    return a.D == 128 ? launch_tiles<128, __nv_bfloat16, __nv_bfloat16, false>(mk, mv, p, st)
                      : launch_tiles<64, __nv_bfloat16, __nv_bfloat16, false>(mk, mv, p, st);
  return a.D == 128 ? launch_tiles<128, __half, __half, false>(mk, mv, p, st)
                    : launch_tiles<64, __half, __half, false>(mk, mv, p, st);
}

cudaError_t window_attention_error_word(uint32_t* code, bool clear) { return read_tu_error_word(code, clear); }

}  // namespace vcb
