// Attention over 16-bit K/V with a sliding window and sinks: tensor maps and
// dispatch of the tile kernel (tile_attention.cuh).
#include "tile_attention.cuh"

namespace vcb {
namespace {

TilePlan plan_of(const WindowAttnArgs& a) {
  const int64_t G = a.Hq / a.Hkv;
  return tile_plan(a.B * a.Hkv, a.Sq * G, G, a.Sk, visibility(a.window, a.sinks, a.causal));
}

}  // namespace

int64_t window_attention_workspace(const WindowAttnArgs& a) {
  return plan_of(a).part_rows() * (a.D + 2) * 4;
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
  p.vis = visibility(a.window, a.sinks, a.causal);
  p.scale_log2 = a.sm_scale * kLog2e;
  p.lengths = a.kv_lengths;
  set_plan(p, t, a.workspace, a.D);
  if (a.dtype == VC_DTYPE_BF16)
    return a.D == 128 ? launch_tiles<128, __nv_bfloat16, __nv_bfloat16, kTensors>(mk, mv, p, st)
                      : launch_tiles<64, __nv_bfloat16, __nv_bfloat16, kTensors>(mk, mv, p, st);
  return a.D == 128 ? launch_tiles<128, __half, __half, kTensors>(mk, mv, p, st)
                    : launch_tiles<64, __half, __half, kTensors>(mk, mv, p, st);
}

cudaError_t window_attention_error_word(uint32_t* code, bool clear) { return read_tu_error_word(code, clear); }

}  // namespace vcb
