// Chunks of queries over the 4-bit cache: dispatch of the tile kernel
// (tile_attention.cuh) with its dequantising producers.
#include "tile_attention.cuh"

namespace vcb {
namespace {

TilePlan plan_of(const Kv4AttnArgs& a) {
  const int64_t G = a.Hq / a.cache.Hkv;
  int64_t keys = a.cache.width * a.cache.page_size;
  if (a.max_length > 0) keys = min64(keys, a.max_length);
  return tile_plan(a.cache.B * a.cache.Hkv, a.Sq * G, G, keys, visibility(a.window, a.sinks, a.causal));
}

}  // namespace

int64_t kv4_chunk_workspace(const Kv4AttnArgs& a) {
  const TilePlan t = plan_of(a);
  return t.splits == 1 ? 0 : a.cache.B * a.Hq * a.Sq * t.splits * (a.D + 2) * 4;
}

int kv4_chunk_attention(const Kv4AttnArgs& a, cudaStream_t st) {
  const TilePlan t = plan_of(a);
  TileParams p{};
  p.q = a.q;
  p.out = a.out;
  p.qsb = a.qsb; p.qsh = a.qsh; p.qss = a.qss;
  p.osb = a.osb; p.osh = a.osh; p.oss = a.oss;
  p.Hkv = static_cast<int>(a.cache.Hkv);
  p.BH = static_cast<int>(a.cache.B * a.cache.Hkv);
  p.Sq = a.Sq;
  p.G = static_cast<int>(a.Hq / a.cache.Hkv);
  p.rows = static_cast<int>(a.Sq * p.G);
  p.pairs = static_cast<int>(t.pairs);
  p.splits = static_cast<int>(t.splits);
  p.vis = visibility(a.window, a.sinks, a.causal);
  p.scale_log2 = a.sm_scale * kLog2e;
  p.lengths = a.lengths;
  p.q_lengths = a.q_lengths;
  p.pages = kv4_pages(a.cache);
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + int64_t(p.BH) * p.rows * t.splits * a.D);
  const CUtensorMap none{};   // K/V come from the cache's records
  if (a.dtype == VC_DTYPE_BF16)
    return a.D == 128 ? launch_tiles<128, __half, __nv_bfloat16, true>(none, none, p, st)
                      : launch_tiles<64, __half, __nv_bfloat16, true>(none, none, p, st);
  return a.D == 128 ? launch_tiles<128, __half, __half, true>(none, none, p, st)
                    : launch_tiles<64, __half, __half, true>(none, none, p, st);
}

cudaError_t kv4_chunk_error_word(uint32_t* code, bool clear) { return read_tu_error_word(code, clear); }

}  // namespace vcb
