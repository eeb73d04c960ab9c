// C ABI of the operators that attend to the paged cache: attention (with weight sums), block bounds, block choice.
// No allocation, no synchronisation, no exceptions: every entry returns a triattn_status.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/triattn_b200.h"
#include "attend.cuh"
#include "attend_tma.cuh"
#include "attend_umma.cuh"
#include "blocks.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "tensor_map.cuh"

using namespace triattn;

namespace {

// Which attention kernel serves a call, from its geometry alone.
//   decode   at most 16 query rows per KV head (query tokens x group size), block sizes that are multiples of 8: cache tiles by
//            tiled TMA, products on mma.sync
//   tree     more rows (head dimensions 64 and 128): the same ring, products on tcgen05, 128 rows or, above that, 256 per CTA
//   general  everything else: tiles gathered token by token with cp.async
enum class AttendKind { kGeneral, kDecode, kTree };
struct AttendPlan {
  AttendKind kind;
  int tile, rows;  // tokens per tile, query rows per row tile
  int mt;          // general kernel: 16-row groups of the tile
  bool split_p;    // at most 8 rows: probabilities in two bf16 parts
  int runs, min_tiles, box;  // runs per KV head
  size_t part_o, part_ml, bytes;
};

long long attend_max_tiles(const triattn_paged_layout& Y, int max_q, int num_listed, int tile, int rows) {
  long long blocks = Y.max_blocks_per_req;
  if (num_listed > 0) blocks = std::min<long long>(blocks, num_listed);
  const long long tiles = (blocks * Y.block_size + tile - 1) / tile;
  const long long row_tiles = ((long long)max_q * Y.group_size + rows - 1) / rows;
  return tiles * row_tiles * Y.num_reqs;
}

// Runs per KV head on `slots` resident CTAs: as many as fit, or as fit twice where once leaves over 7 % of the slots idle.
int attend_max_runs(int slots, int heads) {
  int runs = slots / heads;
  if (runs * heads * 100 < slots * 93) runs = std::max(1, 2 * slots / heads);
  return runs;
}

// The stride of an axis with one entry says nothing: give it the value the tensor maps want.
triattn_paged_layout with_plain_strides(const triattn_paged_layout& L) {
  triattn_paged_layout Y = L;
  if (Y.num_blocks == 1) Y.block_stride = std::max(Y.block_size * Y.token_stride, Y.num_kv_heads * Y.head_stride);
  if (Y.num_kv_heads == 1) Y.head_stride = Y.block_stride;
  else if (Y.num_blocks == 1) Y.block_stride = (Y.block_stride + Y.head_stride - 1) / std::max<int64_t>(Y.head_stride, 1) * Y.head_stride;
  return Y;
}

// Can the layer's K and V be described by the tensor maps of attend_tma.cuh?
bool tileable(const triattn_paged_layout& Y) {
  const int64_t strides[3] = {Y.block_stride, Y.token_stride, Y.head_stride};
  for (int64_t s : strides)
    if (s <= 0 || s >= (1ll << 35)) return false;
  return Y.block_size % 8 == 0 && Y.block_stride % Y.head_stride == 0 &&
         Y.num_blocks * (Y.block_stride / Y.head_stride) < (1ll << 31);
}

// Tiles per warp up to which one CTA takes all of a KV head's tiles.  One request, 8 heads, on the device: 150 tokens 8.5 us whole and 9.2
// in parts with the launch that joins them, 300 tokens 9.6 and 10.8, 517 (three tiles per warp) 11.8 and 11.1, 1100 16.7 and 11.9.
constexpr int kDecodeWholeTiles = 2;

AttendPlan attend_plan(const triattn_paged_layout& Y, int max_q, int num_listed) {
  AttendPlan a{};
  const long long R = (long long)max_q * Y.group_size;
  a.split_p = R <= 8;
  a.min_tiles = 1;
  int ctas = kSMs;
  if (R <= 16 && tileable(Y)) {
    a.kind = AttendKind::kDecode;
    a.tile = Y.head_dim == 64 ? kDecodeTile<64> : Y.head_dim == 128 ? kDecodeTile<128> : kDecodeTile<256>;
    a.rows = a.split_p ? 8 : 16;
    a.min_tiles = kDecodeWarps;
  } else if (tileable(Y) && Y.head_dim <= 128) {
    a.kind = AttendKind::kTree;
    a.tile = kTreeTile;
    a.rows = R <= 128 ? 128 : 256;
    a.min_tiles = 2;
  } else {
    a.kind = AttendKind::kGeneral;
    a.tile = kAttendTile;
    a.mt = R <= 16 ? 1 : R <= 32 ? 2 : 4;
    a.rows = a.split_p ? 8 : 16 * a.mt;
    if (Y.head_dim <= 128) ctas = 2 * kSMs;
  }
  for (a.box = a.tile; a.box > 8 && Y.block_size % a.box; a.box /= 2) {
  }
  const long long most = attend_max_tiles(Y, max_q, num_listed, a.tile, a.rows);
  a.runs = (int)std::min<long long>(attend_max_runs(ctas, Y.num_kv_heads), most);
  // a few tiles per warp and head: one CTA per head does them all, and nothing is left to join
  if (a.kind == AttendKind::kDecode && most <= kDecodeWholeTiles * kDecodeWarps) a.runs = 1;
  a.part_o = (size_t)2 * a.runs * Y.num_kv_heads * a.rows * Y.head_dim * sizeof(float);
  a.part_ml = (size_t)2 * a.runs * Y.num_kv_heads * a.rows * 2 * sizeof(float);
  a.bytes = round_up(a.part_o, 256) + round_up(a.part_ml, 256);
  return a;
}

int validate_attend(const triattn_paged_layout* Y, int max_q, int num_listed) {
  const int rc = validate_layout(Y);
  if (rc != TRIATTN_OK) return rc;
  if (max_q <= 0 || num_listed < 0) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (max_q > kAttendMaxQuery || Y->group_size > 64) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if (Y->head_dim != 64 && Y->head_dim != 128 && Y->head_dim != 256) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  // token positions are 32-bit
  if ((long long)Y->max_blocks_per_req * Y->block_size > (1ll << 30) || (long long)num_listed * Y->block_size > (1ll << 30))
    return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if (Y->num_kv_heads > 65535) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  return TRIATTN_OK;
}

// K or V of a layer as (64 channels, token mod 8, 64-channel part, token / 8, head slot): see attend_tma.cuh.  The last
// block holds only num_kv_heads slots: the extent stops there, so no box reaches behind the cache.
bool encode_cache_map(CUtensorMap* map, const void* base, const triattn_paged_layout& Y, int box) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  const cuuint64_t parts = (cuuint64_t)Y.head_dim / 64;
  const cuuint64_t slots = (cuuint64_t)(Y.num_blocks - 1) * (cuuint64_t)(Y.block_stride / Y.head_stride) + (cuuint64_t)Y.num_kv_heads;
  const cuuint64_t dims[5] = {64, 8, parts, (cuuint64_t)Y.block_size / 8, slots};
  const cuuint64_t strides[4] = {(cuuint64_t)Y.token_stride * 2, 128, (cuuint64_t)Y.token_stride * 16, (cuuint64_t)Y.head_stride * 2};
  const cuuint32_t boxes[5] = {64, 8, (cuuint32_t)parts, (cuuint32_t)box / 8, 1}, elem[5] = {1, 1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dims, strides, boxes, elem,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool SP>
int launch_decode(const AttendParams& p, const AttendPlan& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  constexpr size_t smem = decode_smem_bytes<D, SP>();
  if (!ensure_dynamic_smem<attend_decode_kernel<D, SP>>(smem)) return TRIATTN_ERR_CUDA;
  return launch_kernel(attend_decode_kernel<D, SP>, dim3((unsigned)(a.runs * p.Hkv)), dim3(kDecodeThreads), smem, st, true, p, km, vm, a.runs);
}

template <int D, int NT>
int launch_tree(const AttendParams& p, const AttendPlan& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  constexpr size_t smem = tree_smem_bytes<D, NT>();
  if (!ensure_dynamic_smem<attend_tree_kernel<D, NT>>(smem)) return TRIATTN_ERR_CUDA;
  return launch_kernel(attend_tree_kernel<D, NT>, dim3((unsigned)(a.runs * p.Hkv)), dim3(kTreeThreads<NT>), smem, st, true, p, km, vm, a.runs);
}

template <int D>
int launch_attend(const AttendParams& p, const AttendPlan& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  if (a.kind == AttendKind::kDecode)
    return a.split_p ? launch_decode<D, true>(p, a, km, vm, st) : launch_decode<D, false>(p, a, km, vm, st);
  if constexpr (D <= 128) {
    if (a.kind == AttendKind::kTree) return a.rows == 128 ? launch_tree<D, 1>(p, a, km, vm, st) : launch_tree<D, 2>(p, a, km, vm, st);
  }
#define TRIATTN_LAUNCH(MT, SP)                                                                                            \
  {                                                                                                                       \
    if (!ensure_dynamic_smem<attend_paged_kernel<D, MT, SP>>(attend_smem_bytes<D, MT>())) return TRIATTN_ERR_CUDA;         \
    return launch_kernel(attend_paged_kernel<D, MT, SP>, dim3((unsigned)(a.runs * p.Hkv)), dim3(kAttendThreads),                    \
                         attend_smem_bytes<D, MT>(), st, true, p, a.runs);                                                \
  }
  if (a.split_p) TRIATTN_LAUNCH(1, true)
  if (a.mt == 1) TRIATTN_LAUNCH(1, false)
  if (a.mt == 2) TRIATTN_LAUNCH(2, false)
  TRIATTN_LAUNCH(4, false)
#undef TRIATTN_LAUNCH
}

template <int D>
int launch_attend_all(const AttendParams& p, const AttendPlan& a, const CUtensorMap& km, const CUtensorMap& vm,
                      int max_row_tiles, const CUtensorMap* observe_map, int observe_box, int observe_runs, cudaStream_t st) {
  int rc = launch_attend<D>(p, a, km, vm, st);
  if (rc != TRIATTN_OK) return rc;
  if (a.runs > 1) {  // (with one run per head every segment is whole)
    const int chunks = (a.rows + 7) / 8, live = (p.max_q * p.g + 7) / 8;  // CTAs per row tile; of them with rows, where there is one tile
    const dim3 grid((unsigned)(max_row_tiles > 1 ? max_row_tiles * chunks : std::min(chunks, live)), (unsigned)p.Hkv, (unsigned)p.B);
    rc = launch_kernel(attend_combine_kernel<D>, grid, dim3(kCombineThreads), 0, st, true, p, a.runs, a.tile, a.rows);
  }
  if (rc != TRIATTN_OK || p.sums == nullptr) return rc;
  if (observe_map != nullptr) {
    constexpr size_t smem = observe_mma_smem_bytes<D>();
    if (!ensure_dynamic_smem<attend_observe_mma_kernel<D>>(smem)) return TRIATTN_ERR_CUDA;
    for (int row0 = 0; row0 < p.max_q * p.g; row0 += kObserveRowsMax<D>) {
      AttendParams o = p;
      o.box = observe_box;
      rc = launch_kernel(attend_observe_mma_kernel<D>, dim3((unsigned)(observe_runs * p.Hkv)), dim3(kObserveMmaThreads), smem, st,
                         true, o, *observe_map, observe_runs, row0);
      if (rc != TRIATTN_OK) return rc;
    }
    return TRIATTN_OK;
  }
  if (!ensure_dynamic_smem<attend_observe_kernel<D>>(observe_smem_bytes<D>())) return TRIATTN_ERR_CUDA;
  return launch_kernel(attend_observe_kernel<D>, dim3((unsigned)(observe_runs * p.Hkv)), dim3(kAttendThreads),
                       observe_smem_bytes<D>(), st, true, p, observe_runs);
}

template <int D>
int launch_scores(const SelectBlocksParams& p, dim3 grid, int per_warp, cudaStream_t st) {
  if (!ensure_dynamic_smem<block_scores_kernel<D>>(score_smem_bytes<D>())) return TRIATTN_ERR_CUDA;
  return launch_kernel(block_scores_kernel<D>, grid, dim3(kScoreThreads), score_smem_bytes<D>(), st, true, p, per_warp);
}

}  // namespace

extern "C" {

size_t triattn_attend_workspace_bytes(const triattn_paged_layout* layout, int max_query_len, int num_listed) {
  if (validate_attend(layout, max_query_len, num_listed) != TRIATTN_OK) return 0;
  return attend_plan(with_plain_strides(*layout), max_query_len, num_listed).bytes;
}

int triattn_attend_paged(const triattn_paged_layout* layout, const void* k_cache, const void* v_cache,
                         const int32_t* block_table, const int32_t* seq_lens, const int32_t* query_start_loc,
                         const void* q, int64_t q_token_stride, int64_t q_head_stride, int num_query_tokens,
                         int max_query_len, float scale, const int64_t* tree_mask, const int32_t* block_list,
                         int num_listed, float* weight_sums, int reset_weight_sums, void* out,
                         int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
                         size_t workspace_bytes, uint32_t* device_status, void* stream) {
  if (block_list == nullptr) num_listed = 0;
  int rc = validate_attend(layout, max_query_len, num_listed);
  if (rc != TRIATTN_OK) return rc;
  if (!k_cache || !v_cache || !block_table || !seq_lens || !query_start_loc || !lse || !workspace)
    return TRIATTN_ERR_INVALID_ARGUMENT;
  if (num_query_tokens < 0 || !(scale > 0.f) || !std::isfinite(scale) || (block_list && num_listed <= 0))
    return TRIATTN_ERR_INVALID_ARGUMENT;
  if (num_query_tokens == 0) return TRIATTN_OK;
  if (!q || !out) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(q) || !aligned16(out) || !aligned16(workspace) ||
      q_token_stride % 8 || q_head_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
    return TRIATTN_ERR_MISALIGNED;
  const triattn_paged_layout Y = with_plain_strides(*layout);
  const AttendPlan a = attend_plan(Y, max_query_len, num_listed);
  if (workspace_bytes < a.bytes) return TRIATTN_ERR_WORKSPACE_TOO_SMALL;
  AttendParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_ts = q_token_stride;
  p.q_hs = q_head_stride;
  p.k = static_cast<const unsigned char*>(k_cache);
  p.v = static_cast<const unsigned char*>(v_cache);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.qsl = query_start_loc;
  p.tree = tree_mask;
  p.block_list = block_list;
  p.num_listed = num_listed;
  p.B = Y.num_reqs;
  p.Hkv = Y.num_kv_heads;
  p.g = Y.group_size;
  p.bs = Y.block_size;
  p.num_blocks = Y.num_blocks;
  p.max_blocks = Y.max_blocks_per_req;
  p.block_stride = Y.block_stride;
  p.token_stride = Y.token_stride;
  p.head_stride = Y.head_stride;
  p.N = num_query_tokens;
  p.max_q = max_query_len;
  p.box = a.box;
  p.min_tiles = a.min_tiles;
  p.slots_per_block = tileable(Y) ? (int)(Y.block_stride / Y.head_stride) : 0;
  p.scale_log2 = scale * kLog2e;
  p.out = static_cast<uint16_t*>(out);
  p.o_ts = out_token_stride;
  p.o_hs = out_head_stride;
  p.lse = lse;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + round_up(a.part_o, 256));
  p.sums = weight_sums;
  p.reset_sums = reset_weight_sums ? 1 : 0;
  p.status = device_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int row_tiles = (int)(((long long)max_query_len * Y.group_size + a.rows - 1) / a.rows);
  CUtensorMap km{}, vm{}, om{};
  const bool tiled = tileable(Y);
  if (a.kind != AttendKind::kGeneral && (!encode_cache_map(&km, k_cache, Y, a.box) || !encode_cache_map(&vm, v_cache, Y, a.box)))
    return TRIATTN_ERR_CUDA;
  int observe_runs = 0, observe_box = 128;
  if (weight_sums != nullptr) {
    observe_runs = (int)std::min<long long>(attend_max_runs(tiled || Y.head_dim > 128 ? kSMs : 2 * kSMs, Y.num_kv_heads),
                                            attend_max_tiles(Y, 1, num_listed, tiled ? 128 : kAttendTile, 64));
    for (; Y.block_size % observe_box && observe_box > 8; observe_box /= 2) {
    }
    if (tiled && !encode_cache_map(&om, k_cache, Y, observe_box)) return TRIATTN_ERR_CUDA;
  }
  const CUtensorMap* observe_map = tiled ? &om : nullptr;
  switch (Y.head_dim) {
    case 64: return launch_attend_all<64>(p, a, km, vm, row_tiles, observe_map, observe_box, observe_runs, st);
    case 128: return launch_attend_all<128>(p, a, km, vm, row_tiles, observe_map, observe_box, observe_runs, st);
    default: return launch_attend_all<256>(p, a, km, vm, row_tiles, observe_map, observe_box, observe_runs, st);
  }
}

int triattn_update_block_bounds(const triattn_paged_layout* layout, const void* const* k_layer_ptrs,
                                const int32_t* block_table, const int32_t* first_tokens, const int32_t* seq_lens,
                                void* bounds, uint32_t* device_status, void* stream) {
  const int rc = validate_layout(layout);
  if (rc != TRIATTN_OK) return rc;
  if (!k_layer_ptrs || !block_table || !first_tokens || !seq_lens || !bounds) return TRIATTN_ERR_INVALID_ARGUMENT;
  const triattn_paged_layout& Y = *layout;
  if (Y.head_dim != 64 && Y.head_dim != 128 && Y.head_dim != 256) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if ((long long)Y.max_blocks_per_req * Y.block_size > (1ll << 30)) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if (!aligned16(bounds)) return TRIATTN_ERR_MISALIGNED;
  BoundsParams p{};
  p.k_ptrs = k_layer_ptrs;
  p.bounds = static_cast<uint16_t*>(bounds);
  p.block_table = block_table;
  p.first = first_tokens;
  p.seq_lens = seq_lens;
  p.B = Y.num_reqs;
  p.Hkv = Y.num_kv_heads;
  p.D = Y.head_dim;
  p.bs = Y.block_size;
  p.num_blocks = Y.num_blocks;
  p.max_blocks = Y.max_blocks_per_req;
  p.block_stride = Y.block_stride;
  p.token_stride = Y.token_stride;
  p.head_stride = Y.head_stride;
  p.status = device_status;
  const long long pairs = (long long)Y.num_layers * Y.num_reqs;
  const long long warps = (long long)Y.max_blocks_per_req * Y.num_kv_heads;
  // eight CTAs per SM; a step that touches one block per request gets one CTA per (layer, request)
  const long long gx = std::max<long long>(1, std::min((warps + 7) / 8, kSMs * 8 / pairs));
  return launch_kernel(block_bounds_kernel, dim3((unsigned)gx, (unsigned)Y.num_reqs, (unsigned)Y.num_layers),
                       dim3(kBoundsThreads), 0, static_cast<cudaStream_t>(stream), true, p);
}

size_t triattn_select_blocks_workspace_bytes(const triattn_paged_layout* layout) {
  if (validate_layout(layout) != TRIATTN_OK) return 0;
  return round_up((size_t)layout->num_reqs * layout->num_kv_heads * layout->max_blocks_per_req * sizeof(float), 256);
}

int triattn_select_blocks(const triattn_paged_layout* layout, const void* q, int64_t q_token_stride,
                          int64_t q_head_stride, int num_query_tokens, int max_query_len,
                          const int32_t* query_start_loc, const void* bounds, const int32_t* block_table,
                          const int32_t* seq_lens, int num_selected, int sink_blocks, int recent_blocks,
                          int32_t* block_list, void* workspace, size_t workspace_bytes, uint32_t* device_status,
                          void* stream) {
  int rc = validate_attend(layout, max_query_len, 0);
  if (rc != TRIATTN_OK) return rc;
  if (!query_start_loc || !bounds || !block_table || !seq_lens || !block_list || !workspace) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (num_query_tokens < 0 || num_selected <= 0 || sink_blocks < 0 || recent_blocks < 0) return TRIATTN_ERR_INVALID_ARGUMENT;
  const triattn_paged_layout& Y = *layout;
  // what is always read has to fit: the sink, the recent blocks and the blocks of the query's own tokens
  const long long own = (max_query_len + Y.block_size - 2) / Y.block_size + 1;
  if (num_selected < sink_blocks + std::max<long long>(recent_blocks, own)) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (num_query_tokens > 0 && !q) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (!aligned16(bounds) || !aligned16(workspace) || !aligned16(q) || q_token_stride % 8 || q_head_stride % 8)
    return TRIATTN_ERR_MISALIGNED;
  if (workspace_bytes < triattn_select_blocks_workspace_bytes(layout)) return TRIATTN_ERR_WORKSPACE_TOO_SMALL;
  SelectBlocksParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_ts = q_token_stride;
  p.q_hs = q_head_stride;
  p.qsl = query_start_loc;
  p.bounds = static_cast<const uint16_t*>(bounds);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.B = Y.num_reqs;
  p.Hkv = Y.num_kv_heads;
  p.g = Y.group_size;
  p.bs = Y.block_size;
  p.num_blocks = Y.num_blocks;
  p.max_blocks = Y.max_blocks_per_req;
  p.N = num_query_tokens;
  p.max_q = max_query_len;
  p.num_selected = num_selected;
  p.sink = sink_blocks;
  p.recent = recent_blocks;
  p.scores = static_cast<float*>(workspace);
  p.block_list = block_list;
  p.status = device_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long rows = (long long)Y.num_reqs * Y.num_kv_heads;
  // up to 32 blocks per warp, fewer while the grid does not hold two CTAs per SM
  int per_warp = 32;
  const auto grid_x = [&](int n) { return (Y.max_blocks_per_req + 8ll * n - 1) / (8 * n); };
  while (per_warp > 4 && grid_x(per_warp) * rows < 2 * kSMs) per_warp /= 2;
  const dim3 grid((unsigned)grid_x(per_warp), (unsigned)Y.num_kv_heads, (unsigned)Y.num_reqs);
  switch (Y.head_dim) {
    case 64: rc = launch_scores<64>(p, grid, per_warp, st); break;
    case 128: rc = launch_scores<128>(p, grid, per_warp, st); break;
    default: rc = launch_scores<256>(p, grid, per_warp, st); break;
  }
  if (rc != TRIATTN_OK) return rc;
  const int cap = (int)std::min<long long>((Y.max_blocks_per_req + 3ll) / 4 * 4, 32768);
  const size_t smem = (size_t)cap * 4;
  if (!ensure_dynamic_smem<pick_blocks_kernel>(smem)) return TRIATTN_ERR_CUDA;
  return launch_kernel(pick_blocks_kernel, dim3((unsigned)Y.num_kv_heads, (unsigned)Y.num_reqs), dim3(kPickThreads), smem, st,
                       true, p, cap);
}

}  // extern "C"
