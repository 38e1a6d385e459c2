// Host side of the two matrix-core kernels of tree_attention: which of them a call takes, how its work is shared
// out, and its launches.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "tree_attn_rows.h"
#include "tree_attn_tiles.h"

namespace kg_gfx950 {

inline long long tree_items(const TreeArgs& a, int block) {  // at most, where `starts` ascend
  return a.heads * ((long long)a.tokens * a.group / block + std::min(a.batch, a.tokens));
}
// What they take: 16-bit queries, heads of a multiple of 16 up to 256, rows of 16-byte pieces, strides of tree_row, sums of
// units in 31 bits.
inline bool tree_matrix_takes(const TreeArgs& a, int cache_bytes) {
  auto whole = [&](const void* p, std::initializer_list<long long> strides, int bytes, int unit) {
    bool ok = (uintptr_t)p % unit == 0;
    for (long long s : strides) ok = ok && s * bytes % unit == 0;
    return ok;
  };
  for (long long s : {a.k_page, a.v_page})
    if (s > 0xffffffffLL) return false;
  if (a.k_scale != nullptr)
    for (long long s : {a.ks_page, a.ks_row, a.vs_page, a.vs_row})
      if (s > 0xffffffffLL) return false;
  if ((long long)a.tokens * a.heads_q > kTreeMostUnits || tree_items(a, 16) > kTreeMostUnits) return false;
  return a.d % 16 == 0 && a.d <= 256 && whole(a.q, {a.q_token, a.q_head}, 2, 16) && whole(a.out, {a.o_token, a.o_head}, 2, 4) &&
         whole(a.k, {a.k_page, a.k_head, a.k_row}, cache_bytes, 16) && whole(a.v, {a.v_page, a.v_head, a.v_row}, cache_bytes, 16) &&
         a.k_row <= 1 << 24 && a.v_row <= 1 << 24 && a.pages > 0 && a.per > 0;
}

struct TreePlan {
  int width;     // padded head
  bool tiles;    // tree_attn_tiles_kernel
  int blocks16;  // 16-row blocks of a wave
  TreeSplit split;
  bool join;
  size_t bytes;
};
// Rows in fours that a launch of the join can have, a wave each: its work-items are counted in 32 bits.
constexpr long long kTreeMostQuads = (1ll << 26) - 4;
// Shares of a call: as many workgroups as run at once, or as there can be units (the table's reach bounds a
// request's keys, the batch's tokens its blocks of rows).
inline TreePlan tree_plan(const TreeArgs& a, int cache_bytes, bool may_split, long long most_bytes) {
  TreePlan p;
  p.width = a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256;
  const long long rows = ((long long)a.tokens + a.batch - 1) / a.batch * a.group;  // of a request and key head, on average
  p.tiles = rows > 16 || a.page_size % 16 != 0;
  p.blocks16 = p.tiles && rows > 64 && p.width < 256 ? 2 : 1;
  p.split.block = 16 * p.blocks16 * (p.tiles ? treet::kWaves : 1);
  p.split.width = p.width;
  const long long round = p.tiles ? (p.width == 256 ? 32 : 64)
                                  : ((cache_bytes == 2 && p.width >= 128) || p.width == 256 ? 32 : 64) * treer::kWaves;
  const long long reach = (long long)a.per * a.page_size;
  const long long items = tree_items(a, p.split.block);
  const long long units = items * std::max(1ll, (reach + round - 1) / round);
  may_split = may_split && reach > round && units < kTreeMostUnits && items * p.split.block / kTreeJoinRows <= kTreeMostQuads;
  p.split.round = may_split ? (int)round : 0;
  p.split.grid = (int)std::min<long long>(may_split ? units : items, p.width == 256 ? 256 : 512);
  const long long record = 2ll * p.split.block * (p.width + kTreePad) * (long long)sizeof(float);
  if (may_split) p.split.grid = (int)std::min<long long>(p.split.grid, most_bytes / record);
  p.join = may_split;
  p.split.partial = nullptr;
  p.bytes = may_split ? (size_t)(p.split.grid * record) : 0;
  return p;
}

template <typename Tag, typename C>
hipError_t launch_tree(const TreeArgs& a, const TreePlan& p, hipStream_t stream) {
#define KG_TREE_ROWS(WIDTH) \
  hipLaunchKernelGGL((tree_attn_rows_kernel<Tag, C, WIDTH>), dim3(p.split.grid), dim3(treer::kThreads), 0, stream, a, p.split)
#define KG_TREE_TILES(WIDTH, NQ) \
  hipLaunchKernelGGL((tree_attn_tiles_kernel<Tag, C, WIDTH, NQ>), dim3(p.split.grid), dim3(treet::kThreads), 0, stream, a, p.split)
  if (p.width == 256) {
    if (p.tiles) KG_TREE_TILES(256, 1);
    else KG_TREE_ROWS(256);
  } else if (p.width == 128) {
    if (!p.tiles) KG_TREE_ROWS(128);
    else if (p.blocks16 == 1) KG_TREE_TILES(128, 1);
    else KG_TREE_TILES(128, 2);
  } else {
    if (!p.tiles) KG_TREE_ROWS(64);
    else if (p.blocks16 == 1) KG_TREE_TILES(64, 1);
    else KG_TREE_TILES(64, 2);
  }
#undef KG_TREE_TILES
#undef KG_TREE_ROWS
  if (p.join) {
    const long long quads = tree_items(a, p.split.block) * (p.split.block / kTreeJoinRows);  // of rows
    // many: 16 records and more of an item, if all workgroups have work
    const bool many = p.split.grid / std::max(1ll, tree_items(a, p.split.block)) >= 16, few = quads <= 4096;
#define KG_TREE_JOIN(WIDTH, WAVES)                                                                                      \
  hipLaunchKernelGGL((tree_attn_join_kernel<Tag, WIDTH, WAVES>),                                                        \
                     dim3((unsigned)((quads * WAVES + tree_join_waves(WAVES) - 1) / tree_join_waves(WAVES))),           \
                     dim3(64 * tree_join_waves(WAVES)), 0, stream, a, p.split)
    if (p.width == 256) {
      if (few && many) KG_TREE_JOIN(256, 8);
      else if (few) KG_TREE_JOIN(256, 4);
      else KG_TREE_JOIN(256, 1);
    } else if (p.width == 128) {
      if (few && many) KG_TREE_JOIN(128, 16);
      else if (few) KG_TREE_JOIN(128, 4);
      else KG_TREE_JOIN(128, 1);
    } else {
      if (few && many) KG_TREE_JOIN(64, 16);
      else if (few) KG_TREE_JOIN(64, 4);
      else KG_TREE_JOIN(64, 1);
    }
#undef KG_TREE_JOIN
  }
  return hipGetLastError();
}

}  // namespace kg_gfx950
