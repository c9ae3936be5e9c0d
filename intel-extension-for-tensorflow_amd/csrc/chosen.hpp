// What the kernels share whose rows are grouped by the weights they chose: loads of the three types, and the tiles of rows of a
// grouped order.
#ifndef ITEXHIP_CHOSEN_HPP_
#define ITEXHIP_CHOSEN_HPP_

#include "chosen_rules.hpp"
#include "common.hpp"

namespace itexhip {

constexpr int kMaxGroups = 1024;
constexpr int64_t kMaxRows = 1 << 30;

inline bool is_chosen_type(int t) { return t == ITEXHIP_FLOAT || is_float16_type(t); }
inline int64_t element_size(int t) { return t == ITEXHIP_FLOAT ? 4 : 2; }

template <int T>
__device__ __forceinline__ float load_value(const void* base, int64_t i) {
  if constexpr (T == ITEXHIP_FLOAT) return static_cast<const float*>(base)[i];
  else if constexpr (T == ITEXHIP_BFLOAT16) return bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
}

// Eight elements from the i-th on; the address of the first is a multiple of 16 bytes
template <int T>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&x)[8]) {
  if constexpr (T == ITEXHIP_FLOAT) {
    const f4* from = reinterpret_cast<const f4*>(static_cast<const float*>(base) + i);
    const f4 a = from[0], b = from[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j] = a[j]; x[4 + j] = b[j]; }
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = (w[j / 2] >> (16 * (j % 2))) & 0xffffu;
      x[j] = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
  }
}

// Launches of up to 2^23 workgroups, since a grid has fewer than 2^32 threads: f(first, count) for each
template <class F>
inline void launch_blocks(int64_t blocks, F&& f) {
  in_pieces(0, blocks, [&](int64_t begin, int64_t end) { f(begin, static_cast<unsigned>(end - begin)); }, 1LL << 23);
}

// The tiles that tiles_bound counts
struct RowTile {
  int group;       // groups: the rows of no group
  int begin, rows; // places
};
// The groups' tiles, counted by all lanes of a wavefront; a lane has `each` neighbouring groups.  Offsets are cut to 0 .. n, so that
// whatever they hold, places are.
struct GroupUnit {
  int group;          // -1: there are not that many units
  int begin, rows;    // the group's places
  int tiles;          // of the group
  int64_t index;      // within the group
};
enum Tiles : int { kAllTiles, kFullTiles, kLastTiles };  // of a group; kLastTiles: those that are not full
template <bool REST, int KIND = kAllTiles>
struct TileCount {
  const int32_t* offsets;
  int groups, n, per_tile, each;
  int begin, rows;    // of the lane's first group
  int mine, sum;      // tiles of the lane's groups; and with those of the lanes below
  __device__ __forceinline__ int at(int g) const { return g > groups ? n : min(max(offsets[g], 0), n); }
  __device__ __forceinline__ int tiles_of(int rows) const {
    return KIND == kFullTiles ? rows / per_tile : KIND == kLastTiles ? rows % per_tile != 0 : (rows + per_tile - 1) / per_tile;
  }
  __device__ __forceinline__ TileCount(const int32_t* offsets, int groups, int n, int per_tile)
      : offsets(offsets), groups(groups), n(n), per_tile(per_tile) {
    const int lane = static_cast<int>(__lane_id()), parts = groups + (REST ? 1 : 0);
    each = (parts + 63) / 64;
    const int g0 = min(lane * each, parts), g1 = min(g0 + each, parts);
    begin = rows = mine = 0;
    if (g0 < g1) {
      begin = at(g0);
      rows = max(at(g0 + 1) - begin, 0);
      mine = tiles_of(rows);
      for (int g = g0 + 1; g < g1; ++g) mine += tiles_of(max(at(g + 1) - at(g), 0));
    }
    sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int below = __shfl_up(sum, d);
      if (lane >= d) sum += below;
    }
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, 63); }
  // Whose the index-th unit is where every tile has `units` of them; the same for all lanes
  __device__ __forceinline__ GroupUnit find(int64_t units, int64_t index) const {
    const unsigned long long past = __ballot(sum * units > index);
    if (past == 0) return GroupUnit{-1, 0, 0, 0, 0};
    const int owner = __builtin_ctzll(past);
    int64_t rank = index - (__builtin_amdgcn_readlane(sum, owner) - __builtin_amdgcn_readlane(mine, owner)) * units;
    int first = __builtin_amdgcn_readlane(begin, owner), count = __builtin_amdgcn_readlane(rows, owner);
    for (int g = owner * each;;) {
      const int tiles = tiles_of(count);
      if (rank >= 0 && rank < tiles * units) return GroupUnit{g, first, count, tiles, rank};
      rank -= tiles * units;
      if (++g >= groups + (REST ? 1 : 0)) return GroupUnit{-1, 0, 0, 0, 0};  // (offsets that are none, whose tiles do not add up)
      first = __builtin_amdgcn_readfirstlane(at(g));
      count = __builtin_amdgcn_readfirstlane(max(at(g + 1) - first, 0));
    }
  }
};
template <bool REST>
__device__ __forceinline__ RowTile find_tile(const int32_t* __restrict__ offsets, int groups, int n, int per_tile, int index) {
  const GroupUnit u = TileCount<REST>(offsets, groups, n, per_tile).find(1, index);
  const int before = static_cast<int>(u.index) * per_tile;
  return RowTile{u.group, u.begin + before, min(per_tile, u.rows - before)};
}

}  // namespace itexhip
#endif  // ITEXHIP_CHOSEN_HPP_
