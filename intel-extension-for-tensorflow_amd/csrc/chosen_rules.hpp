// Which kernel a call of the operators takes whose rows are grouped by the weights they chose, and how its work is cut: rules on sizes alone,
// without HIP, so that they can be compiled and looked at anywhere.
#ifndef ITEXHIP_CHOSEN_RULES_HPP_
#define ITEXHIP_CHOSEN_RULES_HPP_

#include <cstdint>

namespace itexhip {

// Tiles of up to `per_tile` places of the order, group by group; with REST the rows of no group are a group of their own behind the
// others.  How many there are is known on the device only: a launch has room for tiles_bound of them, and those beyond the
// last find group = -1.
inline int64_t tiles_bound(int64_t n, int groups, int per_tile, bool rest) {
  const int64_t parts = groups + (rest ? 1 : 0);
  const int64_t open = n < parts ? n : parts;  // groups that can have a tile that is not full
  return open + (n - open) / per_tile;
}

// ------------------------------------------------------------------------------------------------
// Experts' products
// ------------------------------------------------------------------------------------------------
struct ProductSizes {
  int64_t slots, top_k;  // slots = tokens * top_k
  int experts;
  int64_t pitch, N;      // bytes of a row's codes, 64 to each K step; channels
  bool up, gated;
};
constexpr int kFewRows = 16;    // rows whose codes a workgroup makes, up
constexpr int kFewPlaces = 16;  // rows of the way back in one launch
constexpr int kFewBytes = 64 * 1024;  // codes that a workgroup keeps in LDS
constexpr int kWorkgroups = 256;      // of tiles: one for each CU; they take the tiles in turns
constexpr int kTileSteps = 4;         // K steps that a tile has to have

// up: a workgroup makes the codes of its tokens itself where they are about 32 elements a thread; beyond, a launch that makes them once is shorter
inline bool few_up(const ProductSizes& s) {
  const int64_t tokens = s.slots / s.top_k, each = s.slots > s.experts ? (s.slots + s.experts - 1) / s.experts : 1;
  return tokens <= kFewRows && each * s.pitch <= 8192 && tokens * s.pitch <= kFewBytes / 2;
}
// down, one launch : three in us: 2 rows of 768 to 14336 7 : 12 to 32 : 34, 4 of 1536 and 4096 11 : 16 and 18 : 15, 8 of 768 and 1536 10 : 13 and 13 : 17,
// where there are few channels 12 : 12, 16 of 768 13 : 13.  8 of 1536 are 12288 bytes: the rule leaves them to the three launches, 17 for 13; 3 rows were not measured
inline bool few_down(const ProductSizes& s) {
  const int64_t bytes = s.slots * s.pitch;
  return s.slots <= kFewPlaces && (s.slots <= 2 || bytes <= 8192) && bytes <= kFewBytes;
}
// Few strips: eight wavefronts each instead of four, so that the device has enough on their way (896 strips of 4096: 46 -> 39 us), unless that
// leaves a wavefront a handful of chunks (736 of 1024: 13 -> 15)
inline bool few_strips(const ProductSizes& s) {
  return tiles_bound(s.slots, s.experts, 32, false) * ((s.N + 31) / 32) < (s.pitch / 32 >= 64 ? 1024 : 512);
}

// Strips of 32 channels by 4 or 8 wavefronts, tiles of 256 rows by 128 or 256 columns of weights.
// Tiles cost a workgroup about 10 us whatever they hold, and have to be enough of them (rows of tiles a workgroup); strips read
// an expert's weights again for every 32 rows.  Measured, tiles : strips in us, 8 experts of 4096 x 4096, gated, at 16, 32, 64 rows each 67 : 57, 68 : 75, 75 : 130, not gated 49 : 44,
// 54 : 66, 66 : 99; 32 of 1408 x 2048, not gated, at 8, 16 30 : 29, 32 : 38; 4 of 14336 x 4096 (64 tiles) at 32, 64 134 : 101, 162 : 171;
// 8 of 1024 x 1024, gated (64 tiles), at 64, 128, 256 18 : 13, 24 : 21, 25 : 30, not gated (32 tiles) at 256, 512 33 : 31, 39 : 50.  At three of the 70 sizes that were
// measured the rule takes the longer one: 24 for 21 and 33 for 31 of the last, 38 for 32 of 1408 x 2048 at 16.  Rows are counted by slots: with
// experts on other devices an expert here has fewer than the rule takes it to have.
enum ProductKernel { kStrips4, kStrips8, kTiles128, kTiles256 };
inline ProductKernel product_kernel(const ProductSizes& s) {
  const int64_t width = s.gated ? 128 : 256, each = s.slots / s.experts, tiles = s.experts * ((s.N + width - 1) / width);
  const bool near = !s.up || s.slots / s.top_k * s.pitch < (1LL << 32);  // up: codes in reach of 32 bits
  if (each >= (s.gated ? 24 : 12) && each * tiles >= kWorkgroups * (s.pitch >= 2048 ? 12 : 32) && s.pitch / 64 >= kTileSteps && near)
    return tiles * ((each + 255) / 256) < kWorkgroups * 3 / 4 ? kTiles128 : kTiles256;  // half as many channels a tile where they are too few for the device
  return few_strips(s) ? kStrips8 : kStrips4;
}

// ------------------------------------------------------------------------------------------------
// Adapters
// ------------------------------------------------------------------------------------------------
constexpr int kMaxSplits = 6;
constexpr int kEnoughTiles = 512;

// Many places an adapter: tiles of 64 of them, which read A a quarter as often; 16 where most would be empty or tiles few
inline bool long_tiles(int64_t tokens, int adapters) { return tokens > 32 * static_cast<int64_t>(adapters) && tiles_bound(tokens, adapters, 64, false) >= 64; }
// of the product with B, `width` columns a workgroup: 64 places where that leaves enough workgroups
inline bool long_expand(int64_t tokens, int adapters, int64_t columns, int width) {
  return long_tiles(tokens, adapters) && tiles_bound(tokens, adapters, 64, true) * ((columns + width - 1) / width) >= kEnoughTiles;
}
// Shares of K: enough workgroups for the device where tiles are few, of at least 256 k each.  parts: workgroups that divide a tile's rows of A
inline int splits_of(int64_t tokens, int adapters, int64_t parts, int64_t in) {
  const int64_t tiles = tiles_bound(tokens, adapters, long_tiles(tokens, adapters) ? 64 : 16, false) * parts;
  int64_t n = tiles == 0 ? 1 : (kEnoughTiles + tiles - 1) / tiles;
  n = n < (in + 255) / 256 ? n : (in + 255) / 256;
  return static_cast<int>(n < kMaxSplits ? n : kMaxSplits);
}
inline int shrink_parts(int rank) { return rank <= 64 ? 1 : (rank + 63) / 64; }  // of a slice
// Rows of the middle that any call of up to this many tokens needs: a share's tiles hold at most 64 tokens each
inline int64_t middle_rows(int64_t tokens) {
  const int64_t most = kMaxSplits * tokens, few = 64 * 2 * kEnoughTiles;
  return most < few ? most : few > tokens ? few : tokens;
}
// One launch where a workgroup's part of x A^T is short and reading A again for every 1024 columns costs less than a second launch
inline bool one_launch(int64_t tokens, int adapters, int rank, int n_slices, int64_t in, int64_t columns) {
  const int64_t blocks = (columns + 1023) / 1024 + n_slices - 1;
  return rank <= 16 && in <= 2048 && tiles_bound(tokens, adapters, 16, false) * blocks * rank * in * 2 <= (4 << 20);
}

}  // namespace itexhip
#endif  // ITEXHIP_CHOSEN_RULES_HPP_
