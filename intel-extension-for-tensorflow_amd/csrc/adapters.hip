// Low-rank adapters of many requests beside a shared projection: x A^T of each row's adapter, then the base plus its product with B^T.
#include <type_traits>

#include "chosen.hpp"
#include "qgemm_common.hpp"

namespace itexhip {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kMaxSplits = 16;

struct AdapterArgs {
  itexhip_adapters_params p;
  const void *x, *a, *b, *base;
  const int32_t *offsets, *rows, *ranks;
  const float* scales;
  void* out;
  float* middle;   // [splits][tokens][deep]: x A^T by place of the order, a share of K each
  int tokens, deep, splits, per_split;  // deep = n_slices * rank; per_split: K steps of 32 of a share
  int in, columns;  // of x; of the output
  int64_t first;    // workgroup of the launch
  int blocks[ITEXHIP_ADAPTER_MAX_SLICES];  // blocks of 64 columns up to the end of each slice
};

__device__ __forceinline__ int token_of(const AdapterArgs& A, int place) { return min(max(A.rows[place], 0), A.tokens - 1); }
__device__ __forceinline__ int rank_of(const AdapterArgs& A, int group) { return A.ranks == nullptr ? A.p.rank : min(max(A.ranks[group], 0), A.p.rank); }

// An operand of the 16-row products: a lane holds 8 consecutive k of row lane % 16, those from 8 (lane / 16) on.
struct Eight {
  float v[8];
};
template <int T>
using operand_t = std::conditional_t<T == ITEXHIP_BFLOAT16, v8bf, std::conditional_t<T == ITEXHIP_HALF, v8h, Eight>>;

// D += P Q^T over 32 k: a lane's four results are rows 4 (lane / 16) .. + 3 of P and row lane % 16 of Q.  In fp32 each of the
// products takes four k, one of every lane's 8: the order of k is the same in both operands.
template <int T, class V>
__device__ __forceinline__ v4f product(const V& p, const V& q, v4f d) {
  if constexpr (T == ITEXHIP_BFLOAT16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, d, 0, 0, 0);
  } else if constexpr (T == ITEXHIP_HALF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, d, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(p.v[j], q.v[j], d, 0, 0, 0);
    return d;
  }
}
// Elements k .. k + 7 of a row that has `count` of them; zeros behind.  VEC: rows are aligned to 16 bytes and count is a multiple of 8
template <int T, bool VEC>
__device__ __forceinline__ operand_t<T> load_operand(const void* base, int64_t row, int k, int count) {
  operand_t<T> o;
  if constexpr (VEC) {
    if (k < count) {
      if constexpr (T == ITEXHIP_FLOAT) {
        load8<T>(base, row + k, o.v);
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + row + k);
        __builtin_memcpy(&o, &w, 16);
      }
    } else {
      __builtin_memset(&o, 0, sizeof(o));
    }
  } else {
    if constexpr (T == ITEXHIP_FLOAT) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o.v[j] = k + j < count ? static_cast<const float*>(base)[row + k + j] : 0.0f;
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = k + 2 * j < count ? static_cast<const uint16_t*>(base)[row + k + 2 * j] : 0u;
        const uint32_t hi = k + 2 * j + 1 < count ? static_cast<const uint16_t*>(base)[row + k + 2 * j + 1] : 0u;
        w[j] = lo | hi << 16;
      }
      __builtin_memcpy(&o, w, 16);
    }
  }
  return o;
}

// the elements from the count-th on become zeros
template <int T>
__device__ __forceinline__ void cut(operand_t<T>& o, int count) {
  if constexpr (T == ITEXHIP_FLOAT) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = j < count ? o.v[j] : 0.0f;
  } else {
    uint32_t w[4];
    __builtin_memcpy(w, &o, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] &= (2 * j < count ? 0xffffu : 0u) | (2 * j + 1 < count ? 0xffff0000u : 0u);
    __builtin_memcpy(&o, w, 16);
  }
}

// x A^T.  A workgroup has 16 places of one adapter, 16 of its rows of A and a share of K, which its wavefronts divide.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void shrink_kernel(const AdapterArgs A) {
  __shared__ __align__(16) float sums[4][16 * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = A.first + blockIdx.x;
  const int tile_of_a = static_cast<int>(id % ((A.deep + 15) / 16)), rest = static_cast<int>(id / ((A.deep + 15) / 16));
  const int split = rest % A.splits;
  const RowTile t = find_tile<false>(A.offsets, A.p.adapters, A.tokens, 16, rest / A.splits);
  if (t.group < 0) return;
  const int r = tile_of_a * 16 + (lane & 15), rank = rank_of(A, t.group);
  const bool there = r < A.deep && r % A.p.rank < rank;
  const int64_t x_row = static_cast<int64_t>(token_of(A, t.begin + min(lane & 15, t.rows - 1))) * A.p.x_stride;
  const int64_t a_row = (static_cast<int64_t>(t.group) * A.deep + min(r, A.deep - 1)) * A.in;
  const int first = split * A.per_split, last = min(first + A.per_split, (A.in + 31) / 32);
  v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = first + wave; c < last; c += 4) {
    const int k = c * 32 + (lane >> 4) * 8;
    const operand_t<T> a = load_operand<T, VEC>(A.a, a_row, k, there ? A.in : 0);
    const operand_t<T> x = load_operand<T, VEC>(A.x, x_row, k, A.in);
    d = product<T>(a, x, d);
  }
  *reinterpret_cast<v4f*>(&sums[wave][(lane & 15) * 16 + (lane >> 4) * 4]) = d;
  __syncthreads();
  const int place = threadIdx.x >> 4, column = tile_of_a * 16 + (threadIdx.x & 15);
  if (place < t.rows && column < A.deep) {
    float sum = sums[0][threadIdx.x];
    for (int w = 1; w < 4; ++w) sum += sums[w][threadIdx.x];
    A.middle[(static_cast<int64_t>(split) * A.tokens + t.begin + place) * A.deep + column] = sum;
  }
}

// A power of two that brings a row's largest absolute value (its bits) to 2^8 .. 2^9, and its inverse
__device__ __forceinline__ void power_of(uint32_t bits, float* up, float* down) {
  const int e = min(max(static_cast<int>(bits >> 23), 20), 240);  // of 2^(e - 127)
  *up = __uint_as_float(static_cast<uint32_t>(262 - e) << 23);
  *down = __uint_as_float(static_cast<uint32_t>(e - 8) << 23);
}

// out = base + scale (x A^T) B^T.  A wavefront has 16 places of one adapter and 64 columns of one slice: a product's row q = 4 g + i of
// its j-th tile of B stands for column 16 g + 4 j + i, so that a lane ends with 16 neighbouring columns of a row.  The middle's values are the sum of two
// numbers of the type; in half precision times a power of two that keeps a row's largest in range.
template <int T>
__global__ __launch_bounds__(256) void expand_kernel(const AdapterArgs A) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = A.first + blockIdx.x;
  const int fours = (A.blocks[A.p.n_slices - 1] + 3) / 4, index = static_cast<int>(id / fours);
  const int block = static_cast<int>(id - static_cast<int64_t>(index) * fours) * 4 + wave;
  if (block >= A.blocks[A.p.n_slices - 1]) return;
  const RowTile t = find_tile<true>(A.offsets, A.p.adapters, A.tokens, 16, index);
  if (t.group < 0) return;
  const bool none = t.group == A.p.adapters;
  if (none && A.out == A.base) return;
  int slice = 0;
  while (block >= A.blocks[slice]) ++slice;
  const int slice_begin = slice == 0 ? 0 : static_cast<int>(A.p.slice_end[slice - 1]), slice_end = static_cast<int>(A.p.slice_end[slice]);
  const int column0 = slice_begin + (block - (slice == 0 ? 0 : A.blocks[slice - 1])) * 64;
  const int place = t.begin + min(lane & 15, t.rows - 1), group4 = lane >> 4;
  v4f d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) d[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  float scale = 0.0f, down = 1.0f;
  if (!none) {
    const int rank = rank_of(A, t.group);
    scale = A.scales[t.group];
    const int64_t at = static_cast<int64_t>(place) * A.deep + slice * A.p.rank, share = static_cast<int64_t>(A.tokens) * A.deep;
    auto middle = [&](int r, float (&v)[8]) {
      if (r < rank) {
        load8<ITEXHIP_FLOAT>(A.middle, at + r, v);
        for (int s = 1; s < A.splits; ++s) {
          float w[8];
          load8<ITEXHIP_FLOAT>(A.middle, at + s * share + r, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r + i >= rank) v[i] = 0.0f;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      }
    };
    float up = 1.0f;
    if constexpr (T == ITEXHIP_HALF) {
      uint32_t top = 0;
      for (int r0 = 0; r0 < rank; r0 += 32) {
        float v[8];
        middle(r0 + group4 * 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      power_of(top, &up, &down);
    }
    for (int r0 = 0; r0 < rank; r0 += 32) {
      const int r = r0 + group4 * 8;
      float v[8];
      middle(r, v);
      operand_t<T> hi, lo;
      if constexpr (T == ITEXHIP_FLOAT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) hi.v[i] = v[i];
      } else {
        uint32_t wh[4], wl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = v[2 * i] * up, b = v[2 * i + 1] * up;
          wh[i] = f32x2_to_bits16<T>(a, b);
          const float ha = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(wh[i] & 0xffffu) : f16_bits_to_f32(wh[i] & 0xffffu);
          const float hb = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(wh[i] >> 16) : f16_bits_to_f32(wh[i] >> 16);
          wl[i] = f32x2_to_bits16<T>(a - ha, b - hb);
        }
        __builtin_memcpy(&hi, wh, 16);
        __builtin_memcpy(&lo, wl, 16);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = lane & 15, column = column0 + (q >> 2) * 16 + j * 4 + (q & 3);
        const int64_t b_row = (static_cast<int64_t>(t.group) * A.columns + min(column, slice_end - 1)) * A.p.rank;
        operand_t<T> b = load_operand<T, true>(A.b, b_row, r, (rank + 7) / 8 * 8);
        if (rank % 8 != 0) cut<T>(b, rank - r);
        d[j] = product<T>(b, hi, d[j]);
        if constexpr (T != ITEXHIP_FLOAT) d[j] = product<T>(b, lo, d[j]);
      }
    }
  }
  if ((lane & 15) >= t.rows) return;
  const int64_t token = token_of(A, place);
  const int first = column0 + group4 * 16;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int column = first + j * 4 + i;
      if (column >= slice_end) continue;
      const float base = load_value<T>(A.base, token * A.p.base_stride + column);
      if (none) store_output<T>(A.out, token * A.p.out_stride + column, base);
      else store_output<T>(A.out, token * A.p.out_stride + column, base + scale * (d[j][i] * down));
    }
}

int check(const itexhip_adapters_params* p, const char* name) {
  ITEXHIP_REQUIRE(p != nullptr, "%s: null parameters", name);
  ITEXHIP_REQUIRE(is_chosen_type(p->type), "%s: the type is float, bfloat16 or half", name);
  ITEXHIP_REQUIRE(p->adapters >= 1 && p->adapters <= kMaxGroups, "%s: 1 .. 1024 adapters, got %d", name, p->adapters);
  ITEXHIP_REQUIRE(p->rank >= 8 && p->rank <= 256 && p->rank % 8 == 0, "%s: rank is a multiple of 8, 8 .. 256, got %d", name, p->rank);
  ITEXHIP_REQUIRE(p->n_slices >= 1 && p->n_slices <= ITEXHIP_ADAPTER_MAX_SLICES, "%s: 1 .. 4 slices, got %d", name, p->n_slices);
  ITEXHIP_REQUIRE(p->tokens >= 0 && p->tokens < kMaxRows, "%s: tokens are 0 .. 2^30 - 1", name);
  ITEXHIP_REQUIRE(p->in >= 1 && p->in <= (1 << 20), "%s: in is 1 .. 2^20", name);
  int64_t before = 0;
  for (int i = 0; i < p->n_slices; ++i) {
    ITEXHIP_REQUIRE(p->slice_end[i] > before && p->slice_end[i] <= (1 << 20), "%s: slice_end ascends from 1 to at most 2^20", name);
    before = p->slice_end[i];
  }
  ITEXHIP_REQUIRE(p->x_stride >= p->in && p->x_stride < (1LL << 31), "%s: x_stride is at least in and below 2^31", name);
  for (const int64_t s : {p->base_stride, p->out_stride})
    ITEXHIP_REQUIRE(s >= before && s < (1LL << 31), "%s: base_stride and out_stride are at least the columns and below 2^31", name);
  return ITEXHIP_OK;
}

// Shares of K for one tile of rows: enough workgroups for the device where tokens are few
int splits_of(int64_t in) {
  const int64_t n = (in + 511) / 512;
  return static_cast<int>(n < kMaxSplits ? n : kMaxSplits);
}

template <int T>
void run_adapters(AdapterArgs A, hipStream_t st) {
  const bool vec = A.in % 8 == 0 && aligned(A.x, 16) && aligned(A.a, 16) && (A.p.x_stride * element_size(T)) % 16 == 0;
  const int steps = (A.in + 31) / 32;
  A.per_split = (steps + A.splits - 1) / A.splits;
  const auto shrink = vec ? shrink_kernel<T, true> : shrink_kernel<T, false>;
  launch_blocks(tiles_bound(A.tokens, A.p.adapters, 16, false) * A.splits * ((A.deep + 15) / 16), [&](int64_t first, unsigned count) {
    A.first = first;
    shrink<<<count, 256, 0, st>>>(A);
  });
  launch_blocks(tiles_bound(A.tokens, A.p.adapters, 16, true) * ((A.blocks[A.p.n_slices - 1] + 3) / 4), [&](int64_t first, unsigned count) {
    A.first = first;
    expand_kernel<T><<<count, 256, 0, st>>>(A);
  });
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int64_t itexhip_adapters_workspace(const itexhip_adapters_params* p) {
  if (check(p, "itexhip_adapters_workspace") != ITEXHIP_OK) return 0;
  return (static_cast<int64_t>(splits_of(p->in)) * p->tokens * p->n_slices * p->rank * 4 + 255) / 256 * 256 + 256;
}

extern "C" int itexhip_adapters(const itexhip_adapters_params* p, const void* x, const int32_t* offsets, const int32_t* rows, const void* a, const void* b,
                                const int32_t* ranks, const float* scales, const void* base, void* out, void* workspace, void* stream) {
  if (const int e = check(p, "itexhip_adapters")) return e;
  if (p->tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(x && offsets && rows && a && b && scales && base && out && workspace, "itexhip_adapters: null buffer");
  const size_t size = static_cast<size_t>(element_size(p->type));
  ITEXHIP_REQUIRE(aligned(x, size) && aligned(a, size) && aligned(base, size) && aligned(out, size) && aligned(offsets, 4) && aligned(rows, 4) &&
                      aligned(ranks, 4) && aligned(scales, 4),
                  "itexhip_adapters: buffers are aligned to their elements");
  ITEXHIP_REQUIRE(aligned(b, 16) && aligned(workspace, 16), "itexhip_adapters: b and the workspace are aligned to 16 bytes");
  ITEXHIP_REQUIRE(out != base || p->out_stride == p->base_stride, "itexhip_adapters: in place, base_stride and out_stride are the same");
  AdapterArgs A{};
  A.p = *p;
  A.x = x;
  A.a = a;
  A.b = b;
  A.base = base;
  A.offsets = offsets;
  A.rows = rows;
  A.ranks = ranks;
  A.scales = scales;
  A.out = out;
  A.middle = static_cast<float*>(workspace);
  A.tokens = static_cast<int>(p->tokens);
  A.deep = p->n_slices * p->rank;
  A.splits = splits_of(p->in);
  A.in = static_cast<int>(p->in);
  A.columns = static_cast<int>(p->slice_end[p->n_slices - 1]);
  int64_t begin = 0;
  for (int i = 0, blocks = 0; i < p->n_slices; ++i) {
    blocks += static_cast<int>((p->slice_end[i] - begin + 63) / 64);
    A.blocks[i] = blocks;
    begin = p->slice_end[i];
  }
  hipStream_t st = as_stream(stream);
  if (p->type == ITEXHIP_FLOAT) run_adapters<ITEXHIP_FLOAT>(A, st);
  else if (p->type == ITEXHIP_BFLOAT16) run_adapters<ITEXHIP_BFLOAT16>(A, st);
  else run_adapters<ITEXHIP_HALF>(A, st);
  ITEXHIP_CHECK_LAUNCH("itexhip_adapters");
  return ITEXHIP_OK;
}
