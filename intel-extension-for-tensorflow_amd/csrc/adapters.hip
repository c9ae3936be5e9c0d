// Low-rank adapters of many requests beside a shared projection: x A^T of each row's adapter, then the base plus its product with B^T.
#include <type_traits>

#include "chosen.hpp"
#include "qgemm_common.hpp"

namespace itexhip {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

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
  int vec;          // runs of columns of base and out are aligned
  int blocks[ITEXHIP_ADAPTER_MAX_SLICES];  // a workgroup's columns: how many such blocks there are up to the end of each slice
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

// N neighbouring elements (an even number), aligned to 16 bytes, or to all of them if that is less
template <int T, int N>
constexpr int run_alignment() { return N * (T == ITEXHIP_FLOAT ? 4 : 2) < 16 ? N * (T == ITEXHIP_FLOAT ? 4 : 2) : 16; }
template <int T, int N>
struct Run {
  static constexpr int WORDS = N * (T == ITEXHIP_FLOAT ? 4 : 2) / 4;
  uint32_t w[WORDS];
  // PASSING: past the caches' order of use, for tensors that do not stay in them
  template <bool PASSING = false>
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    if constexpr (PASSING && WORDS == 4) {
      const v4i v = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(static_cast<const char*>(base) + i * (T == ITEXHIP_FLOAT ? 4 : 2)));
      __builtin_memcpy(w, &v, 16);
      return;
    }
    __builtin_memcpy(w, __builtin_assume_aligned(static_cast<const char*>(base) + i * (T == ITEXHIP_FLOAT ? 4 : 2), run_alignment<T, N>()), 4 * WORDS);
  }
  template <bool PASSING = false>
  __device__ __forceinline__ void store(void* base, int64_t i) const {
    if constexpr (PASSING && WORDS == 4) {
      v4i v;
      __builtin_memcpy(&v, w, 16);
      __builtin_nontemporal_store(v, reinterpret_cast<v4i*>(static_cast<char*>(base) + i * (T == ITEXHIP_FLOAT ? 4 : 2)));
      return;
    }
    __builtin_memcpy(__builtin_assume_aligned(static_cast<char*>(base) + i * (T == ITEXHIP_FLOAT ? 4 : 2), run_alignment<T, N>()), w, 4 * WORDS);
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (T == ITEXHIP_FLOAT) return __uint_as_float(w[j]);
    const uint32_t h = (w[j / 2] >> (16 * (j % 2))) & 0xffffu;
    return T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
  }
  __device__ __forceinline__ void set(int j, float x, float y) {  // elements j and j + 1, j even
    if constexpr (T == ITEXHIP_FLOAT) {
      w[j] = __float_as_uint(x);
      w[j + 1] = __float_as_uint(y);
    } else {
      w[j / 2] = f32x2_to_bits16<T>(x, y);
    }
  }
  // one by one, of a row that ends `count` elements on
  __device__ __forceinline__ void load_some(const void* base, int64_t i, int count) {
#pragma unroll
    for (int j = 0; j < N; j += 2) set(j, j < count ? load_value<T>(base, i + j) : 0.0f, j + 1 < count ? load_value<T>(base, i + j + 1) : 0.0f);
  }
  __device__ __forceinline__ void store_some(void* base, int64_t i, int count) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) {
        if constexpr (T == ITEXHIP_FLOAT) static_cast<uint32_t*>(base)[i + j] = w[j];
        else static_cast<uint16_t*>(base)[i + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2)));
      }
  }
};

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

// x A^T.  A workgroup has 16 RT places of one adapter, up to 16 CT of one slice's rows of A and a share of K.  Its wavefronts take the
// share's steps of 32 in turns, so that together they read 256 consecutive bytes of a row, and add up in LDS.  Operands go straight from
// memory to registers: x is read once, A stays in L2.  8192 tokens of 4096, rank 64 (bfloat16): 21 to 23 us, 2.9 to 3.2 TB/s of x, with A four times as many
// bytes from L2 again.  One token: 4 us, a launch and two round trips to memory.
template <int T, bool VEC, int RT, int CT>
__global__ __launch_bounds__(256) void shrink_kernel(const AdapterArgs A) {
  constexpr int PITCH = 16 * CT + 4;
  __shared__ __align__(16) float sums[4][16 * RT * PITCH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups_of = (A.p.rank + 16 * CT - 1) / (16 * CT);
  int64_t id = A.first + blockIdx.x;
  const int split = static_cast<int>(id % A.splits);
  id /= A.splits;
  const int which = static_cast<int>(id % (groups_of * A.p.n_slices)), slice = which / groups_of, r0 = which % groups_of * 16 * CT;
  const RowTile t = find_tile<false>(A.offsets, A.p.adapters, A.tokens, 16 * RT, static_cast<int>(id / (groups_of * A.p.n_slices)));
  if (t.group < 0) return;
  const int rank = rank_of(A, t.group), k0 = (lane >> 4) * 8;
  int64_t x_row[RT], a_row[CT];
  int there[CT];
#pragma unroll
  for (int i = 0; i < RT; ++i) x_row[i] = static_cast<int64_t>(token_of(A, t.begin + min(i * 16 + (lane & 15), t.rows - 1))) * A.p.x_stride;
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const int r = r0 + j * 16 + (lane & 15);
    there[j] = r < rank ? A.in : 0;  // rows behind the rank are not read
    a_row[j] = (static_cast<int64_t>(t.group) * A.deep + slice * A.p.rank + min(r, A.p.rank - 1)) * A.in;
  }
  const int first = split * A.per_split, last = min(first + A.per_split, (A.in + 31) / 32);
  v4f d[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) d[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto load = [&](int c, operand_t<T> (&x)[RT], operand_t<T> (&a)[CT]) {
    const int k = c * 32 + k0;
#pragma unroll
    for (int i = 0; i < RT; ++i) x[i] = load_operand<T, VEC>(A.x, x_row[i], k, A.in);
#pragma unroll
    for (int j = 0; j < CT; ++j) a[j] = load_operand<T, VEC>(A.a, a_row[j], k, there[j]);
  };
  auto multiply = [&](const operand_t<T> (&x)[RT], const operand_t<T> (&a)[CT]) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) d[i][j] = product<T>(a[j], x[i], d[i][j]);
  };
  constexpr int AT_ONCE = 4;
  int c = first + wave;
  for (; c + 4 * (AT_ONCE - 1) < last; c += 4 * AT_ONCE) {
    operand_t<T> x[AT_ONCE][RT], a[AT_ONCE][CT];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) load(c + 4 * u, x[u], a[u]);
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) multiply(x[u], a[u]);
  }
  for (; c < last; c += 4) {
    operand_t<T> x[RT], a[CT];
    load(c, x, a);
    multiply(x, a);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) *reinterpret_cast<v4f*>(&sums[wave][(i * 16 + (lane & 15)) * PITCH + j * 16 + (lane >> 4) * 4]) = d[i][j];
  __syncthreads();
  constexpr int FOURS = 4 * CT;  // of a row
  for (int n = threadIdx.x; n < 16 * RT * FOURS; n += 256) {
    const int place = n / FOURS, r = n % FOURS * 4;
    if (place >= t.rows || r0 + r >= A.p.rank) continue;  // (rank is a multiple of 8)
    v4f sum = *reinterpret_cast<const v4f*>(&sums[0][place * PITCH + r]);
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const v4f more = *reinterpret_cast<const v4f*>(&sums[w][place * PITCH + r]);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += more[i];
    }
    *reinterpret_cast<v4f*>(A.middle + (static_cast<int64_t>(split) * A.tokens + t.begin + place) * A.deep + slice * A.p.rank + r0 + r) = sum;
  }
}

// A power of two that brings a row's largest absolute value (its bits) to 2^8 .. 2^9, and its inverse
__device__ __forceinline__ void power_of(uint32_t bits, float* up, float* down) {
  const int e = min(max(static_cast<int>(bits >> 23), 20), 240);  // of 2^(e - 127)
  *up = __uint_as_float(static_cast<uint32_t>(262 - e) << 23);
  *down = __uint_as_float(static_cast<uint32_t>(e - 8) << 23);
}

// out = base + scale (x A^T) B^T.  A wavefront has 16 NT columns of one slice, whose rows of B it keeps in registers (KS steps of 32 of the rank),
// and goes through up to ROWS places of one adapter, 16 at a time.  A lane's column of the j-th tile is NT (lane % 16) + j of them, so that it ends
// with NT neighbouring columns of four rows and 16 lanes with a run of 16 NT.  The workgroup adds up the shares of x A^T and holds them in LDS as operands: the
// sum of two numbers of the type (one of bfloat16 alone would be off by 2^-9 of it); in half precision times a power of two that keeps a
// row's largest in range.  Bound by memory: 8192 tokens of 14336 columns, rank 64, take 118 to 123 us for 470 MB, 3.8 to 4.0 TB/s, the next 16 rows' base on its way
// while the last ones are multiplied (without that 241).  With x A^T, a pass of 64 rows a workgroup took 144 us, 128 147, 256 162; three wavefronts a SIMD 147, two 162;
// stores past the caches' order of use 144 -> 136.
template <int T, int KS, int NT, int ROWS>
__global__ __launch_bounds__(256, KS <= 2 ? 3 : 2) void expand_kernel(const AdapterArgs A) {
  constexpr int SIZE = T == ITEXHIP_FLOAT ? 4 : 2, PARTS = T == ITEXHIP_FLOAT ? 1 : 2;
  constexpr int PITCH = KS * 32 * SIZE + 16;
  __shared__ __align__(16) uint8_t operands[2][PARTS][16 * PITCH];
  __shared__ float downs[2][16];
  __shared__ int tokens[ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all = A.blocks[A.p.n_slices - 1];
  const int64_t id = A.first + blockIdx.x;
  const int index = static_cast<int>(id / all), block = static_cast<int>(id - static_cast<int64_t>(index) * all);
  const RowTile t = find_tile<true>(A.offsets, A.p.adapters, A.tokens, ROWS, index);
  if (t.group < 0) return;
  const bool none = t.group == A.p.adapters;
  if (none && A.out == A.base) return;
  int slice = 0;
  while (block >= A.blocks[slice]) ++slice;
  const int slice_begin = slice == 0 ? 0 : static_cast<int>(A.p.slice_end[slice - 1]), slice_end = static_cast<int>(A.p.slice_end[slice]);
  const int column0 = slice_begin + ((block - (slice == 0 ? 0 : A.blocks[slice - 1])) * 4 + wave) * (16 * NT);
  const int column = column0 + (lane & 15) * NT;  // the lane's first
  const int rank = none ? 0 : rank_of(A, t.group);
  const float scale = none ? 0.0f : A.scales[t.group];
  const bool vec = A.vec && column + NT <= slice_end;

  operand_t<T> b[KS][NT];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = s * 32 + (lane >> 4) * 8;
      const int64_t row = (static_cast<int64_t>(none ? 0 : t.group) * A.columns + min(column + j, slice_end - 1)) * A.p.rank;
      b[s][j] = load_operand<T, true>(A.b, row, r, (rank + 7) / 8 * 8);
      if (rank % 8 != 0) cut<T>(b[s][j], rank - r);
    }

  for (int n = threadIdx.x; n < ROWS; n += 256) tokens[n] = token_of(A, t.begin + min(n, t.rows - 1));
  const int row = threadIdx.x >> 4, part = threadIdx.x & 15;  // 16 threads a row of operands
  constexpr int EACH = KS * 2;  // r that a thread has, in pairs from 2 part on
  struct Round {
    float v[EACH];
    Run<T, NT> base[4];  // of the lane's rows, 4 (lane / 16) .. + 3
  };
  auto load_middle = [&](int n, Round& q) {
    const float* from = A.middle + static_cast<int64_t>(t.begin + min(n * 16 + row, t.rows - 1)) * A.deep + slice * A.p.rank + part * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float2 sum = {0.0f, 0.0f};
      if (s * 32 + part * 2 < rank) {
        sum = *reinterpret_cast<const float2*>(from + s * 32);
        for (int o = 1; o < A.splits; o += 5) {  // five at a time on their way
          float2 more[5];
#pragma unroll
          for (int i = 0; i < 5; ++i) more[i] = *reinterpret_cast<const float2*>(from + s * 32 + static_cast<int64_t>(min(o + i, A.splits - 1)) * A.tokens * A.deep);
#pragma unroll
          for (int i = 0; i < 5; ++i) {
            sum.x += o + i < A.splits ? more[i].x : 0.0f;
            sum.y += o + i < A.splits ? more[i].y : 0.0f;
          }
        }
      }
      q.v[2 * s] = sum.x;
      q.v[2 * s + 1] = s * 32 + part * 2 + 1 < rank ? sum.y : 0.0f;
    }
  };
  auto load_base = [&](int n, Round& q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = n * 16 + (lane >> 4) * 4 + i;
      if (m >= t.rows || column >= slice_end) continue;
      const int64_t at = static_cast<int64_t>(tokens[m]) * A.p.base_stride + column;
      if (vec) q.base[i].template load<(ROWS > 16)>(A.base, at);
      else q.base[i].load_some(A.base, at, slice_end - column);
    }
  };
  const int rounds = (t.rows + 15) / 16;
  Round now, next;
  load_middle(0, now);
  __syncthreads();
  load_base(0, now);
  for (int n = 0; n < rounds; ++n) {
    const int parity = n & 1;
    float up = 1.0f, down = 1.0f;
    if constexpr (T == ITEXHIP_HALF) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) top = max(top, __float_as_uint(now.v[i]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < 16; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
      power_of(top, &up, &down);
      if (part == 0) downs[parity][row] = down;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint8_t* const to = operands[parity][0] + row * PITCH + (s * 32 + part * 2) * SIZE;
      if constexpr (T == ITEXHIP_FLOAT) {
        *reinterpret_cast<float2*>(to) = float2{now.v[2 * s], now.v[2 * s + 1]};
      } else {
        const float a = now.v[2 * s] * up, c = now.v[2 * s + 1] * up;
        const uint32_t hi = f32x2_to_bits16<T>(a, c);
        const float ha = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(hi & 0xffffu) : f16_bits_to_f32(hi & 0xffffu);
        const float hc = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(hi >> 16) : f16_bits_to_f32(hi >> 16);
        *reinterpret_cast<uint32_t*>(to) = hi;
        *reinterpret_cast<uint32_t*>(operands[parity][PARTS - 1] + row * PITCH + (s * 32 + part * 2) * SIZE) = f32x2_to_bits16<T>(a - ha, c - hc);
      }
    }
    __syncthreads();  // (one a round: the next one's operands go to the other half)
    if (n + 1 < rounds) {
      load_middle(n + 1, next);
      load_base(n + 1, next);
    }
    v4f d[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) d[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < PARTS; ++h) {
        operand_t<T> o;
        __builtin_memcpy(&o, operands[parity][h] + (lane & 15) * PITCH + (s * 32 + (lane >> 4) * 8) * SIZE, sizeof(o));
#pragma unroll
        for (int j = 0; j < NT; ++j) d[j] = product<T>(o, b[s][j], d[j]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = n * 16 + (lane >> 4) * 4 + i;
      if (m >= t.rows || column >= slice_end) continue;
      const float factor = T == ITEXHIP_HALF ? downs[parity][(lane >> 4) * 4 + i] : 1.0f;
      Run<T, NT> y = now.base[i];
      if (!none) {
#pragma unroll
        for (int j = 0; j < NT; j += 2)
          y.set(j, now.base[i].at(j) + scale * (d[j][i] * factor), now.base[i].at(j + 1) + scale * (d[j + 1][i] * factor));
      }
      const int64_t at = static_cast<int64_t>(tokens[m]) * A.p.out_stride + column;
      if (vec) y.template store<(ROWS > 16)>(A.out, at);
      else y.store_some(A.out, at, slice_end - column);
    }
    now = next;
  }
}

// Both products in one launch, for ranks up to 16: a workgroup makes x A^T of its 16 places and one slice for itself, 16 wavefronts a share of K each, and
// goes on with 1024 columns, whose B and base travel meanwhile.  A is read once for every such block of columns, from L2 but for the first time.
// One launch : two in us (runs differ by the host's pace), 1 token of 1024 to 4096 columns 6.6 : 7.7-9.4, of 2048 7.5 : 7.9-9.3, of 4096 9.5 : 8.4-9.7;
// 64 of 1024 to 1024, an adapter each, 7.5 : 8.7-10.8; 1000 of 512 to 2048 8.4 : 9.3-11.6, 4000 of 512 to 1024 (4 MB of A read in all) 13.6-14.2 :
// 13.2-14.0; 2000 of 1024 to 4096 (16 MB) 21 : 16.  fp32 and ranks of 32 do not fit the registers of 16 wavefronts.
constexpr int kOnceWaves = 16;
template <int T>
__global__ __launch_bounds__(64 * kOnceWaves) void once_kernel(const AdapterArgs A) {
  constexpr int NT = 4, PITCH = 32 * 2 + 16, SUMS = 16 + 4;
  __shared__ __align__(16) float sums[kOnceWaves][16 * SUMS];
  __shared__ __align__(16) uint8_t operands[2][16 * PITCH];
  __shared__ float downs[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all = A.blocks[A.p.n_slices - 1];
  const int64_t id = A.first + blockIdx.x;
  const int index = static_cast<int>(id / all), block = static_cast<int>(id - static_cast<int64_t>(index) * all);
  const RowTile t = find_tile<true>(A.offsets, A.p.adapters, A.tokens, 16, index);
  if (t.group < 0) return;
  const bool none = t.group == A.p.adapters;
  if (none && A.out == A.base) return;
  int slice = 0;
  while (block >= A.blocks[slice]) ++slice;
  const int slice_begin = slice == 0 ? 0 : static_cast<int>(A.p.slice_end[slice - 1]), slice_end = static_cast<int>(A.p.slice_end[slice]);
  const int column0 = slice_begin + ((block - (slice == 0 ? 0 : A.blocks[slice - 1])) * kOnceWaves + wave) * (16 * NT);
  const int column = column0 + (lane & 15) * NT;  // the lane's first
  const int rank = none ? 0 : rank_of(A, t.group);
  const float scale = none ? 0.0f : A.scales[t.group];
  const bool vec = A.vec && column + NT <= slice_end;
  const int place = lane & 15, k0 = (lane >> 4) * 8;
  const int64_t x_row = static_cast<int64_t>(token_of(A, t.begin + min(place, t.rows - 1))) * A.p.x_stride;

  // B and the base travel while x A^T is made
  operand_t<T> b[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t row = (static_cast<int64_t>(none ? 0 : t.group) * A.columns + min(column + j, slice_end - 1)) * A.p.rank;
    b[j] = load_operand<T, true>(A.b, row, k0, (rank + 7) / 8 * 8);
  }
  Run<T, NT> base[4];
  int64_t token[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = (lane >> 4) * 4 + i;
    if (m >= t.rows || column >= slice_end) continue;
    token[i] = token_of(A, t.begin + m);
    const int64_t at = token[i] * A.p.base_stride + column;
    if (vec) base[i].load(A.base, at);
    else base[i].load_some(A.base, at, slice_end - column);
  }
  v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
  if (!none) {
    const int there = place < rank ? A.in : 0;  // rows behind the rank are not read
    const int64_t a_row = (static_cast<int64_t>(t.group) * A.deep + slice * A.p.rank + min(place, A.p.rank - 1)) * A.in;
    const int steps = (A.in + 31) / 32;
    constexpr int AT_ONCE = 8;
    for (int c = wave; c < steps; c += AT_ONCE * kOnceWaves) {  // (steps behind the last are of zeros)
      operand_t<T> x[AT_ONCE], a[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int k = (c + u * kOnceWaves) * 32 + k0;
        x[u] = load_operand<T, true>(A.x, x_row, k, A.in);
        a[u] = load_operand<T, true>(A.a, a_row, k, there);
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) d = product<T>(a[u], x[u], d);
    }
  }
  *reinterpret_cast<v4f*>(&sums[wave][place * SUMS + (lane >> 4) * 4]) = d;
  __syncthreads();
  {  // a wavefront for each place, its lanes for its values
    float v = 0.0f;
    if (lane < rank) {  // (behind the rank an x that is not finite has left zeros times it)
#pragma unroll
      for (int w = 0; w < kOnceWaves; ++w) v += sums[w][wave * SUMS + lane];
    }
    float up = 1.0f, down = 1.0f;
    if constexpr (T == ITEXHIP_HALF) {
      uint32_t top = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m)));
      power_of(top, &up, &down);
      if (lane == 0) downs[wave] = down;
    }
    if (lane < 32) {  // (zeros from 16 on)
      const float a = v * up;
      const uint32_t hi = f32_to_bits16<T>(a);
      const float h = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi);
      *reinterpret_cast<uint16_t*>(operands[0] + wave * PITCH + lane * 2) = static_cast<uint16_t>(hi);
      *reinterpret_cast<uint16_t*>(operands[1] + wave * PITCH + lane * 2) = static_cast<uint16_t>(f32_to_bits16<T>(a - h));
    }
  }
  __syncthreads();
  if (column0 >= slice_end) return;  // the whole wavefront
  v4f y[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) y[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < NT; ++j)
    if (rank % 8 != 0) cut<T>(b[j], rank - k0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    operand_t<T> o;
    __builtin_memcpy(&o, operands[h] + place * PITCH + k0 * 2, sizeof(o));
#pragma unroll
    for (int j = 0; j < NT; ++j) y[j] = product<T>(o, b[j], y[j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = (lane >> 4) * 4 + i;
    if (m >= t.rows || column >= slice_end) continue;
    const float factor = T == ITEXHIP_HALF ? downs[m] : 1.0f;
    Run<T, NT> r = base[i];
    if (!none) {
#pragma unroll
      for (int j = 0; j < NT; j += 2)
        r.set(j, base[i].at(j) + scale * (y[j][i] * factor), base[i].at(j + 1) + scale * (y[j + 1][i] * factor));
    }
    const int64_t at = token[i] * A.p.out_stride + column;
    if (vec) r.store(A.out, at);
    else r.store_some(A.out, at, slice_end - column);
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

template <int T, bool VEC, int RT, int CT>
void launch_shrink(AdapterArgs A, hipStream_t st) {
  const int64_t parts = static_cast<int64_t>((A.p.rank + 16 * CT - 1) / (16 * CT)) * A.p.n_slices;
  const int steps = (A.in + 31) / 32;
  A.per_split = (steps + A.splits - 1) / A.splits;
  launch_blocks(tiles_bound(A.tokens, A.p.adapters, 16 * RT, false) * parts * A.splits, [&](int64_t first, unsigned count) {
    A.first = first;
    shrink_kernel<T, VEC, RT, CT><<<count, 256, 0, st>>>(A);
  });
}
template <int T, bool VEC, int RT>
void launch_shrink(const AdapterArgs& A, hipStream_t st) {
  if (A.p.rank <= 16) launch_shrink<T, VEC, RT, 1>(A, st);
  else if (A.p.rank <= 32) launch_shrink<T, VEC, RT, 2>(A, st);
  else launch_shrink<T, VEC, RT, 4>(A, st);
}

template <int T, int KS, int NT, int ROWS>
void launch_expand(AdapterArgs A, hipStream_t st) {
  int64_t begin = 0;
  for (int i = 0, blocks = 0; i < A.p.n_slices; ++i) {
    blocks += static_cast<int>((A.p.slice_end[i] - begin + 64 * NT - 1) / (64 * NT));
    A.blocks[i] = blocks;
    begin = A.p.slice_end[i];
  }
  launch_blocks(tiles_bound(A.tokens, A.p.adapters, ROWS, true) * A.blocks[A.p.n_slices - 1], [&](int64_t first, unsigned count) {
    A.first = first;
    expand_kernel<T, KS, NT, ROWS><<<count, 256, 0, st>>>(A);
  });
}
template <int T, int KS, int NT>
void launch_expand(const AdapterArgs& A, hipStream_t st) {
  if (long_expand(A.tokens, A.p.adapters, A.columns, 64 * NT)) launch_expand<T, KS, NT, 64>(A, st);
  else launch_expand<T, KS, NT, 16>(A, st);
}
template <int T>
void launch_expand(const AdapterArgs& A, hipStream_t st) {
  constexpr int NT = T == ITEXHIP_FLOAT ? 4 : 8;  // 16 bytes of a lane's row; fewer where more would not fit the registers
  if (A.p.rank <= 32) launch_expand<T, 1, NT>(A, st);
  else if (A.p.rank <= 64) launch_expand<T, 2, NT>(A, st);
  else if (A.p.rank <= 128) launch_expand<T, 4, 4>(A, st);
  else launch_expand<T, 8, T == ITEXHIP_FLOAT ? 2 : 4>(A, st);
}

template <int T>
void launch_once(AdapterArgs A, hipStream_t st) {
  constexpr int COLUMNS = 64 * kOnceWaves;
  int64_t begin = 0;
  for (int i = 0, blocks = 0; i < A.p.n_slices; ++i) {
    blocks += static_cast<int>((A.p.slice_end[i] - begin + COLUMNS - 1) / COLUMNS);
    A.blocks[i] = blocks;
    begin = A.p.slice_end[i];
  }
  launch_blocks(tiles_bound(A.tokens, A.p.adapters, 16, true) * A.blocks[A.p.n_slices - 1], [&](int64_t first, unsigned count) {
    A.first = first;
    once_kernel<T><<<count, 64 * kOnceWaves, 0, st>>>(A);
  });
}
template <int T>
void run_adapters(AdapterArgs A, hipStream_t st) {
  const int64_t size = element_size(T);
  const bool vec = A.in % 8 == 0 && aligned(A.x, 16) && aligned(A.a, 16) && (A.p.x_stride * size) % 16 == 0;
  A.vec = aligned(A.base, 16) && aligned(A.out, 16) && (A.p.base_stride * size) % 16 == 0 && (A.p.out_stride * size) % 16 == 0;
  for (int i = 0; i + 1 < A.p.n_slices; ++i) A.vec = A.vec && (A.p.slice_end[i] * size) % 16 == 0;
  if constexpr (T != ITEXHIP_FLOAT) {
    if (vec && one_launch(A.tokens, A.p.adapters, A.p.rank, A.p.n_slices, A.in, A.columns)) return launch_once<T>(A, st);
  }
  const bool wide = long_tiles(A.tokens, A.p.adapters);
  if (vec) wide ? launch_shrink<T, true, 4>(A, st) : launch_shrink<T, true, 1>(A, st);
  else wide ? launch_shrink<T, false, 4>(A, st) : launch_shrink<T, false, 1>(A, st);
  launch_expand<T>(A, st);
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int64_t itexhip_adapters_workspace(const itexhip_adapters_params* p) {
  if (check(p, "itexhip_adapters_workspace") != ITEXHIP_OK) return 0;
  return (middle_rows(p->tokens) * p->n_slices * p->rank * 4 + 255) / 256 * 256 + 256;
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
  A.splits = splits_of(p->tokens, p->adapters, static_cast<int64_t>(p->n_slices) * shrink_parts(p->rank), p->in);
  A.in = static_cast<int>(p->in);
  A.columns = static_cast<int>(p->slice_end[p->n_slices - 1]);
  hipStream_t st = as_stream(stream);
  if (p->type == ITEXHIP_FLOAT) run_adapters<ITEXHIP_FLOAT>(A, st);
  else if (p->type == ITEXHIP_BFLOAT16) run_adapters<ITEXHIP_BFLOAT16>(A, st);
  else run_adapters<ITEXHIP_HALF>(A, st);
  ITEXHIP_CHECK_LAUNCH("itexhip_adapters");
  return ITEXHIP_OK;
}
