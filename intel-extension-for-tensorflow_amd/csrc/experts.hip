// The experts' quantized products: rows of activations to codes, the products of each row's expert, each token's sum of its experts.
#include "chosen.hpp"
#include "qgemm_common.hpp"

namespace itexhip {
namespace {

// ------------------------------------------------------------------------------------------------
// Rows to codes.  s = max(absmax / 127, 2^-100); code = rne(x / s) of the quotient itself: the product with the reciprocal is
// next to it, and the remainder x - n s, which is a multiple of ulp(s) / 2 below 2 s and therefore exact in one fma, tells
// whether the nearest integer is n or a neighbour, and where it is halfway.
// Rows of codes are `pitch` bytes (K rounded up to 64), zeros behind K: the packed weights' K steps.
// A workgroup has a row and keeps it between the two passes.  8192 rows of 14336 (bfloat16) take 68 us, 5.2 TB/s read and written (85 with every
// element through its remainder).
// ------------------------------------------------------------------------------------------------
constexpr float kLeastScale = 0x1p-100f;

__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float n = __builtin_rintf(x * inv);
  const float r = fmaf(-n, s, x), half = 0.5f * s;
  if (r > half) n += 1.0f;
  else if (r < -half) n -= 1.0f;
  else if ((r == half || r == -half) && (static_cast<int>(n) & 1)) n += r > 0.0f ? 1.0f : -1.0f;
  return static_cast<int>(n);
}
// Eight codes in two words.  The fma with 3 2^22 brings the nearest integer of x / s (1 + e), |e| <= 2^-24, into the low byte; it is that of the quotient
// too where what is left over is 2^-15 or more away from a half, since the two are 127 2^-24 apart at most.  One element in 16000 is not and has
// its wavefront go through the exact remainders.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[8];
  float farthest = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fmaf(x[j], inv, kMagic);
    b[j] = __float_as_uint(a);
    farthest = fmaxf(farthest, fabsf(fmaf(x[j], inv, -(a - kMagic))));
  }
  if (farthest > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = static_cast<uint32_t>(code_of(x[j], s, inv));
  }
  uint2 w;
  w.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
  w.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[7], b[6], 0x0c0c0400u), __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400u), 0x05040100u);
  return w;
}
// of a row's largest absolute value, as its bits (those of NaN are above infinity's)
__device__ __forceinline__ float scale_of(uint32_t absmax_bits) {
  if (absmax_bits >= 0x7f800000u) return __builtin_nanf("");
  return fmaxf(__uint_as_float(absmax_bits) / 127.0f, kLeastScale);
}

// HELD: runs of 8 elements that a thread keeps between the two passes, up to 7 (14336 elements a row; 8 and more were not measured); 0: it reads them again
template <int T, bool VEC, int HELD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, int64_t stride, int K, int pitch, int8_t* __restrict__ codes,
                                                            float* __restrict__ scales, int64_t first) {
  __shared__ uint32_t most[4];
  const int64_t row = first + blockIdx.x, base = row * stride;
  auto load = [&](int k, float (&v)[8]) {
    if (VEC && k + 8 <= K) {
      load8<T>(x, base + k, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < K ? load_value<T>(x, base + k + j) : 0.0f;
    }
  };
  uint32_t top = 0;
  auto largest = [&](const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  };
  float held[HELD > 0 ? HELD : 1][8];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) load(h * 2048 + threadIdx.x * 8, held[h]);
#pragma unroll
    for (int h = 0; h < HELD; ++h) largest(held[h]);
  } else {
    for (int k = threadIdx.x * 8; k < K; k += 2048) {
      float v[8];
      load(k, v);
      largest(v);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(most[0], most[1]), max(most[2], most[3]));
  const float s = scale_of(top), inv = 1.0f / s;
  const bool finite = s == s;
  if (threadIdx.x == 0) scales[row] = s;
  auto store = [&](int k, const float (&v)[8]) {
    *reinterpret_cast<uint2*>(codes + row * pitch + k) = finite ? codes_of(v, s, inv) : uint2{0u, 0u};
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (h * 2048 + static_cast<int>(threadIdx.x) * 8 < pitch) store(h * 2048 + threadIdx.x * 8, held[h]);
  } else {
    for (int k = threadIdx.x * 8; k < pitch; k += 2048) {
      float v[8];
      load(k, v);
      store(k, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Products
// ------------------------------------------------------------------------------------------------
struct ProductArgs {
  const int8_t* codes;       // [rows of the source][pitch]
  const float* row_scales;   // of the source's rows
  const int8_t* packed;      // [experts][each][panel]
  const float* scales;       // [experts][each][N]
  const int32_t *offsets, *rows;
  void* out;                 // up: h, [place][N];  down: fp32, [slot][N]
  const void* x;             // the source itself, for kernels that make the codes
  int64_t x_stride;
  bool x_vec;                // its rows are aligned to 16 bytes
  int64_t panel;
  int experts, slots, top_k; // slots = tokens * top_k
  int K;
  int few;                   // rows of a tile whose workgroups make its codes, at most kFewRows
  int pitch, chunks, N;      // chunks of 32 k, an even number
  int strips;                // of 32 channels
  int64_t first;             // workgroup of the launch
  int activation;
};

__device__ __forceinline__ float activate(int activation, float x) {
  switch (activation) {
    case ITEXHIP_ACT_RELU: return x <= 0.0f ? 0.0f : x;  // (NaN stays, which a maximum would drop)
    case ITEXHIP_ACT_GELU_APPROX: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_GELU_TANH, 0.0f, 0.0f}, x);
    case ITEXHIP_ACT_GELU_EXACT: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_GELU_ERF, 0.0f, 0.0f}, x);
    case ITEXHIP_ACT_SWISH: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_SWISH, 1.0f, 0.0f}, x);
    default: return x;
  }
}

// Where a place's codes are, and (down) where its result goes.  What `rows` holds is cut to the slots there are.
__device__ __forceinline__ int slot_of(const ProductArgs& A, int place) { return min(max(A.rows[place], 0), A.slots - 1); }

// Codes and scales of a few rows in LDS, by all wavefronts of a workgroup: each has a share of one row.  `at` gives a row's first element.
// All of them wait twice.
template <int T, int WAVES, class F>
__device__ __forceinline__ void quantize_few(const void* x, bool vec, int rows, int K, int pitch, int8_t* codes, float* scales, uint32_t (&most)[WAVES], F&& at) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int shares = max(1, WAVES / rows), share = wave / rows;
  for (int r0 = 0; r0 < rows; r0 += WAVES) {  // (more rows than wavefronts: in turns)
    const int row = r0 + (rows <= WAVES ? wave % rows : wave);
    const bool there = row < rows && share < shares;
    const int64_t base = at(min(row, rows - 1));
    auto load = [&](int k, float (&v)[8]) {
      if (vec && k + 8 <= K) {
        load8<T>(x, base + k, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < K ? load_value<T>(x, base + k + j) : 0.0f;
      }
    };
    uint32_t top = 0;
    if (there) {
      for (int k = (share * 64 + lane) * 8; k < K; k += shares * 512) {
        float v[8];
        load(k, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
    if (lane == 0) most[wave] = top;
    __syncthreads();
    if (there) {
      if (rows <= WAVES)
        for (int o = 0; o < shares; ++o) top = max(top, most[row + o * rows]);
      const float s = scale_of(top), inv = 1.0f / s;
      if (share == 0 && lane == 0) scales[row] = s;
      for (int k = (share * 64 + lane) * 8; k < pitch; k += shares * 512) {
        float v[8];
        load(k, v);
        *reinterpret_cast<uint2*>(codes + row * pitch + k) = s == s ? codes_of(v, s, inv) : uint2{0u, 0u};
      }
    }
    __syncthreads();
  }
}

// Weights that one workgroup reads once: past the caches' order of use
__device__ __forceinline__ v4i load_once(const int8_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p)); }

// Few rows an expert: each wavefront streams a share of the K chunks of a strip of 32 channels past up to 32 rows, the next chunks on
// their way while the last ones are multiplied; the shares' sums meet in LDS.  The rows' codes come from the caches, or (SOURCE: the
// type of x) the workgroup makes them itself, which saves a launch where rows are very few.
// Bound by memory: one token's two experts of 4096 x 14336, gate and up, 235 MB, take 40 us (5.8 TB/s), 64 tokens through 64 experts of
// 2048 x 1408, 369 MB, 55 to 57 with the codes' launch (6.5 TB/s; the profiler has 59 for this one alone, 54 at best).  With each batch of chunks waited for before the next is asked for the latter took 70.
// OUT: type of h (up), or 0: fp32 by slot (down).
template <int OUT, bool GATED, int WAVES, int SOURCE>
__global__ __launch_bounds__(64 * WAVES) void experts_stream_kernel(const ProductArgs A) {
  constexpr int EACH = GATED ? 2 : 1, PITCH = 36;
  constexpr bool UP = OUT != 0, FUSED = SOURCE != 0;
  __shared__ __align__(16) int sums[EACH][WAVES][32 * PITCH];
  __shared__ float few_scales[kFewRows];
  __shared__ uint32_t most[WAVES];
  extern __shared__ __align__(16) int8_t few_codes[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = A.first + blockIdx.x;
  const int index = static_cast<int>(id / A.strips), strip = static_cast<int>(id - static_cast<int64_t>(index) * A.strips);
  const RowTile t = find_tile<false>(A.offsets, A.experts, A.slots, FUSED ? A.few : 32, index);
  if (t.group < 0) return;
  const int8_t* weights = A.packed + static_cast<int64_t>(t.group) * EACH * A.panel + static_cast<int64_t>(strip) * A.chunks * kChunkBytes + lane * 16;
  v16i acc[EACH];
#pragma unroll
  for (int w = 0; w < EACH; ++w)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[w][r] = 0;
  constexpr int AT_ONCE = 4;
  struct Batch {
    v4i b[AT_ONCE][EACH];
  };
  // chunks c, c + WAVES ...; behind the last one that chunk again, which is not multiplied
  auto load = [&](int c, Batch& to) {
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
      for (int w = 0; w < EACH; ++w) to.b[u][w] = load_once(weights + w * A.panel + static_cast<int64_t>(min(c + u * WAVES, A.chunks - 1)) * kChunkBytes);
  };
  Batch now, next;
  load(wave, now);
  const int8_t* source;
  if constexpr (FUSED) {
    quantize_few<SOURCE, WAVES>(A.x, A.x_vec, t.rows, A.K, A.pitch, few_codes, few_scales, most,
                                [&](int r) { return static_cast<int64_t>(slot_of(A, t.begin + r) / A.top_k) * A.x_stride; });
    source = few_codes + min(lane & 31, t.rows - 1) * A.pitch + (lane >> 5) * 16;
  } else {
    const int place = t.begin + min(lane & 31, t.rows - 1);
    const int row = UP ? slot_of(A, place) / A.top_k : place;
    source = A.codes + static_cast<int64_t>(row) * A.pitch + (lane >> 5) * 16;
  }
  for (int c = wave; c < A.chunks; c += AT_ONCE * WAVES) {
    v4i a[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) a[u] = *reinterpret_cast<const v4i*>(source + min(c + u * WAVES, A.chunks - 1) * 32);
    if (c + AT_ONCE * WAVES < A.chunks) load(c + AT_ONCE * WAVES, next);
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (c + u * WAVES >= A.chunks) break;
#pragma unroll
      for (int w = 0; w < EACH; ++w) acc[w] = __builtin_amdgcn_mfma_i32_32x32x32_i8(now.b[u][w], a[u], acc[w], 0, 0, 0);
    }
    now = next;
  }
  // the shares' sums, then four channels of a row a thread
  const int m = threadIdx.x >> 3, n0 = strip * 32 + (threadIdx.x & 7) * 4;
#pragma unroll
  for (int w = 0; w < EACH; ++w)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<v4i*>(&sums[w][wave][(lane & 31) * PITCH + g * 8 + (lane >> 5) * 4]) =
          v4i{acc[w][4 * g], acc[w][4 * g + 1], acc[w][4 * g + 2], acc[w][4 * g + 3]};
  __syncthreads();
  if (m >= t.rows) return;
  const int place = t.begin + m;
  const int slot = slot_of(A, place);
  const float s = FUSED ? few_scales[m % kFewRows] : A.row_scales[UP ? slot / A.top_k : place];
  float v[EACH][4];
#pragma unroll
  for (int w = 0; w < EACH; ++w) {
    v4i sum = *reinterpret_cast<const v4i*>(&sums[w][0][m * PITCH + (threadIdx.x & 7) * 4]);
#pragma unroll
    for (int o = 1; o < WAVES; ++o) sum += *reinterpret_cast<const v4i*>(&sums[w][o][m * PITCH + (threadIdx.x & 7) * 4]);
    const float* of = A.scales + (static_cast<int64_t>(t.group) * EACH + w) * A.N;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[w][j] = static_cast<float>(sum[j]) * (s * of[min(n0 + j, A.N - 1)]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float y = v[0][j];
    if constexpr (UP) {
      y = activate(A.activation, y);
      if constexpr (GATED) y = y * v[1][j];
      if (n0 + j < A.N) store_output<OUT>(A.out, static_cast<int64_t>(place) * A.N + n0 + j, y);
    } else {
      if (n0 + j < A.N) static_cast<float*>(A.out)[static_cast<int64_t>(slot) * A.N + n0 + j] = y;
    }
  }
}

// The way back of very few choices in one launch: a workgroup has a strip of 32 channels of every expert that is chosen.  Its
// wavefronts divide the experts and, within one, the chunks of K; every place of the order is a row of every product, and where the sums meet each place
// takes its own expert's.  Then the strip's part of each token is all there.  One token's two experts of 14336 x 4096, 118 MB, take 28 us, of which the codes,
// made by every workgroup for itself while its first chunks travel, are about 3; three launches took 48.
struct FewArgs {
  const int32_t* experts;
  const float* weights;
  const void* addend;
  int64_t addend_stride, out_stride;
  int tokens;
};
constexpr int kFewWaves = 16;
template <int T>
__global__ __launch_bounds__(64 * kFewWaves) void experts_few_down_kernel(const ProductArgs A, const FewArgs F) {
  constexpr int PITCH = 36;
  __shared__ __align__(16) int sums[kFewWaves][kFewPlaces * PITCH];  // of a share: a place's own expert
  __shared__ float results[kFewPlaces][32];
  __shared__ float row_scales[kFewPlaces];
  __shared__ uint32_t most[kFewWaves];
  extern __shared__ __align__(16) int8_t few_codes[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), strip = blockIdx.x;
  // the lane's place (the upper lanes hold them again), its slot and expert, -1: none here
  const int place = lane & (kFewPlaces - 1);
  const int slot = slot_of(A, min(place, A.slots - 1));
  int expert = F.experts[slot];
  if (place >= A.slots || expert < 0 || expert >= A.experts) expert = -1;
  // experts in the order of their first places
  int order = -1, number = 0;
  for (int p = 0; p < A.slots; ++p) {
    const int e = __builtin_amdgcn_readlane(expert, p);
    if (e < 0) continue;
    const unsigned long long same = __ballot(expert == e);
    if (__builtin_ctzll(same) != p) continue;
    if (expert == e) order = number;
    ++number;
  }
  number = __builtin_amdgcn_readfirstlane(number);
  if (number > 0) {  // (the same for all wavefronts: they all saw the same values)
    const int shares = kFewWaves / number, mine = wave % number, share = wave / number;
    const int e = __builtin_amdgcn_readlane(expert, __builtin_ctzll(__ballot(order == mine)));
    const int8_t* weights = A.packed + static_cast<int64_t>(e) * A.panel + static_cast<int64_t>(strip) * A.chunks * kChunkBytes + lane * 16;
    constexpr int AT_ONCE = 8;
    v4i now[AT_ONCE], next[AT_ONCE];
    auto load = [&](int c, v4i (&to)[AT_ONCE]) {
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) to[u] = load_once(weights + static_cast<int64_t>(min(c + u * shares, A.chunks - 1)) * kChunkBytes);
    };
    if (share < shares) load(share, now);
    quantize_few<T, kFewWaves>(A.x, A.x_vec, A.slots, A.K, A.pitch, few_codes, row_scales, most, [&](int r) { return r * A.x_stride; });
    if (share < shares) {
      const int8_t* source = few_codes + min(lane & 31, A.slots - 1) * A.pitch + (lane >> 5) * 16;
      v16i acc;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] = 0;
      for (int c = share; c < A.chunks; c += AT_ONCE * shares) {
        if (c + AT_ONCE * shares < A.chunks) load(c + AT_ONCE * shares, next);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          if (c + u * shares >= A.chunks) break;
          acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(now[u], *reinterpret_cast<const v4i*>(source + (c + u * shares) * 32), acc, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) now[u] = next[u];
      }
      if ((lane & 31) == place && order == mine) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4i*>(&sums[share][place * PITCH + g * 8 + (lane >> 5) * 4]) = v4i{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
      }
    }
    __syncthreads();
    // a thread for each place and channel
    const int p = threadIdx.x >> 5, n = threadIdx.x & 31;
    const int to = __shfl(slot, p), which = __shfl(order, p), its = __shfl(expert, p);
    if (p < A.slots && which >= 0) {
      int sum = 0;
      for (int o = 0; o < shares; ++o) sum += sums[o][p * PITCH + n];
      results[to][n] = static_cast<float>(sum) * (row_scales[p] * A.scales[static_cast<int64_t>(its) * A.N + min(strip * 32 + n, A.N - 1)]);
    }
    __syncthreads();
  }
  const int token = threadIdx.x >> 5, n = strip * 32 + (threadIdx.x & 31);
  if (token >= F.tokens || n >= A.N) return;
  float sum = 0.0f;
  for (int c = 0; c < A.top_k; ++c) {
    const int its = F.experts[token * A.top_k + c];
    if (its >= 0 && its < A.experts) sum = sum + F.weights[token * A.top_k + c] * results[token * A.top_k + c][threadIdx.x & 31];
  }
  if (F.addend != nullptr) sum = sum + load_value<T>(F.addend, token * F.addend_stride + n);
  store_output<T>(A.out, token * F.out_stride + n, sum);
}

// ------------------------------------------------------------------------------------------------
// Many rows an expert: tiles of BM places of one expert and BN channels (gated: BN / 2 of the gate and the same BN / 2 of the up weight, so
// that a wavefront ends with both sums of a value), K in steps of 64.  Four wavefronts of (BM / 2) x (BN / 2) accumulators in
// MFMA tiles of 32 x 32, the tiles of rows in turns.  Both operands reach LDS by direct loads, three steps ahead in a ring of four; a step's fragments are read
// during the step before it, one load or read behind each MFMA, so that one wavefront a SIMD keeps the matrix core fed.
// Activation rows lie in LDS 16 to a KiB, a row's four 16-byte pieces in the lanes of a quad, turned by (row / 4) so that the 16 lanes
// served at a time read 16 different bank groups; weights are packed in fragment order and copied as they are.
//
// Tiles are numbered expert by expert, within an expert in groups of up to 8 tiles of rows, there column by column, and each XCD has
// a contiguous run of the experts' last tiles, which are not full, and then of the others: its 32 workgroups share a few columns of weights and up to 8 tiles of rows in their L2.  A workgroup
// stays for all its tiles: the last steps of one fetch the first ones of the next, which then travel while results are written.
//
// 4096 tokens, 2 of 8 experts of 4096 x 14336, gate and up (1.92 TOP): launches apart from one another 1.07 ms, 1.01 at best, 1.8 to 1.9 POP/s; the way back 0.56, 0.55 at best, 1.7 to 1.8.  The board's power bounds it: the matrix
// cores are busy 50 % of the cycles at 1.74 GHz (the way back 43 % at 1.93), so what costs energy costs time.  Steps alone took 0.87 ms of 1.02, as long as this library's MatMul of as many
// rows of one weight; the results' arithmetic, which no matrix instruction covers, makes the difference.  A tile of 256 x 256 has the fewest operand bytes for
// its products that registers allow.  Bases in scalar registers and one offset for all weights' loads of a step brought 1049 to 1015 us.
// ------------------------------------------------------------------------------------------------
constexpr int kTileGroup = 8;  // tiles of rows that share a column
// MFMA tiles of results that go through a wavefront's piece of LDS at a time: 128 bytes of a row
constexpr int tile_pair(int element, int out_tn) { return element == 2 && out_tn >= 2 ? 2 : 1; }
constexpr int tile_lds(int element, int out_tn, int bm, int bn) {
  return 4 * (bm + bn) * 64 + 3 * (bn + 2 * bm) * 4 + 4 * 32 * (tile_pair(element, out_tn) * 32 * element + 16);
}

// The activation of 16 values, chosen once for them
__device__ __forceinline__ void activate16(int activation, float (&y)[16]) {
#define ITEXHIP_EACH(ACT) _Pragma("unroll") for (int r = 0; r < 16; ++r) y[r] = activate(ACT, y[r])
  if (activation == ITEXHIP_ACT_SWISH) ITEXHIP_EACH(ITEXHIP_ACT_SWISH);
  else if (activation == ITEXHIP_ACT_RELU) ITEXHIP_EACH(ITEXHIP_ACT_RELU);
  else if (activation == ITEXHIP_ACT_GELU_APPROX) ITEXHIP_EACH(ITEXHIP_ACT_GELU_APPROX);
  else if (activation == ITEXHIP_ACT_GELU_EXACT) ITEXHIP_EACH(ITEXHIP_ACT_GELU_EXACT);
#undef ITEXHIP_EACH
}

// A pointer that all lanes have, in scalar registers, for loads written as assembly: a memory instruction reads them five wait states after the
// vector instructions that wrote them at the earliest, and the compiler counts those for its own loads only
__device__ __forceinline__ const int8_t* uniform(const int8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
  uint64_t q = static_cast<uint64_t>(hi) << 32 | lo;
  asm volatile("s_nop 4" : "+s"(q));
  return reinterpret_cast<const int8_t*>(q);
}

// lds_dma16 to OFFSET behind lds_addr, the sum formed in m0
template <int OFFSET>
__device__ __forceinline__ void lds_dma16_at(const void* base, uint32_t lane_offset, uint32_t lds_addr) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_offset), "s"(base), "s"(lds_addr), "i"(OFFSET) : "memory", "m0", "scc");
}

// SWISH: the activation, known when compiled; with the others beside it this one's code would be fetched around them
template <int OUT, bool GATED, bool SWISH, int BM, int BN>
__global__ __launch_bounds__(256) void experts_tile_kernel(const ProductArgs A) {
  constexpr bool UP = OUT != 0;
  constexpr int EACH = GATED ? 2 : 1, NSTAGE = 4, AHEAD = 3;
  constexpr int TM = BM / 64, TN = BN / 64;                       // MFMA tiles of a wavefront
  constexpr int A_LOADS = BM / 16, B_LOADS = BN / 16;             // of 1 KiB a step
  constexpr int A_PER_WAVE = A_LOADS / 4, B_PER_WAVE = B_LOADS / 4, NLD = A_PER_WAVE + B_PER_WAVE;
  constexpr int STAGE = (A_LOADS + B_LOADS) * kChunkBytes, B_REGION = A_LOADS * kChunkBytes;
  constexpr int NSLICE = 2 * TN;
  constexpr int OUT_TN = TN / EACH, WIDTH = BN / EACH;            // MFMA tiles of results; channels of a tile
  static_assert(A_LOADS % 4 == 0 && B_LOADS % 4 == 0 && TN % EACH == 0 && NSLICE % 4 == 0, "loads and tiles divide among wavefronts");
  extern __shared__ __align__(16) uint8_t lds[];
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds));
  // behind the ring, for three tiles: scales of its BN channels, wavefront by wavefront, scales of its rows and their slots; then the
  // wavefronts' pieces for results
  constexpr int PANEL = BN + 2 * BM;
  float* const panels = reinterpret_cast<float*>(lds + NSTAGE * STAGE);
  uint8_t* const buffers = lds + NSTAGE * STAGE + 3 * PANEL * 4;

  const int columns = (A.N + WIDTH - 1) / WIDTH;
  // this XCD's tiles: an eighth of the experts' last ones, which are not full, then an eighth of the others; only the offsets tell how many
  const TileCount<false, kFullTiles> full(A.offsets, A.experts, A.slots, BM);
  const TileCount<false, kLastTiles> last(A.offsets, A.experts, A.slots, BM);
  const int xcd = blockIdx.x & 7;
  const int64_t all_full = static_cast<int64_t>(full.total()) * columns, all_last = static_cast<int64_t>(last.total()) * columns;
  const int64_t last_begin = all_last * xcd / 8, last_run = all_last * (xcd + 1) / 8 - last_begin;
  const int64_t full_begin = all_full * xcd / 8, run = last_run + all_full * (xcd + 1) / 8 - full_begin;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave & 1, wn = wave >> 1, lrow = lane & 31, lgrp = lane >> 5;
  const int q_row = lane >> 2, q_piece = (lane & 3) ^ ((q_row >> 2) & 3);
  // column tile c of the block: which weight, and its first channel from the tile's on
  auto which_of = [](int c) { return GATED ? c % TN / OUT_TN : 0; };
  auto channel_of = [](int c) { return (GATED ? c / TN * OUT_TN + c % OUT_TN : c) * 32; };

  struct Work {
    bool there;
    int begin, rows, n_base;
  };
  // Where a tile's operands are loaded from: bases that are the same for the wavefront, and a lane's offsets from them
  struct Source {
    const int8_t* a;
    uint32_t row[A_PER_WAVE];
    const int8_t* b[B_PER_WAVE];
  };
  auto find = [&](int64_t local, Work& w, Source& src, float* panel) {
    w.there = local < run;
    if (!w.there) return;
    const bool whole = local >= last_run;
    const GroupUnit u = whole ? full.find(columns, full_begin + local - last_run) : last.find(columns, last_begin + local);
    w.there = u.group >= 0;
    if (!w.there) return;
    int tile_m, tile_n;
    if (whole) {
      const int group = __builtin_amdgcn_readfirstlane(static_cast<int>(u.index / (kTileGroup * columns)));
      const int in_group = static_cast<int>(u.index - static_cast<int64_t>(group) * (kTileGroup * columns));
      const int group_rows = min(kTileGroup, u.tiles - group * kTileGroup);
      tile_n = __builtin_amdgcn_readfirstlane(in_group / group_rows);
      tile_m = group * kTileGroup + in_group - tile_n * group_rows;
    } else {
      tile_n = static_cast<int>(u.index);
      tile_m = u.rows / BM;
    }
    w.begin = u.begin + tile_m * BM;
    w.rows = min(BM, u.rows - tile_m * BM);
    w.n_base = tile_n * WIDTH;
    static_for<A_PER_WAVE>([&](auto c) {
      const int in_tile = min((wave * A_PER_WAVE + static_cast<int>(c)) * 16 + q_row, w.rows - 1);
      const uint32_t row = UP ? slot_of(A, w.begin + in_tile) / A.top_k : in_tile;
      src.row[c] = row * static_cast<uint32_t>(A.pitch) + q_piece * 16;  // up: all codes are below 4 GiB, which the host checks
    });
    src.a = UP ? A.codes : A.codes + static_cast<int64_t>(w.begin) * A.pitch;
    const int8_t* const weights = A.packed + static_cast<int64_t>(u.group) * EACH * A.panel;
    static_for<B_PER_WAVE>([&](auto c) {
      const int ld = wave * B_PER_WAVE + static_cast<int>(c), strip = min((w.n_base + channel_of(ld >> 1)) >> 5, A.strips - 1);
      src.b[c] = weights + which_of(ld >> 1) * A.panel + (static_cast<int64_t>(strip) * A.chunks + (ld & 1)) * kChunkBytes;
    });
    static_assert(BM == 256 && BN <= 256, "a thread for each row and channel");
    {
      const int place = w.begin + min(static_cast<int>(threadIdx.x), w.rows - 1), slot = slot_of(A, place);
      panel[BN + threadIdx.x] = A.row_scales[UP ? slot / A.top_k : place];
      reinterpret_cast<int*>(panel)[BN + BM + threadIdx.x] = slot;
      const int c = threadIdx.x % BN >> 5, n = min(w.n_base + channel_of(c) + static_cast<int>(threadIdx.x & 31), A.N - 1);
      if (threadIdx.x < BN) panel[threadIdx.x] = A.scales[(static_cast<int64_t>(u.group) * EACH + which_of(c)) * A.N + n];
    }
  };
  const uint32_t lane16 = lane * 16;
  auto issue = [&](auto c, const Source& src, uint32_t step_b, int stage) {
    constexpr int ci = decltype(c)::value;
    const uint32_t to = lds_base + stage * STAGE + wave * (ci < A_PER_WAVE ? A_PER_WAVE : B_PER_WAVE) * kChunkBytes;
    if constexpr (ci < A_PER_WAVE) lds_dma16_at<ci * kChunkBytes>(src.a, src.row[ci], to);
    else lds_dma16_at<B_REGION + (ci - A_PER_WAVE) * kChunkBytes>(src.b[ci - A_PER_WAVE], step_b, to);
  };
  const int fq = lrow & 15, fh = lrow >> 4;
  const uint32_t frag_a[2] = {static_cast<uint32_t>(fh * kChunkBytes + ((4 * fq + ((0 + lgrp) ^ ((fq >> 2) & 3))) << 4)),
                              static_cast<uint32_t>(fh * kChunkBytes + ((4 * fq + ((2 + lgrp) ^ ((fq >> 2) & 3))) << 4))};
  auto read_a = [&](int stage, int kc, int i) {
    return *reinterpret_cast<const v4i*>(lds + stage * STAGE + (2 * i + wm) * (2 * kChunkBytes) + frag_a[kc]);
  };
  auto read_b = [&](int stage, int kc, int j) {
    return *reinterpret_cast<const v4i*>(lds + stage * STAGE + B_REGION + ((wn * TN + j) * 2 + kc) * kChunkBytes + lane * 16);
  };

  const int KT = A.chunks / 2;  // at least AHEAD: the last steps of a tile fetch the first ones of the next
  Work now, next;
  Source src, next_src;   // src: of the step that is loaded next; its second offset:
  uint32_t step_b = lane16;
  find(blockIdx.x >> 3, now, src, panels);
  if (!now.there) return;
  auto make_uniform = [](Source& s) {
    s.a = uniform(s.a);
    static_for<B_PER_WAVE>([&](auto c) { s.b[c] = uniform(s.b[c]); });
  };
  make_uniform(src);
  static_for<AHEAD>([&](auto k) {
    static_for<NLD>([&](auto c) { issue(c, src, step_b, decltype(k)::value); });
    src.a += 64;
    step_b += 2 * kChunkBytes;
  });
  wait_vmcnt<(AHEAD - 2) * NLD>();
  __syncthreads();

  int ring = 0;  // stage of the tile's first step
  int64_t number = blockIdx.x >> 3;
  for (int slot = 0;; slot = slot == 2 ? 0 : slot + 1) {
    // (a third panel: a wavefront may be here while another one still is at the results of the tile before)
    number += gridDim.x >> 3;
    find(number, next, next_src, panels + (slot == 2 ? 0 : slot + 1) * PANEL);
    const bool more = __builtin_amdgcn_readfirstlane(next.there);  // what is fetched behind the last tile is not used
    v16i acc[TN * TM];
    static_for<TN * TM>([&](auto t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][r] = 0;
    });
    // The steps of a tile whose wavefronts use TU of their TM tiles of rows: the last tile of an expert costs by 64 rows
    auto multiply = [&](auto used) {
      constexpr int TU = decltype(used)::value, FA = 2 * TU;
      v4i fa0[FA], fa1[FA], fb[4];
      static_for<FA>([&](auto x) { fa0[x] = read_a(ring, decltype(x)::value / TU, decltype(x)::value % TU); });
      static_for<2>([&](auto d) { fb[d] = read_b(ring, decltype(d)::value / TN, decltype(d)::value % TN); });
      auto step = [&](int kt, const v4i (&at)[FA], v4i (&then)[FA]) {
        const int st_now = (ring + kt) & (NSTAGE - 1), st_next = (ring + kt + 1) & (NSTAGE - 1), st_fill = (ring + kt + AHEAD) & (NSTAGE - 1);
        if (kt + AHEAD == KT) {
          if (more) src = next_src;
          else src.a -= static_cast<int64_t>(KT) * 64;
          make_uniform(src);
          step_b = lane16;
        }
        static_for<NSLICE>([&](auto sl) {
          constexpr int s = decltype(sl)::value, kc = s / TN, j = s % TN;
          static_for<TU>([&](auto i) {
            constexpr int ii = decltype(i)::value, t = j * TM + ii;
            acc[t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[s % 4], at[kc * TU + ii], acc[t], 0, 0, 0);
            if constexpr (ii == 0) {
              constexpr int sn = s + 2;  // weight fragments are read two slices ahead
              if constexpr (sn < NSLICE) fb[sn % 4] = read_b(st_now, sn / TN, sn % TN);
              else fb[sn % 4] = read_b(st_next, (sn - NSLICE) / TN, (sn - NSLICE) % TN);
            }
            if constexpr (ii == TU - 1) {
              static_for<NLD>([&](auto c) {
                if constexpr (decltype(c)::value * NSLICE / NLD == s) issue(c, src, step_b, st_fill);
              });
            }
            if constexpr (s < NSLICE / 2) {  // activation fragments of the next step during the first half
              constexpr int Q = NSLICE / 2 * TU, q = s * TU + ii, shift = Q >= 2 * FA ? 1 : 0;
              static_for<FA>([&](auto x) {
                if constexpr (decltype(x)::value * Q / FA + shift == q) then[decltype(x)::value] = read_a(st_next, decltype(x)::value / TU, decltype(x)::value % TU);
              });
            }
            __builtin_amdgcn_sched_barrier(0);
          });
        });
        src.a += 64;
        step_b += 2 * kChunkBytes;
        wait_vmcnt<(AHEAD - 2) * NLD>();
        __syncthreads();
      };
      int kt = 0;
      if (KT & 1) {
        step(0, fa0, fa1);
        static_for<FA>([&](auto x) { fa0[x] = fa1[x]; });
        kt = 1;
      }
      for (; kt < KT; kt += 2) {
        step(kt, fa0, fa1);
        step(kt + 1, fa1, fa0);
      }
    };
    const int used = __builtin_amdgcn_readfirstlane((now.rows + 63) / 64);
    static_for<TM>([&](auto less) {
      if (used == static_cast<int>(less) + 1) multiply(std::integral_constant<int, decltype(less)::value + 1>{});
    });
    ring = (ring + KT) & (NSTAGE - 1);

    // ---- results.  A lane has groups of 4 channels of one row; they go through a private piece of LDS (32 rows of a few channels and
    // a pad) to rows of contiguous bytes.
    // (lane numbers that the compiler does not know: what follows from them is not kept in registers, of which there are none, throughout the steps)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int erow = el & 31, egrp = el >> 5;
    constexpr int ESZ = UP ? (OUT == ITEXHIP_FLOAT ? 4 : 2) : 4;
    constexpr int PAIR = tile_pair(ESZ, OUT_TN), ROWB = PAIR * 32 * ESZ, PITCH = ROWB + 16;
    uint8_t* const buffer = buffers + wave * (32 * PITCH);
    constexpr int LPR = ROWB / 16, RPP = 64 / LPR;   // lanes a row, rows a store
    const bool whole_rows = ((static_cast<uint32_t>(A.N) * ESZ | static_cast<uint32_t>(reinterpret_cast<uintptr_t>(A.out))) & 15) == 0;
    const float* const scale0 = panels + slot * PANEL + wn * TN * 32 + egrp * 4;
    const float* const row_scale = panels + slot * PANEL + BN;
    const int* const slots = reinterpret_cast<const int*>(row_scale + BM);
    static_for<TM>([&](auto tile) {
      constexpr int i = decltype(tile)::value;
      const int m0 = (2 * i + wm) * 32;
      if (m0 >= now.rows) return;  // the same for the whole wavefront
      const float s = row_scale[m0 + erow];
      static_for<OUT_TN / PAIR>([&](auto pair) {
        static_for<PAIR>([&](auto half) {
          constexpr int j = decltype(pair)::value * PAIR + decltype(half)::value;
          float y[16];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f4 of = *reinterpret_cast<const f4*>(scale0 + j * 32 + g * 8);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[g * 4 + r] = static_cast<float>(acc[j * TM + i][g * 4 + r]) * (s * of[r]);
          }
          if constexpr (UP) activate16(SWISH ? ITEXHIP_ACT_SWISH : A.activation, y);
          if constexpr (GATED) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const f4 of = *reinterpret_cast<const f4*>(scale0 + (OUT_TN + j) * 32 + g * 8);
#pragma unroll
              for (int r = 0; r < 4; ++r) y[g * 4 + r] *= static_cast<float>(acc[(OUT_TN + j) * TM + i][g * 4 + r]) * (s * of[r]);
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint8_t* const to = buffer + erow * PITCH + (decltype(half)::value * 32 + g * 8 + egrp * 4) * ESZ;
            const float* const v = y + g * 4;
            if constexpr (ESZ == 4) *reinterpret_cast<f4*>(to) = f4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<uint2*>(to) = uint2{f32x2_to_bits16<UP ? OUT : ITEXHIP_HALF>(v[0], v[1]), f32x2_to_bits16<UP ? OUT : ITEXHIP_HALF>(v[2], v[3])};
          }
        });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int n0 = now.n_base + (wn * OUT_TN + decltype(pair)::value * PAIR) * 32;
#pragma unroll
        for (int p = 0; p < 32 / RPP; ++p) {
          const int r = p * RPP + el / LPR, n = n0 + el % LPR * (16 / ESZ);
          const v4i v = *reinterpret_cast<const v4i*>(buffer + r * PITCH + el % LPR * 16);
          if (m0 + r >= now.rows || n >= A.N) continue;
          const int64_t row = UP ? now.begin + m0 + r : slots[m0 + r];
          uint8_t* const to = static_cast<uint8_t*>(A.out) + (row * A.N + n) * ESZ;
          if (whole_rows) {
            *reinterpret_cast<v4i*>(to) = v;
          } else {
#pragma unroll
            for (int w = 0; w < 16 / ESZ; ++w) {
              if (n + w >= A.N) continue;
              if constexpr (ESZ == 4) *reinterpret_cast<int*>(to + w * 4) = v[w];
              else *reinterpret_cast<uint16_t*>(to + w * 2) = static_cast<uint16_t>(static_cast<uint32_t>(v[w / 2]) >> (16 * (w % 2)));
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      });
    });
    if (!more) break;
    now = next;
  }
  wait_vmcnt<0>();  // no load may still be writing LDS when another workgroup has it
}

// out[t] = addend[t] + sum of the weighted results of the token's choices, in their order.  4096 tokens of 2 choices of 4096 (201 MB) take 43 us,
// 4.7 TB/s.  The results are fp32: 16 bits would round every part once more.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ experts, const float* __restrict__ weights,
                                                      const void* addend, int64_t addend_stride, void* out, int64_t out_stride, int num_experts, int top_k,
                                                      int N, int64_t first) {
  const int64_t token = first + blockIdx.x;
  constexpr int W = VEC ? 4 : 1;
  for (int n = threadIdx.x * W; n < N; n += 256 * W) {
    float sum[W];
#pragma unroll
    for (int j = 0; j < W; ++j) sum[j] = 0.0f;
    for (int c = 0; c < top_k; ++c) {
      const int e = experts[token * top_k + c];
      if (e < 0 || e >= num_experts) continue;
      const float w = weights[token * top_k + c];
      const float* from = y + (token * top_k + c) * static_cast<int64_t>(N) + n;
      float v[W];
      if constexpr (VEC) {
        const f4 q = *reinterpret_cast<const f4*>(from);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = q[j];
      } else {
        v[0] = from[0];
      }
#pragma unroll
      for (int j = 0; j < W; ++j) sum[j] = sum[j] + w * v[j];
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (addend != nullptr) sum[j] = sum[j] + load_value<T>(addend, token * addend_stride + n + j);
      store_output<T>(out, token * out_stride + n + j, sum[j]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
int64_t pitch_of(int64_t K) { return (K + 63) / 64 * 64; }

int check(const itexhip_experts_params* p, const char* name) {
  ITEXHIP_REQUIRE(p != nullptr, "%s: null parameters", name);
  ITEXHIP_REQUIRE(is_chosen_type(p->type), "%s: the type is float, bfloat16 or half", name);
  ITEXHIP_REQUIRE(p->experts >= 1 && p->experts <= kMaxGroups, "%s: 1 .. 1024 experts, got %d", name, p->experts);
  ITEXHIP_REQUIRE(p->top_k >= 1 && p->top_k <= 32, "%s: top_k is 1 .. 32", name);
  ITEXHIP_REQUIRE(p->tokens >= 0 && p->tokens < kMaxRows / p->top_k, "%s: tokens * top_k is below 2^30", name);
  ITEXHIP_REQUIRE(p->hidden >= 1 && p->hidden <= kMaxK && p->inner >= 1 && p->inner <= kMaxK, "%s: hidden and inner are 1 .. 65536", name);
  ITEXHIP_REQUIRE(p->activation == ITEXHIP_ACT_NONE || p->activation == ITEXHIP_ACT_RELU || p->activation == ITEXHIP_ACT_GELU_APPROX ||
                      p->activation == ITEXHIP_ACT_GELU_EXACT || p->activation == ITEXHIP_ACT_SWISH,
                  "%s: activation is none, relu, gelu or swish", name);
  for (const int64_t s : {p->x_stride, p->addend_stride, p->out_stride})
    ITEXHIP_REQUIRE(s >= p->hidden && s < (1LL << 31), "%s: a stride is at least hidden and below 2^31", name);
  return ITEXHIP_OK;
}

// The workspace: codes of the rows, their scales, (down) the products by slot
struct Layout {
  int64_t codes, scales, results, total;
};
int64_t padded(int64_t n) { return (n + 255) / 256 * 256; }
Layout layout_of(const itexhip_experts_params& p, bool up) {
  const int64_t rows = up ? p.tokens : p.tokens * p.top_k;
  Layout l;
  l.codes = 0;
  l.scales = padded(rows * pitch_of(up ? p.hidden : p.inner));
  l.results = l.scales + padded(rows * 4);
  l.total = l.results + (up ? 0 : padded(rows * p.hidden * 4));
  return l;
}

ProductSizes sizes_of(const ProductArgs& A, bool up, bool gated) { return ProductSizes{A.slots, A.top_k, A.experts, A.pitch, A.N, up, gated}; }

template <int T>
void launch_quantize(const void* x, int64_t stride, int64_t rows, int64_t K, const ProductArgs& A, hipStream_t st) {
  const bool vec = aligned(x, 16) && (stride * element_size(T)) % 16 == 0;
  const auto kernel = !vec           ? quantize_rows_kernel<T, false, 0>
                      : K <= 1 * 2048 ? quantize_rows_kernel<T, true, 1>
                      : K <= 2 * 2048 ? quantize_rows_kernel<T, true, 2>
                      : K <= 4 * 2048 ? quantize_rows_kernel<T, true, 4>
                      : K <= 7 * 2048 ? quantize_rows_kernel<T, true, 7>
                                      : quantize_rows_kernel<T, true, 0>;
  launch_blocks(rows, [&](int64_t first, unsigned count) {
    kernel<<<count, 256, 0, st>>>(x, stride, static_cast<int>(K), A.pitch, const_cast<int8_t*>(A.codes), const_cast<float*>(A.row_scales), first);
  });
}

template <int OUT, bool GATED, int WAVES, int SOURCE>
int launch_stream(ProductArgs A, hipStream_t st) {
  A.few = A.slots / A.top_k;  // (tokens: an expert has no more rows, unless a token names it twice, which is one more tile)
  const int per_tile = SOURCE != 0 ? A.few : 32, lds = SOURCE != 0 ? A.few * A.pitch : 0;
  static unsigned long long configured;
  const auto kernel = experts_stream_kernel<OUT, GATED, WAVES, SOURCE>;
  if (SOURCE != 0 && !device_bit(&configured, false)) {
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kFewBytes);
    if (err != hipSuccess) return hip_fail(err, "hipFuncSetAttribute(experts_stream_kernel)");
    device_bit(&configured, true);
  }
  launch_blocks(tiles_bound(A.slots, A.experts, per_tile, false) * A.strips, [&](int64_t first, unsigned count) {
    A.first = first;
    kernel<<<count, 64 * WAVES, lds, st>>>(A);
  });
  return ITEXHIP_OK;
}
template <int OUT, bool GATED, bool SWISH, int BM, int BN>
int launch_tiles(ProductArgs A, hipStream_t st) {
  constexpr int WIDTH = GATED ? BN / 2 : BN, LDS = tile_lds(OUT == ITEXHIP_BFLOAT16 || OUT == ITEXHIP_HALF ? 2 : 4, WIDTH / 64, BM, BN);
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static unsigned long long configured;
  const auto kernel = experts_tile_kernel<OUT, GATED, SWISH, BM, BN>;
  if (!device_bit(&configured, false)) {
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (err != hipSuccess) return hip_fail(err, "hipFuncSetAttribute(experts_tile_kernel)");
    device_bit(&configured, true);
  }
  const int64_t tiles = tiles_bound(A.slots, A.experts, BM, false) * ((A.N + WIDTH - 1) / WIDTH);
  const int64_t grid = tiles < kWorkgroups ? (tiles + 7) / 8 * 8 : kWorkgroups;
  kernel<<<static_cast<unsigned>(grid), 256, LDS, st>>>(A);
  return ITEXHIP_OK;
}
template <int OUT, bool GATED>
int launch_products(const ProductArgs& A, hipStream_t st) {
  constexpr bool SWISH = GATED;
  const bool swish = SWISH && A.activation == ITEXHIP_ACT_SWISH;
  switch (product_kernel(sizes_of(A, OUT != 0, GATED))) {
    case kTiles128: return swish ? launch_tiles<OUT, GATED, SWISH, 256, 128>(A, st) : launch_tiles<OUT, GATED, false, 256, 128>(A, st);
    case kTiles256: return swish ? launch_tiles<OUT, GATED, SWISH, 256, 256>(A, st) : launch_tiles<OUT, GATED, false, 256, 256>(A, st);
    case kStrips8: return launch_stream<OUT, GATED, 8, 0>(A, st);
    default: return launch_stream<OUT, GATED, 4, 0>(A, st);
  }
}

ProductArgs product_args(const itexhip_experts_params& p, bool up, const Layout& l, void* workspace, const int32_t* offsets, const int32_t* rows,
                         const int8_t* packed, const float* scales, void* out) {
  const int64_t K = up ? p.hidden : p.inner, N = up ? p.inner : p.hidden;
  ProductArgs A{};
  A.codes = static_cast<int8_t*>(workspace) + l.codes;
  A.row_scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.scales);
  A.packed = packed;
  A.scales = scales;
  A.offsets = offsets;
  A.rows = rows;
  A.out = out;
  A.panel = itexhip_qgemm_packed_bytes(K, N);
  A.experts = p.experts;
  A.slots = static_cast<int>(p.tokens * p.top_k);
  A.top_k = p.top_k;
  A.K = static_cast<int>(K);
  A.pitch = static_cast<int>(pitch_of(K));
  A.chunks = A.pitch / 32;
  A.N = static_cast<int>(N);
  A.strips = static_cast<int>((N + 31) / 32);
  A.activation = p.activation;
  return A;
}

template <int T>
int run_up(const itexhip_experts_params& p, const void* x, const int32_t* offsets, const int32_t* rows, const int8_t* packed, const float* scales,
            void* h, void* workspace, hipStream_t st) {
  const Layout l = layout_of(p, true);
  ProductArgs A = product_args(p, true, l, workspace, offsets, rows, packed, scales, h);
  A.x = x;
  A.x_stride = p.x_stride;
  A.x_vec = aligned(x, 16) && (p.x_stride * element_size(T)) % 16 == 0;
  const ProductSizes sizes = sizes_of(A, true, p.gated != 0);
  if (few_up(sizes)) {
    if (p.gated) return few_strips(sizes) ? launch_stream<T, true, 8, T>(A, st) : launch_stream<T, true, 4, T>(A, st);
    return few_strips(sizes) ? launch_stream<T, false, 8, T>(A, st) : launch_stream<T, false, 4, T>(A, st);
  }
  launch_quantize<T>(x, p.x_stride, p.tokens, p.hidden, A, st);
  return p.gated ? launch_products<T, true>(A, st) : launch_products<T, false>(A, st);
}

template <int T>
int run_down(const itexhip_experts_params& p, const void* h, const int32_t* experts, const int32_t* offsets, const int32_t* rows, const int8_t* packed,
              const float* scales, const float* weights, const void* addend, void* out, void* workspace, hipStream_t st) {
  const Layout l = layout_of(p, false);
  float* const results = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.results);
  ProductArgs A = product_args(p, false, l, workspace, offsets, rows, packed, scales, results);
  A.x = h;
  A.x_stride = p.inner;
  A.x_vec = aligned(h, 16) && (p.inner * element_size(T)) % 16 == 0;
  if (few_down(sizes_of(A, false, false))) {
    static unsigned long long configured;
    const auto kernel = experts_few_down_kernel<T>;
    if (!device_bit(&configured, false)) {
      const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kFewBytes);
      if (err != hipSuccess) return hip_fail(err, "hipFuncSetAttribute(experts_few_down_kernel)");
      device_bit(&configured, true);
    }
    A.out = out;
    const FewArgs F{experts, weights, addend, p.addend_stride, p.out_stride, static_cast<int>(p.tokens)};
    kernel<<<static_cast<unsigned>(A.strips), 64 * kFewWaves, static_cast<size_t>(A.slots) * A.pitch, st>>>(A, F);
    return ITEXHIP_OK;
  }
  launch_quantize<T>(h, p.inner, A.slots, p.inner, A, st);
  if (const int e = launch_products<0, false>(A, st)) return e;
  const auto combine = p.hidden % 4 == 0 ? combine_kernel<T, true> : combine_kernel<T, false>;
  launch_blocks(p.tokens, [&](int64_t first, unsigned count) {
    combine<<<count, 256, 0, st>>>(results, experts, weights, addend, p.addend_stride, out, p.out_stride, p.experts, p.top_k, A.N, first);
  });
  return ITEXHIP_OK;
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int64_t itexhip_experts_workspace(const itexhip_experts_params* p) {
  if (check(p, "itexhip_experts_workspace") != ITEXHIP_OK) return 0;
  const int64_t up = layout_of(*p, true).total, down = layout_of(*p, false).total;
  return (up > down ? up : down) + 256;
}

extern "C" int itexhip_experts_up(const itexhip_experts_params* p, const void* x, const int32_t* offsets, const int32_t* rows, const int8_t* packed,
                                  const float* scales, void* h, void* workspace, void* stream) {
  if (const int e = check(p, "itexhip_experts_up")) return e;
  if (p->tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(x && offsets && rows && packed && scales && h && workspace, "itexhip_experts_up: null buffer");
  ITEXHIP_REQUIRE(aligned(x, element_size(p->type)) && aligned(h, element_size(p->type)) && aligned(offsets, 4) && aligned(rows, 4) && aligned(scales, 4),
                  "itexhip_experts_up: buffers are aligned to their elements");
  ITEXHIP_REQUIRE(aligned(packed, 16) && aligned(workspace, 16), "itexhip_experts_up: packed weights and workspace are aligned to 16 bytes");
  hipStream_t st = as_stream(stream);
  const int status = p->type == ITEXHIP_FLOAT      ? run_up<ITEXHIP_FLOAT>(*p, x, offsets, rows, packed, scales, h, workspace, st)
                     : p->type == ITEXHIP_BFLOAT16 ? run_up<ITEXHIP_BFLOAT16>(*p, x, offsets, rows, packed, scales, h, workspace, st)
                                                   : run_up<ITEXHIP_HALF>(*p, x, offsets, rows, packed, scales, h, workspace, st);
  if (status != ITEXHIP_OK) return status;
  ITEXHIP_CHECK_LAUNCH("itexhip_experts_up");
  return ITEXHIP_OK;
}

extern "C" int itexhip_experts_down(const itexhip_experts_params* p, const void* h, const int32_t* experts, const int32_t* offsets, const int32_t* rows,
                                    const int8_t* packed, const float* scales, const float* weights, const void* addend, void* out, void* workspace,
                                    void* stream) {
  if (const int e = check(p, "itexhip_experts_down")) return e;
  if (p->tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(h && experts && offsets && rows && packed && scales && weights && out && workspace, "itexhip_experts_down: null buffer");
  const size_t size = static_cast<size_t>(element_size(p->type));
  ITEXHIP_REQUIRE(aligned(h, size) && aligned(addend, size) && aligned(out, size) && aligned(experts, 4) && aligned(offsets, 4) && aligned(rows, 4) &&
                      aligned(scales, 4) && aligned(weights, 4),
                  "itexhip_experts_down: buffers are aligned to their elements");
  ITEXHIP_REQUIRE(aligned(packed, 16) && aligned(workspace, 16), "itexhip_experts_down: packed weights and workspace are aligned to 16 bytes");
  ITEXHIP_REQUIRE(addend != out || p->addend_stride == p->out_stride, "itexhip_experts_down: in place, addend_stride and out_stride are the same");
  hipStream_t st = as_stream(stream);
  const int status = p->type == ITEXHIP_FLOAT      ? run_down<ITEXHIP_FLOAT>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st)
                     : p->type == ITEXHIP_BFLOAT16 ? run_down<ITEXHIP_BFLOAT16>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st)
                                                   : run_down<ITEXHIP_HALF>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st);
  if (status != ITEXHIP_OK) return status;
  ITEXHIP_CHECK_LAUNCH("itexhip_experts_down");
  return ITEXHIP_OK;
}
