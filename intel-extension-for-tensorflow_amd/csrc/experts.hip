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
// of a row's largest absolute value, as its bits (those of NaN are above infinity's)
__device__ __forceinline__ float scale_of(uint32_t absmax_bits) {
  if (absmax_bits >= 0x7f800000u) return __builtin_nanf("");
  return fmaxf(__uint_as_float(absmax_bits) / 127.0f, kLeastScale);
}

template <int T, bool VEC>
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
  for (int k = threadIdx.x * 8; k < K; k += 2048) {
    float v[8];
    load(k, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(most[0], most[1]), max(most[2], most[3]));
  const float s = scale_of(top), inv = 1.0f / s;
  const bool finite = s == s;
  if (threadIdx.x == 0) scales[row] = s;
  for (int k = threadIdx.x * 8; k < pitch; k += 2048) {
    float v[8];
    load(k, v);
    int c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = finite ? code_of(v[j], s, inv) : 0;
    *reinterpret_cast<uint2*>(codes + row * pitch + k) = uint2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
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
  int64_t panel;
  int experts, slots, top_k; // slots = tokens * top_k
  int pitch, chunks, N;      // chunks of 32 k, an even number
  int strips;                // of 32 channels
  int64_t first;             // workgroup of the launch
  int activation;
};

__device__ __forceinline__ float activate(int activation, float x) {
  switch (activation) {
    case ITEXHIP_ACT_RELU: return fmaxf(x, 0.0f);
    case ITEXHIP_ACT_GELU_APPROX: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_GELU_TANH, 0.0f, 0.0f}, x);
    case ITEXHIP_ACT_GELU_EXACT: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_GELU_ERF, 0.0f, 0.0f}, x);
    case ITEXHIP_ACT_SWISH: return apply_eltwise(itexhip_eltwise{ITEXHIP_ELT_SWISH, 1.0f, 0.0f}, x);
    default: return x;
  }
}

// Where a place's codes are, and (down) where its result goes.  What `rows` holds is cut to the slots there are.
__device__ __forceinline__ int slot_of(const ProductArgs& A, int place) { return min(max(A.rows[place], 0), A.slots - 1); }

// Few rows an expert: each wavefront streams a share of the K chunks of a strip of 32 channels past up to 32 RT rows, whose
// codes come from the caches; the shares' sums meet in LDS.  OUT: type of h (up), or 0: fp32 by slot (down).
template <int OUT, bool GATED, int RT>
__global__ __launch_bounds__(256) void experts_stream_kernel(const ProductArgs A) {
  constexpr int WAVES = 4, EACH = GATED ? 2 : 1, PITCH = 36;
  constexpr bool UP = OUT != 0;
  __shared__ __align__(16) int sums[EACH][WAVES][32 * PITCH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = A.first + blockIdx.x;
  const int index = static_cast<int>(id / A.strips), strip = static_cast<int>(id - static_cast<int64_t>(index) * A.strips);
  const RowTile t = find_tile<false>(A.offsets, A.experts, A.slots, 32 * RT, index);
  if (t.group < 0) return;
  const int8_t* source[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int place = t.begin + min(i * 32 + (lane & 31), t.rows - 1);
    const int row = UP ? slot_of(A, place) / A.top_k : place;
    source[i] = A.codes + static_cast<int64_t>(row) * A.pitch + (lane >> 5) * 16;
  }
  const int8_t* weights = A.packed + static_cast<int64_t>(t.group) * EACH * A.panel + static_cast<int64_t>(strip) * A.chunks * kChunkBytes + lane * 16;
  v16i acc[EACH][RT];
#pragma unroll
  for (int w = 0; w < EACH; ++w)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[w][i][r] = 0;
  auto load = [&](int c, v4i (&b)[EACH], v4i (&a)[RT]) {
#pragma unroll
    for (int w = 0; w < EACH; ++w) b[w] = *reinterpret_cast<const v4i*>(weights + w * A.panel + static_cast<int64_t>(c) * kChunkBytes);
#pragma unroll
    for (int i = 0; i < RT; ++i) a[i] = *reinterpret_cast<const v4i*>(source[i] + c * 32);
  };
  auto multiply = [&](const v4i (&b)[EACH], const v4i (&a)[RT]) {
#pragma unroll
    for (int w = 0; w < EACH; ++w)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[w][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[w], a[i], acc[w][i], 0, 0, 0);
  };
  constexpr int AT_ONCE = 4;
  int c = wave;
  for (; c + (AT_ONCE - 1) * WAVES < A.chunks; c += AT_ONCE * WAVES) {
    v4i b[AT_ONCE][EACH], a[AT_ONCE][RT];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) load(c + u * WAVES, b[u], a[u]);
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) multiply(b[u], a[u]);
  }
  for (; c < A.chunks; c += WAVES) {
    v4i b[EACH], a[RT];
    load(c, b, a);
    multiply(b, a);
  }
  // row tile by row tile: the shares' sums, then four channels of a row a thread
  const int m = threadIdx.x >> 3, n0 = strip * 32 + (threadIdx.x & 7) * 4;
  static_for<RT>([&](auto tile) {
    constexpr int i = decltype(tile)::value;
    if (i * 32 >= t.rows) return;  // the same for all
    if (i > 0) __syncthreads();
#pragma unroll
    for (int w = 0; w < EACH; ++w)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<v4i*>(&sums[w][wave][(lane & 31) * PITCH + g * 8 + (lane >> 5) * 4]) =
            v4i{acc[w][i][4 * g], acc[w][i][4 * g + 1], acc[w][i][4 * g + 2], acc[w][i][4 * g + 3]};
    __syncthreads();
    if (i * 32 + m >= t.rows) return;
    const int place = t.begin + i * 32 + m;
    const int slot = slot_of(A, place), row = UP ? slot / A.top_k : place;
    const float s = A.row_scales[row];
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
  });
}

// out[t] = addend[t] + sum of the weighted results of the token's choices, in their order
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

template <int T>
void launch_quantize(const void* x, int64_t stride, int64_t rows, int64_t K, int8_t* codes, float* scales, hipStream_t st) {
  const bool vec = aligned(x, 16) && (stride * element_size(T)) % 16 == 0;
  const auto kernel = vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
  launch_blocks(rows, [&](int64_t first, unsigned count) {
    kernel<<<count, 256, 0, st>>>(x, stride, static_cast<int>(K), static_cast<int>(pitch_of(K)), codes, scales, first);
  });
}

template <int OUT, bool GATED, int RT>
void launch_stream(ProductArgs A, hipStream_t st) {
  launch_blocks(tiles_bound(A.slots, A.experts, 32 * RT, false) * A.strips, [&](int64_t first, unsigned count) {
    A.first = first;
    experts_stream_kernel<OUT, GATED, RT><<<count, 256, 0, st>>>(A);
  });
}
template <int OUT, bool GATED>
void launch_products(const ProductArgs& A, hipStream_t st) {
  if (A.slots > 64 * A.experts) launch_stream<OUT, GATED, 4>(A, st);
  else launch_stream<OUT, GATED, 1>(A, st);
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
  A.pitch = static_cast<int>(pitch_of(K));
  A.chunks = A.pitch / 32;
  A.N = static_cast<int>(N);
  A.strips = static_cast<int>((N + 31) / 32);
  A.activation = p.activation;
  return A;
}

template <int T>
void run_up(const itexhip_experts_params& p, const void* x, const int32_t* offsets, const int32_t* rows, const int8_t* packed, const float* scales,
            void* h, void* workspace, hipStream_t st) {
  const Layout l = layout_of(p, true);
  const ProductArgs A = product_args(p, true, l, workspace, offsets, rows, packed, scales, h);
  launch_quantize<T>(x, p.x_stride, p.tokens, p.hidden, const_cast<int8_t*>(A.codes), const_cast<float*>(A.row_scales), st);
  if (p.gated) launch_products<T, true>(A, st);
  else launch_products<T, false>(A, st);
}

template <int T>
void run_down(const itexhip_experts_params& p, const void* h, const int32_t* experts, const int32_t* offsets, const int32_t* rows, const int8_t* packed,
              const float* scales, const float* weights, const void* addend, void* out, void* workspace, hipStream_t st) {
  const Layout l = layout_of(p, false);
  float* const results = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.results);
  const ProductArgs A = product_args(p, false, l, workspace, offsets, rows, packed, scales, results);
  launch_quantize<T>(h, p.inner, A.slots, p.inner, const_cast<int8_t*>(A.codes), const_cast<float*>(A.row_scales), st);
  launch_products<0, false>(A, st);
  const auto combine = p.hidden % 4 == 0 ? combine_kernel<T, true> : combine_kernel<T, false>;
  launch_blocks(p.tokens, [&](int64_t first, unsigned count) {
    combine<<<count, 256, 0, st>>>(results, experts, weights, addend, p.addend_stride, out, p.out_stride, p.experts, p.top_k, A.N, first);
  });
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
  if (p->type == ITEXHIP_FLOAT) run_up<ITEXHIP_FLOAT>(*p, x, offsets, rows, packed, scales, h, workspace, st);
  else if (p->type == ITEXHIP_BFLOAT16) run_up<ITEXHIP_BFLOAT16>(*p, x, offsets, rows, packed, scales, h, workspace, st);
  else run_up<ITEXHIP_HALF>(*p, x, offsets, rows, packed, scales, h, workspace, st);
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
  hipStream_t st = as_stream(stream);
  if (p->type == ITEXHIP_FLOAT) run_down<ITEXHIP_FLOAT>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st);
  else if (p->type == ITEXHIP_BFLOAT16) run_down<ITEXHIP_BFLOAT16>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st);
  else run_down<ITEXHIP_HALF>(*p, h, experts, offsets, rows, packed, scales, weights, addend, out, workspace, st);
  ITEXHIP_CHECK_LAUNCH("itexhip_experts_down");
  return ITEXHIP_OK;
}
