// Rows of heads: norm and rotation of queries and keys, appending to the 4-bit cache, reading its rows back.
#include <math.h>

#include "common.hpp"
#include "kv4.hpp"

namespace itexhip {
namespace {

struct HeadsArgs {
  itexhip_heads_params p;
  const void *q, *k, *v;
  const float *q_weight, *k_weight;
  const int32_t* positions;
  const double* freqs;
  const int64_t* slots;
  void *q_out, *k_out;
  uint8_t* cache;
  int64_t tokens, num_slots, page_bytes;
  int page_shift, page_size, dp;
  int passes_q, passes_k, passes, parts;  // passes: groups of 64 / LPH heads of one tensor; a wavefront takes every parts-th
};

template <int T>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
  if constexpr (T == ITEXHIP_FLOAT) return static_cast<const float*>(base)[i];
  else if constexpr (T == ITEXHIP_BFLOAT16) return bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
}
template <int T>
__device__ __forceinline__ void load4(const void* base, int64_t i, float (&x)[4]) {
  if constexpr (T == ITEXHIP_FLOAT) {
    const f4 v = *reinterpret_cast<const f4*>(static_cast<const float*>(base) + i);
    for (int j = 0; j < 4; ++j) x[j] = v[j];
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[2] = {v.x, v.y};
    for (int j = 0; j < 4; ++j) {
      const uint32_t h = (w[j / 2] >> (16 * (j % 2))) & 0xffffu;
      x[j] = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
  }
}
template <int T>
__device__ __forceinline__ void store4(void* base, int64_t i, const float (&x)[4]) {
  if constexpr (T == ITEXHIP_FLOAT) {
    *reinterpret_cast<f4*>(static_cast<float*>(base) + i) = f4{x[0], x[1], x[2], x[3]};
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) =
        uint2{f32x2_to_bits16<T>(x[0], x[1]), f32x2_to_bits16<T>(x[2], x[3])};
  }
}

template <int LPH, class V>
__device__ __forceinline__ V head_sum(V x) {
#pragma unroll
  for (int m = 1; m < LPH; m *= 2) x += __shfl_xor(x, m);
  return x;
}
template <int LPH, class V>
__device__ __forceinline__ V head_max(V x) {
#pragma unroll
  for (int m = 1; m < LPH; m *= 2) {
    const V y = __shfl_xor(x, m);
    x = x > y ? x : y;
  }
  return x;
}

// cosine and sine of 2 pi t, |t| <= 1/2, times the factor
__device__ __forceinline__ void turn(float t, double factor, float* c, float* s) {
  sincospif(2.0f * t, s, c);
  const float f = static_cast<float>(factor);
  *c *= f;
  *s *= f;
}
__device__ __forceinline__ void turn(double t, double factor, double* c, double* s) {
  sincospi(2.0 * t, s, c);
  *c *= factor;
  *s *= factor;
}

// A lane's four pairs of a head, the pairs 4 chunk .. 4 chunk + 3 of head_dim / 2: those below rotary_dim / 2 are rotated.
template <class Real>
struct Pairs {
  Real a[4], b[4];
};

// Norm and rotation in fp32 or fp64; lanes without pairs hold zeros and keep them.
template <int LPH, class Real>
__device__ __forceinline__ void norm_rotate(const HeadsArgs& A, Pairs<Real>& x, bool norm, const float (&wa)[4], const float (&wb)[4],
                                            int rotated, const Real (&c)[4], const Real (&s)[4]) {
  if (norm) {
    Real sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += x.a[j] * x.a[j] + x.b[j] * x.b[j];
    sum = head_sum<LPH>(sum);
    const Real r = Real(1) / sqrt(sum / static_cast<Real>(A.p.head_dim) + static_cast<Real>(A.p.eps));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x.a[j] = x.a[j] * r * static_cast<Real>(wa[j]);
      x.b[j] = x.b[j] * r * static_cast<Real>(wb[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j < rotated) {
      const Real a = x.a[j], b = x.b[j];
      x.a[j] = a * c[j] - b * s[j];
      x.b[j] = b * c[j] + a * s[j];
    }
  }
}

__device__ __forceinline__ uint32_t half_of(double x) { return f32_to_f16_bits(static_cast<float>(x)); }
template <class Real> __device__ __forceinline__ Real saturate(Real x) { return x > Real(65504) ? Real(65504) : x < Real(-65504) ? Real(-65504) : x; }

// Parameters and codes of a head whose pairs are spread over LPH lanes.  `error` bounds how far the pairs are off, relative to
// the largest of them.  Returns whether a rounding (of scale, offset or a code) is closer to its border than that.
template <int LPH, class Real>
__device__ __forceinline__ bool quantize_head(Pairs<Real>& x, bool active, Real error, uint32_t* scale_bits, uint32_t* offset_bits,
                                              uint32_t (&code)[8]) {
  bool nan = false;
  Real hi = Real(-65504), lo = Real(65504);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    nan = nan || x.a[j] != x.a[j] || x.b[j] != x.b[j];
    x.a[j] = saturate(x.a[j]);
    x.b[j] = saturate(x.b[j]);
    if (active) {
      hi = x.a[j] > hi ? x.a[j] : hi;
      hi = x.b[j] > hi ? x.b[j] : hi;
      lo = x.a[j] < lo ? x.a[j] : lo;
      lo = x.b[j] < lo ? x.b[j] : lo;
    }
  }
  hi = head_max<LPH>(hi);
  lo = -head_max<LPH>(-lo);
  const int lane = __lane_id();
  nan = ((__ballot(nan && active) >> (lane & ~(LPH - 1))) & (LPH == 64 ? ~0ull : (1ull << (LPH & 63)) - 1)) != 0;
  const double largest = hi > -lo ? hi : -lo, e = static_cast<double>(error) * largest;
  const double step = (static_cast<double>(hi) - static_cast<double>(lo)) / 15.0;
  const uint32_t sb = half_of(step);
  const double scale = f16_bits_to_f32(sb);
  const double middle = static_cast<double>(lo) + 8.0 * scale;
  const uint32_t ob = half_of(middle);
  const Real offset = f16_bits_to_f32(ob), sc = f16_bits_to_f32(sb);
  bool close = error > 0 && (half_of(step - e) != half_of(step + e) || half_of(middle - e) != half_of(middle + e));
  const Real near = static_cast<Real>(0.5) - static_cast<Real>(e / scale + 2e-6);  // never reached in fp64 (error is 0 there)
  auto one = [&](Real v) -> uint32_t {
    if (sc == 0) return 8;
    const Real t = (v - offset) / sc, r = rint(t);
    if (sizeof(Real) == 4) close = close || !(fabs(t - r) < near);
    return static_cast<uint32_t>(static_cast<int>(r < -8 ? Real(-8) : r > 7 ? Real(7) : r) + 8);
  };
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    code[j] = one(x.a[j]);
    code[4 + j] = one(x.b[j]);
  }
  if (nan) {
    *scale_bits = *offset_bits = 0x7e00;
#pragma unroll
    for (int j = 0; j < 8; ++j) code[j] = 8;
    return false;
  }
  *scale_bits = sb;
  *offset_bits = ob;
  return close && active;
}

// One wavefront takes one token: its cosines and sines once, then groups of 64 / LPH heads, LPH lanes a head, four pairs a
// lane.  In the half layout the two ends of a rotated pair lie rotary_dim / 2 apart, so a lane's eight dimensions are two
// runs of four, otherwise one of eight.
//
// The codes of the cache are those of the 64-bit formulas: a key computed again by another call (a shared prefix, a resumed
// sequence) has the same codes.  The fp32 pass knows how far it may be off and tells when a rounding is closer to its border
// than that, for about one head in a hundred; those are done again in fp64.
template <int T, int LPH, bool VEC, bool APPEND>
__global__ __launch_bounds__(256) void heads_kernel(const HeadsArgs A) {
  __shared__ __align__(8) uint8_t lds_codes[APPEND ? 4 * 64 * 8 : 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int64_t token = unit / A.parts;
  if (token >= A.tokens) return;
  const int part = static_cast<int>(unit - token * A.parts);
  const int sub = lane & (LPH - 1), group = lane / LPH;
  const int D = A.p.head_dim, half_rot = A.p.rotary_dim / 2, pair0 = 4 * sub;
  const bool active = pair0 < D / 2;
  const int rotated = active ? (half_rot - pair0 < 0 ? 0 : half_rot - pair0 > 4 ? 4 : half_rot - pair0) : 0;
  const bool split = !A.p.interleaved && pair0 < half_rot;  // VEC: the whole chunk is rotated or none of it
  const int run0 = split ? pair0 : 2 * pair0, run1 = split ? pair0 + half_rot : 2 * pair0 + 4;
  auto dim_a = [&](int j) { return !A.p.interleaved && pair0 + j < half_rot ? pair0 + j : 2 * (pair0 + j); };
  auto dim_b = [&](int j) { return !A.p.interleaved && pair0 + j < half_rot ? pair0 + j + half_rot : 2 * (pair0 + j) + 1; };

  auto load = [&](const void* src, int64_t at, Pairs<float>& x) {
    if constexpr (VEC) {
      float u[4] = {}, w[4] = {};
      if (active) {
        load4<T>(src, at + run0, u);
        load4<T>(src, at + run1, w);
      }
      x.a[0] = u[0]; x.a[1] = split ? u[1] : u[2]; x.a[2] = split ? u[2] : w[0]; x.a[3] = split ? u[3] : w[2];
      x.b[0] = split ? w[0] : u[1]; x.b[1] = split ? w[1] : u[3]; x.b[2] = split ? w[2] : w[1]; x.b[3] = w[3];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = pair0 + j < D / 2;
        x.a[j] = in ? load1<T>(src, at + dim_a(j)) : 0.0f;
        x.b[j] = in ? load1<T>(src, at + dim_b(j)) : 0.0f;
      }
    }
  };
  auto store = [&](void* dst, int64_t at, const Pairs<float>& x) {
    if constexpr (VEC) {
      if (!active) return;
      const float u[4] = {x.a[0], split ? x.a[1] : x.b[0], split ? x.a[2] : x.a[1], split ? x.a[3] : x.b[1]};
      const float w[4] = {split ? x.b[0] : x.a[2], split ? x.b[1] : x.b[2], split ? x.b[2] : x.a[3], x.b[3]};
      store4<T>(dst, at + run0, u);
      store4<T>(dst, at + run1, w);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (pair0 + j >= D / 2) continue;
        store_output<T>(dst, at + dim_a(j), x.a[j]);
        store_output<T>(dst, at + dim_b(j), x.b[j]);
      }
    }
  };

  double phase[4] = {};
  float c[4] = {}, s[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j < rotated) {
      const double t = static_cast<double>(A.positions[token]) * A.freqs[pair0 + j];
      phase[j] = t - rint(t);
      turn(static_cast<float>(phase[j]), A.p.attention_factor, &c[j], &s[j]);
    }
  }
  int64_t slot = -1, page_at = 0;
  if constexpr (APPEND) {
    slot = A.slots[token];
    if (slot >= 0 && slot < A.num_slots) page_at = (slot >> A.page_shift) * A.page_bytes;
    else slot = -1;
  }
  float wa[4] = {1, 1, 1, 1}, wb[4] = {1, 1, 1, 1};
  int loaded = -1;
  for (int pass = part; pass < A.passes; pass += A.parts) {
    const int role = pass < A.passes_q ? 0 : pass < A.passes_q + A.passes_k ? 1 : 2;
    if (APPEND && role > 0 && slot < 0) break;
    const int first = role == 0 ? 0 : role == 1 ? A.passes_q : A.passes_q + A.passes_k;
    const int head = (pass - first) * (64 / LPH) + group, heads = role == 0 ? A.p.q_heads : A.p.kv_heads;
    const void* src = role == 0 ? A.q : role == 1 ? A.k : A.v;
    const int64_t* st = role == 0 ? A.p.q_strides : role == 1 ? A.p.k_strides : A.p.v_strides;
    const float* weight = role == 0 ? A.q_weight : role == 1 ? A.k_weight : nullptr;
    const bool there = head < heads;  // lanes beyond the last head run along on its values and store nothing
    const int64_t at = token * st[0] + (there ? head : heads - 1) * st[1];
    Pairs<float> x;
    load(src, at, x);
    if (weight != nullptr && loaded != role) {
      loaded = role;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (pair0 + j < D / 2) {
          wa[j] = weight[dim_a(j)];
          wb[j] = weight[dim_b(j)];
        }
      }
    }
    if (role == 0 || !APPEND) {
      norm_rotate<LPH, float>(A, x, weight != nullptr, wa, wb, rotated, c, s);
      const int64_t* so = role == 0 ? A.p.q_out_strides : A.p.k_out_strides;
      if (there) store(role == 0 ? A.q_out : A.k_out, token * so[0] + head * so[1], x);
      continue;
    }
    if constexpr (APPEND) {
      const Pairs<float> raw = x;
      uint32_t code[8], scale_bits, offset_bits;
      bool close;
      if (role == 1) {
        norm_rotate<LPH, float>(A, x, weight != nullptr, wa, wb, rotated, c, s);
        close = quantize_head<LPH, float>(x, active, 2e-6f, &scale_bits, &offset_bits, code);
      } else {
        close = quantize_head<LPH, float>(x, active, 0.0f, &scale_bits, &offset_bits, code);
      }
      if (__any(close)) {
        Pairs<double> y;
        double cd[4] = {}, sd[4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y.a[j] = raw.a[j];
          y.b[j] = raw.b[j];
          if (role == 1 && j < rotated) turn(phase[j], A.p.attention_factor, &cd[j], &sd[j]);
        }
        if (role == 1) norm_rotate<LPH, double>(A, y, weight != nullptr, wa, wb, rotated, cd, sd);
        quantize_head<LPH, double>(y, active, 0.0, &scale_bits, &offset_bits, code);
      }
      // to the order of the dimensions through LDS, eight codes a lane
      uint8_t* mine = lds_codes + wave * 512 + group * (LPH * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!active) continue;


        mine[dim_a(j)] = static_cast<uint8_t>(code[j]);
        mine[dim_b(j)] = static_cast<uint8_t>(code[4 + j]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      uint32_t packed = 0x88888888u;  // the padding of a head: codes that stand for the offset, never used
      if (active) {
        const uint2 w = *reinterpret_cast<const uint2*>(mine + 8 * sub);
        packed = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          packed |= ((w.x >> (8 * j)) & 15u) << (4 * j);
          packed |= ((w.y >> (8 * j)) & 15u) << (16 + 4 * j);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const Kv4Block block{A.page_size, A.dp};
      if (there && 8 * sub < A.dp) {
        uint8_t* to = A.cache + page_at + static_cast<int64_t>(head) * block.bytes();
        const int in_page = static_cast<int>(slot & (A.page_size - 1));
        *reinterpret_cast<uint32_t*>(to + (role == 1 ? block.key_codes(in_page) + 4 * sub : block.value_codes(in_page, sub))) = packed;
        if (sub == 0) {
          uint8_t* par = to + (role == 1 ? block.key_params(in_page) : block.value_params(in_page));
          *reinterpret_cast<uint16_t*>(par) = static_cast<uint16_t>(scale_bits);
          *reinterpret_cast<uint16_t*>(par + 8) = static_cast<uint16_t>(offset_bits);
        }
      }
    }
  }
}

// Rows of the cache as values: one lane takes eight dimensions of a token's key and value
template <int T>
__global__ __launch_bounds__(256) void gather_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots, int64_t units,
                                                     int kv_heads, int head_dim, int dp, int page_size, int page_shift, int64_t num_slots,
                                                     int64_t page_bytes, void* __restrict__ k_out, void* __restrict__ v_out) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (unit >= units) return;
  const int chunks = head_dim / 8;
  const int64_t row = unit / chunks;
  const int dword = static_cast<int>(unit - row * chunks);
  const int64_t token = row / kv_heads;
  const int head = static_cast<int>(row - token * kv_heads);
  const int64_t slot = slots[token];
  const bool in = slot >= 0 && slot < num_slots;
  const Kv4Block block{page_size, dp};
  const uint8_t* from = cache + (in ? (slot >> page_shift) * page_bytes : 0) + static_cast<int64_t>(head) * block.bytes();
  const int place = in ? static_cast<int>(slot & (page_size - 1)) : 0;
  auto one = [&](int codes, int params, void* out) {
    const uint32_t w = in ? *reinterpret_cast<const uint32_t*>(from + codes) : 0;
    const float scale = in ? f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(from + params)) : 0.0f;
    const float offset = in ? f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(from + params + 8)) : 0.0f;
    float x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = fmaf(scale, static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8), offset);
      y[j] = fmaf(scale, static_cast<float>(static_cast<int>((w >> (16 + 4 * j)) & 15u) - 8), offset);
    }
    store4<T>(out, row * head_dim + 8 * dword, x);
    store4<T>(out, row * head_dim + 8 * dword + 4, y);
  };
  if (k_out != nullptr) one(block.key_codes(place) + 4 * dword, block.key_params(place), k_out);
  if (v_out != nullptr) one(block.value_codes(place, dword), block.value_params(place), v_out);
}

constexpr int64_t kMaxStride = 1ll << 40;

int check_heads(const char* who, const itexhip_heads_params* p, int64_t tokens) {
  ITEXHIP_REQUIRE(p != nullptr, "%s: null parameters", who);
  ITEXHIP_REQUIRE(p->type == ITEXHIP_FLOAT || is_float16_type(p->type), "%s: type is float, bfloat16 or half", who);
  ITEXHIP_REQUIRE(p->head_dim >= 2 && p->head_dim <= 256 && p->head_dim % 2 == 0, "%s: head_dim is even, 2 to 256", who);
  ITEXHIP_REQUIRE(p->q_heads >= 0 && p->q_heads <= 65535 && p->kv_heads >= 0 && p->kv_heads <= 65535, "%s: heads are 0 to 65535", who);
  ITEXHIP_REQUIRE(p->rotary_dim >= 0 && p->rotary_dim <= p->head_dim && p->rotary_dim % 2 == 0,
                  "%s: rotary_dim is even, 0 to head_dim", who);
  ITEXHIP_REQUIRE(p->eps >= 0.0 && p->eps < 1e30, "%s: eps is finite and not negative", who);
  ITEXHIP_REQUIRE(isfinite(p->attention_factor), "%s: attention_factor is finite", who);
  ITEXHIP_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "%s: tokens are 0 to 2^31 - 1", who);
  const int64_t* all[5] = {p->q_strides, p->k_strides, p->v_strides, p->q_out_strides, p->k_out_strides};
  for (const int64_t* s : all)
    for (int i = 0; i < 2; ++i)
      ITEXHIP_REQUIRE(s[i] > -kMaxStride && s[i] < kMaxStride, "%s: a stride of %lld elements", who, static_cast<long long>(s[i]));
  return ITEXHIP_OK;
}

template <int T, bool APPEND>
void launch(const HeadsArgs& A, int lph, bool vec, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((A.tokens * A.parts + 3) / 4)), block(256);
  if (!vec) heads_kernel<T, 32, false, APPEND><<<grid, block, 0, stream>>>(A);
  else if (lph == 8) heads_kernel<T, 8, true, APPEND><<<grid, block, 0, stream>>>(A);
  else if (lph == 16) heads_kernel<T, 16, true, APPEND><<<grid, block, 0, stream>>>(A);
  else heads_kernel<T, 32, true, APPEND><<<grid, block, 0, stream>>>(A);
}

template <bool APPEND>
int run(HeadsArgs& A, hipStream_t stream, const char* who) {
  const itexhip_heads_params& p = A.p;
  const size_t esize = p.type == ITEXHIP_FLOAT ? 4 : 2, vector = 4 * esize;
  bool vec = p.head_dim % 8 == 0 && (p.rotary_dim % 8 == 0);
  auto ok = [&](const void* x, const int64_t* s) { vec = vec && (x == nullptr || (aligned(x, vector) && s[0] % 4 == 0 && s[1] % 4 == 0)); };
  ok(A.q, p.q_strides);
  ok(A.k, p.k_strides);
  ok(A.v, p.v_strides);
  ok(A.q_out, p.q_out_strides);
  ok(A.k_out, p.k_out_strides);
  const int lph = !vec ? 32 : p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32, group = 64 / lph;
  A.passes_q = A.q != nullptr ? (p.q_heads + group - 1) / group : 0;
  A.passes_k = A.k != nullptr ? (p.kv_heads + group - 1) / group : 0;
  A.passes = A.passes_q + A.passes_k * (APPEND ? 2 : 1);
  if (A.passes == 0 || A.tokens == 0) return ITEXHIP_OK;
  // few tokens: a token's groups of heads go to several wavefronts, each with its own cosines and sines
  const int64_t waves = 8192;
  A.parts = static_cast<int>(A.tokens >= waves ? 1 : (waves + A.tokens - 1) / A.tokens < A.passes ? (waves + A.tokens - 1) / A.tokens : A.passes);
  if (p.type == ITEXHIP_FLOAT) launch<ITEXHIP_FLOAT, APPEND>(A, lph, vec, stream);
  else if (p.type == ITEXHIP_BFLOAT16) launch<ITEXHIP_BFLOAT16, APPEND>(A, lph, vec, stream);
  else launch<ITEXHIP_HALF, APPEND>(A, lph, vec, stream);
  ITEXHIP_CHECK_LAUNCH(who);
  return ITEXHIP_OK;
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int itexhip_rope_frequencies(int scaling, int rotary_dim, double base, double factor, double original_context, double low,
                                        double high, double* freqs, double* attention_factor) {
  const char* who = "itexhip_rope_frequencies";
  const double two_pi = 6.283185307179586476925286766559;
  ITEXHIP_REQUIRE(scaling >= ITEXHIP_ROPE_NONE && scaling <= ITEXHIP_ROPE_YARN, "%s: unknown scaling %d", who, scaling);
  ITEXHIP_REQUIRE(rotary_dim >= 2 && rotary_dim <= 256 && rotary_dim % 2 == 0, "%s: rotary_dim is even, 2 to 256", who);
  ITEXHIP_REQUIRE(base > 1.0 && isfinite(base), "%s: base is over 1", who);
  ITEXHIP_REQUIRE(scaling == ITEXHIP_ROPE_NONE || (factor >= 1.0 && isfinite(factor)), "%s: factor is at least 1", who);
  ITEXHIP_REQUIRE(scaling != ITEXHIP_ROPE_NTK || rotary_dim > 2, "%s: NTK scaling takes a rotary_dim over 2", who);
  ITEXHIP_REQUIRE(scaling < ITEXHIP_ROPE_LLAMA3 || (original_context > 0.0 && isfinite(original_context) && low > 0.0 && high > low && isfinite(high)),
                  "%s: original_context and 0 < low < high are wanted", who);
  ITEXHIP_REQUIRE(freqs != nullptr && attention_factor != nullptr, "%s: null output", who);
  const int n = rotary_dim / 2;
  const double b = scaling == ITEXHIP_ROPE_NTK ? base * pow(factor, rotary_dim / (rotary_dim - 2.0)) : base;
  // the index at which a pair makes `turns` turns within the original context
  auto index_of = [&](double turns) { return rotary_dim * log(original_context / (turns * two_pi)) / (2.0 * log(base)); };
  double from = 0, to = 0;
  if (scaling == ITEXHIP_ROPE_YARN) {
    from = fmax(floor(index_of(high)), 0.0);
    to = fmin(ceil(index_of(low)), rotary_dim - 1.0);
  }
  for (int i = 0; i < n; ++i) {
    const double f = pow(b, -2.0 * i / rotary_dim) / two_pi;
    double kept = 1.0;  // share of the frequency that is not divided by the factor
    if (scaling == ITEXHIP_ROPE_LINEAR) kept = 0.0;
    if (scaling == ITEXHIP_ROPE_LLAMA3) kept = (original_context * f - low) / (high - low);
    if (scaling == ITEXHIP_ROPE_YARN) kept = 1.0 - (i - from) / fmax(to - from, 0.001);
    kept = fmin(fmax(kept, 0.0), 1.0);
    freqs[i] = scaling == ITEXHIP_ROPE_NONE || scaling == ITEXHIP_ROPE_NTK ? f : f / factor * (1.0 - kept) + f * kept;
  }
  *attention_factor = scaling == ITEXHIP_ROPE_YARN ? 0.1 * log(factor) + 1.0 : 1.0;
  return ITEXHIP_OK;
}

extern "C" int itexhip_qk_norm_rope(const itexhip_heads_params* p, int64_t tokens, const void* q, const void* k, const float* q_weight,
                                    const float* k_weight, const int32_t* positions, const double* freqs, void* q_out, void* k_out,
                                    void* stream) {
  const char* who = "itexhip_qk_norm_rope";
  if (const int st = check_heads(who, p, tokens)) return st;
  if (tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE((q == nullptr) == (q_out == nullptr) && (k == nullptr) == (k_out == nullptr), "%s: an input without its output or the reverse", who);
  ITEXHIP_REQUIRE(p->rotary_dim == 0 || (positions != nullptr && freqs != nullptr), "%s: a rotation takes positions and freqs", who);
  auto same = [](const int64_t* a, const int64_t* b) { return a[0] == b[0] && a[1] == b[1]; };
  ITEXHIP_REQUIRE((q == nullptr || q != q_out || same(p->q_strides, p->q_out_strides)) && (k == nullptr || k != k_out || same(p->k_strides, p->k_out_strides)),
                  "%s: in place the strides are the same", who);
  const size_t esize = p->type == ITEXHIP_FLOAT ? 4 : 2;
  ITEXHIP_REQUIRE(aligned(q, esize) && aligned(k, esize) && aligned(q_out, esize) && aligned(k_out, esize) && aligned(q_weight, 4) &&
                  aligned(k_weight, 4) && aligned(positions, 4) && aligned(freqs, 8), "%s: an array is not aligned to its elements", who);
  HeadsArgs A = {};
  A.p = *p;
  A.q = q; A.k = k; A.q_weight = q_weight; A.k_weight = k_weight; A.positions = positions; A.freqs = freqs;
  A.q_out = q_out; A.k_out = k_out; A.tokens = tokens;
  return run<false>(A, as_stream(stream), who);
}

extern "C" int64_t itexhip_kv4_page_bytes(const itexhip_kv4_cache* c) {
  if (const char* wrong = kv4_invalid(c)) {
    set_error("itexhip_kv4_page_bytes: %s", wrong);
    return 0;
  }
  return static_cast<int64_t>(c->kv_heads) * Kv4Block{c->page_size, kv4_padded(c->head_dim)}.bytes();
}

extern "C" int itexhip_kv4_append(const itexhip_heads_params* p, const itexhip_kv4_cache* c, int64_t tokens, const void* q, const void* k,
                                  const void* v, const float* q_weight, const float* k_weight, const int32_t* positions,
                                  const double* freqs, const int64_t* slots, void* q_out, void* cache, void* stream) {
  const char* who = "itexhip_kv4_append";
  if (const int st = check_heads(who, p, tokens)) return st;
  if (const char* wrong = kv4_invalid(c)) {
    set_error("%s: %s", who, wrong);
    return ITEXHIP_INVALID_ARGUMENT;
  }
  ITEXHIP_REQUIRE(p->head_dim == c->head_dim && p->kv_heads == c->kv_heads, "%s: the rows' heads (%d of %d) are not the cache's (%d of %d)", who,
                  p->kv_heads, p->head_dim, c->kv_heads, c->head_dim);
  if (tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(k != nullptr && v != nullptr && slots != nullptr && cache != nullptr, "%s: null keys, values, slots or cache", who);
  ITEXHIP_REQUIRE((q == nullptr) == (q_out == nullptr), "%s: an input without its output or the reverse", who);
  ITEXHIP_REQUIRE(p->rotary_dim == 0 || (positions != nullptr && freqs != nullptr), "%s: a rotation takes positions and freqs", who);
  ITEXHIP_REQUIRE(q == nullptr || q != q_out || (p->q_strides[0] == p->q_out_strides[0] && p->q_strides[1] == p->q_out_strides[1]),
                  "%s: in place the strides are the same", who);
  const size_t esize = p->type == ITEXHIP_FLOAT ? 4 : 2;
  ITEXHIP_REQUIRE(aligned(q, esize) && aligned(k, esize) && aligned(v, esize) && aligned(q_out, esize) && aligned(q_weight, 4) &&
                  aligned(k_weight, 4) && aligned(positions, 4) && aligned(freqs, 8) && aligned(slots, 8) && aligned(cache, 16),
                  "%s: an array is not aligned to its elements (the cache to 16 bytes)", who);
  HeadsArgs A = {};
  A.p = *p;
  A.q = q; A.k = k; A.v = v; A.q_weight = q_weight; A.k_weight = k_weight; A.positions = positions; A.freqs = freqs; A.slots = slots;
  A.q_out = q_out; A.cache = static_cast<uint8_t*>(cache); A.tokens = tokens;
  A.page_size = c->page_size;
  A.page_shift = log2_of(c->page_size);
  A.num_slots = c->num_pages * c->page_size;
  A.dp = kv4_padded(c->head_dim);
  A.page_bytes = itexhip_kv4_page_bytes(c);
  return run<true>(A, as_stream(stream), who);
}

extern "C" int itexhip_kv4_gather(const itexhip_kv4_cache* c, int type, int64_t tokens, const void* cache, const int64_t* slots, void* k_out,
                                  void* v_out, void* stream) {
  const char* who = "itexhip_kv4_gather";
  if (const char* wrong = kv4_invalid(c)) {
    set_error("%s: %s", who, wrong);
    return ITEXHIP_INVALID_ARGUMENT;
  }
  ITEXHIP_REQUIRE(type == ITEXHIP_FLOAT || is_float16_type(type), "%s: type is float, bfloat16 or half", who);
  ITEXHIP_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "%s: tokens are 0 to 2^31 - 1", who);
  if (tokens == 0 || (k_out == nullptr && v_out == nullptr)) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(cache != nullptr && slots != nullptr, "%s: null cache or slots", who);
  ITEXHIP_REQUIRE(aligned(cache, 16) && aligned(slots, 8) && aligned(k_out, 16) && aligned(v_out, 16),
                  "%s: cache and outputs are 16-byte aligned, slots to their elements", who);
  const int64_t units = tokens * c->kv_heads * (c->head_dim / 8);
  ITEXHIP_REQUIRE(units < (1ll << 31) * 128, "%s: too many values for one call", who);
  const int dp = kv4_padded(c->head_dim);
  const dim3 grid(static_cast<unsigned>((units + 255) / 256)), block(256);
  auto go = [&](auto kernel) {
    kernel<<<grid, block, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(cache), slots, units, c->kv_heads, c->head_dim, dp, c->page_size,
                                                  log2_of(c->page_size), c->num_pages * c->page_size, itexhip_kv4_page_bytes(c), k_out, v_out);
  };
  if (type == ITEXHIP_FLOAT) go(gather_kernel<ITEXHIP_FLOAT>);
  else if (type == ITEXHIP_BFLOAT16) go(gather_kernel<ITEXHIP_BFLOAT16>);
  else go(gather_kernel<ITEXHIP_HALF>);
  ITEXHIP_CHECK_LAUNCH(who);
  return ITEXHIP_OK;
}
