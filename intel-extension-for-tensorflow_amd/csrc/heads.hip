// Rows of heads: norm and rotation of queries and keys, appending to the 4-bit cache, reading its rows back.
#include <math.h>

#include <type_traits>

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
  int passes_k, passes_v, passes;  // groups of 64 / LPH heads of a token's keys, values, all with the queries
  int64_t share;                   // passes a wavefront
};

template <int T>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
  if constexpr (T == ITEXHIP_FLOAT) return static_cast<const float*>(base)[i];
  else if constexpr (T == ITEXHIP_BFLOAT16) return bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
}
template <int T>
__device__ __forceinline__ void store8(void* base, int64_t i, const float (&x)[8]) {
  if constexpr (T == ITEXHIP_FLOAT) {
    f4* to = reinterpret_cast<f4*>(static_cast<float*>(base) + i);
    to[0] = f4{x[0], x[1], x[2], x[3]};
    to[1] = f4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) =
        uint4{f32x2_to_bits16<T>(x[0], x[1]), f32x2_to_bits16<T>(x[2], x[3]), f32x2_to_bits16<T>(x[4], x[5]), f32x2_to_bits16<T>(x[6], x[7])};
  }
}

// Over the LPH lanes of a head.  Lanes 1, 2, 4 and 8 apart meet within the vector unit; of a mirrored row any lane of the
// other half will do, since its half agrees by then.
template <int CTRL, class V>
__device__ __forceinline__ V from_lane(V x) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one or two registers");
  int w[sizeof(V) / 4];
  __builtin_memcpy(w, &x, sizeof(V));
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) w[i] = __builtin_amdgcn_update_dpp(w[i], w[i], CTRL, 0xf, 0xf, false);
  __builtin_memcpy(&x, w, sizeof(V));
  return x;
}
template <int LPH, class V, class F>
__device__ __forceinline__ V over_head(V x, F&& f) {
  if constexpr (LPH > 1) x = f(x, from_lane<0xb1>(x));    // quad_perm 1 0 3 2
  if constexpr (LPH > 2) x = f(x, from_lane<0x4e>(x));    // quad_perm 2 3 0 1
  if constexpr (LPH > 4) x = f(x, from_lane<0x141>(x));   // row_half_mirror
  if constexpr (LPH > 8) x = f(x, from_lane<0x140>(x));   // row_mirror
  if constexpr (LPH > 16) x = f(x, __shfl_xor(x, 16));
  return x;
}

// cosine and sine of 2 pi t for |t| <= 1/2, to about 1e-15: sine and cosine of the angle to the nearest quarter turn, |y| <= pi / 4,
// by their Taylor sums (the first terms left out are y^17 / 17! < 5e-17 and y^16 / 16! < 2e-15), put back by the quarter
__device__ __forceinline__ void turn(double t, double factor, double* c, double* s) {
  const double quarter = rint(4.0 * t);
  const double y = fma(quarter, -0.25, t) * 6.283185307179586, z = y * y;
  double a = fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0);
  a = fma(z, a, -1.0 / 39916800.0);
  a = fma(z, a, 1.0 / 362880.0);
  a = fma(z, a, -1.0 / 5040.0);
  a = fma(z, a, 1.0 / 120.0);
  a = fma(z, a, -1.0 / 6.0);
  a = fma(z * y, a, y);
  double b = fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0);
  b = fma(z, b, -1.0 / 3628800.0);
  b = fma(z, b, 1.0 / 40320.0);
  b = fma(z, b, -1.0 / 720.0);
  b = fma(z, b, 1.0 / 24.0);
  b = fma(z, b, -0.5);
  b = fma(z, b, 1.0);
  const int n = static_cast<int>(quarter);
  const double cs = (n & 1) ? a : b, sn = (n & 1) ? b : a;
  *c = ((n + 1) & 2) ? -cs * factor : cs * factor;
  *s = (n & 2) ? -sn * factor : sn * factor;
}

__device__ __forceinline__ uint32_t half_of(double x) { return f32_to_f16_bits(static_cast<float>(x)); }

// Two runs of NPL dimensions of a head, held by one lane
template <class Real, int NPL>
struct Runs {
  Real x[2][NPL];
};

template <int LPH, int NPL, class Real>
__device__ __forceinline__ void norm(const HeadsArgs& A, Runs<Real, NPL>& v, const float (&weight)[2][NPL]) {
  Real sum = 0;
#pragma unroll
  for (int j = 0; j < 2 * NPL; ++j) sum = fma(v.x[j / NPL][j % NPL], v.x[j / NPL][j % NPL], sum);
  sum = over_head<LPH>(sum, [](Real a, Real b) { return a + b; });
  const Real r = Real(1) / sqrt(sum / static_cast<Real>(A.p.head_dim) + static_cast<Real>(A.p.eps));
#pragma unroll
  for (int j = 0; j < 2 * NPL; ++j) v.x[j / NPL][j % NPL] = v.x[j / NPL][j % NPL] * r * static_cast<Real>(weight[j / NPL][j % NPL]);
}

// The lane's pairs, each turned by what turn_of(pair) gives: the first `rotated` of them, with WHOLE all or none.  `across`: a pair's
// ends are in the two runs, otherwise neighbours in one
template <bool WHOLE, int NPL, class Real, class F>
__device__ __forceinline__ void rotate(Runs<Real, NPL>& v, bool across, int rotated, F&& turn_of) {
  auto pair = [&](int j, Real& a, Real& b) {
    Real c, s;
    turn_of(j, &c, &s);
    const Real u = a, w = b;
    a = fma(u, c, -(w * s));
    b = fma(w, c, u * s);
  };
  if (rotated == 0) return;
  if (across) {
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (WHOLE || j < rotated) pair(j, v.x[0][j], v.x[1][j]);
    asm volatile("; ends of pairs in two runs");  // (two branches that end alike would be merged, with the runs in memory)
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) pair(j, v.x[2 * j / NPL][2 * j % NPL], v.x[2 * j / NPL][2 * j % NPL + 1]);
  }
}

// Parameters and codes of a head whose dimensions are spread over LPH lanes (`mine`: this lane has some).  Real: double for keys; values
// are float until the quotient.
template <int LPH, int NPL, class Real>
__device__ __forceinline__ void quantize_head(Runs<Real, NPL>& v, bool mine, uint32_t* scale_bits, uint32_t* offset_bits, uint32_t (&code)[2][NPL]) {
  bool nan = false;
  Real most = Real(-65504), least = Real(65504);
#pragma unroll
  for (int j = 0; j < 2 * NPL; ++j) {
    Real& x = v.x[j / NPL][j % NPL];
    nan = nan || x != x;
    x = fmin(fmax(x, Real(-65504)), Real(65504));
    most = fmax(most, x);
    least = fmin(least, x);
  }
  const double hi = over_head<LPH>(mine ? most : Real(-65504), [](Real a, Real b) { return fmax(a, b); });
  const double lo = over_head<LPH>(mine ? least : Real(65504), [](Real a, Real b) { return fmin(a, b); });
  const int lane = __lane_id();
  nan = ((__ballot(nan && mine) >> (lane & ~(LPH - 1))) & ((1ull << LPH) - 1)) != 0;
  const uint32_t sb = half_of((hi - lo) / 15.0);
  const double scale = f16_bits_to_f32(sb);
  const uint32_t ob = half_of(fma(8.0, scale, lo));
  const double offset = f16_bits_to_f32(ob), inv = scale == 0.0 || nan ? 0.0 : 1.0 / scale;
  // A quotient that is a half exactly has to come out as one: the product with the reciprocal is off by 2^-52 of it, and adding
  // and subtracting 3 2^11 rounds it to a multiple of 2^-40.  Then 3 2^51 + 8 brings 8 and the nearest integer, ties to even, into
  // the low word (quotients are below 2^30: an offset is off by at most 16, a scale at least 2^-24).
#pragma unroll
  for (int j = 0; j < 2 * NPL; ++j) {
    double t = (static_cast<double>(v.x[j / NPL][j % NPL]) - offset) * inv;
    t = ((t + 6144.0) - 6144.0) + 6755399441055752.0;
    uint32_t word[2];
    __builtin_memcpy(word, &t, 8);
    code[j / NPL][j % NPL] = static_cast<uint32_t>(min(max(static_cast<int>(word[0]), 0), 15));
  }
  *scale_bits = nan ? 0x7e00u : sb;
  *offset_bits = nan ? 0x7e00u : ob;
}

// A pass is 64 / LPH heads of one token's keys, values or queries, in this order: LPH lanes a head, NPL pairs a lane.  In the half
// layout the two ends of a rotated pair lie rotary_dim / 2 apart, so a lane's dimensions are two runs of NPL, otherwise one of
// 2 NPL; runs are 16-byte loads where alignment and sizes allow (VEC; NPL = 8 of 16-bit types).  The passes of all tokens in
// a row are cut into equal shares for as many wavefronts as the device holds; a share's next pass is being loaded while one
// is worked on, and a token's cosines and sines are computed once for its passes in a share.
//
// Queries are normed and rotated in fp32.  Keys go through 64 bits all the way to their codes: a key computed by another call (a
// shared prefix, a resumed sequence) has the same codes then, whichever way the arithmetic is ordered.
//
// Norm and rotation of 8192 tokens (32 heads and 8 of 128, bfloat16, 168 MB read and written) take 43 us, 3.9 TB/s, where a copy
// has 5.1.  Appending them takes 31 us for the queries (4.3 TB/s) and 32 for keys and values, 34 MB and 9 MB of cache: there a
// SIMD's two wavefronts issue 500 vector instructions for a pass of 16 dimensions a lane, a good part of them in 64 bits, which is half
// of the time, and wait for the other half.  12 heads and 1 of 80 keep a third of the lanes at work: norm and rotation of 8192 tokens 20 us,
// 1.7 TB/s, appending 38.  One token takes 4 to 5 us: a launch and one chain of loads.
//
// Wavefronts a SIMD: what registers allow without spills, or as nearly.  Measured, 8192 tokens, in us: appending and reading back bfloat16 2 : 3 72.6 : 72.2
// (and more for few tokens), fp32 3 : 4 119 : 111; norm and rotation bfloat16 3 : 4 : 6 43 : 43 : 77, fp32 3 : 4 : 6 : 8 73 : 71 : 76 : 110.
constexpr int occupancy_of(int npl, bool vec, bool append) { return !append ? 4 : npl == 8 ? 2 : vec ? 4 : 3; }
// Passes a wavefront from which an append's queries go through a launch of their own, which has more wavefronts and no 64-bit
// registers: one launch : two, with the read-back, bfloat16 at 6 passes 24 : 26 us, 12 40 : 38, 18 67 : 59, 24 86 : 76; fp32 at 12 60 : 63, 24 113 : 111
constexpr int kOwnLaunch = 16;
template <int T, int NPL, int LPH, bool VEC, bool APPEND>
__global__ __launch_bounds__(256, occupancy_of(NPL, VEC, APPEND)) void heads_kernel(const HeadsArgs A) {
  constexpr bool DWORDS = VEC && NPL == 8;  // a run is a dword of codes
  constexpr int WORDS = VEC ? NPL * (T == ITEXHIP_FLOAT ? 4 : 2) / 4 : NPL;
  using Angle = std::conditional_t<APPEND, double, float>;
  __shared__ __align__(16) Angle lds_turns[4][128][2];  // a wavefront's token: cosine and sine of each pair
  __shared__ __align__(8) uint8_t lds_codes[APPEND && !DWORDS ? 4 * 64 * 2 * NPL : 8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t begin = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * A.share;
  const int64_t end = begin + A.share < A.tokens * A.passes ? begin + A.share : A.tokens * A.passes;
  if (begin >= end) return;
  const int sub = lane & (LPH - 1), group = lane / LPH;
  const int D = A.p.head_dim, half_rot = A.p.rotary_dim / 2, pair0 = NPL * sub;
  const bool mine = pair0 < D / 2;
  const int rotated = mine ? (half_rot - pair0 < 0 ? 0 : half_rot - pair0 > NPL ? NPL : half_rot - pair0) : 0;
  const bool split = !A.p.interleaved && pair0 < half_rot;  // VEC: all the lane's pairs are rotated or none
  const int run0 = split ? pair0 : 2 * pair0, run1 = split ? pair0 + half_rot : 2 * pair0 + NPL;
  // without VEC: run 0 holds the pairs' first ends, run 1 the second ones, wherever they are
  auto dim_of = [&](int r, int j) {
    if constexpr (VEC) return (r == 0 ? run0 : run1) + j;
    else return !A.p.interleaved && pair0 + j < half_rot ? pair0 + j + r * half_rot : 2 * (pair0 + j) + r;
  };
  auto in_head = [&](int j) { return VEC ? mine : pair0 + j < D / 2; };

  struct Raw { uint32_t w[2][WORDS]; };
  auto load = [&](const void* src, int64_t at, Raw& raw) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (VEC) {
        const char* from = static_cast<const char*>(src) + (at + (r == 0 ? run0 : run1)) * (T == ITEXHIP_FLOAT ? 4 : 2);
        if (mine) {
          if constexpr (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(from);
            raw.w[r][0] = v.x; raw.w[r][1] = v.y; raw.w[r][2] = v.z; raw.w[r][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(from);
            raw.w[r][0] = v.x; raw.w[r][1] = v.y;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (in_head(j)) raw.w[r][j] = __float_as_uint(load1<T>(src, at + dim_of(r, j)));
      }
    }
  };
  auto widen = [&](const Raw& raw, auto& v) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        float x;
        if constexpr (!VEC || T == ITEXHIP_FLOAT) {
          x = __uint_as_float(raw.w[r][j]);
        } else {
          const uint32_t h = (raw.w[r][j / 2] >> (16 * (j % 2))) & 0xffffu;
          x = T == ITEXHIP_BFLOAT16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
        v.x[r][j] = in_head(j) ? x : 0.0f;
      }
    }
  };
  auto store = [&](void* dst, int64_t at, const Runs<float, NPL>& v) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (VEC) {
        if (!mine) continue;
        char* to = static_cast<char*>(dst) + (at + (r == 0 ? run0 : run1)) * (T == ITEXHIP_FLOAT ? 4 : 2);
        if constexpr (T == ITEXHIP_FLOAT) {
          *reinterpret_cast<f4*>(to) = f4{v.x[r][0], v.x[r][1], v.x[r][2], v.x[r][3]};
        } else {
          uint32_t w[WORDS];
#pragma unroll
          for (int j = 0; j < WORDS; ++j) w[j] = f32x2_to_bits16<T>(v.x[r][2 * j], v.x[r][2 * j + 1]);
          if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(to) = uint4{w[0], w[1], w[2], w[3]};
          else *reinterpret_cast<uint2*>(to) = uint2{w[0], w[1]};
        }
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (in_head(j)) store_output<T>(dst, at + dim_of(r, j), v.x[r][j]);
      }
    }
  };

  enum { kKeys, kValues, kQueries };
  struct Pass { int64_t token, slot; int position, role, head, there; };  // no padding: its copy would be an array in memory
  auto pass_of = [&](int64_t token, int pass, Raw& to) {
    Pass q;
    q.token = token;
    q.role = pass < A.passes_k ? kKeys : pass < A.passes_k + A.passes_v ? kValues : kQueries;
    const int first = q.role == kKeys ? 0 : q.role == kValues ? A.passes_k : A.passes_k + A.passes_v;
    const int heads = q.role == kQueries ? A.p.q_heads : A.p.kv_heads;
    const int64_t st = q.role == kQueries ? A.p.q_strides[0] : q.role == kKeys ? A.p.k_strides[0] : A.p.v_strides[0];
    const int64_t sh = q.role == kQueries ? A.p.q_strides[1] : q.role == kKeys ? A.p.k_strides[1] : A.p.v_strides[1];
    q.head = (pass - first) * (64 / LPH) + group;
    q.there = q.head < heads;  // lanes beyond the last head run along on its values and store nothing
    // by vector loads: the next wait for LDS would be a wait for a scalar one too, a pass before it is wanted
    int at = static_cast<int>(token);
    asm("" : "+v"(at));
    q.position = half_rot > 0 ? A.positions[at] : 0;
    q.slot = 0;
    if constexpr (APPEND) q.slot = A.slots[at];
    load(q.role == kQueries ? A.q : q.role == kKeys ? A.k : A.v, token * st + (q.there ? q.head : heads - 1) * sh, to);
    return q;
  };
  Raw raw, next;
  int64_t token = begin / A.passes;
  int pass = static_cast<int>(begin - token * A.passes);
  Pass now = pass_of(token, pass, raw);
  double freq[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) freq[n] = lane + 64 * n < half_rot ? A.freqs[lane + 64 * n] : 0.0;
  float weight[2][NPL];
  int64_t turned = -1;  // the token that lds_turns is for
  int weights_of = -1;
  for (int64_t i = begin; i < end; ++i) {
    Pass then = now;
    if (++pass == A.passes) {
      pass = 0;
      ++token;
    }
    if (i + 1 < end) then = pass_of(token, pass, next);
    const float* w = now.role == kQueries ? A.q_weight : now.role == kKeys ? A.k_weight : nullptr;
    if (w != nullptr && weights_of != now.role) {
      weights_of = now.role;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < NPL; ++j) weight[r][j] = in_head(j) ? w[dim_of(r, j)] : 0.0f;
    }
    if (half_rot > 0 && turned != now.token && now.role != kValues) {
      turned = now.token;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int pair = lane + 64 * n;
        if (pair >= half_rot) break;
        const double t = static_cast<double>(now.position) * freq[n];
        double c, s;
        turn(t - rint(t), A.p.attention_factor, &c, &s);
        lds_turns[wave][pair][0] = static_cast<Angle>(c);
        lds_turns[wave][pair][1] = static_cast<Angle>(s);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    auto turn_of = [&](int j, auto* c, auto* s) {
      const Angle* at = lds_turns[wave][VEC ? pair0 + j : min(pair0 + j, half_rot - 1)];
      *c = static_cast<std::remove_reference_t<decltype(*c)>>(at[0]);
      *s = static_cast<std::remove_reference_t<decltype(*s)>>(at[1]);
    };
    if (now.role == kQueries || !APPEND) {
      Runs<float, NPL> v;
      widen(raw, v);
      if (w != nullptr) norm<LPH>(A, v, weight);
      rotate<VEC, NPL, float>(v, !VEC || split, rotated, turn_of);
      const int64_t st = now.role == kQueries ? A.p.q_out_strides[0] : A.p.k_out_strides[0], sh = now.role == kQueries ? A.p.q_out_strides[1] : A.p.k_out_strides[1];
      if (now.there) store(now.role == kQueries ? A.q_out : A.k_out, now.token * st + now.head * sh, v);
    } else if constexpr (APPEND) {
      uint32_t code[2][NPL], scale_bits, offset_bits;
      if (now.role == kKeys) {
        Runs<double, NPL> v;
        widen(raw, v);
        if (w != nullptr) norm<LPH>(A, v, weight);
        rotate<VEC, NPL, double>(v, !VEC || split, rotated, turn_of);
        quantize_head<LPH, NPL>(v, mine, &scale_bits, &offset_bits, code);
      } else {
        Runs<float, NPL> v;
        widen(raw, v);
        quantize_head<LPH, NPL>(v, mine, &scale_bits, &offset_bits, code);
      }
      const int64_t its = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(now.slot >> 32))) << 32 |
                          static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(now.slot)));
      const bool placed = its >= 0 && its < A.num_slots;
      const int64_t slot = placed ? its : 0, page_at = (slot >> A.page_shift) * A.page_bytes;
      now.there = now.there && placed;
      const Kv4Block block{A.page_size, A.dp};
      uint8_t* to = A.cache + page_at + static_cast<int64_t>(now.head) * block.bytes();
      const int place = static_cast<int>(slot & (A.page_size - 1));
      auto put = [&](int dword, uint32_t packed) {
        *reinterpret_cast<uint32_t*>(to + (now.role == kKeys ? block.key_codes(place) + 4 * dword : block.value_codes(place, dword))) = packed;
      };
      // the padding of a head: codes that stand for the offset; nothing uses them
      if constexpr (DWORDS) {
        uint32_t packed[2] = {0, 0};
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) packed[r] |= code[r][j] << (4 * j);
        if (now.there) {
          if (mine) {
            put(run0 / 8, packed[0]);
            put(run1 / 8, packed[1]);
          } else if (16 * sub < A.dp) {
            put(2 * sub, 0x88888888u);
            put(2 * sub + 1, 0x88888888u);
          }
        }
      } else {
        // to the order of the dimensions through LDS; the lane then has 2 NPL consecutive ones
        uint8_t* codes = lds_codes + (wave * 64 + group * LPH) * 2 * NPL;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (VEC) {
            if (mine) *reinterpret_cast<uint32_t*>(codes + dim_of(r, 0)) = code[r][0] | code[r][1] << 8 | code[r][2] << 16 | code[r][3] << 24;
          } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j)
              if (in_head(j)) codes[dim_of(r, j)] = static_cast<uint8_t>(code[r][j]);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        static_assert(NPL == 4 || DWORDS, "a dword a lane");
        uint32_t packed = 0x88888888u;
        if (mine) {
          const uint2 u = *reinterpret_cast<const uint2*>(codes + 8 * sub);
          packed = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            packed |= ((u.x >> (8 * j)) & 15u) << (4 * j);
            packed |= ((u.y >> (8 * j)) & 15u) << (16 + 4 * j);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (now.there && 8 * sub < A.dp) put(sub, packed);
      }
      if (now.there && sub == 0) {
        uint8_t* par = to + (now.role == kKeys ? block.key_params(place) : block.value_params(place));
        *reinterpret_cast<uint16_t*>(par) = static_cast<uint16_t>(scale_bits);
        *reinterpret_cast<uint16_t*>(par + 8) = static_cast<uint16_t>(offset_bits);
      }
    }
    raw = next;
    now = then;
  }
}

// Rows of the cache as values: one lane takes eight dimensions of a token's key and value.  A launch has fewer than 2^32 of these
// units, from `first` on, so a unit's place comes from divisions in 32 bits.
template <int T>
__global__ __launch_bounds__(256) void gather_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots, int64_t first, uint32_t units,
                                                     uint32_t kv_heads, int head_dim, int dp, int page_size, int page_shift, int64_t num_slots,
                                                     int64_t page_bytes, void* __restrict__ k_out, void* __restrict__ v_out) {
  const uint32_t unit = blockIdx.x * 256u + threadIdx.x;
  if (unit >= units) return;
  const uint32_t chunks = static_cast<uint32_t>(head_dim) / 8, row = unit / chunks, token = row / kv_heads;
  const int dword = static_cast<int>(unit - row * chunks), head = static_cast<int>(row - token * kv_heads);
  const int64_t slot = slots[first + token], at = (first * kv_heads + row) * head_dim + 8 * dword;
  const bool in = slot >= 0 && slot < num_slots;
  const Kv4Block block{page_size, dp};
  const uint8_t* from = cache + (in ? (slot >> page_shift) * page_bytes : 0) + static_cast<int64_t>(head) * block.bytes();
  const int place = in ? static_cast<int>(slot & (page_size - 1)) : 0;
  auto one = [&](int codes, int params, void* out) {
    const uint32_t w = in ? *reinterpret_cast<const uint32_t*>(from + codes) : 0;
    const float scale = in ? f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(from + params)) : 0.0f;
    const float offset = in ? f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(from + params + 8)) : 0.0f;
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = fmaf(scale, static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8), offset);
      x[4 + j] = fmaf(scale, static_cast<float>(static_cast<int>((w >> (16 + 4 * j)) & 15u) - 8), offset);
    }
    store8<T>(out, at, x);
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

template <int T, int NPL, int LPH, bool VEC, bool APPEND>
void launch(HeadsArgs& A, hipStream_t stream) {
  // as many wavefronts as the device holds at once, or one a pass
  const int64_t all = A.tokens * A.passes, held = 1024 * occupancy_of(NPL, VEC, APPEND);
  A.share = (all + held - 1) / held;
  const int64_t waves = (all + A.share - 1) / A.share;
  heads_kernel<T, NPL, LPH, VEC, APPEND><<<dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, stream>>>(A);
}
template <int T, bool APPEND>
void launch_runs(HeadsArgs& A, int npl, int lph, bool vec, hipStream_t stream) {
  if constexpr (T != ITEXHIP_FLOAT) {
    if (npl == 8) {
      if (lph == 4) launch<T, 8, 4, true, APPEND>(A, stream);
      else if (lph == 8) launch<T, 8, 8, true, APPEND>(A, stream);
      else launch<T, 8, 16, true, APPEND>(A, stream);
      return;
    }
  }
  if (!vec) launch<T, 4, 32, false, APPEND>(A, stream);
  else if (lph == 8) launch<T, 4, 8, true, APPEND>(A, stream);
  else if (lph == 16) launch<T, 4, 16, true, APPEND>(A, stream);
  else launch<T, 4, 32, true, APPEND>(A, stream);
}

template <bool APPEND>
int run(HeadsArgs& A, hipStream_t stream, const char* who) {
  const itexhip_heads_params& p = A.p;
  const size_t esize = p.type == ITEXHIP_FLOAT ? 4 : 2;
  // runs of `n` elements as one load: sizes, strides and addresses are multiples of it
  auto runs_of = [&](int n) {
    auto ok = [&](const void* x, const int64_t* s) { return x == nullptr || (aligned(x, n * esize) && s[0] % n == 0 && s[1] % n == 0); };
    return p.head_dim % (2 * n) == 0 && p.rotary_dim % (2 * n) == 0 && ok(A.q, p.q_strides) && ok(A.k, p.k_strides) && ok(A.v, p.v_strides) &&
           ok(A.q_out, p.q_out_strides) && ok(A.k_out, p.k_out_strides);
  };
  const int npl = p.type != ITEXHIP_FLOAT && runs_of(8) ? 8 : 4;
  const bool vec = npl == 8 || runs_of(4);
  const int lph = !vec ? 32 : (p.head_dim <= 64 ? 32 : p.head_dim <= 128 ? 64 : 128) / npl, group = 64 / lph;
  A.passes_k = A.k != nullptr ? (p.kv_heads + group - 1) / group : 0;
  A.passes_v = APPEND ? A.passes_k : 0;
  A.passes = A.passes_k + A.passes_v + (A.q != nullptr ? (p.q_heads + group - 1) / group : 0);
  if (A.passes == 0 || A.tokens == 0) return ITEXHIP_OK;
  if constexpr (APPEND) {
    if (A.q != nullptr && A.tokens * A.passes >= kOwnLaunch * 1024ll * occupancy_of(npl, vec, true)) {
      HeadsArgs Q = A;
      Q.k = Q.v = nullptr;
      if (const int st = run<false>(Q, stream, who)) return st;
      A.passes = A.passes_k + A.passes_v;
    }
  }
  if (p.type == ITEXHIP_FLOAT) launch_runs<ITEXHIP_FLOAT, APPEND>(A, npl, lph, vec, stream);
  else if (p.type == ITEXHIP_BFLOAT16) launch_runs<ITEXHIP_BFLOAT16, APPEND>(A, npl, lph, vec, stream);
  else launch_runs<ITEXHIP_HALF, APPEND>(A, npl, lph, vec, stream);
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
  const int64_t per_token = static_cast<int64_t>(c->kv_heads) * (c->head_dim / 8);
  const int dp = kv4_padded(c->head_dim);
  auto go = [&](auto kernel) {
    in_pieces(0, tokens, [&](int64_t begin, int64_t end) {
      const uint32_t units = static_cast<uint32_t>((end - begin) * per_token);
      kernel<<<dim3((units + 255) / 256), dim3(256), 0, as_stream(stream)>>>(
          static_cast<const uint8_t*>(cache), slots, begin, units, static_cast<uint32_t>(c->kv_heads), c->head_dim, dp, c->page_size,
          log2_of(c->page_size), c->num_pages * c->page_size, itexhip_kv4_page_bytes(c), k_out, v_out);
    }, kElementsPerLaunch / per_token);
  };
  if (type == ITEXHIP_FLOAT) go(gather_kernel<ITEXHIP_FLOAT>);
  else if (type == ITEXHIP_BFLOAT16) go(gather_kernel<ITEXHIP_BFLOAT16>);
  else go(gather_kernel<ITEXHIP_HALF>);
  ITEXHIP_CHECK_LAUNCH(who);
  return ITEXHIP_OK;
}
