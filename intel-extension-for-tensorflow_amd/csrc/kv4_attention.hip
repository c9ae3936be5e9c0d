// Attention over the paged 4-bit cache.
#include <math.h>

#include <type_traits>

#include "common.hpp"
#include "kv4.hpp"

namespace itexhip {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

constexpr int kMostSplitRows = 64;     // rows of a sequence, times heads of a kv head, that split kernels always take
constexpr int kMostGroups = 1024;      // workgroups of a split kernel
// Copies of the rows in a tile's 16 columns, see Engine; tokens that a workgroup of four wavefronts takes at a time
constexpr int copies_of(bool f32, int64_t rows) { return f32 || rows > 8 ? 1 : rows > 4 ? 2 : 4; }
constexpr int step_of(int copies) { return copies == 4 ? 256 : 128; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kProbExponent = 9.0f;  // probabilities are held as 2^9 p, up to 2^14 p above the maximum so far: half keeps 11 bits down to 2^-23

// Probabilities times scales as halves: 2^(score log2(e) + ref) scale.  ref goes by the largest score and a power of two over the scales
// (scale_bound, an exponent more than was seen), so that they are below 2^10, and 5 bits are left for scores to rise in
// without a look at them (kMostExponent).  The largest score and the largest scale may be different tokens', though, and a large
// scale without probability would take the others' bits: ref falls no further than to where the largest product of a token's own
// probability and scale is 2^4, of which 2^-29 is lost then.  Where that holds ref above what scale_bound asks for,
// scale_bound becomes the present tile's, and scores above raise_at come to be looked at again.
constexpr float kMostExponent = 15.0f, kOwnExponent = 4.0f;
// log2 of a half: a straight line between powers of two, at most 0.09 below it; above it for subnormals, by 9 at most (2^-5 in place of 2^4)
__device__ __forceinline__ float log2_of_half(uint32_t bits) { return fmaf(static_cast<float>(bits & 0x7fffu), 1.0f / 1024.0f, -15.0f); }
__device__ __forceinline__ float log2_over(uint32_t bound) { return static_cast<float>(static_cast<int>(bound >> 10) - 14); }
__device__ __forceinline__ uint32_t bound_of(uint32_t bound, uint32_t most) { return most > bound ? min(most + 0x400u, 0x7bffu) : bound; }
// ref for a tile whose largest score asks for `bound` (with the bound of the scales), its largest product for `own`
__device__ __forceinline__ float lower(float ref, bool first, float bound, float own) {
  const float to = fmaxf(kProbExponent + 1.0f - bound, kOwnExponent - own);
  return first ? to : fminf(ref, to);
}

struct AttArgs {
  const void* q;
  const uint8_t* cache;
  const int32_t *table, *cu_q, *kv_len;
  void* out;
  float* lse;
  int64_t* prefix;   // [num_seqs + 1] steps before each sequence, then the share of a workgroup
  float *part_ml, *part_o;
  int64_t table_stride, total_q, page_bytes, num_pages;
  int64_t q_st, q_sh, o_st, o_sh;
  float scale;
  int q_heads, kv_heads, group, num_seqs, max_q_len, causal, window, head_dim, page_size, page_shift, vec, groups;
};

// One sequence's rows and tokens, whatever the arrays say
struct Seq {
  int64_t first;   // row of q
  int n, len, lo;  // rows to compute, tokens, first token that any row sees (multiple of 32)
  int before;      // position of the first row, by all rows that the sequence has; not below -2^30, where no row sees a token either
  int64_t steps;   // of STEP tokens; at least one if there are rows
};
template <int STEP = 128>
__device__ __forceinline__ Seq sequence(const AttArgs& A, int b) {
  Seq s;
  const int total = static_cast<int>(A.total_q), end = A.cu_q[b + 1], from = min(max(A.cu_q[b], 0), total);
  const int all = end < from ? 0 : end - from;
  s.first = from;
  s.n = min(min(all, total - from), A.max_q_len);
  const int room = static_cast<int>(A.table_stride << A.page_shift);  // at most 2^30
  s.len = min(max(A.kv_len[b], 0), room);
  s.before = max(s.len - all, -(1 << 30));
  s.lo = A.window > 0 ? max(s.before - A.window + 1, 0) & ~31 : 0;
  s.steps = s.n == 0 ? 0 : s.len > s.lo ? (s.len - s.lo + STEP - 1) / STEP : 1;
  return s;
}

// One instruction takes one scalar register and no literals: the masks stay in scalar registers, what is or-ed in a vector register
struct CodeBits {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u;        // the codes
  uint32_t low_one = 0x64006400u, high_one = 0x54005400u; // halves of 1024 and 64
  __device__ __forceinline__ void pin() { asm("" : "+s"(low), "+s"(high), "+v"(low_one), "+v"(high_one)); }
  __device__ __forceinline__ uint32_t at_64(uint32_t x) const { return (x & high) | high_one; }
  __device__ __forceinline__ uint32_t at_1024(uint32_t x) const { return (x & low) | low_one; }
};
__device__ __forceinline__ half2v as_half2(uint32_t u) { half2v h; __builtin_memcpy(&h, &u, 4); return h; }
__device__ __forceinline__ uint32_t as_bits(half2v h) { uint32_t u; __builtin_memcpy(&u, &h, 4); return u; }
__device__ __forceinline__ float low_half(uint32_t u) { return static_cast<float>(as_half2(u)[0]); }
__device__ __forceinline__ float high_half(uint32_t u) { return static_cast<float>(as_half2(u)[1]); }

template <int T>
__device__ __forceinline__ float load_q(const void* q, int64_t i) {
  if constexpr (T == ITEXHIP_FLOAT) return static_cast<const float*>(q)[i];
  else if constexpr (T == ITEXHIP_BFLOAT16) return bf16_bits_to_f32(static_cast<const uint16_t*>(q)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(q)[i]);
}

// Wavefronts a SIMD of a split kernel, and so its workgroups: registers for 2 (256; two tiles of rows of 128 dimensions spill 2 of theirs in
// 16-bit types and 28 in fp32, other kernels none), and longer shares than with 3, where every other wait is for memory
// anyway; 3 where they fit (fp32 of 128: but for 2) and tokens are small or their products long.  44 to 157 scalar
// registers are held in lanes of vector registers.  Measured 2 : 3 in us, half or
// bfloat16 heads of 128: one sequence of 131072 35 : 44, of 65536 (8 rows) 26 : 35, 64 of up to 8192 80 : 80; heads of 64: 32 sequences
// of up to 4096 33.7 : 32.1, one of 32768 22.6 : 19.7; fp32, 32 sequences of up to 4096, 4 heads of 128 80 : 77.  4 spill (138 for 86).
constexpr int occupancy_of(int nb, int dp, bool f32) { return dp == 256 ? 1 : nb == 1 && (dp == 64 || f32) ? 3 : 2; }

// A wavefront's 16 NB rows against 16 TILES tokens at a time, everything in registers.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds, for its query column c, the scores of tokens 4 g .. 4 g + 3
// of each tile, which is the layout that the second product O^T = V^T P^T takes as its operand, so probabilities never
// leave the lane.  (The order of the 32 tokens within that product is the same on both sides and otherwise free.)
//
// Codes become operands without conversions.  A code c four bits up in a half whose exponent is that of 64 is the number
// 64 + c, in its lowest bits with the exponent of 1024 it is 1024 + c: an and-or for two codes.  For keys the excess of 72 (64
// and the 8 that the codes are held over) is taken back once a column (corr, the product's initial value), and scale and
// offset of a token are applied to its score: q . k = scale (q . code) + offset sum(q).  An excess of 1032 would save two shifts
// of seven instructions for eight codes, but costs four bits of the score.  For values the excess is subtracted (exactly:
// averages of many values would cancel against it), the scale is multiplied into the probability before that is
// rounded to half, and offset times probability is summed apart in fp32: codes and products of 11 bits are exact, the one
// rounding is that of the probability.
//
// Probabilities times scales have to fit a half: see above for `ref`, p = 2^(score log2(e) + ref).
//
// Queries are multiplied by a power of two of their row so that half holds what bfloat16 does.  In fp32 the products are
// fp32 MFMAs on fp32 operands, and codes are numbers of -8 .. 7: with an excess to take back the sums would be larger than the
// score and round accordingly (5 drafted tokens over 1500 of heads of 64: off by 7.3e-7 of the values, without it by 4.5e-7).
//
// Few rows (one token of a few heads) would leave most of the 16 columns empty and a softmax of nothing in most lanes.  They are
// repeated COPIES times instead, and copy b of the columns (the lanes' `block`) has the softmax of tile b only: its lanes take their
// scores from that tile's product, and put zeros into the other tiles' places of the second product.  Both products are what they were;
// of the vector instructions those for scales, exponentials and sums are a COPIES-th a token.  The copies' maxima are
// kept alike, their sums are added at the end.  (64 sequences of up to 8192 tokens, 4 rows: 87 us without copies, 80 with four.)
//
// Codes are read once by one workgroup: nontemporal loads leave the caches to the rest (80 us for 91).
template <int T, int DP, int NB, int COPIES>
struct Engine {
  static constexpr bool F32 = T == ITEXHIP_FLOAT;
  static_assert(COPIES == 1 || (NB == 1 && !F32), "copies");
  static constexpr int TILES = COPIES == 4 ? 4 : 2, TOKENS = 16 * TILES, OWN = COPIES == 1 ? TILES : 1, WIDTH = 16 / COPIES;  // OWN: tiles whose scores a lane has
  static constexpr int NKK = DP / 32, E = DP / 16, NV = DP <= 128 ? 1 : 2;
  half8v q16[F32 ? 1 : NB][NKK];
  float q32[F32 ? NB : 1][NKK][8];
  f4 corr[NB];  // what a product of 16-bit types starts from: minus the excess of the codes
  float sumq[NB], qs[NB], m[NB], raise_at[NB], ref[NB], l[NB], po[NB];
  uint32_t scale_bound;  // half bits that no value's scale exceeds without a look: an exponent with all ones below
  int limit[NB], start[NB];  // the tokens that column c of block nb sees: start <= t < limit
  f4 o[NB][E];
  int min_limit, max_start;  // over the wavefront's rows
  int seq_len;               // tokens of the sequence
  int lane, c, g, block;
  CodeBits bits;
  uint32_t kraw[TILES][NKK];
  u4v vraw[TILES][NV], kp[OWN], vp[OWN];
  const uint8_t* own_params;  // with copies: where kp came from
  const __attribute__((address_space(4))) int32_t* table;
  const uint8_t* head_base;
  int64_t page_bytes;
  int last_tile, shift, num_pages;
  uint32_t k_lane, v_lane, p_lane, vp_more;

  __device__ __forceinline__ void init(const AttArgs& A, const Seq& s, int kv_head, int row0) {
    lane = threadIdx.x & 63;
    c = lane & 15;
    g = lane >> 4;
    block = COPIES == 1 ? 0 : c / WIDTH;
    const int rows = s.n * A.group;
    auto limit_of = [&](int row) { return A.causal ? max(s.before + row / A.group + 1, 0) : s.len; };
    auto start_of = [&](int row) { return A.window > 0 ? max(s.before + row / A.group - A.window + 1, 0) : 0; };
    min_limit = limit_of(row0);
    max_start = start_of(min(row0 + 16 * NB, rows) - 1);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + nb * 16 + c % WIDTH;
      const bool in = row < rows;
      limit[nb] = in ? limit_of(row) : 0;
      start[nb] = in ? start_of(row) : 0;
      const int64_t at = in ? (s.first + row / A.group) * A.q_st + static_cast<int64_t>(kv_head * A.group + row % A.group) * A.q_sh : 0;
      float x[NKK][8], most = 0.0f, sum = 0.0f;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        const int d0 = (g * NKK + kk) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[kk][j] = 0.0f;
        if (in && d0 < A.head_dim) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[kk][j] = load_q<T>(A.q, at + d0 + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[kk][j]));
      }
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      float back = 1.0f, excess = 0.0f;
      if constexpr (!F32) {
        // the row's largest magnitude to 1 .. 2: exact but for what is 2^-14 of it and smaller, off by at most 2^-25 of it
        int ex = 0;
        if (most > 1e-30f && most < 3e38f) ex = static_cast<int>((__float_as_uint(most) >> 23) & 255) - 127;
        const float by = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        back = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // operand order: register r holds the codes in bits 4 r .. of a dword's two halves, dimensions r and r + 4
            const _Float16 h = static_cast<_Float16>(x[kk][j] * by);
            q16[nb][kk][(j & 3) * 2 + (j >> 2)] = h;
            const float f = static_cast<float>(h);
            sum += f;
          }
        }
        excess = 72.0f * sum;
      } else {
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            q32[nb][kk][j] = x[kk][j];
            sum += x[kk][j];
          }
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      excess += __shfl_xor(excess, 16);
      excess += __shfl_xor(excess, 32);
      sumq[nb] = sum;
      corr[nb] = f4{-excess, -excess, -excess, -excess};
      qs[nb] = fmaxf(A.scale * kLog2e * back, 1.2e-38f);
      m[nb] = raise_at[nb] = -INFINITY;
      ref[nb] = kProbExponent + (F32 ? 0.0f : 15.0f);
      l[nb] = po[nb] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[nb][e] = f4{0, 0, 0, 0};
    }
    scale_bound = 0x03ffu;  // exponent 2^-15 (subnormals): scales below 2^-14
  }

  // The tokens from .. to - 1 of a sequence; `table` may be read at the pages of those only.
  __device__ __forceinline__ void open(const AttArgs& A, const int32_t* pages, int kv_head, int to) {
    table = (const __attribute__((address_space(4))) int32_t*)(pages);
    last_tile = (to - 1) & ~15;
    shift = A.page_shift;
    num_pages = static_cast<int>(A.num_pages);
    page_bytes = A.page_bytes;
    const Kv4Block block{A.page_size, DP};
    head_base = A.cache + static_cast<int64_t>(kv_head) * block.bytes();
    k_lane = c * (DP / 2) + g * (DP / 8);
    v_lane = block.value_codes(4 * g, DP == 64 ? c / 2 : c);
    p_lane = block.key_params(4 * g);
    vp_more = block.value_params(0) - block.key_params(0);
  }
  // Pages of the tiles at t, t + 16, ... (beyond the last tile: that one's again, masked by its tokens)
  __device__ __forceinline__ void fetch_pages(int t, int (&pages)[TILES]) const {
#pragma unroll
    for (int i = 0; i < TILES; ++i) pages[i] = table[min(t + 16 * i, last_tile) >> shift];
  }
  // Where tile i of the step at t is; a page that is none: page 0 (masked)
  __device__ __forceinline__ const uint8_t* tile(int page, int t, int i, int* place) const {
    *place = min(t + 16 * i, last_tile) & ((1 << shift) - 1);
    return head_base + (page >= 0 && page < num_pages ? page : 0) * page_bytes;
  }
  __device__ __forceinline__ bool valid(int page) const { return page >= 0 && page < num_pages; }

  // What a lane (16 g + c) loads of a step's tiles of 16 tokens:
  //   keys      token c of a tile, dwords g NKK .. g NKK + NKK - 1 of its row
  //   values    tokens 4 g .. 4 g + 3 of a tile, dword c (and c + 16; a half of dword c / 2 if a head has 8 of them)
  //   params    of tokens 4 g .. 4 g + 3 of the tiles that the lane has scores of: four scales, four offsets
  __device__ __forceinline__ void load_keys(const int (&pages)[TILES], int t) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      int place;
      const uint8_t* base = tile(pages[i], t, i, &place);
      const uint8_t* kr = base + place * (DP / 2);
      if constexpr (NKK == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(kr + k_lane);
        kraw[i][0] = w.x;
        kraw[i][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < NKK / 4; ++j) {
          const u4v w = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(kr + k_lane + 16 * j));
#pragma unroll
          for (int n = 0; n < 4; ++n) kraw[i][4 * j + n] = w[n];
        }
      }
      if constexpr (COPIES == 1) kp[i] = *reinterpret_cast<const u4v*>(base + place * 4 + p_lane);
      else own_params = i == 0 || block == i ? base + place * 4 : own_params;
    }
    if constexpr (COPIES > 1) {
      own_params += p_lane;
      kp[0] = *reinterpret_cast<const u4v*>(own_params);
    }
  }
  __device__ __forceinline__ void load_values(const int (&pages)[TILES], int t) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      int place;
      const uint8_t* base = tile(pages[i], t, i, &place);
#pragma unroll
      for (int j = 0; j < NV; ++j) vraw[i][j] = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(base + place * (DP / 2) + v_lane + 256 * j));
      if constexpr (COPIES == 1) vp[i] = *reinterpret_cast<const u4v*>(base + place * 4 + vp_more + p_lane);
    }
    if constexpr (COPIES > 1) vp[0] = *reinterpret_cast<const u4v*>(own_params + vp_more);
  }

  // code n of a dword whose codes have their highest bits flipped, less the 8 that it is held over
  static __device__ __forceinline__ float signed_code(uint32_t flipped, int n) { return static_cast<float>(static_cast<int>(flipped << (28 - 4 * n)) >> 28); }
  __device__ __forceinline__ half8v key_operand(uint32_t w) const {
    const u4v u = {bits.at_64(w << 4), bits.at_64(w), bits.at_64(w >> 4), bits.at_64(w >> 8)};
    half8v h;
    __builtin_memcpy(&h, &u, 16);
    return h;
  }

  __device__ __forceinline__ void rescale(int nb, float a) {
    l[nb] *= a;
    po[nb] *= a;
#pragma unroll
    for (int e = 0; e < E; ++e) o[nb][e] *= a;
  }

  // The sums are held relative to 2^-ref, which falls with the maximum of the scores and with the scales: either has grown
  __device__ __forceinline__ void raise(const float (&p)[NB][4 * OWN], uint32_t most) {
    auto over_lanes = [](float x) {
#pragma unroll
      for (int d = WIDTH; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
      return x;
    };
    if constexpr (F32) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float top = p[nb][0];
#pragma unroll
        for (int j = 1; j < 4 * OWN; ++j) top = fmaxf(top, p[nb][j]);
        top = over_lanes(top);
        const float was = m[nb];
        if (top > was) {
          m[nb] = raise_at[nb] = top;
          const float by = was == -INFINITY ? top * qs[nb] : (top - was) * qs[nb];
          ref[nb] -= by;
          rescale(nb, was == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-by));
        }
      }
    } else {
#pragma unroll
      for (int d = WIDTH; d < 64; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
      most = (most > 0x7bffu ? 0x7bffu : most) | 0x3ffu;  // NaN comes through the products
      scale_bound = bound_of(scale_bound, most);
      bool held = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float top = p[nb][0], own = -INFINITY;
#pragma unroll
        for (int j = 1; j < 4 * OWN; ++j) top = fmaxf(top, p[nb][j]);
        top = over_lanes(top);
#pragma unroll
        for (int j = 0; j < 4 * OWN; ++j) own = fmaxf(own, fmaf(p[nb][j], qs[nb], log2_of_half(vp[j / 4][j % 4 / 2] >> (16 * (j & 1)))));
        own = over_lanes(own);
        if (top > -INFINITY) {
          const float bound = fmaf(top, qs[nb], log2_over(scale_bound)), to = lower(ref[nb], m[nb] == -INFINITY, bound, own);
          if (to != ref[nb]) {
            rescale(nb, m[nb] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(to - ref[nb]));
            ref[nb] = to;
          }
          m[nb] = fmaxf(m[nb], top);
          held = held || to + bound > kMostExponent;
        }
      }
      if (__any(held)) scale_bound = most;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) raise_at[nb] = m[nb] == -INFINITY ? -INFINITY : (kMostExponent - log2_over(scale_bound) - ref[nb]) * __builtin_amdgcn_rcpf(qs[nb]);
    }
  }

  // One step: `pages` are its own, `next` (at `tn`) those of the step to load behind it
  __device__ __forceinline__ void step(bool mask, const int (&pages)[TILES], int t0, const int (&next)[TILES], int tn) {
    auto tile_of = [&](int i) { return COPIES == 1 ? i : block; };  // of the lane's i-th four scores
    float p[NB][4 * OWN];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      f4 own;
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        f4 s = F32 ? f4{0, 0, 0, 0} : corr[nb];
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          if constexpr (!F32) {
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_operand(kraw[i][kk]), q16[nb][kk], s, 0, 0, 0);
          } else {
#pragma unroll
            for (int n = 0; n < 8; ++n)
              s = __builtin_amdgcn_mfma_f32_16x16x4f32(signed_code(kraw[i][kk] ^ 0x88888888u, n), q32[nb][kk][n], s, 0, 0, 0);
          }
        }
        if (COPIES == 1 || i == 0) {
          own = s;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) own[j] = block == i ? s[j] : own[j];
        }
        if (COPIES > 1 && i + 1 < TILES) continue;
        constexpr int last = OWN - 1;
        const int k = COPIES == 1 ? i : last;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sc = kp[k][j / 2], of = kp[k][2 + j / 2];
          const float ks = (j & 1) ? high_half(sc) : low_half(sc), ko = (j & 1) ? high_half(of) : low_half(of);
          p[nb][4 * k + j] = fmaf(ks, own[j], fmaf(ko, sumq[nb], 0.0f));
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_keys(next, tn);
    __builtin_amdgcn_sched_barrier(0);
    if (mask) {
      uint32_t nan = 0;  // bit 4 i + j: the value of token 4 g + j of the lane's tile i is NaN and only some rows may see it
      bool ok[OWN];
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        if (COPIES == 1) ok[COPIES == 1 ? i : 0] = valid(pages[i]);
        else ok[0] = i == 0 || block == i ? valid(pages[i]) : ok[0];
      }
      // tokens beyond the last one hold whatever memory held: their values must not reach a product, not even times zero
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t keep = (j & 1) ? 0x0000ffffu : 0xffff0000u;
          const uint32_t sc = (vp[i][j / 2] >> (16 * (j & 1))) & 0x7fffu, of = (vp[i][2 + j / 2] >> (16 * (j & 1))) & 0x7fffu;
          const bool beyond = t0 + 16 * tile_of(i) + 4 * g + j >= seq_len || !ok[i];
          if (beyond || sc >= 0x7c00u || of >= 0x7c00u) {
            if (!beyond) nan |= 1u << (4 * i + j);
            vp[i][j / 2] &= keep;
            vp[i][2 + j / 2] &= keep;
          }
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int k = 0; k < 4 * OWN; ++k) {
          const int t = t0 + 16 * tile_of(k / 4) + 4 * g + k % 4;
          const bool seen = ok[k / 4] && t < limit[nb] && t >= start[nb];
          p[nb][k] = seen ? p[nb][k] : -INFINITY;
          if (seen && (nan >> k & 1)) l[nb] = NAN;
        }
      }
    }
    uint32_t most = 0;
    bool over = false;
    if constexpr (!F32) {
      typedef unsigned short us2 __attribute__((ext_vector_type(2)));
      us2 two = {0, 0};
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        us2 x[2];
        __builtin_memcpy(x, &vp[i], 8);
        two = __builtin_elementwise_max(two, __builtin_elementwise_max(x[0], x[1]));
      }
      most = two[0] > two[1] ? two[0] : two[1];
      over = most > scale_bound;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float top = p[nb][0];
#pragma unroll
      for (int j = 1; j < 4 * OWN; ++j) top = fmaxf(top, p[nb][j]);
      over = over || top > raise_at[nb];
    }
    if (__any(over)) raise(p, most);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < 4 * OWN; ++j) {
        p[nb][j] = __builtin_amdgcn_exp2f(fmaf(p[nb][j], qs[nb], ref[nb]));
        l[nb] += p[nb][j];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!F32) {
      half8v pb[NB][TILES / 2];  // of tiles 2 u and 2 u + 1
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        uint32_t two[2 * OWN];
#pragma unroll
        for (int j = 0; j < 4 * OWN; j += 2) {
          half2v h;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t sc = vp[j / 4][j % 4 / 2], of = vp[j / 4][2 + j % 4 / 2];
            po[nb] = fmaf(p[nb][j + k], k ? high_half(of) : low_half(of), po[nb]);
            float x = fmaf(p[nb][j + k], k ? high_half(sc) : low_half(sc), 0.0f);
            asm("" : "+v"(x));  // (merged with the conversion it would be an instruction that writes half a register, at twice the time)
            h[k] = static_cast<_Float16>(x);
          }
          two[j / 2] = as_bits(h);
        }
#pragma unroll
        for (int u = 0; u < TILES / 2; ++u) {
          u4v a;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (COPIES == 1) a[k] = two[k];
            else a[k] = block == 2 * u + k / 2 ? two[k & 1] : 0;
          }
          __builtin_memcpy(&pb[nb][u], &a, 16);
        }
      }
      // a lane's eight tokens of one dimension, two a register: first the halves of two tokens' dwords that hold its code
#pragma unroll
      for (int at = 0; at < TILES / 2 * (E / 4); ++at) {
        const int u = at / (E / 4), part = at % (E / 4);  // two tiles, four dimensions: a half of a dword
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u4v& d = vraw[2 * u + i][part / 2 % NV];
            if constexpr (DP == 64) w[2 * i + j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], (c & 1) ? 0x07060302u : 0x05040100u);
            else w[2 * i + j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], (part & 1) ? 0x07060302u : 0x05040100u);
          }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          u4v a;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = n < 2 ? w[k] : w[k] >> 8;
            const half2v h = (n & 1) ? as_half2(bits.at_64(x)) + half2v{-72, -72}
                               : as_half2(bits.at_1024(x)) + half2v{-1032, -1032};
            a[k] = as_bits(h);
          }
          half8v v;
          __builtin_memcpy(&v, &a, 16);
          const int e = part * 4 + n;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[nb][u], o[nb][e], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sc = vp[i][j / 2], of = vp[i][2 + j / 2];
          const float vs = (j & 1) ? high_half(sc) : low_half(sc), vo = (j & 1) ? high_half(of) : low_half(of);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const uint32_t d = vraw[i][e / 8][j] ^ 0x88888888u;
            const float v = fmaf(DP == 64 ? signed_code(d >> (16 * (c & 1)), e) : signed_code(d, e & 7), vs, vo);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[nb][4 * i + j], o[nb][e], 0, 0, 0);
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(next, tn);
    __builtin_amdgcn_sched_barrier(0);
  }

  // Tokens from, from + stride, ..., TOKENS each, up to `to`
  __device__ __forceinline__ void run(const AttArgs& A, const int32_t* pages, int kv_head, int from, int to, int stride, int len) {
    if (from >= to) return;
    seq_len = len;
    bits.pin();
    open(A, pages, kv_head, to);
    int now[TILES], next[TILES], later[TILES];
    fetch_pages(from, now);
    fetch_pages(from + stride, next);
    load_keys(now, from);
    load_values(now, from);
    for (int t = from; t < to; t += stride) {
      fetch_pages(t + 2 * stride, later);
      bool all = t + TOKENS <= min_limit && t >= max_start;
#pragma unroll
      for (int i = 0; i < TILES; ++i) all = all && valid(now[i]);
      step(!all, now, t, next, t + stride);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        now[i] = next[i];
        next[i] = later[i];
      }
    }
  }

  // the first of the four or eight dimensions that o[..][e][r], e = 0 .. 3 (+ 4), belong to
  __device__ __forceinline__ int dim_of(int e, int r) const {
    return DP == 64 ? 4 * (4 * g + r) + e : 8 * (4 * g + r) + (e & 7) + 128 * (e >> 3);
  }

  // The parts of a row's sums that the four lanes of a column, and the copies, hold apart
  template <int BY>  // what the lane BY further on has, among 16
  static __device__ __forceinline__ float turned(float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + BY, 0xf, 0xf, true)); }
  __device__ __forceinline__ void close() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int d = WIDTH; d < 64; d *= 2) l[nb] += __shfl_xor(l[nb], d);
      if constexpr (!F32) {
#pragma unroll
        for (int d = WIDTH; d < 64; d *= 2) po[nb] += __shfl_xor(po[nb], d);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if constexpr (COPIES > 1) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              o[nb][e][r] += turned<8>(o[nb][e][r]);
              if constexpr (COPIES == 4) o[nb][e][r] += turned<4>(o[nb][e][r]);
            }
          }
          o[nb][e] += po[nb];
        }
      }
      l[nb] = fmaf(0.0f, o[nb][0][0], l[nb]);  // a value that is not finite and that all rows of a step saw is in all dimensions' sums so far
    }
  }
  // What the sums are relative to, in units of log2
  __device__ __forceinline__ float top_of(int nb) const { return m[nb] == -INFINITY ? -INFINITY : -ref[nb]; }

  // o / l and the log-sum-exp of the rows; `top` in units of log2
  __device__ __forceinline__ void finish(const AttArgs& A, const Seq& s, int kv_head, int row0, const float (&top)[NB], const float (&sum)[NB]) const {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + nb * 16 + c;
      if (row >= s.n * A.group) continue;
      const int head = kv_head * A.group + row % A.group;
      const int64_t q_row = s.first + row / A.group;
      const bool empty = sum[nb] == 0.0f;
      const float inv = empty ? 0.0f : 1.0f / sum[nb];
      if (g == 0 && A.lse != nullptr)
        A.lse[q_row * A.q_heads + head] = empty ? -INFINITY : kLn2 * (top[nb] + log2f(sum[nb]));
      const int64_t at = q_row * A.o_st + head * A.o_sh;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = dim_of(e, r);
          if (d >= A.head_dim) continue;
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = o[nb][e + j][r] * inv;
          if (A.vec) {
            if constexpr (F32) *reinterpret_cast<f4*>(static_cast<float*>(A.out) + at + d) = f4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.out) + at + d) = uint2{f32x2_to_bits16<T>(v[0], v[1]), f32x2_to_bits16<T>(v[2], v[3])};
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) store_output<T>(A.out, at + d + j, v[j]);
          }
        }
      }
    }
  }
};

// Sequences of few rows, in tiles of 16 NB: the tokens are what is divided.  The steps of all sequences, kv heads and tiles in a
// row, [sequence][kv head][tile][step], are cut into equal shares, one a workgroup, whatever the lengths are and without the host
// knowing them.  A share may end one (sequence, head), hold several whole ones and begin another: whole ones are written out,
// the two at its ends leave their sums in the workspace for combine_kernel.
//
// What bounds it: 64 sequences of up to 8192 tokens (8 kv heads of 128, 378 MB) take 79 us with combine_kernel, 4.8 TB/s, where a copy
// has 5.1 and a launch that only reads 6.9: vector instructions are issued for 60 % of the time (and-or, shift and subtraction of
// the codes: 144 for 64 tokens of a wavefront's 400), matrix instructions for 15 %.  Loads two steps ahead instead of one: 85 us.  One
// sequence of 131072 tokens (143 MB) takes 33 us.  One of 2000 takes 13, a chain of latencies: 9 us for lengths, pages, the
// first codes and the sums of four wavefronts, 4 for the second launch.
template <int NB>
__device__ __forceinline__ int tiles_of(const AttArgs& A, const Seq& s) { return (s.n * A.group + 16 * NB - 1) / (16 * NB); }
template <int T, int DP, int NB, int COPIES>
__global__ __launch_bounds__(256, occupancy_of(NB, DP, T == ITEXHIP_FLOAT)) void split_kernel(const AttArgs A) {
  constexpr int STEP = step_of(COPIES);
  __shared__ int64_t scan[5];
  __shared__ int64_t found[2];
  __shared__ float lds_ml[4][2][16 * NB];
  __shared__ float lds_o[2][NB * (DP / 16) * 4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // steps of all sequences, then the sequence in which this workgroup's share begins
  auto prefix_of = [&](int base, int64_t& inclusive, int64_t& all) {
    const int b = base + tid;
    int64_t x = 0;
    if (b < A.num_seqs) {
      const Seq s = sequence<STEP>(A, b);
      x = s.steps * A.kv_heads * tiles_of<NB>(A, s);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) scan[wave] = x;
    __syncthreads();
    all = scan[0] + scan[1] + scan[2] + scan[3];
    for (int w = 0; w < wave; ++w) x += scan[w];
    inclusive = x;
  };
  int b = 0;
  int64_t total = 0, from = 0, share, begin, end;
  auto cut = [&] {
    share = (total + gridDim.x - 1) / gridDim.x;
    begin = share * blockIdx.x;
    end = begin + share < total ? begin + share : total;
  };
  if (A.num_seqs == 1) {  // nothing to look for
    const Seq s = sequence<STEP>(A, 0);
    total = s.steps * A.kv_heads * tiles_of<NB>(A, s);
    cut();
    if (blockIdx.x == 0 && tid == 0) A.prefix[0] = 0;
  } else {
    int64_t inclusive, all, before = 0;
    for (int base = 0; base < A.num_seqs; base += 256) {
      prefix_of(base, inclusive, all);
      total += all;
    }
    cut();
    if (tid == 0) found[0] = -1;
    for (int base = 0; base < A.num_seqs; base += 256) {
      if (A.num_seqs > 256) prefix_of(base, inclusive, all);
      const int at = base + tid;
      __syncthreads();
      if (at < A.num_seqs) {
        const Seq s = sequence<STEP>(A, at);
        const int64_t mine = s.steps * A.kv_heads * tiles_of<NB>(A, s), first = before + inclusive - mine;
        if (begin >= first && begin < first + mine) {
          found[0] = at;
          found[1] = first;
        }
        if (blockIdx.x == 0) A.prefix[at] = first;
      }
      before += all;
    }
    __syncthreads();
    b = static_cast<int>(found[0]);
    from = found[1];
  }
  if (blockIdx.x == 0 && tid == 0) A.prefix[A.num_seqs] = share;
  if (begin >= end) return;

  for (int64_t at = begin; at < end;) {
    const Seq s = sequence<STEP>(A, b);
    if (s.steps == 0) {
      ++b;
      continue;
    }
    const int64_t rel = at - from;
    const int tiles = tiles_of<NB>(A, s), item = static_cast<int>(rel / s.steps), head = item / tiles, row0 = (item - head * tiles) * 16 * NB;
    const int64_t s0 = rel - item * s.steps, left = s.steps - s0, n = left < end - at ? left : end - at;
    const bool whole = n == s.steps;

    Engine<T, DP, NB, COPIES> eng;
    eng.init(A, s, head, row0);
    const int first = s.lo + static_cast<int>(s0) * STEP, last = first + static_cast<int>(n) * STEP;
    eng.run(A, A.table + b * A.table_stride, head, first + STEP / 4 * wave, last < s.len ? last : s.len, STEP, s.len);
    eng.close();

    // the four wavefronts' sums into those of the first
    float top[NB], sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (eng.g == 0) {
        lds_ml[wave][0][nb * 16 + eng.c] = eng.top_of(nb);
        lds_ml[wave][1][nb * 16 + eng.c] = eng.l[nb];
      }
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int k = nb * 16 + eng.c;
      top[nb] = fmaxf(fmaxf(lds_ml[0][0][k], lds_ml[1][0][k]), fmaxf(lds_ml[2][0][k], lds_ml[3][0][k]));
      const float ref = top[nb] == -INFINITY ? 0.0f : top[nb];
      sum[nb] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum[nb] += lds_ml[w][1][k] * __builtin_amdgcn_exp2f(lds_ml[w][0][k] - ref);
      const float mine = __builtin_amdgcn_exp2f(lds_ml[wave][0][k] - ref);
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) eng.o[nb][e] *= mine;
    }
    for (int half = 2; half >= 1; half /= 2) {
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < DP / 16; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds_o[wave - half][(nb * (DP / 16) + e) * 4 + r][lane] = eng.o[nb][e][r];
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < DP / 16; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) eng.o[nb][e][r] += lds_o[wave][(nb * (DP / 16) + e) * 4 + r][lane];
      }
      __syncthreads();
    }
    if (wave == 0) {
      if (whole) {
        eng.finish(A, s, head, row0, top, sum);
      } else {
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s0 == 0 ? 1 : 0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int row = nb * 16 + eng.c;
          if (row0 + row >= s.n * A.group) continue;
          if (eng.g == 0) {
            A.part_ml[(slot * 16 * NB + row) * 2] = top[nb];
            A.part_ml[(slot * 16 * NB + row) * 2 + 1] = sum[nb];
          }
          float* to = A.part_o + (slot * 16 * NB + row) * DP;
#pragma unroll
          for (int e = 0; e < DP / 16; e += 4)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              *reinterpret_cast<f4*>(to + eng.dim_of(e, r)) = f4{eng.o[nb][e][r], eng.o[nb][e + 1][r], eng.o[nb][e + 2][r], eng.o[nb][e + 3][r]};
        }
      }
    }
    at += n;
    if (rel + n == s.steps * A.kv_heads * tiles) {
      ++b;
      from = at;
    }
  }
}

// One row of a (sequence, kv head) that several workgroups shared: their sums, in the order of the tokens, so that equal calls give equal
// bits.  All partial maxima and sums are read at once by as many threads, then the outputs by groups of DP / 4 (one thread going
// through them: 54 us for a sequence of 131072 tokens where this took 39); 4 to 6 us, most of it the launch.
template <int T, int DP, int NB, int COPIES>
__global__ __launch_bounds__(256) void combine_kernel(const AttArgs A) {
  constexpr int STEP = step_of(COPIES);
  constexpr int LANES = DP / 4, PARTS = 256 / LANES, CHUNK = kMostGroups;
  __shared__ float lds_o[PARTS][DP];
  __shared__ float lds_l[4], lds_top[4], weight[CHUNK];
  const int b = blockIdx.z, head = blockIdx.y, row = blockIdx.x, tid = threadIdx.x;
  const Seq s = sequence<STEP>(A, b);
  if (row >= s.n * A.group) return;
  const int item = head * tiles_of<NB>(A, s) + row / (16 * NB);
  const int64_t share = A.prefix[A.num_seqs], i0 = A.prefix[b] + item * s.steps;
  if (share < 1 || i0 < 0) return;  // (another call is writing the workspace)
  const int64_t w0 = i0 / share, w1 = min((i0 + s.steps - 1) / share, static_cast<int64_t>(A.groups) - 1);
  if (w0 >= w1) return;
  const int count = static_cast<int>(w1 - w0 + 1);  // at most the workgroups of the split kernel, kMostGroups
  auto at = [&](int i) { return (2 * (w0 + i) + (i == 0 ? 1 : 0)) * 16 * NB + row % (16 * NB); };
  const int lane = tid % LANES, part = tid / LANES;
  // every thread takes the maxima and sums of up to CHUNK / 256 parts
  float tops[CHUNK / 256], sums[CHUNK / 256], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < CHUNK / 256; ++k) {
    const int i = tid + 256 * k;
    tops[k] = -INFINITY;
    sums[k] = 0.0f;
    if (i < count) {
      const float2 v = *reinterpret_cast<const float2*>(A.part_ml + at(i) * 2);
      tops[k] = v.x;
      sums[k] = v.y;
    }
    top = fmaxf(top, tops[k]);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (tid % 64 == 0) lds_top[tid / 64] = top;
  __syncthreads();
  top = fmaxf(fmaxf(lds_top[0], lds_top[1]), fmaxf(lds_top[2], lds_top[3]));
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < CHUNK / 256; ++k) {
    const float w = __builtin_amdgcn_exp2f(tops[k] - ref);
    weight[tid + 256 * k] = w;
    sum += sums[k] * w;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (tid % 64 == 0) lds_l[tid / 64] = sum;
  __syncthreads();
  sum = lds_l[0] + lds_l[1] + lds_l[2] + lds_l[3];
  f4 o = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = part; i < count; i += PARTS) o += *reinterpret_cast<const f4*>(A.part_o + at(i) * DP + 4 * lane) * weight[i];
  *reinterpret_cast<f4*>(&lds_o[part][4 * lane]) = o;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) o += *reinterpret_cast<const f4*>(&lds_o[i][4 * lane]);
  const int q_head = head * A.group + row % A.group;
  const int64_t q_row = s.first + row / A.group;
  const bool empty = sum == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / sum;
  if (lane == 0 && A.lse != nullptr) A.lse[q_row * A.q_heads + q_head] = empty ? -INFINITY : kLn2 * (top + log2f(sum));
  if (4 * lane >= A.head_dim) return;
  const int64_t to = q_row * A.o_st + q_head * A.o_sh + 4 * lane;
#pragma unroll
  for (int j = 0; j < 4; ++j) store_output<T>(A.out, to + j, o[j] * inv);
}

// Sequences of more rows in fp32: a wavefront takes 16 NB rows through all the tokens that they see, codes straight from the caches to its
// registers.  fp32 MFMAs (a 16th of half's rate) and a conversion for every code they take bound it: 2048 tokens, 32 heads
// over 8 of 128, 698 us, 49 TFLOP/s.
template <int T, int DP, int NB>
__global__ __launch_bounds__(256) void rows_kernel(const AttArgs A) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.z, head = blockIdx.y;
  const Seq s = sequence(A, b);
  const int rows = s.n * A.group, row0 = (static_cast<int>(blockIdx.x) * 4 + wave) * 16 * NB;
  if (row0 >= rows) return;
  Engine<T, DP, NB, 1> eng;
  eng.init(A, s, head, row0);
  const int first = row0 / A.group, last = (row0 + 16 * NB < rows ? row0 + 16 * NB - 1 : rows - 1) / A.group;
  int to = s.len, from = s.lo;
  if (A.causal) {
    to = s.before + last + 1;
    to = to < 0 ? 0 : to;
  }
  if (A.window > 0) {
    from = s.before + first - A.window + 1;
    from = (from < 0 ? 0 : from) & ~31;
  }
  eng.run(A, A.table + b * A.table_stride, head, from, to, 32, s.len);
  eng.close();
  float top[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) top[nb] = eng.top_of(nb);
  eng.finish(A, s, head, row0, top, eng.l);
}

// Sequences of many rows on half MFMAs.  A workgroup goes through the tokens that its rows see, TT at a time, 32 rows a wavefront: all
// its threads turn a tile's codes into operands in LDS, once for all rows, and the wavefronts read them as whole fragments.
// 32 x 32 x 16 products with the same transposition as in Engine: S^T = K Q^T gives lane 32 h + c the scores of column c for tokens
// 8 i + 4 h + 0 .. 3, which O^T = V^T P^T takes as they are.
//
// LDS holds a fragment as 64 lanes of 16 bytes.  Keys: [32 tokens][16 dimensions], lane 32 h + token: dimensions 8 h .. 8 h + 7 in the
// order of key_operand.  Values: [16 tokens][32 dimensions], lane 32 h + dimension: tokens 4 h .. 4 h + 3 and 8 + 4 h .. + 3.
//
// What bounds it: 8192 tokens, 32 heads over 8 kv heads of 128, bfloat16, take 665 to 700 us, 785 to 830 TFLOP/s of the two products.  The matrix cores
// are busy for a third of that, vector instructions are issued for half of it (a scale, an exponential, a sum and a conversion for
// each score), and a wavefront does one after the other: two on a SIMD overlap them in part.  Measured and slower: four wavefronts of
// 32 rows (995), 64 rows a wavefront (1100), three wavefronts a SIMD (spills, 1280), the products pinned between the vector
// instructions (737), staging by half the wavefronts (730), raised wave priorities (757), each beside 720 to 740 of its day; queries by single
// elements cost every call 11 us.
//
// A wavefront stages tokens of one group of 16 at a time, which lie in one page: page and addresses are scalar.
template <int DP> constexpr int kTile = DP == 256 ? 32 : 64;
template <int DP> constexpr int kWaves = DP == 256 ? 4 : 8;
template <int T, int DP>
__global__ __launch_bounds__(64 * kWaves<DP>, kWaves<DP> / 4) void prompt_kernel(const AttArgs A) {
  constexpr int WAVES = kWaves<DP>, TT = kTile<DP>, TB = TT / 32, KK = DP / 16, DB = DP / 32, U = TT / 16, THREADS = 64 * WAVES, DW = DP / 8;
  constexpr bool FOLD = T == ITEXHIP_HALF;  // scales of values go into the probabilities, as in Engine; else into the operands, a rounding to half
  typedef float f16v __attribute__((ext_vector_type(16)));
  __shared__ u4v lds_k[2][TB * KK * 64], lds_v[2][U * DB * 64], lds_vp[2][TT / 4];
  __shared__ f4 lds_kp[2][TT / 2];  // of two tokens: scale and offset - 72 scale, the excess of the codes taken back
  // A bit a token: [..][0] seen by some row, [..][1] its value is not finite; without FOLD [..][1] is all of 16 tokens if some value of
  // theirs may be none as a half, and lds_nans says which are not finite
  __shared__ __align__(16) uint16_t lds_flags[2][2][4];
  __shared__ __align__(8) uint16_t lds_nans[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % A.kv_heads, b = blockIdx.z;  // neighbouring workgroups, on different dies, take different heads
  const Seq s = sequence(A, b);
  const int rows = s.n * A.group, tile_rows = 32 * WAVES;
  const int tiles = (rows + tile_rows - 1) / tile_rows;
  const int at_tile = tiles - 1 - static_cast<int>(blockIdx.x / A.kv_heads);  // the longest first
  if (at_tile < 0) return;
  const int row0 = at_tile * tile_rows + 32 * wave, row = row0 + c;
  auto limit_of = [&](int r) { return A.causal ? max(s.before + r / A.group + 1, 0) : s.len; };
  auto start_of = [&](int r) { return A.window > 0 ? max(s.before + r / A.group - A.window + 1, 0) : 0; };
  // of the workgroup and the wavefront
  const int first_row = at_tile * tile_rows, last_row = min(first_row + tile_rows, rows) - 1;
  const int from = start_of(first_row) & ~(TT - 1), to = min(limit_of(last_row), s.len);
  const bool there = row0 < rows;
  const int w_last = min(row0 + 32, rows) - 1;
  const int w_to = there ? limit_of(w_last) : 0, w_from = start_of(row0), w_all_to = limit_of(row0), w_all_from = there ? start_of(w_last) : 0;

  // queries, as in Engine::init
  half8v q[KK];
  float sumq = 0.0f, qs;
  const bool in = row < rows;
  const int limit = in ? limit_of(row) : 0, start = in ? start_of(row) : 0;
  {
    float x[KK][8], most = 0.0f;
    const int64_t at = in ? (s.first + row / A.group) * A.q_st + static_cast<int64_t>(head * A.group + row % A.group) * A.q_sh : 0;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d0 = kk * 16 + hi * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[kk][j] = 0.0f;
      if (in && d0 < A.head_dim) {  // (a branch around all eight: they become one load)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[kk][j] = load_q<T>(A.q, at + d0 + j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[kk][j]));
    }
    most = fmaxf(most, __shfl_xor(most, 32));
    int ex = 0;
    if (most > 1e-30f && most < 3e38f) ex = static_cast<int>((__float_as_uint(most) >> 23) & 255) - 127;
    const float by = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
    qs = fmaxf(A.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + ex) << 23), 1.2e-38f);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const _Float16 h = static_cast<_Float16>(x[kk][j] * by);
        q[kk][(j & 3) * 2 + (j >> 2)] = h;
        sumq += static_cast<float>(h);
      }
    }
    sumq += __shfl_xor(sumq, 32);
  }
  float m = -INFINITY, raise_at = -INFINITY, l = 0.0f, po = 0.0f, ref = kProbExponent + (FOLD ? 15.0f : 0.0f);
  f16v o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  uint32_t scale_bound = 0x03ffu;

  CodeBits bits;
  bits.pin();
  const Kv4Block block{A.page_size, DP};
  const uint8_t* head_base = A.cache + static_cast<int64_t>(head) * block.bytes();
  const int32_t* table = A.table + b * A.table_stride;
  // Tasks of a group of 16 tokens: keys (token, pair of dwords), values (half, dword, pair of codes).  A wavefront has its tasks in one
  // group, or (DP = 256) in both one after the other.
  constexpr int KG = 16 * DW / 2, VG = 2 * DW * 4, STAGERS = U * VG / 64 < WAVES ? U * VG / 64 : WAVES, N = U * VG / (64 * STAGERS);
  static_assert(KG == VG && VG % 64 == 0 && (64 * STAGERS) % VG == 0, "the wavefronts of a group");
  const bool stages = wave < STAGERS;
  const int in_group = tid % VG;
  auto group_of = [&](int i) { return i * (64 * STAGERS / VG) + wave / (VG / 64); };
  const int k_token = in_group & 15, k_pair = in_group >> 4, v_pair = in_group & 3, v_dword = (in_group >> 2) % DW, v_half = (in_group >> 2) / DW;
  const uint32_t k_lane = k_token * (DP / 2) + 8 * k_pair, v_lane = block.value_codes(4 * v_half, v_dword), vp_lane = block.value_params(4 * v_half),
                 par_lane = block.key_params(4 * (lane & 3)) + (lane & 4) * A.page_size;  // keys' of four tokens, values' of four tokens
  uint2 kraw[N];
  u4v vraw[N][2], vpar[N][2];
  u4v par = {0, 0, 0, 0};
  int page[N], par_page = -1, par_next = -1;  // parameters: a group for each of the first wavefronts, which the others wait for anyway
  auto good = [&](int p) { return p >= 0 && p < A.num_pages; };
  // Pages, read a tile ahead of the loads that need them; by vector loads, since the wait for a scalar one would be the wait for
  // all of LDS too and come at once
  int next[N];
  auto look_up = [&](int t0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int at = min(t0 + 16 * group_of(i), to - 1) >> A.page_shift;
      asm("" : "+v"(at));
      next[i] = table[at];
    }
    int at = min(t0 + 16 * (wave % U), to - 1) >> A.page_shift;
    asm("" : "+v"(at));
    par_next = table[at];
  };
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < N; ++i) page[i] = __builtin_amdgcn_readfirstlane(next[i]);
    par_page = __builtin_amdgcn_readfirstlane(par_next);
    look_up(t0 + TT);
    if (wave < U) {
      const uint8_t* params = head_base + (good(par_page) ? par_page : 0) * A.page_bytes + ((t0 + 16 * wave) & (A.page_size - 1)) * 4;
      if (lane < 8) par = *reinterpret_cast<const u4v*>(params + par_lane);
    }
    if (!stages) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int place = (t0 + 16 * group_of(i)) & (A.page_size - 1);
      const uint8_t* base = head_base + (good(page[i]) ? page[i] : 0) * A.page_bytes;
      const uint8_t *codes = base + place * (DP / 2), *params = base + place * 4;
      kraw[i] = *reinterpret_cast<const uint2*>(codes + k_lane);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        vraw[i][k] = *reinterpret_cast<const u4v*>(codes + v_lane + k * (8 * DP / 2));
        if (!FOLD) vpar[i][k] = *reinterpret_cast<const u4v*>(params + vp_lane + k * 32);
      }
    }
  };
  auto stage = [&](int t0, int buf) {
    if (!stages) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = group_of(i), tg = t0 + 16 * u, t = 16 * u + k_token;
      u4v* to_k = &lds_k[buf][((t / 32) * KK + k_pair) * 64 + t % 32];
      to_k[0] = u4v{bits.at_64(kraw[i].x << 4), bits.at_64(kraw[i].x), bits.at_64(kraw[i].x >> 4), bits.at_64(kraw[i].x >> 8)};
      to_k[32] = u4v{bits.at_64(kraw[i].y << 4), bits.at_64(kraw[i].y), bits.at_64(kraw[i].y >> 4), bits.at_64(kraw[i].y >> 8)};
      if (!FOLD && (!good(page[i]) || tg + 16 > s.len)) {  // tokens beyond the last one or without a page become zeros
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t2 = tg + 8 * (k / 2) + 4 * v_half + 2 * (k & 1);
          const uint32_t keep = !good(page[i]) ? 0 : (t2 < s.len ? 0xffffu : 0u) | (t2 + 1 < s.len ? 0xffff0000u : 0u);
          vpar[i][k / 2][k & 1] &= keep;
          vpar[i][k / 2][2 + (k & 1)] &= keep;
        }
      }
      const uint32_t pick = (v_pair & 2) ? 0x07060302u : 0x05040100u;
      const int shift = (v_pair & 1) * 8;
      u4v a, z;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = __builtin_amdgcn_perm(vraw[i][k / 2][2 * (k & 1) + 1], vraw[i][k / 2][2 * (k & 1)], pick) >> shift;
        half2v first = as_half2(bits.at_1024(x)) + half2v{-1032, -1032}, second = as_half2(bits.at_64(x)) + half2v{-72, -72};
        if constexpr (!FOLD) {
          const uint32_t vs = vpar[i][k / 2][k & 1], vo = vpar[i][k / 2][2 + (k & 1)];
          first = __builtin_elementwise_fma(first, as_half2(vs), as_half2(vo));
          second = __builtin_elementwise_fma(second, as_half2(vs), as_half2(vo));
        }
        a[k] = as_bits(first);
        z[k] = as_bits(second);
      }
      u4v* to_v = &lds_v[buf][(u * DB + v_dword / 4) * 64 + v_half * 32 + (v_dword & 3) * 8 + 2 * v_pair];
      to_v[0] = a;
      to_v[1] = z;
    }
  };
  auto stage_params = [&](int t0, int buf) {
    if (wave >= U) return;
    const int tg = t0 + 16 * wave;
    auto odd = [](uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; };
    // without FOLD: a value is at most 8 |scale| + |offset|; what append saturated comes to up to 65536, which a half does not hold
    auto most = [&](int j) { return as_bits(__builtin_elementwise_fma(as_half2(par[j] & 0x7fff7fffu), half2v{8, 8}, as_half2(par[2 + j] & 0x7fff7fffu))); };
    const bool far = FOLD ? odd(par[0]) || odd(par[1]) || odd(par[2]) || odd(par[3]) : odd(most(0)) || odd(most(1));
    const bool any_far = !FOLD && __any(lane >= 4 && lane < 8 && far);
    uint32_t valid = 0xffffu, nans = 0;
    if (!good(par_page) || tg + 16 > s.len || (FOLD ? __any(lane >= 4 && lane < 8 && far) : any_far)) {
      const int n = good(par_page) ? min(max(s.len - tg, 0), 16) : 0;
      valid = (1u << n) - 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // token 4 (lane - 4) + j
        const uint32_t vs = par[j / 2] >> (16 * (j & 1)), vo = par[2 + j / 2] >> (16 * (j & 1));
        const bool is_nan = (vs & 0x7c00u) == 0x7c00u || (vo & 0x7c00u) == 0x7c00u;
        const uint64_t lanes = __ballot(lane >= 4 && lane < 8 && is_nan) >> 4;
        nans |= static_cast<uint32_t>((lanes & 1) | (lanes & 2) << 3 | (lanes & 4) << 6 | (lanes & 8) << 9) << j;
      }
      nans &= valid;
      if (FOLD) {
        const uint32_t keep = (valid & ~nans) >> (4 * (lane & 3));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (lane >= 4 && !(keep >> j & 1)) {
            const uint32_t other = (j & 1) ? 0x0000ffffu : 0xffff0000u;
            par[j / 2] &= other;
            par[2 + j / 2] &= other;
          }
        }
      }
    }
    if (lane == 0) {
      lds_flags[buf][0][wave] = static_cast<uint16_t>(valid);
      lds_flags[buf][1][wave] = static_cast<uint16_t>(FOLD ? nans : any_far ? 0xffffu : 0u);
      if (!FOLD) lds_nans[buf][wave] = static_cast<uint16_t>(nans);
    }
    if (lane < 4) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float ks0 = low_half(par[j]), ks1 = high_half(par[j]);
        lds_kp[buf][2 * (4 * wave + lane) + j] = f4{ks0, fmaf(-72.0f, ks0, low_half(par[2 + j])), ks1, fmaf(-72.0f, ks1, high_half(par[2 + j]))};
      }
    } else if (lane < 8) {
      lds_vp[buf][4 * wave + lane - 4] = par;
    }
  };
  auto rescale = [&](float by) {  // after ref -= by
    const float a = __builtin_amdgcn_exp2f(-by);
    l *= a;
    po *= a;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] *= a;
  };

  if (from < to) {
    look_up(from);
    fetch(from);
    stage_params(from, 0);
    stage(from, 0);
  }
  __syncthreads();
  constexpr uint64_t kAll = TT == 64 ? ~0ull : (1ull << (TT & 63)) - 1;
  for (int t0 = from, buf = 0; t0 < to; t0 += TT, buf ^= 1) {
    const bool more = t0 + TT < to;
    const u4v flags = *reinterpret_cast<const u4v*>(lds_flags[buf]);
    if (more) fetch(t0 + TT);
    const uint64_t valid = (flags[0] | static_cast<uint64_t>(flags[1]) << 32) & kAll;
    uint64_t nans = (flags[2] | static_cast<uint64_t>(flags[3]) << 32) & kAll;
    if constexpr (!FOLD) {
      // values that are not finite reach the rows that see them through l, the products as finite ones; values beyond a half are its
      // largest, 65504 for at most 65536: 2^-11 of it
      if (nans != 0) {
        const uint2 bits_of = *reinterpret_cast<const uint2*>(lds_nans[buf]);
        nans = (bits_of.x | static_cast<uint64_t>(bits_of.y) << 32) & kAll;
        half8v* all = reinterpret_cast<half8v*>(lds_v[buf]);
        constexpr _Float16 top = static_cast<_Float16>(65504.0f);
        for (int k = tid; k < U * DB * 64; k += THREADS) {
          half8v a = all[k];
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = a[j] != a[j] ? static_cast<_Float16>(0) : a[j] > top ? top : a[j] < -top ? -top : a[j];
          all[k] = a;
        }
        __syncthreads();
      }
    }
    if (t0 < w_to && t0 + TT > w_from) {
      const bool mask = valid != kAll || nans != 0 || t0 + TT > w_all_to || t0 < w_all_from;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        // fragments are asked for ahead of the products that take them: the keys' at once, the values' before the softmax
        half8v kf[KK], vf[2][DB];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) __builtin_memcpy(&kf[kk], &lds_k[buf][(tb * KK + kk) * 64 + lane], 16);
        f16v sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kk], q[kk], sc, 0, 0, 0);
#pragma unroll
        for (int d = 0; d < DB; ++d) __builtin_memcpy(&vf[0][d], &lds_v[buf][(2 * tb * DB + d) * 64 + lane], 16);
        u4v vp[FOLD ? 4 : 1];
        float p[16], top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const f4 par = lds_kp[buf][tb * 16 + 4 * (k / 2) + 2 * hi + k % 2];
          p[2 * k] = fmaf(par[0], sc[2 * k], par[1] * sumq);
          p[2 * k + 1] = fmaf(par[2], sc[2 * k + 1], par[3] * sumq);
        }
        if constexpr (FOLD) {
#pragma unroll
          for (int k = 0; k < 4; ++k) vp[k] = lds_vp[buf][tb * 8 + 2 * k + hi];
        }
        if (mask) {
          const uint32_t here = static_cast<uint32_t>(valid >> (32 * tb)) >> (4 * hi), nan_here = static_cast<uint32_t>(nans >> (32 * tb)) >> (4 * hi);
          const int first = t0 + 32 * tb + 4 * hi, below = limit - first, above = start - first;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = 8 * (r / 4) + r % 4;  // from the lane's first token of the block
            const bool seen = (here >> at & 1) && at < below && at >= above;
            p[r] = seen ? p[r] : -INFINITY;
            if (seen && (nan_here >> at & 1)) l = NAN;
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, p[r]);
        uint32_t most = 0;
        if constexpr (FOLD) {
          typedef unsigned short us2 __attribute__((ext_vector_type(2)));
          us2 two = {0, 0};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            us2 x[2];
            __builtin_memcpy(x, &vp[k], 8);
            two = __builtin_elementwise_max(two, __builtin_elementwise_max(x[0], x[1]));
          }
          most = two[0] > two[1] ? two[0] : two[1];
        }
        if (__any(top > raise_at || (FOLD && most > scale_bound))) {
          top = fmaxf(top, __shfl_xor(top, 32));
          if constexpr (FOLD) {
            most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
            most = (most > 0x7bffu ? 0x7bffu : most) | 0x3ffu;
            scale_bound = bound_of(scale_bound, most);
            uint32_t least = 0xffffu;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint32_t x = vp[k / 2][k % 2];
              asm volatile("" : "+v"(x));  // (not ahead of the branch, where the results would take registers that spill)
              least = min(least, min(x & 0xffffu, x >> 16));
            }
            float own = INFINITY;  // where no scale is far below the bound, that holds for the products too
            if (__any(log2_over(scale_bound) - log2_of_half(least) > kProbExponent + 1.0f - kOwnExponent)) {
              own = -INFINITY;
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                uint32_t x = vp[r / 4][r % 4 / 2];
                asm volatile("" : "+v"(x));
                own = fmaxf(own, fmaf(p[r], qs, log2_of_half(x >> (16 * (r & 1)))));
              }
              own = fmaxf(own, __shfl_xor(own, 32));
            }
            bool held = false;
            if (top > -INFINITY) {
              const float bound = fmaf(top, qs, log2_over(scale_bound)), to = lower(ref, m == -INFINITY, bound, own);
              if (to != ref) rescale(m == -INFINITY ? 0.0f : ref - to);
              ref = to;
              m = fmaxf(m, top);
              held = to + bound > kMostExponent;
            }
            if (__any(held)) scale_bound = most;
            raise_at = m == -INFINITY ? -INFINITY : (kMostExponent - log2_over(scale_bound) - ref) * __builtin_amdgcn_rcpf(qs);
          } else if (top > m) {
            const float by = m == -INFINITY ? top * qs : (top - m) * qs;
            ref -= by;
            rescale(m == -INFINITY ? 0.0f : by);
            m = top;
            raise_at = top + 5.0f / qs;
          }
        }
        half8v pb[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = __builtin_amdgcn_exp2f(fmaf(p[r], qs, ref));
          l += x;
          if constexpr (FOLD) {
            const uint32_t vs = vp[r / 4][r % 4 / 2], vo = vp[r / 4][2 + r % 4 / 2];
            po = fmaf(x, (r & 1) ? high_half(vo) : low_half(vo), po);
            x = fmaf(x, (r & 1) ? high_half(vs) : low_half(vs), 0.0f);
            asm("" : "+v"(x));  // (merged with the conversion it would be an instruction that writes half a register, at twice the time)
          }
          pb[r / 8][r % 8] = static_cast<_Float16>(x);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) __builtin_memcpy(&vf[1][d], &lds_v[buf][((2 * tb + 1) * DB + d) * 64 + lane], 16);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[u][d], pb[u], o[d], 0, 0, 0);
        }
      }
    }
    if (more) {
      stage_params(t0 + TT, buf ^ 1);
      stage(t0 + TT, buf ^ 1);
    }
    __syncthreads();
  }

  l += __shfl_xor(l, 32);
  if constexpr (FOLD) po += __shfl_xor(po, 32);
  if (!in) return;
  const int q_head = head * A.group + row % A.group;
  const int64_t q_row = s.first + row / A.group, at = q_row * A.o_st + q_head * A.o_sh;
  const bool empty = l == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / l;
  if (hi == 0 && A.lse != nullptr) A.lse[q_row * A.q_heads + q_head] = empty ? -INFINITY : kLn2 * (log2f(l) - ref);
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dim = 32 * d + 8 * i + 4 * hi;
      if (dim >= A.head_dim) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (o[d][4 * i + j] + (FOLD ? po : 0.0f)) * inv;
      if (A.vec) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.out) + at + dim) = uint2{f32x2_to_bits16<T>(v[0], v[1]), f32x2_to_bits16<T>(v[2], v[3])};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) store_output<T>(A.out, at + dim + j, v[j]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
struct Plan {
  int blocks;      // NB
  int copies;
  bool split;
  int64_t groups;  // workgroups of the split kernel
  size_t prefix, ml, o;
};

// Of more than kMostSplitRows rows, whether the tokens are divided (split_kernel) or the rows alone (prompt_kernel, rows_kernel).  Those
// give a workgroup one tile of rows and all the tokens, and leave CUs idle where there are few tiles: as long as each has a CU of its own, the
// time is that of one, 9 us and so much a token of the longest sequence.  split_kernel's is 25 us and so much a row and token, and
// what combine_kernel takes for a row.  In us, 8 kv heads of 128 and 4 query heads each but where noted (the constants are these sizes'; others
// go by the formula), rows alone : tokens divided, sequences x rows of tokens
//   bfloat16  16 x 17 of 4096 137 : 90, 64 of 16384 595 : 57, 512 of 16384 599 : 288, 4 x 128 of 4096 158 : 95, 100 of 2000 83 : 32, 2 x 200 of
//             1000 49 : 64, 300 of 300 22 : 46, 1000 of 1000 47 : 95, 1000 of 4096 161 : 203; heads of 256: 128 of 16384 1218 : 204;
//             12 heads of 64: 4 x 128 of 1024 37 : 36, 512 of 512 25 : 28
//   fp32      128 of 4096 676 : 110, 4 x 128 of 4096 676 : 353, 512 of 4096 674 : 355; 12 heads of 64: 512 of 512 54 : 34, 2048 of 2048 193 : 194
// The longest sequence is taken to be as long as the table is wide (the host knows no lengths) or what a window leaves of it.
bool tokens_are_divided(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c, int64_t rows, int dp) {
  const bool f32 = p->type == ITEXHIP_FLOAT;
  const int64_t tile = f32 ? (dp == 256 ? 64 : 128) : dp == 256 ? 128 : 256, all = static_cast<int64_t>(p->num_seqs) * c->kv_heads;
  if ((rows + tile - 1) / tile * all > 256) return false;
  double tokens = static_cast<double>(p->table_stride) * c->page_size;
  if (p->window > 0) tokens = fmin(tokens, static_cast<double>(p->window) + p->max_q_len);
  const double by_rows = 9.0 + tokens * (f32 ? 0.165 : dp == 256 ? 0.072 : 0.0366);
  const double divided = 25.0 + static_cast<double>(rows * all) * (tokens * (f32 ? 5.6e-6 : 1.1e-6) + 1.0 / 600.0);
  return divided < by_rows;
}

// Workgroups of a split kernel of `blocks` tiles of 16 rows: what the device holds, or one a step
int64_t groups_of(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c, int step, int blocks, int64_t rows) {
  const int64_t full = 256 * occupancy_of(blocks, kv4_padded(c->head_dim), p->type == ITEXHIP_FLOAT);
  const int64_t steps = static_cast<int64_t>(p->num_seqs) * c->kv_heads * ((p->table_stride * c->page_size + step - 1) / step);
  const int64_t bound = (steps < full ? steps : full) * ((rows + 16 * blocks - 1) / (16 * blocks));
  return bound < 1 ? 1 : bound < full ? bound : full;
}
size_t prefix_bytes(int num_seqs) { return (static_cast<size_t>(num_seqs) + 1) * 8 + 15 & ~size_t{15}; }

Plan plan_of(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c) {
  Plan plan = {};
  const int dp = kv4_padded(c->head_dim);
  const int64_t rows = static_cast<int64_t>(p->max_q_len) * (p->q_heads / c->kv_heads);
  plan.blocks = rows <= 16 || dp == 256 ? 1 : 2;
  plan.copies = copies_of(p->type == ITEXHIP_FLOAT, rows);
  plan.split = rows <= kMostSplitRows || tokens_are_divided(p, c, rows, dp);
  if (plan.split) {
    plan.groups = groups_of(p, c, step_of(plan.copies), plan.blocks, rows);
    plan.prefix = prefix_bytes(p->num_seqs);
    plan.ml = static_cast<size_t>(plan.groups) * 2 * 16 * plan.blocks * 2 * 4;
    plan.o = static_cast<size_t>(plan.groups) * 2 * 16 * plan.blocks * dp * 4;
  }
  return plan;
}

// What the plan of this call and of every call of fewer sequences, rows or pages needs: which kernel takes a call goes by its own sizes, and
// a program keeps one workspace for calls of many.
size_t workspace_bytes(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c) {
  const int dp = kv4_padded(c->head_dim);
  const int64_t rows = static_cast<int64_t>(p->max_q_len) * (p->q_heads / c->kv_heads), lone = dp == 256 ? rows : rows < 16 ? rows : 16;
  const size_t part = 2 * 16 * static_cast<size_t>(dp + 2) * 4;
  const size_t one = groups_of(p, c, 128, 1, lone) * part, two = rows > lone ? groups_of(p, c, 128, 2, rows) * 2 * part : 0;
  return prefix_bytes(p->num_seqs) + (one > two ? one : two) + 16;
}

int check(const char* who, const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c) {
  if (const char* wrong = kv4_invalid(c)) {
    set_error("%s: %s", who, wrong);
    return ITEXHIP_INVALID_ARGUMENT;
  }
  ITEXHIP_REQUIRE(p != nullptr, "%s: null parameters", who);
  ITEXHIP_REQUIRE(p->type == ITEXHIP_FLOAT || is_float16_type(p->type), "%s: type is float, bfloat16 or half", who);
  ITEXHIP_REQUIRE(p->q_heads >= 1 && p->q_heads <= 65535 && p->q_heads % c->kv_heads == 0, "%s: q_heads is a multiple of kv_heads, at most 65535", who);
  ITEXHIP_REQUIRE(p->num_seqs >= 0 && p->num_seqs <= 65535, "%s: num_seqs is 0 to 65535", who);
  ITEXHIP_REQUIRE(p->max_q_len >= 0 && static_cast<int64_t>(p->max_q_len) * p->q_heads < (1ll << 30),
                  "%s: max_q_len times q_heads is 0 to 2^30 - 1", who);
  ITEXHIP_REQUIRE(p->total_q >= 0 && p->total_q < (1ll << 31), "%s: total_q is 0 to 2^31 - 1", who);
  ITEXHIP_REQUIRE(p->scale > 0.0f && isfinite(p->scale), "%s: scale is finite and positive", who);
  ITEXHIP_REQUIRE(p->window >= 0, "%s: window is not negative", who);
  ITEXHIP_REQUIRE(p->table_stride >= 0 && p->table_stride <= (1ll << 30) / c->page_size, "%s: table_stride times page_size is 0 to 2^30", who);
  const int64_t* all[2] = {p->q_strides, p->out_strides};
  for (const int64_t* s : all)
    for (int i = 0; i < 2; ++i)
      ITEXHIP_REQUIRE(s[i] > -(1ll << 40) && s[i] < (1ll << 40), "%s: a stride of %lld elements", who, static_cast<long long>(s[i]));
  return ITEXHIP_OK;
}

template <int T, int DP, int NB>
void launch(const AttArgs& A, const Plan& plan, hipStream_t stream) {
  const int rows = A.max_q_len * A.group;
  if (plan.split) {
    auto both = [&](auto copies) {
      split_kernel<T, DP, NB, copies.value><<<dim3(static_cast<unsigned>(plan.groups)), dim3(256), 0, stream>>>(A);
      if (plan.groups > 1) combine_kernel<T, DP, NB, copies.value><<<dim3(rows, A.kv_heads, A.num_seqs), dim3(256), 0, stream>>>(A);
    };
    if constexpr (T != ITEXHIP_FLOAT && NB == 1) {
      if (plan.copies == 4) both(std::integral_constant<int, 4>{});
      else if (plan.copies == 2) both(std::integral_constant<int, 2>{});
      else both(std::integral_constant<int, 1>{});
    } else {
      both(std::integral_constant<int, 1>{});
    }
  } else {
    if constexpr (T == ITEXHIP_FLOAT) {
      rows_kernel<T, DP, NB><<<dim3((rows + 64 * NB - 1) / (64 * NB), A.kv_heads, A.num_seqs), dim3(256), 0, stream>>>(A);
    } else {
      constexpr int tile = 32 * kWaves<DP>;
      prompt_kernel<T, DP><<<dim3(A.kv_heads * ((rows + tile - 1) / tile), 1, A.num_seqs), dim3(2 * tile), 0, stream>>>(A);
    }
  }
}
template <int T, int DP>
void launch_blocks(const AttArgs& A, const Plan& plan, hipStream_t stream) {
  if (plan.blocks == 1) launch<T, DP, 1>(A, plan, stream);
  else if constexpr (DP != 256) launch<T, DP, 2>(A, plan, stream);
}
template <int T>
void launch_dims(const AttArgs& A, const Plan& plan, hipStream_t stream) {
  const int dp = kv4_padded(A.head_dim);
  if (dp == 64) launch_blocks<T, 64>(A, plan, stream);
  else if (dp == 128) launch_blocks<T, 128>(A, plan, stream);
  else launch_blocks<T, 256>(A, plan, stream);
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int64_t itexhip_kv4_attention_workspace(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c) {
  if (check("itexhip_kv4_attention_workspace", p, c) != ITEXHIP_OK) return 0;
  return static_cast<int64_t>(workspace_bytes(p, c));
}

extern "C" int itexhip_kv4_attention(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c, const void* q, const void* cache,
                                     const int32_t* block_table, const int32_t* cu_q, const int32_t* kv_len, void* workspace, void* out,
                                     float* lse, void* stream) {
  const char* who = "itexhip_kv4_attention";
  if (const int st = check(who, p, c)) return st;
  if (p->num_seqs == 0 || p->max_q_len == 0 || p->total_q == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(q != nullptr && cache != nullptr && cu_q != nullptr && kv_len != nullptr && workspace != nullptr && out != nullptr &&
                  (block_table != nullptr || p->table_stride == 0), "%s: null array", who);
  const size_t esize = p->type == ITEXHIP_FLOAT ? 4 : 2;
  ITEXHIP_REQUIRE(aligned(q, esize) && aligned(out, esize) && aligned(cache, 16) && aligned(workspace, 16) && aligned(block_table, 4) &&
                  aligned(cu_q, 4) && aligned(kv_len, 4) && aligned(lse, 4), "%s: an array is not aligned to its elements (cache and workspace to 16 bytes)", who);
  const Plan plan = plan_of(p, c);
  AttArgs A = {};
  A.q = q;
  A.cache = static_cast<const uint8_t*>(cache);
  A.table = block_table;
  A.cu_q = cu_q;
  A.kv_len = kv_len;
  A.out = out;
  A.lse = lse;
  char* w = static_cast<char*>(workspace);
  A.prefix = reinterpret_cast<int64_t*>(w);
  A.part_ml = reinterpret_cast<float*>(w + plan.prefix);
  A.part_o = reinterpret_cast<float*>(w + plan.prefix + plan.ml);
  A.table_stride = p->table_stride;
  A.total_q = p->total_q;
  A.page_bytes = itexhip_kv4_page_bytes(c);
  A.num_pages = c->num_pages;
  A.q_st = p->q_strides[0]; A.q_sh = p->q_strides[1];
  A.o_st = p->out_strides[0]; A.o_sh = p->out_strides[1];
  A.scale = p->scale;
  A.q_heads = p->q_heads;
  A.kv_heads = c->kv_heads;
  A.group = p->q_heads / c->kv_heads;
  A.num_seqs = p->num_seqs;
  A.max_q_len = p->max_q_len;
  A.causal = p->causal != 0;
  A.window = p->window < 1 << 30 ? p->window : 1 << 30;  // no sequence is longer; positions from -2^30 on less this stay in 32 bits
  A.head_dim = c->head_dim;
  A.page_size = c->page_size;
  A.page_shift = log2_of(c->page_size);
  A.groups = static_cast<int>(plan.groups);
  A.vec = aligned(out, 4 * esize) && A.o_st % 4 == 0 && A.o_sh % 4 == 0;
  if (p->type == ITEXHIP_FLOAT) launch_dims<ITEXHIP_FLOAT>(A, plan, as_stream(stream));
  else if (p->type == ITEXHIP_BFLOAT16) launch_dims<ITEXHIP_BFLOAT16>(A, plan, as_stream(stream));
  else launch_dims<ITEXHIP_HALF>(A, plan, as_stream(stream));
  ITEXHIP_CHECK_LAUNCH(who);
  return ITEXHIP_OK;
}
