// Attention over the paged 4-bit cache.
#include <math.h>

#include "common.hpp"
#include "kv4.hpp"

namespace itexhip {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;             // tokens a workgroup takes at a time, 32 a wavefront
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kProbExponent = 14.0f; // probabilities are held as 2^14 p: half keeps 11 bits of them down to 2^-28

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
  int q_heads, kv_heads, group, num_seqs, max_q_len, causal, window, head_dim, page_size, page_shift, vec;
};

// One sequence's rows and tokens, whatever the arrays say
struct Seq {
  int64_t first;   // row of q
  int n, len, lo;  // new tokens, tokens, first token that any row sees (multiple of 32)
  int64_t steps;   // of kStep tokens; at least one if there are rows
};
__device__ __forceinline__ Seq sequence(const AttArgs& A, int b) {
  Seq s;
  int64_t from = A.cu_q[b], to = A.cu_q[b + 1];
  from = from < 0 ? 0 : from > A.total_q ? A.total_q : from;
  to = to < from ? from : to > A.total_q ? A.total_q : to;
  s.first = from;
  s.n = static_cast<int>(to - from < A.max_q_len ? to - from : A.max_q_len);
  const int64_t room = A.table_stride << A.page_shift;
  int64_t len = A.kv_len[b];
  s.len = static_cast<int>(len < 0 ? 0 : len > room ? room : len);
  int64_t lo = A.window > 0 ? static_cast<int64_t>(s.len) - s.n - A.window + 1 : 0;
  s.lo = static_cast<int>(lo < 0 ? 0 : lo) & ~31;
  s.steps = s.n == 0 ? 0 : s.len > s.lo ? (s.len - s.lo + kStep - 1) / kStep : 1;
  return s;
}

__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t a, uint32_t o) { return (x & a) | o; }
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

// What a lane loads of 32 tokens (two tiles of 16, each in one page): lane = 16 g + c.
//   keys      token c of a tile, dwords g NKK .. g NKK + NKK - 1 of its row
//   values    tokens 4 g .. 4 g + 3 of a tile, dword c (and c + 16; a half of dword c / 2 if a head has 8 of them)
//   params    of tokens 4 g .. 4 g + 3: four scales, four offsets
template <int DP>
struct Raw {
  static constexpr int NKK = DP / 32, NV = DP <= 128 ? 1 : 2;
  uint32_t k[2][NKK];
  u4v v[2][NV], kp[2], vp[2];
  bool ok[2];
};

// A wavefront's 16 NB rows against 32 tokens at a time, everything in registers.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds, for its query column c, the scores of tokens 4 g .. 4 g + 3
// of each tile, which is the layout that the second product O^T = V^T P^T takes as its operand, so probabilities never
// leave the lane.  (The order of the 32 tokens within that product is the same on both sides and otherwise free.)
//
// Codes become operands without conversions.  A code c in the low bits of a half whose exponent is that of 1024 is the
// number 1024 + c, four bits further up with the exponent of 64 it is 64 + c: one and-or for two codes.  For keys the excess is
// taken back once a column (corr, the product's initial value) and scale and offset of a token are applied to its score:
// q . k = scale (q . code) + offset sum(q).  For values the excess is subtracted (exactly) and scale and offset applied in
// packed half arithmetic: long averages of values would otherwise cancel against the excess.
//
// Queries are multiplied by a power of two of their row so that half holds what bfloat16 does.  In fp32 the products are
// fp32 MFMAs on fp32 operands.
template <int T, int DP, int NB>
struct Engine {
  static constexpr bool F32 = T == ITEXHIP_FLOAT;
  static constexpr int NKK = DP / 32, E = DP / 16, NV = Raw<DP>::NV;
  half8v q16[F32 ? 1 : NB][NKK];
  float q32[F32 ? NB : 1][NKK][8];
  float corr[NB], sumq[NB], qs[NB], m[NB], l[NB];
  int limit[NB], start[NB];  // the tokens that column c of block nb sees: start <= t < limit
  f4 o[NB][E];
  int min_limit, max_start;  // over the wavefront's rows
  int lane, c, g;

  __device__ __forceinline__ void init(const AttArgs& A, const Seq& s, int kv_head, int row0) {
    lane = threadIdx.x & 63;
    c = lane & 15;
    g = lane >> 4;
    const int rows = s.n * A.group;
    auto sees = [&](int row, int* from, int* to) {
      const int pos = s.len - s.n + row / A.group;
      *to = A.causal ? (pos + 1 < 0 ? 0 : pos + 1) : s.len;
      *from = A.window > 0 && pos - A.window + 1 > 0 ? pos - A.window + 1 : 0;
    };
    int unused;
    sees(row0, &unused, &min_limit);
    const int last = row0 + 16 * NB - 1;
    sees(last < rows ? last : rows - 1, &max_start, &unused);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + nb * 16 + c;
      const bool in = row < rows;
      limit[nb] = start[nb] = 0;
      if (in) sees(row, &start[nb], &limit[nb]);
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
            excess += f * ((j & 1) ? 72.0f : 1032.0f);
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            q32[nb][kk][j] = x[kk][j];
            sum += x[kk][j];
          }
        }
        excess = 8.0f * sum;
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      excess += __shfl_xor(excess, 16);
      excess += __shfl_xor(excess, 32);
      sumq[nb] = sum;
      corr[nb] = -excess;
      qs[nb] = fmaxf(A.scale * kLog2e * back, 1.2e-38f);
      m[nb] = -INFINITY;
      l[nb] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[nb][e] = f4{0, 0, 0, 0};
    }
  }

  // Loads of the tiles at t0 and t0 + 16; a tile that ends before `from` or starts at `to` or beyond, or has no page, is not ok and holds zeros
  __device__ __forceinline__ void load(const AttArgs& A, const int32_t* table, int kv_head, int t0, int to, Raw<DP>& r) const {
    const Kv4Block block{A.page_size, DP};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = t0 + 16 * i;
      int page = t < to ? table[t >> A.page_shift] : -1;
      page = __builtin_amdgcn_readfirstlane(page);
      r.ok[i] = page >= 0 && page < A.num_pages;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) r.k[i][kk] = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) r.v[i][j] = u4v{0, 0, 0, 0};
      r.kp[i] = r.vp[i] = u4v{0, 0, 0, 0};
      if (r.ok[i]) {
        const uint8_t* base = A.cache + page * A.page_bytes + static_cast<int64_t>(kv_head) * block.bytes();
        const int place = t & (A.page_size - 1);
        const uint8_t* kr = base + block.key_codes(place + c) + g * (DP / 8);
        if constexpr (NKK == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(kr);
          r.k[i][0] = w.x;
          r.k[i][1] = w.y;
        } else {
#pragma unroll
          for (int j = 0; j < NKK / 4; ++j) {
            const u4v w = *reinterpret_cast<const u4v*>(kr + 16 * j);
#pragma unroll
            for (int n = 0; n < 4; ++n) r.k[i][4 * j + n] = w[n];
          }
        }
        const uint8_t* vr = base + block.value_codes(place + 4 * g, DP == 64 ? c / 2 : c);
#pragma unroll
        for (int j = 0; j < NV; ++j) r.v[i][j] = *reinterpret_cast<const u4v*>(vr + 256 * j);
        r.kp[i] = *reinterpret_cast<const u4v*>(base + block.key_params(place + 4 * g));
        r.vp[i] = *reinterpret_cast<const u4v*>(base + block.value_params(place + 4 * g));
      }
    }
  }

  __device__ __forceinline__ half8v key_operand(uint32_t w) const {
    const uint32_t v = w >> 8;
    const u4v u = {and_or(w, 0x000f000fu, 0x64006400u), and_or(w, 0x00f000f0u, 0x54005400u), and_or(v, 0x000f000fu, 0x64006400u),
                   and_or(v, 0x00f000f0u, 0x54005400u)};
    half8v h;
    __builtin_memcpy(&h, &u, 16);
    return h;
  }

  // The scores of a column become probabilities (times 2^14), the sums so far are rescaled where the maximum has grown
  __device__ __forceinline__ void softmax(int nb, float (&x)[8]) {
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__any(top > m[nb])) {
      const float now = fmaxf(m[nb], top);
      const float a = now == m[nb] ? 1.0f : __builtin_amdgcn_exp2f((m[nb] - now) * qs[nb]);
      m[nb] = now;
      l[nb] *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) o[nb][e] *= a;
    }
    const float ref = kProbExponent - (m[nb] == -INFINITY ? 0.0f : m[nb] * qs[nb]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], qs[nb], ref));
      l[nb] += x[j];
    }
  }

  __device__ __forceinline__ void step(const Raw<DP>& r, int t0) {
    const bool mask = !(r.ok[0] && r.ok[1] && t0 + 32 <= min_limit && t0 >= max_start);
    u4v vp[2] = {r.vp[0], r.vp[1]};
    uint32_t nan = 0;  // bit 4 i + j: the value of token 4 g + j of tile i is NaN and only some rows may see it
    if (mask) {
      // tokens beyond the last one hold whatever memory held: their values must not reach a product, not even times zero
      const int last = limit_of_wave();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t keep = (j & 1) ? 0x0000ffffu : 0xffff0000u;
          const uint32_t sc = (vp[i][j / 2] >> (16 * (j & 1))) & 0x7fffu, of = (vp[i][2 + j / 2] >> (16 * (j & 1))) & 0x7fffu;
          const bool beyond = t0 + 16 * i + 4 * g + j >= last;
          if (beyond || sc >= 0x7c00u || of >= 0x7c00u) {
            if (!beyond) nan |= 1u << (4 * i + j);
            vp[i][j / 2] &= keep;
            vp[i][2 + j / 2] &= keep;
          }
        }
      }
    }
    float p[NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f4 s = f4{corr[nb], corr[nb], corr[nb], corr[nb]};
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          if constexpr (!F32) {
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_operand(r.k[i][kk]), q16[nb][kk], s, 0, 0, 0);
          } else {
#pragma unroll
            for (int n = 0; n < 8; ++n)
              s = __builtin_amdgcn_mfma_f32_16x16x4f32(static_cast<float>((r.k[i][kk] >> (4 * n)) & 15u), q32[nb][kk][n], s, 0, 0, 0);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sc = r.kp[i][j / 2], of = r.kp[i][2 + j / 2];
          const float ks = (j & 1) ? high_half(sc) : low_half(sc), ko = (j & 1) ? high_half(of) : low_half(of);
          float x = fmaf(ks, s[j], ko * sumq[nb]);
          if (mask) {
            const int t = t0 + 16 * i + 4 * g + j;
            const bool seen = r.ok[i] && t < limit[nb] && t >= start[nb];
            x = seen ? x : -INFINITY;
            if (seen && (nan >> (4 * i + j) & 1)) l[nb] = NAN;
          }
          p[nb][4 * i + j] = x;
        }
      }
      softmax(nb, p[nb]);
    }
    if constexpr (!F32) {
      half8v pb[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[nb][j] = static_cast<_Float16>(p[nb][j]);
      }
      // a lane's eight tokens of one dimension, two a register: first the halves of two tokens' dwords that hold its code
#pragma unroll
      for (int part = 0; part < E / 4; ++part) {  // four dimensions each: a half of a dword
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u4v& d = r.v[i][part / 2 % NV];
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
            half2v h = (n & 1) ? as_half2(and_or(x, 0x00f000f0u, 0x54005400u)) + half2v{-72, -72}
                               : as_half2(and_or(x, 0x000f000fu, 0x64006400u)) + half2v{-1032, -1032};
            h = __builtin_elementwise_fma(h, as_half2(vp[k / 2][k & 1]), as_half2(vp[k / 2][2 + (k & 1)]));
            a[k] = as_bits(h);
          }
          half8v v;
          __builtin_memcpy(&v, &a, 16);
          const int e = part * 4 + n;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[nb], o[nb][e], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sc = vp[i][j / 2], of = vp[i][2 + j / 2];
          const float vs = (j & 1) ? high_half(sc) : low_half(sc), vo = (j & 1) ? high_half(of) : low_half(of);
          const float low = fmaf(-8.0f, vs, vo);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const uint32_t d = r.v[i][e / 8][j];
            const uint32_t code = DP == 64 ? (d >> (16 * (c & 1) + 4 * e)) & 15u : (d >> (4 * (e & 7))) & 15u;
            const float v = fmaf(static_cast<float>(code), vs, low);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[nb][4 * i + j], o[nb][e], 0, 0, 0);
          }
        }
      }
    }
  }

  int seq_len;  // tokens of the sequence
  __device__ __forceinline__ int limit_of_wave() const { return seq_len; }

  // the first of the four or eight dimensions that o[..][e][r], e = 0 .. 3 (+ 4), belong to
  __device__ __forceinline__ int dim_of(int e, int r) const {
    return DP == 64 ? 4 * (4 * g + r) + e : 8 * (4 * g + r) + (e & 7) + 128 * (e >> 3);
  }

  __device__ __forceinline__ void sum_l() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      l[nb] += __shfl_xor(l[nb], 16);
      l[nb] += __shfl_xor(l[nb], 32);
    }
  }

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
        A.lse[q_row * A.q_heads + head] = empty ? -INFINITY : kLn2 * (top[nb] - kProbExponent + log2f(sum[nb]));
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

// Rows of every sequence fit one tile of 16 NB: the tokens are what is divided.  The steps of all sequences and kv heads in a
// row, [sequence][kv head][step], are cut into equal shares, one a workgroup, whatever the lengths are and without the host
// knowing them.  A share may end one (sequence, head), hold several whole ones and begin another: whole ones are written out,
// the two at its ends leave their sums in the workspace for combine_kernel.
template <int T, int DP, int NB>
__global__ __launch_bounds__(256) void split_kernel(const AttArgs A) {
  __shared__ int64_t scan[5];
  __shared__ int64_t found[2];
  __shared__ float lds_ml[4][2][16 * NB];
  __shared__ float lds_o[2][NB * (DP / 16) * 4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  // steps of all sequences, then the sequence in which this workgroup's share begins
  auto prefix_of = [&](int base, int64_t& inclusive, int64_t& all) {
    const int b = base + tid;
    int64_t x = b < A.num_seqs ? sequence(A, b).steps * A.kv_heads : 0;
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
  int64_t total = 0, inclusive, all;
  for (int base = 0; base < A.num_seqs; base += 256) {
    prefix_of(base, inclusive, all);
    total += all;
  }
  const int64_t share = (total + gridDim.x - 1) / gridDim.x;
  const int64_t begin = share * blockIdx.x, end = begin + share < total ? begin + share : total;
  if (tid == 0) found[0] = -1;
  int64_t before = 0;
  for (int base = 0; base < A.num_seqs; base += 256) {
    if (base > 0 || A.num_seqs > 256) prefix_of(base, inclusive, all);
    const int b = base + tid;
    __syncthreads();
    if (b < A.num_seqs) {
      const int64_t mine = sequence(A, b).steps * A.kv_heads, from = before + inclusive - mine;
      if (begin >= from && begin < from + mine) {
        found[0] = b;
        found[1] = from;
      }
      if (blockIdx.x == 0) A.prefix[b] = from;
    }
    before += all;
  }
  if (blockIdx.x == 0 && tid == 0) A.prefix[A.num_seqs] = share;
  __syncthreads();
  if (begin >= end) return;
  int b = static_cast<int>(found[0]);
  int64_t from = found[1];

  for (int64_t at = begin; at < end;) {
    const Seq s = sequence(A, b);
    if (s.steps == 0) {
      ++b;
      continue;
    }
    const int64_t rel = at - from;
    const int head = static_cast<int>(rel / s.steps);
    const int64_t s0 = rel - head * s.steps, left = s.steps - s0, n = left < end - at ? left : end - at;
    const bool whole = n == s.steps;

    Engine<T, DP, NB> eng;
    eng.init(A, s, head, 0);
    eng.seq_len = s.len;
    const int32_t* table = A.table + b * A.table_stride;
    const int t_begin = s.lo + static_cast<int>(s0) * kStep + 32 * wave;
    Raw<DP> now, next;
    eng.load(A, table, head, t_begin, s.len, now);
    for (int i = 0; i < static_cast<int>(n); ++i) {
      const int t = t_begin + i * kStep;
      if (t >= s.len) break;
      if (i + 1 < n) eng.load(A, table, head, t + kStep, s.len, next);
      eng.step(now, t);
      now = next;
    }
    eng.sum_l();

    // the four wavefronts' sums into those of the first
    float top[NB], sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (eng.g == 0) {
        lds_ml[wave][0][nb * 16 + eng.c] = eng.m[nb] == -INFINITY ? -INFINITY : eng.m[nb] * eng.qs[nb];
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
        eng.finish(A, s, head, 0, top, sum);
      } else {
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s0 == 0 ? 1 : 0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int row = nb * 16 + eng.c;
          if (row >= s.n * A.group) continue;
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
    if (rel + n == s.steps * A.kv_heads) {
      ++b;
      from = at;
    }
  }
}

// One row of a (sequence, kv head) that several workgroups shared: their sums, in the order of the tokens
template <int T, int DP, int NB>
__global__ __launch_bounds__(256) void combine_kernel(const AttArgs A) {
  __shared__ float lds_o[256 / (DP / 4)][DP];
  __shared__ float lds_l[256 / (DP / 4)];
  const int b = blockIdx.z, head = blockIdx.y, row = blockIdx.x;
  const Seq s = sequence(A, b);
  if (row >= s.n * A.group) return;
  const int64_t share = A.prefix[A.num_seqs], i0 = A.prefix[b] + head * s.steps;
  const int64_t w0 = i0 / share, w1 = (i0 + s.steps - 1) / share;
  if (w0 == w1) return;
  const int count = static_cast<int>(w1 - w0 + 1);
  auto at = [&](int i) { return (2 * (w0 + i) + (i == 0 ? 1 : 0)) * 16 * NB + row; };
  constexpr int LANES = DP / 4, PARTS = 256 / LANES;
  const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  float top = -INFINITY;
  for (int i = 0; i < count; ++i) top = fmaxf(top, A.part_ml[at(i) * 2]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  f4 o = {0, 0, 0, 0};
  for (int i = part; i < count; i += PARTS) {
    const int64_t k = at(i);
    const float w = __builtin_amdgcn_exp2f(A.part_ml[k * 2] - ref);
    sum += A.part_ml[k * 2 + 1] * w;
    o += *reinterpret_cast<const f4*>(A.part_o + k * DP + 4 * lane) * w;
  }
  *reinterpret_cast<f4*>(&lds_o[part][4 * lane]) = o;
  if (lane == 0) lds_l[part] = sum;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) {
    o += *reinterpret_cast<const f4*>(&lds_o[i][4 * lane]);
    sum += lds_l[i];
  }
  const int q_head = head * A.group + row % A.group;
  const int64_t q_row = s.first + row / A.group;
  const bool empty = sum == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / sum;
  if (lane == 0 && A.lse != nullptr) A.lse[q_row * A.q_heads + q_head] = empty ? -INFINITY : kLn2 * (top - kProbExponent + log2f(sum));
  if (4 * lane >= A.head_dim) return;
  const int64_t to = q_row * A.o_st + q_head * A.o_sh + 4 * lane;
#pragma unroll
  for (int j = 0; j < 4; ++j) store_output<T>(A.out, to + j, o[j] * inv);
}

// Sequences of more rows: a wavefront takes 16 NB rows through all the tokens that they see
template <int T, int DP, int NB>
__global__ __launch_bounds__(256) void rows_kernel(const AttArgs A) {
  const int wave = threadIdx.x >> 6, b = blockIdx.z, head = blockIdx.y;
  const Seq s = sequence(A, b);
  const int rows = s.n * A.group, row0 = (static_cast<int>(blockIdx.x) * 4 + wave) * 16 * NB;
  if (row0 >= rows) return;
  Engine<T, DP, NB> eng;
  eng.init(A, s, head, row0);
  eng.seq_len = s.len;
  const int first = row0 / A.group, last = (row0 + 16 * NB < rows ? row0 + 16 * NB - 1 : rows - 1) / A.group;
  int to = s.len, from = s.lo;
  if (A.causal) {
    to = s.len - s.n + last + 1;
    to = to < 0 ? 0 : to;
  }
  if (A.window > 0) {
    from = s.len - s.n + first - A.window + 1;
    from = (from < 0 ? 0 : from) & ~31;
  }
  const int32_t* table = A.table + b * A.table_stride;
  Raw<DP> now, next;
  if (from < to) eng.load(A, table, head, from, to, now);
  for (int t = from; t < to; t += 32) {
    if (t + 32 < to) eng.load(A, table, head, t + 32, to, next);
    eng.step(now, t);
    now = next;
  }
  eng.sum_l();
  float top[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) top[nb] = eng.m[nb] == -INFINITY ? -INFINITY : eng.m[nb] * eng.qs[nb];
  eng.finish(A, s, head, row0, top, eng.l);
}

// ---------------------------------------------------------------------------------------------------------------------
struct Plan {
  int blocks;      // NB
  bool split;
  int64_t groups;  // workgroups of the split kernel
  size_t prefix, ml, o, bytes;
};

Plan plan_of(const itexhip_kv4_attention_params* p, const itexhip_kv4_cache* c) {
  Plan plan = {};
  const int dp = kv4_padded(c->head_dim);
  const int64_t rows = static_cast<int64_t>(p->max_q_len) * (p->q_heads / c->kv_heads);
  const int most = dp == 256 ? 1 : p->type == ITEXHIP_FLOAT ? 2 : 4;
  plan.blocks = rows <= 16 || most == 1 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
  plan.split = rows <= 16 * plan.blocks;
  if (plan.split) {
    const int64_t bound = static_cast<int64_t>(p->num_seqs) * c->kv_heads * ((p->table_stride * c->page_size + kStep - 1) / kStep);
    const int64_t full = plan.blocks == 1 ? 1024 : 512;
    plan.groups = bound < 1 ? 1 : bound < full ? bound : full;
    plan.prefix = (static_cast<size_t>(p->num_seqs) + 1) * 8 + 15 & ~size_t{15};
    plan.ml = static_cast<size_t>(plan.groups) * 2 * 16 * plan.blocks * 2 * 4;
    plan.o = static_cast<size_t>(plan.groups) * 2 * 16 * plan.blocks * dp * 4;
  }
  plan.bytes = plan.prefix + plan.ml + plan.o + 16;
  return plan;
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
  ITEXHIP_REQUIRE(p->max_q_len >= 0 && static_cast<int64_t>(p->max_q_len) * (p->q_heads / c->kv_heads) < (1ll << 30),
                  "%s: max_q_len times the heads of a kv head is 0 to 2^30", who);
  ITEXHIP_REQUIRE(p->total_q >= 0 && p->total_q < (1ll << 31), "%s: total_q is 0 to 2^31 - 1", who);
  ITEXHIP_REQUIRE(p->scale > 0.0f && isfinite(p->scale), "%s: scale is finite and positive", who);
  ITEXHIP_REQUIRE(p->window >= 0, "%s: window is not negative", who);
  ITEXHIP_REQUIRE(p->table_stride >= 0 && p->table_stride * c->page_size <= (1ll << 30), "%s: table_stride times page_size is 0 to 2^30", who);
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
    split_kernel<T, DP, NB><<<dim3(static_cast<unsigned>(plan.groups)), dim3(256), 0, stream>>>(A);
    if (plan.groups > 1) combine_kernel<T, DP, NB><<<dim3(rows, A.kv_heads, A.num_seqs), dim3(256), 0, stream>>>(A);
  } else {
    rows_kernel<T, DP, NB><<<dim3((rows + 64 * NB - 1) / (64 * NB), A.kv_heads, A.num_seqs), dim3(256), 0, stream>>>(A);
  }
}
template <int T, int DP>
void launch_blocks(const AttArgs& A, const Plan& plan, hipStream_t stream) {
  if (plan.blocks == 1) launch<T, DP, 1>(A, plan, stream);
  else if (plan.blocks == 2) { if constexpr (DP != 256) launch<T, DP, 2>(A, plan, stream); }
  else if constexpr (T != ITEXHIP_FLOAT && DP != 256) launch<T, DP, 4>(A, plan, stream);
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
  return static_cast<int64_t>(plan_of(p, c).bytes);
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
  A.window = p->window;
  A.head_dim = c->head_dim;
  A.page_size = c->page_size;
  A.page_shift = log2_of(c->page_size);
  A.vec = aligned(out, 4 * esize) && A.o_st % 4 == 0 && A.o_sh % 4 == 0;
  if (p->type == ITEXHIP_FLOAT) launch_dims<ITEXHIP_FLOAT>(A, plan, as_stream(stream));
  else if (p->type == ITEXHIP_BFLOAT16) launch_dims<ITEXHIP_BFLOAT16>(A, plan, as_stream(stream));
  else launch_dims<ITEXHIP_HALF>(A, plan, as_stream(stream));
  ITEXHIP_CHECK_LAUNCH(who);
  return ITEXHIP_OK;
}
