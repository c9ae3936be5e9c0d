// A router's choice of experts, and the order of rows by what they chose.
#include <math.h>

#include "chosen.hpp"

namespace itexhip {
namespace {

// ------------------------------------------------------------------------------------------------
// Router.  LPT lanes hold a token's ranks in 64 bits, PER consecutive experts each, so that LPT = 16 lets a wavefront choose for
// four tokens at once.  What is chosen or left out becomes NaN, which neither a maximum nor an equality sees: top_k rounds of
// one maximum over the lanes and the lowest expert that equals it.  8192 tokens, 8 of 256 experts in groups, logistic scores (fp32): 14 us for 8 MB, bound
// by vector instructions, 1700 of a wavefront: 500 for the scores, 140 a round.
// ------------------------------------------------------------------------------------------------
struct RouteArgs {
  itexhip_route_params p;
  const void* logits;
  const float* bias;
  int32_t* experts;
  float* weights;
  int64_t tokens, first;  // first: workgroup of the launch
};

// Over a token's lanes.  Lanes 1, 2, 4 and 8 apart meet within the vector unit; of a mirrored row any lane of the other half will
// do, since its half agrees by then.
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
template <int LPT, class V, class F>
__device__ __forceinline__ V over_lanes(V x, F&& f) {
  static_assert(LPT == 16 || LPT == 64, "lanes a token");
  x = f(x, from_lane<0xb1>(x));    // quad_perm 1 0 3 2
  x = f(x, from_lane<0x4e>(x));    // quad_perm 2 3 0 1
  x = f(x, from_lane<0x141>(x));   // row_half_mirror
  x = f(x, from_lane<0x140>(x));   // row_mirror
  if constexpr (LPT > 16) {
    x = f(x, __shfl_xor(x, 16));
    x = f(x, __shfl_xor(x, 32));
  }
  return x;
}

// e^x to about 2^-52: n ln 2 taken off with ln 2 in two parts, so that |r| <= ln 2 / 2, and the Taylor sum of e^r (the first term left
// out is r^14 / 14! < 5e-18).  Below 2^-1074 it is 0, beyond 2^1024 infinite; NaN stays.
__device__ __forceinline__ double exp64(double x) {
  x = x < -800.0 ? -800.0 : x > 800.0 ? 800.0 : x;
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0x1.62e42fefa38p-1, x);
  r = fma(n, -0x1.ef35793c7673p-45, r);
  double p = fma(r, 1.0 / 6227020800.0, 1.0 / 479001600.0);
  p = fma(r, p, 1.0 / 39916800.0);
  p = fma(r, p, 1.0 / 3628800.0);
  p = fma(r, p, 1.0 / 362880.0);
  p = fma(r, p, 1.0 / 40320.0);
  p = fma(r, p, 1.0 / 5040.0);
  p = fma(r, p, 1.0 / 720.0);
  p = fma(r, p, 1.0 / 120.0);
  p = fma(r, p, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return ldexp(p, static_cast<int>(n));
}
// 1 / (1 + e^-x): the reciprocal instruction's value and two steps of Newton's iteration (the sum is 1 at least; infinite from 2^1024 on)
__device__ __forceinline__ double sigmoid(double x) {
  const double d = 1.0 + exp64(-x);
  double r = __builtin_amdgcn_rcp(d);
  r = fma(fma(-d, r, 1.0), r, r);
  r = fma(fma(-d, r, 1.0), r, r);
  return d > 1e308 ? 0.0 : r;
}
// x is not a number any more: its upper word decides that
__device__ __forceinline__ double spoiled_if(bool condition, double x) {
  uint32_t w[2];
  __builtin_memcpy(w, &x, 8);
  w[1] = condition ? 0x7ff80000u : w[1];
  __builtin_memcpy(&x, w, 8);
  return x;
}

// VEC: a lane's logits are aligned to 16 bytes and there are as many as it can hold, or none
template <int T, int LPT, int PER, bool VEC>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs A) {
  constexpr int TOKENS = 256 / LPT;  // of a workgroup
  extern __shared__ __align__(16) uint8_t lds[];
  const int local = threadIdx.x / LPT, sub = threadIdx.x & (LPT - 1);
  const int64_t token = (A.first + blockIdx.x) * TOKENS + local;
  const bool live = token < A.tokens;
  const int E = A.p.experts, k = A.p.top_k;
  const bool softmax = A.p.score == ITEXHIP_ROUTE_SOFTMAX;
  const int64_t row = (live ? token : A.tokens - 1) * A.p.logits_stride;
  const double inf = __builtin_inf(), nan = __builtin_nan("");
  auto max_of = [](double a, double b) { return fmax(a, b); };
  auto sum_of = [](double a, double b) { return a + b; };

  double rank[PER];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < PER; i += 8) {
      float x[8];
      load8<T>(A.logits, row + min(sub * PER, E - PER) + i, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) rank[i + j] = sub * PER < E ? static_cast<double>(x[j]) : nan;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = sub * PER + i;
      const double x = load_value<T>(A.logits, row + min(e, E - 1));
      rank[i] = e < E ? x : nan;
    }
  }
  double top = 0.0, total = 1.0;
  if (softmax) {
    top = -inf;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = fmax(top, rank[i]);
    top = over_lanes<LPT>(top, max_of);
    if (top == -inf) top = 0.0;  // nothing but -infinity: scores of 0
    total = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double z = exp64(rank[i] - top);
      if (sub * PER + i < E) total += z;
      rank[i] = z;
    }
    total = over_lanes<LPT>(total, sum_of);
    total = total == 0.0 ? 1.0 : total;
    const double inv = 1.0 / total;
#pragma unroll
    for (int i = 0; i < PER; ++i) rank[i] = rank[i] * inv;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) rank[i] = sigmoid(rank[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = sub * PER + i;
    if (A.bias != nullptr && e < E) rank[i] += static_cast<double>(A.bias[e]);
    rank[i] = e >= E ? nan : rank[i] != rank[i] ? -inf : rank[i];
  }

  if (A.p.groups > 1) {
    const int G = A.p.groups, size = E / G;
    double* const ranks = reinterpret_cast<double*>(lds) + static_cast<size_t>(local) * (LPT * PER + 64);
    double* const values = ranks + LPT * PER;
    auto put = [&](int g, double best, double second) {
      const double value = A.p.group_best == 2 ? best + second : best;
      values[g] = value != value ? -inf : value;
    };
    auto take = [](double r, double& best, double& second) {
      second = fmax(second, fmin(best, r));
      best = fmax(best, r);
    };
    const int lanes = size / PER;  // of a group, where groups are whole lanes
    const bool whole = size % PER == 0 && (lanes & (lanes - 1)) == 0;
    if (whole) {
      double best = -inf, second = -inf;
#pragma unroll
      for (int i = 0; i < PER; ++i) take(rank[i], best, second);
      for (int d = 1; d < lanes; d *= 2) {
        const double b = __shfl_xor(best, d), s = __shfl_xor(second, d);
        second = fmax(fmin(best, b), fmax(second, s));
        best = fmax(best, b);
      }
      if (sub % lanes == 0 && sub * PER < E) put(sub / lanes, best, second);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) ranks[sub * PER + i] = rank[i];
      __syncthreads();
      for (int g = sub; g < G; g += LPT) {
        double best = -inf, second = -inf;
        for (int i = 0; i < size; ++i) take(ranks[g * size + i], best, second);
        put(g, best, second);
      }
    }
    __syncthreads();
    unsigned long long open = 0;  // groups that are left, the same in all of a token's lanes
    for (int g = sub; g < G; g += LPT) {
      int ahead = 0;
      for (int o = 0; o < G; ++o) ahead += values[o] > values[g] || (values[o] == values[g] && o < g);
      if (ahead < A.p.top_groups) open |= 1ull << g;
    }
    open = over_lanes<LPT>(open, [](unsigned long long a, unsigned long long b) { return a | b; });
    if (whole) {
      const bool shut = !((open >> min(sub / lanes, G - 1)) & 1);
#pragma unroll
      for (int i = 0; i < PER; ++i) rank[i] = spoiled_if(shut, rank[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int g = min(sub * PER + i, E - 1) / size;
        rank[i] = spoiled_if(!((open >> g) & 1), rank[i]);
      }
    }
  }

  // the j-th choice and its score stay with lane j % LPT, which has up to two (32 / LPT) of them
  constexpr int KEEP = 32 / LPT > 0 ? (32 + LPT - 1) / LPT : 1;
  int chosen[KEEP];
#pragma unroll
  for (int n = 0; n < KEEP; ++n) chosen[n] = 0;
  for (int j = 0; j < k; ++j) {
    double best = rank[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = fmax(best, rank[i]);
    best = over_lanes<LPT>(best, max_of);
    int id = 1 << 30;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i) id = rank[i] == best ? i : id;
    id += id < PER ? sub * PER : 0;
    id = over_lanes<LPT>(id, [](int a, int b) { return min(a, b); });
    const int mine = id - sub * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) rank[i] = spoiled_if(i == mine, rank[i]);
#pragma unroll
    for (int n = 0; n < KEEP; ++n)
      if (n * LPT + sub == j) chosen[n] = min(id, E - 1);
  }
  double score[KEEP], sum = 0.0;
#pragma unroll
  for (int n = 0; n < KEEP; ++n) {
    const double x = load_value<T>(A.logits, row + chosen[n]);
    score[n] = softmax ? exp64(x - top) / total : sigmoid(x);
    if (n * LPT + sub < k) sum += score[n];
  }
  sum = A.p.renormalise ? over_lanes<LPT>(sum, sum_of) : 1.0;
#pragma unroll
  for (int n = 0; n < KEEP; ++n) {
    const int j = n * LPT + sub;
    if (!live || j >= k) continue;
    A.experts[token * k + j] = chosen[n];
    A.weights[token * k + j] = static_cast<float>((sum == 0.0 ? 0.0 : score[n] / sum) * static_cast<double>(A.p.scale));
  }
}

template <int T, int LPT, int PER>
void launch_route(RouteArgs A, hipStream_t st) {
  constexpr int TOKENS = 256 / LPT;
  const bool vec = PER >= 8 && A.p.experts % PER == 0 && aligned(A.logits, 16) && (A.p.logits_stride * element_size(T)) % 16 == 0;
  const auto kernel = vec ? route_kernel<T, LPT, PER, PER >= 8> : route_kernel<T, LPT, PER, false>;
  const size_t lds = A.p.groups > 1 ? TOKENS * (LPT * PER + 64) * sizeof(double) : 0;
  launch_blocks((A.tokens + TOKENS - 1) / TOKENS, [&](int64_t first, unsigned count) {
    A.first = first;
    kernel<<<count, 256, lds, st>>>(A);
  });
}
template <int T>
void launch_route(const RouteArgs& A, hipStream_t st) {
  // Few tokens: more lanes each, whose instructions one after the other are what takes the time.  64 lanes : 16 lanes in us for 8 of 256 experts in groups, 64
  // tokens 7.5 : 9.8, 1024 7.9 : 10.0, 2048 8.5 : 10.2, 4096 11.5 : 10.3, 8192 18.7 : 13.8; 8 of 128 6.1 : 8.5, 6.4 : 8.7, 6.9 : 8.8, 9.4 : 8.9, 14.8 : 11.2;
  // so 64 lanes would be the shorter ones up to some 2048 tokens
  if (A.p.experts <= 64) launch_route<T, 16, 4>(A, st);
  else if (A.p.experts <= 256 && A.tokens <= 1024) launch_route<T, 64, 4>(A, st);
  else if (A.p.experts <= 256) launch_route<T, 16, 16>(A, st);
  else launch_route<T, 64, 16>(A, st);
}

// ------------------------------------------------------------------------------------------------
// Order of rows by group: a counting sort.  The rows are cut into runs, one a workgroup, whose wavefronts take consecutive shares.
// A first launch counts each run's groups; in the second a wavefront knows where its rows of a group begin: behind all smaller
// groups, the group's rows of earlier runs and those of the run's earlier wavefronts.  Rows of one group within 64 keep their
// order by their number among the lanes.  One workgroup does both where there are few rows.  65536 rows in 256 groups: 4 us to count, 12 to order, round
// trips for the runs' counts, the groups' sums and the rows one after the other; up to 1024 rows 2.5 to 4.
// ------------------------------------------------------------------------------------------------
constexpr int kOrderWaves = 4;
constexpr int kRunRows = 1024, kMostRuns = 256;
int runs_of(int64_t n) {
  const int64_t runs = (n + kRunRows - 1) / kRunRows;
  return static_cast<int>(runs < kMostRuns ? runs : kMostRuns);
}

__device__ __forceinline__ int key_of(const int32_t* group_of, int i, int groups) {
  const int g = group_of[i];
  return g < 0 || g >= groups ? groups : g;
}

// counts of each wavefront's share [begin, end) of the rows into LDS
__device__ __forceinline__ void count_share(const int32_t* group_of, int begin, int end, int groups, int* bins) {
  const int lane = threadIdx.x & 63;
  for (int g = lane; g <= groups; g += 64) bins[g] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int i = begin + lane; i < end; i += 64) atomicAdd(&bins[key_of(group_of, i, groups)], 1);
}

__global__ __launch_bounds__(64 * kOrderWaves) void count_rows_kernel(const int32_t* __restrict__ group_of, int n, int groups, int per_run,
                                                                      int32_t* __restrict__ counts) {
  extern __shared__ int bins[];
  const int wave = threadIdx.x >> 6, stride = groups + 1, share = (per_run + kOrderWaves - 1) / kOrderWaves;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_run;
  const int last = static_cast<int>(min(first + per_run, static_cast<int64_t>(n)));
  const int begin = static_cast<int>(min(first + static_cast<int64_t>(wave) * share, static_cast<int64_t>(last)));
  count_share(group_of, begin, min(begin + share, last), groups, bins + wave * stride);
  __syncthreads();
  for (int g = threadIdx.x; g <= groups; g += 64 * kOrderWaves) {
    int sum = 0;
    for (int w = 0; w < kOrderWaves; ++w) sum += bins[w * stride + g];
    counts[static_cast<int64_t>(blockIdx.x) * stride + g] = sum;
  }
}

// counts: of the runs, or null where there is but one
__global__ __launch_bounds__(64 * kOrderWaves) void order_rows_kernel(const int32_t* __restrict__ group_of, int n, int groups, int per_run,
                                                                      const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                                                                      int32_t* __restrict__ rows) {
  extern __shared__ int bins[];  // of the wavefronts, then the total of each group
  __shared__ int wave_sum[kOrderWaves];
  constexpr int THREADS = 64 * kOrderWaves;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, stride = groups + 1, share = (per_run + kOrderWaves - 1) / kOrderWaves;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_run;
  const int last = static_cast<int>(min(first + per_run, static_cast<int64_t>(n)));
  const int begin = static_cast<int>(min(first + static_cast<int64_t>(wave) * share, static_cast<int64_t>(last))), end = min(begin + share, last);
  int* const total = bins + kOrderWaves * stride;
  count_share(group_of, begin, end, groups, bins + wave * stride);
  __syncthreads();
  // each thread a run of groups: totals, where the groups begin, and from there where each wavefront's rows do
  const int each = (stride + THREADS - 1) / THREADS;
  const int g0 = min(static_cast<int>(threadIdx.x) * each, stride), g1 = min(g0 + each, stride);
  for (int g = threadIdx.x; g < stride; g += THREADS) {
    int all = 0, before = 0;
    if (counts != nullptr) {
      constexpr int AT_ONCE = 16;
      const int runs = gridDim.x, run = blockIdx.x;
      for (int r = 0; r < runs; r += AT_ONCE) {
        int c[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) c[i] = counts[static_cast<int64_t>(min(r + i, runs - 1)) * stride + g];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          all += r + i < runs ? c[i] : 0;
          before += r + i < run ? c[i] : 0;
        }
      }
    } else {
      for (int w = 0; w < kOrderWaves; ++w) all += bins[w * stride + g];
    }
    total[g] = all;
    int at = before;
    for (int w = 0; w < kOrderWaves; ++w) {
      const int c = bins[w * stride + g];
      bins[w * stride + g] = at;
      at += c;
    }
  }
  __syncthreads();
  int mine = 0;
  for (int g = g0; g < g1; ++g) mine += total[g];
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int below = __shfl_up(sum, d);
    if (lane >= d) sum += below;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int start = sum - mine;
  for (int w = 0; w < wave; ++w) start += wave_sum[w];
  for (int g = g0; g < g1; ++g) {
    if (blockIdx.x == 0) offsets[g] = start;  // offsets[groups]: where the rows of no group begin
    for (int w = 0; w < kOrderWaves; ++w) bins[w * stride + g] += start;
    start += total[g];
  }
  __syncthreads();
  int* const next = bins + wave * stride;
  int bits = 1;
  while ((1 << bits) <= groups) ++bits;
  for (int i0 = begin; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const bool there = i < end;
    const int key = there ? key_of(group_of, i, groups) : 0;
    unsigned long long same = __ballot(there);  // lanes with this lane's group
    for (int b = 0; b < bits; ++b) {
      const bool set = (key >> b) & 1;
      const unsigned long long with = __ballot(set);
      same &= set ? with : ~with;
    }
    const int ahead = __popcll(same & ((1ull << lane) - 1));
    const int at = there ? next[key] + ahead : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (there) {
      rows[at] = i;
      if (ahead == 0) next[key] = at + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

int check_groups(int64_t n, int groups) {
  ITEXHIP_REQUIRE(groups >= 1 && groups <= kMaxGroups, "itexhip_group_rows: 1 .. 1024 groups, got %d", groups);
  ITEXHIP_REQUIRE(n >= 0 && n < kMaxRows, "itexhip_group_rows: rows are 0 .. 2^30 - 1");
  return ITEXHIP_OK;
}

}  // namespace
}  // namespace itexhip

using namespace itexhip;

extern "C" int itexhip_route(const itexhip_route_params* p, int64_t tokens, const void* logits, const float* bias, int32_t* experts_out,
                             float* weights_out, void* stream) {
  ITEXHIP_REQUIRE(p != nullptr, "itexhip_route: null parameters");
  ITEXHIP_REQUIRE(is_chosen_type(p->type), "itexhip_route: the type is float, bfloat16 or half");
  ITEXHIP_REQUIRE(p->experts >= 1 && p->experts <= kMaxGroups, "itexhip_route: 1 .. 1024 experts, got %d", p->experts);
  ITEXHIP_REQUIRE(p->score == ITEXHIP_ROUTE_SOFTMAX || p->score == ITEXHIP_ROUTE_SIGMOID, "itexhip_route: score is softmax or sigmoid");
  ITEXHIP_REQUIRE(p->groups >= 1 && p->groups <= 64 && p->experts % p->groups == 0, "itexhip_route: 1 .. 64 groups of equally many experts");
  ITEXHIP_REQUIRE(p->top_groups >= 1 && p->top_groups <= p->groups, "itexhip_route: top_groups is 1 .. groups");
  const int size = p->experts / p->groups;
  ITEXHIP_REQUIRE(p->group_best == 1 || (p->group_best == 2 && size >= 2), "itexhip_route: group_best is 1, or 2 where groups have two experts");
  ITEXHIP_REQUIRE(p->top_k >= 1 && p->top_k <= 32 && p->top_k <= size * p->top_groups,
                  "itexhip_route: top_k is 1 .. 32 and no more than the experts of top_groups groups");
  ITEXHIP_REQUIRE(isfinite(p->scale), "itexhip_route: scale is finite");
  ITEXHIP_REQUIRE(tokens >= 0 && tokens < kMaxRows, "itexhip_route: tokens are 0 .. 2^30 - 1");
  ITEXHIP_REQUIRE(p->logits_stride >= 0 && p->logits_stride < (1LL << 31), "itexhip_route: bad logits_stride");
  if (tokens == 0) return ITEXHIP_OK;
  ITEXHIP_REQUIRE(logits && experts_out && weights_out, "itexhip_route: null buffer");
  ITEXHIP_REQUIRE(aligned(logits, element_size(p->type)) && aligned(bias, 4) && aligned(experts_out, 4) && aligned(weights_out, 4),
                  "itexhip_route: buffers are aligned to their elements");
  const RouteArgs A{*p, logits, bias, experts_out, weights_out, tokens, 0};
  hipStream_t st = as_stream(stream);
  if (p->type == ITEXHIP_FLOAT) launch_route<ITEXHIP_FLOAT>(A, st);
  else if (p->type == ITEXHIP_BFLOAT16) launch_route<ITEXHIP_BFLOAT16>(A, st);
  else launch_route<ITEXHIP_HALF>(A, st);
  ITEXHIP_CHECK_LAUNCH("itexhip_route");
  return ITEXHIP_OK;
}

extern "C" int64_t itexhip_group_rows_workspace(int64_t n, int groups) {
  if (check_groups(n, groups) != ITEXHIP_OK) return 0;
  return (static_cast<int64_t>(runs_of(n)) * (groups + 1) * 4 + 16 + 15) / 16 * 16;
}

extern "C" int itexhip_group_rows(int64_t n, int groups, const int32_t* group_of, int32_t* offsets_out, int32_t* rows_out, void* workspace,
                                  void* stream) {
  if (const int e = check_groups(n, groups)) return e;
  ITEXHIP_REQUIRE(offsets_out && (n == 0 || (group_of && rows_out && workspace)), "itexhip_group_rows: null buffer");
  ITEXHIP_REQUIRE(aligned(group_of, 4) && aligned(offsets_out, 4) && aligned(rows_out, 4) && aligned(workspace, 16),
                  "itexhip_group_rows: buffers are aligned to their elements, the workspace to 16 bytes");
  hipStream_t st = as_stream(stream);
  const int runs = n == 0 ? 1 : runs_of(n), per_run = n == 0 ? 1 : static_cast<int>((n + runs - 1) / runs);
  const size_t bins = static_cast<size_t>(groups + 1) * 4;
  int32_t* const counts = runs > 1 ? static_cast<int32_t*>(workspace) : nullptr;
  if (runs > 1)
    count_rows_kernel<<<runs, 64 * kOrderWaves, bins * kOrderWaves, st>>>(group_of, static_cast<int>(n), groups, per_run, counts);
  order_rows_kernel<<<runs, 64 * kOrderWaves, bins * (kOrderWaves + 1), st>>>(group_of, static_cast<int>(n), groups, per_run, counts, offsets_out,
                                                                               rows_out);
  ITEXHIP_CHECK_LAUNCH("itexhip_group_rows");
  return ITEXHIP_OK;
}
