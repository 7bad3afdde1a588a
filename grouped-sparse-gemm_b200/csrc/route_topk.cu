// Router logits to the top-k experts and weights that dispatch_plan and moe_finalize take.
//
//   score = softmax or sigmoid of the logits; experts are ranked by score + bias, or by the logit where there is no bias (the
//   scores rise with it), groups of neighbouring experts by the sum of their two best keys (their best one without a bias),
//   ties going to the lowest index; the weights are the scores of the chosen, over their sum if asked for, times a factor.
//
// A warp takes a token: its keys lie in registers as unsigned numbers that order like them, every round of the selection is
// two warp-wide integer reductions (largest key, lowest expert that has it).  Keys with a bias are sums of 32-bit roundings,
// so two that lie closer together than those can be off might come out in the wrong order: where a selected key is that
// close to the next one, the row is done again in 64 bits.  That is rare where keys differ (3 rows in 10000 of 256 experts, random
// float32 or bf16 logits and a random bias), but equal keys are as close as keys can be: bf16 logits with one bias for all make a third of
// the rows doubtful, saturated sigmoids all of them.
// Bound: issue slots for many rows (16384 x 128, top-8 of softmax: 10.7 us, 554 instructions a row, 77 % of the slots; 16384 x 256, top-8
// of sigmoid with bias, 29 us, from 4 of 8 groups 52, bf16 logits 59; those with a bias of zeros 111, all rows doubtful 120), latency of
// the reductions for few (64 x 256, the same with groups: 7.2 to 7.8 us, with a doubtful row among them 9.7, a third of them 16).  One
// kernel for all options, keys found anew every round, took 15.6 us for the first.
#include <algorithm>
#include <climits>

#include "common.cuh"

namespace pnv {
namespace {

constexpr int kWarps = 8;                // of a block
constexpr int kBlocks = 8;               // of an SM at most: further rows are walked over
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  const float* bias;             // or nullptr
  float* weights;
  int* ids;
  long long rows, stride;
  int experts, topk, groups, topk_groups, group_size;
  unsigned group_inv;            // ceil(2^20 / group_size)
  int bf16, sigmoid, renormalize;
  float scale;
};

__device__ __forceinline__ float logit_at(const RouteArgs& a, const void* row, int e) {
  return a.bf16 ? __uint_as_float((uint32_t)__ldg(static_cast<const unsigned short*>(row) + e) << 16)
                : __ldg(static_cast<const float*>(row) + e);
}

// Unsigned numbers that order like the keys; 0 stands for an expert that cannot be chosen, 1 for a NaN.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);                         // (-0 counts as 0)
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  if ((b & 0x7FFFFFFFFFFFFFFFull) > 0x7FF0000000000000ull) return 1ull;
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float key_of(uint32_t o) { return o == 1u ? -INFINITY : __uint_as_float((o >> 31) ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ double key_of(unsigned long long o) {
  return o == 1ull ? -INFINITY : __longlong_as_double((long long)((o >> 63) ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kAll, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}

__device__ __forceinline__ float sigmoid_of(float l) { return rcp_approx(1.f + ex2_approx(l * -kLog2e)); }
__device__ __forceinline__ double sigmoid_of(double l) { return 1.0 / (1.0 + exp(-l)); }
__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// exp(l - mx), 1 where the two are the same infinity, 0 everywhere in a row of nothing but -infinity; NaN where either is one.
template <class F>
__device__ __forceinline__ F softmax_part(F l, F mx) { return mx == (F)-INFINITY ? (F)0 : l == mx ? (F)1 : exp_of(l - mx); }

// The largest logit; a NaN where all scores of the row are to be NaN.  With a bias any NaN makes every key one, so that the choice
// is none.  Without one a NaN ranks last and does not count beside a number, but where nothing is above -infinity the row must not
// get the zeros of one that was masked.
template <bool kBias>
__device__ __forceinline__ float row_max(const RouteArgs& a, const void* row, int lane) {
  uint32_t m = 0;
  bool nan = false;
  for (int e = lane; e < a.experts; e += 32) {
    const float l = logit_at(a, row, e);
    nan |= isnan(l);
    m = max(m, order_of(l));
  }
  m = warp_max(m);
  if ((kBias || m <= order_of(-INFINITY)) && __any_sync(kAll, nan)) return __uint_as_float(0x7FFFFFFFu);
  return key_of(m);
}
// The largest of the chosen lanes' logits (none of them a NaN).
__device__ __forceinline__ float best_of(float logit, bool chosen) { return key_of(warp_max(chosen ? order_of(logit) : 0u)); }

template <class F>
__device__ __forceinline__ F softmax_sum(const RouteArgs& a, const void* row, int lane, F mx) {
  F sum = 0;
  for (int e = lane; e < a.experts; e += 32) sum += softmax_part((F)logit_at(a, row, e), mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  return sum;
}

// Two neighbouring keys, the larger one first, are too close for 32 bits to order where their difference is within what both can
// be off.  A sigmoid is off by 1.2e-7 (the largest of 2^31 values between -100 and 100 against 64 bits), a softmax by 1.5e-6 (its
// sum over 1024), the sum with the bias by half a unit, 6e-8 of the key; a group's sum of two keys by twice that, of either key,
// and half a unit of its own.  large: the largest magnitude among them.
__device__ __forceinline__ bool too_close(float larger, float smaller, float terms, float large, bool sigmoid) {
  return larger - smaller <= terms * (sigmoid ? fmaf(1.5e-7f, large, 3e-7f) : fmaf(3.8e-6f, large, 3.8e-6f));
}

// Lane r < topk returns expert r of the row, best first, and its key; logit[j] is that of expert 32 j + lane.  doubtful: (32 bits
// with a bias) the order is not certain.
template <class F, class O, int VPL, bool kBias, bool kGroups>
__device__ __forceinline__ int select(const RouteArgs& a, const void* row, const float (&logit)[VPL], int lane, O& picked_key, bool& doubtful) {
  constexpr bool kCheck = kBias && sizeof(F) == 4;
  O key[VPL];
  {
    F mx = 0, total = 1;
    if (kBias && !a.sigmoid) {
      mx = (F)row_max<kBias>(a, row, lane);
      total = softmax_sum<F>(a, row, lane, mx);
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = j * 32 + lane;
      key[j] = 0;
      if (e < a.experts) {
        F k = (F)logit[j];
        if (kBias) k = (a.sigmoid ? sigmoid_of(k) : softmax_part(k, mx) / total) + (F)__ldg(a.bias + e);
        key[j] = order_of(k);
      }
    }
  }
  doubtful = false;
  if constexpr (kGroups) {
    O mine = 0;                          // lane g: the score of group g
    int g = 0;
    float large = 0.f;                   // the largest magnitude of a group's best
    O first = 0, second = 0;             // this lane's two best of a group
    auto take = [&](O k) {
      if (kBias) second = max(second, min(first, k));
      first = max(first, k);
    };
    auto close_group = [&]() {
      const O best = warp_max(first);
      O score = best;
      if (kBias) {
        const int owner = __ffs(__ballot_sync(kAll, first == best)) - 1;
        const O next = warp_max(lane == owner ? second : first);
        score = next == 0 ? best : order_of(key_of(best) + key_of(next));
        if (kCheck && fabsf((float)key_of(best)) < INFINITY) large = fmaxf(large, fabsf((float)key_of(best)));
      }
      if (lane == g) mine = score;
      first = second = 0;
      ++g;
    };
    if (a.group_size % 32 == 0) {        // whole registers belong to a group
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        take(key[j]);
        if ((j + 1) * 32 % a.group_size == 0 && g < a.groups) close_group();
      }
    } else {
#pragma unroll 1
      while (g < a.groups) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) take((((unsigned)(j * 32 + lane) * a.group_inv) >> 20) == (unsigned)g ? key[j] : (O)0);
        close_group();
      }
    }
    unsigned kept = 0;
    F last = 0;
#pragma unroll 1
    for (int r = 0; r <= a.topk_groups && r < a.groups; ++r) {
      const O best = warp_max(mine);
      if (r == a.topk_groups) {          // (the order among the kept does not matter, only the border)
        if (kCheck) doubtful |= too_close((float)last, (float)key_of(best), 2.f, large + fabsf((float)last), a.sigmoid);
        break;
      }
      const int chosen = __ffs(__ballot_sync(kAll, mine == best && lane < a.groups)) - 1;
      last = key_of(best);
      kept |= 1u << chosen;
      if (lane == chosen) mine = 0;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const unsigned of = ((unsigned)(j * 32 + lane) * a.group_inv) >> 20;
      if (of >= 32 || !((kept >> of) & 1)) key[j] = 0;
    }
  }
  // Up to eight keys a lane are sorted first (equal ones in the order of their experts): a round then looks at one key a lane,
  // and the lane that had the best one moves up.
  constexpr bool kSorted = VPL <= 8;
  int expert[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) expert[j] = j * 32 + lane;
  if constexpr (kSorted) {
#pragma unroll
    for (int i = 1; i < VPL; ++i)
#pragma unroll
      for (int j = i; j > 0; --j) {
        const bool swap = key[j] > key[j - 1];
        const O hi = swap ? key[j] : key[j - 1], lo = swap ? key[j - 1] : key[j];
        const int he = swap ? expert[j] : expert[j - 1], le = swap ? expert[j - 1] : expert[j];
        key[j - 1] = hi; key[j] = lo;
        expert[j - 1] = he; expert[j] = le;
      }
  }
  int picked = 0;
  picked_key = 0;
  F last = 0;
  const int rounds = kCheck ? a.topk + 1 : a.topk;        // one more to see how close the next one is
#pragma unroll 1
  for (int r = 0; r < rounds; ++r) {
    O first = key[0];
    int mine = expert[0];
    if constexpr (!kSorted) {
#pragma unroll
      for (int j = 1; j < VPL; ++j)
        if (key[j] > first) { first = key[j]; mine = expert[j]; }
    }
    const O best = warp_max(first);
    if (kCheck && best == 0) break;      // (only the round beyond the last: there are topk experts to choose from)
    const unsigned with = __ballot_sync(kAll, first == best);
    int e = __shfl_sync(kAll, mine, __ffs(with) - 1);
    if (with & (with - 1)) e = __reduce_min_sync(kAll, first == best ? mine : INT_MAX);
    if constexpr (kSorted) {
      if (mine == e) {
#pragma unroll
        for (int j = 0; j + 1 < VPL; ++j) { key[j] = key[j + 1]; expert[j] = expert[j + 1]; }
        key[VPL - 1] = 0;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (expert[j] == e) key[j] = 0;
    }
    if (kCheck) {
      const F k = key_of(best);
      if (r > 0) doubtful |= too_close((float)last, (float)k, 1.f, fabsf((float)last), a.sigmoid);
      last = k;
    }
    if (lane == r) { picked = e; picked_key = best; }
  }
  return picked;
}

template <int VPL>
__device__ __forceinline__ void load_row(const RouteArgs& a, const void* row, int lane, float (&logit)[VPL]) {
#pragma unroll
  for (int j = 0; j < VPL; ++j) logit[j] = j * 32 + lane < a.experts ? logit_at(a, row, j * 32 + lane) : 0.f;
}

template <int VPL, bool kGroups>
__device__ __noinline__ int select_exactly(const RouteArgs& a, const void* row, int lane) {
  float logit[VPL];
  load_row(a, row, lane, logit);
  bool ignored;
  unsigned long long key;
  return select<double, unsigned long long, VPL, true, kGroups>(a, row, logit, lane, key, ignored);
}

template <int VPL, bool kBias, bool kGroups>
__global__ void __launch_bounds__(kWarps * 32)
route_topk_kernel(const RouteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * kWarps;
  const long long row_bytes = a.stride * (a.bf16 ? 2 : 4);
  long long t = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  float logit[VPL], next[VPL];
  if (t < a.rows) load_row(a, static_cast<const uint8_t*>(a.logits) + t * row_bytes, lane, next);
  for (; t < a.rows; t += step) {
    const uint8_t* row = static_cast<const uint8_t*>(a.logits) + t * row_bytes;
#pragma unroll
    for (int j = 0; j < VPL; ++j) logit[j] = next[j];
    if (t + step < a.rows) load_row(a, row + step * row_bytes, lane, next);
    bool doubtful;
    uint32_t key;
    int e = select<float, uint32_t, VPL, kBias, kGroups>(a, row, logit, lane, key, doubtful);
    if constexpr (kBias) {
      if (doubtful) e = select_exactly<VPL, kGroups>(a, row, lane);
    }
    float mine = 0.f;                    // the logit of this lane's choice: without a bias its key says it
    if (lane < a.topk) mine = kBias ? logit_at(a, row, e) : key == 1u ? __uint_as_float(0x7FFFFFFFu) : key_of(key);
    // Renormalized scores may be smaller than 32 bits go: the chosen are then put over the best of them.
    float w = 0.f;
    if (a.sigmoid) {
      constexpr float kSmall = -17.f;    // 1 + exp(l) is 1 in 32 bits below
      float over = 0.f;
      if (a.renormalize && !__any_sync(kAll, lane < a.topk && !(mine < kSmall))) {
        over = best_of(mine, lane < a.topk);
        if (over == -INFINITY) over = 0.f;
      }
      if (lane < a.topk) w = mine < kSmall ? expf(mine - over) : __fdiv_rn(1.f, 1.f + expf(-mine));
    } else {
      float mx = -INFINITY;              // without bias and groups the first choice has it, if it is a number
      if (!kBias && !kGroups) mx = __shfl_sync(kAll, mine, 0);
      if (kBias || kGroups || !(mx > -INFINITY)) mx = row_max<kBias>(a, row, lane);
      if (kBias && a.renormalize && mx < INFINITY) mx = best_of(mine, lane < a.topk);      // (a row's infinity leaves the others 0)
      if (lane < a.topk) w = softmax_part(mine, mx);
      if (!a.renormalize) {
        const float total = softmax_sum<float>(a, row, lane, mx);
        w = total > 0.f ? __fdiv_rn(w, total) : total;             // (a NaN stays one)
      }
    }
    if (a.renormalize) {
      float sum = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
      w = sum == 0.f ? 0.f : __fdiv_rn(w, sum);
    }
    if (lane < a.topk) {
      a.ids[t * a.topk + lane] = e;
      a.weights[t * a.topk + lane] = w * a.scale;
    }
  }
}

using RouteKernel = void (*)(const RouteArgs);
template <bool kBias, bool kGroups>
RouteKernel route_kernel(int vpl) {
  return vpl <= 1 ? route_topk_kernel<1, kBias, kGroups> : vpl <= 2 ? route_topk_kernel<2, kBias, kGroups>
       : vpl <= 4 ? route_topk_kernel<4, kBias, kGroups> : vpl <= 8 ? route_topk_kernel<8, kBias, kGroups>
       : vpl <= 16 ? route_topk_kernel<16, kBias, kGroups> : route_topk_kernel<32, kBias, kGroups>;
}

}  // namespace
}  // namespace pnv

using namespace pnv;

extern "C" int pnv_route_topk(const void* logits, int logits_are_bf16, int64_t stride, int64_t rows, int experts, int topk, int sigmoid,
                              const float* bias, int groups, int topk_groups, int renormalize, float scale, float* weights,
                              int32_t* ids, int sm_count, pnv_stream_t stream) {
  PNV_REQUIRE(rows >= 0 && rows < (1LL << 31), "bad row count");
  PNV_REQUIRE(experts >= 1 && experts <= PNV_ROUTE_MAX_EXPERTS, "route_topk: 1 to %d experts, got %d", PNV_ROUTE_MAX_EXPERTS, experts);
  PNV_REQUIRE(groups >= 1 && groups <= 32 && experts % groups == 0, "groups must divide the experts, at most 32, got %d", groups);
  PNV_REQUIRE(topk_groups >= 1 && topk_groups <= groups, "topk_groups must be in [1, groups], got %d", topk_groups);
  PNV_REQUIRE(topk >= 1 && topk <= 32 && topk <= experts / groups * topk_groups,
              "topk must be in [1, 32] and leave every choice an expert, got %d of %d", topk, experts / groups * topk_groups);
  if (rows == 0) return PNV_OK;
  PNV_REQUIRE(logits && weights && ids, "null pointer argument");
  PNV_REQUIRE(stride >= experts, "rows must not overlap");
  PNV_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (logits_are_bf16 ? 2 : 4) == 0 && reinterpret_cast<uintptr_t>(bias) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(weights) % 4 == 0 && reinterpret_cast<uintptr_t>(ids) % 4 == 0,
              "route_topk: a buffer is not aligned to its elements");
  const int group_size = experts / groups;
  // (e * ceil(2^20 / size)) >> 20 is e / size for e below 1024: the product is off by less than e / 2^20 < 1 / size)
  RouteArgs a{logits, bias, weights, (int*)ids, rows, stride, experts, topk, groups, topk_groups, group_size,
              (unsigned)(((1 << 20) + group_size - 1) / group_size), logits_are_bf16, sigmoid, renormalize, scale};
  const int vpl = ceil_div_i(experts, 32);
  const RouteKernel kernel = bias != nullptr ? groups > 1 ? route_kernel<true, true>(vpl) : route_kernel<true, false>(vpl)
                                             : groups > 1 ? route_kernel<false, true>(vpl) : route_kernel<false, false>(vpl);
  const long long blocks = std::min<long long>((rows + kWarps - 1) / kWarps, (long long)kBlocks * (sm_count > 0 ? sm_count : 148));
  PNV_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kWarps * 32), 0, (cudaStream_t)stream, pdl_enabled(), a));
  return PNV_OK;
}
