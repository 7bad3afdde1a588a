// Dense linear layers: out = act(x w^T + bias) + residual, or act(gate) * up + residual where the rows of w hold gates and
// ups in blocks of 32 (gated), on bf16 operands or on 8-bit codes with block scales (norm.cu says which).  The sum, the bias,
// the activation and the residual are fp32, rounded once on the way out.
//
// Two kernels.
//
//   split    one CTA per 128 weight rows x 16 to 128 tokens, weight rows along the tensor core's M: token tiles as narrow
//            as a decode step wants.  Where there are fewer tiles than SMs a cluster of up to eight CTAs shares a tile's K and
//            sends its partial sums to the CTAs that own their tokens by copies between their shared memories, which add them in a
//            fixed order: no workspace, no atomics.
//   pair     persistent; a CTA pair multiplies 256 tokens x 128 to 256 weight rows with one instruction, tokens along M, so that
//            a thread of the epilogue holds neighbouring features of one token.  Large products.
//
// What bounds them, and measured times (a library product of the same operands, without bias, activation and residual, in
// parentheses).  Products in a row take the SM clock from 1.9 GHz to what power allows, at once:
//   pair     the tensor pipe at that clock: 8192 x 28672 x 4096 gated 1150 us, 1.67 PFLOP/s, 1.61 million cycles at 1.43 GHz, tensor
//            pipe 89 % busy (1190); in a loop of seconds 1340 us, as many cycles at 1.21 GHz (1390).  8-bit operands: 8192 x 7168 x
//            2048 88 us, 130000 cycles at 1.54 GHz (84), with a residual 100, 143000 to 146000 cycles at 1.52 GHz; in a loop 107
//            us, 130000 cycles at 1.31 GHz (103), with a residual 120 to 123, 136000 at 1.22 GHz.
//   split    latency where little is read: 16 x 256 x 7168 to float32 4.7 us (10.7); what a CTA takes in, 85 bytes a cycle, and
//            the way of the partial sums, 16 bytes a cycle, otherwise: 64 x 4096 x 7168 gated on 8-bit operands 8.4 us, 30 MB
//            (12.9).
//
// Accumulation.  The tensor core adds to its fp32 accumulators with truncation: over K = 7168 the sums of random products
// come out 7e-6 too small in magnitude (relative 8e-6, against 3e-7 of fp32 arithmetic).  That is nothing beside a rounding
// to bf16: 8192 x 28672 x 4096, gated, is off from 64 bits by 1.658332e-3, sums in fp32 arithmetic by 1.658307e-3, and a library
// product of these operands, activated in 64 bits, by as much as here; the other rounding is taken by 4 outputs in a thousand, where
// fp32 arithmetic takes it by 0.7.  It would show in float32 results (router logits), so the split kernel lets an accumulator grow
// over 512 K only there and adds those pieces in registers: 5e-7, sums of one sign 9e-7 too small (1.3e-6 at most).
//
// Every mbarrier wait is bounded; one that gives up records a code in g_linear_status and the roles fall through to the end,
// where tensor memory is freed.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "device_once.cuh"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace pnv {
namespace {

__device__ int g_linear_status = 0;
enum LinearStatus : int { kLinProducer = 11, kLinMmaFull = 12, kLinMmaAcc = 13, kLinEpilogue = 14, kLinSums = 15, kLinResidual = 16 };

constexpr int kSmemMax = 227 * 1024;
constexpr int kStageRow = 128;           // bytes of K per operand row and pipeline stage: one 128-byte swizzle row
constexpr int kTileRows = 128;           // rows of one CTA's M operand
constexpr int kABytes = kTileRows * kStageRow;
constexpr int kBarBytes = 1024;

struct LinearArgs {
  void* out;
  const void* bias;                      // or nullptr
  const __nv_bfloat16* residual;         // or nullptr
  const uint8_t* x_sf;                   // 8-bit operands
  const uint8_t* w_sf;
  long long residual_stride;
  int rows, features, n_out;             // n_out: features, or half of them (gated)
  int k_bytes;                           // bytes of K in a row of either operand
  int m_tiles, n_tiles, tile_n, band;    // pair kernel: along tokens and along features, the features of a tile, tiles of a band
  int out_f32, bias_f32, gated, kind;    // kind: PNV_ACT_*
  GatedAct act;
  int vec_out, vec_residual, vec_bias;   // may these be accessed 16 bytes at a time
  int tma;                               // pair kernel: do outputs leave and residuals come by TMA copies
};

// What an epilogue does between bias and residual.  Kernels are compiled for each: with all the activations' code in one
// epilogue, jumped over four times a block, a block of 64 features took 2200 cycles where nothing was to be activated.
enum Mode : int { kNothing = 0, kActivate = 1, kGate = 2 };

// ---- epilogue arithmetic -------------------------------------------------------------------------

// The exponential and the reciprocal are good to 1e-7, the exponent's product is rounded first: off by 1.5e-7 for gates of unit size,
// 9e-7 at -20, 1.7e-6 at -40 (of 1.7e-16), less than a thousandth of a bf16 unit.
__device__ __forceinline__ float silu_f32(float g) { return g * rcp_approx(1.f + ex2_approx(g * -kLog2e)); }

// v / 2 erfc(-v / sqrt(2)).  In 1 + erf a negative v cancels (6 % off at -5, nothing left from -6).  With a = |v|, t = 1 / (1 + 0.35 a):
// erfc(a / sqrt(2)) / 2 = exp(-a^2 / 2) t Q(t), where t Q(t) is smooth; Q is its polynomial of degree 8 with the smallest
// relative error over a < 14.5 (weighted least squares, 3.2e-8), above which the exponential is 0.  Off by 10 + v^2 units of 2^-23 at
// most (v^2: what the exponent's rounding does).  4096 x 8192 x 4096 180 us, 1 + erff 178, erfcf 226.
__device__ __forceinline__ float gelu_f32(float v) {
  const float a = fabsf(v) > 16.f ? 16.f : fabsf(v);           // (an infinity would meet a zero; a NaN stays one)
  const float t = rcp_approx(fmaf(a, 0.35f, 1.f));
  constexpr float kQ[9] = {0.139621302f, 0.139863536f, 0.119821183f, 0.105552927f, -0.023213394f, 0.159321249f, -0.255840391f, 0.144031614f,
                           -0.0291580297f};
  float q = kQ[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) q = fmaf(q, t, kQ[i]);
  const float y = a * (t * q) * ex2_approx(a * a * (-0.5f * kLog2e));
  return v > 0.f ? v - y : -y;
}

template <int E>
__device__ __forceinline__ void add_bias(float (&v)[E], const LinearArgs& a, int col) {
  if (a.bias == nullptr) return;
  if (a.bias_f32) {
    const float* b = static_cast<const float*>(a.bias) + col;
    if (a.vec_bias && col + E <= a.features) {
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(b + j));
        v[j] += t.x; v[j + 1] += t.y; v[j + 2] += t.z; v[j + 3] += t.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (col + j < a.features) v[j] += __ldg(b + j);
    }
  } else {
    const unsigned short* b = static_cast<const unsigned short*>(a.bias) + col;
    if (a.vec_bias && col + E <= a.features) {
#pragma unroll
      for (int j = 0; j < E; j += 8) {
        float f[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(b + j)), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] += f[i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (col + j < a.features) v[j] += __uint_as_float((uint32_t)__ldg(b + j) << 16);
    }
  }
}

__device__ __forceinline__ float bias_at(const LinearArgs& a, int col) {
  if (col >= a.features) return 0.f;
  return a.bias_f32 ? __ldg(static_cast<const float*>(a.bias) + col)
                    : __uint_as_float((uint32_t)__ldg(static_cast<const unsigned short*>(a.bias) + col) << 16);
}

template <int E>
__device__ __forceinline__ void activate(float (&v)[E], const LinearArgs& a) {
  switch (a.kind) {
    case PNV_ACT_RELU:
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];        // (a NaN stays one)
      break;
    case PNV_ACT_SILU:
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = silu_f32(v[j]);
      break;
    case PNV_ACT_GELU:
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = gelu_f32(v[j]);
      break;
    default:
      break;
  }
}

template <int E>
__device__ __forceinline__ void gate(const float (&g)[E], const float (&u)[E], float (&y)[E], const LinearArgs& a) {
  if (a.kind == PNV_ACT_SITU) {
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = situ_short(g[j], u[j], a.act.beta, a.act.inv_beta, a.act.linear_beta, a.act.inv_linear);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = silu_f32(g[j]) * u[j];
  }
}

// v: outputs col .. col + E - 1 of token `row`.
template <int E>
__device__ __forceinline__ void add_residual(float (&v)[E], const LinearArgs& a, int row, int col) {
  if (a.residual == nullptr) return;
  const __nv_bfloat16* r = a.residual + row * a.residual_stride + col;
  if (a.vec_residual && col + E <= a.n_out) {
#pragma unroll
    for (int j = 0; j < E; j += 8) {
      float f[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(r + j)), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j + i] += f[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (col + j < a.n_out) v[j] += __uint_as_float((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(r) + j) << 16);
  }
}
// The one rounding.
template <int E>
__device__ __forceinline__ void store_outputs(const float (&v)[E], const LinearArgs& a, int row, int col) {
  const bool whole = col + E <= a.n_out;
  if (a.out_f32) {
    float* o = static_cast<float*>(a.out) + (long long)row * a.n_out + col;
    if (a.vec_out && whole) {
#pragma unroll
      for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (col + j < a.n_out) o[j] = v[j];
    }
    return;
  }
  uint32_t w[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) w[j] = as_u32(__floats2bfloat162_rn(v[2 * j], v[2 * j + 1]));
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + (long long)row * a.n_out + col;
  if (whole && a.vec_out) {
#pragma unroll
    for (int j = 0; j < E / 2; j += 4) *reinterpret_cast<uint4*>(o + 2 * j) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (col + j < a.n_out) reinterpret_cast<unsigned short*>(o)[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
  }
}

// Instructions of a stage that meet any K at all (the last stage of a K that is no multiple of 128 bytes has fewer: blocks past
// K are not multiplied, whatever scale they carry).
__device__ __forceinline__ int stage_mmas(int k_bytes, int stage) { return min(4, (k_bytes - stage * kStageRow + 31) / 32); }

// The four instructions of one stage (fewer where mmas says so); a and b: descriptors of the stage's operand tiles, 32 bytes of
// K are 2 units of their address field.  kMx8: the scale words of its four K-blocks sit at sfa and sfb.
// idesc: of the first block; the others differ in the scale byte that they name.
template <int CTAS, bool kMx8>
__device__ __forceinline__ void issue_one(uint32_t d, uint64_t a, uint64_t b, int i, uint32_t idesc, uint32_t accumulate, uint32_t sfa, uint32_t sfb) {
  if constexpr (kMx8) ptx::tc_mma_mxf8<CTAS>(d, a + 2 * i, b + 2 * i, idesc | ptx::mma_mxf8_scale_byte(i), accumulate, sfa, sfb);
  else ptx::tc_mma_bf16<CTAS>(d, a + 2 * i, b + 2 * i, idesc, accumulate);
}
template <int CTAS, bool kMx8>
__device__ __forceinline__ void issue_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int mmas, bool first, uint32_t sfa, uint32_t sfb) {
  issue_one<CTAS, kMx8>(d, a, b, 0, idesc, first ? 0u : 1u, sfa, sfb);
  if (mmas == 4) {
#pragma unroll
    for (int i = 1; i < 4; ++i) issue_one<CTAS, kMx8>(d, a, b, i, idesc, 1u, sfa, sfb);
  } else {
#pragma unroll
    for (int i = 1; i < 3; ++i)
      if (i < mmas) issue_one<CTAS, kMx8>(d, a, b, i, idesc, 1u, sfa, sfb);
  }
}
template <bool kMx8>
__device__ __forceinline__ constexpr uint32_t product_idesc(int n, int m) { return kMx8 ? ptx::mma_mxf8_idesc(n, m) : ptx::mma_bf16_idesc(n, m); }

// After a wait gave up: time for the copies in flight to land before the CTA leaves.
__device__ __forceinline__ void linger() {
#pragma unroll 1
  for (int i = 0; i < 2000; ++i) __nanosleep(1000);
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// ---- split kernel ----------------------------------------------------------------------------------

// Two warps issue, each every other stage into accumulators of its own: one alone takes 450 cycles a stage (four products and
// a commit 270, the rest its waits), whatever the width of the tile.
constexpr int kIssuers = 2;

template <int BN, bool kMx8>
struct SplitCfg {
  static_assert(BN == 16 || BN == 32 || BN == 64 || BN == 128, "token tiles of 16, 32, 64 or 128");
  static constexpr int kGroups = BN >= 64 ? 2 : 1;                   // epilogue warps per quarter of the lanes
  static constexpr int kEpiWarps = 4 * kGroups;
  static constexpr int kThreads = (4 + kEpiWarps) * 32;              // producer, two issuers, an idle warp, epilogue
  static constexpr int kCols = BN / kGroups;                         // accumulator columns of an epilogue warp
  static constexpr int kBBytes = BN * kStageRow;
  static constexpr int kStageBytes = kABytes + kBBytes + (kMx8 ? 1024 : 0);
  static constexpr int kSumBytes = BN * kTileRows * 4;               // partial sums of this CTA's share of the outputs
  static constexpr int kMaxStages = 12;
  static constexpr int kFit = (kSmemMax - 1024 - kBarBytes - kSumBytes) / kStageBytes;
  // A multiple of the issuers, so that the same one meets every turn of a stage: a wait for a parity cannot tell the turn it wants
  // from the one two before, so a warp that skips turns may find a stage full that is still being filled.
  static constexpr int kStages = (kFit < kMaxStages ? kFit : kMaxStages) / kIssuers * kIssuers;
  // stages after which the accumulators are emptied into registers: 512 K in each of the two (float32 results only)
  static constexpr int kChunk = 16;
  // tensor memory: the issuers' accumulators, twice where they are emptied on the way, then the scales
  static constexpr int kBuffers = kMx8 ? 1 : 2;
  static constexpr int kColSf = kBuffers * kIssuers * BN;
  static constexpr int kColsUsed = kColSf + (kMx8 ? 8 * kStages : 0);
  static constexpr int kTmemCols = kColsUsed <= 32 ? 32 : kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kSumBytes + kBarBytes;
  static_assert(kColsUsed <= 512 && kStages > kIssuers && kStages % kIssuers == 0, "tensor-memory column map or pipeline");
};

template <int BN, bool kMx8, int kMode>
__global__ void __launch_bounds__(SplitCfg<BN, kMx8>::kThreads, 1)
linear_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LinearArgs a,
                    const int split) {
  using C = SplitCfg<BN, kMx8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  float* sums = reinterpret_cast<float*>(stages + C::kStages * C::kStageBytes);      // [CTA it came from][token of this CTA][feature]
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + C::kStages * C::kStageBytes + C::kSumBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* sums_full = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_full + 1);
  // (the shuffle tells the compiler that the roles below are the same for a whole warp)
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)ptx::cluster_ctarank() : 0;
  const int ft = (int)blockIdx.x / split, tt = (int)blockIdx.y;      // feature tile, token tile
  if (warp == 0) {
    if (ptx::elect_one()) {
      ptx::prefetch_tensormap(&map_w);
      ptx::prefetch_tensormap(&map_x);
      for (int s = 0; s < C::kStages; ++s) {
        ptx::mbar_init(full + s, 1);
        ptx::mbar_init(empty + s, 1);
      }
      for (int b = 0; b < 2; ++b) {
        ptx::mbar_init(acc_full + b, kIssuers);
        ptx::mbar_init(acc_empty + b, C::kEpiWarps);
      }
      ptx::mbar_init(sums_full, 1);
      ptx::fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (split > 1) ptx::cluster_arrive();  // (waited for before the first copy into another CTA: its barrier has to be there)
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  const int k_stages = (a.k_bytes + kStageRow - 1) / kStageRow;
  const int ks0 = (int)((long long)rank * k_stages / split), n = (int)((long long)(rank + 1) * k_stages / split) - ks0;
  const int chunk_stages = !kMx8 && a.out_f32 ? C::kChunk : n;
  const int chunks = (n + chunk_stages - 1) / chunk_stages;
  const int share = BN / split;          // tokens of the tile whose outputs this CTA makes
  const int tokens = min(BN, a.rows - tt * BN), own = min(share, tokens - rank * share);      // of the tile; of them this CTA's
  if (warp == 0) {
    // ---- producer
    const int n_kt = k_stages;           // an atom of scales has the 128 codes of a stage
    int stage = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (int ks = ks0; ks < ks0 + n; ++ks) {
      if (!ptx::mbar_wait_warp(empty + stage, phase ^ 1)) {
        atomicExch(&g_linear_status, kLinProducer);
        linger();
        break;
      }
      uint8_t* st = stages + stage * C::kStageBytes;
      if (ptx::elect_one()) {
        ptx::mbar_arrive_expect_tx(full + stage, C::kStageBytes);
        ptx::tma_load_3d(st, &map_w, full + stage, ks * kStageRow, ft * kTileRows, 0);
        ptx::tma_load_3d(st + kABytes, &map_x, full + stage, ks * kStageRow, tt * BN, 0);
        if constexpr (kMx8) {            // (token tiles of 64 share an atom of scales in twos, narrower ones are the only one)
          ptx::bulk_load(st + kABytes + C::kBBytes, a.w_sf + ((long long)ft * n_kt + ks) * 512, 512, full + stage);
          ptx::bulk_load(st + kABytes + C::kBBytes + 512, a.x_sf + ((long long)(tt * BN / 128) * n_kt + ks) * 512, 512, full + stage);
        }
      }
      __syncwarp();
      if (++stage == C::kStages) { stage = 0; phase ^= 1; }
    }
  } else if (warp <= kIssuers) {
    // ---- issuers
    const int me = warp - 1;
    const uint32_t sfb_shift = (uint32_t)(tt * BN & 127) / 32;         // tokens 64 on of an atom: two columns on
    int stage = me;
    uint32_t phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int chunk = 0; ok && chunk < chunks; ++chunk) {
      const int lo = chunk * chunk_stages + me, hi = min(n, (chunk + 1) * chunk_stages), buf = chunk & 1;
      if (!ptx::mbar_wait_warp(acc_empty + buf, ((chunk >> 1) & 1) ^ 1)) {
        atomicExch(&g_linear_status, kLinMmaAcc);
        break;
      }
      ptx::tc_fence_after();
      const uint32_t d = tmem + (buf * kIssuers + me) * BN;
      if (lo >= hi) {                    // the last chunk can be too short for both
        if (ptx::elect_one()) ptx::mbar_arrive(acc_full + buf);
        __syncwarp();
      }
#pragma unroll 1
      for (int i = lo; i < hi; i += kIssuers) {
        if (!ptx::mbar_wait_warp(full + stage, phase)) {
          atomicExch(&g_linear_status, kLinMmaFull);
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t st = ptx::smem_u32(stages + stage * C::kStageBytes);
        if (ptx::elect_one()) {
          const uint32_t sfa = tmem + C::kColSf + 8 * stage, sfb = sfa + 4;
          if constexpr (kMx8) {
            ptx::tc_cp_32x128b_warpx4(sfa, ptx::smem_desc(st + kABytes + C::kBBytes, 128, 0, 0));
            ptx::tc_cp_32x128b_warpx4(sfb, ptx::smem_desc(st + kABytes + C::kBBytes + 512, 128, 0, 0));
          }
          issue_stage<1, kMx8>(d, ptx::smem_desc(st, 1024, 16, 2), ptx::smem_desc(st + kABytes, 1024, 16, 2), product_idesc<kMx8>(BN, kTileRows),
                               stage_mmas(a.k_bytes, ks0 + i), i == lo, sfa, sfb + sfb_shift);
          ptx::tc_commit(empty + stage);
          if (i + kIssuers >= hi) ptx::tc_commit(acc_full + buf);
        }
        __syncwarp();
        stage += kIssuers;
        if (stage >= C::kStages) { stage -= C::kStages; phase ^= 1; }
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue: the accumulators' pieces are added in registers, then go to the CTAs that own their tokens
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;                 // lane quarter of this warp
    const int col0 = (warp - 4) / 4 * C::kCols;
    float sum[C::kCols];
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) sum[j] = 0.f;
#pragma unroll 1
    for (int chunk = 0; chunk < chunks; ++chunk) {
      const int buf = chunk & 1;
      if (!ptx::mbar_wait_warp(acc_full + buf, (chunk >> 1) & 1)) {
        atomicExch(&g_linear_status, kLinEpilogue);
        break;
      }
      ptx::tc_fence_after();
      const int used = min(kIssuers, n - chunk * chunk_stages);        // accumulators that hold anything
#pragma unroll 1
      for (int j = 0; j < used; ++j) {
        const uint32_t src = tmem + lanes + (buf * kIssuers + j) * BN + col0;
        if constexpr (C::kCols == 16) {
          uint32_t r[16];
          ptx::tc_ld_32x16(src, r);
          ptx::tc_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] += __uint_as_float(r[i]);
        } else {
#pragma unroll
          for (int h = 0; h < C::kCols; h += 32) {
            uint32_t r[32];
            ptx::tc_ld_32x32(src + h, r);
            ptx::tc_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[h + i] += __uint_as_float(r[i]);
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(acc_empty + buf);
    }
    const int feature = (warp & 3) * 32 + lane;
    // every load and product of this CTA is over: with partners the first stages' memory takes what goes to them
    float* part = split > 1 ? reinterpret_cast<float*>(stages) : sums;
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) part[(col0 + j) * kTileRows + feature] = sum[j];
    if (split > 1) {
      ptx::fence_proxy_async_smem();
      ptx::cluster_wait();
      named_barrier(1, C::kEpiWarps * 32);
      // tokens [r * share, (r + 1) * share) go to CTA r, as the rank-th part of what it adds
      for (int r = warp - 4; r < split; r += C::kEpiWarps) {
        const int rows = min(share, tokens - r * share);
        if (rows > 0 && ptx::elect_one())
          ptx::bulk_copy_cluster(sums + rank * share * kTileRows, part + r * share * kTileRows, rows * kTileRows * 4, sums_full, r);
        __syncwarp();
      }
    }
  }
  __syncwarp();
  // Outputs are made in pieces of eight neighbouring features of a token; a thread's pieces have the same features.  Gated:
  // features [64 b, 64 b + 32) are gates, the next 32 their ups.
  constexpr int kPieces = kMode == kGate ? 8 : 16;
  static_assert(C::kThreads % kPieces == 0, "a thread keeps its features from token to token");
  const int piece = (int)threadIdx.x % kPieces;
  const int f = kMode == kGate ? (piece >> 2) * 64 + (piece & 3) * 8 : piece * 8, col = ft * kTileRows + f;
  float bias[8], up_bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = up_bias[j] = 0.f;
  if (col < a.features) {
    add_bias(bias, a, col);
    if (kMode == kGate) add_bias(up_bias, a, col + 32);
  }
  ptx::tc_fence_before();
  if (split > 1) {
    if (warp < 4) ptx::cluster_wait();
    if (warp == 0 && own > 0) {
      if (ptx::elect_one()) ptx::mbar_arrive_expect_tx(sums_full, (uint32_t)(split * own * kTileRows * 4));
      __syncwarp();
      if (!ptx::mbar_wait_warp(sums_full, 0)) {
        atomicExch(&g_linear_status, kLinSums);
        linger();
      }
    }
    __syncthreads();
    ptx::cluster_arrive();               // this CTA has all that the others sent it
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kTmemCols);
  }

  // ---- this CTA's share of the tile's outputs
  if (col < a.features) {
    const int out_col = kMode == kGate ? (col - f) / 2 + (piece >> 2) * 32 + (piece & 3) * 8 : col;
#pragma unroll(kMode == kGate ? 1 : 2)
    for (int token = (int)threadIdx.x / kPieces; token < own; token += C::kThreads / kPieces) {
      const int row = tt * BN + rank * share + token;
      float v[8], up[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = up[j] = 0.f;
      const float4* src = reinterpret_cast<const float4*>(sums + token * kTileRows + f);
#pragma unroll 4
      for (int r = 0; r < split; ++r, src += share * (kTileRows / 4)) {
        const float4 p = src[0], q = src[1];
        v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
        v[4] += q.x; v[5] += q.y; v[6] += q.z; v[7] += q.w;
        if constexpr (kMode == kGate) {
          const float4 s = src[8], t = src[9];
          up[0] += s.x; up[1] += s.y; up[2] += s.z; up[3] += s.w;
          up[4] += t.x; up[5] += t.y; up[6] += t.z; up[7] += t.w;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += bias[j];
      if constexpr (kMode == kGate) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) up[j] += up_bias[j];
        gate(v, up, y, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = y[j];
      } else if constexpr (kMode == kActivate) {
        activate(v, a);
      }
      add_residual(v, a, row, out_col);
      store_outputs(v, a, row, out_col);
    }
  }
  if (split > 1) ptx::cluster_wait();    // what this CTA sent has arrived: its memory may go
}

// ---- pair kernel -----------------------------------------------------------------------------------
//
// Six stages of 32 KB (8-bit operands: five of 34 KB with the scales) beside 32 KB in which residuals arrive and outputs leave:
// with twice that for the epilogue and a stage less the products waited (8192 x 7168 x 2048: 83 us instead of 77).  Eight
// epilogue warps: a thread keeps its 128 accumulators in registers, so that where there is one accumulator (8-bit operands and
// tiles of 256 features: the scale words need the other's columns) it is free again after 130 cycles.

template <bool kMx8>
struct PairCfg {
  static constexpr int kTileM = 256, kTileN = 256;                   // tokens and (at most) features of a pair's tile
  static constexpr int kGroups = 2, kEpiWarps = 4 * kGroups;         // epilogue warps: one per quarter of the lanes and group
  static constexpr int kThreads = (2 + kEpiWarps) * 32;              // producer, issuer, epilogue (168 registers a thread)
  static constexpr int kBBytes = 128 * kStageRow;                    // half of the features, at most
  static constexpr int kSfBytes = kMx8 ? 512 + 1024 : 0;             // own tokens' scales, those of the tile's features
  static constexpr int kStageBytes = kABytes + kBBytes + (kMx8 ? 2048 : 0);
  static constexpr int kStagingBytes = kEpiWarps * 4096;             // a warp's 32 tokens x 64 features of residual and output
  static constexpr int kStages = (kSmemMax - 1024 - kBarBytes - kStagingBytes) / kStageBytes;
  // Two accumulators, so that a tile's products are made while the one before is read.  8-bit operands: the scale words need
  // columns too, so there are two of up to 192 features, or one; its readers hand it back as soon as they have it in registers.
  // (Tiles of 192 in several waves, two against one: 2048 x 7168 x 2048 25.4 us against 26.6, with a residual 27.4 against 29.1.)
  static constexpr int kAccWidth = kMx8 ? 192 : kTileN;
  static constexpr int kTmemCols = 512;
  __host__ __device__ static constexpr int accs(int tile_n) { return tile_n <= kAccWidth ? 2 : 1; }
  __host__ __device__ static constexpr int col_sf(int tile_n) { return tile_n <= kAccWidth ? 2 * kAccWidth : kTileN; }
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kStagingBytes + kBarBytes;
  static_assert(col_sf(kAccWidth) + (kMx8 ? 12 * kStages : 0) <= kTmemCols && col_sf(kTileN) + (kMx8 ? 12 * kStages : 0) <= kTmemCols,
                "tensor-memory column map overflows");
};

// Tiles in bands along the tokens, features outer within a band: the tiles that run at one time share activations and weights
// in L2, and the weights are read from memory once per band.
__device__ __forceinline__ void pair_tile(int tile, const LinearArgs& a, int& mt, int& nt) {
  const int band = tile / (a.band * a.n_tiles), in = tile - band * a.band * a.n_tiles;
  const int height = min(a.band, a.m_tiles - band * a.band);
  nt = in / height;
  mt = band * a.band + in - nt * height;
}
// Eight tiles of 256 tokens, or 16 or 32 where their activations fill no more than a third of L2.  In loops of seconds, 8192 x
// 28672 x 4096: 8 / 16 / 32 tiles take 1385 / 1350 / 1467 us, 8-bit operands 780 / 752 / 745; 16384 x 4096 x 14336 1501 / 1560 /
// 1655.
constexpr int kLowBand = 8, kHighBand = 32;
constexpr long long kBandBytes = 40LL << 20;

__device__ __forceinline__ int tile_nt(int tile, const LinearArgs& a) {
  int mt, nt;
  pair_tile(tile, a, mt, nt);
  return nt;
}

template <bool kMx8, int kMode>
__global__ void __launch_bounds__(PairCfg<kMx8>::kThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_w_sf, const __grid_constant__ CUtensorMap map_x_sf,
                   const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_out_32,
                   const __grid_constant__ CUtensorMap map_res, const __grid_constant__ CUtensorMap map_res_32, const LinearArgs a) {
  using C = PairCfg<kMx8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* staging = stages + C::kStages * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::kStagingBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* res_full = acc_empty + 2;                                  // one per epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + C::kEpiWarps);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  if (warp == 0) {
    if (ptx::elect_one()) {
      ptx::prefetch_tensormap(&map_w);
      ptx::prefetch_tensormap(&map_x);
      for (int s = 0; s < C::kStages; ++s) {
        ptx::mbar_init(full + s, 1);
        ptx::mbar_init(empty + s, 1);
      }
      for (int b = 0; b < 2; ++b) {
        ptx::mbar_init(acc_full + b, 1);
        ptx::mbar_init(acc_empty + b, 2 * C::kEpiWarps);
      }
      for (int w = 0; w < C::kEpiWarps; ++w) ptx::mbar_init(res_full + w, 1);
      ptx::fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == 1) {
    ptx::tmem_alloc<2>(tmem_slot, C::kTmemCols);
    ptx::tmem_relinquish<2>();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  const int k_stages = (a.k_bytes + kStageRow - 1) / kStageRow;
  const int tiles = a.m_tiles * a.n_tiles, pairs = (int)gridDim.x / 2;
  const int accs = C::accs(a.tile_n);
  if (warp == 0) {
    // ---- producer, in both CTAs: own tokens, own half of the features; completion is counted on the first CTA's barrier
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int tile = (int)blockIdx.x / 2; ok && tile < tiles; tile += pairs) {
      int mt, nt;
      pair_tile(tile, a, mt, nt);
#pragma unroll 1
      for (int ks = 0; ks < k_stages; ++ks) {
        if (!ptx::mbar_wait_warp(empty + stage, phase ^ 1)) {
          atomicExch(&g_linear_status, kLinProducer);
          ok = false;
          break;
        }
        uint8_t* st = stages + stage * C::kStageBytes;
        if (ptx::elect_one()) {
          if (rank == 0) ptx::mbar_arrive_expect_tx(full + stage, (uint32_t)(2 * (kABytes + a.tile_n / 2 * kStageRow + C::kSfBytes)));
          ptx::tma_load_3d_pair(st, &map_x, full + stage, 0, ks * kStageRow, mt * 256 + (int)rank * 128, 0);
          ptx::tma_load_3d_pair(st + kABytes, &map_w, full + stage, 0, ks * kStageRow, nt * a.tile_n + (int)rank * a.tile_n / 2, 0);
          if constexpr (kMx8) {
            ptx::tma_load_3d_pair(st + kABytes + C::kBBytes, &map_x_sf, full + stage, 0, 0, ks, mt * 2 + (int)rank);
            ptx::tma_load_3d_pair(st + kABytes + C::kBBytes + 512, &map_w_sf, full + stage, 0, 0, ks, nt * a.tile_n / 128);
          }
        }
        __syncwarp();
        if (++stage == C::kStages) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) linger();
  } else if (warp == 1 && rank == 0) {
    // ---- issuer
    const uint32_t idesc = product_idesc<kMx8>(a.tile_n, C::kTileM);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int tile = (int)blockIdx.x / 2; ok && tile < tiles; tile += pairs) {
      if (!ptx::mbar_wait_warp(acc_empty + acc, acc_phase ^ 1)) {
        atomicExch(&g_linear_status, kLinMmaAcc);
        break;
      }
      ptx::tc_fence_after();
      // a tile that starts in the middle of a 128-feature atom of scales: two columns (64 features) on
      const uint32_t sfb_shift = kMx8 ? (uint32_t)((tile_nt(tile, a) * a.tile_n) & 127) / 32 : 0u;
#pragma unroll 1
      for (int ks = 0; ks < k_stages; ++ks) {
        if (!ptx::mbar_wait_warp(full + stage, phase)) {
          atomicExch(&g_linear_status, kLinMmaFull);
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t st = ptx::smem_u32(stages + stage * C::kStageBytes);
        if (ptx::elect_one()) {
          const uint32_t sfa = tmem + C::col_sf(a.tile_n) + 12 * stage, sfb = sfa + 4;
          if constexpr (kMx8) {
            const uint32_t sf = st + kABytes + C::kBBytes;
            ptx::tc_cp_32x128b_warpx4<2>(sfa, ptx::smem_desc(sf, 128, 0, 0));
            ptx::tc_cp_32x128b_warpx4<2>(sfb, ptx::smem_desc(sf + 512, 128, 0, 0));
            ptx::tc_cp_32x128b_warpx4<2>(sfb + 4, ptx::smem_desc(sf + 1024, 128, 0, 0));
          }
          issue_stage<2, kMx8>(tmem + acc * C::kAccWidth, ptx::smem_desc(st, 1024, 16, 2), ptx::smem_desc(st + kABytes, 1024, 16, 2), idesc,
                               stage_mmas(a.k_bytes, ks), ks == 0, sfa, sfb + sfb_shift);
          ptx::tc_commit_pair(empty + stage);
          if (ks + 1 == k_stages) ptx::tc_commit_pair(acc_full + acc);
        }
        __syncwarp();
        if (++stage == C::kStages) { stage = 0; phase ^= 1; }
      }
      if (++acc == accs) { acc = 0; acc_phase ^= 1; }
    }
  } else if (warp >= 2) {
    // ---- epilogue: a tile's blocks of 64 features go to the two groups in turn, a thread has one token's.  Outputs leave and
    // residuals come through 4 KB of shared memory per warp and TMA copies of 32 tokens x 64 features (128-byte swizzle; of 32
    // features, 64-byte swizzle, where a tile ends with them or gates leave half), a thread reading its residuals from where it
    // puts its outputs.  With loads and stores of its own, 32 rows apart from lane to lane, the epilogue of a tile with a residual
    // took 10000 cycles, where the products of K = 2048 take 8200.  What copies cannot take goes the other way (slow).
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    uint8_t* mine = staging + (warp - 2) * 4096;
    const bool staged_res = a.residual != nullptr && a.tma != 0;
    int acc = 0;
    uint32_t acc_phase = 0, res_phase = 0;
    bool ok = true;
    const auto is_wide = [&](int block) { return kMode != kGate && a.tile_n - block * 64 >= 64; };
    // The residual of a block of a tile (tokens from row0 on) is asked for; lane 0, whose stores from there have been read.
    const auto ask = [&](int row0, int nt, int block) {
      const int col = nt * a.tile_n + block * 64;
      const bool wide = is_wide(block);
      ptx::mbar_arrive_expect_tx(res_full + warp - 2, wide ? 4096 : 2048);
      ptx::tma_load_3d(mine, wide ? &map_res : &map_res_32, res_full + warp - 2, kMode == kGate ? col / 2 : col, row0, 0);
    };
    const int last_blocks = (a.tile_n + 63) / 64;
    if (staged_res && group < last_blocks && (int)blockIdx.x / 2 < tiles && lane == 0) {
      int mt, nt;
      pair_tile((int)blockIdx.x / 2, a, mt, nt);
      ask(mt * 256 + (int)rank * 128 + quarter * 32, nt, group);
    }
    __syncwarp();
#pragma unroll 1
    for (int tile = (int)blockIdx.x / 2; ok && tile < tiles; tile += pairs) {
      int mt, nt;
      pair_tile(tile, a, mt, nt);
      const int row0 = mt * 256 + (int)rank * 128 + quarter * 32, row = row0 + lane;
      float bias[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int block = group + 2 * i, col = nt * a.tile_n + block * 64;
        bias[i][0] = bias[i][1] = 0.f;
        if (a.bias != nullptr && block < last_blocks) {
          bias[i][0] = bias_at(a, col + lane);
          bias[i][1] = bias_at(a, col + 32 + lane);
        }
      }
      if (!ptx::mbar_wait_warp(acc_full + acc, acc_phase)) {
        atomicExch(&g_linear_status, kLinEpilogue);
        linger();
        break;
      }
      ptx::tc_fence_after();
      uint32_t r[2][2][32];              // (columns past the tile hold whatever they hold and are not used)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t src = tmem + ((uint32_t)quarter << 21) + acc * C::kAccWidth + (group + 2 * i) * 64;
        ptx::tc_ld_32x32(src, r[i][0]);
        ptx::tc_ld_32x32(src + 32, r[i][1]);
      }
      ptx::tc_ld_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(acc_empty + acc, 0);
      if (++acc == accs) { acc = 0; acc_phase ^= 1; }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int block = group + 2 * i, col = nt * a.tile_n + block * 64, out_col = kMode == kGate ? col / 2 : col;
        if (!ok || block >= last_blocks) continue;
        // features of the block that belong to the tile (a multiple of 32) and to the matrix
        const int width = min(min(64, a.tile_n - block * 64), a.features - col);
        if (staged_res) {
          if (!ptx::mbar_wait_warp(res_full + warp - 2, res_phase)) {
            atomicExch(&g_linear_status, kLinResidual);
            linger();
            ok = false;
            continue;
          }
          res_phase ^= 1;
        } else if (a.tma) {
          if (lane == 0) ptx::bulk_wait_read_all();
          __syncwarp();
        }
        if (a.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            r[i][0][j] = __float_as_uint(__uint_as_float(r[i][0][j]) + __shfl_sync(0xffffffffu, bias[i][0], j));
            r[i][1][j] = __float_as_uint(__uint_as_float(r[i][1][j]) + __shfl_sync(0xffffffffu, bias[i][1], j));
          }
        }
        const bool wide = is_wide(block);
        if (__builtin_expect(a.tma, 1)) {
          // this thread's row of the box, 16-byte pieces swizzled by the row (what lies past the matrix is not copied out)
          uint8_t* line = mine + lane * (wide ? 128 : 64);
          const int swz = wide ? lane & 7 : (lane >> 1) & 3;
#pragma unroll
          for (int h = 0; h < (kMode == kGate ? 32 : 64); h += 8) {
            if (kMode != kGate && h == 32 && !wide) break;
            float v[8];
            if constexpr (kMode == kGate) {
              float g[8], u[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) { g[j] = __uint_as_float(r[i][0][h + j]); u[j] = __uint_as_float(r[i][1][h + j]); }
              gate(g, u, v, a);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[i][h / 32][h % 32 + j]);
              if constexpr (kMode == kActivate) activate(v, a);
            }
            uint4* at = reinterpret_cast<uint4*>(line + (((h / 8) ^ swz) << 4));
            if (staged_res) {
              float f[8];
              unpack8(*at, f);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += f[j];
            }
            *at = make_uint4(as_u32(__floats2bfloat162_rn(v[0], v[1])), as_u32(__floats2bfloat162_rn(v[2], v[3])),
                             as_u32(__floats2bfloat162_rn(v[4], v[5])), as_u32(__floats2bfloat162_rn(v[6], v[7])));
          }
          ptx::fence_proxy_async_smem();
        } else if (row < a.rows) {
#pragma unroll
          for (int h = 0; h < (kMode == kGate ? 32 : 64); h += 8) {
            if (h < width) {             // (gated: a whole block or nothing)
              float v[8];
              if constexpr (kMode == kGate) {
                float g[8], u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) { g[j] = __uint_as_float(r[i][0][h + j]); u[j] = __uint_as_float(r[i][1][h + j]); }
                gate(g, u, v, a);
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[i][h / 32][h % 32 + j]);
                if constexpr (kMode == kActivate) activate(v, a);
              }
              add_residual(v, a, row, out_col + h);
              store_outputs(v, a, row, out_col + h);
            }
          }
        }
        __syncwarp();
        if (lane == 0) {
          if (a.tma && row0 < a.rows && width > 0) {
            ptx::tma_store_3d(wide ? &map_out : &map_out_32, mine, out_col, row0, 0);
            ptx::bulk_commit();
          }
          if (staged_res) {              // the next block's residual, once the copies have read this one's outputs
            ptx::bulk_wait_read_all();
            if (block + 2 < last_blocks) {
              ask(row0, nt, block + 2);
            } else if (tile + pairs < tiles) {
              int mt2, nt2;
              pair_tile(tile + pairs, a, mt2, nt2);
              ask(mt2 * 256 + (int)rank * 128 + quarter * 32, nt2, group);
            }
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0) ptx::bulk_wait_all();
  }
  __syncwarp();
  ptx::tc_fence_before();
  ptx::cluster_sync();                   // (the partner's barriers and tensor memory are in use until both are here)
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<2>(tmem, C::kTmemCols);
  }
}

// ---- host side -------------------------------------------------------------------------------------

// A tiled view [rows][width] of `type`, rows `stride` bytes apart, in boxes of box_rows x box_width.  (Encoding one takes a
// third of a microsecond.)
int make_view(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t width, uint64_t rows, uint64_t stride, uint32_t box_width,
              uint32_t box_rows, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion, uint64_t layers = 1, uint32_t box_layers = 1) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(PNV_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[3] = {width, rows, layers};
  cuuint64_t strides[2] = {stride, stride * rows};
  cuuint32_t box[3] = {box_width, box_rows, box_layers};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PNV_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (width=%llu rows=%llu stride=%llu)", (int)r,
                (unsigned long long)width, (unsigned long long)rows, (unsigned long long)stride);
  return PNV_OK;
}

// An operand [rows][k_bytes] in boxes of 128 bytes of K (128-byte swizzle).
int operand_map(CUtensorMap* map, const void* base, uint64_t k_bytes, uint64_t rows, uint64_t stride, uint32_t box_rows) {
  return make_view(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, k_bytes, rows, stride, kStageRow, box_rows, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
// A scale buffer as [row atoms][K atoms][128 words], in boxes of `atoms` row atoms of one K atom.  (A tiled copy, unlike a
// plain bulk copy, can count its bytes on the partner's barrier.)
int scale_map(CUtensorMap* map, const void* base, uint64_t row_atoms, uint64_t k_atoms, uint32_t atoms) {
  return make_view(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 128, k_atoms, 512, 128, 1, CU_TENSOR_MAP_SWIZZLE_NONE,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, row_atoms, atoms);
}
// bf16 rows, `stride` elements apart, in boxes of 64 or 32 columns x 32 rows (128- or 64-byte swizzle): outputs and residuals.
int rows_map(CUtensorMap* map, const void* base, uint64_t width, uint64_t rows, uint64_t stride, uint32_t box) {
  return make_view(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, width, rows, stride * 2, box, 32,
                   box == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

constexpr int kMaxSplitLog = 3;          // clusters of 1, 2, 4 or 8 CTAs

int current_device(int& dev) {
  PNV_CUDA(cudaGetDevice(&dev));
  PNV_REQUIRE(dev >= 0 && dev < kMaxDevices, "unexpected CUDA device index %d", dev);
  return PNV_OK;
}
int set_up_failed(cudaError_t err) {
  cudaGetLastError();                    // (it is reported here, and is not to be found by whoever asks next)
  return fail(PNV_ERR_CUDA, "linear kernel set-up failed: %s", cudaGetErrorString(err));
}

// Per kernel and device, once: the shared-memory carve-out.
template <class Kernel>
int prepare(Kernel kernel, DeviceOnce& once, size_t smem) {
  int dev = 0;
  if (int rc = current_device(dev)) return rc;
  const cudaError_t err = once(dev, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
  return err == cudaSuccess ? PNV_OK : set_up_failed(err);
}

// Per device, once: how many clusters of 2^i CTAs run at one time.  Every kernel here fills an SM's shared memory with one CTA,
// so one of them answers for all.
int cluster_capacity(const int** out) {
  using C = SplitCfg<16, false>;
  static DeviceOnce setup, asked;
  static int clusters[kMaxDevices][kMaxSplitLog + 1] = {};
  const auto kernel = linear_split_kernel<16, false, kNothing>;
  if (int rc = prepare(kernel, setup, C::kSmem)) return rc;
  int dev = 0;
  if (int rc = current_device(dev)) return rc;
  const cudaError_t err = asked(dev, [&] {
    cudaError_t e = cudaSuccess;
    for (int i = 0; i <= kMaxSplitLog && e == cudaSuccess; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(8 << 7);
      cfg.blockDim = dim3(C::kThreads);
      cfg.dynamicSmemBytes = C::kSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&clusters[dev][i], kernel, &cfg);
    }
    return e;
  });
  if (err != cudaSuccess) return set_up_failed(err);
  *out = clusters[dev];
  return PNV_OK;
}

// ---- which kernel, tile and split: the cheapest by a model of their time ---------------------------------
//
// The constants are a fit, in units of 1/1.9 ns, to measured times of all the candidates for eight weights from 256 x 7168 to
// 28672 x 4096 and 1 to 4096 tokens, both operand types (two thousand calls): off by a tenth on average; the candidate that it
// picks is 1.2 % slower than the best one on average and 18 % at worst.  Two changes came after the fit and are not in it: the split
// kernel's bias is read ahead (a few tenths of a microsecond, for all its candidates), and pair tiles of 192 features have two
// accumulators on 8-bit operands too (up to 5 % in several waves; an entry of their own that made them cheaper took them where
// others are faster: K = 1024 with a residual lost 10 %).

struct Plan {
  int tokens;                            // split kernel: tokens of a tile; 0: pair kernel
  int split;                             // split kernel: CTAs that share a tile's K
  int width;                             // pair kernel: features of a tile
  long long cost;
};

Plan make_plan(const LinearArgs& a, bool mx8, const int* clusters, int sm_count) {
  const long long stages = ceil_div_i(a.k_bytes, kStageRow), feature_tiles = ceil_div_i(a.features, kTileRows);
  const auto waves_of = [](long long tiles, int room) { return tiles <= room ? 1LL : (tiles + room - 1) / room; };
  Plan best{0, 0, 0, -1};
  const auto offer = [&](const Plan& p) {
    if (best.cost < 0 || p.cost < best.cost) best = p;
  };
  for (int log = 4; log <= 7; ++log) {
    const int tokens = 1 << log;
    // Tiles no wider than they need be.  (Scale words start at multiples of 64 tokens: narrower tiles only on their own.)
    if (tokens > 16 && tokens / 2 >= a.rows) break;
    if (mx8 && tokens < 64 && tokens < a.rows) continue;
    const long long token_tiles = (a.rows + tokens - 1) >> log, tiles = token_tiles * feature_tiles;
    if (token_tiles > 65535) continue;   // (a grid's limit)
    for (int i = 0; i <= kMaxSplitLog; ++i) {
      const int split = 1 << i, room = std::min(clusters[i], sm_count >> i);
      if (room < 1 || (split > 1 && (tiles > room || stages < 2 * split))) break;
      const long long mine = (stages + split - 1) >> i;
      // a stage: what is issued for it, its bytes, or the weights' bytes of all CTAs
      const long long stage = std::max(std::max(213, 171 + tokens), (int)(std::min<long long>(tiles * split, sm_count) * kABytes / 5670));
      const long long sums = split > 1 ? 1690 + 20 * tokens + 10 * split : 0;        // on their way between the CTAs
      offer(Plan{tokens, split, 0, 4360 + waves_of(tiles, room) * (mine * stage + sums + 47 * tokens)});
    }
  }
  const int pairs = std::min(clusters[1], sm_count / 2);
  if (!a.out_f32 && pairs >= 1) {
    // Widths of 32 features; of 64 where the scales' atoms or the gates' blocks ask for it.
    const long long m_tiles = (a.rows + 255) >> 8;
    for (int width = 256; width >= 128; width -= mx8 || a.gated ? 64 : 32) {
      const long long tiles = m_tiles * ((a.features + width - 1) / width);
      if (tiles >= (1LL << 31) / kHighBand) continue;
      // a stage: its products (2 cycles a feature at full clock) and waits; a tile at least what its epilogue takes
      const long long stage = mx8 ? 236 + 19 * width / 10 : 84 + 23 * width / 10;
      offer(Plan{0, 1, width, 5760 + waves_of(tiles, pairs) * std::max(stages * stage, 3980LL) + 10 * width});
    }
  }
  return best;
}

template <class Kernel, class... Args>
cudaError_t launch_clusters(Kernel kernel, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

struct Operands {
  const void* x;
  const void* w;
  long long x_stride;                    // bytes
};

template <int BN, bool kMx8, int kMode>
int launch_split(const Operands& o, const LinearArgs& a, int split, cudaStream_t stream) {
  using C = SplitCfg<BN, kMx8>;
  static DeviceOnce setup;
  if (int rc = prepare(linear_split_kernel<BN, kMx8, kMode>, setup, C::kSmem)) return rc;
  CUtensorMap map_w, map_x;
  if (int rc = operand_map(&map_w, o.w, a.k_bytes, a.features, a.k_bytes, kTileRows)) return rc;
  if (int rc = operand_map(&map_x, o.x, a.k_bytes, a.rows, o.x_stride, BN)) return rc;
  const dim3 grid((unsigned)(ceil_div_i(a.features, kTileRows) * split), (unsigned)ceil_div_i(a.rows, BN));
  PNV_CUDA(launch_clusters(linear_split_kernel<BN, kMx8, kMode>, grid, C::kThreads, C::kSmem, split, stream, map_w, map_x, a, split));
  return PNV_OK;
}

template <bool kMx8, int kMode>
int launch_pair(const Operands& o, LinearArgs a, int width, int sm_count, cudaStream_t stream) {
  using C = PairCfg<kMx8>;
  static DeviceOnce setup;
  if (int rc = prepare(linear_pair_kernel<kMx8, kMode>, setup, C::kSmem)) return rc;
  a.tile_n = width;
  a.m_tiles = ceil_div_i(a.rows, 256);
  a.n_tiles = ceil_div_i(a.features, width);
  a.band = kLowBand;
  while (a.band < kHighBand && 2LL * a.band * 256 * a.k_bytes <= kBandBytes) a.band *= 2;
  const int pairs = std::min(sm_count / 2, a.m_tiles * a.n_tiles);
  CUtensorMap map_w, map_x, map_w_sf = {}, map_x_sf = {};
  if (int rc = operand_map(&map_w, o.w, a.k_bytes, a.features, a.k_bytes, a.tile_n / 2)) return rc;
  if (int rc = operand_map(&map_x, o.x, a.k_bytes, a.rows, o.x_stride, 128)) return rc;
  if (kMx8) {
    const int k_atoms = ceil_div_i(a.k_bytes, 128);
    if (int rc = scale_map(&map_w_sf, a.w_sf, sf_row_atoms(a.features), k_atoms, 2)) return rc;
    if (int rc = scale_map(&map_x_sf, a.x_sf, sf_row_atoms(a.rows), k_atoms, 1)) return rc;
  }
  a.tma = a.vec_out && (a.residual == nullptr || a.vec_residual);
  CUtensorMap map_out = {}, map_out_32 = {}, map_res = {}, map_res_32 = {};
  if (a.tma) {
    if (int rc = rows_map(&map_out, a.out, a.n_out, a.rows, a.n_out, 64)) return rc;
    if (int rc = rows_map(&map_out_32, a.out, a.n_out, a.rows, a.n_out, 32)) return rc;
    if (a.residual != nullptr) {
      if (int rc = rows_map(&map_res, a.residual, a.n_out, a.rows, a.residual_stride, 64)) return rc;
      if (int rc = rows_map(&map_res_32, a.residual, a.n_out, a.rows, a.residual_stride, 32)) return rc;
    }
  }
  PNV_CUDA(launch_clusters(linear_pair_kernel<kMx8, kMode>, dim3((unsigned)(2 * pairs)), C::kThreads, C::kSmem, 2, stream, map_w, map_x, map_w_sf,
                           map_x_sf, map_out, map_out_32, map_res, map_res_32, a));
  return PNV_OK;
}

template <bool kMx8, int kMode>
int run_linear(const Operands& o, const LinearArgs& a, int sm_count, cudaStream_t stream) {
  const int* clusters = nullptr;
  if (int rc = cluster_capacity(&clusters)) return rc;
  const Plan p = make_plan(a, kMx8, clusters, sm_count);
  PNV_REQUIRE(p.cost >= 0, "linear: too many rows for one call");
  switch (p.tokens) {
    case 0: return launch_pair<kMx8, kMode>(o, a, p.width, std::min(2 * clusters[1], sm_count), stream);
    case 16: return launch_split<16, kMx8, kMode>(o, a, p.split, stream);
    case 32: return launch_split<32, kMx8, kMode>(o, a, p.split, stream);
    case 64: return launch_split<64, kMx8, kMode>(o, a, p.split, stream);
    default: return launch_split<128, kMx8, kMode>(o, a, p.split, stream);
  }
}

bool at(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int linear_common(bool mx8, void* out, int out_is_f32, const void* x, long long x_stride, const uint8_t* x_sf, const void* w, const uint8_t* w_sf,
                  const void* bias, int bias_is_f32, const void* residual, long long residual_stride, long long rows, int features, int k,
                  int act_kind, int gated, float beta, float linear_beta, int sm_count, cudaStream_t stream) {
  PNV_REQUIRE(rows >= 0 && rows < (1LL << 31) - 256, "bad row count");
  PNV_REQUIRE(features >= 1 && k >= 1, "features and k must be positive");
  PNV_REQUIRE(features < (1 << 30) && k < (1 << 29), "features or k too large");
  LinearArgs a{};
  if (gated) {
    PNV_REQUIRE(act_kind == PNV_ACT_SILU || act_kind == PNV_ACT_SITU, "activation must be 'silu' or 'situ' when gated, got kind %d", act_kind);
    if (int rc = make_gated_act(act_kind, beta, linear_beta, a.act)) return rc;
    PNV_REQUIRE(features % 64 == 0, "gated: features (gates and ups in 64-row blocks) must be a multiple of 64, got %d", features);
  } else {
    PNV_REQUIRE(act_kind == PNV_ACT_NONE || act_kind == PNV_ACT_RELU || act_kind == PNV_ACT_SILU || act_kind == PNV_ACT_GELU,
                "activation must be 'none', 'relu', 'silu' or 'gelu' unless gated, got kind %d", act_kind);
  }
  const int n_out = gated ? features / 2 : features;
  if (mx8) PNV_REQUIRE(k % kSfBlock == 0, "K must be a multiple of %d, got %d", kSfBlock, k);
  else PNV_REQUIRE(k % 8 == 0, "K must be a multiple of 8, got %d", k);
  if (rows == 0) return PNV_OK;
  PNV_REQUIRE(out && x && w && (!mx8 || (x_sf && w_sf)), "null pointer argument");
  const long long k_bytes = mx8 ? k : 2LL * k, stride_bytes = mx8 ? x_stride : 2 * x_stride;
  PNV_REQUIRE(x_stride >= k && stride_bytes % 16 == 0, "rows of x must not overlap and start at multiples of 16 bytes");
  PNV_REQUIRE(at(x, 16) && at(w, 16), "the operands must be 16-byte aligned");
  PNV_REQUIRE(!mx8 || (at(x_sf, 16) && at(w_sf, 16)), "the scales must be 16-byte aligned");
  PNV_REQUIRE(at(out, out_is_f32 ? 4 : 2) && at(bias, bias_is_f32 ? 4 : 2) && at(residual, 2), "a buffer is not aligned to its elements");
  PNV_REQUIRE(residual == nullptr || residual_stride >= n_out, "rows of the residual must not overlap");
  a.out = out;
  a.bias = bias;
  a.residual = static_cast<const __nv_bfloat16*>(residual);
  a.x_sf = x_sf;
  a.w_sf = w_sf;
  a.residual_stride = residual_stride;
  a.rows = (int)rows;
  a.features = features;
  a.n_out = n_out;
  a.k_bytes = (int)k_bytes;
  a.out_f32 = out_is_f32;
  a.bias_f32 = bias_is_f32;
  a.gated = gated;
  a.kind = act_kind;
  // (pieces of a row start at multiples of 8 outputs)
  a.vec_out = (long long)n_out * (out_is_f32 ? 4 : 2) % 16 == 0 && at(out, 16);
  a.vec_residual = residual_stride % 8 == 0 && at(residual, 16);
  a.vec_bias = at(bias, 16);
  if (sm_count <= 0) sm_count = 148;
  const Operands o{x, w, stride_bytes};
  if (gated) return mx8 ? run_linear<true, kGate>(o, a, sm_count, stream) : run_linear<false, kGate>(o, a, sm_count, stream);
  if (act_kind != PNV_ACT_NONE)
    return mx8 ? run_linear<true, kActivate>(o, a, sm_count, stream) : run_linear<false, kActivate>(o, a, sm_count, stream);
  return mx8 ? run_linear<true, kNothing>(o, a, sm_count, stream) : run_linear<false, kNothing>(o, a, sm_count, stream);
}

}  // namespace
}  // namespace pnv

using namespace pnv;

extern "C" int pnv_linear(void* out, int out_is_f32, const void* x, int64_t x_stride, const void* w, const void* bias, int bias_is_f32,
                          const void* residual, int64_t residual_stride, int64_t rows, int features, int k, int act_kind, int gated,
                          float beta, float linear_beta, int sm_count, pnv_stream_t stream) {
  return linear_common(false, out, out_is_f32, x, x_stride, nullptr, w, nullptr, bias, bias_is_f32, residual, residual_stride, rows,
                       features, k, act_kind, gated, beta, linear_beta, sm_count, (cudaStream_t)stream);
}

extern "C" int pnv_linear_mx8(void* out, const uint8_t* x, const uint8_t* x_sf, const uint8_t* w, const uint8_t* w_sf, const void* bias,
                              int bias_is_f32, const void* residual, int64_t residual_stride, int64_t rows, int features, int k,
                              int act_kind, int gated, float beta, float linear_beta, int sm_count, pnv_stream_t stream) {
  return linear_common(true, out, 0, x, k, x_sf, w, w_sf, bias, bias_is_f32, residual, residual_stride, rows, features, k, act_kind, gated,
                       beta, linear_beta, sm_count, (cudaStream_t)stream);
}

extern "C" int pnv_linear_plan(int mx8, int64_t rows, int features, int k, int out_is_f32, int gated, int sm_count, int* tokens, int* split,
                               int* width) {
  PNV_REQUIRE(tokens && split && width, "null pointer argument");
  PNV_REQUIRE(rows >= 1 && rows < (1LL << 31) - 256 && features >= 1 && features < (1 << 30) && k >= 1 && k < (1 << 29), "sizes out of range");
  LinearArgs a{};
  a.rows = (int)rows;
  a.features = features;
  a.k_bytes = mx8 ? k : 2 * k;
  a.out_f32 = out_is_f32;
  a.gated = gated;
  const int* clusters = nullptr;
  if (int rc = cluster_capacity(&clusters)) return rc;
  const Plan p = make_plan(a, mx8 != 0, clusters, sm_count > 0 ? sm_count : 148);
  PNV_REQUIRE(p.cost >= 0, "linear: too many rows for one call");
  *tokens = p.tokens;
  *split = p.split;
  *width = p.width;
  return PNV_OK;
}

extern "C" int pnv_linear_device_status(int* status_out) {
  PNV_REQUIRE(status_out, "null pointer argument");
  PNV_CUDA(cudaDeviceSynchronize());
  PNV_CUDA(cudaMemcpyFromSymbol(status_out, g_linear_status, sizeof(int)));
  int zero = 0;
  PNV_CUDA(cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int)));
  return PNV_OK;
}
