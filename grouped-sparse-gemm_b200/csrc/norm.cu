// The root-mean-square norm ahead of a block, with the residual's addition, and the 8-bit quantizer of the dense products.
//
//   v = x + residual;  n = v / sqrt(mean(v^2) + eps) * weight        (all in 32 bits)
//   residual_out = bf16(v), y = bf16(n), (q, q_sf) = 8-bit codes of n
// Codes and y are both rounded from n itself: codes made of the rounded y would carry two roundings.
//
// The 8-bit format: e4m3 codes with one e8m0 scale (a power of two, byte b stands for 2^(b - 127)) per 32 elements, the
// smallest that leaves the block's largest magnitude at 448 or below, so that no element saturates; a block of zeros has
// scale 1, a block that holds an infinity or a NaN scale byte 0xFF (NaN) and NaN codes.  Scales lie in the same 512-byte
// atoms as the grouped GEMM's (common.cuh), slop filled with 1.0: a product multiplies what it finds there by zeros.
#include "common.cuh"
#include "mx8.cuh"

namespace pnv {
namespace {

constexpr int kVecElems = 8;             // elements a lane holds of each of its pieces: 16 bytes of bf16

struct NormArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* residual;         // or nullptr
  const void* weight;
  __nv_bfloat16* y;                      // or nullptr
  __nv_bfloat16* residual_out;
  uint8_t* q;                            // or nullptr
  uint8_t* q_sf;
  long long x_stride, residual_stride;
  long long rows, padded_rows;           // rows up to padded_rows only have scales, of slop
  int width, weight_f32;
  int team;                              // threads per row, a multiple of 32; a block has one row where it is above 32
  float eps;
};

// How a lane reaches the eight neighbouring elements of one of its pieces, piece i of a row.
//   kWhole    elements 8 i to 8 i + 7, one 16-byte access
//   kShifted  rows that start anywhere, at the same place within 16 bytes in every buffer: elements 8 i - s on, where s is how far
//             the row starts behind a 16-byte boundary, so that all accesses but a row's first and last are whole
//   kSingle   elements 8 i on, one by one
enum Access : int { kWhole = 0, kShifted = 1, kSingle = 2 };

// Elements at, at + 1, ... of a row of `width` (zeros outside of it).
template <int kAccess>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int at, int width) {
  if constexpr (kAccess == kWhole) {
    return __ldg(reinterpret_cast<const uint4*>(row + at));
  } else {
    if (kAccess == kShifted && at >= 0 && at + 8 <= width) return __ldg(reinterpret_cast<const uint4*>(row + at));
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      h[j] = at + j >= 0 && at + j < width ? __ldg(reinterpret_cast<const unsigned short*>(row) + at + j) : 0u;
    return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
}
template <int kAccess>
__device__ __forceinline__ void store8(__nv_bfloat16* row, int at, int width, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = as_u32(__floats2bfloat162_rn(f[2 * j], f[2 * j + 1]));
  if (kAccess == kWhole || (kAccess == kShifted && at >= 0 && at + 8 <= width)) {
    *reinterpret_cast<uint4*>(row + at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j >= 0 && at + j < width)
        reinterpret_cast<unsigned short*>(row)[at + j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
  }
}
// Eight weights from element `at` on.  Shifted, they are cut out of the two whole pieces that hold them: shift = elements by which
// `at` is short of the second one's start, the same for a row.
template <int kAccess>
__device__ __forceinline__ void load_weight8(const void* weight, int f32, int at, int shift, int width, float (&w)[8]) {
  if (f32) {
    const float* p = static_cast<const float*>(weight) + at;
    if (kAccess == kWhole) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = at + j >= 0 && at + j < width ? __ldg(p + j) : 0.f;
    }
    return;
  }
  const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(weight);
  if constexpr (kAccess != kShifted) {
    unpack8(load8<kAccess>(p, at, width), w);
  } else {
    const uint4 hi = load8<kShifted>(p, at + shift, width);
    if (shift == 0) {
      unpack8(hi, w);
      return;
    }
    const uint4 lo = load8<kShifted>(p, at + shift - 8, width);
    uint32_t v[9] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, 0u};
    const int skip = 8 - shift;          // elements of the first piece that are not wanted
    if (skip & 4) {
#pragma unroll
      for (int j = 0; j < 6; ++j) v[j] = v[j + 2];
    }
    if (skip & 2) {
#pragma unroll
      for (int j = 0; j < 5; ++j) v[j] = v[j + 1];
    }
    if (skip & 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __funnelshift_r(v[j], v[j + 1], 16);
    }
    unpack8(make_uint4(v[0], v[1], v[2], v[3]), w);
  }
}

// A team of `team` threads takes a row and keeps all of it in registers, V pieces of eight elements a thread, so that
// memory is read once.  Bound: HBM (9 bytes and 1/32 per element with both outputs): 16384 x 7168 in 159 to 167 us, 6.35 to 6.67
// TB/s, in a loop of seconds 171 to 179, 0.90 to 0.95 of a copy: power takes the clock to 1.63 GHz there.
template <int V, int kAccess>
__global__ void __launch_bounds__(512)
add_rms_norm_kernel(const NormArgs a) {
  __shared__ float s_sum[16];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x % a.team, per_block = blockDim.x / a.team;
  const long long row = (long long)blockIdx.x * per_block + threadIdx.x / a.team;
  const int n_kt = (a.width + 127) / 128;
  uint8_t* sf_row = a.q_sf + ((row >> 7) * n_kt) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
  if (row >= a.rows) {                   // (whole teams, so whole warps; with team > 32 the whole block)
    if (a.q != nullptr && row < a.padded_rows)
      for (int i = lane; i < n_kt; i += a.team) *reinterpret_cast<uint32_t*>(sf_row + i * 512LL) = kMx8SlopWord;
    return;
  }
  const int shift = kAccess == kShifted ? (int)((unsigned)row * (unsigned)a.width & 7u) : 0;
  const int n = (a.width + shift + kVecElems - 1) / kVecElems;
  const __nv_bfloat16* x = a.x + row * a.x_stride;
  float v[V][8];
  float sum = 0.f;
  {
    uint4 raw[V];
#pragma unroll
    for (int p = 0; p < V; ++p) {
      const int i = p * a.team + lane;
      raw[p] = i < n ? load8<kAccess>(x, 8 * i - shift, a.width) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (a.residual != nullptr) {
      const __nv_bfloat16* r = a.residual + row * a.residual_stride;
      uint4 more[V];
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const int i = p * a.team + lane;
        more[p] = i < n ? load8<kAccess>(r, 8 * i - shift, a.width) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const int i = p * a.team + lane;
        float f[8];
        unpack8(raw[p], v[p]);
        unpack8(more[p], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[p][j] += f[j];
        if (i < n) store8<kAccess>(a.residual_out + row * a.width, 8 * i - shift, a.width, v[p]);
      }
    } else {
#pragma unroll
      for (int p = 0; p < V; ++p) unpack8(raw[p], v[p]);
    }
  }
  // squares are added eight by eight, then those sums: in one chain of 40 the roundings add up to what moves a code in a million
#pragma unroll
  for (int p = 0; p < V; ++p) {
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = fmaf(v[p][2 * j + 1], v[p][2 * j + 1], v[p][2 * j] * v[p][2 * j]);
    sum += (s[0] + s[1]) + (s[2] + s[3]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (a.team > 32) {
    if ((lane & 31) == 0) s_sum[lane >> 5] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < a.team / 32; ++w) sum += s_sum[w];
  }
  const float rstd = __frsqrt_rn(__fdiv_rn(sum, (float)a.width) + a.eps);
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const int i = p * a.team + lane;
    if (i < n) {
      float w[8];
      load_weight8<kAccess>(a.weight, a.weight_f32, 8 * i - shift, shift, a.width, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[p][j] = __fmul_rn(__fmul_rn(v[p][j], rstd), w[j]);
      if (a.y != nullptr) store8<kAccess>(a.y + row * a.width, 8 * i - shift, a.width, v[p]);
    }
    if (kAccess != kShifted && a.q != nullptr) {       // four lanes hold a block, sixteen the four blocks of a word of scales
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[p][j]) & 0x7FFFFFFFu);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t byte = i < n ? mx8_scale_byte(m) : kMx8One;
      if (i < n) {
        const float inv = mx8_inverse(byte);
        reinterpret_cast<uint2*>(a.q + row * a.width)[i] = make_uint2(mx8_codes4(v[p], 0, byte, inv), mx8_codes4(v[p], 4, byte, inv));
      }
      uint32_t word = byte << (8 * ((lane >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      if ((lane & 15) == 0 && (i >> 4) < n_kt) *reinterpret_cast<uint32_t*>(sf_row + (i >> 4) * 512LL) = word;
    }
  }
}

constexpr int kQuantThreads = 256;

// A lane takes a block of 32 elements, four lanes the blocks of one word of scales ("quad": 128 elements of a row).  Quads
// of all rows are laid end to end, rows padded to whole atoms among them: their scales are written here too.  Bound: HBM
// (8192 x 14336: 53 us, 356 MB at 6.7 TB/s).
__global__ void __launch_bounds__(kQuantThreads)
quant_mx8_kernel(const __nv_bfloat16* __restrict__ x, long long x_stride, unsigned rows, unsigned quads, int K, int n_kt,
                 uint8_t* __restrict__ q, uint8_t* __restrict__ q_sf) {
  pdl_wait();
  pdl_launch_dependents();
  const unsigned quad = blockIdx.x * (kQuantThreads / 4) + threadIdx.x / 4;
  const unsigned row = quad / (unsigned)n_kt;
  const int atom = (int)(quad - row * (unsigned)n_kt), part = threadIdx.x & 3;
  const int kb = atom * 4 + part;
  uint32_t byte = kMx8One;
  if (quad < quads && row < rows && kb < K / kSfBlock) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(x + row * x_stride) + kb * 64LL;
    uint32_t w[16];
    if (((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(x_stride * 2)) & 31) == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(w[8 * h]), "=r"(w[8 * h + 1]), "=r"(w[8 * h + 2]), "=r"(w[8 * h + 3]), "=r"(w[8 * h + 4]), "=r"(w[8 * h + 5]),
              "=r"(w[8 * h + 6]), "=r"(w[8 * h + 7]) : "l"(src + 32 * h) : "memory");
    } else {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint4 t = __ldg(reinterpret_cast<const uint4*>(src) + h);
        w[4 * h] = t.x; w[4 * h + 1] = t.y; w[4 * h + 2] = t.z; w[4 * h + 3] = t.w;
      }
    }
    uint32_t m = 0;                      // magnitudes of bf16 numbers order like their bits, infinities and NaNs above all
#pragma unroll
    for (int i = 0; i < 16; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    byte = mx8_scale_byte(max(m & 0xFFFFu, m >> 16) << 16);
    const float inv = mx8_inverse(byte);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f[4] = {bf16_lo(w[2 * i]), bf16_hi(w[2 * i]), bf16_lo(w[2 * i + 1]), bf16_hi(w[2 * i + 1])};
      c[i] = mx8_codes4(f, 0, byte, inv);
    }
    uint4* dst = reinterpret_cast<uint4*>(q + (long long)row * K + kb * 32LL);
    dst[0] = make_uint4(c[0], c[1], c[2], c[3]);
    dst[1] = make_uint4(c[4], c[5], c[6], c[7]);
  }
  uint32_t word = byte << (8 * part);
  word |= __shfl_xor_sync(0xffffffffu, word, 1);
  word |= __shfl_xor_sync(0xffffffffu, word, 2);
  if (part == 0 && quad < quads)
    *reinterpret_cast<uint32_t*>(q_sf + ((long long)(row >> 7) * n_kt + atom) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4) = word;
}

template <int V>
cudaError_t launch_norm(const NormArgs& a, Access access, dim3 grid, dim3 block, cudaStream_t s) {
  return launch_pdl(access == kWhole ? add_rms_norm_kernel<V, kWhole> : access == kShifted ? add_rms_norm_kernel<V, kShifted>
                                                                                          : add_rms_norm_kernel<V, kSingle>,
                    grid, block, 0, s, pdl_enabled(), a);
}

bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace pnv

using namespace pnv;

extern "C" int pnv_add_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                                int weight_is_f32, float eps, int64_t rows, int width, void* y, void* residual_out, uint8_t* q,
                                uint8_t* q_sf, int sm_count, pnv_stream_t stream) {
  PNV_REQUIRE(rows >= 0 && rows < (1LL << 31), "bad row count");
  PNV_REQUIRE(width >= 1 && width <= PNV_NORM_MAX_WIDTH, "add_rms_norm: rows of 1 to %d elements, got %d", PNV_NORM_MAX_WIDTH, width);
  PNV_REQUIRE(y != nullptr || q != nullptr, "add_rms_norm: at least one of y and q is written");
  PNV_REQUIRE((q == nullptr) == (q_sf == nullptr), "null pointer argument");
  PNV_REQUIRE(q == nullptr || width % kSfBlock == 0, "8-bit output: the width must be a multiple of %d, got %d", kSfBlock, width);
  PNV_REQUIRE(eps >= 0.f, "eps must not be negative");
  if (rows == 0) return PNV_OK;
  PNV_REQUIRE(x && weight && (residual == nullptr) == (residual_out == nullptr), "null pointer argument");
  PNV_REQUIRE(x_stride >= width && (residual == nullptr || residual_stride >= width), "rows must not overlap");
  PNV_REQUIRE(aligned_to(x, 2) && aligned_to(residual, 2) && aligned_to(weight, weight_is_f32 ? 4 : 2) && aligned_to(y, 2) &&
                  aligned_to(residual_out, 2) && aligned_to(q, 8) && aligned_to(q_sf, 4),
              "add_rms_norm: a buffer is not aligned to its elements (codes 8 bytes, scales 4)");
  // Whole 16-byte accesses; else shifted ones, where all rows lie alike within 16 bytes (odd widths, 8-bit output not among them);
  // else element by element.  16384 x 4097, bf16 output and residual: 132 us shifted, 316 element by element (4096: 80 whole).
  const bool aligned = aligned_to(x, 16) && aligned_to(residual, 16) && aligned_to(weight, 16) && aligned_to(y, 16) && aligned_to(residual_out, 16);
  const bool alike = x_stride % 8 == width % 8 && (residual == nullptr || residual_stride % 8 == width % 8);
  const Access access = !aligned || !alike ? kSingle : width % 8 == 0 ? kWhole : width + 7 <= PNV_NORM_MAX_WIDTH ? kShifted : kSingle;
  const int n = ceil_div_i(width + (access == kShifted ? 7 : 0), kVecElems);
  if (sm_count <= 0) sm_count = 148;
  // Many rows: as few threads a row as hold it with five pieces each (16384 x 7168 with both outputs: 167 us; with seven 180,
  // the fewer rows of an SM are then not enough to keep memory busy while one of them is added up; with three 228).  Rows that
  // leave SMs without work: two pieces each (up to 512 threads), so that a row takes as little time as it can.
  int team = 32;
  while (team < 512 && ceil_div_i(n, team) > (rows <= 2LL * sm_count ? 2 : 5)) team *= 2;
  const int threads = team > 32 ? team : 128;
  NormArgs a{(const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, weight, (__nv_bfloat16*)y, (__nv_bfloat16*)residual_out, q, q_sf,
             x_stride, residual_stride, rows, q ? (rows + 127) / 128 * 128 : rows, width, weight_is_f32, team, eps};
  const long long blocks = (a.padded_rows + threads / team - 1) / (threads / team);
  const dim3 grid((unsigned)blocks), block((unsigned)threads);
  cudaStream_t s = (cudaStream_t)stream;
  switch (ceil_div_i(n, team)) {
    case 1: PNV_CUDA(launch_norm<1>(a, access, grid, block, s)); break;
    case 2: PNV_CUDA(launch_norm<2>(a, access, grid, block, s)); break;
    case 3: PNV_CUDA(launch_norm<3>(a, access, grid, block, s)); break;
    case 4: PNV_CUDA(launch_norm<4>(a, access, grid, block, s)); break;
    case 5: PNV_CUDA(launch_norm<5>(a, access, grid, block, s)); break;
    case 6: PNV_CUDA(launch_norm<6>(a, access, grid, block, s)); break;
    case 7: PNV_CUDA(launch_norm<7>(a, access, grid, block, s)); break;
    default: PNV_CUDA(launch_norm<8>(a, access, grid, block, s)); break;
  }
  return PNV_OK;
}

extern "C" int pnv_quant_mx8(const void* x, int64_t x_stride, int64_t rows, int k, uint8_t* q, uint8_t* q_sf, pnv_stream_t stream) {
  PNV_REQUIRE(k > 0 && k % kSfBlock == 0, "K must be a multiple of %d, got %d", kSfBlock, k);
  PNV_REQUIRE(rows >= 0 && rows < (1LL << 31), "bad row count");
  if (rows == 0) return PNV_OK;
  PNV_REQUIRE(x && q && q_sf, "null pointer argument");
  PNV_REQUIRE(x_stride >= k && x_stride % 8 == 0, "rows must not overlap and start at multiples of 16 bytes");
  PNV_REQUIRE(aligned_to(x, 16) && aligned_to(q, 16) && aligned_to(q_sf, 4),
              "quant_mx8: the bf16 rows and the codes must be 16-byte aligned, the scales 4-byte");
  const int n_kt = sf_k_atoms(k);
  const long long quads = (rows + 127) / 128 * 128 * n_kt;
  PNV_REQUIRE(quads < (1LL << 32) - kQuantThreads, "too many rows");
  PNV_CUDA(launch_pdl(quant_mx8_kernel, dim3((unsigned)((quads + kQuantThreads / 4 - 1) / (kQuantThreads / 4))), dim3(kQuantThreads), 0,
                      (cudaStream_t)stream, pdl_enabled(), (const __nv_bfloat16*)x, (long long)x_stride, (unsigned)rows, (unsigned)quads, k,
                      n_kt, q, q_sf));
  return PNV_OK;
}
