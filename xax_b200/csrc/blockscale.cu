// Block-scaled e4m3 casts: one float32 multiplier per 128 columns of a row (activations) or per 128 x 128 square
// (weights), alone and fused behind RMSNorm (with the residual's addition) and SiLU(gate) * up.
//
//   amax = max |v| over the block
//   inv  = max(amax * (1/448), 2^-126); 1 where amax is 0, infinite or NaN
//   q    = e4m3(v * (1/inv)), round to nearest even, clipped to +-448; NaN stays NaN
//
// so the block stands for q * inv.  Everything between the bf16 inputs and q is float32: one rounding to 8 bits at
// the end (the floor of 2^-126 keeps 1/inv finite; with it the largest value of a normal block lands on 448).
//
// All are bandwidth kernels.  A thread owns 16 consecutive values: one 32-byte load (half the load instructions of two
// 16-byte ones, and whole sectors), one 16-byte store; the eight threads of a block of 128 are eight neighbouring lanes
// and its maximum takes three shuffles.  Measured, of the copy rate: 8192 x 4096 by rows 16.6 us = 0.93, 14336 x 4096 by squares
// 29.2 us = 0.92, RMSNorm with residual of 8192 x 4096 36.6 us = 0.98.  Decode-sized calls take 2 to 4 us on the GPU.
#include "common.cuh"
#include "quant_device.cuh"

namespace xaxb {

constexpr int kPiece = 16;               // values per thread and piece
constexpr int kBlockPieces = 128 / kPiece;

struct Packed16 {  // 16 bf16
  uint32_t w[8];
};

__device__ __forceinline__ Packed16 load16(const __nv_bfloat16* p) {
  Packed16 r;
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
               : "l"(p));
  return r;
}

__device__ __forceinline__ void store16(__nv_bfloat16* p, const Packed16& r) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]), "l"(p)
               : "memory");
}

__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Magnitudes compare as unsigned bit patterns, which puts NaN above infinity: a NaN in a block reaches its amax.
__device__ __forceinline__ uint32_t magnitude16(const float (&v)[kPiece]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kPiece; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return m;
}
__device__ __forceinline__ uint32_t magnitude16(const Packed16& p) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = __vmaxu2(m, p.w[j] & 0x7FFF7FFFu);
  return max(m << 16, m & 0xFFFF0000u);
}

__device__ __forceinline__ uint32_t lanes8_max(uint32_t m) {
#pragma unroll
  for (int o = 1; o < kBlockPieces; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ float block_inv_scale(uint32_t amax_bits) {
  const float inv = fmaxf(__uint_as_float(amax_bits) * (1.0f / 448.0f), 0x1p-126f);
  return amax_bits == 0 || amax_bits >= 0x7F800000u ? 1.0f : inv;
}

__device__ __forceinline__ uint4 cast16(const float (&v)[kPiece], float scale) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = e4m3x2(v[4 * j] * scale, v[4 * j + 1] * scale) | (e4m3x2(v[4 * j + 2] * scale, v[4 * j + 3] * scale) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 cast16(const Packed16& p, float scale) {
  float v[kPiece];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[2 * j] = low(p.w[j]), v[2 * j + 1] = high(p.w[j]);
  return cast16(v, scale);
}

// n / d for n < 2^31 by a multiplication with a precomputed reciprocal: with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(m, n) + n) >> l.
struct FastDiv {
  uint32_t d, m, l;
};
static FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while (l < 32 && (1ull << l) < d) ++l;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), l};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv f) { return (__umulhi(f.m, n) + n) >> f.l; }

// ---- bf16 rows, a block per 128 columns.  Piece number p = row * pieces_per_row + (columns / 16), rows padded to
// whole blocks, so inv[p / 8] is the block's place in the row-major [rows, blocks] result for every width.
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const __nv_bfloat16* __restrict__ x, uint32_t pieces,
                                                              FastDiv per_row, int cols, uint8_t* __restrict__ q,
                                                              float* __restrict__ inv) {
  pdl_trigger();
  const uint32_t p = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = div_by(p, per_row), col = (p - row * per_row.d) * kPiece;
  const bool here = p < pieces && col < (uint32_t)cols;
  const int64_t at = (int64_t)row * cols + col;
  pdl_wait();
  Packed16 v = {};
  if (here) v = load16(x + at);
  const float s = block_inv_scale(lanes8_max(magnitude16(v)));
  if (here) {
    *reinterpret_cast<uint4*>(q + at) = cast16(v, 1.0f / s);
    if (p % kBlockPieces == 0) inv[p / kBlockPieces] = s;
  }
}

// ---- 128 x 128 squares: one CTA each, four pieces per thread kept (packed) in registers across the maximum.
__global__ void __launch_bounds__(256) quantize_squares_kernel(const __nv_bfloat16* __restrict__ x, int64_t rows, int cols,
                                                               uint8_t* __restrict__ q, float* __restrict__ inv) {
  pdl_trigger();
  __shared__ uint32_t warp_max[8];
  const int64_t row0 = (int64_t)blockIdx.x * 128 + threadIdx.x / kBlockPieces;
  const int col = blockIdx.y * 128 + (threadIdx.x % kBlockPieces) * kPiece;
  pdl_wait();
  Packed16 v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    v[u] = {};
    if (row0 + u * 32 < rows && col < cols) v[u] = load16(x + (row0 + u * 32) * cols + col);
  }
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) m = max(m, magnitude16(v[u]));
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, warp_max[i]);
  const float s = block_inv_scale(m), r = 1.0f / s;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (row0 + u * 32 < rows && col < cols) *reinterpret_cast<uint4*>(q + (row0 + u * 32) * cols + col) = cast16(v[u], r);
  if (threadIdx.x == 0) inv[(int64_t)blockIdx.x * gridDim.y + blockIdx.y] = s;
}

// ---- RMSNorm of x (+ residual): t = x + residual and the norm in float32, one CTA per row, the row in registers.  A row
// is one dependent chain (load, sum over the CTA, normalise, maximum, store), so an SM overlaps as many as it has CTAs:
// many rows run narrow CTAs with more pieces per thread, few rows spread over more threads.
template <int NP, int NT>
__global__ void __launch_bounds__(NT) rmsnorm_blocks_kernel(const __nv_bfloat16* __restrict__ x,
                                                            const __nv_bfloat16* __restrict__ residual,
                                                            const __nv_bfloat16* __restrict__ weight, float eps, int cols,
                                                            int blocks, __nv_bfloat16* __restrict__ sum,
                                                            uint8_t* __restrict__ q, float* __restrict__ inv) {
  pdl_trigger();
  __shared__ float warp_sum[NT / 32];
  const int64_t row = blockIdx.x;
  pdl_wait();
  constexpr bool kWeightEarly = NP <= 2;  // off the chain behind the sum, where registers allow
  Packed16 px[NP], pr[NP], pw[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (threadIdx.x + k * NT) * kPiece;
    px[k] = {}, pr[k] = {};
    if (col < cols) px[k] = load16(x + row * cols + col);
    if (col < cols && residual) pr[k] = load16(residual + row * cols + col);
    if (col < cols && kWeightEarly) pw[k] = load16(weight + col);
  }
  float v[NP][kPiece];
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (threadIdx.x + k * NT) * kPiece;
    Packed16 total;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[k][2 * j] = low(px[k].w[j]) + low(pr[k].w[j]);
      v[k][2 * j + 1] = high(px[k].w[j]) + high(pr[k].w[j]);
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(total.w[j]) : "f"(v[k][2 * j + 1]), "f"(v[k][2 * j]));
    }
    if (col < cols && residual) store16(sum + row * cols + col, total);
#pragma unroll
    for (int j = 0; j < kPiece; ++j) ss = fmaf(v[k][j], v[k][j], ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) ss += warp_sum[i];
  const float n = 1.0f / sqrtf(ss / (float)cols + eps);  // both correctly rounded: once per thread and row
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int piece = threadIdx.x + k * NT, col = piece * kPiece;
    if (col < cols) {
      const Packed16 w = kWeightEarly ? pw[k] : load16(weight + col);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[k][2 * j] *= n * low(w.w[j]);
        v[k][2 * j + 1] *= n * high(w.w[j]);
      }
    }
    const float s = block_inv_scale(lanes8_max(magnitude16(v[k])));
    if (col < cols) {
      *reinterpret_cast<uint4*>(q + row * cols + col) = cast16(v[k], 1.0f / s);
      if (piece % kBlockPieces == 0) inv[row * blocks + piece / kBlockPieces] = s;
    }
  }
}

// ---- silu(gate) * up, gate and up the two halves of a row of the fused gate | up product.

// 4 / (1 + e^x) to a few units: e^x = 2^h (1 + l) with h = x log2 e rounded and l = x - h ln 2, from the approximate
// exponential and reciprocal (2^-22 each).  x is kept from -88 up, where e^x is nothing beside 1, and h below 128; past
// that e^x is infinite in float32 and the result 0.  NaN comes back in the product with the gate.  (Four times the value,
// since the reciprocal itself would be denormal, and flushed, from x = 87.3 up, where gate times it is not yet.)
__device__ __forceinline__ float four_over_one_plus_exp(float x) {
  x = fmaxf(x, -88.0f);
  const float h = fminf(x * 1.4426950408889634f, 127.99999f);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(h));
  e = fmaf(e, fmaf(h, -0.6931471805599453f, x), e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0.25f, 0.25f)));
  return r;
}

__device__ __forceinline__ float silu_mul(float g, float u) { return 0.25f * g * four_over_one_plus_exp(-g) * u; }

// A grid of resident CTAs walks the pieces; the next piece's loads are under way while one is computed.  An exponential, a
// reciprocal and a dozen more instructions per value take about as long as its bytes (4099 x 5632: 20.5 us = 5.7 TB/s, 0.86
// of the copy rate, with 55 % of the special-function unit and 70 % of the issue slots; 27.5 us with the library's
// exponential and division or with approximations that treat denormals).
__global__ void __launch_bounds__(256) silu_mul_blocks_kernel(const __nv_bfloat16* __restrict__ gate_up, int64_t ld,
                                                              uint32_t pieces, FastDiv per_row, int dim,
                                                              uint8_t* __restrict__ q, float* __restrict__ inv) {
  pdl_trigger();
  const uint32_t step = gridDim.x * 256u;
  Packed16 g, u;
  auto ask = [&](uint32_t p) {
    const uint32_t row = div_by(p, per_row), col = (p - row * per_row.d) * kPiece;
    g = {}, u = {};
    if (p < pieces && col < (uint32_t)dim) {
      g = load16(gate_up + row * ld + col);
      u = load16(gate_up + row * ld + dim + col);
    }
  };
  uint32_t p = blockIdx.x * 256u + threadIdx.x;
  pdl_wait();
  ask(p);
  // (pieces is a multiple of 8 and CTAs start at multiples of 256: the eight lanes of a block stay together.  p cannot
  // wrap: pieces < 2^31 and step < 2^20.)
  for (uint32_t base = blockIdx.x * 256u; base < pieces; base += step, p += step) {
    const Packed16 gn = g, un = u;
    if (base + step < pieces) ask(p + step);
    float h[kPiece];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[2 * j] = silu_mul(low(gn.w[j]), low(un.w[j]));
      h[2 * j + 1] = silu_mul(high(gn.w[j]), high(un.w[j]));
    }
    const float s = block_inv_scale(lanes8_max(magnitude16(h)));
    const uint32_t row = div_by(p, per_row), col = (p - row * per_row.d) * kPiece;
    if (p < pieces && col < (uint32_t)dim) {
      *reinterpret_cast<uint4*>(q + (int64_t)row * dim + col) = cast16(h, 1.0f / s);
      if (p % kBlockPieces == 0) inv[p / kBlockPieces] = s;
    }
  }
}

static bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// What the four casts ask of a [rows, cols] result.
static int check_rows(const char* what, int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols % kPiece != 0) {
    set_last_error("%s: rows (%lld) must be positive and the width (%lld) a positive multiple of %d", what, (long long)rows,
                   (long long)cols, kPiece);
    return XAXB_BAD_ARGUMENT;
  }
  if (cols > (1 << 24) || rows > 0x7fffffff || rows * ((cols + 127) / 128) * kBlockPieces > 0x7fffff00ll) {
    set_last_error("%s: [%lld, %lld] has more than 2^31 pieces of %d values", what, (long long)rows, (long long)cols, kPiece);
    return XAXB_BAD_ARGUMENT;
  }
  return XAXB_OK;
}

template <int NP, int NT>
static void launch_rmsnorm_blocks(cudaStream_t s, const void* x, const void* residual, const void* weight, float eps,
                                  int64_t rows, int cols, void* sum, void* q, float* inv) {
  launch_kernel(rmsnorm_blocks_kernel<NP, NT>, dim3((unsigned)rows), dim3(NT), 0, s, 1, static_cast<const __nv_bfloat16*>(x),
                static_cast<const __nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(weight), eps, cols,
                (cols + 127) / 128, static_cast<__nv_bfloat16*>(sum), static_cast<uint8_t*>(q), inv);
}

}  // namespace xaxb

using namespace xaxb;

extern "C" {

int xaxb_quantize_blocks(xaxb_ctx* ctx, void* stream, const void* x_bf16, int64_t rows, int64_t cols, int block_rows,
                         void* q_e4m3, float* inv_scale) {
  if (!ctx || !x_bf16 || !q_e4m3 || !inv_scale || misaligned(x_bf16, 32) || misaligned(q_e4m3, 16) ||
      (block_rows != 1 && block_rows != 128)) {
    set_last_error("quantize_blocks: x must be 32-byte aligned, q 16-byte aligned, block_rows 1 or 128");
    return XAXB_BAD_ARGUMENT;
  }
  if (int rc = check_rows("quantize_blocks", rows, cols)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(x_bf16);
  const int64_t blocks = (cols + 127) / 128;
  if (block_rows == 128) {
    if (blocks > 65535) {
      set_last_error("quantize_blocks: at most 65535 squares side by side");
      return XAXB_BAD_ARGUMENT;
    }
    launch_kernel(quantize_squares_kernel, dim3((unsigned)((rows + 127) / 128), (unsigned)blocks), dim3(256), 0, s, 1, x, rows,
                  (int)cols, static_cast<uint8_t*>(q_e4m3), inv_scale);
    return check_launch("quantize_squares_kernel");
  }
  const uint32_t per_row = (uint32_t)(blocks * kBlockPieces), pieces = (uint32_t)(rows * per_row);
  launch_kernel(quantize_blocks_kernel, dim3((pieces + 255) / 256), dim3(256), 0, s, 1, x, pieces, fast_div(per_row), (int)cols,
                static_cast<uint8_t*>(q_e4m3), inv_scale);
  return check_launch("quantize_blocks_kernel");
}

int xaxb_rmsnorm_blocks(xaxb_ctx* ctx, void* stream, const void* x_bf16, const void* residual_bf16, const void* weight_bf16,
                        float eps, int64_t rows, int64_t cols, void* sum_bf16, void* q_e4m3, float* inv_scale) {
  if (!ctx || !x_bf16 || !weight_bf16 || !q_e4m3 || !inv_scale || (residual_bf16 != nullptr) != (sum_bf16 != nullptr) ||
      misaligned(x_bf16, 32) || misaligned(residual_bf16, 32) || misaligned(weight_bf16, 32) || misaligned(sum_bf16, 32) ||
      misaligned(q_e4m3, 16)) {
    set_last_error("rmsnorm_blocks: bf16 tensors must be 32-byte aligned, q 16-byte aligned; a sum goes with a residual");
    return XAXB_BAD_ARGUMENT;
  }
  if (int rc = check_rows("rmsnorm_blocks", rows, cols)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int pieces = (int)((cols + 127) / 128) * kBlockPieces;
  if (pieces > 2048) {
    set_last_error("rmsnorm_blocks: rows of at most 32768 values, got %lld", (long long)cols);
    return XAXB_UNSUPPORTED;
  }
  const bool many = rows >= 4 * reinterpret_cast<const Ctx*>(ctx)->num_sms;
#define XAXB_NORM(NP, NT) \
  launch_rmsnorm_blocks<NP, NT>(s, x_bf16, residual_bf16, weight_bf16, eps, rows, (int)cols, sum_bf16, q_e4m3, inv_scale)
  if (pieces <= 128) XAXB_NORM(1, 128);
  else if (pieces <= 256 && many) XAXB_NORM(2, 128);
  else if (pieces <= 256) XAXB_NORM(1, 256);
  else if (pieces <= 512 && many) XAXB_NORM(2, 256);
  else if (pieces <= 512) XAXB_NORM(1, 512);
  else if (pieces <= 1024) XAXB_NORM(2, 512);
  else XAXB_NORM(4, 512);
#undef XAXB_NORM
  return check_launch("rmsnorm_blocks_kernel");
}

int xaxb_silu_mul_blocks(xaxb_ctx* ctx, void* stream, const void* gate_up_bf16, int64_t ld, int64_t rows, int64_t dim,
                         void* q_e4m3, float* inv_scale) {
  if (!ctx || !gate_up_bf16 || !q_e4m3 || !inv_scale || misaligned(gate_up_bf16, 32) || misaligned(q_e4m3, 16) || ld % 16 != 0 ||
      ld < 2 * dim) {
    set_last_error("silu_mul_blocks: gate_up must be 32-byte aligned, q 16-byte aligned, ld a multiple of 16 and at least twice the width");
    return XAXB_BAD_ARGUMENT;
  }
  if (int rc = check_rows("silu_mul_blocks", rows, dim)) return rc;
  const uint32_t per_row = (uint32_t)((dim + 127) / 128 * kBlockPieces), pieces = (uint32_t)(rows * per_row);
  const unsigned ctas = (pieces + 255) / 256, resident = 4u * reinterpret_cast<const Ctx*>(ctx)->num_sms;
  launch_kernel(silu_mul_blocks_kernel, dim3(ctas < resident ? ctas : resident), dim3(256), 0, static_cast<cudaStream_t>(stream), 1,
                static_cast<const __nv_bfloat16*>(gate_up_bf16), ld, pieces, fast_div(per_row), (int)dim,
                static_cast<uint8_t*>(q_e4m3), inv_scale);
  return check_launch("silu_mul_blocks_kernel");
}

}  // extern "C"
