// Product of two block-scaled e4m3 matrices:
//
//   out[m, n] = bf16( sum_kb a_inv[m, kb] * b_inv[n / 128, kb] * P[m, n, kb] + bias[n] + residual[m, n] )
//   P[m, n, kb] = sum over the 128 values k of block kb of a[m, k] * b[n, k]
//
// with a [M, K] (activations, a multiplier per row and block of 128) and b [N, K] (weights, one per 128 x 128 square).
#include "gemm_device.cuh"

namespace xaxb {

struct GemmBlocksParams {
  const uint8_t* a;
  const uint8_t* b;
  long long lda, ldb;
  int M, N, K;
  int num_k_blocks;
  const float* a_inv;  // [M, num_k_blocks]
  const float* b_inv;  // [ceil(N / 128), num_k_blocks]
  const __nv_bfloat16* bias;
  const __nv_bfloat16* residual;
  long long ldr;
  __nv_bfloat16* out;
  long long ldo;
};

__device__ __forceinline__ float e4m3_value(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// 64 x 64 outputs per CTA of 256 threads, 16 per thread, operands widened to float32 in shared memory 32 columns at
// a time; the partial sums of a block of 128 are scaled once, like the tensor-core kernels do it.
__global__ void __launch_bounds__(256) gemm_blocks_kernel(const GemmBlocksParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float as[32][65], bs[32][65];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  float acc[4][4] = {}, part[4][4];
  for (int kb = 0; kb < p.num_k_blocks; ++kb) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[i][j] = 0.0f;
    for (int k0 = kb * 128; k0 < kb * 128 + 128; k0 += 32) {
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i / 32, c = i % 32, k = k0 + c;
        as[c][r] = m0 + r < p.M && k < p.K ? e4m3_value(p.a[(m0 + r) * p.lda + k]) : 0.0f;
        bs[c][r] = n0 + r < p.N && k < p.K ? e4m3_value(p.b[(n0 + r) * p.ldb + k]) : 0.0f;
      }
      __syncthreads();
#pragma unroll 4
      for (int c = 0; c < 32; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[c][tm + 16 * i], bs[c][tn + 16 * j], part[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + tm + 16 * i;
      const float sa = m < p.M ? __ldg(p.a_inv + (long long)m * p.num_k_blocks + kb) : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tn + 16 * j;
        const float sb = n < p.N ? __ldg(p.b_inv + (long long)(n / 128) * p.num_k_blocks + kb) : 0.0f;
        acc[i][j] = fmaf(part[i][j], sa * sb, acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      float f = acc[i][j];
      if (p.bias) f += __bfloat162float(p.bias[n]);
      if (p.residual) f += __bfloat162float(p.residual[m * p.ldr + n]);
      p.out[m * p.ldo + n] = __float2bfloat16_rn(f);
    }
}

}  // namespace xaxb

using namespace xaxb;

extern "C" int xaxb_gemm_fp8_blocks(xaxb_ctx* ctx_, void* stream, const void* a_e4m3, int64_t lda, const float* a_inv,
                                    const void* b_e4m3, int64_t ldb, const float* b_inv, int64_t M, int64_t N, int64_t K,
                                    const void* bias_bf16, const void* residual_bf16, int64_t ldr, void* out_bf16,
                                    int64_t ldo) {
  if (!ctx_ || !a_e4m3 || !a_inv || !b_e4m3 || !b_inv || !out_bf16 || M <= 0 || N <= 0 || K <= 0) {
    set_last_error("gemm_fp8_blocks: null pointer or non-positive shape");
    return XAXB_BAD_ARGUMENT;
  }
  const uintptr_t pointers = reinterpret_cast<uintptr_t>(a_e4m3) | reinterpret_cast<uintptr_t>(b_e4m3) |
                             reinterpret_cast<uintptr_t>(bias_bf16) | reinterpret_cast<uintptr_t>(residual_bf16) |
                             reinterpret_cast<uintptr_t>(out_bf16);
  if (K % 16 != 0 || lda % 16 != 0 || ldb % 16 != 0 || lda < K || ldb < K || N % 8 != 0 || ldo % 8 != 0 || ldo < N ||
      (residual_bf16 && (ldr % 8 != 0 || ldr < N)) || (pointers & 15) || M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) {
    set_last_error("gemm_fp8_blocks: K, lda, ldb must be multiples of 16, N, ldo, ldr of 8, row strides no smaller than the "
                   "rows, and all tensors 16-byte aligned (M %lld N %lld K %lld)", (long long)M, (long long)N, (long long)K);
    return XAXB_BAD_ARGUMENT;
  }
  GemmBlocksParams p;
  p.a = static_cast<const uint8_t*>(a_e4m3), p.lda = lda, p.a_inv = a_inv;
  p.b = static_cast<const uint8_t*>(b_e4m3), p.ldb = ldb, p.b_inv = b_inv;
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.num_k_blocks = (int)((K + 127) / 128);
  p.bias = static_cast<const __nv_bfloat16*>(bias_bf16);
  p.residual = static_cast<const __nv_bfloat16*>(residual_bf16), p.ldr = ldr;
  p.out = static_cast<__nv_bfloat16*>(out_bf16), p.ldo = ldo;
  const int64_t tiles_m = (M + 63) / 64;
  if (tiles_m > 65535) {
    set_last_error("gemm_fp8_blocks: at most %d rows", 65535 * 64);
    return XAXB_BAD_ARGUMENT;
  }
  launch_kernel(gemm_blocks_kernel, dim3((unsigned)((N + 63) / 64), (unsigned)tiles_m), dim3(256), 0,
                static_cast<cudaStream_t>(stream), 1, p);
  return check_launch("gemm_blocks_kernel");
}
