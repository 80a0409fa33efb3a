// Product of two block-scaled e4m3 matrices:
//
//   out[m, n] = bf16( sum_kb a_inv[m, kb] * b_inv[n / 128, kb] * P[m, n, kb] + bias[n] + residual[m, n] )
//   P[m, n, kb] = sum over the 128 values k of block kb of a[m, k] * b[n, k]
//
// with a [M, K] (activations, a multiplier per row and block of 128) and b [N, K] (weights, one per 128 x 128 square).
#include "gemm_device.cuh"
#include "quant_device.cuh"

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
  int* d_status;
};

constexpr int kSiteBlkProducer = 51, kSiteBlkMma = 52, kSiteBlkMmaAcc = 53, kSiteBlkPromote = 54;

// Barrier over the 128 promoting threads.
__device__ __forceinline__ void promote_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// A bounded wait that goes on although the CTA has given up: for copies that must land before the CTA may leave.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity, int* d_status) {
  const unsigned long long t0 = globaltimer_ns(), limit = wait_limit_ns(d_status);
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < limit) {
  }
}

// Distributed-shared-memory load that stays behind the barrier in front of it.
__device__ __forceinline__ float4 ld_dsmem_f4_ordered(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// bf16(f + bias + residual) of eight neighbouring columns, 16 bytes.
__device__ __forceinline__ void finish8(const GemmBlocksParams& p, float (&f)[8], int m, int n) {
  if (p.bias) {
    float v[8];
    unpack8(__ldg(reinterpret_cast<const uint4*>(p.bias + n)), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] += v[j];
  }
  if (p.residual) {
    float v[8];
    unpack8(*reinterpret_cast<const uint4*>(p.residual + m * p.ldr + n), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] += v[j];
  }
  *reinterpret_cast<uint4*>(p.out + m * p.ldo + n) = pack8(f);
}

// ---------------------------------------------------------------------------------------
// Few rows: weight streaming.  The weights are the MMA's 128-row operand and NT rows of activations its columns, so a
// decode step moves 16 KB of weights and only NT * 128 bytes of activations per K block.  A cluster of S CTAs shares
// the K blocks of one tile; each CTA leaves its part of the result in shared memory and the cluster adds the parts
// over distributed shared memory in rank order (no atomics: the same bits every time).
//   warp 0     TMA producer (weight and activation tiles into a ring)
//   warp 1     one thread issues the four MMAs of a K block into the next tensor-memory buffer; their commit both
//              frees the ring stage and hands the block to the promoting warps
//   warps 2-5  promotion: thread = weight row; acc[t] += partial[t] * (a_inv[t, kb] * b_inv[kb]) in float32 registers
template <int NT>
struct BlocksDecodeCfg {
  static constexpr int kCtasPerSm = NT == 128 ? 2 : 3;
  static constexpr int kWeightBytes = kBM * kBKBytes;
  static constexpr int kStageBytes = kWeightBytes + NT * kBKBytes;
  static constexpr int kStages = NT == 16 ? 4 : 3;
  static constexpr int kBufs = NT == 16 ? 4 : 2;           // tensor-memory buffers of NT columns
  static constexpr int kTmemCols = kBufs * NT;              // kCtasPerSm times this is at most 512
  static constexpr int kScaleBlocks = NT <= 32 ? 32 : 16;  // K blocks whose multipliers are staged at a time
  static constexpr int kPipeBytes = kStages * kStageBytes;
  static constexpr int kParkFloats = kBM + 4;              // floats per token of the parked result
  static constexpr int kSmemBytes = kPipeBytes + kScaleBlocks * NT * 4 + 256;
  static_assert(NT * kParkFloats * 4 <= kPipeBytes, "the parked result overlays the ring");
  // A stage's commit barrier must not complete a second time before the promoting warps have seen the first: the
  // block that uses the stage next has to wait for a buffer that they free after that.
  static_assert(kBufs <= kStages, "a stage comes round no sooner than a buffer");
  static_assert(kCtasPerSm * kTmemCols <= 512 && (kCtasPerSm + 1) * (kSmemBytes + 1024) > 228 * 1024,
                "shared memory must keep more CTAs off the SM than tensor memory serves");
};

template <int NT>
__global__ void __launch_bounds__(kGemmThreads, BlocksDecodeCfg<NT>::kCtasPerSm)
gemm_blocks_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                          const GemmBlocksParams p, const int S) {
  using Cfg = BlocksDecodeCfg<NT>;
  constexpr int kStages = Cfg::kStages, kBufs = Cfg::kBufs;
  constexpr uint32_t kIdesc = umma_idesc(kFmtE4M3, kFmtE4M3, 0, 0, kBM, NT);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* smem_w = smem;
  uint8_t* smem_x = smem + kStages * Cfg::kWeightBytes;
  float* scales = reinterpret_cast<float*>(smem + Cfg::kPipeBytes);  // [kScaleBlocks][NT]
  float* park = reinterpret_cast<float*>(smem);                      // [NT][kParkFloats], after the main loop
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kPipeBytes + Cfg::kScaleBlocks * NT * 4);  // [kStages]
  uint64_t* done = full + kStages;                                   // [kStages]
  uint64_t* buf_free = done + kStages;                               // [kBufs]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(buf_free + kBufs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int tile_n = blockIdx.x / S;
  const int n0 = tile_n * kBM, m0 = blockIdx.y * NT;
  const int kb0 = (int)((long long)p.num_k_blocks * rank / S);
  const int nkb = (int)((long long)p.num_k_blocks * (rank + 1) / S) - kb0;  // at least 1: S <= num_k_blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(full + s, 1), mbar_init(done + s, 1);
    for (int b = 0; b < kBufs; ++b) mbar_init(buf_free + b, 4);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();  // tensor memory is allocated: the next kernel may be scheduled
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, i = 0;
      uint32_t phase = 0;
      for (; i < nkb; ++i) {
        if (i >= kStages &&
            !mbar_wait(done + stage, phase ^ 1, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkProducer))
          break;
        mbar_arrive_expect_tx(full + stage, Cfg::kStageBytes);
        tma_load_2d(smem_w + stage * Cfg::kWeightBytes, &tmap_w, full + stage, (kb0 + i) * kBKBytes, n0);
        tma_load_2d(smem_x + stage * NT * kBKBytes, &tmap_x, full + stage, (kb0 + i) * kBKBytes, m0);
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
      if (*abort_flag)  // the stages in flight land before the CTA leaves
        for (int j = i > kStages ? i - kStages : 0; j < i; ++j) mbar_drain(full + j % kStages, (j / kStages) & 1, p.d_status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      for (int i = 0; i < nkb; ++i) {
        if (i >= kBufs && !mbar_wait(buf_free + buf, buf_phase ^ 1, abort_flag, p.d_status,
                                     XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkMmaAcc))
          break;
        if (!mbar_wait(full + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkMma)) break;
        tc_fence_after_sync();
        const uint64_t w_desc = umma_desc_kmajor_sw128(smem_u32(smem_w + stage * Cfg::kWeightBytes));
        const uint64_t x_desc = umma_desc_kmajor_sw128(smem_u32(smem_x + stage * NT * kBKBytes));
#pragma unroll
        for (int k = 0; k < kBKBytes / 32; ++k) umma_f8(tmem_base + buf * NT, w_desc + 2 * k, x_desc + 2 * k, kIdesc, k != 0);
        umma_commit(done + stage);
        if (++stage == kStages) stage = 0, phase ^= 1;
        if (++buf == kBufs) buf = 0, buf_phase ^= 1;
      }
    }
  } else {
    const int quarter = warp & 3, t = threadIdx.x - 64;
    const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16);
    const float* b_inv = p.b_inv + (long long)tile_n * p.num_k_blocks + kb0;
    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.0f;
    int stage = 0, buf = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int in_chunk = i % Cfg::kScaleBlocks;
      if (in_chunk == 0) {  // the combined multipliers of the next blocks
        if (i > 0) promote_sync();
        const int n = min(Cfg::kScaleBlocks, nkb - i);
        const int m = m0 + t % NT;
        const float* a_inv = p.a_inv + (long long)m * p.num_k_blocks + kb0 + i;
#pragma unroll 4
        for (int b = t / NT; b < n; b += 128 / NT)
          scales[b * NT + t % NT] = m < p.M ? __ldg(a_inv + b) * __ldg(b_inv + i + b) : 0.0f;
        promote_sync();
      }
      if (ok) ok = mbar_wait(done + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkPromote);
      ok = __all_sync(0xffffffffu, ok);  // (a warp that gave up still takes part in the barriers above)
      if (ok) {
        tc_fence_after_sync();
        const float* sc = scales + in_chunk * NT;
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          uint32_t r[16];
          tmem_ld_x16(taddr + buf * NT + c, r);
          tmem_ld_wait();
          if (c + 16 == NT) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(buf_free + buf);
          }
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sc + c + j);
            acc[c + j] = fmaf(__uint_as_float(r[j]), s4.x, acc[c + j]);
            acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), s4.y, acc[c + j + 1]);
            acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), s4.z, acc[c + j + 2]);
            acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), s4.w, acc[c + j + 3]);
          }
        }
      }
      if (++stage == kStages) stage = 0, phase ^= 1;
      if (++buf == kBufs) buf = 0;
    }
    // The last block's commit covers every MMA, and every MMA every copy: the ring is free.
    if (ok) {
      float* mine = park + quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < NT; ++j) mine[j * Cfg::kParkFloats] = acc[j];
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  if (S > 1)
    cluster_sync_all();  // every CTA's part is visible to the cluster
  else
    __syncthreads();

  // This CTA adds its share of the tile's (token, 8 weight rows) items over the ranks.
  if (!*abort_flag) {
    const int items = min(NT, p.M - m0) * (kBM / 8);
    const int hi = items * (rank + 1) / S;
    const uint32_t park_addr = smem_u32(park);
    for (int it = items * rank / S + threadIdx.x; it < hi; it += kGemmThreads) {
      const int tok = it / (kBM / 8), r8 = it % (kBM / 8) * 8, n = n0 + r8;
      if (n >= p.N) continue;
      const uint32_t off = park_addr + (uint32_t)(tok * Cfg::kParkFloats + r8) * 4u;
      float f[8] = {};
      for (int src = 0; src < S; ++src) {
        const uint32_t at = S > 1 ? dsmem_addr(off, (uint32_t)src) : off;
        const float4 lo = ld_dsmem_f4_ordered(at), hi4 = ld_dsmem_f4_ordered(at + 16);
        f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w;
        f[4] += hi4.x, f[5] += hi4.y, f[6] += hi4.z, f[7] += hi4.w;
      }
      finish8(p, f, m0 + tok, n);
    }
  }
  __syncwarp();
  if (S > 1) cluster_sync_all();  // the peers have finished reading this CTA's part
  __syncthreads();
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// How many CTAs share a tile's K blocks.
static int pick_split(int tiles, int num_k_blocks, int num_sms) {
  int best = 1;
  double best_t = 1e30;
  for (int s = 1; s <= 8 && s <= num_k_blocks; ++s) {
    const double per_sm = (tiles * s + num_sms - 1) / num_sms;
    const double t = per_sm * ((num_k_blocks + s - 1) / s) * 0.37 + (s > 1 ? 1.5 + 0.1 * s : 0.0);
    if (t < best_t) best_t = t, best = s;
  }
  return best;
}

template <int NT>
static int launch_decode(const Ctx* ctx, cudaStream_t stream, const GemmBlocksParams& p) {
  using Cfg = BlocksDecodeCfg<NT>;
  CUtensorMap tw, tx;
  if (int rc = make_tmap_2d(ctx, &tw, p.b, 1, (uint64_t)p.K, (uint64_t)p.N, (uint64_t)p.ldb, kBKBytes, kBM)) return rc;
  if (int rc = make_tmap_2d(ctx, &tx, p.a, 1, (uint64_t)p.K, (uint64_t)p.M, (uint64_t)p.lda, kBKBytes, NT)) return rc;
  if (int rc = ensure_dynamic_smem<gemm_blocks_decode_kernel<NT>>(ctx, Cfg::kSmemBytes, "gemm_blocks_decode_kernel")) return rc;
  const int tiles_n = (p.N + kBM - 1) / kBM, tiles_m = (p.M + NT - 1) / NT;
  const int S = pick_split(tiles_n * tiles_m, p.num_k_blocks, ctx->num_sms);
  cudaError_t e = launch_kernel(gemm_blocks_decode_kernel<NT>, dim3((unsigned)(tiles_n * S), (unsigned)tiles_m),
                                dim3(kGemmThreads), Cfg::kSmemBytes, stream, (unsigned)S, tw, tx, p, S);
  if (e != cudaSuccess) {
    set_last_error("gemm_blocks_decode_kernel launch: %s", cudaGetErrorString(e));
    return XAXB_LAUNCH_FAILED;
  }
  return check_launch("gemm_blocks_decode_kernel");
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
  const Ctx* ctx = reinterpret_cast<const Ctx*>(ctx_);
  p.d_status = ctx->d_status;
  if ((M + 127) / 128 > 65535) {
    set_last_error("gemm_fp8_blocks: at most %d rows", 65535 * 128);
    return XAXB_BAD_ARGUMENT;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M <= 16) return launch_decode<16>(ctx, s, p);
  if (M <= 32) return launch_decode<32>(ctx, s, p);
  if (M <= 64) return launch_decode<64>(ctx, s, p);
  return launch_decode<128>(ctx, s, p);
}
