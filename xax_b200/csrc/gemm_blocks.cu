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

constexpr int kSiteBlkProducer = 51, kSiteBlkMma = 52, kSiteBlkPromote = 53;

// Barrier over the decode kernel's promoting threads.
template <int kThreads>
__device__ __forceinline__ void promote_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
}

// mbar_wait for barriers that complete within a microsecond: polls before it turns to the clock and the limit, which
// lives in global memory.
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* d_status,
                                               int code) {
#pragma unroll 1
  for (int i = 0; i < 1000; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait(bar, parity, abort_flag, d_status, code);
}

// For a producer that has given up: nothing has moved for the wait limit; a millisecond more for the copies asked for last.
__device__ __forceinline__ void wait_for_last_copies() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 1000000ull) {
  }
}

// A store into the shared memory of a CTA of the cluster.
__device__ __forceinline__ void st_dsmem_f4(uint32_t cluster_addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// Barrier over one warpgroup of the pair kernel (two of them promote).
__device__ __forceinline__ void warpgroup_sync(int which) {
  if (which == 0)
    asm volatile("bar.sync 1, 128;" ::: "memory");
  else
    asm volatile("bar.sync 2, 128;" ::: "memory");
}

// Shared-memory loads that stay where they are written.
__device__ __forceinline__ float lds_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
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

// (a, b) += (x * s, y * t), two float32 in one instruction.  (Volatile, which keeps the additions between the loads they
// overlap with: left to the compiler they gathered behind the last one.)
__device__ __forceinline__ void fma2(float& a, float& b, uint32_t x, uint32_t y, float s, float t) {
  asm volatile("{\n\t.reg .b64 c, v, w;\n\t"
               "mov.b64 c, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {%4, %5};\n\t"
               "fma.rn.f32x2 c, v, w, c;\n\t"
               "mov.b64 {%0, %1}, c;\n\t}"
               : "+f"(a), "+f"(b)
               : "r"(x), "r"(y), "f"(s), "f"(t));
}

// ---------------------------------------------------------------------------------------
// Few rows: weight streaming.  For up to 64 tokens the weights are the MMA's 128-row operand and NT rows of activations its
// columns, so a decode step moves 16 KB of weights and only NT * 128 bytes of activations per K block.  A cluster of S
// CTAs shares the K blocks of one tile; each CTA pushes its part of the result into the shared memory of the CTA that
// owns the token, which adds the parts in rank order (no atomics: the same bits every time).  (Pulling the parts took
// S remote round trips per item, 7000 of 38000 cycles for 128 x 4096 x 14336, S = 4; one bulk copy per owner in place of
// the threads' 16-byte pushes 20.0 us against 19.0.)
//   promoting warps  thread = weight row; acc[t] += partial[t] * (a_inv[t, kb] * b_inv[kb]) in float32 registers.  With
//                    NT = 128 the operands change places: thread = token, two warpgroups of 64 weight rows each, and the
//                    combined multiplier is one value a thread instead of one a column.
//   next warp        TMA producer (weight and activation tiles into a ring)
//   next two warps   one thread each issues the four MMAs of every other K block into the next tensor-memory buffer (one
//                    thread those of all blocks where the ring is too short for two, see issue_step)
// Finding a barrier complete, an MMA and a commit cost the issuing thread 65 to 200 cycles each, which is what a chain of K
// blocks runs at, so one barrier opens a block (full[s] counts its copies and the promoting warps that free its buffer,
// arriving on the stage that the block will use) and one closes it (the commit on done[s] frees the stage and hands the
// product over).
// What bounds it is the operand bytes that an SM keeps in flight, so the ring takes all the shared memory that the CTAs
// which will be resident together leave (`stages`, from the launcher).  Measured (graph of launches, operands past L2):
// 1 x 28672 x 4096 20.9 us = 5.6 TB/s, 0.86 of the copy rate (224 tiles on 148 SMs; the rest is that imbalance);
// 64 x 4096 x 14336 15.9, 128 x 4096 x 14336 18.9, 64 x 2048 x 5632 7.9, 1 x 4096 x 4096 5.3 us, of which start, first
// copies, the two cluster barriers and the pushes are 3 (16 tokens) to 6 us (128).
// kAlone: for launches of at most one CTA an SM, which leaves NT = 128 room for 32-column readouts and four buffers.
template <int NT, bool kAlone>
struct BlocksDecodeCfg {
  static constexpr bool kTokenRows = NT == 128;            // the token is the accumulator's row, else the weight row is
  static constexpr int kGroups = NT == 128 ? 2 : 1;        // promoting warpgroups
  static constexpr int kCols = NT / kGroups;               // accumulator columns per promoting thread
  static constexpr int kThreads = NT == 128 ? 384 : 224;
  // Registers of two CTAs of NT = 128: their 384 threads start with 80 each; the warpgroup of the producer and the
  // issuers gives up what the promoting ones need.
  static constexpr bool kMoveRegs = NT == 128 && !kAlone;
  static constexpr int kPromoteRegs = 104, kIssueRegs = 32;
  static_assert(kGroups * kPromoteRegs + kIssueRegs <= 3 * 80, "register split");
  static constexpr int kCtasPerSm = kAlone ? 1 : NT == 16 ? 3 : 2;  // at most: registers, tensor memory
  static constexpr int kWeightBytes = kBM * kBKBytes;
  static constexpr int kStageBytes = kWeightBytes + NT * kBKBytes;
  static constexpr int kMaxStages = 12;
  static constexpr int kBufs = NT == 32 ? 3 : kMoveRegs ? 2 : 4;  // tensor-memory buffers of NT columns
  static constexpr int kTmemCols = NT == 32 ? 128 : kBufs * NT;
  static constexpr int kScaleBlocks = 16;                  // K blocks whose multipliers are staged at a time
  static constexpr int kLoad = NT == 16 || kMoveRegs ? 16 : 32;  // columns per readout (what the registers allow)
  static constexpr int kPartFloats = kBM + 4;              // floats per token of a CTA's part of the result
  static constexpr int kPartBytes = (kTokenRows ? 1 : 2) * NT * kPartFloats * 4;  // (two: one to turn it round in)
  static constexpr int kExtraBytes = kScaleBlocks * NT * 4 + (2 * kMaxStages + 2) * 8;
  static constexpr int kSmemPerSm = 228 * 1024, kSmemReserved = 1024;
  // The CTAs of a cluster (one on an SM) keep the parts beside the ring, so that none waits for another's ring before it
  // pushes (64 x 4096 x 14336: 16.5 -> 16.0 us, 64 x 2048 x 5632: 8.3 -> 7.9), except where that leaves NT = 128 four
  // stages instead of six (128 x 4096 x 14336: 19.0 -> 19.3).
  static constexpr bool kBeside = NT < 128;
  static constexpr int beside_bytes(bool split) { return kBeside && split ? kPartBytes : 0; }
  // The ring that leaves room for `ctas` CTAs on an SM, and for no more of them than tensor memory serves.
  static constexpr int stages_for(int ctas, bool split) {
    const int n = (kSmemPerSm / ctas - kSmemReserved - kExtraBytes - beside_bytes(split)) / kStageBytes;
    return n < kMaxStages ? n : kMaxStages;
  }
  // Two threads may issue if neither can test a stage's barrier a phase early.  A thread that turns to block i has found
  // block i - 2 open, so the blocks up to i - 2 - kBufs are done; the stage's block before, i - stages, is among them, or
  // is the same thread's (stages even).
  static constexpr int issue_step(int stages) { return stages % 2 == 0 || stages >= kBufs + 2 ? 2 : 1; }
  static constexpr int smem_bytes(int stages, bool split) {
    return stages * kStageBytes + kExtraBytes + beside_bytes(split);
  }
  static constexpr int kMinStages = kBufs > 3 ? kBufs : 3;
  static_assert(NT * kPartFloats * 4 <= kMinStages * kStageBytes, "the parts overlay the ring");
  static_assert(stages_for(kCtasPerSm, false) >= kMinStages, "a stage comes round no sooner than a buffer");
  static_assert(kMoveRegs || stages_for(1, true) >= kMinStages, "a cluster's CTAs");
  static_assert(kCtasPerSm * kTmemCols <= 512, "tensor memory");
};

template <int NT, bool kAlone>
__global__ void __launch_bounds__(BlocksDecodeCfg<NT, kAlone>::kThreads, BlocksDecodeCfg<NT, kAlone>::kCtasPerSm)
gemm_blocks_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                          const GemmBlocksParams p, const int S, const int stages) {
  using Cfg = BlocksDecodeCfg<NT, kAlone>;
  constexpr int kBufs = Cfg::kBufs, kPromoteWarps = 4 * Cfg::kGroups;
  constexpr uint32_t kIdesc = umma_idesc(kFmtE4M3, kFmtE4M3, 0, 0, kBM, NT);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* smem_w = smem;
  uint8_t* smem_x = smem + stages * Cfg::kWeightBytes;
  float* scales = reinterpret_cast<float*>(smem + stages * Cfg::kStageBytes);  // [kScaleBlocks][NT]
  // [S][NT / S][kPartFloats], this CTA's tokens; over the ring, or beside it
  float* parts = reinterpret_cast<float*>(Cfg::kBeside && S > 1 ? smem + stages * Cfg::kStageBytes + Cfg::kExtraBytes : smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + Cfg::kScaleBlocks * NT);  // [stages]
  uint64_t* done = full + Cfg::kMaxStages;                                     // [stages]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + Cfg::kMaxStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int tile_n = blockIdx.x / S;
  const int n0 = tile_n * kBM, m0 = blockIdx.y * NT;
  const int kb0 = (int)((long long)p.num_k_blocks * rank / S);
  const int nkb = (int)((long long)p.num_k_blocks * (rank + 1) / S) - kb0;  // at least 1: S <= num_k_blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(full + s, 1 + kPromoteWarps), mbar_init(done + s, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == kPromoteWarps + 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  if (Cfg::kBeside && S > 1) cluster_arrive();  // waited for before the first push: the cluster's CTAs are all there
  pdl_trigger();  // tensor memory is allocated: the next kernel may be scheduled
  // The first weight tiles are asked into L2 while the previous kernel ends (nothing in flight writes weights, and L2 is
  // the point of coherence); everything that reads or writes global memory for good waits for it.
  if (warp == kPromoteWarps && lane == 0)
    for (int i = 0; i < min(4, nkb); ++i) tma_prefetch_l2_2d(&tmap_w, (kb0 + i) * kBKBytes, n0);
  pdl_wait();

  if (warp >= kPromoteWarps) {
    if constexpr (Cfg::kMoveRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kIssueRegs));
    if (warp == kPromoteWarps && lane == 0) {
      // ------------------------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < nkb; ++i) {
        if (i >= stages &&
            !mbar_wait_soon(done + stage, phase ^ 1, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkProducer))
          break;
        mbar_arrive_expect_tx(full + stage, Cfg::kStageBytes);
        tma_load_2d(smem_w + stage * Cfg::kWeightBytes, &tmap_w, full + stage, (kb0 + i) * kBKBytes, n0);
        tma_load_2d(smem_x + stage * NT * kBKBytes, &tmap_x, full + stage, (kb0 + i) * kBKBytes, m0);
        if (++stage == stages) stage = 0, phase ^= 1;
      }
      if (*abort_flag) wait_for_last_copies();
    } else if ((warp == kPromoteWarps + 1 || warp == kPromoteWarps + 2) && lane == 0) {
      // ------------------------------------------------------------------ MMA issuers
      const int step = Cfg::issue_step(stages), first = warp - (kPromoteWarps + 1);
      int stage = first, buf = first;
      uint32_t phase = 0;
      for (int i = first < step ? first : nkb; i < nkb; i += step) {
        if (!mbar_wait_soon(full + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkMma)) break;
        tc_fence_after_sync();
        const uint64_t w_desc = umma_desc_kmajor_sw128(smem_u32(smem_w + stage * Cfg::kWeightBytes));
        const uint64_t x_desc = umma_desc_kmajor_sw128(smem_u32(smem_x + stage * NT * kBKBytes));
#pragma unroll
        for (int k = 0; k < kBKBytes / 32; ++k)
          umma_f8(tmem_base + buf * NT, (Cfg::kTokenRows ? x_desc : w_desc) + 2 * k, (Cfg::kTokenRows ? w_desc : x_desc) + 2 * k,
                  kIdesc, k != 0);
        umma_commit(done + stage);
        if ((stage += step) >= stages) stage -= stages, phase ^= 1;
        if ((buf += step) >= kBufs) buf -= kBufs;
      }
    }
  } else {
    // ------------------------------------------------------------------ promotion
    // A stage's commit barrier never completes a second time before these warps have seen the first: the block that
    // uses the stage next waits for a buffer that they free after that (stages >= kBufs).
    if constexpr (Cfg::kMoveRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kPromoteRegs));
    const int quarter = warp & 3, col0 = (warp >> 2) * Cfg::kCols, t = threadIdx.x;
    const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + col0;
    float acc[Cfg::kCols];
#pragma unroll
    for (int j = 0; j < Cfg::kCols; ++j) acc[j] = 0.0f;
    int stage = 0, buf = 0, next = kBufs % stages;  // next: the stage of the block that will use this one's buffer
    uint32_t phase = 0;
    bool ok = true;
    if (lane == 0) {  // all buffers start free
#pragma unroll
      for (int b = 0; b < kBufs; ++b) mbar_arrive(full + b);
    }
#pragma unroll 1
    for (int i = 0; i < nkb; ++i) {
      const int in_chunk = i % Cfg::kScaleBlocks;
      if (in_chunk == 0) {  // the combined multipliers of the next blocks
        if (i > 0) promote_sync<128 * Cfg::kGroups>();
        constexpr int kEach = Cfg::kScaleBlocks * NT / (128 * Cfg::kGroups);  // a thread's, all asked for at once
        const int m = min(m0 + t % NT, p.M - 1), b0 = t / NT * kEach;         // (rows past M are never stored)
        const float *a_inv = p.a_inv + (long long)m * p.num_k_blocks + kb0, *b_inv = p.b_inv + (long long)tile_n * p.num_k_blocks + kb0;
        float v[kEach], w[kEach];
#pragma unroll
        for (int b = 0; b < kEach; ++b) {
          const int at = min(i + b0 + b, nkb - 1);
          v[b] = __ldg(a_inv + at), w[b] = __ldg(b_inv + at);
        }
#pragma unroll
        for (int b = 0; b < kEach; ++b) scales[(b0 + b) * NT + t % NT] = v[b] * w[b];
        promote_sync<128 * Cfg::kGroups>();
      }
      if (!mbar_try_wait(done + stage, phase) && ok)
        ok = mbar_wait_soon(done + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSiteBlkPromote);
      ok = __all_sync(0xffffffffu, ok);  // (a warp that gave up still takes part in the barriers above)
      if (ok) {
        tc_fence_after_sync();
        const uint32_t sc = smem_u32(scales + in_chunk * NT + (Cfg::kTokenRows ? quarter * 32 + lane : 0));
        const uint32_t from = taddr + buf * NT;
#pragma unroll
        for (int c = 0; c < Cfg::kCols; c += Cfg::kLoad) {
          uint32_t r[Cfg::kLoad];
          if constexpr (Cfg::kLoad == 32)
            tmem_ld_x32(from + c, r);
          else
            tmem_ld_x16(from + c, r);
          // the columns' multipliers, on their way together with the products (left to the compiler each is read right
          // before its use: 770 cycles a block for 64 tokens)
          float4 mul[Cfg::kTokenRows ? 1 : Cfg::kLoad / 4];
          if constexpr (Cfg::kTokenRows) {
            const float v = lds_f1(sc);
            mul[0] = make_float4(v, v, v, v);
          } else {
#pragma unroll
            for (int j = 0; j < Cfg::kLoad / 4; ++j) mul[j] = lds_f4(sc + (c + 4 * j) * 4);
          }
          tmem_ld_wait();
          if (c + Cfg::kLoad == Cfg::kCols) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + next);
          }
#pragma unroll
          for (int j = 0; j < Cfg::kLoad; j += 4) {
            const float4 m4 = mul[Cfg::kTokenRows ? 0 : j / 4];
            fma2(acc[c + j], acc[c + j + 1], r[j], r[j + 1], m4.x, m4.y);
            fma2(acc[c + j + 2], acc[c + j + 3], r[j + 2], r[j + 3], m4.z, m4.w);
          }
        }
      }
      if (++stage == stages) stage = 0, phase ^= 1;
      if (++next == stages) next = 0;
      if (++buf == kBufs) buf = 0;
    }
    // Every block is done, and with it every copy: this CTA's ring is free.  Threads whose row is a token hold neighbouring
    // columns and can push 16 bytes at a time; the others first turn their part round in shared memory (scalar pushes
    // were slower than all of it: 20 us against 9 for 64 x 2048 x 5632).
    const int per = NT / S, tokens = min(NT, p.M - m0);  // tokens per owner (a power of two); those that exist
    const int row = quarter * 32 + lane;
    float* turned = Cfg::kTokenRows || S == 1 ? parts : parts + NT * Cfg::kPartFloats;
    if (!Cfg::kTokenRows && ok) {
#pragma unroll
      for (int j = 0; j < Cfg::kCols; ++j)
        if (j < tokens) turned[j * Cfg::kPartFloats + row] = acc[j];
    }
    tc_fence_before_sync();
    __syncwarp();
    if (S > 1) {
      if (!Cfg::kBeside) cluster_arrive();  // the rings of the whole cluster are free
      cluster_wait();
    }
    if (S == 1 || !Cfg::kTokenRows) promote_sync<128 * Cfg::kGroups>();
    if (ok && Cfg::kTokenRows && row < tokens) {
      const uint32_t mine = smem_u32(parts) + (uint32_t)((rank * per + row % per) * Cfg::kPartFloats + col0) * 4u;
      const uint32_t at = S > 1 ? dsmem_addr(mine, (uint32_t)(row / per)) : mine;
#pragma unroll
      for (int j = 0; j < Cfg::kCols; j += 4) st_dsmem_f4(at + j * 4, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    } else if (ok && !Cfg::kTokenRows && S > 1) {
      for (int it = t; it < tokens * (kBM / 4); it += 128 * Cfg::kGroups) {
        const int tok = it / (kBM / 4), r4 = it % (kBM / 4) * 4;
        const float4 v = *reinterpret_cast<const float4*>(turned + tok * Cfg::kPartFloats + r4);
        const uint32_t mine = smem_u32(parts) + (uint32_t)((rank * per + tok % per) * Cfg::kPartFloats + r4) * 4u;
        st_dsmem_f4(dsmem_addr(mine, (uint32_t)(tok / per)), v.x, v.y, v.z, v.w);
      }
    }
    if (S > 1)
      cluster_sync_all();  // every part has arrived
    else
      promote_sync<128 * Cfg::kGroups>();
    if (!*abort_flag) {
      const int items = min(per, tokens - rank * per) * (kBM / 8);
      for (int it = t; it < items; it += 128 * Cfg::kGroups) {
        const int tok = it / (kBM / 8), r8 = it % (kBM / 8) * 8, n = n0 + r8;
        if (n >= p.N) continue;
        const float* from = parts + tok * Cfg::kPartFloats + r8;
        float f[8] = {};
#pragma unroll
        for (int src = 0; src < 8; ++src) {
          if (src < S) {
            const float4 lo = *reinterpret_cast<const float4*>(from + src * per * Cfg::kPartFloats);
            const float4 hi = *reinterpret_cast<const float4*>(from + src * per * Cfg::kPartFloats + 4);
            f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w;
            f[4] += hi.x, f[5] += hi.y, f[6] += hi.z, f[7] += hi.w;
          }
        }
        finish8(p, f, m0 + rank * per + tok, n);
      }
    }
  }
  if (warp >= kPromoteWarps && S > 1) {  // the two barriers of the cluster above (barriers are all that may follow here:
    __syncwarp();                        // with NT = 128 these warps are down to 32 registers)
    if (!Cfg::kBeside) cluster_arrive();
    cluster_wait();
    cluster_sync_all();
  }
  __syncthreads();
  if (warp == kPromoteWarps + 1) {
    if (*abort_flag) wait_for_last_copies();  // (and MMAs)
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// How many CTAs share a tile's K blocks: as many as keep one CTA on an SM, since what a second one brings is less than the
// cluster's two barriers and pushes cost (64 x 28672 x 4096, 224 tiles: 24.9 us undivided, 33.0 with two; 16 x 6144 x 4096,
// 48 tiles: 11.1, 8.0 and 7.9 us with 1, 2 and 4).  Clusters of eight find room for their CTAs on one SM each in few places
// (64 x 2048 x 5632, 16 tiles: 8.6 us with 4, 13.3 with 8), so they are for few tiles; a CTA keeps four blocks at least.
static int pick_split(long long tiles, int num_k_blocks, int num_sms) {
  int s = 1;
  while (s < 8 && tiles * s * 2 <= (s == 4 ? 64 : num_sms) && num_k_blocks >= 8 * s) s *= 2;
  return s;
}

template <int NT, bool kAlone>
static int launch_decode_as(const Ctx* ctx, cudaStream_t stream, const GemmBlocksParams& p, int tiles_n, int tiles_m, int S,
                            int per_sm) {
  using Cfg = BlocksDecodeCfg<NT, kAlone>;
  CUtensorMap tw, tx;
  if (int rc = make_tmap_2d(ctx, &tw, p.b, 1, (uint64_t)p.K, (uint64_t)p.N, (uint64_t)p.ldb, kBKBytes, kBM)) return rc;
  if (int rc = make_tmap_2d(ctx, &tx, p.a, 1, (uint64_t)p.K, (uint64_t)p.M, (uint64_t)p.lda, kBKBytes, NT)) return rc;
  if (int rc = ensure_dynamic_smem<gemm_blocks_decode_kernel<NT, kAlone>>(ctx, Cfg::kSmemPerSm - Cfg::kSmemReserved,
                                                                          "gemm_blocks_decode_kernel"))
    return rc;
  const int stages = Cfg::stages_for(per_sm < Cfg::kCtasPerSm ? per_sm : Cfg::kCtasPerSm, S > 1);
  cudaError_t e = launch_kernel(gemm_blocks_decode_kernel<NT, kAlone>, dim3((unsigned)(tiles_n * S), (unsigned)tiles_m),
                                dim3(Cfg::kThreads), Cfg::smem_bytes(stages, S > 1), stream, (unsigned)S, tw, tx, p, S, stages);
  if (e != cudaSuccess) {
    set_last_error("gemm_blocks_decode_kernel launch: %s", cudaGetErrorString(e));
    return XAXB_LAUNCH_FAILED;
  }
  return check_launch("gemm_blocks_decode_kernel");
}

template <int NT>
static int launch_decode(const Ctx* ctx, cudaStream_t stream, const GemmBlocksParams& p) {
  const int tiles_n = (p.N + kBM - 1) / kBM, tiles_m = (p.M + NT - 1) / NT;
  const int S = pick_split((long long)tiles_n * tiles_m, p.num_k_blocks, ctx->num_sms);
  const long long ctas = (long long)tiles_n * tiles_m * S;
  const int per_sm = (int)((ctas + ctx->num_sms - 1) / ctx->num_sms < 4 ? (ctas + ctx->num_sms - 1) / ctx->num_sms : 4);
  if (NT == 128 && per_sm == 1) return launch_decode_as<NT, NT == 128>(ctx, stream, p, tiles_n, tiles_m, S, per_sm);
  return launch_decode_as<NT, false>(ctx, stream, p, tiles_n, tiles_m, S, per_sm);
}

// ---------------------------------------------------------------------------------------
// Many rows: 256 x 256 tiles, each by a pair of CTAs on two SMs (tcgen05.mma.cta_group::2; CTA r of the pair loads rows
// 128 r .. of both operand tiles and keeps rows 128 r .. of the result).  A K block's product goes to one of two
// tensor-memory buffers of 256 columns, always freshly written; two warpgroups of promoting threads (thread = row,
// 128 columns each: one weight square) read it out, scale it and add it to float32 registers while the tensor
// core fills the other buffer.
//
// Per 128-byte K block the tensor core needs 512 cycles and the packed multiply-adds of two warps per scheduler 256, so the
// promotion could hide behind the MMAs, but a block takes about 900 (62 % of the tensor pipe).  It is a chain of signals: 350
// cycles from a buffer's release until the issuing thread sees it, 512 of MMAs, 400 from the commit until the promoting
// warps see that, 330 until they have read it, shared by two buffers.  (Without readout and promotion 341 us of 433, and no
// less with a quarter of the MMAs; but three buffers of 160 columns do not help, 573 us, or 510 without readout and promotion:
// a block costs about the same however narrow.)  4096 x 28672 x 4096: 405 to 450 us from GPU to GPU in a graph = 2.1 to 2.4
// PFLOP/s; for seconds on end 480 us, 1455 MHz at the power cap, where the product without block scales takes 385 at 1255
// MHz.  2048 x 8192 x 2048: 37 to 43.  Not faster: 128 x 256 tiles on single CTAs, whose releases are local but which read
// half as much again out of L2 (467 against 419 us); halves of 128 columns with barriers of their own (578); opening the
// next block before the last columns of this one are added (490).  To keep the chain short
//   * two warps issue, one the even and one the odd K blocks (different buffers, nothing to order between them);
//   * one barrier opens a K block: full[s] counts both CTAs' copies AND the 16 warps that free the buffer, the latter
//     arriving on the stage that the block two further on will use;
//   * one commit closes it, multicast to both CTAs: done[s] frees the stage and hands the product over;
//   * a spare warp brings the multipliers through shared memory (loads by the promoting threads, however early, had them
//     wait for L2 behind every barrier: 594 us).
// Registers: three warpgroups start with 168 each; the issuing one gives up what the promoting ones need.
constexpr int kPairThreads = 384;
constexpr int kPairLaunchRegs = 168, kPairPromoteRegs = 192, kPairIssueRegs = 120;
static_assert(2 * kPairPromoteRegs + kPairIssueRegs <= 3 * kPairLaunchRegs, "register split");
constexpr int kPairTile = 256;
constexpr int kPairStages = 5;
static_assert(kPairStages >= 2 + 2, "two issuing threads on a ring of odd length: see BlocksDecodeCfg::issue_step");
constexpr int kPairOperandBytes = kBM * kBKBytes;          // per CTA, operand and stage
constexpr int kPairStageBytes = 2 * kPairOperandBytes;
constexpr int kPairOutBytes = kBM * 128;                   // 128 rows of 64 bf16: one TMA store
constexpr int kPairScaleFloats = 132;                      // per stage: 128 row multipliers, 2 of squares, the tile's corner
constexpr int kPairSmemBytes = kPairStages * (kPairStageBytes + kPairScaleFloats * 4) + 4 * kPairOutBytes + 128;
static_assert(kPairSmemBytes <= 227 * 1024, "shared memory of a CTA");
constexpr int kSitePairProducer = 55, kSitePairMma = 56, kSitePairPromote = 57, kSitePairScales = 58;

__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((uint16_t)3)
               : "memory");
}

// Two float32 to two bf16, the first in the low half, in one instruction.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void add8(float* f, const uint4 v) {
  float w[8];
  unpack8(v, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] += w[j];
}

__global__ void __launch_bounds__(kPairThreads, 1)
gemm_blocks_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                        const __grid_constant__ CUtensorMap tmap_out, const GemmBlocksParams p, const int tiles_m,
                        const int tiles_n, const int band) {
  constexpr uint32_t kIdesc = umma_idesc(kFmtE4M3, kFmtE4M3, 0, 0, 2 * kBM, kPairTile);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kPairStages * kPairOperandBytes;
  uint8_t* smem_out = smem + kPairStages * kPairStageBytes;
  float* smem_scale = reinterpret_cast<float*>(smem_out + 4 * kPairOutBytes);  // [kPairStages][kPairScaleFloats]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_scale + kPairStages * kPairScaleFloats);  // [kPairStages], the leader's
  uint64_t* done = full + kPairStages;                                         // [kPairStages], in each CTA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + kPairStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int num_tiles = tiles_m * tiles_n, nkb = p.num_k_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) mbar_init(full + s, 2 + 16), mbar_init(done + s, 2);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    prefetch_tmap(&tmap_out);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before anyone signals across the pair
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();  // tensor memory is allocated: the next kernel may be scheduled
  pdl_wait();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairIssueRegs));
    if (warp == 8) {
      // ---------------------------------------------------------------- TMA producer (both CTAs)
      if (lane == 0) {
        int stage = 0;
        long long g = 0;  // K blocks so far, over all tiles
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
          int tm, tn;
          tile_coords(band, tile, tiles_m, tiles_n, tm, tn);
          const int m0 = tm * kPairTile + (int)rank * kBM, n0 = tn * kPairTile + (int)rank * kBM;
          for (int kb = 0; kb < nkb; ++kb, ++g) {
            if (g >= kPairStages) {
              ok = mbar_wait_soon(done + stage, phase ^ 1, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSitePairProducer);
              if (!ok) break;
            }
            const uint32_t leader_full = dsmem_addr(smem_u32(full + stage), 0);
            mbar_arrive_expect_tx_cluster(leader_full, kPairStageBytes);
            tma_load_2d_pair(smem_a + stage * kPairOperandBytes, &tmap_a, leader_full, kb * kBKBytes, m0);
            tma_load_2d_pair(smem_b + stage * kPairOperandBytes, &tmap_b, leader_full, kb * kBKBytes, n0);
            if (++stage == kPairStages) stage = 0, phase ^= 1;
          }
        }
        if (!ok) wait_for_last_copies();
      }
    } else if (warp <= 10 && rank == 0) {
      // ---------------------------------------------------------------- MMA issuers (leader only)
      if (lane == 0) {
        const int parity = warp - 9;
        const uint32_t d_tmem = tmem_base + parity * kPairTile;
        const long long tiles_here = pair < num_tiles ? (num_tiles - pair + num_pairs - 1) / num_pairs : 0;
        const long long blocks = tiles_here * nkb;
        int stage = parity;
        uint32_t phase = 0;
        for (long long g = parity; g < blocks; g += 2) {
          if (!mbar_wait_soon(full + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSitePairMma)) break;
          tc_fence_after_sync();
          const uint64_t a_desc = umma_desc_kmajor_sw128(smem_u32(smem_a + stage * kPairOperandBytes));
          const uint64_t b_desc = umma_desc_kmajor_sw128(smem_u32(smem_b + stage * kPairOperandBytes));
#pragma unroll
          for (int k = 0; k < kBKBytes / 32; ++k) umma_pair<true>(d_tmem, a_desc + 2 * k, b_desc + 2 * k, kIdesc, k != 0);
          umma_commit_both(done + stage);
          stage += 2;
          if (stage >= kPairStages) stage -= kPairStages, phase ^= 1;
        }
      }
    } else if (warp == 11) {
      // ---------------------------------------------------------------- multipliers (both CTAs)
      // Lane l brings rows l, l + 32, l + 64, l + 96 of a_inv (and lanes 0 and 1 the squares' multipliers) two K blocks at a
      // time, the next two on their way while these are handed out, and with them the tile's first row and column.  Block g's place in the ring is free once block
      // g - 3 is done: its MMAs began after every promoting warp had given back the buffer of block g - 5.
      float next[2][4], next_b[2], now[2][4], now_b[2];
      const float *a_inv[4] = {}, *b_inv = nullptr;
      int corner = 0, next_corner = 0;  // lane 2: the tile's first row; lane 3: its first column
      auto enter_tile = [&](int tile) {
        int tm, tn;
        tile_coords(band, tile, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * kPairTile + (int)rank * kBM + lane, n0 = tn * kPairTile + (lane & 1) * 128;
        next_corner = lane == 2 ? m0 - lane : tn * kPairTile;
        // (rows and columns past the matrix have zero products; they get some multiplier that exists)
#pragma unroll
        for (int i = 0; i < 4; ++i) a_inv[i] = p.a_inv + (long long)min(m0 + 32 * i, p.M - 1) * nkb;
        b_inv = p.b_inv + (long long)(min(n0, p.N - 1) / 128) * nkb;
      };
      auto ask = [&](int kb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = min(kb + j, nkb - 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) next[j][i] = __ldg(a_inv[i] + at);
          next_b[j] = __ldg(b_inv + at);
        }
      };
      if (pair < num_tiles) {
        enter_tile(pair);
        ask(0);
      }
      int stage = 0, wait_stage = kPairStages - 3;
      uint32_t wait_phase = 1;  // of block g - 3; the first three blocks find their places free
      long long g = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        for (int kb0 = 0; kb0 < nkb && ok; kb0 += 2) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) now[j][i] = next[j][i];
            now_b[j] = next_b[j];
          }
          corner = kb0 == 0 ? next_corner : corner;
          if (kb0 + 2 < nkb) {
            ask(kb0 + 2);
          } else if (tile + num_pairs < num_tiles) {
            enter_tile(tile + num_pairs);
            ask(0);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (kb0 + j < nkb) {
              if (g >= 3 && ok)
                ok = mbar_wait_soon(done + wait_stage, wait_phase, abort_flag, p.d_status,
                                    XAXB_DEVICE_TIMEOUT * 1000 + kSitePairScales);
              ok = __all_sync(0xffffffffu, ok);
              float* to = smem_scale + stage * kPairScaleFloats;
#pragma unroll
              for (int i = 0; i < 4; ++i) to[lane + 32 * i] = now[j][i];
              if (lane < 4) to[128 + lane] = lane < 2 ? now_b[j] : __int_as_float(corner);
              __syncwarp();
              if (lane == 0) mbar_arrive(done + stage);
              ++g;
              if (++stage == kPairStages) stage = 0;
              if (++wait_stage == kPairStages) wait_stage = 0, wait_phase ^= 1;
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ promotion and epilogue (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairPromoteRegs));
    const int quarter = warp & 3, half = warp >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + half * 128;
    uint8_t* out_blocks = smem_out + half * 2 * kPairOutBytes;
    int stage = 0, next = 2 % kPairStages;  // the block's stage, and that of the block that will use its buffer next
    uint32_t phase = 0;
    int buf = 0;
    bool ok = true;
    if (lane == 0) {  // both buffers start free
      mbar_arrive_cluster(dsmem_addr(smem_u32(full), 0));
      mbar_arrive_cluster(dsmem_addr(smem_u32(full + 1), 0));
    }
    const uint32_t leader_full = dsmem_addr(smem_u32(full), 0);
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      int m0 = 0, n0 = 0;
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
#pragma unroll 1
      for (int kb = 0; kb < nkb; ++kb) {
        if (!mbar_try_wait(done + stage, phase) && ok)
          ok = mbar_wait_soon(done + stage, phase, abort_flag, p.d_status, XAXB_DEVICE_TIMEOUT * 1000 + kSitePairPromote);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          tc_fence_after_sync();
          const uint32_t from = taddr + buf * kPairTile;
          // Five readouts, each asked for while the one before is added (a wait covers all that are on their way, so
          // there is one at a time; 32 + 16 columns are what the registers hold beside the 128 sums).
          uint32_t r[32], t[16];
          tmem_ld_x32(from, r);
          const float* scale = smem_scale + stage * kPairScaleFloats;
          const float sc = scale[row] * scale[128 + half];
          if (kb == nkb - 1) m0 = __float_as_int(scale[130]), n0 = __float_as_int(scale[131]) + half * 128;
#pragma unroll
          for (int c = 0; c < 128; c += 48) {
            tmem_ld_wait();
            if (c < 96) {
              tmem_ld_x16(from + c + 32, t);
            } else {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(leader_full + next * 8);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) fma2(acc[c + i], acc[c + i + 1], r[i], r[i + 1], sc, sc);
            if (c < 96) {
              tmem_ld_wait();
              tmem_ld_x32(from + c + 48, r);
#pragma unroll
              for (int i = 0; i < 16; i += 2) fma2(acc[c + 32 + i], acc[c + 33 + i], t[i], t[i + 1], sc, sc);
            }
          }
        }
        buf ^= 1;
        if (++stage == kPairStages) stage = 0, phase ^= 1;
        if (++next == kPairStages) next = 0;
      }
      // The tile's rows, 128 columns a thread, to two staging blocks and from there by TMA, which clips at M and N.
      if (p.bias) {
#pragma unroll
        for (int c = 0; c < 128; c += 8)
          if (n0 + c < p.N) add8(&acc[c], __ldg(reinterpret_cast<const uint4*>(p.bias + n0 + c)));
      }
      if (p.residual && m0 + row < p.M) {
        const __nv_bfloat16* residual = p.residual + (m0 + row) * p.ldr + n0;
#pragma unroll
        for (int c = 0; c < 128; c += 8)
          if (n0 + c < p.N) add8(&acc[c], *reinterpret_cast<const uint4*>(residual + c));
      }
      if (quarter < 2 && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      warpgroup_sync(half);
#pragma unroll
      for (int c = 0; c < 128; c += 8)
        *reinterpret_cast<uint4*>(out_blocks + c / 64 * kPairOutBytes + sw128_offset(row, c % 64 / 8)) =
            make_uint4(bf16x2(acc[c], acc[c + 1]), bf16x2(acc[c + 2], acc[c + 3]), bf16x2(acc[c + 4], acc[c + 5]),
                       bf16x2(acc[c + 6], acc[c + 7]));
      fence_proxy_async_smem();
      warpgroup_sync(half);
      if (quarter < 2 && lane == 0 && ok) {  // a block each
        const int n = n0 + quarter * 64;
        if (n < p.N && m0 < p.M)
          asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                       ::"l"(&tmap_out), "r"(smem_u32(out_blocks + quarter * kPairOutBytes)), "r"(n), "r"(m0)
                       : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
    if (quarter < 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // no arrival or operand read of the peer can still target a CTA that leaves
  if (warp == 9) {
    tc_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// How many CTA pairs can be resident at once (not every SM has a partner).
static int blocks_resident_pairs(const Ctx* ctx) {
  static int pairs = 0;
  if (pairs == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * (ctx->num_sms / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, gemm_blocks_pair_kernel, &cfg);
    pairs = e == cudaSuccess && n > 0 ? n : ctx->num_sms / 2 - 8;
  }
  return pairs;
}

static int launch_pair(const Ctx* ctx, cudaStream_t stream, const GemmBlocksParams& p) {
  CUtensorMap ta, tb, tout;
  if (int rc = make_tmap_2d(ctx, &ta, p.a, 1, (uint64_t)p.K, (uint64_t)p.M, (uint64_t)p.lda, kBKBytes, kBM)) return rc;
  if (int rc = make_tmap_2d(ctx, &tb, p.b, 1, (uint64_t)p.K, (uint64_t)p.N, (uint64_t)p.ldb, kBKBytes, kBM)) return rc;
  if (int rc = make_tmap_2d(ctx, &tout, p.out, 2, (uint64_t)p.N, (uint64_t)p.M, (uint64_t)p.ldo * 2, 64, kBM)) return rc;
  if (int rc = ensure_dynamic_smem<gemm_blocks_pair_kernel>(ctx, kPairSmemBytes, "gemm_blocks_pair_kernel")) return rc;
  const int tiles_m = (p.M + kPairTile - 1) / kPairTile, tiles_n = (p.N + kPairTile - 1) / kPairTile;
  const long long tiles = (long long)tiles_m * tiles_n;
  const int max_pairs = blocks_resident_pairs(ctx);
  const int pairs = tiles < max_pairs ? (int)tiles : max_pairs;
  cudaError_t e = launch_kernel(gemm_blocks_pair_kernel, dim3((unsigned)(2 * pairs)), dim3(kPairThreads), kPairSmemBytes, stream,
                                2u, ta, tb, tout, p, tiles_m, tiles_n, 16);
  if (e != cudaSuccess) {
    set_last_error("gemm_blocks_pair_kernel launch: %s", cudaGetErrorString(e));
    return XAXB_LAUNCH_FAILED;
  }
  return check_launch("gemm_blocks_pair_kernel");
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
  const long long pair_tiles = ((M + kPairTile - 1) / kPairTile) * ((N + kPairTile - 1) / kPairTile);
  if (pair_tiles > 0x3fffffff) {
    set_last_error("gemm_fp8_blocks: [%lld, %lld] has too many tiles", (long long)M, (long long)N);
    return XAXB_BAD_ARGUMENT;
  }
  // The pair kernel from where 128 x 128 tiles no longer fit one on an SM: 512 x 4096 x 4096 (128 tiles) 17.9 us on them and
  // 19.1 on pairs, 768 x 4096 x 4096 (192 tiles) 26.9 and 20.2, 256 x 28672 x 4096 52.4 and 35.9.
  if (M > 128 && ((M + kBM - 1) / kBM) * ((N + kBM - 1) / kBM) > ctx->num_sms) return launch_pair(ctx, s, p);
  if (M <= 16) return launch_decode<16>(ctx, s, p);
  if (M <= 32) return launch_decode<32>(ctx, s, p);
  if (M <= 64) return launch_decode<64>(ctx, s, p);
  return launch_decode<128>(ctx, s, p);
}
