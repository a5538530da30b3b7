// 8-bit integer projections:
//   out[M,N] = epi( (round(x / sx) . w^T) * sx[row] * sw[col] + bias[col] )
// x is quantized per row (sx = amax / 127, k_quant_rows), w [N, K] int8 comes with a
// scale per output channel.  Products and sums are exact in int32.  Epilogues: bias,
// bias + GELU (out in x's type or fp32), bias + fp32 residual.
#pragma once

#include "gemm.cuh"
#include "kv8.cuh"

namespace b200 {

enum Dt : int { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };

// x [M, K] (row stride ldx elements) -> codes int8 [M, ldq], scale [M].  A row with an
// infinity or NaN gets a NaN scale, so its outputs are NaN.  One CTA a row; the row is
// read twice, the second time from L1/L2.
template <int DT>
__global__ void __launch_bounds__(256) k_quant_rows(const void* x, long long ldx, int8_t* q, long long ldq,
                                                    float* scale, int M, int K) {
  __shared__ unsigned tops[8];
  griddep_sync();
  const int tid = threadIdx.x;
  const size_t row = blockIdx.x;
  auto at = [&](int k) -> float {
    if constexpr (DT == DT_F32) return static_cast<const float*>(x)[row * ldx + k];
    else return h16_to_f(static_cast<const uint16_t*>(x)[row * ldx + k], DT == DT_BF16);
  };
  unsigned top = 0;
  for (int k = tid; k < K; k += 256) top = max(top, __float_as_uint(at(k)) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
  for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
  const float s = top < 0x7f800000u ? __fmul_rn(__uint_as_float(top), 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  if (tid == 0) scale[row] = s;
  for (int k = tid; k < K; k += 256) {
    const float r = s > 0.f ? rintf(__fdiv_rn(at(k), s)) : 0.f;
    q[row * ldq + k] = static_cast<int8_t>(static_cast<int>(fminf(fmaxf(r, -127.f), 127.f)));
  }
}

struct GemmI8Params {
  int M, N, K;
  const float* sx;     // [M]
  const float* sw;     // [N]
  const float* bias;   // [N], may be null
  const float* resid;  // fp32 [M, N], row stride ld_resid, may be null
  long long ld_resid;
  void* out;           // [M, N], row stride ld_out
  long long ld_out;
  int gelu, dt;        // output type
};

// kind::i8 instruction descriptor: int32 accumulators (bits 4-5 = 2), signed 8-bit A and B, both K-major
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void umma_i8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}

// One row's `cols` (up to 32) results from column col0 on: v holds the int32 sums.
__device__ __forceinline__ void gemm_i8_row(const GemmI8Params& p, int row, int col0, float (&v)[32]) {
  const int cols = min(32, p.N - col0);
  if (row >= p.M || cols <= 0) return;
  const float sx = __ldg(p.sx + row);
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const int c = min(col0 + j, p.N - 1);
    float y = __fmul_rn(__fmul_rn(static_cast<float>(__float_as_int(v[j])), sx), __ldg(p.sw + c));
    if (p.bias) y = __fadd_rn(y, __ldg(p.bias + c));
    if (p.gelu) y = gelu_as(y);
    if (p.resid) y += __ldg(p.resid + row * p.ld_resid + c);
    v[j] = y;
  }
  if (p.dt == DT_F32) {
    float* o = static_cast<float*>(p.out) + row * p.ld_out + col0;
    for (int j = 0; j < cols; ++j) o[j] = v[j];
  } else {
    uint16_t* o = static_cast<uint16_t*>(p.out) + row * p.ld_out + col0;
    for (int j = 0; j < cols; ++j) o[j] = static_cast<uint16_t>(f_to_h16(v[j], p.dt == DT_BF16));
  }
}

// The persistent schedule of k_gemm_tn with 128-byte K slices of 8-bit operands.
template <int BN, int STAGES>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    k_gemm_i8(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const GemmI8Params p) {
  constexpr int A_BYTES = 128 * 128, STAGE_BYTES = A_BYTES + BN * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ntl = (p.N + BN - 1) / BN, ntiles = (p.M + 127) / 128 * ntl;
  const int my_tiles = (ntiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int nk = (p.K + 127) / 128;
  constexpr uint32_t TMEM_COLS = 2 * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 256);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_sync();

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmW);
      int it = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int t = static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
        const int m0 = (t / ntl) * 128, n0 = (t % ntl) * BN;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, abort_flag, DERR_WAIT_SLOT)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * STAGE_BYTES;
          mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
          tma_load_2d(st, &tmA, &full[s], kb * 128, m0);
          tma_load_2d(st + A_BYTES, &tmW, &full[s], kb * 128, n0);
        }
      }
      if (*abort_flag)
        for (int j = (it > STAGES ? it - STAGES : 0); j < it; ++j) mbar_wait_drain(&full[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_i8(128, BN);
      int it = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int b = i & 1;
        if (i >= 2 && !mbar_wait(&acc_empty[b], ((i >> 1) - 1) & 1, abort_flag, DERR_WAIT_MMA)) break;
        tc_fence_after();
        const uint32_t dcol = tmem + b * BN;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag, DERR_WAIT_TMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES), b_addr = a_addr + A_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8_ss(dcol, make_sdesc(a_addr + kk * 32, 16, 1024, UMMA_SW128),
                       make_sdesc(b_addr + kk * 32, 16, 1024, UMMA_SW128), idesc, (kb | kk) != 0 ? 1u : 0u);
          tc_commit(&empty[s]);
        }
        if (!ok) break;
        tc_commit(&acc_full[b]);
      }
      if (*abort_flag) {
        tc_commit(drain);
        mbar_wait_drain(drain, 0);
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    for (int i = 0; i < my_tiles; ++i) {
      const int b = i & 1;
      const int t = static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
      const int row = (t / ntl) * 128 + q * 32 + lane, n0 = (t % ntl) * BN;
      const bool ok = mbar_wait_warp(&acc_full[b], (i >> 1) & 1, abort_flag, DERR_WAIT_MMA);
      if (!ok || *abort_flag) break;
      tc_fence_after();
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
        float v[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(q * 32) << 16) + b * BN + c, v);
        gemm_i8_row(p, row, n0 + c, v);
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[b]);
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace b200
