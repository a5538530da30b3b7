// 8-bit integer projections:
//   out[M,N] = epi( (round(x / sx) . w^T) * sx[row] * sw[col] + bias[col] )
// x is quantized per row (sx = amax / 127, k_quant_rows), w [N, K] int8 comes with a
// scale per output channel.  Products and sums are exact in int32.  Epilogues: bias,
// bias + GELU (out in x's type or fp32), bias + fp32 residual.  fp32 results take GELU's erf from
// erff; 16-bit ones take the form of gelu_as, within 2e-6, which their own rounding hides but for
// results near 0 (8192x1024x4096 of fp32: 71 us, with gelu_as 61).
#pragma once

#include "gemm2.cuh"
#include "kv8.cuh"

namespace b200 {

enum Dt : int { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };

// 16 consecutive values of a row from k on (zeros past K); vec: all 16 exist and the address is 16-byte aligned
template <int DT>
__device__ __forceinline__ void load_row16(const void* x, size_t base, int k, int K, bool vec, float (&v)[16]) {
  if (vec) {
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(x) + base + k) + i);
        v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float u[8];
        unpack8<DT == DT_BF16>(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + base + k) + i), u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = u[j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (k + j >= K) v[j] = 0.f;
      else if constexpr (DT == DT_F32) v[j] = __ldg(static_cast<const float*>(x) + base + k + j);
      else v[j] = h16_to_f(__ldg(static_cast<const uint16_t*>(x) + base + k + j), DT == DT_BF16);
    }
  }
}

// x [M, K] (row stride ldx elements) -> codes int8 [M, ldq], scale [M].  A row with an
// infinity or NaN gets a NaN scale, so its outputs are NaN.  TPR threads a row: a warp for
// 2048 rows or more of up to 2048 values (32768x1024 fp16 in 23 us, 4.4 TB/s), else 256
// (333x1001 bf16: the product 10.2 us, with a warp a row 12.7); the row is read twice,
// the second time from L1.
// Memory-bound.  vec: x's rows start 16-byte aligned.  Only the K codes of a row are
// written, 16 at a time where they start on 16 bytes.
template <int DT, int TPR>
__global__ void __launch_bounds__(256) k_quant_rows(const void* x, long long ldx, int8_t* q, long long ldq,
                                                    float* scale, int M, int K, int vec) {
  __shared__ unsigned tops[8];
  griddep_sync();
  const int tid = threadIdx.x % TPR;
  const size_t row = static_cast<size_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (TPR == 32 && row >= static_cast<size_t>(M)) return;
  const size_t base = row * ldx;
  auto one = [&](int k) {  // rows that start off 16 bytes: lanes side by side, a value each
    if (k >= K) return 0.f;
    if constexpr (DT == DT_F32) return __ldg(static_cast<const float*>(x) + base + k);
    else return h16_to_f(__ldg(static_cast<const uint16_t*>(x) + base + k), DT == DT_BF16);
  };
  unsigned top = 0;
  if (vec) {
    for (int k = tid * 16; k < K; k += TPR * 16) {
      float v[16];
      load_row16<DT>(x, base, k, K, k + 16 <= K, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
  } else {
#pragma unroll 8
    for (int k = tid; k < K; k += TPR) top = max(top, __float_as_uint(one(k)) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (TPR > 32) {
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    __syncthreads();
    for (int i = 0; i < TPR / 32; ++i) top = max(top, tops[i]);
  }
  const float s = top < 0x7f800000u ? __fmul_rn(__uint_as_float(top), 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  if (tid == 0) scale[row] = s;
  const bool live = s > 0.f;                // false: a row of zeros, or NaN
  const bool small = s < 1e-30f;            // 1 / s could overflow: divide
  const float inv = __fdiv_rn(1.f, s);
  if (!vec) {
#pragma unroll 2
    for (int k = tid; k < K; k += 4 * TPR) {
      const uint32_t w = live ? quantize4(one(k), one(k + TPR), one(k + 2 * TPR), one(k + 3 * TPR), s, inv, small) : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j * TPR < K) q[row * ldq + k + j * TPR] = static_cast<int8_t>(w >> (8 * j));
    }
    return;
  }
  for (int k = tid * 16; k < K; k += TPR * 16) {
    float v[16];
    load_row16<DT>(x, base, k, K, k + 16 <= K, v);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (live) {
      w.x = quantize4(v[0], v[1], v[2], v[3], s, inv, small);
      w.y = quantize4(v[4], v[5], v[6], v[7], s, inv, small);
      w.z = quantize4(v[8], v[9], v[10], v[11], s, inv, small);
      w.w = quantize4(v[12], v[13], v[14], v[15], s, inv, small);
    }
    int8_t* to = q + row * ldq + k;
    if (k + 16 <= K && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      *reinterpret_cast<uint4*>(to) = w;
    } else {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k + j < K) to[j] = static_cast<int8_t>(x[j >> 2] >> (8 * (j & 3)));
    }
  }
}

enum I8Epilogue : int { I8_BIAS = 0, I8_GELU = 1, I8_RESID = 2 };

struct GemmI8Params {
  int M, N, K;
  const float* sx;     // [M]
  const float* sw;     // [N]
  const float* bias;   // [N], may be null
  const float* resid;  // I8_RESID: fp32 [M, N], row stride ld_resid
  long long ld_resid;
  void* out;           // [M, N], row stride ld_out
  long long ld_out;
  int vec_resid;       // resid's rows are 16-byte aligned
  int tma_out;         // out's rows are 16-byte aligned: tiles leave by TMA store
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

template <int DT>
struct I8Out {
  static constexpr int CC = DT == DT_F32 ? 16 : 32;  // columns of a 64-byte chunk row
};
constexpr int I8_STG_WARP = 4096 + 1024;  // per epilogue warp: two 2 KB chunk slots, then 128 columns' scales and biases

// Scales and biases of the 128 columns from col0 on into the warp's own shared memory (0 past N).
__device__ __forceinline__ void i8_columns(const GemmI8Params& p, int col0, float* cols, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = col0 + lane + 32 * i;
    cols[lane + 32 * i] = c < p.N ? __ldg(p.sw + c) : 0.f;
    cols[128 + lane + 32 * i] = p.bias != nullptr && c < p.N ? __ldg(p.bias + c) : 0.f;
  }
  __syncwarp();
}

// Epilogue of `width` (<= 128) columns of an accumulator tile for one warp: 32 rows from row0, one a lane.
// Chunks of 64 bytes a row are staged (SWIZZLE_64B) in the warp's two slots and leave by TMA store, or, where
// out's rows are not 16-byte aligned, element by element along the rows.
template <int DT, int EPI>
__device__ __forceinline__ void i8_epilogue(const CUtensorMap* tmO, const GemmI8Params& p, uint32_t taddr, int width,
                                            int col0, int row0, uint8_t* stg, int& gc, int lane) {
  constexpr int CC = I8Out<DT>::CC;
  const float* cols = reinterpret_cast<const float*>(stg + 4096);
  const uint32_t sw = static_cast<uint32_t>((lane >> 1) & 3);
  const int row = row0 + lane;
  const float sx = row < p.M ? __ldg(p.sx + row) : 0.f;
  const uint64_t sx2 = f2pk(sx, sx);
#pragma unroll 1
  for (int c = 0; c < width; c += CC, ++gc) {
    const int col = col0 + c;
    if (col >= p.N) break;
    float v[CC];
    if constexpr (DT == DT_F32) tmem_ld16(taddr + c, v);
    else tmem_ld32(taddr + c, v);
    if constexpr (EPI == I8_RESID) {
      if (row < p.M) {
        const float* r = p.resid + row * p.ld_resid + col;
        float u[CC];
        if (p.vec_resid && col + CC <= p.N) {
#pragma unroll
          for (int j = 0; j < CC; j += 4) {
            const float4 w = *reinterpret_cast<const float4*>(r + j);  // (not __ldg: resid may be out)
            u[j] = w.x; u[j + 1] = w.y; u[j + 2] = w.z; u[j + 3] = w.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < CC; ++j) u[j] = col + j < p.N ? r[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < CC; ++j)
          v[j] = __fadd_rn(u[j], __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(v[j])), sx), cols[c + j]),
                                           cols[128 + c + j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < CC; j += 2) {
        uint64_t y = f2pk(__int2float_rn(__float_as_int(v[j])), __int2float_rn(__float_as_int(v[j + 1])));
        y = f2mul(f2mul(y, sx2), *reinterpret_cast<const uint64_t*>(cols + c + j));
        y = f2add(y, *reinterpret_cast<const uint64_t*>(cols + 128 + c + j));
        f2upk(y, v[j], v[j + 1]);
        if constexpr (EPI == I8_GELU && DT == DT_F32) {
          v[j] = gelu_erf(v[j]);
          v[j + 1] = gelu_erf(v[j + 1]);
        } else if constexpr (EPI == I8_GELU) {
          gelu_as2(v[j], v[j + 1]);
        }
      }
    }
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if constexpr (DT == DT_F32) w[j] = __float_as_uint(v[j]);
      else w[j] = pack2<DT == DT_BF16>(v[2 * j], v[2 * j + 1]);
    }
    uint8_t* slot = stg + (gc & 1) * 2048;
    if (lane == 0) bulk_wait_read_1();  // the slot's previous chunk has left
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(slot + lane * 64 + ((j ^ sw) << 4)) =
          make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    if (p.tma_out) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(tmO, slot, col, row0);
        bulk_commit();
      }
    } else {
      __syncwarp();
      const int rows = min(32, p.M - row0);
      if constexpr (DT == DT_F32) {
        for (int r = lane >> 4; r < rows; r += 2) {
          const int j = lane & 15;
          if (col + j < p.N)
            static_cast<float*>(p.out)[(row0 + r) * p.ld_out + col + j] = *reinterpret_cast<const float*>(
                slot + r * 64 + (((j >> 2) ^ ((r >> 1) & 3)) << 4) + (j & 3) * 4);
        }
      } else {
        for (int r = 0; r < rows; ++r)
          if (col + lane < p.N)
            static_cast<uint16_t*>(p.out)[(row0 + r) * p.ld_out + col + lane] = *reinterpret_cast<const uint16_t*>(
                slot + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
      }
    }
  }
}

// The persistent schedule of k_gemm_tn with 128-byte K slices of 8-bit operands.
template <int BN, int STAGES>
struct GemmI8Smem {
  static constexpr int A_BYTES = 128 * 128, STAGE_BYTES = A_BYTES + BN * 128;
  static constexpr int STG_OFF = STAGES * STAGE_BYTES, BAR_OFF = STG_OFF + 8 * I8_STG_WARP;
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;
};
template <int BN, int STAGES, int DT, int EPI>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    k_gemm_i8(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
              const __grid_constant__ CUtensorMap tmO, const GemmI8Params p) {
  using L = GemmI8Smem<BN, STAGES>;
  constexpr int A_BYTES = L::A_BYTES, STAGE_BYTES = L::STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
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
    uint8_t* stg = smem + L::STG_OFF + (warp - 2) * I8_STG_WARP;
    int gc = 0;
    for (int i = 0; i < my_tiles; ++i) {
      const int b = i & 1;
      const int t = static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
      const int row0 = (t / ntl) * 128 + q * 32, col0 = (t % ntl) * BN + half * (BN / 2);
      i8_columns(p, col0, reinterpret_cast<float*>(stg + 4096), lane);
      const bool ok = mbar_wait_warp(&acc_full[b], (i >> 1) & 1, abort_flag, DERR_WAIT_MMA);
      if (!ok || *abort_flag) break;
      tc_fence_after();
      i8_epilogue<DT, EPI>(&tmO, p, tmem + (static_cast<uint32_t>(q * 32) << 16) + b * BN + half * (BN / 2), BN / 2, col0,
                           row0, stg, gc, lane);
      tc_fence_before();
      mbar_arrive(&acc_empty[b]);
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// The same on CTA pairs, after k_gemm2_tn: one 256x256 tile a pair, each CTA staging its 128 rows of x's codes and
// 128 rows of w per 128-byte K slice.  Measured, row quantization included: 8192x4096x4096 bf16 111 us (2.47 PFLOP/s),
// 32768x1024x4096 143 us, with GELU 170 us (the epilogue), 32768x4096x1024 onto the residual 199 us.
__host__ __device__ constexpr int gemm2_i8_stages(int ew) { return ew == 16 ? 4 : 5; }
template <int EW>
struct Gemm2I8Smem {
  static constexpr int A_BYTES = 128 * 128, STAGE_BYTES = 2 * A_BYTES;
  static constexpr int STG_OFF = gemm2_i8_stages(EW) * STAGE_BYTES, BAR_OFF = STG_OFF + EW * I8_STG_WARP;
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;
};
__device__ __forceinline__ void umma_i8_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}\n"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u),
        "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
template <int DT, int EPI, int EW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * EW, 1)
    k_gemm2_i8(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
               const __grid_constant__ CUtensorMap tmO, const GemmI8Params p) {
  constexpr int STAGES = gemm2_i8_stages(EW), CW = 256 / (EW / 4);  // columns a warp
  using L = Gemm2I8Smem<EW>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cid = static_cast<int>(blockIdx.x) >> 1, ncl = static_cast<int>(gridDim.x) >> 1;
  const int ntl = (p.N + 255) / 256, ntiles = (p.M + 255) / 256 * ntl;
  const int my_tiles = (ntiles - cid + ncl - 1) / ncl;
  const int nk = (p.K + 127) / 128;
  constexpr uint32_t TMEM_COLS = 512;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * EW);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
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
        const int t = cid + i * ncl;
        const int m0 = (t / ntl) * 256, n0 = (t % ntl) * 256;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, abort_flag, DERR_WAIT_SLOT)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * L::STAGE_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE_BYTES);
          const uint32_t fbar = mapa_shared(smem_u32(&full[s]), 0);
          tma_load_2d_pair(st, &tmA, fbar, kb * 128, m0 + 128 * static_cast<int>(rank));
          tma_load_2d_pair(st + L::A_BYTES, &tmW, fbar, kb * 128, n0 + 128 * static_cast<int>(rank));
        }
      }
      if (*abort_flag && rank == 0)
        for (int j = (it > STAGES ? it - STAGES : 0); j < it; ++j) mbar_wait_drain(&full[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc_i8(256, 256);
      int it = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int b = i & 1;
        if (i >= 2 && !mbar_wait(&acc_empty[b], ((i >> 1) - 1) & 1, abort_flag, DERR_WAIT_MMA)) break;
        tc_fence_after();
        const uint32_t dcol = tmem + b * 256;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag, DERR_WAIT_TMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * L::STAGE_BYTES), b_addr = a_addr + L::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8_ss_pair(dcol, make_sdesc(a_addr + kk * 32, 16, 1024, UMMA_SW128),
                            make_sdesc(b_addr + kk * 32, 16, 1024, UMMA_SW128), idesc, (kb | kk) != 0 ? 1u : 0u);
          tc_commit_pair(&empty[s], 0x3);
        }
        if (!ok) break;
        tc_commit_pair(&acc_full[b], 0x3);
      }
      if (*abort_flag) {
        tc_commit_pair(drain, 0x1);
        mbar_wait_drain(drain, 0);
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    uint8_t* stg = smem + L::STG_OFF + (warp - 2) * I8_STG_WARP;
    const uint32_t empty_leader0 = mapa_shared(smem_u32(&acc_empty[0]), 0);
    int gc = 0;
    for (int i = 0; i < my_tiles; ++i) {
      const int b = i & 1;
      const int t = cid + i * ncl;
      const int row0 = (t / ntl) * 256 + 128 * static_cast<int>(rank) + q * 32, col0 = (t % ntl) * 256 + part * CW;
      i8_columns(p, col0, reinterpret_cast<float*>(stg + 4096), lane);
      const bool ok = mbar_wait_warp(&acc_full[b], (i >> 1) & 1, abort_flag, DERR_WAIT_MMA);
      if (!ok || *abort_flag) break;
      tc_fence_after();
      i8_epilogue<DT, EPI>(&tmO, p, tmem + (static_cast<uint32_t>(q * 32) << 16) + b * 256 + part * CW, CW, col0, row0,
                           stg, gc, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(empty_leader0 + b * 8);
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

// Few rows (M <= 64): one kernel that quantizes and multiplies.  The weight is what has to be read, so w's rows fill
// the 128 rows of the tcgen05 step and x's rows its N = 16 .. 64 columns, and a cluster of CTAs splits K:
//   - each CTA's slices of w (128 rows x 128 bytes, at most LIN_SLICES) come by TMA while
//   - its warps find the rows' maxima over the CTA's part of K, exchange them in the cluster, and write the codes of
//     x in SWIZZLE_128B order;
//   - the partial int32 sums (exact, so any order gives the same bits) go to shared memory, and each CTA adds and
//     finishes a share of the rows through distributed shared memory.
// Latency-bound.  Against the quantizer and the 128x128 kernel one after the other: 1x1024x4096 GELU 8.3 -> 5.4 us,
// 64x4096x1024 residual 18.9 -> 10.6 us (device time in a CUDA graph; 8 warps a CTA up to 16 rows, where 16 take
// 6.1 us, and 16 above, where 8 take 13.9 us: the quantization's instructions).
constexpr int LIN_ROWS = 64, LIN_SLICES = 8, LIN_MAX_CLUSTER = 8, LIN_MAX_WARPS = 16;

struct LinSmallParams {
  GemmI8Params g;      // (g.sx unused)
  const void* x;
  long long ldx;
  int vec, out_type, epi;
  int pad, slices, cluster;  // rows of x rounded up to 16, K slices a CTA, CTAs a cluster
};
struct LinSmallSmem {
  static constexpr int W_SLICE = 128 * 128;
  int x_off, meta_off, total;
  __host__ __device__ LinSmallSmem(int pad, int slices) {
    const int w = slices * W_SLICE, acc = pad * 128 * 4;
    x_off = w > acc ? w : (acc + 1023) / 1024 * 1024;
    meta_off = x_off + slices * pad * 128;
    total = meta_off + 2 * LIN_ROWS * 4 + 64 + 1024;
  }
};
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

template <int DT>
__global__ void __launch_bounds__(32 * LIN_MAX_WARPS, 1) k_lin_small(const __grid_constant__ CUtensorMap tmW, const LinSmallParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  const LinSmallSmem L(p.pad, p.slices);
  unsigned* tops = reinterpret_cast<unsigned*>(smem + L.meta_off);
  float* sx = reinterpret_cast<float*>(tops + LIN_ROWS);
  uint64_t* full = reinterpret_cast<uint64_t*>(sx + LIN_ROWS);
  uint64_t* done = full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank()), n0 = static_cast<int>(blockIdx.x) / p.cluster * 128;
  const int M = p.g.M, K = p.g.K;
  const int s0 = rank * p.slices, ns = max(0, min(p.slices, (K + 127) / 128 - s0));  // this CTA's slices
  const int k0 = s0 * 128, k1 = min(K, k0 + ns * 128);
  const uint32_t cols = p.pad <= 32 ? 32 : 64;
  if (tid == 0) {
    mbar_init(full, 1);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_sync();
  if (tid == 0 && ns > 0) {
    mbar_arrive_expect_tx(full, ns * LinSmallSmem::W_SLICE);
    for (int s = 0; s < ns; ++s) tma_load_2d(smem + s * LinSmallSmem::W_SLICE, &tmW, full, (s0 + s) * 128, n0);
  }
  __syncwarp();
  // the rows' maxima over this CTA's part of K: four rows a warp side by side, 16 values a lane of each
  for (int r0 = warp; r0 < M; r0 += 4 * warps) {
    unsigned top[4] = {0, 0, 0, 0};
    for (int k = k0 + lane * 16; k < k1; k += 512) {
      float v[4][16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + warps * i < M) load_row16<DT>(p.x, (r0 + warps * i) * p.ldx, k, k1, p.vec && k + 16 <= k1, v[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + warps * i < M)
#pragma unroll
          for (int j = 0; j < 16; ++j) top[i] = max(top[i], __float_as_uint(v[i][j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[i] = __reduce_max_sync(0xffffffffu, top[i]);
      if (lane == 0 && r0 + warps * i < M) tops[r0 + warps * i] = top[i];
    }
  }
  __syncthreads();
  cluster_sync_all();
  if (tid < M) {
    unsigned each[LIN_MAX_CLUSTER], top = 0;
#pragma unroll
    for (int c = 0; c < LIN_MAX_CLUSTER; ++c) each[c] = ld_cluster_u32(mapa_shared(smem_u32(tops + tid), c & (p.cluster - 1)));
#pragma unroll
    for (int c = 0; c < LIN_MAX_CLUSTER; ++c) top = max(top, each[c]);
    sx[tid] = top < 0x7f800000u ? __fmul_rn(__uint_as_float(top), 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  }
  __syncthreads();
  for (int r0 = warp; r0 < M; r0 += 4 * warps)
    for (int k = lane * 16; k < ns * 128; k += 512) {
      float v[4][16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + warps * i < M) load_row16<DT>(p.x, (r0 + warps * i) * p.ldx, k0 + k, k1, p.vec && k0 + k + 16 <= k1, v[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + warps * i;
        if (r >= M) break;
        const float s = sx[r], inv = __fdiv_rn(1.f, s);
        const bool small = s < 1e-30f;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (s > 0.f) {  // false: a row of zeros, or NaN
          w.x = quantize4(v[i][0], v[i][1], v[i][2], v[i][3], s, inv, small);
          w.y = quantize4(v[i][4], v[i][5], v[i][6], v[i][7], s, inv, small);
          w.z = quantize4(v[i][8], v[i][9], v[i][10], v[i][11], s, inv, small);
          w.w = quantize4(v[i][12], v[i][13], v[i][14], v[i][15], s, inv, small);
        }
        *reinterpret_cast<uint4*>(smem + L.x_off + (k >> 7) * p.pad * 128 + sw128_off(r, (k >> 4) & 7)) = w;
      }
    }
  fence_proxy_async_smem();
  __syncthreads();
  bool ok = true;
  if (ns > 0) {
    if (warp == 1 && lane == 0) {
      if (mbar_wait(full, 0, abort_flag, DERR_WAIT_TMA)) {
        tc_fence_after();
        const uint32_t idesc = make_idesc_i8(128, p.pad);
        for (int s = 0; s < ns; ++s) {
          const uint32_t a = smem_u32(smem + s * LinSmallSmem::W_SLICE), b = smem_u32(smem + L.x_off + s * p.pad * 128);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8_ss(tmem, make_sdesc(a + kk * 32, 16, 1024, UMMA_SW128), make_sdesc(b + kk * 32, 16, 1024, UMMA_SW128),
                       idesc, (s | kk) != 0 ? 1u : 0u);
        }
        tc_commit(done);
      } else {
        mbar_wait_drain(full, 0);
      }
    }
    __syncwarp();
    ok = mbar_wait_warp(done, 0, abort_flag, DERR_WAIT_MMA);
    if (ok) tc_fence_after();
  }
  // the sums, [row of x][column], over the slices of w (which every product has read)
  int* acc = reinterpret_cast<int*>(smem);
  __syncthreads();
  for (int c = (warp >> 2) * 16; c < p.pad; c += warps * 4) {
    float v[16];
    if (ns > 0 && ok) {
      tmem_ld16(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[(c + j) * 128 + (warp & 3) * 32 + lane] = __float_as_int(v[j]);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  const int col = n0 + (tid & 127);
  if (col < p.g.N) {
    const float sw = __ldg(p.g.sw + col), bias = p.g.bias ? __ldg(p.g.bias + col) : 0.f;
#pragma unroll 4
    for (int m = rank + p.cluster * (tid >> 7); m < M; m += (warps >> 2) * p.cluster) {
      const uint32_t at = smem_u32(acc + m * 128 + (tid & 127));
      int each[LIN_MAX_CLUSTER], sum = 0;  // one round trip for all
#pragma unroll
      for (int c = 0; c < LIN_MAX_CLUSTER; ++c) each[c] = c < p.cluster ? static_cast<int>(ld_cluster_u32(mapa_shared(at, c))) : 0;
#pragma unroll
      for (int c = 0; c < LIN_MAX_CLUSTER; ++c) sum += each[c];
      float y = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), sx[m]), sw), bias);
      if (p.epi == I8_GELU) y = p.out_type == DT_F32 ? gelu_erf(y) : gelu_as(y);
      if (p.epi == I8_RESID) y = __fadd_rn(p.g.resid[m * p.g.ld_resid + col], y);
      const long long to = m * p.g.ld_out + col;
      if (p.out_type == DT_F32) static_cast<float*>(p.g.out)[to] = y;
      else static_cast<uint16_t*>(p.g.out)[to] = static_cast<uint16_t>(f_to_h16(y, p.out_type == DT_BF16));
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

}  // namespace b200
