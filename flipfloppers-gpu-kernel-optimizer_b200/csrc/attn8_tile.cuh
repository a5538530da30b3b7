// Attention over the 8-bit paged cache for many rows (chunks of prompts): the same
// operator as attn8.cuh on tcgen05.  A CTA takes 256 rows of one key head (query heads
// of its group times new tokens) as two 128-row tiles and walks the keys in tiles of
// 128:
//   warps 1-3    bring the codes from the pages to registers a tile ahead, widen them to
//                fp16 whole numbers (exact) and store K and V in the swizzled layouts the
//                MMAs read, once for both row tiles; Q likewise at the start of an item;
//   warp 0       issues S = Q K^T and O += P V for the two tiles in turn;
//   warps 4-11   softmax, a warpgroup a row tile, one row a thread; P overwrites S in
//                tensor memory.  While one tile is in its exponentials the tensor core
//                works for the other.
// Scales: with w = s + log2(V scale), P = 2^(w - max w + 14) carries a key's V scale (P <= 2^14,
// and O needs no scale of its own), and the softmax's sum takes P / (V scale).  K's scale
// multiplies the score.  A tile with a V of zeros, or with V scales outside 2^-40 .. 2^40, is `far`: there
// P / (V scale) could leave fp32's range on either side (a scale of 2^-100 and 16384 keys make 2^14 * 2^100 * 2^14).
// From the first such tile of an item on, the sum takes exponentials of the scores themselves, twice as many, with a
// reference of its own, and V of zeros weighs nothing in the products.  The newest block's
// 16-bit values are brought into fp16 by a power of two for each token (exact to 2^-24
// of the token's largest value); infinities and NaN of its V stay out of the products (0 times them would reach rows
// that do not see the token) and join their channel of the rows that see them at the end.
// Bound: the softmax (the exponentials alone, 16 a clock and SM, take 2048 clocks for two 128x128 tiles; a row's 128
// weights take its one thread about 2500).  Measured: 2048 tokens over 17200 keys, 16 heads of 64, 338 us (403 TFLOP/s);
// 1024 tokens over 8000 keys, 32/8 heads of 128, 257 us.
#pragma once

#include <type_traits>

#include "attn8.cuh"

namespace b200 {

template <int D>
struct Attn8TileCfg {
  static constexpr int BN = 128, ST = 2, ROWS = 256, THREADS = 384, CONV = 96;
  static constexpr int ATOM = D >= 64 ? 64 : D;      // channels a swizzle row
  static constexpr int ROWB = ATOM * 2;              // its bytes
  static constexpr uint32_t SWZ = ATOM == 64 ? UMMA_SW128 : UMMA_SW64;
  static constexpr int NBOX = D / ATOM;
  static constexpr int Q_BYTES = 128 * D * 2;        // one row tile
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int OFF_KV = 2 * Q_BYTES;         // stage s: K, then V
  static constexpr int OFF_KEY = OFF_KV + ST * 2 * KV_BYTES;        // [ST][3][BN]: K factor, log2 V scale, 1 / V scale
  static constexpr int OFF_QF = OFF_KEY + ST * 3 * BN * 4;          // [2][ROWS] row factors, by item parity
  static constexpr int OFF_AHEAD = OFF_QF + 2 * ROWS * 4;           // [ROWS] see attn8_weights_far
  static constexpr int OFF_BAR = OFF_AHEAD + ROWS * 4;
  static constexpr int TOTAL = OFF_BAR + 256;        // + line + alignment
  // tensor memory: S/P of the tiles at 0 and 128, O at 256 and 256 + D
  static constexpr uint32_t TM_O = 256;
};

struct Attn8Item {
  int b, head, row0;     // first of its 256 rows
  int t0, q_len, len, full, nkt;
  int rows;              // of the sequence and key head
};
__device__ __forceinline__ int attn8_limit(const Attn8Item& it, int row, int group) {
  const int i = row / group;
  return i < it.q_len ? max(0, it.len - it.q_len + i + 1) : 0;
}
// item `at` of the line (longest first within a sequence)
__device__ __forceinline__ Attn8Item attn8_item(const Attn8Params& p, const int* line, int at) {
  Attn8Item it;
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (line[mid] <= at) lo = mid; else hi = mid;
  }
  it.b = lo;
  attn8_sequence(p, lo, it.t0, it.q_len, it.len);
  const int group = p.heads / p.c.kv_heads;
  it.rows = it.q_len * group;
  const int tiles = (it.rows + 255) / 256, i = at - line[lo];
  it.head = i % p.c.kv_heads;
  it.row0 = (tiles - 1 - i / p.c.kv_heads) * 256;
  it.full = it.len & ~(p.c.page - 1);
  it.nkt = (attn8_limit(it, min(it.rows, it.row0 + 256) - 1, group) + 127) / 128;
  return it;
}

template <int D>
__device__ __forceinline__ uint32_t attn8_off(int rows, int row, int d) {  // of channel d in a [rows, D] operand tile
  using C = Attn8TileCfg<D>;
  const int box = d / C::ATOM, ch = (d % C::ATOM) >> 3;
  const uint32_t sw = C::ATOM == 64 ? (row & 7) : ((row >> 1) & 3);
  return box * rows * C::ROWB + row * C::ROWB + ((ch ^ sw) << 4) + (d & 7) * 2;
}
// 2^e as a float, and the exponent that brings the largest of 16-bit values (their magnitude bits) to [2^10, 2^11)
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ int exponent_down(unsigned top, int bf16) {
  const float v = h16_to_f(top, bf16);
  if (!(v > 0.f && v < INFINITY)) return 0;
  return max(-126, min(126, static_cast<int>(__float_as_uint(v) >> 23) - 127 - 10));
}
__device__ __forceinline__ uint4 scale8(uint4 w, int bf16, float f) {  // eight 16-bit values times f, as fp16
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = pack_half2(h16_to_f(u[i] & 0xffffu, bf16) * f, h16_to_f(u[i] >> 16, bf16) * f);
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ unsigned top2(unsigned top, uint32_t w) { return __vmaxu2(top, w & 0x7fff7fffu); }

// The newest block's 16-bit tokens as keys [first, have) of a tile, zeros past them, by the three converting warps.  Once
// an item, and a call of its own, so that the codes' registers are not spilled for it (1024 tokens over 8000 keys of 32/8
// heads of 128: 263 us inlined, 257 so).
template <int D>
__device__ __noinline__ void attn8_newest(const uint16_t* k_new, const uint16_t* v_new, int bf16, int first, int have,
                                          uint8_t* ks, uint8_t* vs, float* key, int* far, int tile, int* odd, int item) {
  const int lane = threadIdx.x & 31, cw = (threadIdx.x >> 5) - 1;
  constexpr int LK = D / 8, TK = 32 / LK;  // lanes a token, tokens a warp
  for (int t0 = first + cw * TK; t0 < 128; t0 += 3 * TK) {
    const int t = t0 + lane / LK, d = lane % LK * 8;
    const bool live = t < have;
    uint4 w = live ? __ldg(reinterpret_cast<const uint4*>(k_new + (t - first) * D + d)) : make_uint4(0, 0, 0, 0);
    unsigned top = top2(top2(top2(top2(0u, w.x), w.y), w.z), w.w);
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
    for (int x = 1; x < LK; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
    const int e = exponent_down(top, bf16);
    if (t < 128) {
      *reinterpret_cast<uint4*>(ks + attn8_off<D>(128, t, d)) = scale8(w, bf16, pow2f(-e));
      if (d == 0) key[t] = pow2f(e);
    }
  }
  for (int t = first + 4 * cw; t < 128; t += 12) {  // four tokens a warp
    constexpr int NV = D == 128 ? 2 : 1;             // 16-byte pieces (two channels of four tokens) a lane
    uint4 w[NV];
    const unsigned most = bf16 ? 0x7f7fu : 0x7bffu;  // the largest finite magnitude
    unsigned top[4] = {0, 0, 0, 0};
    unsigned strange = 0;  // bit n: token t + n has a value that is not finite
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const int piece = lane + 32 * x;
      w[x] = piece < D / 2 && t < have
                 ? __ldg(reinterpret_cast<const uint4*>(v_new + (t - first) * D + piece * 8)) : make_uint4(0, 0, 0, 0);
      const uint32_t u[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const unsigned a = u[n >> 1] >> (16 * (n & 1)) & 0x7fffu, b = u[2 + (n >> 1)] >> (16 * (n & 1)) & 0x7fffu;
        top[n] = max(top[n], max(a <= most ? a : 0u, b <= most ? b : 0u));
        if (t + n < have && max(a, b) > most) strange |= 1u << n;
      }
    }
    strange = __reduce_or_sync(0xffffffffu, strange);
    if (strange && lane == 0) *odd = item;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      top[n] = __reduce_max_sync(0xffffffffu, top[n]);
      const bool live = t + n < have;
      // (a token with nothing else than zeros, infinities and NaN: small, and no far one)
      const int e = !live ? 0 : top[n] == 0 && (strange >> n & 1) ? -40 : exponent_down(top[n], bf16);
      const float down = pow2f(-e);
      const bool zero = live && top[n] == 0 && !(strange >> n & 1);
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        const int piece = lane + 32 * x;
        const uint32_t u[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
        if (piece < D / 2) {
          float a = h16_to_f(u[n >> 1] >> (16 * (n & 1)) & 0xffffu, bf16);
          float b = h16_to_f(u[2 + (n >> 1)] >> (16 * (n & 1)) & 0xffffu, bf16);
          if (!(fabsf(a) < INFINITY)) a = 0.f;
          if (!(fabsf(b) < INFINITY)) b = 0.f;
          *reinterpret_cast<uint32_t*>(vs + attn8_off<D>(128, t + n, 2 * piece)) =
              live ? pack_half2(a * down, b * down) : 0u;
        }
      }
      if (lane == 0) {
        key[128 + t + n] = zero ? -INFINITY : static_cast<float>(e);
        key[256 + t + n] = down;
        if (zero || e < -40 || e > 40) *far = tile;
      }
    }
  }
}

// One softmax step of a row: raw scores s (in registers) become weights.  Key factors in shared memory: K scale,
// log2 of the V scale, 1 / V scale.
// A tile of full blocks that the row sees whole: the factors are alike for 16 keys, and with f > 0 a group's
// maximum is that of its raw scores, so that one multiply-add a score is all there is beside the exponential.
__device__ __forceinline__ void attn8_weights(float (&s)[128], const float* key, float qf, float& m, float& l, float& alpha) {
  float f[8], v[8], now = m;
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    f[g] = key[16 * g] * qf;
    v[g] = key[128 + 16 * g];
    float x = fmax3(s[16 * g], s[16 * g + 1], s[16 * g + 2]), y = fmax3(s[16 * g + 3], s[16 * g + 4], s[16 * g + 5]);
    x = fmax3(x, s[16 * g + 6], s[16 * g + 7]);
    y = fmax3(y, s[16 * g + 8], s[16 * g + 9]);
    x = fmax3(x, s[16 * g + 10], s[16 * g + 11]);
    y = fmax3(y, s[16 * g + 12], s[16 * g + 13]);
    now = fmaxf(now, fmaf(fmaxf(fmax3(x, s[16 * g + 14], s[16 * g + 15]), y), f[g], v[g]));
  }
  const float most = now == -INFINITY ? 0.f : now, ref = most - ATTN8_LIFT;
  alpha = fast_exp2(m - most);
  m = now;
  float sum = 0.f;
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const uint64_t f2 = f2pk(f[g], f[g]), v2 = f2pk(v[g] - ref, v[g] - ref);
    uint64_t a0 = f2pk(0.f, 0.f), a1 = a0;
#pragma unroll
    for (int c = 16 * g; c < 16 * g + 16; c += 4) {
      float x, y, z, w;
      f2upk(f2fma(f2pk(s[c], s[c + 1]), f2, v2), x, y);
      f2upk(f2fma(f2pk(s[c + 2], s[c + 3]), f2, v2), z, w);
      s[c] = fast_exp2(x); s[c + 1] = fast_exp2(y); s[c + 2] = fast_exp2(z); s[c + 3] = fast_exp2(w);
      a0 = f2add(a0, f2pk(s[c], s[c + 1]));
      a1 = f2add(a1, f2pk(s[c + 2], s[c + 3]));
    }
    float x, y;
    f2upk(f2add(a0, a1), x, y);
    sum = fmaf(x + y, key[256 + 16 * g], sum);
  }
  l = l * alpha + sum;
}
// The general form: factors key by key, keys from lim on hidden.
__device__ __forceinline__ void attn8_weights_each(float (&s)[128], const float* key, float qf, int k0, int lim, float& m, float& l,
                                                   float& alpha) {
#pragma unroll
  for (int c = 0; c < 128; c += 4) {
    const float4 f = *reinterpret_cast<const float4*>(key + c), v = *reinterpret_cast<const float4*>(key + 128 + c);
    s[c] = k0 + c < lim ? fmaf(s[c], f.x * qf, v.x) : -INFINITY;
    s[c + 1] = k0 + c + 1 < lim ? fmaf(s[c + 1], f.y * qf, v.y) : -INFINITY;
    s[c + 2] = k0 + c + 2 < lim ? fmaf(s[c + 2], f.z * qf, v.z) : -INFINITY;
    s[c + 3] = k0 + c + 3 < lim ? fmaf(s[c + 3], f.w * qf, v.w) : -INFINITY;
  }
  const float now = fmaxf(m, row_max<128>(s));
  const float most = now == -INFINITY ? 0.f : now, ref = most - ATTN8_LIFT;
  alpha = fast_exp2(m - most);
  m = now;
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < 128; c += 4) {
    const float4 v = *reinterpret_cast<const float4*>(key + 256 + c);
    s[c] = fast_exp2(s[c] - ref);
    s[c + 1] = fast_exp2(s[c + 1] - ref);
    s[c + 2] = fast_exp2(s[c + 2] - ref);
    s[c + 3] = fast_exp2(s[c + 3] - ref);
    sum = fmaf(s[c], v.x, fmaf(s[c + 1], v.y, fmaf(s[c + 2], v.z, fmaf(s[c + 3], v.w, sum))));
  }
  l = l * alpha + sum;
}

// The same where V scales may be anything (log2 of the V scale is -inf for zeros): l is relative to
// 2^(m - ATTN8_LIFT + *ahead), *ahead >= 0 (0 before the row's first such tile).  The scores are read twice from tensor
// memory at `ts`, 64 at a time, and the weights written over those that have been read.  Returns (m, l, alpha).  In a
// loop of its own after the ordinary tiles' loop: as a branch within that it took the 17200-key chunk from 338 to 360 us.
__device__ __forceinline__ float3 attn8_weights_far(uint32_t ts, const float* key, float qf, int k0, int lim, float m, float l,
                                                 float* ahead, bool first) {
  float now = m, most = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 128; h += 64) {
    float s[64];
    tmem_ld64(ts + h, s);
#pragma unroll
    for (int c = 0; c < 64; ++c) {
      const float x = k0 + h + c < lim ? s[c] * (key[h + c] * qf) : -INFINITY;
      most = fmaxf(most, x);
      now = fmaxf(now, k0 + h + c < lim ? x + key[128 + h + c] : -INFINITY);
    }
  }
  const float lwas = m - ATTN8_LIFT + (first ? 0.f : *ahead), lref = fmaxf(lwas, most), base = lref == -INFINITY ? 0.f : lref;
  if (now == -INFINITY) now = lref - 200.f;  // zeros only so far: a reference below that of any scale that can follow
  const float top = now == -INFINITY ? 0.f : now, ref = top - ATTN8_LIFT;  // (no key seen yet: every weight is 0)
  float sum = 0.f;
#pragma unroll 1
  for (int h = 0; h < 128; h += 64) {
    float s[64], p[32];
    tmem_ld64(ts + h, s);
#pragma unroll
    for (int c = 0; c < 64; ++c) {
      const float x = k0 + h + c < lim ? s[c] * (key[h + c] * qf) : -INFINITY;
      sum += fast_exp2(x - base);
      s[c] = k0 + h + c < lim ? fast_exp2(x + (key[128 + h + c] - ref)) : 0.f;
    }
#pragma unroll
    for (int c = 0; c < 32; ++c) p[c] = __uint_as_float(pack_half2(s[2 * c], s[2 * c + 1]));
    tmem_st32(ts + h / 2, p);
  }
  const float over = lref - ref;
  *ahead = fmaxf(0.f, over);
  return make_float3(now, (l * fast_exp2(lwas - base) + sum) * fast_exp2(fminf(0.f, over)), fast_exp2(m - top));
}

// Infinities and NaN among the first n tokens of the newest block's V take their channel of a finished row.  Rare, and
// a call of its own, which leaves the registers of the rest alone.
__device__ __noinline__ void attn8_strange(const uint16_t* v, int n, int dim, int bf16, uint16_t* out) {
#pragma unroll 1
  for (int d = 0; d < dim; ++d) {
    float sum = 0.f;
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      const float a = h16_to_f(__ldg(v + ((t >> 2) * dim + d) * 4 + (t & 3)), bf16);
      if (!(fabsf(a) < INFINITY)) sum += a;
    }
    if (sum != 0.f) out[d] = static_cast<uint16_t>(f_to_h16(sum + h16_to_f(out[d], bf16), bf16));  // (what is NaN already stays)
  }
}

template <int D>
__global__ void __launch_bounds__(Attn8TileCfg<D>::THREADS, 1) k_attn8_tile(const Attn8Params p) {
  using C = Attn8TileCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int tot[C::THREADS / 32];
  uint8_t* smem = smem_align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;        // the converting threads
  uint64_t* q_free = bars + 1;    // the item's last S MMA has read Q
  uint64_t* kv_full = bars + 2;   // [ST] the converting threads
  uint64_t* kv_empty = bars + 4;  // [ST] both tiles' PV have read the stage
  uint64_t* s_full = bars + 6;    // [2]
  uint64_t* p_full = bars + 8;    // [2] 128 softmax threads
  uint64_t* o_done = bars + 10;   // [2]
  uint64_t* drain = bars + 12;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* far = reinterpret_cast<int*>(tmem_slot + 2);  // [ST] of the stage's tile: its number plus 1 if it is a far one
  int* odd = far + C::ST;  // [4] of the item: its number plus 1 if the newest V is not all finite
  int* line = reinterpret_cast<int*>(smem + C::TOTAL);  // [batch + 1] first item of each sequence
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.heads / p.c.kv_heads;
  if (tid == 0) {
    mbar_init(q_full, C::CONV);
    mbar_init(q_free, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kv_full[i], C::CONV);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = far[0] = far[1] = odd[0] = odd[1] = odd[2] = odd[3] = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_sync();
  int items = 0, bad = 0;
  for (int b0 = 0; b0 < p.batch; b0 += C::THREADS) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.batch) {
      int t0, q_len, len;
      bad |= !attn8_sequence(p, b, t0, q_len, len);
      n = p.c.kv_heads * ((q_len * group + 255) / 256);
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) tot[warp] = sum;
    __syncthreads();
    int before = items;
    for (int i = 0; i < C::THREADS / 32; ++i) {
      if (i < warp) before += tot[i];
      items += tot[i];
    }
    if (b < p.batch) line[b] = before + sum - n;
    bad = __syncthreads_or(bad);
  }
  if (bad) items = 0;
  const int G = gridDim.x;

  if (warp == 0) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, false), idesc_o = make_idesc_f16(128, D, true);
      auto issue_s = [&](int x, int st) {
        const uint32_t q = smem_u32(smem + x * C::Q_BYTES), k = smem_u32(smem + C::OFF_KV + st * 2 * C::KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int box = kk * 16 / C::ATOM;
          const uint32_t in = kk * 16 % C::ATOM * 2;
          umma_f16_ss(tmem + x * 128, make_sdesc(q + box * 128 * C::ROWB + in, 16, 8 * C::ROWB, C::SWZ),
                      make_sdesc(k + box * 128 * C::ROWB + in, 16, 8 * C::ROWB, C::SWZ), idesc_s, kk > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[x]);
      };
      auto issue_pv = [&](int x, int st, bool first) {
        const uint32_t v = smem_u32(smem + C::OFF_KV + st * 2 * C::KV_BYTES + C::KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_f16_ts(tmem + C::TM_O + x * D, tmem + x * 128 + 8 * kk,
                      make_sdesc(v + kk * 16 * C::ROWB, 128 * C::ROWB, 8 * C::ROWB, C::SWZ), idesc_o, first && kk == 0 ? 0u : 1u);
        tc_commit(&o_done[x]);
      };
      int g = 0, k = 0;  // key tiles and items so far
      bool ok = true;
      for (int at = blockIdx.x; ok && at < items; at += G) {
        const int nkt = attn8_item(p, line, at).nkt;
        if (nkt == 0) continue;
        if (!mbar_wait(q_full, k & 1, abort_flag, DERR_WAIT_SLOT)) break;
        // S overwrites the P that the PV before it has read: it waits for that PV.
        auto scores = [&](int x, int n) {  // of key tile n (counted over items)
          if (n > 0 && !mbar_wait(&o_done[x], (n - 1) & 1, abort_flag, DERR_WAIT_MMA)) return false;
          tc_fence_after();
          issue_s(x, n % C::ST);
          return true;
        };
        ok = mbar_wait(&kv_full[g % C::ST], g / C::ST & 1, abort_flag, DERR_WAIT_SLOT) && scores(0, g) && scores(1, g);
        if (ok && nkt == 1) tc_commit(q_free);
        for (int j = 0; ok && j < nkt; ++j) {
          const int n = g + j;
          const bool more = j + 1 < nkt;
          for (int x = 0; ok && x < 2; ++x) {
            ok = mbar_wait(&p_full[x], n & 1, abort_flag, DERR_WAIT_SOFTMAX);
            if (!ok) break;
            tc_fence_after();
            issue_pv(x, n % C::ST, j == 0);
            if (x == 1) tc_commit(&kv_empty[n % C::ST]);
            if (more)
              ok = (x == 1 || mbar_wait(&kv_full[(n + 1) % C::ST], (n + 1) / C::ST & 1, abort_flag, DERR_WAIT_SLOT)) &&
                   scores(x, n + 1);
          }
          if (ok && j + 2 == nkt) tc_commit(q_free);
        }
        g += nkt;
        ++k;
      }
      if (*abort_flag) {
        tc_commit(drain);
        mbar_wait_drain(drain, 0);
      }
    }
  } else if (warp < 4) {
    const int i = tid - 32, P = p.c.page, psh = p.c.page_shift, cw = warp - 1;
    constexpr int NC = D / 16, ALL = 128 * NC;                 // 16-byte chunks of K, and of V: of a token, of a tile,
    constexpr int MINE = (ALL + C::CONV - 1) / C::CONV;        // of a thread
    uint4 kr[MINE], vr[MINE];
    int g = 0, k = 0;
    bool ok = true;
    for (int at = blockIdx.x; ok && at < items; at += G) {
      const Attn8Item it = attn8_item(p, line, at);
      if (it.nkt == 0) continue;
      // a tile's pages, one a lane: the table's entries a tile ahead of the codes, checked when they are used
      auto tile_entry = [&](int j) {
        const int blk = (j << (7 - psh)) + lane;
        return lane < (128 >> psh) && blk < (it.full >> psh)
                   ? __ldg(p.c.table + static_cast<size_t>(it.b) * p.c.table_width + blk) : 0;
      };
      auto tile_page = [&](int id) {
        if (id < 0 || id >= p.c.num_pages) {
          record_error(DERR_KV_RANGE);
          id = 0;
        }
        return static_cast<uint32_t>(id) * p.c.kv_heads + it.head;
      };
      // byte offset of a key's first code in the pools
      auto block = [&](uint32_t pages, int key) {
        return static_cast<uint64_t>(__shfl_sync(0xffffffffu, pages, key >> psh)) * static_cast<uint32_t>(P * D) +
               static_cast<uint32_t>((key & (P - 1)) * D);
      };
      auto fetch = [&](uint32_t pages) {
#pragma unroll
        for (int u = 0; u < MINE; ++u) {  // (past the full blocks: some page's codes, which are not used)
          const int c = min(i + C::CONV * u, ALL - 1), kt = c / NC, vt = c / (D / 4) * 4;
          const size_t ka = block(pages, kt) + c % NC * 16;
          const size_t va = block(pages, vt) + c % (D / 4) * 16;
          kr[u] = __ldg(reinterpret_cast<const uint4*>(p.c.k_pages + ka));
          vr[u] = __ldg(reinterpret_cast<const uint4*>(p.c.v_pages + va));
        }
      };
      // codes of a tile into L2, two tiles ahead of their use
      auto prefetch = [&](int j, uint32_t pages) {
        for (int c = i; c < D; c += C::CONV) {  // 128 bytes of K and of V each
          const int kt = c * 128 / D;           // the key they begin with
          const size_t at = block(pages, kt) + c * 128 % D;
          if (kt < it.full - 128 * j) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p.c.k_pages + at));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p.c.v_pages + at));
          }
        }
      };
      uint32_t pages = tile_page(tile_entry(0)), pages1 = tile_page(tile_entry(1));
      fetch(pages);
      // Q: rows in turn
      if (k > 0) ok = mbar_wait_warp(q_free, (k - 1) & 1, abort_flag, DERR_WAIT_MMA);
      if (!ok) break;
#pragma unroll 1
      for (int r = i; r < C::ROWS; r += C::CONV) {
        const int row = it.row0 + r, tok = row / group;
        const uint16_t* src = p.q + (it.t0 + tok) * p.ld_q + static_cast<size_t>(it.head * group + row % group) * D;
        const bool live = row < it.rows;
        float f = 1.f, down = 1.f;
        if (p.c.bf16 && live) {
          unsigned top = 0;
          for (int d = 0; d < D; d += 8) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + d);
            top = top2(top2(top2(top2(top, w.x), w.y), w.z), w.w);
          }
          const int e = exponent_down(max(top & 0xffffu, top >> 16), 1);
          f = pow2f(e);
          down = pow2f(-e);
        }
        for (int d = 0; d < D; d += 8) {
          uint4 w = live ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
          if (p.c.bf16) w = scale8(w, 1, down);
          *reinterpret_cast<uint4*>(smem + (r >> 7) * C::Q_BYTES + attn8_off<D>(128, r & 127, d)) = w;
        }
        reinterpret_cast<float*>(smem + C::OFF_QF)[(k & 1) * C::ROWS + r] = f * p.scale_log2;
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);
      prefetch(1, pages1);
      int next = tile_entry(2);
      for (int j = 0; j < it.nkt; ++j, ++g) {
        const int st = g % C::ST, limit = it.full - 128 * j;
        uint8_t* ks = smem + C::OFF_KV + st * 2 * C::KV_BYTES;
        uint8_t* vs = ks + C::KV_BYTES;
        float* key = reinterpret_cast<float*>(smem + C::OFF_KEY) + st * 3 * C::BN;
        float ksc[2], vsc[2];  // of keys i and i + 96
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int kt = min(i + C::CONV * n, 127);
          const size_t ph = __shfl_sync(0xffffffffu, pages, kt >> psh);
          ksc[n] = __ldg(p.c.k_scale + ph);
          vsc[n] = __ldg(p.c.v_scale + ph);
        }
        if (g >= C::ST) ok = mbar_wait_warp(&kv_empty[st], (g / C::ST - 1) & 1, abort_flag, DERR_WAIT_MMA);
        if (!ok) break;
        // the codes as whole numbers; whole tiles without a branch for every chunk
        auto widen_tile = [&](auto every) {
          constexpr bool whole = decltype(every)::value;
#pragma unroll
          for (int u = 0; u < MINE; ++u) {
            const int c = i + C::CONV * u, kt = c / NC, d = c % NC * 16;
            if (MINE * C::CONV > ALL && u == MINE - 1 && c >= ALL) break;
            if (whole || kt < limit) {
              uint4 a, b;
              widen(kr[u].x, a.x, a.y);
              widen(kr[u].y, a.z, a.w);
              widen(kr[u].z, b.x, b.y);
              widen(kr[u].w, b.z, b.w);
              *reinterpret_cast<uint4*>(ks + attn8_off<D>(128, kt, d)) = a;
              *reinterpret_cast<uint4*>(ks + attn8_off<D>(128, kt, d + 8)) = b;
            }
            const int vt = c / (D / 4) * 4, vd = c % (D / 4) * 4;
            if (whole || vt < limit) {
              const __half2 off = __half2half2(__ushort_as_half(0x6480));
#pragma unroll
              for (int t = 0; t < 4; ++t) {  // four channels of token vt + t
                const uint32_t lo = __byte_perm(vr[u].x, vr[u].y, t | (4 + t) << 8);
                const uint32_t hi = __byte_perm(vr[u].z, vr[u].w, t | (4 + t) << 8);
                const uint32_t x = __byte_perm(lo, 0x64646464u, 0x4240), y = __byte_perm(hi, 0x64646464u, 0x4240);
                const __half2 x2 = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
                const __half2 y2 = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
                *reinterpret_cast<uint2*>(vs + attn8_off<D>(128, vt + t, vd)) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&x2), *reinterpret_cast<const uint32_t*>(&y2));
              }
            }
          }
        };
        if (limit >= 128) widen_tile(std::true_type{});
        else widen_tile(std::false_type{});
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int kt = i + C::CONV * n;
          if (kt < min(limit, 128)) {
            const float v = vsc[n];
            key[kt] = ksc[n];
            key[128 + kt] = log2f(v);                // (-inf for zeros)
            key[256 + kt] = v == v ? 1.f / v : 1.f;  // (NaN comes through the logarithm, to visible keys only)
            if (v < 9.0949470e-13f || v > 1.0995116e12f) far[st] = g + 1;  // 2^-40, 2^40
          }
        }
        if (limit < 128) {  // the newest block's tokens, and zeros past them
          const int first = max(limit, 0), have = it.len - 128 * j;  // keys [first, have) of the tile
          const int nrow = p.c.rows ? __ldg(p.c.rows + it.b) : it.b;
          const bool good = nrow >= 0 && nrow < p.c.new_rows;
          if (!good && i == 0) record_error(DERR_KV_RANGE);
          const size_t base = ((static_cast<size_t>(good ? nrow : 0) * 2 + (it.full >> psh & 1)) * p.c.kv_heads + it.head) *
                              static_cast<size_t>(P * D);
          attn8_newest<D>(p.c.k_new + base, p.c.v_new + base, p.c.bf16, first, good ? have : 0, ks, vs, key, far + st, g + 1,
                          odd + (k & 3), k + 1);
        }
        fence_proxy_async_smem();
        mbar_arrive(&kv_full[st]);
        if (j + 1 < it.nkt) {
          pages = pages1;
          pages1 = tile_page(next);  // (before the codes are asked for: a wait for it could be a wait for them)
          next = tile_entry(j + 3);
          prefetch(j + 2, pages1);
          fetch(pages);
        }
      }
      ++k;
    }
  } else {
    const int x = (warp - 4) >> 2, rl = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + x * 128, to = tmem + lanes + C::TM_O + x * D;
    int g = 0, k = 0;
    bool ok = true;
    for (int at = blockIdx.x; ok && at < items; at += G) {
      const Attn8Item it = attn8_item(p, line, at);
      const int row = it.row0 + 128 * x + rl;
      const int lim = attn8_limit(it, row, group), least = attn8_limit(it, it.row0 + 128 * x, group);
      // rows past the sequence's see nothing, and hide every key (a factor that is not positive needs the general form)
      const bool ragged = it.row0 + 128 * x + 128 > it.rows || !(p.scale_log2 > 0.f);
      float m = -INFINITY, l = 0.f;
      float* const ahead = reinterpret_cast<float*>(smem + C::OFF_AHEAD) + 128 * x + rl;
      const float* const qfs = reinterpret_cast<const float*>(smem + C::OFF_QF) + (k & 1) * C::ROWS + 128 * x + rl;
      // P is in place: O takes the new reference, and the MMA warp the weights
      auto hand_over = [&](int j, float alpha) {
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tmem_ld32(to + c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= alpha;
            tmem_st32(to + c, o);
          }
        }
        tc_fence_before();
        mbar_arrive(&p_full[x]);
      };
      int j = 0;
      for (; j < it.nkt; ++j) {
        const int st = (g + j) % C::ST;
        ok = mbar_wait_warp(&kv_full[st], (g + j) / C::ST & 1, abort_flag, DERR_WAIT_SLOT);
        if (!ok || __any_sync(0xffffffffu, far[st] == g + j + 1)) break;
        ok = mbar_wait_warp(&s_full[x], (g + j) & 1, abort_flag, DERR_WAIT_MMA);
        if (!ok) break;
        tc_fence_after();
        float s[128];
        tmem_ld128(ts, s);
        const float* key = reinterpret_cast<const float*>(smem + C::OFF_KEY) + st * 3 * C::BN;
        const float qf = *qfs;
        float alpha;
        if (ragged || 128 * j + 128 > min(least, it.full)) attn8_weights_each(s, key, qf, 128 * j, lim, m, l, alpha);
        else attn8_weights(s, key, qf, m, l, alpha);
        uint32_t pk[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) pk[c] = pack_half2(s[2 * c], s[2 * c + 1]);
        tmem_st64(ts, pk);
        hand_over(j, alpha);
      }
      const bool wide = ok && j < it.nkt;
#pragma unroll 1
      for (bool first = true; ok && j < it.nkt; ++j, first = false) {  // from the item's first far tile on
        const int st = (g + j) % C::ST;
        ok = mbar_wait_warp(&kv_full[st], (g + j) / C::ST & 1, abort_flag, DERR_WAIT_SLOT) &&
             mbar_wait_warp(&s_full[x], (g + j) & 1, abort_flag, DERR_WAIT_MMA);
        if (!ok) break;
        tc_fence_after();
        const float3 now = attn8_weights_far(ts, reinterpret_cast<const float*>(smem + C::OFF_KEY) + st * 3 * C::BN, *qfs,
                                             128 * j, lim, m, l, ahead, first);
        m = now.x, l = now.y;
        hand_over(j, now.z);
      }
      if (!ok) break;
      // (the word is another item's three on at the earliest: this warp has then handed over a tile of the next)
      const bool strange = it.nkt > 0 && odd[k & 3] == k + 1;
      if (it.nkt > 0) {
        g += it.nkt;
        ++k;
        ok = mbar_wait_warp(&o_done[x], (g - 1) & 1, abort_flag, DERR_WAIT_MMA);
        if (!ok || __any_sync(0xffffffffu, *abort_flag != 0)) break;
        tc_fence_after();
      }
      // a row that sees no key is 0; 2^-ahead in two halves, in fp32's range whatever the scales were
      const float down = wide ? fast_exp2(-0.5f * *ahead) : 1.f, inv = lim > 0 ? 1.f / l * down : 0.f;
      const int tok = row / group;
      uint16_t* dst = p.out + (it.t0 + tok) * p.ld_out + static_cast<size_t>(it.head * group + row % group) * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (it.nkt > 0) {
          tmem_ld32(to + c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (row < it.rows) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
              w[n] = lim > 0 ? f_to_h16(o[e + 2 * n] * inv * down, p.c.bf16) | f_to_h16(o[e + 2 * n + 1] * inv * down, p.c.bf16) << 16 : 0u;
            *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (strange && row < it.rows) {
        const int nrow = p.c.rows ? __ldg(p.c.rows + it.b) : it.b;  // (in range: the token was read from there)
        attn8_strange(p.c.v_new + ((static_cast<size_t>(nrow) * 2 + (it.full / p.c.page & 1)) * p.c.kv_heads + it.head) *
                                      static_cast<size_t>(p.c.page * D), lim - it.full, D, p.c.bf16, dst);
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace b200
