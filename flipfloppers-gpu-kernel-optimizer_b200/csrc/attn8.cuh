// Attention of new tokens over the 8-bit paged cache of kv8.cuh:
//   out[r] = sum_j softmax_j(q[r] . k_j * scale) v_j,   k, v = (code - 128) * block scale
// The rows of one key head are its group's query heads times the sequence's new
// tokens; a row of the token at position p sees the keys 0..p.
//
// Decoding reads the cache once and computes little: the bound is HBM.  Every
// WARP streams its own range of 32-token chunks, with no barrier anywhere:
//   - all (sequence, key head, row tile, chunk) work is one line, cut into equal
//     pieces, one a warp, so ragged lengths load every SM alike; a piece that
//     holds only part of a row tile leaves (max, sum, accumulator) to its CTA, the CTA's
//     sums go through the workspace to k_attn8_join, all added in a fixed order; few
//     tiles of short tables are a CTA's each and need no second kernel;
//   - a chunk's K and V are 32 D contiguous bytes each: bulk copies bring them to the
//     warp's own ring of shared memory, Attn8Cfg::STAGES chunks ahead (cp.async of 16
//     bytes a lane asked L2 for every 32-byte sector twice and stopped at 3.2 TB/s;
//     loads to registers kept too little in flight, 3.9 TB/s);
//   - the products run as S^T = K Q^T and O^T = V^T P^T on m16n8k16 tensor-core
//     steps: tokens (channels of V) fill the 16 rows, query rows the 8 columns, so
//     up to 8 rows cost one column tile (NT = 1) and up to 16 two (NT = 2), and the
//     codes are widened to fp16 (exactly: 1024 + c, less 1152) once for all rows;
//   - scores take the block's K scale, and each block's V product its V scale, in
//     fp32: the codes enter the products as whole numbers.
// Measured: 64 sequences of 1 to 8191 tokens, 32/8 heads of 128, 98 us (5.3 TB/s); one of
// 131000 tokens 58 us (4.6 TB/s, 41 to 45 us of it streaming).
// Contraction order is free, so a lane's 16 bytes of K are the fragment elements of
// four steps; key tau(m) = 4 (m/2) + m%2 (+2 for m >= 8) sits in row m, which after
// the 8x8 transposition of P (movmatrix) meets the word of V with the same four keys.
#pragma once

#include "kv8.cuh"

namespace b200 {

constexpr int ATTN8_CHUNK = 32;   // tokens
// Weights meet V in fp16 (in the newest block of a bf16 cache as two bf16 parts), scores, maxima and sums are fp32: a
// weight is off by at most 2^-11 of itself, so an output by less than one rounding of an fp16 result, where weights of
// more bits would take a second product (twice the tensor steps of PV).  They are kept times 2^14 (at most 16384), so
// that fp16 has its eleven bits for those down to 2^-28 of the largest.
constexpr float ATTN8_LIFT = 14.f;
constexpr int ATTN8_MAX_BATCH = 2048;

struct Attn8Params {
  Kv8Cache c;
  const uint16_t* q;     // [tokens, heads, D], row stride ld_q; may be `out`, so it is not read with __ldg
  uint16_t* out;         // [tokens, heads, D], row stride ld_out
  long long ld_q, ld_out;
  const int* cu;         // [batch + 1] first row of each sequence's new tokens
  const int* lens;       // [batch] cached tokens, the new ones included
  int tokens, batch, heads;
  float scale_log2;      // scale * log2(e)
  int warps;             // warps of the launch
  int* plan;             // [batch + 1] first unit of each sequence on the line (written by CTA 0)
  float* part;           // [warps][2][rows][D] accumulators, then [warps][2][rows][2] (max, sum)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same from zero
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// a bf16 pair with its infinities and NaN taken as 0
__device__ __forceinline__ uint32_t finite_only(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
  return x;
}
// Four codes -> two fp16 pairs of c - 128, exact: 0x6400 | c is 1024 + c.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

template <int D, int NT>
struct Attn8Cfg {
  static constexpr int ROWS = 8 * NT;
  // Warps of the SM's one CTA, and chunks in each warp's ring of shared memory: about 200 KB in flight an SM
  static constexpr int WARPS = D == 128 ? (NT == 1 ? 12 : 8) : NT == 1 ? 16 : 12;
  static constexpr int STAGES = D == 128 ? (NT == 1 ? 2 : 3) : D == 64 ? (NT == 1 ? 3 : 4) : 6;
  static constexpr int CB = D >= 64 ? 16 : 8;        // bytes a lane reads of a K row at once
  static constexpr int NCH = D / (4 * CB);           // such reads a row
  static constexpr int K_BYTES = ATTN8_CHUNK * D, STAGE = 2 * K_BYTES;  // K, then V of one chunk
  static constexpr int RING = STAGES * STAGE;        // one warp's
  static constexpr int BAR_OFF = WARPS * RING, TOTAL = BAR_OFF + WARPS * STAGES * 8 + 16;
};

// What one warp knows of the row tile it works on.
struct Attn8Seg {
  int b, head, rt;       // sequence, key head, row tile
  int len, full_tokens;  // cached tokens; those in full blocks
  int q_len, t0;
};

// chunks of a sequence: 32 tokens each of the full blocks, then 16 each of the newest block (as many bytes)
__device__ __forceinline__ int attn8_full_chunks(int full_tokens) { return (full_tokens + ATTN8_CHUNK - 1) / ATTN8_CHUNK; }
__device__ __forceinline__ int attn8_chunks(int len, int page) {
  const int full = len / page * page;
  return attn8_full_chunks(full) + (len - full + 15) / 16;
}
// The line's units: a chunk of full blocks is one, a chunk of the newest block two and the start of a row tile two
// (measured: its rows, pages and first copies take as long as two chunks, 4 us).
constexpr int ATTN8_START = 2, ATTN8_NEWEST = 2;
__device__ __forceinline__ int attn8_units(int len, int page) {
  const int full = len / page * page;
  return ATTN8_START + attn8_full_chunks(full) + (len - full + 15) / 16 * ATTN8_NEWEST;
}
// first chunk that begins at or after unit u of a row tile with `fullc` chunks of full blocks
__device__ __forceinline__ int attn8_chunk_at(int u, int fullc) {
  u -= ATTN8_START;
  return u <= 0 ? 0 : u <= fullc ? u : fullc + (u - fullc + ATTN8_NEWEST - 1) / ATTN8_NEWEST;
}

// SMALL: pages of 16 tokens, so that a chunk has two.
template <int D, int NT, bool SMALL>
struct Attn8Warp {
  using C = Attn8Cfg<D, NT>;
  const Attn8Params& p;
  uint8_t* const ring;
  uint64_t* const bars;      // one a stage
  volatile int* const abort_flag;
  int issued, taken;         // chunks copied and consumed so far (stage and phase follow)
  bool ok;                   // false: a copy never arrived
  const int lane, g, t;
  const uint32_t lane_k, lane_v;  // this lane's byte offsets in a half chunk of K and of V
  Attn8Seg s;
  uint32_t qb[D / 16][NT][2];
  float qf[NT][2];       // score factor of this lane's columns: scale * log2(e) * row factor
  int lim[NT][2];        // keys that this lane's columns see
  int lo_lim, hi_lim;    // least and most of the tile's rows
  float m[NT][2], l[NT][2];
  float acc[D / 16][NT][4];
  // the copies' window: block of lane 0; page ids of 32 blocks from there, and of the next 32
  int window, page_now, page_next;
  size_t newest_at;  // of the newest block's values of this head
  // the products' window, at most one behind: scales of its 32 blocks, and those of the copies' window
  int swindow;
  float ks_now, vs_now, ks_next, vs_next;

  __device__ Attn8Warp(const Attn8Params& pp, uint8_t* smem, int w)
      : p(pp), ring(smem + w * C::RING), bars(reinterpret_cast<uint64_t*>(smem + C::BAR_OFF) + w * C::STAGES),
        abort_flag(reinterpret_cast<volatile int*>(smem + C::BAR_OFF + C::WARPS * C::STAGES * 8)), issued(0), taken(0),
        ok(true), lane(threadIdx.x & 31), g(lane >> 2), t(lane & 3),
        lane_k((4 * (g >> 1) + (g & 1)) * D + t * C::CB), lane_v(t * 4 * D + 16 * g) {}

  __device__ __forceinline__ const uint16_t* row_ptr(int r, bool& ok) const {
    const int group = p.heads / p.c.kv_heads, i = r / group;
    ok = i < s.q_len;
    return p.q + (s.t0 + (ok ? i : 0)) * p.ld_q + static_cast<size_t>(s.head * group + r % group) * D;
  }
  // first of the four channels that this lane contracts in step j
  __device__ __forceinline__ int chan(int j) const {
    constexpr int WPC = C::CB / 4;
    return 4 * C::CB * (j / WPC) + C::CB * t + 4 * (j % WPC);
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }
#pragma unroll
    for (int a = 0; a < D / 16; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][n][e] = 0.f;
  }

  __device__ __forceinline__ void load_rows() {
    clear();
    const int group = p.heads / p.c.kv_heads;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      bool ok;
      const uint16_t* src = row_ptr(s.rt * C::ROWS + 8 * n + g, ok);
      uint2 w[D / 16];
#pragma unroll
      for (int j = 0; j < D / 16; ++j) w[j] = ok ? *reinterpret_cast<const uint2*>(src + chan(j)) : make_uint2(0, 0);
      float f = 1.f;
      if (p.c.bf16) {
        // a power of two brings the row's largest value to [2^10, 2^11): values down to 2^-27 of it stay exact in
        // fp16, smaller ones are off by at most 2^-35 of it
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) top = __vmaxu2(top, __vmaxu2(w[j].x & 0x7fff7fffu, w[j].y & 0x7fff7fffu));
        top = max(top & 0xffffu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = static_cast<int>(top >> 7) - 127 - 10;  // of 2^e = row factor
        if (top < 0x0080u || top >= 0x7f80u) e = 0;     // zero, subnormal, infinity, NaN: as they are
        e = max(-126, min(126, e));
        const float down = __int_as_float((127 - e) << 23);
        f = __int_as_float((127 + e) << 23);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          w[j].x = pack_half2(__uint_as_float(w[j].x << 16) * down, __uint_as_float(w[j].x & 0xffff0000u) * down);
          w[j].y = pack_half2(__uint_as_float(w[j].y << 16) * down, __uint_as_float(w[j].y & 0xffff0000u) * down);
        }
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        qb[j][n][0] = w[j].x;
        qb[j][n][1] = w[j].y;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qf[n][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4) * p.scale_log2;
        const int i = (s.rt * C::ROWS + 8 * n + 2 * t + e) / group;
        lim[n][e] = i < s.q_len ? max(0, s.len - s.q_len + i + 1) : 0;
      }
    }
    const int i0 = s.rt * C::ROWS / group, i1 = min(s.q_len - 1, (s.rt * C::ROWS + C::ROWS - 1) / group);
    lo_lim = max(0, s.len - s.q_len + i0 + 1);
    hi_lim = max(0, s.len - s.q_len + i1 + 1);
  }

  __device__ __forceinline__ int fetch_page(int blk) {
    const int last = s.full_tokens / p.c.page - 1;
    if (last < 0) return 0;
    int id = __ldg(p.c.table + static_cast<size_t>(s.b) * p.c.table_width + min(blk, last));
    if (id < 0 || id >= p.c.num_pages) {
      record_error(DERR_KV_RANGE);
      id = 0;
    }
    return id;
  }
  __device__ __forceinline__ void fetch_scales() {
    const size_t ph = static_cast<size_t>(page_now) * p.c.kv_heads + s.head;
    ks_next = __ldg(p.c.k_scale + ph);
    vs_next = __ldg(p.c.v_scale + ph);
  }
  __device__ __forceinline__ void open_window(int blk) {
    window = swindow = blk;
    page_now = fetch_page(blk + lane);
    page_next = fetch_page(blk + 32 + lane);
    fetch_scales();
    ks_now = ks_next;
    vs_now = vs_next;
  }
  // byte offset of a block of this head in the pools
  __device__ __forceinline__ size_t block_at(int blk) {
    if (blk >= window + 32) {
      window += 32;
      page_now = page_next;
      page_next = fetch_page(window + 32 + lane);
      fetch_scales();
    }
    const size_t page = __shfl_sync(0xffffffffu, page_now, blk - window);
    return (page * p.c.kv_heads + s.head) * static_cast<uint32_t>(p.c.page * D);
  }
  __device__ __forceinline__ void block_scales(int blk, float& ks, float& vs) {
    if (blk >= swindow + 32) {
      swindow += 32;
      ks_now = ks_next;
      vs_now = vs_next;
    }
    ks = __shfl_sync(0xffffffffu, ks_now, blk - swindow);
    vs = __shfl_sync(0xffffffffu, vs_now, blk - swindow);
  }

  // start the copy of chunk c to the next stage; chunks come in order
  __device__ __forceinline__ void issue(int c, int fullc) {
    uint8_t* dst = ring + issued % C::STAGES * C::STAGE;
    uint64_t* bar = bars + issued % C::STAGES;
    ++issued;
    if (c >= fullc) {
      if (lane == 0) {
        const size_t at = newest_at + static_cast<uint32_t>((c - fullc) * 16 * D);
        mbar_arrive_expect_tx(bar, C::STAGE);
        bulk_load(dst, p.c.k_new + at, C::K_BYTES, bar);
        bulk_load(dst + C::K_BYTES, p.c.v_new + at, C::K_BYTES, bar);
      }
      return;
    }
    if constexpr (SMALL) {
      // a half past the full blocks keeps what the stage held: any byte is a code, and its keys are masked
      const bool both = c * ATTN8_CHUNK + 16 < s.full_tokens;
      const size_t a0 = block_at(2 * c), a1 = block_at(both ? 2 * c + 1 : 2 * c);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, both ? 64 * D : 32 * D);
        bulk_load(dst, p.c.k_pages + a0, 16 * D, bar);
        bulk_load(dst + C::K_BYTES, p.c.v_pages + a0, 16 * D, bar);
        if (both) {
          bulk_load(dst + 16 * D, p.c.k_pages + a1, 16 * D, bar);
          bulk_load(dst + C::K_BYTES + 16 * D, p.c.v_pages + a1, 16 * D, bar);
        }
      }
    } else {
      const int tok = c * ATTN8_CHUNK;
      const size_t at = block_at(tok / p.c.page) + static_cast<uint32_t>(tok % p.c.page * D);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, C::STAGE);
        bulk_load(dst, p.c.k_pages + at, C::K_BYTES, bar);
        bulk_load(dst + C::K_BYTES, p.c.v_pages + at, C::K_BYTES, bar);
      }
    }
  }

  // scores of one chunk (log2 units, keys outside the rows' view at -inf) -> P (fp32) and the running maximum
  template <int H>
  __device__ __forceinline__ void softmax_step(float (&sc)[H][NT][4], int tok0, bool masked) {
    if (masked) {
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = tok0 + 16 * h + 4 * (g >> 1) + (g & 1) + (e >> 1) * 2;
            if (key >= lim[n][e & 1]) sc[h][n][e] = -INFINITY;
          }
    }
    float alpha[NT][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(sc[0][n][e], sc[0][n][e + 2]);
        if constexpr (H == 2) x = fmaxf(x, fmaxf(sc[1][n][e], sc[1][n][e + 2]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float now = fmaxf(m[n][e], x);
        const float top = now == -INFINITY ? 0.f : now;  // no key seen yet: every weight is 0
        const float ref = top - ATTN8_LIFT;
        alpha[n][e] = fast_exp2(m[n][e] - top);
        moved |= now != m[n][e];
        m[n][e] = now;
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& v = sc[h][n][e + 2 * r];
            v = fast_exp2(v - ref);
            sum += v;
          }
        l[n][e] = l[n][e] * alpha[n][e] + sum;
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int a = 0; a < D / 16; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[a][n][e] *= alpha[n][e & 1];
    }
  }

  __device__ __forceinline__ void chunk_scores(const uint8_t* src, const float (&ks)[2], float (&sc)[2][NT][4]) {
    uint32_t kw[2][2][D / 16];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int x = 0; x < C::NCH; ++x) {
          const uint8_t* at = src + 16 * h * D + lane_k + 2 * r * D + 4 * x * C::CB;
          if constexpr (C::CB == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            kw[h][r][4 * x] = v.x; kw[h][r][4 * x + 1] = v.y; kw[h][r][4 * x + 2] = v.z; kw[h][r][4 * x + 3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            kw[h][r][2 * x] = v.x; kw[h][r][2 * x + 1] = v.y;
          }
        }
    // each step's product waits for the one before it in the same sum: four sums side by side (two halves of the
    // chunk, even and odd steps)
    float odd[2][NT][4];
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t a[4];
        widen(kw[h][0][j], a[0], a[2]);
        widen(kw[h][1][j], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float (&to)[4] = j & 1 ? odd[h][n] : sc[h][n];
          if (j < 2) mma_f16_first(to, a, qb[j][n][0], qb[j][n][1]);
          else mma_f16(to, a, qb[j][n][0], qb[j][n][1]);
        }
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][n][e] = (sc[h][n][e] + odd[h][n][e]) * (ks[SMALL ? h : 0] * qf[n][e & 1]);
  }

  __device__ __forceinline__ void chunk_values(const uint8_t* src, const float (&vs)[2], int c, const float (&pr)[2][NT][4], bool masked) {
    uint32_t b[2][NT][2];
    float f[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        b[h][n][0] = transpose8x8(pack_half2(pr[h][n][0], pr[h][n][1]));
        b[h][n][1] = transpose8x8(pack_half2(pr[h][n][2], pr[h][n][3]));
#pragma unroll
        for (int e = 0; e < 2; ++e)  // a block that a row does not see adds nothing, whatever its scale
          f[h][n][e] = masked && lim[n][e] <= c * ATTN8_CHUNK + 16 * h ? 0.f : vs[SMALL ? h : 0];
      }
    }
    constexpr int XG = D == 128 ? (NT == 1 ? 2 : 1) : D == 64 && NT == 2 ? 1 : D / 32;  // 32-channel groups at a time: as many sums side by side
#pragma unroll
    for (int x0 = 0; x0 < D / 32; x0 += XG) {
      float o[2 * XG][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int x = 0; x < XG; ++x) {
          const uint4 w = *reinterpret_cast<const uint4*>(src + C::K_BYTES + 16 * h * D + lane_v + 128 * (x0 + x));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t a[4];
            widen(y ? w.z : w.x, a[0], a[2]);
            widen(y ? w.w : w.y, a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (h == 0 || SMALL) mma_f16_first(o[2 * x + y][n], a, b[h][n][0], b[h][n][1]);
              else mma_f16(o[2 * x + y][n], a, b[h][n][0], b[h][n][1]);
            }
          }
        }
        if (h == 1 || SMALL) {
#pragma unroll
          for (int x = 0; x < 2 * XG; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[2 * x0 + x][n][e] = fmaf(o[x][n][e], f[SMALL ? h : 0][n][e & 1], acc[2 * x0 + x][n][e]);
        }
      }
    }
  }

  // 16 tokens of the newest block, 16-bit values
  template <bool BF16>
  __device__ __forceinline__ void newest_chunk(const uint8_t* src, int tok0) {
    float sc[1][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[0][n][e] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; j += 2) {
      uint4 w[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        w[r] = *reinterpret_cast<const uint4*>(src + ((4 * (g >> 1) + (g & 1) + 2 * r) * D + chan(j)) * 2);
      const uint32_t a0[4] = {w[0].x, w[1].x, w[0].y, w[1].y};
      const uint32_t a1[4] = {w[0].z, w[1].z, w[0].w, w[1].w};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (BF16) {  // rows in their own type: read again
          bool live;
          const uint16_t* from = row_ptr(s.rt * C::ROWS + 8 * n + g, live) + chan(j);
          uint2 q0 = *reinterpret_cast<const uint2*>(from), q1 = *reinterpret_cast<const uint2*>(from + 4);
          if (!live) q0 = q1 = make_uint2(0, 0);
          mma_bf16(sc[0][n], a0, q0.x, q0.y);
          mma_bf16(sc[0][n], a1, q1.x, q1.y);
        } else {
          mma_f16(sc[0][n], a0, qb[j][n][0], qb[j][n][1]);
          mma_f16(sc[0][n], a1, qb[j + 1][n][0], qb[j + 1][n][1]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[0][n][e] *= BF16 ? p.scale_log2 : qf[n][e & 1];
    const bool masked = tok0 + 16 > lo_lim;
    softmax_step(sc, tok0, masked);
    uint32_t b[NT][2], bl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float x = sc[0][n][2 * r], y = sc[0][n][2 * r + 1];
        if constexpr (BF16) {
          // bf16 weights keep 8 bits: a second product adds what the first leaves out
          const uint32_t xh = f_to_h16(x, 1), yh = f_to_h16(y, 1);
          const uint32_t xl = f_to_h16(x - h16_to_f(xh, 1), 1), yl = f_to_h16(y - h16_to_f(yh, 1), 1);
          b[n][r] = transpose8x8(xh | yh << 16);
          bl[n][r] = transpose8x8(xl | yl << 16);
        } else {
          b[n][r] = transpose8x8(pack_half2(x, y));
        }
      }
    // of this lane's four tokens, the first `have`
    auto keep = [&](uint4& v, int have) {
      const uint32_t k0 = have >= 2 ? 0xffffffffu : have == 1 ? 0xffffu : 0u;
      const uint32_t k1 = have >= 4 ? 0xffffffffu : have == 3 ? 0xffffu : 0u;
      v.x &= k0; v.z &= k0; v.y &= k1; v.w &= k1;
    };
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      uint4 w[2];
      bool odd = false;  // an infinity or NaN among the values
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        w[y] = *reinterpret_cast<const uint4*>(src + C::K_BYTES + (t * D + 32 * x + 4 * g) * 8 + 16 * y);
        keep(w[y], s.len - (tok0 + 4 * t));  // what lies past the end is never summed
        constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
        const uint32_t top = __vmaxu2(__vmaxu2(w[y].x & 0x7fff7fffu, w[y].y & 0x7fff7fffu),
                                      __vmaxu2(w[y].z & 0x7fff7fffu, w[y].w & 0x7fff7fffu));
        odd |= (top & 0xffffu) >= inf || (top >> 16) >= inf;
      }
      // 0 * infinity must not reach rows that do not see the value: rows are then taken apart by what they see
      const bool strange = __any_sync(0xffffffffu, odd), apart = masked && strange;
      for (int seen = apart ? max(lo_lim, tok0 + 1) : hi_lim; seen <= hi_lim; ++seen) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint4 v = w[y];
          if (apart) keep(v, seen - (tok0 + 4 * t));
          const uint32_t a[4] = {v.x, v.z, v.y, v.w};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float o[4];
            if constexpr (BF16) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] = 0.f;
              mma_bf16(o, a, b[n][0], b[n][1]);
              uint32_t al[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) al[e] = strange ? finite_only(a[e]) : a[e];
              mma_bf16(o, al, bl[n][0], bl[n][1]);
            } else {
              mma_f16_first(o, a, b[n][0], b[n][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!apart || lim[n][e & 1] == seen) acc[2 * x + y][n][e] += o[e];
          }
        }
      }
    }
  }

  // chunks [c0, c1) of the segment
  __device__ __forceinline__ void stream(int c0, int c1) {
    const int fullc = attn8_full_chunks(s.full_tokens);
    // what no row sees is not read
    const int seen = hi_lim <= s.full_tokens ? attn8_full_chunks(hi_lim) : fullc + (hi_lim - s.full_tokens + 15) / 16;
    const int e1 = min(c1, seen);
    if (c0 >= e1) return;
    newest_at = 0;
    if (e1 > fullc) {
      const int row = p.c.rows ? __ldg(p.c.rows + s.b) : s.b;
      if (row < 0 || row >= p.c.new_rows) {
        record_error(DERR_KV_RANGE);
        return;
      }
      newest_at = ((static_cast<size_t>(row) * 2 + (s.full_tokens / p.c.page & 1)) * p.c.kv_heads + s.head) *
                  static_cast<uint32_t>(p.c.page * D);
    }
    open_window(c0 * ATTN8_CHUNK / p.c.page);
    int next = c0;
    while (next < e1 && next < c0 + C::STAGES - 1) issue(next++, fullc);
    for (int c = c0; c < e1; ++c) {
      __syncwarp();  // every lane has read the stage that is filled again
      if (next < e1) issue(next++, fullc);
      const int tok0 = c * ATTN8_CHUNK, stage = taken % C::STAGES;
      float ks[2], vs[2];
      if (c < fullc) {
        if constexpr (SMALL) {
          const bool both = tok0 + 16 < s.full_tokens;
          block_scales(2 * c, ks[0], vs[0]);
          block_scales(both ? 2 * c + 1 : 2 * c, ks[1], vs[1]);
        } else {
          block_scales(tok0 / p.c.page, ks[0], vs[0]);
        }
      }
      if (!mbar_wait_warp(bars + stage, taken / C::STAGES & 1, abort_flag, DERR_WAIT_TMA)) {
        // what is in flight must land before the shared memory is anyone else's
        for (int i = taken; i < issued; ++i) mbar_wait_drain(bars + i % C::STAGES, i / C::STAGES & 1);
        ok = false;
        return;
      }
      ++taken;
      const uint8_t* src = ring + stage * C::STAGE;
      if (c < fullc) {
        const bool masked = min(tok0 + ATTN8_CHUNK, s.full_tokens) > lo_lim;
        float sc[2][NT][4];
        chunk_scores(src, ks, sc);
        if (SMALL && tok0 + ATTN8_CHUNK > s.full_tokens) {
          // the chunk's other half belongs to the newest block
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[1][n][e] = -INFINITY;
        }
        softmax_step(sc, tok0, masked);
        chunk_values(src, vs, c, sc, masked);
      } else if (p.c.bf16) {
        newest_chunk<true>(src, s.full_tokens + (c - fullc) * 16);
      } else {
        newest_chunk<false>(src, s.full_tokens + (c - fullc) * 16);
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ void join_lanes() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
  }
  // the lane's column e of column tile n: channels 32 x + 4 g .. + 3 are acc[2x][.][e, e+2], acc[2x+1][.][e, e+2]
  __device__ __forceinline__ void finish() {
    join_lanes();
    const int group = p.heads / p.c.kv_heads;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = s.rt * C::ROWS + 8 * n + 2 * t + e, i = r / group;
        if (i >= s.q_len) continue;
        const float inv = lim[n][e] > 0 ? 1.f / l[n][e] : 0.f;  // a row that sees no key is 0
        uint16_t* dst = p.out + (s.t0 + i) * p.ld_out + static_cast<size_t>(s.head * group + r % group) * D + 4 * g;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          const float v[4] = {acc[2 * x][n][e] * inv, acc[2 * x][n][e + 2] * inv, acc[2 * x + 1][n][e] * inv,
                              acc[2 * x + 1][n][e + 2] * inv};
          uint2 w;
          w.x = f_to_h16(v[0], p.c.bf16) | f_to_h16(v[1], p.c.bf16) << 16;
          w.y = f_to_h16(v[2], p.c.bf16) | f_to_h16(v[3], p.c.bf16) << 16;
          *reinterpret_cast<uint2*>(dst + 32 * x) = w;
        }
      }
  }
  // (max, sum, accumulator) to [rows][D] at `acc_to` and [rows][2] at `ml_to`
  __device__ __forceinline__ void leave_part(float* acc_to, float* ml_to) {
    join_lanes();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * t + e;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          *reinterpret_cast<float4*>(acc_to + r * D + 32 * x + 4 * g) =
              make_float4(acc[2 * x][n][e], acc[2 * x][n][e + 2], acc[2 * x + 1][n][e], acc[2 * x + 1][n][e + 2]);
        if (g == 0) *reinterpret_cast<float2*>(ml_to + 2 * r) = make_float2(m[n][e], l[n][e]);
      }
  }
};

// sequence b's new tokens; none where they or its length are outside the buffers.  false: cu decreases, so that
// sequences could share rows and the line of work outgrow 32 bits: then nothing is computed at all.
__device__ __forceinline__ bool attn8_sequence(const Attn8Params& p, int b, int& t0, int& q_len, int& len) {
  t0 = __ldg(p.cu + b);
  const int end = __ldg(p.cu + b + 1);
  len = __ldg(p.lens + b);
  q_len = 0;
  if (t0 < 0 || end < t0 || end > p.tokens || len < 0 || len > static_cast<long long>(p.c.table_width) * p.c.page) {
    record_error(DERR_KV_RANGE);
    const bool rises = end >= t0;
    t0 = len = 0;
    return rises;
  }
  q_len = end - t0;
  return true;
}

// OWN: a row tile a CTA, cut among its warps; else the line of units, cut among all warps.
template <int D, int NT, bool SMALL, bool OWN>
__global__ void __launch_bounds__(32 * Attn8Cfg<D, NT>::WARPS, 1) k_attn8(const Attn8Params p) {
  using C = Attn8Cfg<D, NT>;
  extern __shared__ __align__(128) uint8_t smem_attn8[];
  __shared__ int tot[C::WARPS], held[C::WARPS], held_slot[C::WARPS];
  int* line = reinterpret_cast<int*>(smem_attn8 + C::TOTAL);  // [batch + 1] first work unit of each sequence
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  if (tid < C::WARPS * C::STAGES) mbar_init(reinterpret_cast<uint64_t*>(smem_attn8 + C::BAR_OFF) + tid, 1);
  if (tid == 0) *reinterpret_cast<volatile int*>(smem_attn8 + C::BAR_OFF + C::WARPS * C::STAGES * 8) = 0;
  fence_mbar_init();
  griddep_sync();
  const int group = p.heads / p.c.kv_heads;
  int base = 0, bad = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32 * C::WARPS) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.batch) {
      int t0, q_len, len;
      bad |= !attn8_sequence(p, b, t0, q_len, len);
      n = p.c.kv_heads * ((q_len * group + C::ROWS - 1) / C::ROWS) * (OWN ? 1 : attn8_units(len, p.c.page));
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) tot[wid] = sum;
    __syncthreads();
    int before = base;
    for (int i = 0; i < C::WARPS; ++i) {
      if (i < wid) before += tot[i];
      base += tot[i];
    }
    if (b < p.batch) line[b] = before + sum - n;
    bad = __syncthreads_or(bad);
  }
  if (bad) base = 0;
  if (tid == 0) line[p.batch] = base;
  __syncthreads();
  if (!OWN && blockIdx.x == 0)
    for (int i = tid; i <= p.batch; i += 32 * C::WARPS) p.plan[i] = line[i];

  Attn8Warp<D, NT, SMALL> w(p, smem_attn8, wid);
  const int warp = blockIdx.x * C::WARPS + wid;
  // place `at` of the line: its sequence and row tile; the units of the tile, and the place within them
  auto locate = [&](int at, int& units, int& u0) {
    const int b = warp_search(p.batch, at, [&](int i) { return line[i]; });
    int t0, q_len, len;
    attn8_sequence(p, b, t0, q_len, len);
    const int tiles = (q_len * group + C::ROWS - 1) / C::ROWS;
    units = OWN ? 1 : attn8_units(len, p.c.page);
    const int item = (at - line[b]) / units;
    u0 = (at - line[b]) % units;
    w.s.b = b;
    w.s.head = item / tiles;
    w.s.rt = item % tiles;
    w.s.len = len;
    w.s.full_tokens = len / p.c.page * p.c.page;
    w.s.q_len = q_len;
    w.s.t0 = t0;
  };
  static_assert(C::RING >= (C::ROWS * D + 2 * C::ROWS) * 4, "a part fits a warp's ring");
  float* const mine = reinterpret_cast<float*>(smem_attn8 + wid * C::RING);
  auto part = [&](int x) { return reinterpret_cast<const float*>(smem_attn8 + x * C::RING); };
  // row r, channels d .. d + 3 of the parts of warps [w0, w1) added up: (max, sum) comes back, the accumulators in o
  auto add_parts = [&](int w0, int w1, int r, int d, float4& o) {
    float top = -INFINITY;
    for (int x = w0; x < w1; ++x) top = fmaxf(top, part(x)[C::ROWS * D + 2 * r]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = w0; x < w1; ++x) {
      const float f = fast_exp2(part(x)[C::ROWS * D + 2 * r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(part(x) + r * D + d);
      sum = fmaf(part(x)[C::ROWS * D + 2 * r + 1], f, sum);
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    return make_float2(top, sum);
  };

  if constexpr (OWN) {
    for (int at = blockIdx.x; at < base; at += gridDim.x) {  // (the barriers are reached whatever a wait did)
      int units, u0;
      locate(at, units, u0);
      const int chunks = attn8_chunks(w.s.len, p.c.page), per = (chunks + C::WARPS - 1) / C::WARPS;
      if (w.ok && wid * per < chunks) {
        w.load_rows();
        w.stream(wid * per, min(chunks, (wid + 1) * per));
      } else {
        w.clear();
      }
      w.leave_part(mine, mine + C::ROWS * D);
      __syncthreads();
      const int row0 = w.s.rt * C::ROWS, rows = min(C::ROWS, w.s.q_len * group - row0);
      for (int i = tid; i < rows * (D / 4); i += 32 * C::WARPS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, tok = (row0 + r) / group;
        float4 o;
        const float sum = add_parts(0, C::WARPS, r, d, o).y;
        const float inv = w.s.len - w.s.q_len + tok >= 0 ? 1.f / sum : 0.f;  // a row that sees no key is 0
        uint2 out;
        out.x = f_to_h16(o.x * inv, p.c.bf16) | f_to_h16(o.y * inv, p.c.bf16) << 16;
        out.y = f_to_h16(o.z * inv, p.c.bf16) | f_to_h16(o.w * inv, p.c.bf16) << 16;
        *reinterpret_cast<uint2*>(p.out + (w.s.t0 + tok) * p.ld_out +
                                  static_cast<size_t>(w.s.head * group + (row0 + r) % group) * D + d) = out;
      }
      fence_proxy_async_smem();  // the next tile's copies overwrite the parts
      __syncthreads();
    }
    return;
  }

  const int per = (base + p.warps - 1) / p.warps;
  int at = warp * per;
  const int end = min(base, at + per);
  float* const ml = p.part + static_cast<size_t>(p.warps) * 2 * C::ROWS * D;
  int tile_at = -1;  // of the row tile whose part the warp holds at its end: its first unit on the line
  int tile_slot = 0;
  while (w.ok && at < end) {
    int units, u0;
    locate(at, units, u0);
    const int u1 = min(units, u0 + end - at), fullc = attn8_full_chunks(w.s.full_tokens);
    const int c0 = attn8_chunk_at(u0, fullc), c1 = attn8_chunk_at(u1, fullc);
    if (c0 < c1 || units == u1 - u0) {
      w.load_rows();
      w.stream(c0, c1);
    } else {
      w.clear();
    }
    if (u0 == 0 && u1 == units) {
      w.finish();
    } else if (at + u1 - u0 == end) {
      tile_at = at - u0;  // the warp ends here: its neighbours may hold the same tile's other parts
      tile_slot = u0 == 0 ? 1 : 0;
    } else {
      const size_t place = static_cast<size_t>(warp) * 2 * C::ROWS;
      w.leave_part(p.part + place * D, ml + 2 * place);
    }
    at += u1 - u0;
  }

  // The parts that the CTA's warps end with, neighbours of one tile added up in the place of the run's first warp.
  if (tile_at >= 0) w.leave_part(mine, mine + C::ROWS * D);
  if (lane == 0) {
    held[wid] = tile_at;
    held_slot[wid] = tile_slot;
  }
  __syncthreads();
  for (int w0 = 0; w0 < C::WARPS;) {
    int w1 = w0 + 1;
    if (held[w0] >= 0) {
      while (w1 < C::WARPS && held[w1] == held[w0]) ++w1;
      for (int i = tid; i < C::ROWS * (D / 4); i += 32 * C::WARPS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float4 o;
        const float2 ms = add_parts(w0, w1, r, d, o);
        const size_t to = (static_cast<size_t>(blockIdx.x * C::WARPS + w0) * 2 + held_slot[w0]) * C::ROWS + r;
        *reinterpret_cast<float4*>(p.part + to * D + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(ml + 2 * to) = ms;
      }
    }
    w0 = w1;
  }
}

// Adds the parts of the row tiles that several CTAs (or two places of one) share, in a fixed order.  blockIdx.x: a
// place for every row tile (n rows make at most n / ROWS + 1 tiles), blockIdx.y: key head.  Latency is all there is
// to it: the parts' maxima and sums come in one round of loads, the accumulators in another.
constexpr int ATTN8_JOIN_THREADS = 256;

template <int D, int NT>
__global__ void __launch_bounds__(ATTN8_JOIN_THREADS) k_attn8_join(const Attn8Params p) {
  using C = Attn8Cfg<D, NT>;
  constexpr int V4 = D / 4, T = ATTN8_JOIN_THREADS, MOST = 160;  // parts: one a CTA and one more
  __shared__ float2 mls[MOST * C::ROWS];
  __shared__ float4 red[T];
  griddep_sync();
  const int group = p.heads / p.c.kv_heads, u = blockIdx.x, tid = threadIdx.x;
  const int b = warp_search(p.batch, u, [&](int i) {
    return static_cast<int>(static_cast<long long>(__ldg(p.cu + i)) * group / C::ROWS) + i;
  });
  int t0, q_len, len;
  attn8_sequence(p, b, t0, q_len, len);
  const int rt = u - (static_cast<int>(static_cast<long long>(__ldg(p.cu + b)) * group / C::ROWS) + b);
  const int tiles = (q_len * group + C::ROWS - 1) / C::ROWS;
  const int total = p.plan[p.batch];
  if (rt < 0 || rt >= tiles || total == 0) return;
  const int units = attn8_units(len, p.c.page);
  const int per = (total + p.warps - 1) / p.warps;
  const int first = p.plan[b] + (blockIdx.y * tiles + rt) * units;
  const int w0 = first / per, w1 = (first + units - 1) / per;
  if (w0 == w1) return;
  // A CTA's run of parts is in the place of its first warp; the last part is its warp's own if more follows it.
  const int cta0 = w0 / C::WARPS, cta1 = w1 / C::WARPS;
  const bool own = first + units != min(total, (w1 + 1) * per) && w1 % C::WARPS != 0;
  const int parts = cta1 - cta0 + 1 + own, rows = min(C::ROWS, q_len * group - rt * C::ROWS);
  const float* ml = p.part + static_cast<size_t>(p.warps) * 2 * C::ROWS * D;
  auto place = [&](int i) {
    const int w = i == 0 ? w0 : i > cta1 - cta0 ? w1 : (cta0 + i) * C::WARPS;
    return (static_cast<size_t>(w) * 2 + (i == 0)) * C::ROWS;  // the part that begins the tile is its warp's second
  };
  for (int i = tid; i < parts * rows; i += T) {
    const int x = i / rows, r = i % rows;
    mls[i] = *reinterpret_cast<const float2*>(ml + 2 * (place(x) + r));
  }
  __syncthreads();
  const int n = rows * V4;               // (row, four channels) to add up
  const int lanes = max(1, T / n);       // threads that share one's parts
  for (int n0 = 0; n0 < n; n0 += T) {
    const int unit = n0 + tid % min(n, T), sub = n < T ? tid / n : 0;
    const bool on = unit < n && sub < lanes;
    const int r = unit / V4, d = unit % V4 * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (on) {
      float top = -INFINITY;
      for (int x = 0; x < parts; ++x) top = fmaxf(top, mls[x * rows + r].x);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
      for (int x = sub; x < parts; x += lanes) {
        const float4 v = *reinterpret_cast<const float4*>(p.part + (place(x) + r) * D + d);
        const float f = fast_exp2(mls[x * rows + r].x - ref);
        o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
      }
      for (int x = 0; x < parts; ++x) sum = fmaf(mls[x * rows + r].y, fast_exp2(mls[x * rows + r].x - ref), sum);
    }
    if (lanes > 1) {
      red[tid] = o;
      __syncthreads();
    }
    if (on && sub == 0) {
      for (int i = 1; i < lanes; ++i) {
        const float4 v = red[tid + i * n];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      const int row = rt * C::ROWS + r, tok = row / group;
      const float inv = len - q_len + tok >= 0 ? 1.f / sum : 0.f;
      uint2 out;
      out.x = f_to_h16(o.x * inv, p.c.bf16) | f_to_h16(o.y * inv, p.c.bf16) << 16;
      out.y = f_to_h16(o.z * inv, p.c.bf16) | f_to_h16(o.w * inv, p.c.bf16) << 16;
      *reinterpret_cast<uint2*>(p.out + (t0 + tok) * p.ld_out +
                                static_cast<size_t>(blockIdx.y * group + row % group) * D + d) = out;
    }
  }
}

}  // namespace b200
