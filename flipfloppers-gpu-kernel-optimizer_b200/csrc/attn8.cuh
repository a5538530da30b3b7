// Attention of new tokens over the 8-bit paged cache of kv8.cuh:
//   out[r] = sum_j softmax_j(q[r] . k_j * scale) v_j,   k, v = (code - 128) * block scale
// The rows of one key head are its group's query heads times the sequence's new
// tokens; a row of the token at position p sees the keys 0..p.
//
// Decoding reads the cache once and computes little: the bound is HBM.  Every
// WARP streams its own range of 32-token chunks, with no barrier anywhere:
//   - all (sequence, key head, row tile, chunk) work is one line, cut into equal
//     pieces, one a warp, so ragged lengths load every SM alike; a piece that
//     holds only part of a row tile leaves (max, sum, accumulator) in the
//     workspace and k_attn8_join adds the parts in a fixed order;
//   - codes go from HBM to shared memory by cp.async into slots private to the
//     lane that will use them (ATTN8_STAGES chunks ahead), so only the lane's own
//     wait_group orders them;
//   - the products run as S^T = K Q^T and O^T = V^T P^T on m16n8k16 tensor-core
//     steps: tokens (channels of V) fill the 16 rows, query rows the 8 columns, so
//     up to 8 rows cost one column tile (NT = 1) and up to 16 two (NT = 2), and the
//     codes are widened to fp16 (exactly: 1024 + c, less 1152) once for all rows;
//   - scores take the block's K scale, and each block's V product its V scale, in
//     fp32: the codes enter the products as whole numbers.
// Contraction order is free, so a lane's 16 bytes of K are the fragment elements of
// four steps; key tau(m) = 4 (m/2) + m%2 (+2 for m >= 8) sits in row m, which after
// the 8x8 transposition of P (movmatrix) meets the word of V with the same four keys.
#pragma once

#include "kv8.cuh"

namespace b200 {

constexpr int ATTN8_WARPS = 8;
constexpr int ATTN8_CHUNK = 32;   // tokens
constexpr int ATTN8_STAGES = 3;
constexpr int ATTN8_MAX_BATCH = 4096;

struct Attn8Params {
  Kv8Cache c;
  const uint16_t* q;     // [tokens, heads, D], row stride ld_q
  uint16_t* out;         // [tokens, heads, D], row stride ld_out
  long long ld_q, ld_out;
  const int* cu;         // [batch + 1] first row of each sequence's new tokens
  const int* lens;       // [batch] cached tokens, the new ones included
  int tokens, batch, heads;
  int split;             // 1: cut the line of chunks into equal pieces; 0: whole row tiles
  float scale_log2;      // scale * log2(e)
  int warps;             // warps of the launch
  int* plan;             // [batch + 1] first chunk of each sequence on the line (written by CTA 0)
  float* part;           // [warps][2][rows][D] accumulators, then [warps][2][rows][2] (max, sum)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// a bf16 pair with its infinities and NaN taken as 0
__device__ __forceinline__ uint32_t finite_only(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
  return x;
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
  const int n = live ? BYTES : 0;  // 0: the slot is filled with zeros and src is not read
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
  static constexpr int CB = D >= 64 ? 16 : 8;        // bytes a lane copies of a K row at once
  static constexpr int NCH = D / (4 * CB);           // such copies a row
  static constexpr int K_BYTES = ATTN8_CHUNK * D;    // one chunk
  static constexpr int V_BYTES = ATTN8_CHUNK * D;
  static constexpr int S_BYTES = 4 * 32 * 4;         // the chunk's scales, a copy a lane: K and V, two half chunks
  static constexpr int STAGE = K_BYTES + V_BYTES + S_BYTES;
  static constexpr int RING = ATTN8_STAGES * STAGE;  // one warp's
  static constexpr int SMEM = ATTN8_WARPS * RING;
};

// What one warp knows of the row tile it works on.
struct Attn8Seg {
  int b, head, rt;       // sequence, key head, row tile
  int len, full_tokens;  // cached tokens; those in full blocks
  int q_len, t0;
};

// chunks of a sequence: those of the full blocks, then those of the newest block
__device__ __forceinline__ int attn8_chunks(int len, int page) {
  const int full = len / page * page;
  return max(1, (full + ATTN8_CHUNK - 1) / ATTN8_CHUNK + (len - full + ATTN8_CHUNK - 1) / ATTN8_CHUNK);
}

template <int D, int NT>
struct Attn8Warp {
  using C = Attn8Cfg<D, NT>;
  const Attn8Params& p;
  const uint32_t ring;   // shared address of this warp's ring
  const uint8_t* ringp;
  const int lane, g, t;
  Attn8Seg s;
  uint32_t qb[D / 16][NT][2];
  float qf[NT][2];       // score factor of this lane's columns: scale * log2(e) * row factor
  int lim[NT][2];        // keys that this lane's columns see
  int lo_lim, hi_lim;    // least and most of the tile's rows
  float m[NT][2], l[NT][2];
  float acc[D / 16][NT][4];
  int window, page_now, page_next;  // block of lane 0; page ids of 32 blocks from there, and of the next 32

  __device__ Attn8Warp(const Attn8Params& pp, uint8_t* smem, int warp_in_cta)
      : p(pp), ring(smem_u32(smem) + warp_in_cta * C::RING), ringp(smem + warp_in_cta * C::RING),
        lane(threadIdx.x & 31), g(lane >> 2), t(lane & 3) {}

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

  __device__ __forceinline__ void load_rows() {
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
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }
    }
    const int i0 = s.rt * C::ROWS / group, i1 = min(s.q_len - 1, (s.rt * C::ROWS + C::ROWS - 1) / group);
    lo_lim = max(0, s.len - s.q_len + i0 + 1);
    hi_lim = max(0, s.len - s.q_len + i1 + 1);
#pragma unroll
    for (int a = 0; a < D / 16; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][n][e] = 0.f;
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
  __device__ __forceinline__ void open_window(int blk) {
    window = blk;
    page_now = fetch_page(blk + lane);
    page_next = fetch_page(blk + 32 + lane);
  }
  __device__ __forceinline__ size_t page_head(int blk) {
    if (blk >= window + 32) {
      window += 32;
      page_now = page_next;
      page_next = fetch_page(window + 32 + lane);
    }
    return static_cast<size_t>(__shfl_sync(0xffffffffu, page_now, blk - window)) * p.c.kv_heads + s.head;
  }

  // start the copies of chunk c (of full blocks); chunks come in order
  __device__ __forceinline__ void issue_k(int c, int slot) {
    const int P = p.c.page;
    const uint32_t dst = ring + slot * C::STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = c * ATTN8_CHUNK + 16 * h;
      const bool live = tok < s.full_tokens;
      const size_t ph = page_head((live ? tok : c * ATTN8_CHUNK) / P);
      const uint8_t* src = p.c.k_pages + ph * P * D + (tok % P) * D;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 4 * (g >> 1) + (g & 1) + 2 * r;
#pragma unroll
        for (int x = 0; x < C::NCH; ++x)
          copy_async<C::CB>(dst + (((h * 2 + r) * C::NCH + x) * 32 + lane) * C::CB, src + row * D + (4 * x + t) * C::CB,
                            live);
      }
      copy_async<4>(dst + C::K_BYTES + C::V_BYTES + (h * 32 + lane) * 4, p.c.k_scale + ph, live);
    }
    copy_commit();
  }
  __device__ __forceinline__ void issue_v(int c, int slot) {
    const int P = p.c.page;
    const uint32_t dst = ring + slot * C::STAGE + C::K_BYTES;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = c * ATTN8_CHUNK + 16 * h;
      const bool live = tok < s.full_tokens;
      const size_t ph = page_head((live ? tok : c * ATTN8_CHUNK) / P);
      const uint8_t* src = p.c.v_pages + ph * P * D + (tok % P) * D;
#pragma unroll
      for (int x = 0; x < D / 32; ++x)
        copy_async<16>(dst + ((h * (D / 32) + x) * 32 + lane) * 16, src + t * 4 * D + 128 * x + 16 * g, live);
      copy_async<4>(dst + C::V_BYTES + ((2 + h) * 32 + lane) * 4, p.c.v_scale + ph, live);
    }
    copy_commit();
  }

  // scores of one chunk (log2 units, keys outside the rows' view at -inf) -> P (fp32) and the running maximum
  __device__ __forceinline__ void softmax_step(float (&sc)[2][NT][4], int tok0, bool masked) {
    if (masked) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
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
        float x = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float now = fmaxf(m[n][e], x);
        const float ref = now == -INFINITY ? 0.f : now;  // no key seen yet: every weight is 0
        alpha[n][e] = fast_exp2(m[n][e] - ref);
        moved |= now != m[n][e];
        m[n][e] = now;
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
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

  __device__ __forceinline__ void chunk_scores(int c, int slot, float (&sc)[2][NT][4]) {
    const uint8_t* src = ringp + slot * C::STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[2][D / 16];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int x = 0; x < C::NCH; ++x) {
          const uint8_t* at = src + (((h * 2 + r) * C::NCH + x) * 32 + lane) * C::CB;
          if constexpr (C::CB == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            w[r][4 * x] = v.x; w[r][4 * x + 1] = v.y; w[r][4 * x + 2] = v.z; w[r][4 * x + 3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[r][2 * x] = v.x; w[r][2 * x + 1] = v.y;
          }
        }
      const float ks = *reinterpret_cast<const float*>(src + C::K_BYTES + C::V_BYTES + (h * 32 + lane) * 4);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][n][e] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t a[4];
        widen(w[0][j], a[0], a[2]);
        widen(w[1][j], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(sc[h][n], a, qb[j][n][0], qb[j][n][1]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][n][e] *= ks * qf[n][e & 1];
    }
  }

  __device__ __forceinline__ void chunk_values(int c, int slot, const float (&pr)[2][NT][4], bool masked) {
    const uint8_t* src = ringp + slot * C::STAGE + C::K_BYTES;
    uint32_t b[2][NT][2];
    float f[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float vs = *reinterpret_cast<const float*>(src + C::V_BYTES + ((2 + h) * 32 + lane) * 4);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        b[h][n][0] = transpose8x8(pack_half2(pr[h][n][0], pr[h][n][1]));
        b[h][n][1] = transpose8x8(pack_half2(pr[h][n][2], pr[h][n][3]));
#pragma unroll
        for (int e = 0; e < 2; ++e)  // a block that a row does not see adds nothing, whatever its scale
          f[h][n][e] = masked && lim[n][e] <= c * ATTN8_CHUNK + 16 * h ? 0.f : vs;
      }
    }
    const bool one = p.c.page >= ATTN8_CHUNK;  // one scale for the chunk
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      uint4 w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) w[h] = *reinterpret_cast<const uint4*>(src + ((h * (D / 32) + x) * 32 + lane) * 16);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float o[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4];
          widen(y ? w[h].z : w[h].x, a[0], a[2]);
          widen(y ? w[h].w : w[h].y, a[1], a[3]);
          if (h == 0 || !one) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n], a, b[h][n][0], b[h][n][1]);
          if (h == 1 || !one) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[2 * x + y][n][e] = fmaf(o[n][e], f[one ? 0 : h][n][e & 1], acc[2 * x + y][n][e]);
          }
        }
      }
    }
  }

  // a chunk of the newest block, 16-bit values from global memory
  template <bool BF16>
  __device__ __forceinline__ void newest_chunk(int c) {
    const int P = p.c.page, tok0 = s.full_tokens + c * ATTN8_CHUNK, off = c * ATTN8_CHUNK;
    const int row = p.c.rows ? __ldg(p.c.rows + s.b) : s.b;
    if (row < 0 || row >= p.c.new_rows) {
      record_error(DERR_KV_RANGE);
      return;
    }
    const size_t base =
        ((static_cast<size_t>(row) * 2 + (s.full_tokens / P & 1)) * p.c.kv_heads + s.head) * static_cast<size_t>(P) * D;
    float sc[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][n][e] = 0.f;
    // rows in their own type for the scores: bf16 rows are read again
#pragma unroll
    for (int j = 0; j < D / 16; j += 2) {
      uint4 w[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int at = off + 16 * h + 4 * (g >> 1) + (g & 1) + 2 * r;
          w[h][r] = tok0 - off + at < s.len ? *reinterpret_cast<const uint4*>(p.c.k_new + base + at * D + chan(j))
                                            : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint4 q = make_uint4(qb[j][n][0], qb[j][n][1], qb[j + 1][n][0], qb[j + 1][n][1]);
        if constexpr (BF16) {
          bool ok;
          const uint16_t* src = row_ptr(s.rt * C::ROWS + 8 * n + g, ok);
          const uint2 q0 = *reinterpret_cast<const uint2*>(src + chan(j));
          const uint2 q1 = *reinterpret_cast<const uint2*>(src + chan(j + 1));
          q = ok ? make_uint4(q0.x, q0.y, q1.x, q1.y) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a0[4] = {w[h][0].x, w[h][1].x, w[h][0].y, w[h][1].y};
          const uint32_t a1[4] = {w[h][0].z, w[h][1].z, w[h][0].w, w[h][1].w};
          if constexpr (BF16) {
            mma_bf16(sc[h][n], a0, q.x, q.y);
            mma_bf16(sc[h][n], a1, q.z, q.w);
          } else {
            mma_f16(sc[h][n], a0, q.x, q.y);
            mma_f16(sc[h][n], a1, q.z, q.w);
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][n][e] *= BF16 ? p.scale_log2 : qf[n][e & 1];
    const bool masked = tok0 + ATTN8_CHUNK > lo_lim;
    softmax_step(sc, tok0, masked);
    uint32_t b[2][NT][2], bl[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x = sc[h][n][2 * r], y = sc[h][n][2 * r + 1];
          if constexpr (BF16) {
            // bf16 weights keep 8 bits: a second product adds what the first leaves out
            const uint32_t xh = f_to_h16(x, 1), yh = f_to_h16(y, 1);
            const uint32_t xl = f_to_h16(x - h16_to_f(xh, 1), 1), yl = f_to_h16(y - h16_to_f(yh, 1), 1);
            b[h][n][r] = transpose8x8(xh | yh << 16);
            bl[h][n][r] = transpose8x8(xl | yl << 16);
          } else {
            b[h][n][r] = transpose8x8(pack_half2(x, y));
          }
        }
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      uint4 w[2][2];
      bool odd = false;  // an infinity or NaN among the values
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int have = s.len - (tok0 + 16 * h + 4 * t);  // of this lane's four tokens
        const uint32_t k0 = have >= 2 ? 0xffffffffu : have == 1 ? 0xffffu : 0u;
        const uint32_t k1 = have >= 4 ? 0xffffffffu : have == 3 ? 0xffffu : 0u;
        const uint16_t* src = p.c.v_new + base + (static_cast<size_t>(off / 4 + 4 * h + t) * D + 32 * x + 4 * g) * 4;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint4 v = have > 0 ? *reinterpret_cast<const uint4*>(src + 8 * y) : make_uint4(0, 0, 0, 0);
          v.x &= k0; v.z &= k0; v.y &= k1; v.w &= k1;  // what lies past the end is never summed
          w[h][y] = v;
          constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
          const uint32_t top = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                        __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
          odd |= (top & 0xffffu) >= inf || (top >> 16) >= inf;
        }
      }
      // 0 * infinity must not reach rows that do not see the value: rows are then taken apart by what they see
      const bool strange = __any_sync(0xffffffffu, odd), apart = masked && strange;
      for (int seen = apart ? max(lo_lim, tok0 + 1) : hi_lim; seen <= max(hi_lim, apart ? tok0 + 1 : 0); ++seen) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float o[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 v = w[h][y];
            if (apart) {
              const int have = seen - (tok0 + 16 * h + 4 * t);
              const uint32_t k0 = have >= 2 ? 0xffffffffu : have == 1 ? 0xffffu : 0u;
              const uint32_t k1 = have >= 4 ? 0xffffffffu : have == 3 ? 0xffffu : 0u;
              v.x &= k0; v.z &= k0; v.y &= k1; v.w &= k1;
            }
            const uint32_t a[4] = {v.x, v.z, v.y, v.w};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (BF16) {
                mma_bf16(o[n], a, b[h][n][0], b[h][n][1]);
                uint32_t al[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) al[e] = strange ? finite_only(a[e]) : a[e];
                mma_bf16(o[n], al, bl[h][n][0], bl[h][n][1]);
              } else {
                mma_f16(o[n], a, b[h][n][0], b[h][n][1]);
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!apart || lim[n][e & 1] == seen) acc[2 * x + y][n][e] += o[n][e];
        }
      }
    }
  }

  // chunks [c0, c1) of the segment
  __device__ __forceinline__ void stream(int c0, int c1) {
    const int fullc = (s.full_tokens + ATTN8_CHUNK - 1) / ATTN8_CHUNK;
    const int e1 = min(min(c1, fullc), (hi_lim + ATTN8_CHUNK - 1) / ATTN8_CHUNK);  // what no row sees is not read
    if (c0 < e1) {
      open_window(c0 * ATTN8_CHUNK / p.c.page);
      for (int i = 0; i < ATTN8_STAGES - 1; ++i) {
        if (c0 + i < e1) {
          issue_k(c0 + i, i);
          issue_v(c0 + i, i);
        } else {
          copy_commit();
          copy_commit();
        }
      }
      int slot = 0;
      for (int c = c0; c < e1; ++c) {
        const int ahead = c + ATTN8_STAGES - 1, aslot = slot == 0 ? ATTN8_STAGES - 1 : slot - 1;
        float sc[2][NT][4];
        copy_wait<2 * (ATTN8_STAGES - 1) - 1>();
        chunk_scores(c, slot, sc);
        if (ahead < e1) issue_k(ahead, aslot); else copy_commit();
        const int tok0 = c * ATTN8_CHUNK;
        const bool masked = min(tok0 + ATTN8_CHUNK, s.full_tokens) > lo_lim || tok0 + ATTN8_CHUNK > s.full_tokens;
        softmax_step_full(sc, tok0, masked);
        copy_wait<2 * (ATTN8_STAGES - 1) - 1>();
        chunk_values(c, slot, sc, masked);
        if (ahead < e1) issue_v(ahead, aslot); else copy_commit();
        slot = slot + 1 == ATTN8_STAGES ? 0 : slot + 1;
      }
      copy_wait<0>();
    }
    for (int c = max(c0, fullc); c < c1; ++c) {
      if (s.full_tokens + (c - fullc) * ATTN8_CHUNK >= hi_lim) break;
      if (p.c.bf16) newest_chunk<true>(c - fullc);
      else newest_chunk<false>(c - fullc);
    }
  }
  // the last chunk of the full blocks may be half empty: its other half belongs to the newest block
  __device__ __forceinline__ void softmax_step_full(float (&sc)[2][NT][4], int tok0, bool masked) {
    if (tok0 + ATTN8_CHUNK > s.full_tokens) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[1][n][e] = -INFINITY;
    }
    softmax_step(sc, tok0, masked);
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
  __device__ __forceinline__ void leave_part(int warp, int slot) {
    join_lanes();
    const size_t at = (static_cast<size_t>(warp) * 2 + slot) * C::ROWS;
    float* ml = p.part + static_cast<size_t>(p.warps) * 2 * C::ROWS * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const size_t r = at + 8 * n + 2 * t + e;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          *reinterpret_cast<float4*>(p.part + r * D + 32 * x + 4 * g) =
              make_float4(acc[2 * x][n][e], acc[2 * x][n][e + 2], acc[2 * x + 1][n][e], acc[2 * x + 1][n][e + 2]);
        if (g == 0) *reinterpret_cast<float2*>(ml + 2 * r) = make_float2(m[n][e], l[n][e]);
      }
  }
};

// sequence b's new tokens, clipped to what the buffers hold
__device__ __forceinline__ void attn8_sequence(const Attn8Params& p, int b, int& t0, int& q_len, int& len) {
  t0 = __ldg(p.cu + b);
  q_len = __ldg(p.cu + b + 1) - t0;
  len = __ldg(p.lens + b);
  if (t0 < 0 || q_len < 0 || t0 + q_len > p.tokens || len < 0 || len > static_cast<long long>(p.c.table_width) * p.c.page) {
    record_error(DERR_KV_RANGE);
    t0 = q_len = len = 0;
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(32 * ATTN8_WARPS, D == 128 ? 1 : 2) k_attn8(const Attn8Params p) {
  using C = Attn8Cfg<D, NT>;
  extern __shared__ uint8_t smem_attn8[];
  __shared__ int tot[ATTN8_WARPS];
  int* line = reinterpret_cast<int*>(smem_attn8 + C::SMEM);  // [batch + 1] first work unit of each sequence
  griddep_sync();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int group = p.heads / p.c.kv_heads;
  int base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32 * ATTN8_WARPS) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.batch) {
      int t0, q_len, len;
      attn8_sequence(p, b, t0, q_len, len);
      n = p.c.kv_heads * ((q_len * group + C::ROWS - 1) / C::ROWS) * (p.split ? attn8_chunks(len, p.c.page) : 1);
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
    for (int i = 0; i < ATTN8_WARPS; ++i) {
      if (i < wid) before += tot[i];
      base += tot[i];
    }
    if (b < p.batch) line[b] = before + sum - n;
    __syncthreads();
  }
  if (tid == 0) line[p.batch] = base;
  __syncthreads();
  if (p.split && blockIdx.x == 0)
    for (int i = tid; i <= p.batch; i += 32 * ATTN8_WARPS) p.plan[i] = line[i];

  Attn8Warp<D, NT> w(p, smem_attn8, wid);
  const int warp = blockIdx.x * ATTN8_WARPS + wid;
  const int per = (base + p.warps - 1) / p.warps;
  int at = p.split ? warp * per : warp;
  const int end = p.split ? min(base, at + per) : base;
  int b = 0;
  while (at < end) {
    b = warp_search(p.batch, at, [&](int i) { return line[i]; });
    int t0, q_len, len;
    attn8_sequence(p, b, t0, q_len, len);
    const int tiles = (q_len * group + C::ROWS - 1) / C::ROWS;
    const int chunks = p.split ? attn8_chunks(len, p.c.page) : 1;
    const int item = (at - line[b]) / chunks, c0 = (at - line[b]) % chunks;
    w.s.b = b;
    w.s.head = item / tiles;
    w.s.rt = item % tiles;
    w.s.len = len;
    w.s.full_tokens = len / p.c.page * p.c.page;
    w.s.q_len = q_len;
    w.s.t0 = t0;
    w.load_rows();
    if (p.split) {
      const int c1 = min(chunks, c0 + end - at);
      w.stream(c0, c1);
      if (c0 == 0 && c1 == chunks) w.finish();
      else w.leave_part(warp, c0 == 0 ? 1 : 0);
      at += c1 - c0;
    } else {
      w.stream(0, attn8_chunks(len, p.c.page));
      w.finish();
      at += p.warps;
    }
  }
}

// Adds the parts of the row tiles that several warps share, in the warps' order.
// blockIdx.x: a place for every row tile (n rows make at most n / ROWS + 1 tiles),
// blockIdx.y: key head.
template <int D, int NT>
__global__ void __launch_bounds__(128) k_attn8_join(const Attn8Params p) {
  using C = Attn8Cfg<D, NT>;
  griddep_sync();
  const int group = p.heads / p.c.kv_heads, u = blockIdx.x;
  const int b = warp_search(p.batch, u, [&](int i) {
    return static_cast<int>(static_cast<long long>(__ldg(p.cu + i)) * group / C::ROWS) + i;
  });
  int t0, q_len, len;
  attn8_sequence(p, b, t0, q_len, len);
  const int rt = u - (static_cast<int>(static_cast<long long>(__ldg(p.cu + b)) * group / C::ROWS) + b);
  const int tiles = (q_len * group + C::ROWS - 1) / C::ROWS;
  if (rt < 0 || rt >= tiles) return;
  const int chunks = attn8_chunks(len, p.c.page);
  const int per = (p.plan[p.batch] + p.warps - 1) / p.warps;
  const int first = p.plan[b] + (blockIdx.y * tiles + rt) * chunks;
  const int w0 = first / per, w1 = (first + chunks - 1) / per;
  if (w0 == w1) return;
  const float* ml = p.part + static_cast<size_t>(p.warps) * 2 * C::ROWS * D;
  for (int i = threadIdx.x; i < C::ROWS * (D / 4); i += 128) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const int row = rt * C::ROWS + r, tok = row / group;
    if (tok >= q_len) continue;
    float top = -INFINITY;
    for (int w = w0; w <= w1; ++w) {
      const size_t at = (static_cast<size_t>(w) * 2 + (w == w0)) * C::ROWS + r;
      top = fmaxf(top, ml[2 * at]);
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) {
      const size_t at = (static_cast<size_t>(w) * 2 + (w == w0)) * C::ROWS + r;
      const float f = fast_exp2(ml[2 * at] - ref);
      const float4 v = *reinterpret_cast<const float4*>(p.part + at * D + d);
      sum += ml[2 * at + 1] * f;
      o[0] += v.x * f; o[1] += v.y * f; o[2] += v.z * f; o[3] += v.w * f;
    }
    const float inv = len - q_len + tok >= 0 ? 1.f / sum : 0.f;
    uint2 out;
    out.x = f_to_h16(o[0] * inv, p.c.bf16) | f_to_h16(o[1] * inv, p.c.bf16) << 16;
    out.y = f_to_h16(o[2] * inv, p.c.bf16) | f_to_h16(o[3] * inv, p.c.bf16) << 16;
    *reinterpret_cast<uint2*>(p.out + (t0 + tok) * p.ld_out +
                              static_cast<size_t>(blockIdx.y * group + row % group) * D + d) = out;
  }
}

}  // namespace b200
