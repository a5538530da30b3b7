// A paged key/value cache held in 8 bits: appending with the position rotation
// (k_kv8_append) and reading back as 16-bit values (k_kv8_read).
//
// A page holds one block of P tokens of every key head:
//   K [page][head][P][D] uint8,  V [page][head][P/4][D][4] uint8 (four tokens of
//   a channel side by side: one 32-bit word of V is then a matrix fragment's
//   four contraction elements, and attention needs no transposition),
//   a code c standing for (c - 128) * scale, one fp32 scale per page and head.
// The newest two blocks of a sequence are also kept in 16 bits ("newest":
// [row][2][head][P][D] and [..][P/4][D][4], block j in slot j % 2).  A block that
// is not full is read from there; it is quantized once, from its 16-bit values,
// when its last token arrives.  So what the cache holds does not depend on how
// the tokens were split among calls, and a sequence may be shortened to any
// length that the two blocks written last still reach (drafted tokens that were refused).
//
// Arithmetic: rotation in fp32 with separately rounded products, then one
// rounding to 16 bits; scale = amax * (1/127); code = rint(x / scale), clamped to
// +-127.  A block with an infinity or NaN gets a NaN scale: it reads as NaN.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"

namespace b200 {

constexpr int DERR_KV_RANGE = 7;  // a page, position or row index outside its buffer: skipped

struct Kv8Cache {
  uint8_t* k_pages;
  uint8_t* v_pages;
  float* k_scale;
  float* v_scale;
  uint16_t* k_new;       // newest two blocks, 16 bits
  uint16_t* v_new;
  const int* table;      // [batch, table_width] page of each block
  const int* rows;       // [batch] row of the newest-blocks buffers, null = the batch index
  int num_pages, kv_heads, page, head_dim, new_rows, table_width;
  int page_shift, dim_shift;  // their logarithms
  int bf16;              // 16-bit type: 0 fp16, 1 bf16
};

struct Kv8AppendParams {
  Kv8Cache c;
  const uint16_t* qkv;   // [tokens, (heads + 2 kv_heads) * D], row stride ld
  long long ld;
  uint16_t* q_out;       // [tokens, heads, D]
  const int* cu;         // [batch + 1] first row of each sequence's new tokens
  const int* start;      // [batch] tokens already cached
  const float* cos;      // [rope_rows, rot / 2], null = no rotation
  const float* sin;
  int rot, interleaved, rope_rows;
  int tokens, batch, heads;
  int by_token;          // unit = token (few tokens a sequence) instead of unit = block
  unsigned row_recip, q_recip;  // 2^32 / (units of a row), 2^32 / q_each, rounded up (q_each 1: 0)
  int k_each, q_each;    // key heads of K or V that a CTA splits its threads among, query heads that it takes
};

__device__ __forceinline__ float h16_to_f(uint32_t bits, int bf16) {
  return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ uint32_t f_to_h16(float v, int bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_half2(a, b);
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]), pack2<BF16>(v[4], v[5]), pack2<BF16>(v[6], v[7]));
}

// Largest b in [0, n) with key(b) <= u, key non-decreasing and key(0) <= u: each
// round probes 32 places at once, one a lane (two rounds for 1024 sequences).
template <typename F>
__device__ __forceinline__ int warp_search(int n, int u, F key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && key(at) <= u);
    const int last = 31 - __clz(below | 1u);
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Four codes rint(x / s) as signed bytes, x / s rounded to fp32 first; inv = 1 / s, |x| <= 127.5 s unless `divide`.
// t = x * inv + 1.5 * 2^23 has the nearest whole number in its low bits; x * inv is within 2^-16 of the quotient, so
// only quotients that near a half (and scales whose reciprocal could overflow: `divide`) need the division itself.
__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d, float s, float inv, bool divide) {
  const float magic = 12582912.f;
  const float x[4] = {a, b, c, d};
  float t[4], near = 1.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = fmaf(x[i], inv, magic);
    near = fminf(near, fabsf(fabsf(fmaf(x[i], inv, magic - t[i])) - 0.5f));
  }
  if (divide || near < 4e-5f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.f), 127.f) + magic;
  }
  return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                     __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
}
// i / d for i * d < 2^32, with d's reciprocal 2^32 / d rounded up (d >= 2)
__device__ __forceinline__ int over(int i, unsigned recip) { return static_cast<int>(__umulhi(i, recip)); }

// The rotation of one row (a head of a token at position pos) falls into units: a pair of 8-channel vectors
// (i, i + rot/2) that turn together, or a vector on its own (interleaved pairs, channels past rot).
struct Kv8Unit {
  uint4 a, b;
  int da, db;  // first channels; db < 0: one vector only
};
__device__ __forceinline__ int kv8_units(const Kv8AppendParams& p) {
  return (p.c.head_dim >> 3) - (p.interleaved ? 0 : p.rot >> 4);
}
__device__ __forceinline__ void load8(const float* from, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(from)), b = __ldg(reinterpret_cast<const float4*>(from) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <bool BF16>
__device__ __forceinline__ Kv8Unit rotate_unit(const Kv8AppendParams& p, const uint16_t* row, int i, int pos) {
  Kv8Unit u;
  u.db = -1;
  const int half = p.rot >> 1;
  const float* cs = p.cos + static_cast<size_t>(pos) * half;
  const float* sn = p.sin + static_cast<size_t>(pos) * half;
  float x[8], y[8];
  if (p.interleaved) {
    u.da = 8 * i;
    u.a = __ldg(reinterpret_cast<const uint4*>(row + u.da));
    if (u.da < p.rot) {
      const float4 co = __ldg(reinterpret_cast<const float4*>(cs + u.da / 2));
      const float4 si = __ldg(reinterpret_cast<const float4*>(sn + u.da / 2));
      const float c4[4] = {co.x, co.y, co.z, co.w}, s4[4] = {si.x, si.y, si.z, si.w};
      unpack8<BF16>(u.a, x);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        y[j] = __fsub_rn(__fmul_rn(x[j], c4[j / 2]), __fmul_rn(x[j + 1], s4[j / 2]));
        y[j + 1] = __fadd_rn(__fmul_rn(x[j + 1], c4[j / 2]), __fmul_rn(x[j], s4[j / 2]));
      }
      u.a = pack8<BF16>(y);
    }
  } else if (i < p.rot >> 4) {
    u.da = 8 * i;
    u.db = 8 * i + half;
    u.a = __ldg(reinterpret_cast<const uint4*>(row + u.da));
    u.b = __ldg(reinterpret_cast<const uint4*>(row + u.db));
    float co[8], si[8], z[8], w[8];
    load8(cs + u.da, co);
    load8(sn + u.da, si);
    unpack8<BF16>(u.a, x);
    unpack8<BF16>(u.b, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[j] = __fsub_rn(__fmul_rn(x[j], co[j]), __fmul_rn(y[j], si[j]));
      w[j] = __fadd_rn(__fmul_rn(y[j], co[j]), __fmul_rn(x[j], si[j]));
    }
    u.a = pack8<BF16>(z);
    u.b = pack8<BF16>(w);
  } else {
    u.da = 8 * (i + (p.rot >> 4));
    u.a = __ldg(reinterpret_cast<const uint4*>(row + u.da));
  }
  return u;
}

// One block of K (what 0) or V (what 1) of one key head (one past the last only joins the barrier): new tokens
// [lo, hi), `had` earlier ones.
template <bool BF16>
__device__ __forceinline__ void kv8_append_head(const Kv8AppendParams& p, int what, int head, int nrow, int blk, int lo,
                                                int hi, int first, int last, int had, int len, bool full, bool keep,
                                                  int page, const uint16_t* rows, uint16_t* tile, unsigned* top_bits) {
  const Kv8Cache& c = p.c;
  const int nth = blockDim.x / p.k_each, tid = threadIdx.x % nth;  // the head's threads
  const int D = c.head_dim, P = c.page, per_row = kv8_units(p);
  uint4* const tile16 = reinterpret_cast<uint4*>(tile);
  uint16_t* newest = (what ? c.v_new : c.k_new) +
                     ((static_cast<size_t>(nrow) * 2 + (blk & 1)) * c.kv_heads + head) * P * D;
  unsigned top = 0;  // largest |value| as 16 bits: their order is the values' order, NaN above infinity
  auto see = [&](uint32_t x) { top = __vmaxu2(top, x & 0x7fff7fffu); };
  const size_t hoff = static_cast<size_t>(p.heads + (what ? c.kv_heads : 0) + head) * D;
  // tokens [from, to) of the block that begins at position `begin`: to the tile and to the newest blocks
  auto take = [&](int begin, int from, int to, bool to_tile, bool to_newest) {
    if (what == 0) {
      for (int i = tid; i < (to - from) * per_row; i += nth) {
        const int row = over(i, p.row_recip), pos = from + row, at = pos - begin;
        const Kv8Unit x = rotate_unit<BF16>(p, rows + pos * p.ld + hoff, i - row * per_row, pos);
        auto put = [&](uint4 w, int d) {
          if (to_tile) {
            *reinterpret_cast<uint4*>(tile + at * D + d) = w;
            see(w.x); see(w.y); see(w.z); see(w.w);
          }
          if (to_newest) *reinterpret_cast<uint4*>(newest + at * D + d) = w;
        };
        put(x.a, x.da);
        if (x.db >= 0) put(x.b, x.db);
      }
      return;
    }
    // four tokens of eight channels: the rows' vectors, transposed to the layout of V
    const int g0 = (from - begin) >> 2, groups = ((to - begin + 3) >> 2) - g0, vpr = D >> 3, vsh = __ffs(vpr) - 1;
    for (int i = tid; i < groups * vpr; i += nth) {
      const int grp = g0 + (i >> vsh), d = (i & (vpr - 1)) * 8, pos = begin + 4 * grp;
      uint32_t r[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (pos + k >= from && pos + k < to)
          w = __ldg(reinterpret_cast<const uint4*>(rows + (pos + k) * p.ld + hoff + d));
        r[k][0] = w.x; r[k][1] = w.y; r[k][2] = w.z; r[k][3] = w.w;
        see(w.x); see(w.y); see(w.z); see(w.w);
      }
      uint16_t* dst[2] = {tile + (grp * D + d) * 4, newest + (grp * D + d) * 4};
      const bool on[2] = {to_tile, to_newest};
      const bool whole = pos >= from && pos + 4 <= to;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!on[x]) continue;
        if (whole) {
#pragma unroll
          for (int w = 0; w < 4; ++w)  // channels d + 2w, d + 2w + 1
            *reinterpret_cast<uint4*>(dst[x] + 8 * w) =
                make_uint4(__byte_perm(r[0][w], r[1][w], 0x5410), __byte_perm(r[2][w], r[3][w], 0x5410),
                           __byte_perm(r[0][w], r[1][w], 0x7632), __byte_perm(r[2][w], r[3][w], 0x7632));
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pos + k >= from && pos + k < to)
#pragma unroll
              for (int j = 0; j < 8; ++j) dst[x][4 * j + k] = static_cast<uint16_t>(r[k][j >> 1] >> (16 * (j & 1)));
        }
      }
    }
  };
  if (head < c.kv_heads) take(blk * P, lo, hi, full, keep);
  if (!full) return;
  // the block's earlier tokens
  if (head >= c.kv_heads) {
  } else if (what == 0) {
    for (int i = tid; i < had * (D >> 3); i += nth) {
      const uint4 w = reinterpret_cast<const uint4*>(newest)[i];
      tile16[i] = w;
      see(w.x); see(w.y); see(w.z); see(w.w);
    }
  } else {
    for (int i = tid; i < ((had + 3) >> 2) * (D >> 1); i += nth) {  // four tokens of two channels
      uint4 w = reinterpret_cast<const uint4*>(newest)[i];
      const int keep4 = had - (i >> (c.dim_shift - 1)) * 4;  // of the four, the earlier ones
      if (keep4 >= 4) {
        tile16[i] = w;
      } else {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < keep4) {
            tile[8 * i + k] = static_cast<uint16_t>(x[k >> 1] >> (16 * (k & 1)));
            tile[8 * i + 4 + k] = static_cast<uint16_t>(x[2 + (k >> 1)] >> (16 * (k & 1)));
          }
        const uint32_t k0 = keep4 >= 2 ? 0xffffffffu : 0xffffu, k1 = keep4 == 3 ? 0xffffu : 0u;
        w.x &= k0; w.z &= k0; w.y &= k1; w.w &= k1;
      }
      see(w.x); see(w.y); see(w.z); see(w.w);
    }
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) top_bits[threadIdx.x >> 5] = top;
  __syncthreads();
  if (head >= c.kv_heads) return;
  const int warp0 = (threadIdx.x - tid) >> 5;
  top = 0;
  for (int i = 0; i < (nth >> 5); ++i) top = max(top, top_bits[warp0 + i]);
  const float amax = h16_to_f(top, BF16);
  const float scale = amax < INFINITY ? __fmul_rn(amax, 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  const int after = last - ((last - blk) & 1);  // the kept block of this slot
  if (blk == first && had > 0 && after >= first + 2)
    take(after * P, after * P, min(len, (after + 1) * P), false, true);
  const size_t ph = static_cast<size_t>(page) * c.kv_heads + head;
  if (tid == 0) (what ? c.v_scale : c.k_scale)[ph] = scale;
  const bool live = scale > 0.f;      // false for an all-zero block and for NaN: codes are then zero points
  const bool small = scale < 1e-30f;  // 1 / scale could overflow: divide
  const float inv = __fdiv_rn(1.f, scale);
  uint4* out = reinterpret_cast<uint4*>((what ? c.v_pages : c.k_pages) + ph * P * D);
  for (int i = tid; i < P * D / 16; i += nth) {
    uint32_t w[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};  // the zero point
    if (live) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        unpack8<BF16>(tile16[2 * i + h], v);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[2 * h + j] ^= quantize4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], scale, inv, small);
      }
    }
    out[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Unit = one touched block of one sequence.  blockIdx.x: unit (or token, by_token);
// blockIdx.y: k_each heads of K, a head of V, or q_each query heads.
// Memory-bound.  Measured: 18400 tokens of 16 + 2 x 16 heads of 64 in 51 us (3.7 TB/s),
// 128 single tokens of 32/8 heads of 128 in 10 us (the blocks that become whole: chains of
// dependent loads).  Heads of one CTA share the rows of cos and sin through L1 (with a head
// a CTA they came from L2 for every head, twice the bytes of the head itself: 114 us against
// 77 us for 27000 tokens of 16 + 2 x 16 heads).  Shared memory holds the block's 16-bit
// values, in the order of the page's codes, between the maximum and the codes, so that
// nothing is read twice.  Four CTAs an SM (64 registers): with three it took 59 us.
template <bool BF16>
__global__ void __launch_bounds__(256, 4) k_kv8_append(const Kv8AppendParams p) {
  extern __shared__ uint4 smem_kv8[];
  __shared__ unsigned top_bits[8];
  griddep_sync();
  const Kv8Cache& c = p.c;
  const int tid = threadIdx.x, nth = blockDim.x;
  const int D = c.head_dim, P = c.page, psh = c.page_shift, u = blockIdx.x;
  const int k_ctas = (c.kv_heads + p.k_each - 1) / p.k_each;
  const int y = blockIdx.y, what = y < k_ctas ? 0 : y < 2 * k_ctas ? 1 : 2;
  int b;
  if (p.by_token) b = warp_search(p.batch, u, [&](int i) { return __ldg(p.cu + i); });
  // n tokens touch at most n/P + 2 blocks, so cu/P + 2b spaces the sequences apart
  else b = warp_search(p.batch, u, [&](int i) { return (__ldg(p.cu + i) >> psh) + 2 * i; });
  const int t0 = __ldg(p.cu + b), end = __ldg(p.cu + b + 1), start = __ldg(p.start + b);
  if (t0 == end) return;
  // (positions of whole blocks around the tokens fit 32 bits)
  if (t0 < 0 || end < t0 || end > p.tokens || start < 0 || start > 0x7fffff00 - (end - t0)) {
    if (tid == 0) record_error(DERR_KV_RANGE);
    return;
  }
  const int n = end - t0, len = start + n;
  int blk;
  if (p.by_token) {
    const int pos = start + u - t0;
    // the first token of a block in this call stands for the block
    if (u < t0 || u >= end || (u != t0 && (pos & (P - 1)) != 0)) return;
    blk = pos >> psh;
  } else {
    blk = (start >> psh) + u - ((t0 >> psh) + 2 * b);
  }
  const int lo = max(start, blk * P), hi = min(len, (blk + 1) * P);  // positions of the block's new tokens
  if (lo >= hi) return;
  const int nrow = c.rows ? __ldg(c.rows + b) : b;
  if (blk >= c.table_width || nrow < 0 || nrow >= c.new_rows || (p.cos && len > p.rope_rows)) {
    if (tid == 0) record_error(DERR_KV_RANGE);
    return;
  }
  const uint16_t* rows = p.qkv + (t0 - start) * p.ld;  // row of position 0
  const int per_row = kv8_units(p);

  if (what == 2) {
    const int h0 = (y - 2 * k_ctas) * p.q_each, h1 = min(p.heads, h0 + p.q_each);
    for (int i = tid; i < (hi - lo) * p.q_each * per_row; i += nth) {
      const int row = over(i, p.row_recip), at = p.q_each > 1 ? over(row, p.q_recip) : row;
      const int pos = lo + at, h = h0 + row - at * p.q_each;
      if (h >= h1) continue;
      const Kv8Unit x = rotate_unit<BF16>(p, rows + pos * p.ld + static_cast<size_t>(h) * D, i - row * per_row, pos);
      uint16_t* to = p.q_out + (static_cast<size_t>(t0 + pos - start) * p.heads + h) * D;
      *reinterpret_cast<uint4*>(to + x.da) = x.a;
      if (x.db >= 0) *reinterpret_cast<uint4*>(to + x.db) = x.b;
    }
    return;
  }

  const bool full = hi == (blk + 1) * P;
  const int page = full ? __ldg(c.table + static_cast<size_t>(b) * c.table_width + blk) : 0;
  if (page < 0 || page >= c.num_pages) {
    if (tid == 0) record_error(DERR_KV_RANGE);
    return;
  }
  // The newest two blocks keep their 16-bit values.  The first touched block may have its earlier tokens in the slot
  // that a later kept block of the same parity takes over: the first block's CTA then writes that block's values
  // too, after it has read what it needs.
  const int first = start >> psh, last = (len - 1) >> psh, had = lo - blk * P;
  const bool others = (start & (P - 1)) != 0 && blk >= first + 2 && ((blk - first) & 1) == 0;
  const bool keep = blk >= last - 1 && !others;
  if (!full && !keep) return;
  const int sub = threadIdx.x / (blockDim.x / p.k_each), head = (what ? y - k_ctas : y) * p.k_each + sub;
  kv8_append_head<BF16>(p, what, head, nrow, blk, lo, hi, first, last, had, len, full, keep, page, rows,
                        reinterpret_cast<uint16_t*>(smem_kv8) + sub * P * D, top_bits);
}

struct Kv8ReadParams {
  Kv8Cache c;
  const int* cu;      // [batch + 1] first output row of each sequence's window
  const int* start;   // [batch] position of the window's first token
  const int* lens;    // [batch] tokens cached (which blocks are full)
  uint16_t* k_out;    // [tokens, kv_heads, D]
  uint16_t* v_out;
  int tokens, batch;
};

// Windows of tokens as 16-bit rows (18400 tokens of 16 heads of 64 in 26 us, 4.3 TB/s).
// Lanes run along the channels, eight a lane, so rows leave in 16-byte stores: a warp takes
// 8, 4 or 2 tokens of one head (head_dim 32, 64, 128).
template <bool BF16>
__global__ void __launch_bounds__(256) k_kv8_read(const Kv8ReadParams p) {
  griddep_sync();
  const Kv8Cache& c = p.c;
  const int D = c.head_dim, P = c.page, vpr = D >> 3;
  const int per = 256 / vpr;  // tokens a pass
  const int head = blockIdx.y, d = (threadIdx.x % vpr) * 8;
  const int t = blockIdx.x * per + threadIdx.x / vpr;
  // one search a warp, at its first token; the few sequences that follow are walked
  const int first = blockIdx.x * per + (threadIdx.x & ~31) / vpr;
  int b = warp_search(p.batch, first, [&](int i) { return __ldg(p.cu + i); });
  if (t >= p.tokens) return;
  while (b + 1 < p.batch && t >= __ldg(p.cu + b + 1)) ++b;
  const int pos = __ldg(p.start + b) + t - __ldg(p.cu + b), blk = pos >> c.page_shift, at = pos & (P - 1);
  const int nrow = c.rows ? __ldg(c.rows + b) : b;
  const size_t to = (static_cast<size_t>(t) * c.kv_heads + head) * D + d;
  const bool full = blk < __ldg(p.lens + b) >> c.page_shift;
  const int page = blk < c.table_width && pos >= 0 ? __ldg(c.table + static_cast<size_t>(b) * c.table_width + blk) : -1;
  // (rows past the last sequence's are nobody's: their positions may be anything)
  if (pos < 0 || (blk >= c.table_width && t < __ldg(p.cu + b + 1)) || (full ? page < 0 || page >= c.num_pages : nrow < 0 || nrow >= c.new_rows)) {
    record_error(DERR_KV_RANGE);
    *reinterpret_cast<uint4*>(p.k_out + to) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(p.v_out + to) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (!full) {
    const size_t base = ((static_cast<size_t>(nrow) * 2 + (blk & 1)) * c.kv_heads + head) * P * D;
    *reinterpret_cast<uint4*>(p.k_out + to) = *reinterpret_cast<const uint4*>(c.k_new + base + at * D + d);
    const uint16_t* v = c.v_new + base + ((at >> 2) * D + d) * 4 + (at & 3);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v[8 * j] | (static_cast<uint32_t>(v[8 * j + 4]) << 16);
    *reinterpret_cast<uint4*>(p.v_out + to) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  const size_t ph = static_cast<size_t>(page) * c.kv_heads + head;
  const float ks = c.k_scale[ph], vs = c.v_scale[ph];
  const uint2 kw = *reinterpret_cast<const uint2*>(c.k_pages + ph * P * D + at * D + d);
  const uint4* vp = reinterpret_cast<const uint4*>(c.v_pages + ph * P * D + ((at >> 2) * D + d) * 4);
  const uint4 v0 = vp[0], v1 = vp[1];
  const uint32_t vw[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
  float kf[8], vf[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // 0x4b000000 | c is 2^23 + c: the code as a float without a conversion
    const uint32_t kc = __byte_perm(j < 4 ? kw.x : kw.y, 0x4b000000u, 0x7440 | (j & 3));
    const uint32_t vc = __byte_perm(vw[j], 0x4b000000u, 0x7440 | (at & 3));
    kf[j] = __fmul_rn(__uint_as_float(kc) - 8388736.f, ks);
    vf[j] = __fmul_rn(__uint_as_float(vc) - 8388736.f, vs);
  }
  *reinterpret_cast<uint4*>(p.k_out + to) = pack8<BF16>(kf);
  *reinterpret_cast<uint4*>(p.v_out + to) = pack8<BF16>(vf);
}

}  // namespace b200
