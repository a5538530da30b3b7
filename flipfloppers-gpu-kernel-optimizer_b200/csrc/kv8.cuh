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
// length its newest two blocks still reach (drafted tokens that were refused).
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
};

__device__ __forceinline__ float h16_to_f(uint32_t bits, int bf16) {
  return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ uint32_t f_to_h16(float v, int bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ void unpack8(uint4 w, int bf16, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = h16_to_f(u[i] & 0xffffu, bf16);
    v[2 * i + 1] = h16_to_f(u[i] >> 16, bf16);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8], int bf16) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = f_to_h16(v[2 * i], bf16) | (f_to_h16(v[2 * i + 1], bf16) << 16);
  return make_uint4(u[0], u[1], u[2], u[3]);
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

// Eight channels of one head of one token at position pos, from d, rotated.
__device__ __forceinline__ uint4 rotate8(const Kv8AppendParams& p, const uint16_t* row, int d, int pos) {
  const uint4 w = *reinterpret_cast<const uint4*>(row + d);
  if (p.cos == nullptr || d >= p.rot) return w;
  const int half = p.rot >> 1;
  const float* cs = p.cos + static_cast<size_t>(pos) * half;
  const float* sn = p.sin + static_cast<size_t>(pos) * half;
  float x[8], y[8];
  unpack8(w, p.c.bf16, x);
  if (p.interleaved) {  // pairs (2i, 2i + 1)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float co = __ldg(cs + (d + i) / 2), si = __ldg(sn + (d + i) / 2);
      y[i] = __fsub_rn(__fmul_rn(x[i], co), __fmul_rn(x[i + 1], si));
      y[i + 1] = __fadd_rn(__fmul_rn(x[i + 1], co), __fmul_rn(x[i], si));
    }
  } else {  // pairs (i, i + rot/2)
    const bool second = d >= half;
    float o[8];
    unpack8(*reinterpret_cast<const uint4*>(row + (second ? d - half : d + half)), p.c.bf16, o);
    const int f = second ? d - half : d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float co = __ldg(cs + f + i), si = __ldg(sn + f + i);
      const float a = __fmul_rn(x[i], co), b = __fmul_rn(o[i], si);
      y[i] = second ? __fadd_rn(a, b) : __fsub_rn(a, b);
    }
  }
  return pack8(y, p.c.bf16);
}

// Unit = one touched block of one sequence.  blockIdx.x: unit (or token, by_token);
// blockIdx.y = 3 * head + {0: K, 1: V, 2: the head's group of query heads}.
// Memory-bound; shared memory holds the block's 16-bit values between the
// maximum and the codes, so that nothing is read twice.
__global__ void __launch_bounds__(256) k_kv8_append(const Kv8AppendParams p) {
  extern __shared__ uint4 smem_kv8[];
  __shared__ unsigned top_bits[8];
  griddep_sync();
  const Kv8Cache& c = p.c;
  const int tid = threadIdx.x, nth = blockDim.x;
  const int D = c.head_dim, P = c.page, head = blockIdx.y / 3, what = blockIdx.y % 3;
  const int u = blockIdx.x;
  int b, blk;
  if (p.by_token) {
    b = warp_search(p.batch, u, [&](int i) { return __ldg(p.cu + i); });
    const int t0 = __ldg(p.cu + b), pos = __ldg(p.start + b) + u - t0;
    // the first token of a block in this call stands for the block
    if (u < t0 || u >= __ldg(p.cu + b + 1) || (u != t0 && pos % P != 0)) return;
    blk = pos / P;
  } else {
    // n tokens touch at most n/P + 2 blocks, so cu/P + 2b spaces the sequences apart
    b = warp_search(p.batch, u, [&](int i) { return __ldg(p.cu + i) / P + 2 * i; });
    blk = __ldg(p.start + b) / P + u - (__ldg(p.cu + b) / P + 2 * b);
  }
  const int t0 = __ldg(p.cu + b), start = __ldg(p.start + b);
  const int n = __ldg(p.cu + b + 1) - t0, len = start + n;
  const int lo = max(start, blk * P), hi = min(len, (blk + 1) * P);  // positions of the block's new tokens
  if (lo >= hi) return;
  const int nrow = c.rows ? __ldg(c.rows + b) : b;
  if (t0 < 0 || n < 0 || t0 + n > p.tokens || start < 0 || blk >= c.table_width || nrow < 0 || nrow >= c.new_rows ||
      (p.cos && len > p.rope_rows)) {
    if (tid == 0) record_error(DERR_KV_RANGE);
    return;
  }
  const int vpr = D >> 3, vsh = __ffs(vpr) - 1;  // 16-byte vectors a row (a power of two)
  const uint16_t* rows = p.qkv + (t0 - start) * p.ld;  // row of position 0

  if (what == 2) {  // the query heads of this key head's group
    const int group = p.heads / c.kv_heads, per = group * vpr;
    for (int i = tid; i < (hi - lo) * per; i += nth) {
      const int pos = lo + i / per, r = i % per, h = head * group + (r >> vsh), d = (r & (vpr - 1)) * 8;
      const uint16_t* src = rows + pos * p.ld + static_cast<size_t>(h) * D;
      *reinterpret_cast<uint4*>(p.q_out + (static_cast<size_t>(t0 + pos - start) * p.heads + h) * D + d) =
          rotate8(p, src, d, pos);
    }
    return;
  }

  const bool full = hi == (blk + 1) * P;
  const bool keep = blk >= (len - 1) / P - 1;
  uint16_t* newest = (what ? c.v_new : c.k_new) +
                     ((static_cast<size_t>(nrow) * 2 + (blk & 1)) * c.kv_heads + head) * P * D;
  const uint16_t* tile = reinterpret_cast<const uint16_t*>(smem_kv8);
  unsigned top = 0;  // largest |value| as 16 bits: their order is the values' order, NaN above infinity
  auto see = [&](uint4 w) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __vmaxu2(top, x[i] & 0x7fff7fffu);
  };
  const size_t hoff = static_cast<size_t>(p.heads + (what ? c.kv_heads : 0) + head) * D;
  auto load = [&](int pos, int d) {
    const uint16_t* src = rows + pos * p.ld + hoff;
    return what ? *reinterpret_cast<const uint4*>(src + d) : rotate8(p, src, d, pos);
  };
  auto put_newest = [&](int at, int d, uint4 w) {
    if (what) {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      uint16_t* to = newest + ((at >> 2) * D + d) * 4 + (at & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) to[4 * j] = static_cast<uint16_t>(x[j >> 1] >> (16 * (j & 1)));
    } else {
      *reinterpret_cast<uint4*>(newest + at * D + d) = w;
    }
  };
  // The first touched block may have its earlier tokens in the slot that a later
  // kept block of the same parity takes over: the first block's CTA then writes
  // that block's values too, after it has read what it needs.
  const int first = start / P, last = (len - 1) / P, had0 = start - first * P;
  const bool others = had0 > 0 && blk >= first + 2 && ((blk - first) & 1) == 0;
  for (int i = tid; i < (hi - lo) * vpr; i += nth) {
    const int pos = lo + (i >> vsh), d = (i & (vpr - 1)) * 8, at = pos - blk * P;
    if (!full && (!keep || others)) break;
    const uint4 w = load(pos, d);
    if (full) {
      smem_kv8[at * vpr + (d >> 3)] = w;
      see(w);
    }
    if (keep && !others) put_newest(at, d, w);
  }
  if (!full) return;
  // the block's earlier tokens, from the newest blocks
  const int had = lo - blk * P;
  if (what == 0) {
    for (int i = tid; i < had * vpr; i += nth) {
      const uint4 w = *reinterpret_cast<const uint4*>(newest + i * 8);
      smem_kv8[i] = w;
      see(w);
    }
  } else {
    uint16_t* t16 = reinterpret_cast<uint16_t*>(smem_kv8);
    for (int i = tid; i < had * D; i += nth) {
      const int at = i / D, d = i % D;
      const uint32_t x = newest[((at >> 2) * D + d) * 4 + (at & 3)];
      t16[i] = static_cast<uint16_t>(x);
      top = __vmaxu2(top, x & 0x7fffu);
    }
  }
  const int after = last - ((last - blk) & 1);  // the kept block of this slot
  if (blk == first && had > 0 && after >= first + 2) {
    __syncthreads();
    const int from = after * P, to = min(len, from + P);
    for (int i = tid; i < (to - from) * vpr; i += nth) {
      const int d = (i & (vpr - 1)) * 8, at = i >> vsh;
      put_newest(at, d, load(from + at, d));
    }
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) top_bits[tid >> 5] = top;
  __syncthreads();
  for (int i = 0; i < (nth >> 5); ++i) top = max(top, top_bits[i]);
  const float amax = h16_to_f(top, c.bf16);
  const float scale = amax < INFINITY ? __fmul_rn(amax, 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  const int page = __ldg(c.table + static_cast<size_t>(b) * c.table_width + blk);
  if (page < 0 || page >= c.num_pages) {
    if (tid == 0) record_error(DERR_KV_RANGE);
    return;
  }
  const size_t ph = static_cast<size_t>(page) * c.kv_heads + head;
  if (tid == 0) (what ? c.v_scale : c.k_scale)[ph] = scale;
  const bool live = scale > 0.f;  // false for an all-zero block and for NaN: codes are then zero points
  auto code = [&](uint32_t bits) -> uint32_t {
    if (!live) return 128u;
    const float r = rintf(__fdiv_rn(h16_to_f(bits, c.bf16), scale));
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(r, -127.f), 127.f)) + 128);
  };
  uint4* out = reinterpret_cast<uint4*>((what ? c.v_pages : c.k_pages) + ph * P * D);
  for (int i = tid; i < P * D / 16; i += nth) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // K: 16 channels of a token; V: four tokens of four channels
        const int e = what ? ((i * 4 / D) * 4 + k) * D + (i * 4) % D + j : i * 16 + j * 4 + k;
        w[j] |= code(tile[e]) << (8 * k);
      }
    }
    out[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
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

// Windows of tokens as 16-bit rows.  A warp takes four tokens of one head: lanes
// run along the channels, eight a lane, so rows leave in 16-byte stores.
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
  const int pos = __ldg(p.start + b) + t - __ldg(p.cu + b), blk = pos / P, at = pos % P;
  const int nrow = c.rows ? __ldg(c.rows + b) : b;
  const size_t to = (static_cast<size_t>(t) * c.kv_heads + head) * D + d;
  const bool full = (blk + 1) * P <= __ldg(p.lens + b);
  const int page = blk < c.table_width && pos >= 0 ? __ldg(c.table + static_cast<size_t>(b) * c.table_width + blk) : -1;
  if (pos < 0 || (full ? page < 0 || page >= c.num_pages : nrow < 0 || nrow >= c.new_rows)) {
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
    const uint32_t kc = ((j < 4 ? kw.x : kw.y) >> (8 * (j & 3))) & 0xffu;
    const uint32_t vc = (vw[j] >> (8 * (at & 3))) & 0xffu;
    kf[j] = __fmul_rn(static_cast<float>(static_cast<int>(kc) - 128), ks);
    vf[j] = __fmul_rn(static_cast<float>(static_cast<int>(vc) - 128), vs);
  }
  *reinterpret_cast<uint4*>(p.k_out + to) = pack8(kf, c.bf16);
  *reinterpret_cast<uint4*>(p.v_out + to) = pack8(vf, c.bf16);
}

}  // namespace b200
