// Host side of the 8-bit serving operators: argument checks and launches.  Part of
// the library's one translation unit (included by b200_block.cu, whose helpers it uses).
#pragma once

#include "attn8_tile.cuh"
#include "gemm_i8.cuh"

namespace {

// `rows` rows of `width` bytes, `pitch` bytes apart
struct Rows8 {
  const void* at;
  long long rows, pitch, width;
};
// Whether two such ranges share a byte (columns of one wider buffer may lie side by side).
bool overlap(const Rows8& a, const Rows8& b) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0) return false;
  const auto a0 = reinterpret_cast<uintptr_t>(a.at), b0 = reinterpret_cast<uintptr_t>(b.at);
  if (a0 + (a.rows - 1) * a.pitch + a.width <= b0 || b0 + (b.rows - 1) * b.pitch + b.width <= a0) return false;
  const long long pitch = a.rows > 1 ? a.pitch : b.pitch;
  if ((a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) || pitch <= 0) return true;
  long long d = static_cast<long long>(b0 - a0) % pitch;  // b's first column in a's rows
  if (d < 0) d += pitch;
  return d < a.width || d + b.width > pitch;
}

int cache8_check(const B200KvCache8* c) {
  if (!c || !c->k_pages || !c->v_pages || !c->k_scale || !c->v_scale || !c->k_newest || !c->v_newest || !c->table)
    return B200_ERR_ARG;
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return B200_ERR_HEAD_DIM;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return B200_ERR_TILE;
  if (c->batch <= 0 || c->kv_heads <= 0 || c->num_pages <= 0 || c->newest_rows <= 0 || c->table_width <= 0)
    return B200_ERR_ARG;
  if (c->batch > ATTN8_MAX_BATCH || c->kv_heads > 1024) return B200_ERR_TILE;
  // positions are numbered in 32 bits
  if (static_cast<long long>(c->table_width) * c->page_size > 0x7fff0000LL) return B200_ERR_TILE;
  if (!al16(c->k_pages) || !al16(c->v_pages) || !al16(c->k_newest) || !al16(c->v_newest)) return B200_ERR_ALIGN;
  return B200_OK;
}

Kv8Cache cache8_of(const B200KvCache8* a) {
  Kv8Cache c{};
  c.k_pages = static_cast<uint8_t*>(a->k_pages);
  c.v_pages = static_cast<uint8_t*>(a->v_pages);
  c.k_scale = a->k_scale;
  c.v_scale = a->v_scale;
  c.k_new = static_cast<uint16_t*>(a->k_newest);
  c.v_new = static_cast<uint16_t*>(a->v_newest);
  c.table = a->table;
  c.rows = a->rows;
  c.num_pages = a->num_pages;
  c.kv_heads = a->kv_heads;
  c.page = a->page_size;
  c.head_dim = a->head_dim;
  c.new_rows = a->newest_rows;
  c.table_width = a->table_width;
  c.bf16 = a->bf16 != 0;
  c.page_shift = __builtin_ctz(a->page_size);
  c.dim_shift = __builtin_ctz(a->head_dim);
  return c;
}

int kv8_append_impl(const B200KvCache8* c, const void* qkv, long long ld, void* q_out, const int* cu, const int* start,
                    const float* cos, const float* sin, int rot, int interleaved, int rope_rows, int tokens, int heads,
                    cudaStream_t st) {
  if (int rc = cache8_check(c)) return rc;
  if (tokens < 0 || !cu || !start || heads <= 0 || heads % c->kv_heads) return B200_ERR_ARG;
  if (tokens == 0) return B200_OK;
  if (!qkv || !q_out || (cos == nullptr) != (sin == nullptr)) return B200_ERR_ARG;
  if (cos && (rot <= 0 || rot % 16 || rot > c->head_dim || rope_rows <= 0)) return B200_ERR_TILE;
  if (ld < static_cast<long long>(heads + 2 * c->kv_heads) * c->head_dim) return B200_ERR_ARG;
  if (!al16(qkv) || !al16(q_out) || !al16(cos) || !al16(sin) || ld % 8) return B200_ERR_ALIGN;
  const long long row = static_cast<long long>(heads) * c->head_dim * 2;
  if (overlap({q_out, tokens, row, row}, {qkv, tokens, ld * 2, row + 4LL * c->kv_heads * c->head_dim})) return B200_ERR_ARG;
  if (int rc = check_arch()) return rc;
  Kv8AppendParams p{};
  p.c = cache8_of(c);
  p.qkv = static_cast<const uint16_t*>(qkv);
  p.ld = ld;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.cu = cu;
  p.start = start;
  p.cos = cos;
  p.sin = sin;
  p.rot = cos ? rot : 0;
  p.interleaved = interleaved;
  p.rope_rows = rope_rows;
  p.tokens = tokens;
  p.batch = c->batch;
  p.heads = heads;
  const long long by_block = static_cast<long long>(tokens) / c->page_size + 2LL * c->batch;
  if (by_block > 0x7fffffffLL) return B200_ERR_TILE;
  p.by_token = tokens <= by_block;
  const unsigned units = static_cast<unsigned>(p.by_token ? tokens : by_block);
  const int tile = c->page_size * c->head_dim * 2;
  // heads a CTA: for single tokens one of K and V, and query heads that give its threads a unit each; for prompts as
  // many as leave every SM several CTAs and the tiles within 48 KB
  const int threads = p.by_token ? 128 : 256, per_row = c->head_dim / 8 - (interleaved ? 0 : p.rot / 16);
  const bool many = !p.by_token && by_block * c->kv_heads >= 16LL * num_sms();
  p.k_each = 1;
  while (many && p.k_each < 4 && 2 * p.k_each <= c->kv_heads && 2 * p.k_each * tile <= 48 * 1024) p.k_each *= 2;
  const int smem = p.k_each * tile;
  p.q_each = p.by_token ? std::max(1, threads / per_row) : many ? 8 : 4;
  p.row_recip = static_cast<unsigned>((0x100000000ull + per_row - 1) / per_row);
  p.q_recip = p.q_each > 1 ? static_cast<unsigned>((0x100000000ull + p.q_each - 1) / p.q_each) : 0;
  const unsigned slots = 2 * ((c->kv_heads + p.k_each - 1) / p.k_each) + (heads + p.q_each - 1) / p.q_each;
  if (slots > 65535) return B200_ERR_TILE;
  launch_kernel(p.c.bf16 ? k_kv8_append<true> : k_kv8_append<false>, dim3(units, slots), dim3(threads), smem, st, p);
  return launch_status();
}

int kv8_read_impl(const B200KvCache8* c, const int* cu, const int* start, const int* lens, void* k_out, void* v_out,
                  int tokens, cudaStream_t st) {
  if (int rc = cache8_check(c)) return rc;
  if (tokens < 0 || !cu || !start || !lens) return B200_ERR_ARG;
  if (tokens == 0) return B200_OK;
  if (!k_out || !v_out) return B200_ERR_ARG;
  if (!al16(k_out) || !al16(v_out)) return B200_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  Kv8ReadParams p{};
  p.c = cache8_of(c);
  p.cu = cu;
  p.start = start;
  p.lens = lens;
  p.k_out = static_cast<uint16_t*>(k_out);
  p.v_out = static_cast<uint16_t*>(v_out);
  p.tokens = tokens;
  p.batch = c->batch;
  const int per = 256 / (c->head_dim / 8);
  launch_kernel(p.c.bf16 ? k_kv8_read<true> : k_kv8_read<false>, dim3((tokens + per - 1) / per, c->kv_heads), dim3(256), 0, st, p);
  return launch_status();
}

// Rows of a tile: one column tile of 8 where a key head's rows fit it, else two.
int attn8_rows(int max_q_len, int group) { return static_cast<long long>(max_q_len) * group <= 8 ? 8 : 16; }
template <int D, int NT>
constexpr size_t attn8_slots() {  // floats of one SM's partial results
  using C = Attn8Cfg<D, NT>;
  return static_cast<size_t>(C::WARPS) * 2 * C::ROWS * (D + 2);
}

size_t attn8_workspace(int batch, int heads, int kv_heads, int head_dim, int max_q_len) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_q_len <= 0) return 0;
  const bool one = attn8_rows(max_q_len, heads / kv_heads) == 8;
  const size_t floats = head_dim == 32 ? (one ? attn8_slots<32, 1>() : attn8_slots<32, 2>())
                        : head_dim == 64 ? (one ? attn8_slots<64, 1>() : attn8_slots<64, 2>())
                                         : (one ? attn8_slots<128, 1>() : attn8_slots<128, 2>());
  return num_sms() * floats * sizeof(float) + (static_cast<size_t>(batch) + 1) * sizeof(int);
}

template <int D, int NT, bool SMALL>
int launch_attn8(Attn8Params& p, long long rows, cudaStream_t st) {
  using C = Attn8Cfg<D, NT>;
  const int ctas = std::min(num_sms(), 150);  // (the join kernel holds a part a CTA)
  p.warps = ctas * C::WARPS;
  p.plan = reinterpret_cast<int*>(p.part + ctas * attn8_slots<D, NT>());
  // Few tiles of short tables (at most four chunks a warp of a CTA) are a CTA's each, which adds up its parts itself:
  // no second kernel.  Measured (line against CTA, us on the device, one token a sequence): 1 x 1000 keys of 16 heads of
  // 64: 12.1, 8.4; 8 x 2000: 18.0, 11.2; 16 x 1000 (288 tiles): 19.5, 15.5; 16 x 1000 keys of 32/8 heads of 128: 19.1,
  // 11.1; past the bounds 1 x 4000: 13.2, 16.5; 32 x 1000 (576 tiles): 26.2, 28.9; 4 x 3000 of 32/8 heads: 17.3, 20.0.
  const long long tiles = (rows / C::ROWS + std::min(p.batch, p.tokens)) * p.c.kv_heads;
  const bool own = tiles <= 2 * ctas && static_cast<long long>(p.c.table_width) * p.c.page / ATTN8_CHUNK <= 4 * C::WARPS;
  static_assert(C::TOTAL + (ATTN8_MAX_BATCH + 1) * 4 + 128 <= 227 * 1024, "ring and line fit an SM");
  auto kern = own ? k_attn8<D, NT, SMALL, true> : k_attn8<D, NT, SMALL, false>;
  if (int rc = set_smem(reinterpret_cast<const void*>(kern), C::TOTAL + (ATTN8_MAX_BATCH + 1) * 4)) return rc;
  launch_kernel(kern, dim3(own ? static_cast<unsigned>(std::min<long long>(tiles, ctas)) : ctas), dim3(32 * C::WARPS),
                C::TOTAL + (p.batch + 1) * 4, st, p);
  if (int rc = launch_status()) return rc;
  if (own) return B200_OK;
  launch_kernel(k_attn8_join<D, NT>, dim3(static_cast<unsigned>(rows / C::ROWS + p.batch), p.c.kv_heads),
                dim3(ATTN8_JOIN_THREADS), 0, st, p);
  return launch_status();
}

template <int D>
int launch_attn8_tile(Attn8Params& p, long long rows, cudaStream_t st) {
  using C = Attn8TileCfg<D>;
  auto kern = k_attn8_tile<D>;
  constexpr int most = C::TOTAL + (ATTN8_MAX_BATCH + 1) * 4 + 1024;
  static_assert(most <= 227 * 1024, "tiles and line fit an SM");
  if (int rc = set_smem(reinterpret_cast<const void*>(kern), most)) return rc;
  const long long items = (rows / 256 + std::min(p.batch, p.tokens)) * p.c.kv_heads;
  launch_kernel(kern, dim3(static_cast<unsigned>(std::min<long long>(items, num_sms()))), dim3(C::THREADS),
                C::TOTAL + (p.batch + 1) * 4 + 1024, st, p);
  return launch_status();
}

// Whether the 256-row tcgen05 kernel is ahead of the warps' streams.  Its time goes by the waves of 256-row items
// over the SMs, theirs by the rows (new tokens times query heads); a wave takes as long as this many rows.  Measured
// (warps against tiles, us): 8192 rows over 8000 keys, D = 128: 222, 212; D = 64: 147, 165; D = 32: 117, 145;
// 16384 rows, D = 128: 425, 215; D = 64: 274, 166; 8 x 256 rows of 16 heads over 2000 keys, D = 32: 122, 49; 4096
// rows of D = 128: 123, 213.  The items are counted as if the sequences with new tokens had max_q_len each: sequences
// without any, the idle slots of a batch, count for nothing (1 token of 1 of 16 sequences, 8000 keys of 16 heads of 64:
// 14, 245).  One choice for the batch: single tokens beside a chunk that fills the tiles go with it.
bool attn8_many_rows(int tokens, int max_q_len, int group, int kv_heads, int head_dim) {
  const long long rows = static_cast<long long>(tokens) * group, each = std::min<long long>(static_cast<long long>(max_q_len) * group, rows);
  const long long busy = (static_cast<long long>(tokens) + max_q_len - 1) / max_q_len;
  const long long items = (each + 255) / 256 * busy * kv_heads, waves = (items + num_sms() - 1) / num_sms();
  return rows * kv_heads >= waves * (head_dim == 128 ? 8000 : 10000);
}

template <int D>
int launch_attn8_d(Attn8Params& p, bool one, bool many, long long rows, cudaStream_t st) {
  if (many) return launch_attn8_tile<D>(p, rows, st);
  if (p.c.page == 16) return one ? launch_attn8<D, 1, true>(p, rows, st) : launch_attn8<D, 2, true>(p, rows, st);
  return one ? launch_attn8<D, 1, false>(p, rows, st) : launch_attn8<D, 2, false>(p, rows, st);
}

int attn8_impl(const B200KvCache8* c, const void* q, long long ld_q, void* out, long long ld_out, const int* cu,
               const int* lens, int tokens, int heads, int max_q_len, float scale, void* ws, size_t ws_bytes,
               cudaStream_t st) {
  if (int rc = cache8_check(c)) return rc;
  if (tokens < 0 || !cu || !lens || heads <= 0 || heads % c->kv_heads || max_q_len < 0) return B200_ERR_ARG;
  if (tokens == 0) return B200_OK;
  if (!q || !out || max_q_len == 0) return B200_ERR_ARG;
  const long long width = static_cast<long long>(heads) * c->head_dim;
  if (ld_q < width || ld_out < width) return B200_ERR_ARG;
  if (!al16(q) || !al16(out) || ld_q % 8 || ld_out % 8) return B200_ERR_ALIGN;
  const int group = heads / c->kv_heads;
  const long long rows = static_cast<long long>(tokens) * group;
  // rows, and items of 256 rows and a key head, are numbered in 32 bits, and the warps' line of (sequence, head, row tile,
  // unit) work: what is too long for that goes to the 256-row kernel
  if (rows > 0x7fffffffLL || (rows / 256 + c->batch) * c->kv_heads > 0x7fffffffLL) return B200_ERR_TILE;
  const long long chunks = static_cast<long long>(c->table_width) * c->page_size / ATTN8_CHUNK + 1 + ATTN8_START + 8 * ATTN8_NEWEST;
  const bool many = (rows / 8 + c->batch) * c->kv_heads > 0x7fffffffLL / chunks ||
                    attn8_many_rows(tokens, max_q_len, group, c->kv_heads, c->head_dim);
  if (!ws || ws_bytes < attn8_workspace(c->batch, heads, c->kv_heads, c->head_dim, max_q_len)) return B200_ERR_WORKSPACE;
  // a row tile is written after it was read, so `out` may be q itself
  if ((out != q || (tokens > 1 && ld_out != ld_q)) && overlap({out, tokens, ld_out * 2, width * 2}, {q, tokens, ld_q * 2, width * 2}))
    return B200_ERR_ARG;
  if (!al16(ws)) return B200_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  Attn8Params p{};
  p.c = cache8_of(c);
  p.q = static_cast<const uint16_t*>(q);
  p.out = static_cast<uint16_t*>(out);
  p.ld_q = ld_q;
  p.ld_out = ld_out;
  p.cu = cu;
  p.lens = lens;
  p.tokens = tokens;
  p.batch = c->batch;
  p.heads = heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(ws);
  const bool one = attn8_rows(max_q_len, group) == 8;
  switch (c->head_dim) {
    case 32: return launch_attn8_d<32>(p, one, many, rows, st);
    case 64: return launch_attn8_d<64>(p, one, many, rows, st);
    default: return launch_attn8_d<128>(p, one, many, rows, st);
  }
}

// 8-bit [rows, cols] matrix with row pitch ld bytes: boxes of 128 bytes x box_rows, SWIZZLE_128B
int make_map_i8(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  return make_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, rows, cols, ld, 128, box_rows,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

long long i8_pitch(int K) { return (static_cast<long long>(K) + 15) / 16 * 16; }

bool lin_small_fits(int m, int k);

size_t linear_i8_workspace(int M, int K) {
  if (M <= 0 || K <= 0 || lin_small_fits(M, K)) return 0;
  return static_cast<size_t>(M) * i8_pitch(K) + static_cast<size_t>(M) * sizeof(float);
}

int quantize_rows_impl(const void* x, int x_type, long long ld_x, void* codes, long long ld_codes, float* scale, int m,
                       int k, cudaStream_t st) {
  if (x_type < 0 || x_type > 2) return B200_ERR_CONFIG;
  if (m < 0 || k <= 0 || ld_x < k || ld_codes < k) return B200_ERR_ARG;
  if (m == 0) return B200_OK;
  if (!x || !codes || !scale) return B200_ERR_ARG;
  if (int rc = check_arch()) return rc;
  const int vec = al16(x) && ld_x % (x_type == DT_F32 ? 4 : 8) == 0;
  auto run = [&](auto kern, int rows) {
    launch_kernel(kern, dim3((m + rows - 1) / rows), dim3(256), 0, st, x, ld_x, static_cast<int8_t*>(codes), ld_codes, scale,
                  m, k, vec);
    return launch_status();
  };
  // a warp a row where that makes CTAs enough, else a CTA a row
  if (k <= 2048 && m >= 2048) {
    if (x_type == DT_F16) return run(k_quant_rows<DT_F16, 32>, 8);
    if (x_type == DT_BF16) return run(k_quant_rows<DT_BF16, 32>, 8);
    return run(k_quant_rows<DT_F32, 32>, 8);
  }
  if (x_type == DT_F16) return run(k_quant_rows<DT_F16, 256>, 1);
  if (x_type == DT_BF16) return run(k_quant_rows<DT_BF16, 256>, 1);
  return run(k_quant_rows<DT_F32, 256>, 1);
}

template <int DT, int EPI>
int launch_gemm_i8(const GemmI8Params& p, const CUtensorMap& ta, const void* w, long long ld_w, cudaStream_t st) {
  CUtensorMap tw, to{};
  if (p.tma_out)
    if (int rc = make_map_2d(&to, DT == DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                             DT == DT_F32 ? 4 : 2, p.out, p.M, p.N, p.ld_out, I8Out<DT>::CC, 32, CU_TENSOR_MAP_SWIZZLE_64B))
      return rc;
  if (int rc = make_map_i8(&tw, w, p.N, p.K, ld_w, 128)) return rc;
  if (p.M >= 512 && p.N >= 256) {
    const long long tiles = static_cast<long long>((p.M + 255) / 256) * ((p.N + 255) / 256);
    if (tiles > 0x3fffffffLL) return B200_ERR_TILE;
    const dim3 grid(2 * static_cast<unsigned>(std::min<long long>(tiles, num_sms() / 2)));
    auto run = [&](auto kern, int ew, int smem) {
      if (int rc = set_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
      launch_kernel(kern, grid, dim3(64 + 32 * ew), smem, st, ta, tw, to, p);
      return launch_status();
    };
    // 16 epilogue warps where the epilogue sets the speed, GELU over a short K (quantizer included: 32768x1024x4096
    // 171 us, with 8 warps 178; 65536x256x1024 86 against 94), 8 and a deeper ring elsewhere (16384x2048x2048 GELU
    // 80 against 82; 32768x1024x4096 without GELU 145 against 149)
    if constexpr (EPI == I8_GELU)
      if (p.K <= 1024) return run(k_gemm2_i8<DT, EPI, 16>, 16, Gemm2I8Smem<16>::TOTAL);
    return run(k_gemm2_i8<DT, EPI, 8>, 8, Gemm2I8Smem<8>::TOTAL);
  }
  constexpr int BN = 128, STAGES = 5;
  using L = GemmI8Smem<BN, STAGES>;
  auto kern = k_gemm_i8<BN, STAGES, DT, EPI>;
  if (int rc = set_smem(reinterpret_cast<const void*>(kern), L::TOTAL)) return rc;
  const long long tiles = static_cast<long long>((p.M + 127) / 128) * ((p.N + BN - 1) / BN);
  if (tiles > 0x3fffffffLL) return B200_ERR_TILE;
  launch_kernel(kern, dim3(static_cast<unsigned>(std::min<long long>(tiles, num_sms()))), dim3(GEMM_THREADS), L::TOTAL, st,
                ta, tw, to, p);
  return launch_status();
}

// The one-kernel form for few rows: CTAs of a cluster split K, at most LIN_SLICES slices of 128 each.
bool lin_small_fits(int m, int k) { return m <= LIN_ROWS && k <= LIN_MAX_CLUSTER * LIN_SLICES * 128; }

int launch_lin_small(const GemmI8Params& g, const B200LinearI8Args* a, cudaStream_t st) {
  LinSmallParams p{};
  p.g = g;
  p.x = a->x;
  p.ldx = a->ld_x;
  p.vec = al16(a->x) && a->ld_x % (a->x_type == DT_F32 ? 4 : 8) == 0;
  p.out_type = a->out_type;
  p.epi = a->resid ? I8_RESID : a->gelu ? I8_GELU : I8_BIAS;
  p.pad = (a->m + 15) / 16 * 16;
  // as many CTAs a cluster as fill the SMs once, at least those that hold K
  const int tiles = (a->n + 127) / 128, all = (a->k + 127) / 128;
  p.cluster = 1;
  while (p.cluster < LIN_MAX_CLUSTER && p.cluster < all &&
         ((all + p.cluster - 1) / p.cluster > LIN_SLICES || 2LL * p.cluster * tiles <= num_sms()))
    p.cluster *= 2;
  p.slices = (all + p.cluster - 1) / p.cluster;
  if (static_cast<long long>(tiles) * p.cluster > 0x7fffffffLL) return B200_ERR_TILE;
  CUtensorMap tw;
  if (int rc = make_map_i8(&tw, a->w, a->n, a->k, a->ld_w, 128)) return rc;
  auto kern = a->x_type == DT_F16 ? k_lin_small<DT_F16> : a->x_type == DT_BF16 ? k_lin_small<DT_BF16> : k_lin_small<DT_F32>;
  const int smem = LinSmallSmem(p.pad, p.slices).total;
  if (int rc = set_smem(reinterpret_cast<const void*>(kern), LinSmallSmem(LIN_ROWS, LIN_SLICES).total)) return rc;
  launch_kernel_cluster(kern, dim3(static_cast<unsigned>(tiles * p.cluster)), dim3(p.pad == 16 ? 256 : 32 * LIN_MAX_WARPS),
                        smem, st,
                        static_cast<unsigned>(p.cluster), tw, p);
  return launch_status();
}

int linear_i8_impl(const B200LinearI8Args* a, cudaStream_t st) {
  if (!a || a->m < 0 || a->n <= 0 || a->k <= 0) return B200_ERR_ARG;
  if (a->x_type < 0 || a->x_type > 2 || a->out_type < 0 || a->out_type > 2) return B200_ERR_CONFIG;
  if (a->resid && (a->out_type != DT_F32 || a->gelu)) return B200_ERR_CONFIG;
  if (a->m == 0) return B200_OK;
  if (!a->x || !a->w || !a->w_scale || !a->out) return B200_ERR_ARG;
  if (a->ld_x < a->k || a->ld_w < a->k || a->ld_out < a->n || (a->resid && a->ld_resid < a->n)) return B200_ERR_ARG;
  if (a->ld_w % 16 || !al16(a->w)) return B200_ERR_ALIGN;
  // the sums are int32: |sum| <= 127 * 128 * k (a weight may use the code -128)
  if (a->k > 0x7fffffff / (127 * 128)) return B200_ERR_TILE;
  const bool few = lin_small_fits(a->m, a->k);
  if (!few && (!a->workspace || a->workspace_bytes < linear_i8_workspace(a->m, a->k))) return B200_ERR_WORKSPACE;
  // the epilogue reads an element of resid before it writes it, so `out` may be resid itself; x and w are read throughout
  const long long esize = a->out_type == DT_F32 ? 4 : 2, xsize = a->x_type == DT_F32 ? 4 : 2;
  const Rows8 out{a->out, a->m, a->ld_out * esize, a->n * esize};
  if (overlap(out, {a->x, a->m, a->ld_x * xsize, a->k * xsize}) || overlap(out, {a->w, a->n, a->ld_w, a->k}) ||
      overlap(out, {a->w_scale, 1, 0, 4LL * a->n}) || overlap(out, {a->bias, 1, 0, 4LL * a->n}))
    return B200_ERR_ARG;
  if ((a->resid != a->out || (a->m > 1 && a->ld_resid != a->ld_out)) && overlap(out, {a->resid, a->m, a->ld_resid * 4, 4LL * a->n}))
    return B200_ERR_ARG;
  if (!few && !al16(a->workspace)) return B200_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  GemmI8Params p{};
  p.M = a->m;
  p.N = a->n;
  p.K = a->k;
  p.sw = a->w_scale;
  p.bias = a->bias;
  p.resid = a->resid;
  p.ld_resid = a->ld_resid;
  p.vec_resid = a->resid && al16(a->resid) && a->ld_resid % 4 == 0;
  p.out = a->out;
  p.ld_out = a->ld_out;
  if (few) return launch_lin_small(p, a, st);
  const long long pitch = i8_pitch(a->k);
  int8_t* codes = static_cast<int8_t*>(a->workspace);
  float* sx = reinterpret_cast<float*>(codes + static_cast<size_t>(a->m) * pitch);
  if (int rc = quantize_rows_impl(a->x, a->x_type, a->ld_x, codes, pitch, sx, a->m, a->k, st)) return rc;
  CUtensorMap ta;
  if (int rc = make_map_i8(&ta, codes, a->m, a->k, pitch, 128)) return rc;
  p.sx = sx;
  p.tma_out = al16(a->out) && a->ld_out * (a->out_type == DT_F32 ? 4 : 2) % 16 == 0;
  auto go = [&](auto f) { return f(p, ta, a->w, a->ld_w, st); };
  if (a->resid) return go(launch_gemm_i8<DT_F32, I8_RESID>);
  if (a->out_type == DT_F32) return a->gelu ? go(launch_gemm_i8<DT_F32, I8_GELU>) : go(launch_gemm_i8<DT_F32, I8_BIAS>);
  if (a->out_type == DT_BF16) return a->gelu ? go(launch_gemm_i8<DT_BF16, I8_GELU>) : go(launch_gemm_i8<DT_BF16, I8_BIAS>);
  return a->gelu ? go(launch_gemm_i8<DT_F16, I8_GELU>) : go(launch_gemm_i8<DT_F16, I8_BIAS>);
}

}  // namespace

extern "C" {

int b200_kv8_append(const B200KvCache8* cache, const void* qkv, long long ld_qkv, void* q_out, const int* cu,
                    const int* start, const float* cos, const float* sin, int rot, int interleaved, int rope_rows,
                    int tokens, int heads, b200_stream_t stream) {
  return kv8_append_impl(cache, qkv, ld_qkv, q_out, cu, start, cos, sin, rot, interleaved, rope_rows, tokens, heads,
                         static_cast<cudaStream_t>(stream));
}

int b200_kv8_read(const B200KvCache8* cache, const int* cu, const int* start, const int* lens, void* k_out, void* v_out,
                  int tokens, b200_stream_t stream) {
  return kv8_read_impl(cache, cu, start, lens, k_out, v_out, tokens, static_cast<cudaStream_t>(stream));
}

size_t b200_kv8_attention_workspace_bytes(int batch, int heads, int kv_heads, int head_dim, int max_q_len) {
  return attn8_workspace(batch, heads, kv_heads, head_dim, max_q_len);
}

int b200_kv8_attention(const B200KvCache8* cache, const void* q, long long ld_q, void* out, long long ld_out,
                       const int* cu, const int* lens, int tokens, int heads, int max_q_len, float scale,
                       void* workspace, size_t workspace_bytes, b200_stream_t stream) {
  return attn8_impl(cache, q, ld_q, out, ld_out, cu, lens, tokens, heads, max_q_len, scale, workspace, workspace_bytes,
                    static_cast<cudaStream_t>(stream));
}

int b200_quantize_rows_i8(const void* x, int x_type, long long ld_x, void* codes, long long ld_codes, float* scale,
                          int m, int k, b200_stream_t stream) {
  return quantize_rows_impl(x, x_type, ld_x, codes, ld_codes, scale, m, k, static_cast<cudaStream_t>(stream));
}

size_t b200_linear_i8_workspace_bytes(int m, int k) { return linear_i8_workspace(m, k); }

int b200_linear_i8(const B200LinearI8Args* args, b200_stream_t stream) {
  return linear_i8_impl(args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
