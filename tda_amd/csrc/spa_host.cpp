// spa_host.cpp -- C ABI of the paged cache (include/spa.h): argument validation, buffer sizing and
// dispatch.  Every argument that lies in host memory is checked here before any launch; page numbers,
// lengths, starts and counts in device memory are clamped by the kernels.
#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "../../include/spa.h"
#include "spa_params.hpp"

namespace {

constexpr int64_t kMaxPos = (int64_t(1) << 30) - 64;  // positions and row counts stay in int32
constexpr int64_t kMaxRowBytes = int64_t(1) << 25;
constexpr int64_t kMaxStride = int64_t(1) << 50;      // elements: offsets of whole tensors stay in int64
constexpr double kLog2e = 1.4426950408889634074;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool any_dtype(int32_t t) { return t == TDA_DTYPE_F32 || t == TDA_DTYPE_BF16 || t == SDA_DTYPE_F16; }
int64_t bytes_of(int32_t dtype) { return dtype == TDA_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A (lead, H, rows, width) tensor whose rows the kernels read in 16-byte pieces.
int32_t check_rows(const tda_tensor& t, int64_t es) {
  if (!t.data) return TDA_ERR_NULL_POINTER;
  if (t.stride[3] != 1 || !aligned(t.data, 16)) return TDA_ERR_LAYOUT;
  for (int k = 0; k < 3; ++k)
    if (t.stride[k] < 0 || t.stride[k] > kMaxStride || (t.stride[k] * es) % 16) return TDA_ERR_LAYOUT;
  return t.stride[2] * es > kMaxRowBytes ? TDA_ERR_LAYOUT : TDA_OK;
}
int32_t check_cache_sizes(const spa_cache& c) {
  const bool dims = (c.head_dim == 64 && (c.v_head_dim == 64 || c.v_head_dim == 128)) ||
                    (c.head_dim == 128 && (c.v_head_dim == 128 || c.v_head_dim == 256));
  if (!dims) return TDA_ERR_HEAD_DIM;
  if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1))) return SPA_ERR_PAGES;
  if (c.pages < 1 || c.pages > kMaxPos) return SPA_ERR_PAGES;
  if (c.kv_heads < 1 || c.kv_heads > (1 << 20)) return TDA_ERR_SHAPE;
  // a page's heads are counted in 32 bits
  return c.pages * c.kv_heads > kMaxPos || (double)c.pages * c.kv_heads * c.page_size * c.v_head_dim > (double)kMaxStride ? SPA_ERR_PAGES : TDA_OK;
}
int32_t check_cache(const spa_cache& c) {
  if (int32_t rc = check_cache_sizes(c)) return rc;
  for (const void* p : {c.k1, c.k2, c.v}) {
    if (!p) return TDA_ERR_NULL_POINTER;
    if (!aligned(p, 16)) return TDA_ERR_LAYOUT;
  }
  return TDA_OK;
}
int32_t check_at_sizes(const spa_rows& r) {
  return r.sequences < 1 || r.rows < 1 || r.sequences > kMaxPos || r.rows > kMaxPos ? TDA_ERR_SHAPE : TDA_OK;
}
int32_t check_at(const spa_rows& r, const spa_cache& c) {
  if (int32_t rc = check_at_sizes(r)) return rc;
  if (r.starts && r.counts) return SPA_ERR_ROWS;
  if (!r.table || !r.lengths) return TDA_ERR_NULL_POINTER;
  if (r.table_len < 1 || r.table_len > kMaxPos / c.page_size || r.table_stride < 0 || r.table_stride > kMaxStride) return SPA_ERR_PAGES;
  for (const void* p : {r.table, r.lengths, r.starts, r.counts})
    if (!aligned(p, 4)) return TDA_ERR_LAYOUT;
  return TDA_OK;
}

sda::Rows rows_of(const tda_tensor& t) { return {t.data, t.stride[0], t.stride[1], t.stride[2]}; }
spa::Seqs seqs_of(const spa_rows& r, const spa_cache& c) {
  spa::Seqs q;
  q.table = r.table;
  q.lengths = r.lengths;
  q.starts = r.starts;
  q.counts = r.counts;
  q.tstride = r.table_stride;
  q.tlen = (int)r.table_len;
  q.S = (int)r.sequences;
  q.rows = (int)r.rows;
  q.pages = (int)c.pages;
  for (q.pshift = 4; (1 << q.pshift) < c.page_size; ++q.pshift) {}
  return q;
}
int64_t lead_of(const spa_rows& r) { return r.starts ? 1 : r.sequences; }
int32_t done(int e) {
  const int te = tda::timing_end();
  if (e == 0) e = te;
  if (e == 0) return TDA_OK;
  tda::record_hip_error(e);
  return TDA_ERR_HIP;
}

// A launch lays its workgroups out over two grid axes; their number stays in 32 bits.
bool fits_grid(double blocks) { return blocks < 2147483647.0; }

int32_t check_attend_sizes(const spa_attend_args& a) {
  if (int32_t rc = check_cache_sizes(a.cache)) return rc;
  if (int32_t rc = check_at_sizes(a.at)) return rc;
  if (a.heads < 1 || a.heads > (1 << 20) || a.most < 0) return TDA_ERR_SHAPE;
  if (a.heads % a.cache.kv_heads) return SDA_ERR_HEADS;
  // rows of the heads that share a key head are counted in 32 bits, tiles of 16 of them are workgroups
  const double group = (double)(a.heads / a.cache.kv_heads);
  const double per = a.at.starts ? 1.0 : (double)a.at.sequences;
  return group * a.at.rows <= kMaxPos && fits_grid(((group * a.at.rows / 16.0 + 1) * per + a.at.sequences) * a.cache.kv_heads * 8.0)
             ? TDA_OK
             : TDA_ERR_SHAPE;
}

// Workgroups that share a call's tiles where these are fewer: one a CU.
constexpr int64_t kTarget = 256;

// What 128 keys of 128 rows cost next to 128 keys of 16: products and exponentials against bytes.  One long chunk among
// tokens of 23 to 39 sequences behind up to 3000 to 5000, µs at the cost taken and at those beside it: bf16 (64, 64) 81 (86 at 1, 101 at 3),
// (64, 128) 85 (94, 88), (128, 128) 130 (138 at 2), (128, 256) 162 (182 at 2); fp32 (64, 64) 118 (134 at 4, 140 at 8), (128, 128) 242 (279, 263),
// (128, 256) 575 (694 at 6).
int cost_of(int32_t dtype, int64_t d, int64_t dv) {
  if (dtype == TDA_DTYPE_F32) return dv == 256 ? 4 : 6;
  return d == 64 ? 2 : 1;
}

void deal(const spa_attend_args& a, spa::AttendParams& p) {
  const int64_t G = a.heads / a.cache.kv_heads, S = a.at.sequences, hk = a.cache.kv_heads, rows = a.at.rows, dv = a.cache.v_head_dim;
  const bool exact = !a.at.starts && !a.at.counts;  // every sequence has `rows` rows
  const int64_t most = !exact && a.most && a.most < rows ? a.most : rows;
  const int64_t total = (a.at.starts ? 1 : S) * rows * G;  // rows of all sequences, of the heads of a key head
  int64_t few = 0, many = 0;                         // tiles at most
  if (most * G <= spa::kFewRows) {
    p.bound = 0x7fffffff;  // every sequence has small tiles, however many rows it has after all
    few = a.at.starts ? total / spa::kFewRows + (S < total ? S : total) : S * ceil_div(rows * G, spa::kFewRows);
  } else if (exact) {
    p.bound = 0;
    many = S * ceil_div(rows * G, spa::kManyRows);
  } else {
    p.bound = spa::kFewRows;
    few = S < total ? S : total;
    const int64_t big = total / (spa::kFewRows + 1);  // sequences with more rows than that
    many = total / spa::kManyRows + (S < big ? S : big);
  }
  // whether there are few enough tiles to be cut: known of an exact call, else taken to be so when whole tiles of all rows
  // would be
  const int64_t tiles = many ? (exact ? many : total / spa::kManyRows) : ceil_div(total / spa::kFewRows, 8);
  // Small tiles over short tables are taken whole: what the joining launch costs, six microseconds, their other keys cost too from about 1024
  // on (newest tokens of 8 x 250, (16 over 4 heads, 128): 13.0 us, cut 18.2; 8 x 500: 16.7, 18.5; 2 x 1000: 17.7, 18.1).
  const bool brief = !many && a.at.table_len < 1024 / a.cache.page_size;
  // ... or too many by so few that a last round of them leaves CUs idle; how full the rounds are is known of an exact call
  const int64_t all = tiles * hk, rounds = ceil_div(all, kTarget);
  const bool ragged = many && all <= 3 * kTarget && (!exact || 4 * all < 3 * rounds * kTarget);
  const bool cut = (4 * all <= 3 * kTarget || ragged) && hk <= kTarget && !brief;
  p.room = cut ? (int)(kTarget / hk) : 0;
  const int64_t most_tiles = few + many;
  p.grid = (uint32_t)(hk * (most_tiles > p.room ? most_tiles : p.room));
  p.join[0] = cut ? (uint32_t)(few * hk) : 0;
  p.join[1] = cut ? (uint32_t)(many * hk * (spa::kManyRows / 32)) : 0;
  p.join_rows = (int)(exact && rows * G < spa::kFewRows ? rows * G : spa::kFewRows);
  p.cost = cost_of(a.dtype, a.cache.head_dim, dv);
  p.stride = many ? spa::many_floats(dv) : spa::few_floats(dv);
}
int64_t part_bytes(const spa::AttendParams& p, int64_t hk) { return 2 * p.room * hk * p.stride * 4; }

}  // namespace

extern "C" {

int32_t spa_abi_version(void) { return SPA_ABI_VERSION; }

const char* spa_error_string(int32_t code) {
  switch (code) {
    case SPA_ERR_PAGES: return "pages: page_size must be 16, 32, 64, 128 or 256, and pages and table_len page_size at least 1 and below 2^30 - 64";
    case SPA_ERR_ROWS: return "starts and counts exclude each other";
    case TDA_ERR_LAYOUT: return "rows must have a unit last stride, 16-byte alignment and at most 2^25 bytes between them, pages 16-byte alignment";
    case TDA_ERR_ABI: return "abi_version does not match SPA_ABI_VERSION";
    default: return sda_error_string(code);
  }
}

int32_t spa_validate_append(const spa_append_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SPA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (int32_t rc = check_cache(a->cache)) return rc;
  if (int32_t rc = check_at(a->at, a->cache)) return rc;
  if (a->heads < 0 || a->heads > (1 << 20)) return TDA_ERR_SHAPE;
  // a workgroup has at least one token, and a token at most its rows
  if (!fits_grid((double)lead_of(a->at) * a->at.rows * (2.0 * a->heads + 3.0 * a->cache.kv_heads))) return TDA_ERR_SHAPE;
  const int64_t es = bytes_of(a->dtype);
  for (const tda_tensor* t : {&a->k1, &a->k2, &a->v})
    if (int32_t rc = check_rows(*t, es)) return rc;
  if (a->heads)
    for (const tda_tensor* t : {&a->q1, &a->q2, &a->q1_out, &a->q2_out})
      if (int32_t rc = check_rows(*t, es)) return rc;
  if (a->rot < 0 || a->rot % 2 || a->rot > a->cache.head_dim) return SDA_ERR_AXES;
  if (!a->rot) return TDA_OK;
  if (a->axes < 1 || a->axes > SDA_MAX_AXES) return SDA_ERR_AXES;
  int64_t pairs = 0;
  for (int k = 0; k < a->axes; ++k) {
    if (a->sections[k] < 0) return SDA_ERR_AXES;
    pairs += a->sections[k];
  }
  if (pairs != a->rot / 2) return SDA_ERR_AXES;
  if (!a->inv_freq) return TDA_ERR_NULL_POINTER;
  if (!aligned(a->inv_freq, 4)) return TDA_ERR_LAYOUT;
  if (!a->positions) return TDA_OK;
  if (a->position_dtype != 4 && a->position_dtype != 8) return TDA_ERR_DTYPE;
  if (!aligned(a->positions, a->position_dtype)) return TDA_ERR_LAYOUT;
  for (int64_t s : a->position_stride)
    if (s < 0 || s > kMaxStride) return TDA_ERR_LAYOUT;
  return TDA_OK;
}

int32_t spa_append(const spa_append_args* a, void* stream) {
  if (int32_t rc = spa_validate_append(a)) return rc;
  spa::AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.seq = seqs_of(a->at, a->cache);
  p.pool[0] = a->cache.k1;
  p.pool[1] = a->cache.k2;
  p.pool[2] = a->cache.v;
  p.x[0] = rows_of(a->k1);
  p.x[1] = rows_of(a->k2);
  p.x[2] = rows_of(a->v);
  p.Hk = (int)a->cache.kv_heads;
  p.H = (int)a->heads;
  p.D = (int)a->cache.head_dim;
  p.DV = (int)a->cache.v_head_dim;
  p.lead = (int)lead_of(a->at);
  if (p.H) {
    p.q[0] = rows_of(a->q1);
    p.q[1] = rows_of(a->q2);
    p.qo[0] = rows_of(a->q1_out);
    p.qo[1] = rows_of(a->q2_out);
  }
  p.pairs = (int)(a->rot / 2);
  if (p.pairs) {
    int upto = 0;
    for (int k = 0; k < a->axes; ++k) p.upto[k] = upto += a->sections[k];
    p.axes = a->axes;
    p.inter = a->interleaved ? 1 : 0;
    p.inv_freq = a->inv_freq;
    p.pos = a->positions;
    for (int k = 0; k < 3; ++k) p.ps[k] = a->positions ? a->position_stride[k] : 0;
    p.pos64 = a->position_dtype == 8;
  }
  tda::timing_begin(stream);
  return done(spa::launch_append(p, a->dtype, stream));
}

size_t spa_attend_workspace_bytes(const spa_attend_args* a) {
  if (!a || check_attend_sizes(*a)) return 0;
  spa::AttendParams p;
  std::memset(&p, 0, sizeof(p));
  deal(*a, p);
  return (size_t)part_bytes(p, a->cache.kv_heads);
}

int32_t spa_validate_attend(const spa_attend_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SPA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (int32_t rc = check_cache(a->cache)) return rc;
  if (int32_t rc = check_at(a->at, a->cache)) return rc;
  if (!(a->scale >= 1e-30f && a->scale <= 1e30f)) return SDA_ERR_SCALE;
  if (int32_t rc = check_attend_sizes(*a)) return rc;
  if (!a->lambda_param) return TDA_ERR_NULL_POINTER;
  if (!any_dtype(a->lambda_dtype)) return TDA_ERR_DTYPE;
  for (int64_t s : a->lambda_stride)
    if (s < 0 || s > kMaxStride) return TDA_ERR_LAYOUT;
  if (!aligned(a->lambda_param, (uintptr_t)bytes_of(a->lambda_dtype))) return TDA_ERR_LAYOUT;
  for (const tda_tensor* t : {&a->q1, &a->q2, &a->out})
    if (int32_t rc = check_rows(*t, bytes_of(a->dtype))) return rc;
  const size_t need = spa_attend_workspace_bytes(a);
  return need && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)) ? TDA_ERR_WORKSPACE : TDA_OK;
}

int32_t spa_attend(const spa_attend_args* a, void* stream) {
  if (int32_t rc = spa_validate_attend(a)) return rc;
  spa::AttendParams p;
  std::memset(&p, 0, sizeof(p));
  deal(*a, p);
  p.seq = seqs_of(a->at, a->cache);
  p.k[0] = a->cache.k1;
  p.k[1] = a->cache.k2;
  p.v = a->cache.v;
  p.q[0] = rows_of(a->q1);
  p.q[1] = rows_of(a->q2);
  p.out = rows_of(a->out);
  p.lam = {a->lambda_param, a->lambda_stride[0], a->lambda_stride[1], a->lambda_stride[2], a->lambda_dtype};
  p.H = (int)a->heads;
  p.Hk = (int)a->cache.kv_heads;
  p.lead = (int)lead_of(a->at);
  p.c = (float)(a->scale * kLog2e);
  if (p.room) p.part = static_cast<float*>(a->workspace);
  tda::timing_begin(stream);
  return done(spa::launch_attend(p, a->dtype, (int)a->cache.head_dim, (int)a->cache.v_head_dim, stream));
}

}  // extern "C"
