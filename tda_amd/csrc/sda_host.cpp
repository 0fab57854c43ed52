// sda_host.cpp -- C ABI of the softmax differential attention operators (include/sda.h): argument
// validation, buffer sizing and dispatch.  Every argument that lies in host memory is checked here
// before any launch; lengths and offsets in device memory are clamped by the kernels.
#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "../../include/sda.h"
#include "sda_params.hpp"

namespace {

constexpr int64_t kMaxPos = (int64_t(1) << 30) - 64;      // positions and row counts stay in int32
constexpr int64_t kMaxRowBytes = int64_t(1) << 25;        // a tile of 64 rows spans at most 2^31 bytes
constexpr int64_t kMaxCapacity = int64_t(1) << 24;        // a head's codes stay within 32-bit offsets
constexpr int64_t kMaxStride = int64_t(1) << 50;          // elements: offsets of whole tensors stay in int64
constexpr double kLog2e = 1.4426950408889634074;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
bool any_dtype(int32_t t) { return t == TDA_DTYPE_F32 || t == TDA_DTYPE_BF16 || t == SDA_DTYPE_F16; }
int64_t bytes_of(int32_t dtype) { return dtype == TDA_DTYPE_F32 ? 4 : 2; }

// A (B, H, N, width) tensor whose rows the kernels read in 16-byte pieces (fine: any alignment of
// whole elements).
int32_t check_rows(const tda_tensor& t, int64_t es, bool fine = false) {
  if (!t.data) return TDA_ERR_NULL_POINTER;
  if (t.stride[3] != 1) return TDA_ERR_LAYOUT;
  const int64_t unit = fine ? es : 16;
  if (reinterpret_cast<uintptr_t>(t.data) % unit != 0) return TDA_ERR_LAYOUT;
  for (int k = 0; k < 3; ++k) {
    if (t.stride[k] < 0 || t.stride[k] > kMaxStride) return TDA_ERR_LAYOUT;
    if ((t.stride[k] * es) % unit != 0) return TDA_ERR_LAYOUT;
  }
  return t.stride[2] * es > kMaxRowBytes ? TDA_ERR_LAYOUT : TDA_OK;
}
bool head_dims(int64_t d, int64_t dv) {
  return (d == 64 && (dv == 64 || dv == 128)) || (d == 128 && (dv == 128 || dv == 256));
}
int32_t check_lambda(const void* p, const int64_t (&s)[3], int32_t dtype) {
  if (!p) return TDA_ERR_NULL_POINTER;
  if (!any_dtype(dtype)) return TDA_ERR_DTYPE;
  for (int64_t x : s)
    if (x < 0 || x > kMaxStride) return TDA_ERR_LAYOUT;
  return reinterpret_cast<uintptr_t>(p) % bytes_of(dtype) ? TDA_ERR_LAYOUT : TDA_OK;
}
// The kernels take scale log2(e) and its reciprocal in 32 bits.
bool check_scale(float s) { return s >= 1e-30f && s <= 1e30f; }
// Optional arrays of 4-byte elements.
int32_t check_words(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 4) return TDA_ERR_LAYOUT;
  return TDA_OK;
}
int32_t check_workspace(const void* p, size_t have, size_t need) {
  if (!need) return TDA_OK;
  return !p || have < need || reinterpret_cast<uintptr_t>(p) % 16 ? TDA_ERR_WORKSPACE : TDA_OK;
}
// A launch lays its workgroups out over two grid axes of at most 2^32 work-items each.
bool fits_grid(double blocks) { return blocks < 4294967295.0; }

// What the buffer sizes depend on.
template <class A>
int32_t check_sizes(const A& a) {
  if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.seq_len < 1 || a.seq_len_kv < 1) return TDA_ERR_SHAPE;
  if (a.heads % a.kv_heads) return SDA_ERR_HEADS;
  if (!head_dims(a.head_dim, a.v_head_dim)) return TDA_ERR_HEAD_DIM;
  if (a.batch > kMaxPos || a.heads > kMaxPos || a.batch * a.heads > kMaxPos) return TDA_ERR_SHAPE;
  if (a.seq_len > kMaxPos || a.seq_len_kv > kMaxPos) return TDA_ERR_OFFSET;
  // the most workgroups that any launch of the operator takes: one per 16 rows or keys and column group
  return fits_grid((double)a.batch * a.heads * ((double)a.seq_len + a.seq_len_kv + 32) / 16.0 * (a.v_head_dim / 16.0))
             ? TDA_OK
             : TDA_ERR_SHAPE;
}
template <class A>
int32_t check_common(const A& a) {
  if (a.abi_version != SDA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a.dtype)) return TDA_ERR_DTYPE;
  if (a.causal != 0 && a.causal != 1) return TDA_ERR_CAUSAL;
  if (!check_scale(a.scale)) return SDA_ERR_SCALE;
  if (int32_t rc = check_sizes(a)) return rc;
  if (!a.q_offsets && (a.q_offset < -kMaxPos || a.q_offset > kMaxPos - a.seq_len)) return TDA_ERR_OFFSET;
  if (int32_t rc = check_words({a.q_offsets, a.kv_lens, a.lse})) return rc;
  return check_lambda(a.lambda_param, a.lambda_stride, a.lambda_dtype);
}

// What a training forward keeps for the backward.
template <class A>
int32_t check_kept(const A& a) {
  if (int32_t rc = check_rows(a.out2, 4)) return rc;
  return a.dtype == TDA_DTYPE_F32 ? TDA_OK : check_rows(a.out_low, 2);
}

sda::Rows rows_of(const tda_tensor& t) { return {t.data, t.stride[0], t.stride[1], t.stride[2]}; }
sda::Lambda lambda_of(const void* p, const int64_t (&s)[3], int32_t dtype) {
  return {p, s[0], s[1], s[2], dtype};
}

// Few query rows go to the kernels that cut the key axis and read it once per 16 rows of the heads that share
// a key head (a tile): where one tile holds them all, where 64 tiles are all there is, or where the other
// form would read the keys twice as often, once per 128 rows of each query head.  bf16, widths of 128, us, these
// kernels : the others, (batch, heads, kv_heads, rows, keys):
//   (16, 32, 32, 16, 4096) 316 : 352    (16, 32, 32, 32, 4096) 469 : 338    (1, 32, 32, 32, 4096) 52 : 87
//   (1, 16, 4, 8, 4096) 20 : 67         (1, 16, 4, 64, 4096) 52 : 68        (1, 16, 4, 256, 4096) 103 : 69
//   (32, 32, 8, 8, 8192) 495 : 1040     (32, 32, 8, 16, 8192) 938 : 1028    (4, 32, 8, 16, 1024) 44 : 25
//   (64, 64, 1, 4, 8192) 548 : 3390     (4, 16, 4, 64, 2048) 69 : 40        (1, 8, 8, 64, 512) 15 : 17
bool few_rows(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len) {
  const int64_t g = heads / kv_heads, tiles = ceil_div(g * seq_len, 16);
  return tiles == 1 || batch * kv_heads * tiles <= 64 || 2 * tiles <= g * ceil_div(seq_len, 128);
}

int64_t dec_items(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len) {
  return batch * kv_heads * ceil_div(heads / kv_heads * seq_len, 16);
}
// Parts of the key axis: whole tiles of the four waves (128 keys) each, about `target` workgroups in all,
// no part shorter than 128 keys.
void dec_split(int64_t items, int64_t nk, int64_t target, int* nsplit, int* chunk) {
  int64_t want = ceil_div(target, items);
  const int64_t most = ceil_div(nk, 128);
  if (want > most) want = most;
  *chunk = (int)(ceil_div(ceil_div(nk, want), 128) * 128);
  *nsplit = (int)ceil_div(nk, *chunk);
}
// 1024 workgroups over a bf16 or f32 cache, 512 over the 4-bit one, whose kernel holds two to a CU: one
// token over (32, 32 over 8, 8192, 128) of unequal lengths takes 256 us (2048: 274, 4096: 275) and 103 us
// (768: 118, 1024: 112, 2048: 124).
constexpr int64_t kDecTarget = 1024, kKv4Target = 512;
int64_t dec_bytes(int64_t items, int nsplit, int64_t dv) {
  return nsplit > 1 ? items * nsplit * (64 + 32 * dv) * 4 : 0;
}

bool decodes(const sda_fwd_args& a) {
  return !a.out2.data && !a.lse && few_rows(a.batch, a.heads, a.kv_heads, a.seq_len);
}

// Query heads that a workgroup of the key pass sums over: all that share a key head, or fewer where
// that leaves under 512 workgroups (two a CU; causal ones are of unequal length).  Backward of bf16 (B, 16 over
// 4, 4096, 128): B = 2 1031 us (all four 1017, one 1033), B = 4 1923 (one 2001), B = 1 552 (all 760); (1, 32 over
// 1, 4096, 128) 957 us (at least 1024 workgroups 993, all 4468).
int64_t key_group(const sda_bwd_args& a) {
  const int64_t G = a.heads / a.kv_heads, base = a.batch * a.kv_heads * ceil_div(a.seq_len_kv, 128);
  for (int64_t gs = G; gs > 1; --gs)
    if (G % gs == 0 && base * (G / gs) >= 512) return gs;
  return 1;
}
int64_t peak_bytes(const sda_bwd_args& a) { return a.dtype == SDA_DTYPE_F16 ? 256 : 0; }
int64_t stat_bytes(const sda_bwd_args& a) { return round256(6 * a.batch * a.heads * a.seq_len * 4) + peak_bytes(a); }
int64_t part_bytes(const sda_bwd_args& a) {
  const int64_t G = a.heads / a.kv_heads, gs = key_group(a);
  return gs == G ? 0 : G / gs * a.batch * a.kv_heads * a.seq_len_kv * (2 * a.head_dim + a.v_head_dim) * 4;
}

template <class A, class P>
void fill(P& p, const A& a) {
  const tda_tensor *q[2] = {&a.q1, &a.q2}, *k[2] = {&a.k1, &a.k2};
  for (int x = 0; x < 2; ++x) {
    p.q[x] = rows_of(*q[x]);
    p.k[x] = rows_of(*k[x]);
  }
  p.v = rows_of(a.v);
  p.out = rows_of(a.out);
  p.out2 = rows_of(a.out2);
  p.low = rows_of(a.out_low);
  p.lam = lambda_of(a.lambda_param, a.lambda_stride, a.lambda_dtype);
  p.see = {a.causal, (int)(a.q_offsets ? 0 : a.q_offset), a.q_offsets, a.kv_lens};
  p.B = (int)a.batch;
  p.H = (int)a.heads;
  p.Hk = (int)a.kv_heads;
  p.Nq = (int)a.seq_len;
  p.Nk = (int)a.seq_len_kv;
  p.c = (float)(a.scale * kLog2e);
}

int32_t check_cache_sizes(const sda_kv4& c) {
  if (c.batch < 1 || c.kv_heads < 1 || c.capacity < 1) return TDA_ERR_SHAPE;
  if (!head_dims(c.head_dim, c.v_head_dim)) return TDA_ERR_HEAD_DIM;
  if (c.capacity > kMaxCapacity || c.batch > kMaxPos || c.kv_heads > kMaxPos || c.batch * c.kv_heads > kMaxPos) return SDA_ERR_CACHE;
  if (!fits_grid((double)c.batch * c.kv_heads * c.capacity * c.v_head_dim / 2048.0)) return SDA_ERR_CACHE;
  return TDA_OK;
}
int32_t check_cache(const sda_kv4& c) {
  if (int32_t rc = check_cache_sizes(c)) return rc;
  if (!c.k1 || !c.k2 || !c.v || !c.lengths) return TDA_ERR_NULL_POINTER;
  for (const void* p : {c.k1, c.k2, c.v})
    if (reinterpret_cast<uintptr_t>(p) % 16) return TDA_ERR_LAYOUT;
  return reinterpret_cast<uintptr_t>(c.lengths) % 4 ? TDA_ERR_LAYOUT : TDA_OK;
}
void fill_cache(sda::Kv4Params& p, const sda_kv4& c) {
  void* at[3] = {c.k1, c.k2, c.v};
  for (int z = 0; z < 3; ++z) {
    const int64_t w = z < 2 ? c.head_dim : c.v_head_dim;
    p.codes[z] = static_cast<uint8_t*>(at[z]);
    p.pars[z] = reinterpret_cast<uint32_t*>(p.codes[z] + c.batch * c.kv_heads * ceil_div(c.capacity, 4) * 4 * (w / 2));
  }
  p.lengths = c.lengths;
  p.B = (int)c.batch;
  p.Hk = (int)c.kv_heads;
  p.cap = (int)c.capacity;
  p.cap4 = ceil_div(c.capacity, 4) * 4;
  p.D = (int)c.head_dim;
  p.DV = (int)c.v_head_dim;
}
int32_t done(int e) {
  const int te = tda::timing_end();
  if (e == 0) e = te;
  if (e == 0) return TDA_OK;
  tda::record_hip_error(e);
  return TDA_ERR_HIP;
}

}  // namespace

extern "C" {

int32_t sda_abi_version(void) { return SDA_ABI_VERSION; }

const char* sda_error_string(int32_t code) {
  switch (code) {
    case SDA_ERR_HEADS: return "heads must be a multiple of kv_heads";
    case SDA_ERR_SCALE: return "scale must be finite and positive (1e-30 to 1e30)";
    case SDA_ERR_AXES: return "axes, sections or rotated width out of range";
    case SDA_ERR_CACHE: return "4-bit cache: capacity, lengths or row count out of range, or start or counts overlapping lengths";
    case TDA_ERR_HEAD_DIM: return "(head_dim, v_head_dim) must be (64, 64), (64, 128), (128, 128) or (128, 256)";
    case TDA_ERR_CAUSAL: return "causal must be 0 or 1";
    case TDA_ERR_LAYOUT: return "rows must have a unit last stride, 16-byte alignment and at most 2^25 bytes between them, and those of q1, q2 and dout of a backward may not overlap";
    case TDA_ERR_OFFSET: return "seq_len, seq_len_kv and q_offset + seq_len must stay below 2^30 - 64";
    case TDA_ERR_ABI: return "abi_version does not match SDA_ABI_VERSION";
    default: return tda_error_string(code);
  }
}

size_t sda_fwd_workspace_bytes(const sda_fwd_args* a) {
  if (!a || check_sizes(*a) || !decodes(*a)) return 0;
  int nsplit, chunk;
  const int64_t items = dec_items(a->batch, a->heads, a->kv_heads, a->seq_len);
  dec_split(items, a->seq_len_kv, kDecTarget, &nsplit, &chunk);
  return (size_t)dec_bytes(items, nsplit, a->v_head_dim);
}

int32_t sda_validate_fwd(const sda_fwd_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (int32_t rc = check_common(*a)) return rc;
  const int64_t es = bytes_of(a->dtype);
  for (const tda_tensor* t : {&a->q1, &a->k1, &a->q2, &a->k2, &a->v, &a->out})
    if (int32_t rc = check_rows(*t, es)) return rc;
  if (a->out2.data)
    if (int32_t rc = check_kept(*a)) return rc;
  return check_workspace(a->workspace, a->workspace_bytes, sda_fwd_workspace_bytes(a));
}

int32_t sda_fwd(const sda_fwd_args* a, void* stream) {
  if (int32_t rc = sda_validate_fwd(a)) return rc;
  sda::FwdParams p;
  std::memset(&p, 0, sizeof(p));
  fill(p, *a);
  p.lse = a->lse;
  tda::timing_begin(stream);
  if (decodes(*a)) {
    dec_split(dec_items(a->batch, a->heads, a->kv_heads, a->seq_len), a->seq_len_kv, kDecTarget, &p.nsplit, &p.chunk);
    p.part = static_cast<float*>(a->workspace);
    return done(sda::launch_decode(p, a->dtype, (int)a->head_dim, (int)a->v_head_dim, stream));
  }
  return done(sda::launch_fwd(p, a->dtype, (int)a->head_dim, (int)a->v_head_dim, stream));
}

size_t sda_bwd_workspace_bytes(const sda_bwd_args* a) {
  if (!a || check_sizes(*a)) return 0;
  return (size_t)(stat_bytes(*a) + part_bytes(*a));
}

int32_t sda_validate_bwd(const sda_bwd_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (int32_t rc = check_common(*a)) return rc;
  const int64_t es = bytes_of(a->dtype);
  for (const tda_tensor* t : {&a->q1, &a->k1, &a->q2, &a->k2, &a->v, &a->out, &a->dout, &a->dq1, &a->dk1, &a->dq2,
                              &a->dk2, &a->dv})
    if (int32_t rc = check_rows(*t, es)) return rc;
  if (int32_t rc = check_kept(*a)) return rc;
  if (!a->lse) return TDA_ERR_NULL_POINTER;
  // The key pass takes 32 query rows at a time and gives those past the last one a weight of one: they have to read
  // as zeros, which a descriptor of the rows that there are sees to only where each row ends before the next begins.
  // (Weights of zero for them instead took registers: backward of f16 (2, 16, 2048, 64) 235 -> 250 us, f32 (2, 16,
  // 2048, 128/256) 6.43 -> 6.81 ms, bf16 (4, 16, 2048, 64/128) 406 -> 412 us.)
  if (a->seq_len % 32)
    for (const tda_tensor* t : {&a->q1, &a->q2, &a->dout})
      if (t->stride[2] < (t == &a->dout ? a->v_head_dim : a->head_dim)) return TDA_ERR_LAYOUT;
  if (reinterpret_cast<uintptr_t>(a->dlambda) % bytes_of(a->lambda_dtype)) return TDA_ERR_LAYOUT;
  return check_workspace(a->workspace, a->workspace_bytes, sda_bwd_workspace_bytes(a));
}

int32_t sda_bwd(const sda_bwd_args* a, void* stream) {
  if (int32_t rc = sda_validate_bwd(a)) return rc;
  sda::BwdParams p;
  std::memset(&p, 0, sizeof(p));
  fill(p, *a);
  p.dout = rows_of(a->dout);
  p.dq[0] = rows_of(a->dq1);
  p.dq[1] = rows_of(a->dq2);
  p.dk[0] = rows_of(a->dk1);
  p.dk[1] = rows_of(a->dk2);
  p.dv = rows_of(a->dv);
  p.scale = a->scale;
  p.lse = a->lse;
  p.stat = static_cast<float*>(a->workspace);
  if (peak_bytes(*a)) p.peak = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + stat_bytes(*a) - peak_bytes(*a));
  p.gs = (int)key_group(*a);
  p.part = part_bytes(*a) ? reinterpret_cast<float*>(static_cast<char*>(a->workspace) + stat_bytes(*a)) : nullptr;
  p.dlam = a->dlambda;
  const int64_t n[3] = {a->batch, a->heads, a->seq_len};
  for (int k = 0; k < 3; ++k) p.dlam_n[k] = a->lambda_stride[k] ? n[k] : 1;
  tda::timing_begin(stream);
  return done(sda::launch_bwd(p, a->dtype, (int)a->head_dim, (int)a->v_head_dim, stream));
}

int32_t sda_validate_rotary(const sda_rotary_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SDA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (a->position_dtype != 4 && a->position_dtype != 8) return TDA_ERR_DTYPE;
  if (a->batch < 1 || a->seq_len < 1 || a->head_dim < 2 || a->batch > kMaxPos || a->seq_len > kMaxPos ||
      a->head_dim > 8192 || !fits_grid((double)a->batch * a->seq_len))
    return TDA_ERR_SHAPE;
  if (a->axes < 1 || a->axes > SDA_MAX_AXES || a->count < 1 || a->count > SDA_MAX_ROTARY) return SDA_ERR_AXES;
  if (a->rot < 2 || a->rot % 2 || a->rot > a->head_dim) return SDA_ERR_AXES;
  int64_t pairs = 0;
  for (int k = 0; k < a->axes; ++k) {
    if (a->sections[k] < 0) return SDA_ERR_AXES;
    pairs += a->sections[k];
  }
  if (pairs != a->rot / 2) return SDA_ERR_AXES;
  if (!a->positions || !a->inv_freq) return TDA_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(a->positions) % a->position_dtype || reinterpret_cast<uintptr_t>(a->inv_freq) % 4)
    return TDA_ERR_LAYOUT;
  for (int64_t s : a->position_stride)
    if (s < 0 || s > kMaxStride) return TDA_ERR_LAYOUT;
  for (int z = 0; z < a->count; ++z) {
    if (a->heads[z] < 1 || a->heads[z] > (1 << 20)) return TDA_ERR_SHAPE;
    if (int32_t rc = check_rows(a->x[z], bytes_of(a->dtype), true)) return rc;
    if (int32_t rc = check_rows(a->y[z], bytes_of(a->dtype), true)) return rc;
  }
  return TDA_OK;
}

int32_t sda_rotary(const sda_rotary_args* a, void* stream) {
  if (int32_t rc = sda_validate_rotary(a)) return rc;
  sda::RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  int upto = 0;
  for (int k = 0; k < a->axes; ++k) p.upto[k] = upto += a->sections[k];
  for (int z = 0; z < a->count; ++z) {
    p.x[z] = rows_of(a->x[z]);
    p.y[z] = rows_of(a->y[z]);
    p.heads[z] = (int)a->heads[z];
  }
  p.count = a->count;
  p.B = (int)a->batch;
  p.N = (int)a->seq_len;
  p.D = (int)a->head_dim;
  p.pairs = (int)(a->rot / 2);
  p.inter = a->interleaved ? 1 : 0;
  p.axes = a->axes;
  p.pos = a->positions;
  for (int k = 0; k < 3; ++k) p.ps[k] = a->position_stride[k];
  p.pos64 = a->position_dtype == 8;
  p.inv_freq = a->inv_freq;
  p.sign = a->inverse ? -1.f : 1.f;
  tda::timing_begin(stream);
  return done(sda::launch_rotary(p, a->dtype, stream));
}

size_t sda_kv4_bytes(int64_t batch, int64_t kv_heads, int64_t capacity, int64_t width) {
  if (batch < 1 || kv_heads < 1 || capacity < 1 || batch > kMaxPos || kv_heads > kMaxPos || batch * kv_heads > kMaxPos ||
      capacity > kMaxCapacity || (width != 64 && width != 128 && width != 256)) return 0;
  return (size_t)(batch * kv_heads * (ceil_div(capacity, 4) * 4) * (width / 2 + width / 64 * 4));
}

int32_t sda_validate_kv4_append(const sda_kv4_append_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SDA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (int32_t rc = check_cache(a->cache)) return rc;
  if (a->rows < 1 || a->rows > a->cache.capacity) return SDA_ERR_CACHE;
  for (const tda_tensor* t : {&a->k1, &a->k2, &a->v})
    if (int32_t rc = check_rows(*t, bytes_of(a->dtype))) return rc;
  if (int32_t rc = check_words({a->start, a->counts})) return rc;
  // The call writes the lengths while others of its workgroups read start and counts: these may be the lengths
  // themselves (a launch of its own then writes them), but no other part of them.
  for (const int32_t* p : {a->start, a->counts}) {
    const int64_t apart = (int64_t)(reinterpret_cast<intptr_t>(p) - reinterpret_cast<intptr_t>(a->cache.lengths));
    if (p && apart && apart > -4 * a->cache.batch && apart < 4 * a->cache.batch) return SDA_ERR_CACHE;
  }
  return TDA_OK;
}
int32_t sda_kv4_append(const sda_kv4_append_args* a, void* stream) {
  if (int32_t rc = sda_validate_kv4_append(a)) return rc;
  sda::Kv4Params p;
  std::memset(&p, 0, sizeof(p));
  fill_cache(p, a->cache);
  p.x[0] = rows_of(a->k1);
  p.x[1] = rows_of(a->k2);
  p.x[2] = rows_of(a->v);
  p.rows = (int)a->rows;
  p.start = a->start == a->cache.lengths ? nullptr : a->start;
  p.counts = a->counts;
  tda::timing_begin(stream);
  return done(sda::launch_kv4_append(p, a->dtype, stream));
}

int32_t sda_validate_kv4_read(const sda_kv4_read_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SDA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (int32_t rc = check_cache(a->cache)) return rc;
  if (a->rows < 1 || a->rows > a->cache.capacity) return SDA_ERR_CACHE;
  for (const tda_tensor* t : {&a->k1, &a->k2, &a->v})
    if (int32_t rc = check_rows(*t, bytes_of(a->dtype))) return rc;
  return TDA_OK;
}
int32_t sda_kv4_read(const sda_kv4_read_args* a, void* stream) {
  if (int32_t rc = sda_validate_kv4_read(a)) return rc;
  sda::Kv4Params p;
  std::memset(&p, 0, sizeof(p));
  fill_cache(p, a->cache);
  p.x[0] = rows_of(a->k1);
  p.x[1] = rows_of(a->k2);
  p.x[2] = rows_of(a->v);
  p.rows = (int)a->rows;
  tda::timing_begin(stream);
  return done(sda::launch_kv4_read(p, a->dtype, stream));
}

static int32_t check_attend_sizes(const sda_kv4_attend_args& a) {
  if (int32_t rc = check_cache_sizes(a.cache)) return rc;
  if (a.heads < 1 || a.seq_len < 1) return TDA_ERR_SHAPE;
  if (a.heads % a.cache.kv_heads) return SDA_ERR_HEADS;
  return a.heads <= kMaxPos && a.seq_len <= kMaxPos &&
                 fits_grid((double)a.cache.batch * a.heads * a.seq_len * ((double)a.cache.capacity + 256) / 128.0)
             ? TDA_OK
             : TDA_ERR_SHAPE;
}
size_t sda_kv4_attend_workspace_bytes(const sda_kv4_attend_args* a) {
  if (!a || check_attend_sizes(*a)) return 0;
  int nsplit, chunk;
  const int64_t items = dec_items(a->cache.batch, a->heads, a->cache.kv_heads, a->seq_len);
  dec_split(items, a->cache.capacity, kKv4Target, &nsplit, &chunk);
  return (size_t)dec_bytes(items, nsplit, a->cache.v_head_dim);
}
int32_t sda_validate_kv4_attend(const sda_kv4_attend_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (a->abi_version != SDA_ABI_VERSION) return TDA_ERR_ABI;
  if (!any_dtype(a->dtype)) return TDA_ERR_DTYPE;
  if (int32_t rc = check_cache(a->cache)) return rc;
  if (!check_scale(a->scale)) return SDA_ERR_SCALE;
  if (int32_t rc = check_attend_sizes(*a)) return rc;
  if (int32_t rc = check_lambda(a->lambda_param, a->lambda_stride, a->lambda_dtype)) return rc;
  for (const tda_tensor* t : {&a->q1, &a->q2, &a->out})
    if (int32_t rc = check_rows(*t, bytes_of(a->dtype))) return rc;
  return check_workspace(a->workspace, a->workspace_bytes, sda_kv4_attend_workspace_bytes(a));
}
int32_t sda_kv4_attend(const sda_kv4_attend_args* a, void* stream) {
  if (int32_t rc = sda_validate_kv4_attend(a)) return rc;
  sda::Kv4Params p;
  std::memset(&p, 0, sizeof(p));
  fill_cache(p, a->cache);
  p.q[0] = rows_of(a->q1);
  p.q[1] = rows_of(a->q2);
  p.out = rows_of(a->out);
  p.lam = lambda_of(a->lambda_param, a->lambda_stride, a->lambda_dtype);
  p.H = (int)a->heads;
  p.Nq = (int)a->seq_len;
  p.c = (float)(a->scale * kLog2e);
  p.part = static_cast<float*>(a->workspace);
  dec_split(dec_items(a->cache.batch, a->heads, a->cache.kv_heads, a->seq_len), a->cache.capacity, kKv4Target, &p.nsplit, &p.chunk);
  tda::timing_begin(stream);
  return done(sda::launch_kv4_attend(p, a->dtype, stream));
}

}  // extern "C"
