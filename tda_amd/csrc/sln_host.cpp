// sln_host.cpp -- C ABI of the layer norm (include/sln.h): argument validation, buffer sizing and dispatch.
#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <utility>

#include "../../include/sln.h"
#include "sln_params.hpp"

namespace {

constexpr int64_t kMaxRows = (int64_t(1) << 30) - 64;
constexpr int64_t kMaxStride = int64_t(1) << 50;  // elements: offsets of whole tensors stay in int64

bool any_dtype(int32_t t) { return t == TDA_DTYPE_F32 || t == TDA_DTYPE_BF16 || t == SDA_DTYPE_F16; }
int64_t bytes_of(int32_t dtype) { return dtype == TDA_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int32_t check_rows(const tda_tensor& t, int64_t es) {
  if (!t.data) return TDA_ERR_NULL_POINTER;
  if (t.stride[3] != 1 || !aligned(t.data, (uintptr_t)es)) return TDA_ERR_LAYOUT;
  for (int k = 0; k < 3; ++k)
    if (t.stride[k] < 0 || t.stride[k] > kMaxStride) return TDA_ERR_LAYOUT;
  return TDA_OK;
}
template <class A>
int32_t check_sizes(const A& a) {
  if (a.batch < 1 || a.heads < 1 || a.rows < 1 || a.batch > kMaxRows || a.heads > kMaxRows || a.rows > kMaxRows) return TDA_ERR_SHAPE;
  if ((double)a.batch * a.heads * a.rows > (double)kMaxRows) return TDA_ERR_SHAPE;
  if (a.width < 1 || a.width > SLN_MAX_WIDTH) return SLN_ERR_WIDTH;
  return any_dtype(a.dtype) ? TDA_OK : TDA_ERR_DTYPE;
}
template <class A>
int32_t check_common(const A& a) {
  if (a.abi_version != SLN_ABI_VERSION) return TDA_ERR_ABI;
  if (int32_t rc = check_sizes(a)) return rc;
  return a.weight_dtype == TDA_DTYPE_F32 || a.weight_dtype == a.dtype ? TDA_OK : TDA_ERR_DTYPE;
}
template <class A>
int32_t check_weights(const A& a, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned(p, (uintptr_t)bytes_of(a.weight_dtype))) return TDA_ERR_LAYOUT;
  return TDA_OK;
}

// The rows' axes: x's smallest stride last, neighbours merged where every tensor's strides allow it.
template <class A>
void lay_out(const A& a, sln::Params& p, std::initializer_list<std::pair<sln::Tensor*, const tda_tensor*>> ts) {
  const int64_t n[3] = {a.batch, a.heads, a.rows};
  const int64_t stat[3] = {a.heads * a.rows, a.rows, 1};
  int axes[3], k = 0;
  p.groups = a.weight_heads ? (int)a.heads : 1;
  for (int i = 0; i < 3; ++i)
    if (!(a.weight_heads && i == 1)) axes[k++] = i;
  const auto before = [&](int i, int j) { return a.x.stride[i] < a.x.stride[j]; };  // i belongs further in
  for (int i = 0; i < k; ++i)
    for (int j = i + 1; j < k; ++j)
      if (before(axes[i], axes[j])) std::swap(axes[i], axes[j]);
  // from the inside out: an axis joins the one within it when every tensor steps over that as a whole
  int64_t size[3] = {1, 1, 1};
  int at[3] = {-1, -1, -1}, top = 2;  // the axis whose stride an output axis has
  bool any = false;
  for (int i = k - 1; i >= 0; --i) {
    const int x = axes[i];
    if (n[x] == 1) continue;
    bool join = any;
    if (any) {
      const int in = at[top];
      for (const auto& t : ts) join = join && t.second->stride[x] == size[top] * t.second->stride[in];
      join = join && stat[x] == size[top] * stat[in];
    }
    if (join) {
      size[top] *= n[x];
    } else {
      if (any) --top;
      any = true;
      size[top] = n[x];
      at[top] = x;
    }
  }
  for (int i = 0; i < 3; ++i) p.n[i] = (int)size[i];
  p.rows = (int)(size[0] * size[1] * size[2]);
  for (const auto& t : ts) {
    t.first->p = t.second->data;
    t.first->group = a.weight_heads ? t.second->stride[1] : 0;
    for (int i = 0; i < 3; ++i) t.first->s[i] = at[i] < 0 ? 0 : t.second->stride[at[i]];
  }
  p.stats.group = a.weight_heads ? stat[1] : 0;
  for (int i = 0; i < 3; ++i) p.stats.s[i] = at[i] < 0 ? 0 : stat[at[i]];
  p.width = (int)a.width;
  p.center = a.center ? 1 : 0;
  p.weight_type = a.weight_dtype == TDA_DTYPE_F32 ? 0 : 1;
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

int32_t sln_abi_version(void) { return SLN_ABI_VERSION; }

const char* sln_error_string(int32_t code) {
  switch (code) {
    case SLN_ERR_WIDTH: return "width must be 1 to 16384";
    case SLN_ERR_EPS: return "eps must be finite and not negative";
    case TDA_ERR_LAYOUT: return "rows must have a unit last stride, other strides that are not negative, and whole elements' alignment";
    case TDA_ERR_DTYPE: return "dtype must be F32, BF16 or F16, weight_dtype the same or F32";
    case TDA_ERR_ABI: return "abi_version does not match SLN_ABI_VERSION";
    default: return sda_error_string(code);
  }
}

int32_t sln_validate_fwd(const sln_fwd_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (int32_t rc = check_common(*a)) return rc;
  if (!(a->eps >= 0.f && a->eps <= 3.0e38f)) return SLN_ERR_EPS;
  for (const tda_tensor* t : {&a->x, &a->y})
    if (int32_t rc = check_rows(*t, bytes_of(a->dtype))) return rc;
  if (!aligned(a->stats, 8)) return TDA_ERR_LAYOUT;
  return check_weights(*a, {a->weight, a->bias});
}

int32_t sln_fwd(const sln_fwd_args* a, void* stream) {
  if (int32_t rc = sln_validate_fwd(a)) return rc;
  sln::Params p;
  std::memset(&p, 0, sizeof(p));
  lay_out(*a, p, {{&p.x, &a->x}, {&p.y, &a->y}});
  p.stats.p = a->stats;
  p.weight = a->weight;
  p.bias = a->bias;
  p.eps = a->eps;
  tda::timing_begin(stream);
  return done(sln::launch_fwd(p, a->dtype, stream));
}

size_t sln_bwd_workspace_bytes(const sln_bwd_args* a) {
  if (!a || check_sizes(*a) || !(a->dweight || a->dbias)) return 0;
  const int64_t groups = a->weight_heads ? a->heads : 1;
  const int64_t blocks = sln::bwd_blocks((int)a->width, a->dtype, (int)groups, (int)(a->batch * a->heads * a->rows / groups));
  return blocks == 1 ? 0 : (size_t)(groups * blocks * 2 * a->width * 4);
}

int32_t sln_validate_bwd(const sln_bwd_args* a) {
  if (!a) return TDA_ERR_NULL_POINTER;
  if (int32_t rc = check_common(*a)) return rc;
  const int64_t es = bytes_of(a->dtype);
  for (const tda_tensor* t : {&a->x, &a->dy})
    if (int32_t rc = check_rows(*t, es)) return rc;
  if (a->dx.data)
    if (int32_t rc = check_rows(a->dx, es)) return rc;
  if (!a->stats) return TDA_ERR_NULL_POINTER;
  if (!aligned(a->stats, 8)) return TDA_ERR_LAYOUT;
  if (int32_t rc = check_weights(*a, {a->weight, a->dweight, a->dbias})) return rc;
  const size_t need = sln_bwd_workspace_bytes(a);
  return need && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)) ? TDA_ERR_WORKSPACE : TDA_OK;
}

int32_t sln_bwd(const sln_bwd_args* a, void* stream) {
  if (int32_t rc = sln_validate_bwd(a)) return rc;
  sln::Params p;
  std::memset(&p, 0, sizeof(p));
  if (a->dx.data) lay_out(*a, p, {{&p.x, &a->x}, {&p.dy, &a->dy}, {&p.dx, &a->dx}});
  else lay_out(*a, p, {{&p.x, &a->x}, {&p.dy, &a->dy}});
  p.stats.p = const_cast<float*>(a->stats);
  p.weight = a->weight;
  p.dweight = a->dweight;
  p.dbias = a->dbias;
  p.blocks = sln::bwd_blocks(p.width, a->dtype, p.groups, p.rows);
  if ((a->dweight || a->dbias) && p.blocks > 1) p.part = static_cast<float*>(a->workspace);
  tda::timing_begin(stream);
  return done(sln::launch_bwd(p, a->dtype, stream));
}

}  // extern "C"
