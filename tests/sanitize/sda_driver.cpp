// sda_driver.cpp -- runs the host code of the softmax differential attention operators (sda_host.cpp) under
// AddressSanitizer and UndefinedBehaviorSanitizer, with the launchers below in place of the kernels: every
// rejection, extreme sizes and strides, buffer sizes, and the parameter blocks handed to the launchers.
// Exit status 0 when every check holds; a sanitizer report aborts the run.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <limits>

#include "../../include/sda.h"
#include "../../tda_amd/csrc/sda_params.hpp"

static int failures = 0;
#define CHECK(cond)                                                   \
  do {                                                                \
    if (!(cond)) {                                                    \
      std::fprintf(stderr, "%s:%d: check failed: %s\n", __FILE__, __LINE__, #cond); \
      ++failures;                                                     \
    }                                                                 \
  } while (0)

namespace got {
int forwards = 0, decodes = 0, backwards = 0, rotaries = 0, appends = 0, reads = 0, attends = 0, fail_with = 0;
sda::FwdParams fwd;
sda::BwdParams bwd;
sda::RotaryParams rot;
sda::Kv4Params kv4;
template <class P>
int took(int& count, P& last, const P& p) {
  ++count;
  last = p;
  const int e = fail_with;
  fail_with = 0;
  return e;
}
}  // namespace got
namespace sda {
int launch_fwd(const FwdParams& p, int, int, int, void*) { return got::took(got::forwards, got::fwd, p); }
int launch_decode(const FwdParams& p, int, int, int, void*) { return got::took(got::decodes, got::fwd, p); }
int launch_bwd(const BwdParams& p, int, int, int, void*) { return got::took(got::backwards, got::bwd, p); }
int launch_rotary(const RotaryParams& p, int, void*) { return got::took(got::rotaries, got::rot, p); }
int launch_kv4_append(const Kv4Params& p, int, void*) { return got::took(got::appends, got::kv4, p); }
int launch_kv4_read(const Kv4Params& p, int, void*) { return got::took(got::reads, got::kv4, p); }
int launch_kv4_attend(const Kv4Params& p, int, void*) { return got::took(got::attends, got::kv4, p); }
}  // namespace sda

// The host code never reads through these.
static char* const AT = reinterpret_cast<char*>(uintptr_t(1) << 20);
static constexpr int64_t HUGE64 = std::numeric_limits<int64_t>::max();
static constexpr int64_t EXTREMES[] = {std::numeric_limits<int64_t>::min(), -1, 0, int64_t(1) << 31, int64_t(1) << 62, HUGE64};

static tda_tensor rows(int64_t h, int64_t n, int64_t d) {
  tda_tensor t;
  t.data = AT;
  t.stride[0] = h * n * d, t.stride[1] = n * d, t.stride[2] = d, t.stride[3] = 1;
  return t;
}
template <class A>
static void common(A& a, int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t Nk, int64_t D, int64_t DV) {
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SDA_ABI_VERSION, a.dtype = TDA_DTYPE_BF16, a.causal = 1, a.scale = 0.125f;
  a.batch = B, a.heads = H, a.kv_heads = Hk, a.seq_len = N, a.seq_len_kv = Nk, a.head_dim = D, a.v_head_dim = DV;
  a.q1 = a.q2 = rows(H, N, D);
  a.k1 = a.k2 = rows(Hk, Nk, D);
  a.v = rows(Hk, Nk, DV);
  a.out = rows(H, N, DV);
  a.lambda_param = AT;
  a.workspace = AT;
}
static sda_fwd_args fwd_args(int64_t N = 100, int64_t Nk = 300) {
  sda_fwd_args a;
  common(a, 2, 8, 2, N, Nk, 64, 128);
  a.workspace_bytes = sda_fwd_workspace_bytes(&a);
  return a;
}
static sda_bwd_args bwd_args() {
  sda_bwd_args a;
  common(a, 2, 8, 2, 100, 300, 64, 128);
  a.out2 = a.out_low = a.dout = a.out;
  a.dq1 = a.dq2 = a.q1, a.dk1 = a.dk2 = a.k1, a.dv = a.v;
  a.lse = reinterpret_cast<float*>(AT);
  a.workspace_bytes = sda_bwd_workspace_bytes(&a);
  return a;
}
static sda_kv4 cache() { return {2, 2, 70, 64, 128, AT, AT, AT, reinterpret_cast<int32_t*>(AT)}; }

#define REFUSES(make, validate, change, code) \
  do {                                        \
    auto a = make;                            \
    change;                                   \
    CHECK(validate(&a) == (code));            \
  } while (0)

template <class A, class V, class W>
static void extremes(A (*make)(), V validate, W bytes, std::initializer_list<int64_t A::*> fields) {
  for (int64_t A::*f : fields)
    for (int64_t A::*g : fields)
      for (int64_t x : EXTREMES)
        for (int64_t y : EXTREMES) {
          A a = make();
          a.*f = x;
          a.*g = y;
          (void)bytes(&a);
          CHECK(validate(&a) != TDA_OK);
        }
}

static void attention() {
  CHECK(sda_validate_fwd(nullptr) == TDA_ERR_NULL_POINTER && sda_validate_bwd(nullptr) == TDA_ERR_NULL_POINTER);
  CHECK(sda_fwd_workspace_bytes(nullptr) == 0 && sda_bwd_workspace_bytes(nullptr) == 0);
  sda_fwd_args f = fwd_args();
  f.q_offset = 200;
  CHECK(sda_fwd(&f, nullptr) == TDA_OK && got::forwards == 1 && got::fwd.see.qoff == 200 && got::fwd.Hk == 2);
  CHECK(got::fwd.v.sb == f.v.stride[0] && got::fwd.part == nullptr && got::fwd.lam.type == 0);
  f = fwd_args(1, 4000);  // one token: parts of the keys
  CHECK(f.workspace_bytes > 0 && sda_fwd(&f, nullptr) == TDA_OK && got::decodes == 1 && got::fwd.nsplit > 1);
  CHECK(got::fwd.chunk % 128 == 0 && (int64_t)got::fwd.chunk * got::fwd.nsplit >= 4000 &&
        (int64_t)got::fwd.chunk * (got::fwd.nsplit - 1) < 4000);
  CHECK(f.workspace_bytes == (size_t)4 * got::fwd.nsplit * (64 + 32 * 128) * 4);
  f.lse = reinterpret_cast<float*>(AT);  // a training forward of one token
  CHECK(sda_fwd(&f, nullptr) == TDA_OK && got::forwards == 2);
  f = fwd_args();
  got::fail_with = 1;
  CHECK(sda_fwd(&f, nullptr) == TDA_ERR_HIP);
  sda_bwd_args b = bwd_args();
  CHECK(sda_bwd(&b, nullptr) == TDA_OK && got::backwards == 1 && got::bwd.gs == 1 && got::bwd.part != nullptr);
  CHECK(b.workspace_bytes == (size_t)((6 * 16 * 100 * 4 + 255) / 256 * 256 + 4 * 4 * 300 * (2 * 64 + 128) * 4));
  b.lambda_stride[1] = 1;
  CHECK(sda_bwd(&b, nullptr) == TDA_OK && got::bwd.dlam_n[0] == 1 && got::bwd.dlam_n[1] == 8 && got::bwd.dlam_n[2] == 1);

  REFUSES(fwd_args(), sda_validate_fwd, a.abi_version = 7, TDA_ERR_ABI);
  REFUSES(fwd_args(), sda_validate_fwd, a.dtype = 3, TDA_ERR_DTYPE);
  REFUSES(fwd_args(), sda_validate_fwd, a.dtype = SDA_DTYPE_F16, TDA_OK);
  REFUSES(bwd_args(), sda_validate_bwd, a.dtype = SDA_DTYPE_F16, TDA_ERR_WORKSPACE);  // its peaks take room
  b = bwd_args();
  b.dtype = SDA_DTYPE_F16;
  const size_t without = b.workspace_bytes;
  b.workspace_bytes = sda_bwd_workspace_bytes(&b);
  CHECK(b.workspace_bytes == without + 256 && sda_bwd(&b, nullptr) == TDA_OK);
  CHECK(reinterpret_cast<char*>(got::bwd.peak) == AT + 6 * 16 * 100 * 4 + (256 - 6 * 16 * 100 * 4 % 256) % 256);
  CHECK(reinterpret_cast<char*>(got::bwd.part) == reinterpret_cast<char*>(got::bwd.peak) + 256);
  REFUSES(fwd_args(), sda_validate_fwd, a.causal = 2, TDA_ERR_CAUSAL);
  for (float s : {0.f, -1.f, std::nanf(""), std::numeric_limits<float>::infinity(), 1e-31f, 1e31f})
    REFUSES(fwd_args(), sda_validate_fwd, a.scale = s, SDA_ERR_SCALE);
  REFUSES(fwd_args(), sda_validate_fwd, a.kv_heads = 3, SDA_ERR_HEADS);
  REFUSES(fwd_args(), sda_validate_fwd, a.v_head_dim = 96, TDA_ERR_HEAD_DIM);
  REFUSES(fwd_args(), sda_validate_fwd, a.q_offset = HUGE64, TDA_ERR_OFFSET);
  REFUSES(fwd_args(), sda_validate_fwd, a.q_offset = -HUGE64, TDA_ERR_OFFSET);
  REFUSES(fwd_args(), sda_validate_fwd, a.q_offsets = reinterpret_cast<int32_t*>(AT + 2), TDA_ERR_LAYOUT);
  REFUSES(fwd_args(), sda_validate_fwd, a.kv_lens = reinterpret_cast<int32_t*>(AT + 1), TDA_ERR_LAYOUT);
  REFUSES(fwd_args(), sda_validate_fwd, a.lambda_param = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(fwd_args(), sda_validate_fwd, a.lambda_dtype = 3, TDA_ERR_DTYPE);
  REFUSES(fwd_args(), sda_validate_fwd, a.lambda_stride[2] = -1, TDA_ERR_LAYOUT);
  REFUSES(fwd_args(1, 4000), sda_validate_fwd, a.workspace = nullptr, TDA_ERR_WORKSPACE);
  REFUSES(fwd_args(1, 4000), sda_validate_fwd, --a.workspace_bytes, TDA_ERR_WORKSPACE);
  REFUSES(fwd_args(1, 4000), sda_validate_fwd, a.workspace = AT + 8, TDA_ERR_WORKSPACE);
  for (tda_tensor sda_fwd_args::*t : {&sda_fwd_args::q1, &sda_fwd_args::k1, &sda_fwd_args::q2, &sda_fwd_args::k2,
                                      &sda_fwd_args::v, &sda_fwd_args::out}) {
    REFUSES(fwd_args(), sda_validate_fwd, (a.*t).data = nullptr, TDA_ERR_NULL_POINTER);
    REFUSES(fwd_args(), sda_validate_fwd, (a.*t).data = AT + 2, TDA_ERR_LAYOUT);
    REFUSES(fwd_args(), sda_validate_fwd, (a.*t).stride[3] = 2, TDA_ERR_LAYOUT);
    REFUSES(fwd_args(), sda_validate_fwd, (a.*t).stride[2] = (1 << 24) + 8, TDA_ERR_LAYOUT);
    for (int k = 0; k < 3; ++k)
      for (int64_t s : {int64_t(-8), int64_t(3), HUGE64, int64_t(1) << 62})
        REFUSES(fwd_args(), sda_validate_fwd, (a.*t).stride[k] = s, TDA_ERR_LAYOUT);
  }
  REFUSES(fwd_args(), sda_validate_fwd, a.out2 = a.out, TDA_ERR_NULL_POINTER);  // without what it belongs to
  REFUSES(bwd_args(), sda_validate_bwd, a.out2.data = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(bwd_args(), sda_validate_bwd, a.out_low.data = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(bwd_args(), sda_validate_bwd, a.dv.data = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(bwd_args(), sda_validate_bwd, a.dk2.stride[1] = 5, TDA_ERR_LAYOUT);
  REFUSES(bwd_args(), sda_validate_bwd, a.lse = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(bwd_args(), sda_validate_bwd, a.dlambda = AT + 2, TDA_ERR_LAYOUT);
  REFUSES(bwd_args(), sda_validate_bwd, --a.workspace_bytes, TDA_ERR_WORKSPACE);
  using F = sda_fwd_args;
  extremes<F>([] { return fwd_args(); }, sda_validate_fwd, sda_fwd_workspace_bytes,
              {&F::batch, &F::heads, &F::kv_heads, &F::seq_len, &F::seq_len_kv, &F::head_dim, &F::v_head_dim});
  using G = sda_bwd_args;
  extremes<G>([] { return bwd_args(); }, sda_validate_bwd, sda_bwd_workspace_bytes,
              {&G::batch, &G::heads, &G::kv_heads, &G::seq_len, &G::seq_len_kv, &G::head_dim, &G::v_head_dim});
}

static sda_rotary_args rotary_args() {
  sda_rotary_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SDA_ABI_VERSION, a.dtype = SDA_DTYPE_F16;
  a.batch = 2, a.seq_len = 9, a.head_dim = 64, a.rot = 48, a.axes = 3, a.count = 2;
  a.sections[0] = 4, a.sections[1] = 12, a.sections[2] = 8;
  for (int z = 0; z < 2; ++z) a.heads[z] = 3 + z, a.x[z] = a.y[z] = rows(3 + z, 9, 64);
  a.positions = AT, a.position_dtype = 8;
  a.inv_freq = reinterpret_cast<float*>(AT);
  return a;
}
static void rotary() {
  sda_rotary_args r = rotary_args();
  r.inverse = 1;
  CHECK(sda_rotary(&r, nullptr) == TDA_OK && got::rotaries == 1 && got::rot.upto[0] == 4 && got::rot.upto[1] == 16 &&
        got::rot.upto[2] == 24 && got::rot.pairs == 24 && got::rot.sign == -1.f && got::rot.pos64 == 1);
  CHECK(sda_validate_rotary(nullptr) == TDA_ERR_NULL_POINTER);
  REFUSES(rotary_args(), sda_validate_rotary, a.abi_version = 0, TDA_ERR_ABI);
  REFUSES(rotary_args(), sda_validate_rotary, a.dtype = 3, TDA_ERR_DTYPE);
  REFUSES(rotary_args(), sda_validate_rotary, a.position_dtype = 2, TDA_ERR_DTYPE);
  REFUSES(rotary_args(), sda_validate_rotary, a.axes = 0, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.axes = 5, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.count = 5, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.rot = 47, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.rot = 66, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.sections[1] = -1, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.sections[1] = 2147483647, SDA_ERR_AXES);
  REFUSES(rotary_args(), sda_validate_rotary, a.head_dim = 8194, TDA_ERR_SHAPE);
  REFUSES(rotary_args(), sda_validate_rotary, a.heads[1] = 0, TDA_ERR_SHAPE);
  REFUSES(rotary_args(), sda_validate_rotary, a.positions = AT + 4, TDA_ERR_LAYOUT);
  REFUSES(rotary_args(), sda_validate_rotary, a.position_stride[0] = -1, TDA_ERR_LAYOUT);
  REFUSES(rotary_args(), sda_validate_rotary, a.inv_freq = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(rotary_args(), sda_validate_rotary, a.y[1].data = AT + 1, TDA_ERR_LAYOUT);
  REFUSES(rotary_args(), sda_validate_rotary, a.x[0].stride[0] = HUGE64, TDA_ERR_LAYOUT);
  using R = sda_rotary_args;
  extremes<R>(rotary_args, sda_validate_rotary, [](const R*) { return 0; }, {&R::batch, &R::seq_len, &R::head_dim, &R::rot});
}

static sda_kv4_append_args append_args() {
  sda_kv4_append_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SDA_ABI_VERSION, a.dtype = TDA_DTYPE_F32, a.cache = cache(), a.rows = 5;
  a.k1 = a.k2 = rows(2, 5, 64);
  a.v = rows(2, 5, 128);
  return a;
}
static sda_kv4_read_args read_args() {
  sda_kv4_read_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SDA_ABI_VERSION, a.dtype = TDA_DTYPE_BF16, a.cache = cache(), a.rows = 70;
  a.k1 = a.k2 = rows(2, 70, 64);
  a.v = rows(2, 70, 128);
  return a;
}
static sda_kv4_attend_args attend_args() {
  sda_kv4_attend_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SDA_ABI_VERSION, a.dtype = SDA_DTYPE_F16, a.cache = cache(), a.heads = 8, a.seq_len = 3, a.scale = 1.f;
  a.cache.capacity = 700;
  a.q1 = a.q2 = rows(8, 3, 64);
  a.out = rows(8, 3, 128);
  a.lambda_param = AT, a.lambda_dtype = TDA_DTYPE_BF16;
  a.workspace = AT, a.workspace_bytes = sda_kv4_attend_workspace_bytes(&a);
  return a;
}
template <class A, class V>
static void cache_extremes(A (*make)(), V validate) {
  for (int64_t sda_kv4::*f : {&sda_kv4::batch, &sda_kv4::kv_heads, &sda_kv4::capacity, &sda_kv4::head_dim, &sda_kv4::v_head_dim})
    for (int64_t sda_kv4::*g : {&sda_kv4::batch, &sda_kv4::kv_heads, &sda_kv4::capacity})
      for (int64_t x : EXTREMES)
        for (int64_t y : EXTREMES) {
          A a = make();
          a.cache.*f = x;
          a.cache.*g = y;
          (void)sda_kv4_bytes(a.cache.batch, a.cache.kv_heads, a.cache.capacity, a.cache.head_dim);
          CHECK(validate(&a) != TDA_OK);
        }
  REFUSES(make(), validate, a.cache.k2 = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(make(), validate, a.cache.v = AT + 8, TDA_ERR_LAYOUT);
  REFUSES(make(), validate, a.cache.lengths = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(make(), validate, a.cache.lengths = reinterpret_cast<int32_t*>(AT + 2), TDA_ERR_LAYOUT);
  REFUSES(make(), validate, a.abi_version = 9, TDA_ERR_ABI);
  REFUSES(make(), validate, a.dtype = -1, TDA_ERR_DTYPE);
}
static void held() {
  CHECK(sda_kv4_bytes(2, 3, 5, 128) == (size_t)2 * 3 * 8 * (64 + 8) && sda_kv4_bytes(1, 1, 1, 96) == 0);
  sda_kv4_append_args p = append_args();
  CHECK(sda_kv4_append(&p, nullptr) == TDA_OK && got::appends == 1 && got::kv4.cap4 == 72);
  CHECK(reinterpret_cast<char*>(got::kv4.pars[2]) == AT + 2 * 2 * 72 * 64);
  p.start = p.cache.lengths;  // the same as none
  CHECK(sda_kv4_append(&p, nullptr) == TDA_OK && got::kv4.start == nullptr);
  sda_kv4_read_args r = read_args();
  CHECK(sda_kv4_read(&r, nullptr) == TDA_OK && got::reads == 1 && got::kv4.rows == 70);
  sda_kv4_attend_args t = attend_args();
  CHECK(t.workspace_bytes > 0 && sda_kv4_attend(&t, nullptr) == TDA_OK && got::attends == 1 && got::kv4.lam.type == 1);
  CHECK(got::kv4.chunk % 128 == 0 && (int64_t)got::kv4.chunk * got::kv4.nsplit >= 700);
  got::fail_with = 2;
  CHECK(sda_kv4_attend(&t, nullptr) == TDA_ERR_HIP);
  REFUSES(append_args(), sda_validate_kv4_append, a.rows = 0, SDA_ERR_CACHE);
  REFUSES(append_args(), sda_validate_kv4_append, a.rows = 71, SDA_ERR_CACHE);
  REFUSES(append_args(), sda_validate_kv4_append, a.start = reinterpret_cast<int32_t*>(AT + 1), TDA_ERR_LAYOUT);
  REFUSES(append_args(), sda_validate_kv4_append, a.counts = reinterpret_cast<int32_t*>(AT + 2), TDA_ERR_LAYOUT);
  REFUSES(append_args(), sda_validate_kv4_append, a.v.data = nullptr, TDA_ERR_NULL_POINTER);
  REFUSES(read_args(), sda_validate_kv4_read, a.rows = 71, SDA_ERR_CACHE);
  REFUSES(read_args(), sda_validate_kv4_read, a.k1.stride[0] = HUGE64, TDA_ERR_LAYOUT);
  REFUSES(attend_args(), sda_validate_kv4_attend, a.heads = 7, SDA_ERR_HEADS);
  REFUSES(attend_args(), sda_validate_kv4_attend, a.seq_len = HUGE64, TDA_ERR_SHAPE);
  REFUSES(attend_args(), sda_validate_kv4_attend, a.scale = 0.f, SDA_ERR_SCALE);
  REFUSES(attend_args(), sda_validate_kv4_attend, --a.workspace_bytes, TDA_ERR_WORKSPACE);
  for (int64_t x : EXTREMES)
    for (int64_t y : EXTREMES)
      REFUSES(attend_args(), (int32_t)!!sda_validate_kv4_attend, (a.heads = x, a.seq_len = y, (void)sda_kv4_attend_workspace_bytes(&a)), 1);
  CHECK(sda_validate_kv4_append(nullptr) == TDA_ERR_NULL_POINTER && sda_validate_kv4_read(nullptr) == TDA_ERR_NULL_POINTER &&
        sda_validate_kv4_attend(nullptr) == TDA_ERR_NULL_POINTER && sda_kv4_attend_workspace_bytes(nullptr) == 0);
  cache_extremes(append_args, sda_validate_kv4_append);
  cache_extremes(read_args, sda_validate_kv4_read);
  cache_extremes(attend_args, sda_validate_kv4_attend);
}

int main() {
  CHECK(sda_abi_version() == SDA_ABI_VERSION);
  for (int32_t c = -110; c <= 2; ++c) CHECK(sda_error_string(c) && std::strlen(sda_error_string(c)) > 0);
  attention();
  rotary();
  held();
  if (failures) return 1;
  std::puts("all checks passed");
  return 0;
}
