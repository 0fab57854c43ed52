// spa_driver.cpp -- runs the host code of the paged cache (spa_host.cpp) and of the layer norm (sln_host.cpp) under
// AddressSanitizer and UndefinedBehaviorSanitizer, with the launchers below in place of the kernels: rejections,
// extreme sizes and strides, buffer sizes, and the parameter blocks handed to the launchers.  Exit status 0 when
// every check holds; a sanitizer report aborts the run.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <limits>

#include "../../include/sln.h"
#include "../../include/spa.h"
#include "../../tda_amd/csrc/sln_params.hpp"
#include "../../tda_amd/csrc/spa_params.hpp"

static int failures = 0;
#define CHECK(cond)                                                   \
  do {                                                                \
    if (!(cond)) {                                                    \
      std::fprintf(stderr, "%s:%d: check failed: %s\n", __FILE__, __LINE__, #cond); \
      ++failures;                                                     \
    }                                                                 \
  } while (0)

namespace got {
int appends = 0, attends = 0, forwards = 0, backwards = 0, fail_with = 0;
spa::AppendParams append;
spa::AttendParams attend;
sln::Params norm;
template <class P>
int took(int& count, P& last, const P& p) {
  ++count;
  last = p;
  const int e = fail_with;
  fail_with = 0;
  return e;
}
}  // namespace got
namespace spa {
int launch_append(const AppendParams& p, int, void*) { return got::took(got::appends, got::append, p); }
int launch_attend(const AttendParams& p, int, int, int, void*) { return got::took(got::attends, got::attend, p); }
}  // namespace spa
namespace sln {
int launch_fwd(const Params& p, int, void*) { return got::took(got::forwards, got::norm, p); }
int launch_bwd(const Params& p, int, void*) { return got::took(got::backwards, got::norm, p); }
}  // namespace sln
namespace sda {  // never called
int launch_fwd(const FwdParams&, int, int, int, void*) { return 1; }
int launch_decode(const FwdParams&, int, int, int, void*) { return 1; }
int launch_bwd(const BwdParams&, int, int, int, void*) { return 1; }
int launch_rotary(const RotaryParams&, int, void*) { return 1; }
int launch_kv4_append(const Kv4Params&, int, void*) { return 1; }
int launch_kv4_read(const Kv4Params&, int, void*) { return 1; }
int launch_kv4_attend(const Kv4Params&, int, void*) { return 1; }
}  // namespace sda

// The host code never reads through these.
static char* const AT = reinterpret_cast<char*>(uintptr_t(1) << 20);
static int32_t* const INTS = reinterpret_cast<int32_t*>(AT);
static constexpr int64_t HUGE64 = std::numeric_limits<int64_t>::max();
static constexpr int64_t EXTREMES[] = {std::numeric_limits<int64_t>::min(), -1, 0, int64_t(1) << 31, int64_t(1) << 62, HUGE64};

static tda_tensor rows(int64_t h, int64_t n, int64_t d) {
  tda_tensor t;
  t.data = AT;
  t.stride[0] = h * n * d, t.stride[1] = n * d, t.stride[2] = d, t.stride[3] = 1;
  return t;
}
template <class A>
static void place(A& a, int64_t s, int64_t n) {
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SPA_ABI_VERSION;
  a.dtype = TDA_DTYPE_BF16;
  a.cache = {100, 2, 32, 64, 128, AT, AT, AT};
  a.at = {s, n, INTS, 90, 90, INTS, nullptr, nullptr};
  a.heads = 8;
  a.q1 = a.q2 = rows(8, n, 64);
}
static spa_append_args append_args() {
  spa_append_args a;
  place(a, 3, 5);
  a.k1 = a.k2 = rows(2, 5, 64);
  a.v = rows(2, 5, 128);
  a.q1_out = a.q2_out = a.q1;
  a.rot = 64;
  a.axes = 3;
  a.sections[0] = 12, a.sections[1] = 0, a.sections[2] = 20;
  a.inv_freq = reinterpret_cast<float*>(AT);
  a.positions = AT;
  a.position_dtype = 8;
  return a;
}
static spa_attend_args attend_args(int64_t s, int64_t n) {
  spa_attend_args a;
  place(a, s, n);
  a.out = rows(8, n, 128);
  a.scale = 0.125f;
  a.lambda_param = AT;
  a.workspace = AT;
  a.workspace_bytes = spa_attend_workspace_bytes(&a);
  return a;
}

// Every integer argument at its extremes: refused, or taken without an overflow on the way.
template <class A, class F>
static void extremes(A good, std::initializer_list<int64_t A::*> own, F&& call) {
  for (int64_t x : EXTREMES) {
    for (auto m : own) {
      A a = good;
      a.*m = x;
      call(a);
    }
    for (int64_t spa_cache::*m : {&spa_cache::pages, &spa_cache::kv_heads, &spa_cache::page_size, &spa_cache::head_dim, &spa_cache::v_head_dim}) {
      A a = good;
      a.cache.*m = x;
      call(a);
    }
    for (int64_t spa_rows::*m : {&spa_rows::sequences, &spa_rows::rows, &spa_rows::table_stride, &spa_rows::table_len})
      for (int64_t spa_rows::*n : {&spa_rows::sequences, &spa_rows::rows, &spa_rows::table_stride, &spa_rows::table_len}) {
        A a = good;
        a.at.*m = x;
        a.at.*n = x;
        a.at.starts = x & 1 ? INTS : nullptr;
        call(a);
      }
    for (int k = 0; k < 4; ++k) {
      A a = good;
      a.q1.stride[k] = x;
      call(a);
    }
  }
}

static void paged() {
  spa_append_args ap = append_args();
  CHECK(spa_append(&ap, nullptr) == TDA_OK && got::appends == 1);
  CHECK(got::append.pairs == 32 && got::append.upto[0] == 12 && got::append.upto[1] == 12 && got::append.upto[2] == 32);
  CHECK(got::append.lead == 3 && got::append.seq.pshift == 5 && got::append.seq.pages == 100 && got::append.pos64 == 1);
  ap.at.starts = INTS;
  ap.rot = 0;
  ap.heads = 0;
  CHECK(spa_append(&ap, nullptr) == TDA_OK && got::append.lead == 1 && got::append.pairs == 0 && !got::append.q[0].p);
  got::fail_with = 77;
  CHECK(spa_append(&ap, nullptr) == TDA_ERR_HIP && tda_last_hip_error() == 77);
  extremes(append_args(), {&spa_append_args::heads, &spa_append_args::rot}, [](const spa_append_args& a) { spa_append(&a, nullptr); });

  // few rows of every sequence: small tiles; cut where they are few
  const int64_t few = spa::few_floats(128) * 4, many = spa::many_floats(128) * 4;
  spa_attend_args at = attend_args(3, 1);
  CHECK(spa_attend(&at, nullptr) == TDA_OK && got::attends == 1);
  CHECK(got::attend.bound == 0x7fffffff && got::attend.join[0] == 6 && got::attend.join[1] == 0);
  CHECK(got::attend.room > 3 && got::attend.grid == (uint32_t)got::attend.room * 2 && got::attend.part);
  CHECK((int64_t)at.workspace_bytes == got::attend.room * 4 * few);
  at.at.table_len = 31;  // over short tables: whole
  CHECK(spa_attend(&at, nullptr) == TDA_OK && !got::attend.room && !spa_attend_workspace_bytes(&at));
  at = attend_args(20000, 1);  // whole tiles
  CHECK(spa_attend(&at, nullptr) == TDA_OK && got::attend.grid == 40000 && !got::attend.room && !got::attend.join[0] && !at.workspace_bytes);
  at = attend_args(2, 1000);  // 4000 rows of a key head are 32 tiles
  CHECK(spa_attend(&at, nullptr) == TDA_OK && got::attend.bound == 0 && !got::attend.join[0] && got::attend.join[1] == 2 * 32 * 2 * 4);
  at = attend_args(8, 1000);
  CHECK(spa_attend(&at, nullptr) == TDA_OK && got::attend.grid == 8 * 32 * 2 && !got::attend.room && !at.workspace_bytes);
  at = attend_args(8, 1000);  // packed: either form
  at.at.starts = INTS;
  at.workspace_bytes = spa_attend_workspace_bytes(&at);
  CHECK(spa_attend(&at, nullptr) == TDA_OK && got::attend.lead == 1 && got::attend.bound == spa::kFewRows);
  CHECK(got::attend.join[0] == 8 * 2 && got::attend.join[1] == (4000 / 128 + 8) * 2 * 4);
  CHECK((int64_t)at.workspace_bytes == got::attend.room * 4 * many);
  at.most = 4;  // small tiles alone, which have room for any rows
  at.workspace_bytes = spa_attend_workspace_bytes(&at);
  CHECK(spa_attend(&at, nullptr) == TDA_OK && !got::attend.join[1] && got::attend.grid >= (4000 / 16 + 8) * 2);
  extremes(attend_args(3, 5), {&spa_attend_args::heads, &spa_attend_args::most}, [](spa_attend_args a) {
    a.workspace_bytes = spa_attend_workspace_bytes(&a);
    spa_attend(&a, nullptr);
  });
  // the largest calls that are taken: grids stay in 32 bits
  for (int64_t s : {int64_t(1), int64_t(1) << 20, int64_t(1) << 29})
    for (int64_t n : {int64_t(1), int64_t(1) << 20, int64_t(1) << 29})
      for (int packed = 0; packed < 2; ++packed) {
        spa_attend_args a = attend_args(3, 1);
        a.at.sequences = s;
        a.at.rows = n;
        a.at.starts = packed ? INTS : nullptr;
        a.workspace_bytes = spa_attend_workspace_bytes(&a);
        if (spa_attend(&a, nullptr) != TDA_OK) continue;
        const double need = packed ? (double)n * 4 / 16 : (double)s * ((n * 4 + 127) / 128);
        CHECK((double)got::attend.grid >= need / 8);
      }
}

static sln_fwd_args fwd_args(int64_t b, int64_t h, int64_t n, int64_t w) {
  sln_fwd_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SLN_ABI_VERSION;
  a.dtype = TDA_DTYPE_BF16;
  a.batch = b, a.heads = h, a.rows = n, a.width = w;
  a.eps = 1e-5f;
  a.weight_dtype = TDA_DTYPE_F32;
  a.x = a.y = rows(h, n, w);
  return a;
}
static sln_bwd_args bwd_args(int64_t b, int64_t h, int64_t n, int64_t w) {
  sln_bwd_args a;
  std::memset(&a, 0, sizeof(a));
  a.abi_version = SLN_ABI_VERSION;
  a.dtype = TDA_DTYPE_BF16;
  a.batch = b, a.heads = h, a.rows = n, a.width = w;
  a.weight_dtype = TDA_DTYPE_F32;
  a.x = a.dy = a.dx = rows(h, n, w);
  a.stats = reinterpret_cast<float*>(AT);
  a.dweight = a.dbias = a.workspace = AT;
  a.workspace_bytes = sln_bwd_workspace_bytes(&a);
  return a;
}

static void norm() {
  // contiguous rows are one axis; a weight of each head leaves the heads apart
  sln_fwd_args f = fwd_args(2, 3, 50, 100);
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.groups == 1 && got::norm.rows == 300 && got::norm.n[2] == 300);
  CHECK(got::norm.x.s[2] == 100 && got::norm.stats.s[2] == 1);
  f.weight_heads = 1;
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.groups == 3 && got::norm.rows == 100 && got::norm.n[1] == 2 && got::norm.n[2] == 50);
  CHECK(got::norm.x.group == 5000 && got::norm.x.s[1] == 15000 && got::norm.stats.group == 50 && got::norm.stats.s[1] == 150);
  // (B, N, H, w) memory order: the heads are the inner axis, or with weights of heads the rows of all entries one
  for (tda_tensor* t : {&f.x, &f.y}) t->stride[1] = 100, t->stride[2] = 300;
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.n[2] == 50 && got::norm.n[1] == 2 && got::norm.x.s[2] == 300);
  f.weight_heads = 0;
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.rows == 300 && got::norm.n[2] == 3 && got::norm.n[1] == 50 && got::norm.n[0] == 2);
  f.batch = 1;
  f.heads = 1;
  f.rows = 1;
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.rows == 1 && got::norm.n[2] == 1);
  f = fwd_args(2, 3, 50, 100);
  for (tda_tensor* t : {&f.x}) t->stride[0] = t->stride[1] = t->stride[2] = 0;  // one row, broadcast
  CHECK(sln_fwd(&f, nullptr) == TDA_OK && got::norm.rows == 300);
  for (int64_t w : {1, 7, 64, 1000, 4096, 9000, 16384})
    for (int64_t n : {1, 3, 100, 100000}) {
      sln_bwd_args b = bwd_args(1, 2, n, w);
      CHECK(sln_bwd(&b, nullptr) == TDA_OK && (got::norm.part != nullptr) == (got::norm.blocks > 1));
      CHECK(b.workspace_bytes == (got::norm.blocks > 1 ? (size_t)got::norm.blocks * 2 * w * 4 : 0));
    }
  for (int64_t x : EXTREMES)
    for (int k = 0; k < 8; ++k) {
      sln_fwd_args a = fwd_args(2, 3, 50, 100);
      sln_bwd_args b = bwd_args(2, 3, 50, 100);
      int64_t* at[] = {&a.batch, &a.heads, &a.rows, &a.width, &a.x.stride[0], &a.x.stride[1], &a.y.stride[2], &a.y.stride[3]};
      int64_t* bt[] = {&b.batch, &b.heads, &b.rows, &b.width, &b.dy.stride[0], &b.dx.stride[1], &b.x.stride[2], &b.dy.stride[3]};
      *at[k] = *bt[k] = x;
      sln_fwd(&a, nullptr);
      b.workspace_bytes = sln_bwd_workspace_bytes(&b);
      sln_bwd(&b, nullptr);
    }
  got::fail_with = 5;
  f = fwd_args(1, 1, 1, 1);
  CHECK(sln_fwd(&f, nullptr) == TDA_ERR_HIP && tda_last_hip_error() == 5);
  for (int code = -120; code <= 1; ++code) CHECK(std::strlen(sln_error_string(code)) && std::strlen(spa_error_string(code)));
}

int main() {
  paged();
  norm();
  if (failures) return 1;
  std::puts("all checks passed");
  return 0;
}
