// spa_few.hip -- attention over pages for sequences of few query rows (a decoding step), and the launch that joins
// the pieces of either form.
//
// sda_decode.hpp's tiles and waves, its keys and values read from pages: a wave's tile is 32 keys, two halves of
// 16 that lie in one page each.  The keys of all sequences are dealt to about 1024 workgroups by their own
// lengths (find_job), so a batch of unequal conversations is even work.
#include "sda_decode.hpp"
#include "spa_common.hpp"

namespace spa {

using sda::DecParams;
using sda::DecWork;
using sda::f32x4;

template <class Tr, int D_, int DV_>
struct PagedSrc : sda::DenseSrc<Tr, D_, DV_> {
  using Base = sda::DenseSrc<Tr, D_, DV_>;
  using T = typename Base::T;
  using Regs = typename Base::Regs;
  using row = typename Base::row;
  static constexpr int D = D_, DV = DV_, NT = Base::NT, NB = Base::NB, CW = Base::CW, ES = sizeof(T);
  const AttendParams* A;
  Pages pages;
  int hk;

  __device__ __forceinline__ void begin(const DecParams& P, const DecWork& W, int h, int i, bool live) {
    const int kq = lane_id() >> 4, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const T* r = sda::row_of<T>(P.q[x], W.qb, h, W.row0 + i);
#pragma unroll
      for (int t = 0; t < NT; ++t) this->q[x][t] = live ? Base::load8(r + 32 * t + 8 * kq) : typename Base::frag{};
    }
    hk = W.hk;
    pages.begin(A->seq, W.b, (W.k0 + 32 * wv) >> A->seq.pshift);
  }
  __device__ __forceinline__ void load(Regs& g, int t0, int lim) {
    const int n = lane_id() & 15, kq = lane_id() >> 4, ps = A->seq.pshift;
    if (t0 < lim) pages.reach(t0 >> ps);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int key = t0 + 16 * y, rows = rows_before(key, 16, lim), pg = pages.page(key >> ps);
      const uint64_t at = pool_row(pg, A->Hk, hk, ps, key);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const auto r = page_rsrc<D * ES>(A->k[x], at, pg, rows);
#pragma unroll
        for (int t = 0; t < NT; ++t) g.k[x][y][t] = Base::load8(r, (uint32_t)(n * D * ES + (32 * t + 8 * kq) * ES));
      }
      const auto r = page_rsrc<DV * ES>(A->v, at, pg, rows);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int z = 0; z < NB; ++z) {
          const uint32_t off = (uint32_t)((4 * kq + e) * DV * ES + (CW * n + 16 * CW * z) * ES);
          row& to = g.v[4 * y + e][z];
          if constexpr (CW * ES == 8) to = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
          else if constexpr (CW * ES == 16) to = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
          else to = Base::load8(r, off);
        }
    }
  }
};

template <class Tr, int D, int DV>
__global__ void __launch_bounds__(256) few_rows(DecParams P, AttendParams A) {
  extern __shared__ float lds[];
  using T = typename Tr::T;
  const uint32_t bid = tda::grid_bid<256>();
  if (bid >= A.few.grid) return;
  clear_free_rows<T, DV, 256>(A, bid, A.few.grid);
  Job J;
  if (!find_job<kFewRows, true, true>(A.seq, A.H / A.Hk, A.bound, A.few.room, bid / (uint32_t)A.Hk, J)) return;
  const Seq s = J.seq;
  DecWork W;
  W.b = J.s;
  W.hk = (int)(bid % (uint32_t)A.Hk);
  W.rt = J.tile;
  W.qb = s.qb;
  W.row0 = s.row0;
  W.nq = s.cnt;
  W.len = s.len;
  W.off = s.held;
  W.causal = true;
  keys_of(J, max(min(s.len, s.held + s.cnt), 0), W.k0, W.k1);
  W.part = J.parts > 1 ? A.few.part + (int64_t)bid * few_floats(DV) : nullptr;
  PagedSrc<Tr, D, DV> src;
  src.A = &A;
  sda::decode_body(P, W, src, lds);
}

// ------------------------------------------------------------------ joining pieces
// Parts u = 0 .. n - 1 of one value: maximum, sum and weighted sum, in order, eight at a time so that their
// loads are on their way together.
struct Joined { float m, l; };
template <class Stat, class Val, int N>
__device__ __forceinline__ void join_parts(int n, Stat&& stat, Val&& val, float (&a)[N], Joined& j) {
  j.m = sda::kNoMax;
  j.l = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] = 0.f;
  for (int s0 = 0; s0 < n; s0 += 8) {
    float mm[8], ll[8], aa[8][N];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = min(s0 + u, n - 1);
      stat(s, mm[u], ll[u]);
      val(s, aa[u]);
      if (s0 + u >= n) ll[u] = 0.f;
    }
    float top = j.m;
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, mm[u]);
    const float f = sda::exp2_(j.m - top);
    j.l *= f;
    j.m = top;
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] *= f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (ll[u] == 0.f) continue;  // no key of this piece: its sums are not written
      const float w = sda::exp2_(mm[u] - top);
      j.l = __builtin_fmaf(ll[u], w, j.l);
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = __builtin_fmaf(aa[u][e], w, a[e]);
    }
  }
}
__device__ __forceinline__ float over(float a, float l) { return l > 0.f || l != l ? a / l : 0.f; }

// Workgroups 0 .. few.join - 1: a tile of the first form each; then of the second, 32 rows each.
template <class T, int DV>
__global__ void __launch_bounds__(256) join(AttendParams A) {
  const int G = A.H / A.Hk, tid = threadIdx.x;
  uint32_t bid = tda::grid_bid<256>();
  if (bid < A.few.join) {
    Job J;
    if (!find_job<kFewRows, true, false>(A.seq, G, A.bound, A.few.room, bid / (uint32_t)A.Hk, J) || J.parts < 2) return;
    const int hk = (int)(bid % (uint32_t)A.Hk);
    const Seq s = J.seq;
    const int rows = min(kFewRows, s.cnt * G - kFewRows * J.tile);
    const float* base = A.few.part + ((int64_t)J.first * A.Hk + hk) * few_floats(DV);
    const int64_t step = (int64_t)A.Hk * few_floats(DV);
    for (int e = tid; e < rows * DV; e += 256) {
      const int n = e / DV, c = e % DV, q = kFewRows * J.tile + n, h = hk * G + q / s.cnt, i = s.row0 + q % s.cnt;
      float res[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        Joined j;
        float a[1];
        join_parts(J.parts, [&](int u, float& m, float& l) { m = base[u * step + 32 * x + n]; l = base[u * step + 32 * x + 16 + n]; },
                   [&](int u, float(&v)[1]) { v[0] = base[u * step + 64 + (x * kFewRows + n) * DV + c]; }, a, j);
        res[x] = over(a[0], j.l);
      }
      sda::row_of<T>(A.out, s.qb, h, i)[c] = (T)__builtin_fmaf(-sda::lambda_of(A.lam, s.qb, h, i), res[1], res[0]);
    }
    return;
  }
  bid -= A.few.join;
  if (bid >= A.many.join) return;
  constexpr int NO = DV / 32, RG = kManyRows / 32;
  const int rg = (int)(bid % RG);
  const uint32_t item = bid / RG;
  Job J;
  if (!find_job<kManyRows, false, false>(A.seq, G, A.bound, A.many.room, item / (uint32_t)A.Hk, J) || J.parts < 2) return;
  const int hk = (int)(item % (uint32_t)A.Hk);
  const Seq s = J.seq;
  // the second form's pieces: [branch][m, l][128], then [branch][32 rows][4 of a lane's values][lane]
  const float* base = A.many.part + ((int64_t)J.first * A.Hk + hk) * many_floats(DV);
  const int64_t step = (int64_t)A.Hk * many_floats(DV);
  const int l = lane_id(), q = kManyRows * J.tile + 32 * rg + (l & 31);
  if (q >= s.cnt * G) return;
  const int h = hk * G + q % G, i = s.row0 + q / G;
  const float lam = sda::lambda_of(A.lam, s.qb, h, i);
  T* to = sda::row_of<T>(A.out, s.qb, h, i);
  // each branch's maximum and sum over the pieces, then the pieces' values under them, in order
  float top[2], inv[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    Joined j;
    float none[1];
    join_parts(J.parts, [&](int u, float& m, float& z) {
        m = base[u * step + 2 * kManyRows * y + 32 * rg + (l & 31)];
        z = base[u * step + 2 * kManyRows * y + kManyRows + 32 * rg + (l & 31)];
      }, [](int, float(&v)[1]) { v[0] = 0.f; }, none, j);
    top[y] = j.m;
    inv[y] = j.l > 0.f || j.l != j.l ? 1.0f / j.l : 0.f;
  }
  inv[1] *= -lam;
  constexpr int XS = NO < 4 ? NO : 4;  // quads of values a thread has in hand
  f32x4 z[XS] = {};
  const int x0 = (tid >> 6) * NO;
  for (int xs = 0; xs < NO; xs += XS) {
#pragma unroll
    for (int k = 0; k < XS; ++k) z[k] = f32x4{};
    for (int u0 = 0; u0 < J.parts; u0 += 2) {  // two pieces' values on their way
      f32x4 v[2][2][XS];
      float w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float* part = base + min(u0 + u, J.parts - 1) * step;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float sum = part[2 * kManyRows * y + kManyRows + 32 * rg + (l & 31)];
          w[u][y] = u0 + u < J.parts && sum != 0.f  // else no key of this piece: its sums are not written
                        ? sda::exp2_(part[2 * kManyRows * y + 32 * rg + (l & 31)] - top[y]) * inv[y] : 0.f;
#pragma unroll
          for (int k = 0; k < XS; ++k)
            v[u][y][k] = *reinterpret_cast<const f32x4*>(part + 4 * kManyRows + (int64_t)(((y * RG + rg) * NO * 4 + x0 + xs + k) * 64 + l) * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (w[u][y] != 0.f)
#pragma unroll
            for (int k = 0; k < XS; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e) z[k][e] = __builtin_fmaf(w[u][y], v[u][y][k][e], z[k][e]);
    }
#pragma unroll
    for (int k = 0; k < XS; ++k) {
      const int x = x0 + xs + k;
      sda::store4(to + 32 * (x / 4) + 8 * (x % 4) + 4 * (l >> 5), z[k]);
    }
  }
}

// ------------------------------------------------------------------ launches
template <class Tr, int D, int DV>
static int run(const AttendParams& a, hipStream_t st) {
  DecParams p{};
  p.q[0] = a.q[0];
  p.q[1] = a.q[1];
  p.out = a.out;
  p.lam = a.lam;
  p.H = a.H;
  p.Hk = a.Hk;
  p.c = a.c;
  constexpr int LDS = sda::kDecLds<DV>;
  if (LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&few_rows<Tr, D, DV>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return (int)e;
  }
  few_rows<Tr, D, DV><<<tda::grid_of<256>(a.few.grid), 256, LDS, st>>>(p, a);
  tda::launched(st, "spa_few_rows");
  return (int)hipGetLastError();
}
template <class Tr>
static int pick(const AttendParams& p, int d, int dv, hipStream_t st) {
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}
int launch_few(const AttendParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 1 ? pick<sda::TrB>(p, d, dv, st) : dtype == 2 ? pick<sda::TrH>(p, d, dv, st) : pick<sda::TrF>(p, d, dv, st);
}
template <class T>
static int run_join(const AttendParams& p, int dv, hipStream_t st) {
  const dim3 grid = tda::grid_of<256>((int64_t)p.few.join + p.many.join);
  if (dv == 64) join<T, 64><<<grid, 256, 0, st>>>(p);
  else if (dv == 128) join<T, 128><<<grid, 256, 0, st>>>(p);
  else join<T, 256><<<grid, 256, 0, st>>>(p);
  tda::launched(st, "spa_join");
  return (int)hipGetLastError();
}
int launch_attend(const AttendParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  int e = p.few.grid ? launch_few(p, dtype, d, dv, stream) : 0;
  if (!e && p.many.grid) e = launch_many(p, dtype, d, dv, stream);
  if (!e && p.few.join + p.many.join)
    e = dtype == 0 ? run_join<float>(p, dv, st) : dtype == 1 ? run_join<tda::bf16>(p, dv, st) : run_join<_Float16>(p, dv, st);
  return e;
}

}  // namespace spa
