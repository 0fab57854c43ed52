// spa_many.hip -- attention over pages for sequences of many query rows (a chunk of a prompt).
//
// sda_fwd.hip's pass over the keys: 128 rows a workgroup, 8 waves (four groups of 32 rows times the two
// branches), transposed scores, keys and values by direct loads to LDS a stage ahead.  Three things differ.
// A tile's rows are those of all query heads that share a key head, token by token: a chunk of 40 tokens of 4 heads
// fills two tiles instead of a third of each of four, and a tile's positions are few, so little of its last
// stages is hidden.  A stage's rows come from pages: one load instruction takes 1 KB, 1 to 8 rows that lie in one
// page (pages are 16 rows or more), whose number a wave has in a register of 64 table entries.  And where the tiles
// are too few for the chip their keys are cut into pieces (find_job), which a second launch joins.
#include "spa_common.hpp"

namespace spa {

using sda::f32x16;
using sda::f32x4;
using tda::crow;

template <class Tr, int D, int DV>
struct Shape {
  using T = typename Tr::T;
  static constexpr int BN = sizeof(T) == 2 && DV <= 128 ? 64 : 32;  // keys of a stage
  using KT = sda::Tile<Tr, BN, D>;
  using VT = sda::Tile<Tr, BN, DV>;
  static constexpr int STAGE = 2 * KT::BYTES + VT::BYTES;
  static constexpr int XCH = 4 * 32 * DV * 4;  // branch 2's result, f32
  static constexpr int LDS = 2 * STAGE > XCH ? 2 * STAGE : XCH;
  static_assert(KT::LOADS % 8 == 0 && VT::LOADS % 8 == 0, "loads spread evenly over the waves");
};

template <class Tr, int D, int DV>
__global__ void __launch_bounds__(512) many_rows(AttendParams P) {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  using S = Shape<Tr, D, DV>;
  using KT = typename S::KT;
  using VT = typename S::VT;
  constexpr int BN = S::BN, NS = BN / 32, NT = D / 16, NO = DV / 32;
  constexpr int KL = KT::LOADS / 8, VL = VT::LOADS / 8;
  constexpr int KR = 1024 / (D * KT::ES), VR = 1024 / (DV * VT::ES);  // rows of a load
  constexpr int G4 = sizeof(T) == 2 ? 4 : 1;  // fragments read ahead; an fp32 one is eight products itself
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const uint32_t bid = tda::grid_bid<512>();
  if (bid >= P.many.grid) return;
  if (!P.few.grid) clear_free_rows<T, DV, 512>(P, bid, P.many.grid);
  const int G = P.H / P.Hk, hk = (int)(bid % (uint32_t)P.Hk), ps = P.seq.pshift;
  Job J;
  if (!find_job<kManyRows, false, true>(P.seq, G, P.bound, P.many.room, bid / (uint32_t)P.Hk, J)) return;
  const Seq sq = J.seq;
  const int R = sq.cnt * G;
  const int l = lane_id(), n32 = l & 31, g = l >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wv & 3, br = wv >> 2;
  const int r0 = J.tile * kManyRows, r0w = r0 + 32 * rg;
  // positions that the workgroup's, the wave's last rows and the wave's first row see
  const auto sight = [&](int r) { return max(min(sq.len, sq.held + min(r, R - 1) / G + 1), 0); };  // 0 .. 2^30
  int k0p, lim;
  keys_of(J, sight(r0 + kManyRows - 1), k0p, lim);
  const int limw = uniform(min(sight(r0w + 31), lim)), clear = uniform(sight(r0w));
  const int nst = (lim - k0p + BN - 1) / BN;
  const int r = r0w + n32;  // this lane's row
  const bool live = r < R;
  const int qi = sq.row0 + (live ? r / G : 0), h = hk * G + (live ? r % G : 0);
  const int see = live ? sight(r) : 0;

  uint32_t ko[KL], vo[VL];
#pragma unroll
  for (int u = 0; u < KL; ++u) ko[u] = KT::source(8 * u + wv, D * KT::ES) - (uint32_t)((8 * u + wv) * KR * D * KT::ES);
#pragma unroll
  for (int u = 0; u < VL; ++u) vo[u] = VT::source(8 * u + wv, DV * VT::ES) - (uint32_t)((8 * u + wv) * VR * DV * VT::ES);
  Pages pages;
  pages.begin(P.seq, J.s, k0p >> ps);
  // Stage j goes into buffer j % 2; rows behind every row's sight read as zeros (a weight of zero times whatever lies
  // there must stay zero).  Where its rows stand is worked out a stage ahead of its loads, in the middle of the
  // products, and kept in scalar registers.
  constexpr bool SAME = KR == VR;  // keys' and values' loads take the same rows
  uint64_t krow[KL], vrow[VL];
  int krows[KL], vrows[VL];
  auto prepare = [&](int j) {
    const int key = k0p + j * BN;
    pages.reach(key >> ps);
    const auto place = [&](int k, int n, uint64_t& row, int& rows) {
      const int pg = pages.page(k >> ps);
      row = pool_row(pg, P.Hk, hk, ps, k);
      rows = pg >= 0 ? rows_before(k, n, lim) : 0;
    };
#pragma unroll
    for (int u = 0; u < KL; ++u) place(key + (8 * u + wv) * KR, KR, krow[u], krows[u]);
    if constexpr (!SAME) {
#pragma unroll
      for (int u = 0; u < VL; ++u) place(key + (8 * u + wv) * VR, VR, vrow[u], vrows[u]);
    }
  };
  auto issue = [&](int j) {
    char* at = lds + (j & 1) * S::STAGE;
#pragma unroll
    for (int u = 0; u < KL; ++u) {
      const uint64_t row = uniform(krow[u]);
      const int rows = uniform(krows[u]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        KT::load(page_rsrc<D * KT::ES>(P.k[x], row, 0, rows), reinterpret_cast<T*>(at + x * KT::BYTES), 8 * u + wv, ko[u]);
      if constexpr (SAME)
        VT::load(page_rsrc<DV * VT::ES>(P.v, row, 0, rows), reinterpret_cast<T*>(at + 2 * KT::BYTES), 8 * u + wv, vo[u]);
    }
    if constexpr (!SAME) {
#pragma unroll
      for (int u = 0; u < VL; ++u)
        VT::load(page_rsrc<DV * VT::ES>(P.v, uniform(vrow[u]), 0, uniform(vrows[u])), reinterpret_cast<T*>(at + 2 * KT::BYTES), 8 * u + wv, vo[u]);
    }
  };
  if (nst > 0) {
    prepare(0);
    issue(0);
    prepare(1);
  }

  frag qf[NT];
  sda::load_frags<Tr, NT>(live ? sda::row_of<T>(P.q[br], sq.qb, h, qi) : nullptr, g, qf);
  f32x16 o[NO] = {};
  float m = sda::kNoMax, sums[4] = {};

  sda::RowReader<Tr, D> kr;
  sda::ColReader<Tr, DV, true> vr;  // a stage is waited for before its barrier
  const char* kbuf = lds + br * KT::BYTES;
  const char* vbuf = lds + 2 * KT::BYTES;
  kr.init(kbuf);
  vr.init(vbuf);
  auto step = [&](int j, auto half) {  // stage j, in the half of the buffers that its parity names
    constexpr int AT = half * S::STAGE;
    sda::wait_vm<0>();
    tda::lds_barrier();  // stage j is in place, and every wave is done with stage j - 1
    if (j + 1 < nst) issue(j + 1);
    const int k0 = k0p + j * BN;
    if (k0 >= limw) {
      prepare(j + 2);
      return;
    }
    // one sequence of NS NT key fragments, then 2 NS NO value fragments, read a group ahead of their use
    frag f[2][G4];
    auto read = [&](int i) {
#pragma unroll
      for (int u = 0; u < G4; ++u) {
        const int e = i * G4 + u, w = e - NS * NT;
        if (e < NS * NT) f[i & 1][u] = kr.read(kbuf, AT + 32 * D * KT::ES * (e % NS), e / NS);
        else f[i & 1][u] = vr.read(vbuf, AT + 32 * DV * VT::ES * (w / (2 * NO)), w / NO % 2, w % NO);
      }
    };
    f32x16 s[NS] = {};
    read(0);
#pragma unroll
    for (int i = 0; i < NS * NT / G4; ++i) {
      read(i + 1);
#pragma unroll
      for (int u = 0; u < G4; ++u) {
        const int e = i * G4 + u;
        s[e % NS] = Tr::mma32(f[i & 1][u], qf[e / NS], s[e % NS]);
      }
    }
    if (k0 + BN > clear) {
      asm volatile("");  // a branch: few stages need this
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + 32 * x + crow(e, g) >= see) s[x][e] = -__builtin_inff();
    }
    float four[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) four[e % 4] = fmaxf(four[e % 4], s[x][e]);
    float top = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3])) * P.c;
    if (__any(top > m + sda::kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = fmaxf(m, top), f = sda::exp2_(m - to);
      m = to;
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[e] *= f;
#pragma unroll
      for (int x = 0; x < NO; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[x][e] *= f;
    }
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[x][e] = sda::exp2_(__builtin_fmaf(s[x][e], P.c, -m));
        sums[e % 4] += s[x][e];
      }
    frag p[2 * NS];
#pragma unroll
    for (int x = 0; x < 2 * NS; ++x) p[x] = sda::pack8<Tr>(s[x / 2], x % 2);
    prepare(j + 2);  // behind the last stage: rows of none
    constexpr int first = NS * NT / G4, last = first + 2 * NS * NO / G4;
#pragma unroll
    for (int i = first; i < last; ++i) {
      if (i + 1 < last) read(i + 1);
#pragma unroll
      for (int u = 0; u < G4; ++u) {
        const int w = i * G4 + u - NS * NT;
        o[w % NO] = Tr::mma32(f[i & 1][u], p[w / NO], o[w % NO]);
      }
    }
  };
  for (int j = 0; j < nst; j += 2) {
    step(j, std::integral_constant<int, 0>());
    if (j + 1 < nst) step(j + 1, std::integral_constant<int, 1>());
  }

  float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  sum += __shfl_xor(sum, 32);
  if (J.parts > 1) {  // its sums as the lanes hold them
    float* part = P.many.part + (int64_t)bid * many_floats(DV);
    if (g == 0) {
      part[2 * kManyRows * br + 32 * rg + n32] = m;
      part[2 * kManyRows * br + kManyRows + 32 * rg + n32] = sum;
    }
    if (nst > 0) {
      f32x4* to = reinterpret_cast<f32x4*>(part + 4 * kManyRows) + (int64_t)((br * 4 + rg) * NO * 4) * 64 + l;
#pragma unroll
      for (int y = 0; y < NO; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(4 * y + e) * 64] = f32x4{o[y][4 * e], o[y][4 * e + 1], o[y][4 * e + 2], o[y][4 * e + 3]};
    }
    return;
  }
  const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;  // no visible key: zeros
  __syncthreads();  // the stages are read: their place carries branch 2's result
  f32x4* xch = reinterpret_cast<f32x4*>(lds) + rg * (NO * 4 * 64) + l;
  if (br) {
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        xch[(4 * y + e) * 64] = f32x4{o[y][4 * e] * inv, o[y][4 * e + 1] * inv, o[y][4 * e + 2] * inv, o[y][4 * e + 3] * inv};
  }
  __syncthreads();
  if (!br && live) {
    const float lam = sda::lambda_of(P.lam, sq.qb, h, qi);
    T* to = sda::row_of<T>(P.out, sq.qb, h, qi);
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 w = xch[(4 * y + e) * 64];
        f32x4 z;
#pragma unroll
        for (int k = 0; k < 4; ++k) z[k] = __builtin_fmaf(-lam, w[k], o[y][4 * e + k] * inv);
        sda::store4(to + 32 * y + 8 * e + 4 * g, z);
      }
  }
}

template <class Tr, int D, int DV>
static int run(const AttendParams& p, hipStream_t st) {
  using S = Shape<Tr, D, DV>;
  if (S::LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&many_rows<Tr, D, DV>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS);
    if (e != hipSuccess) return (int)e;
  }
  many_rows<Tr, D, DV><<<tda::grid_of<512>(p.many.grid), 512, S::LDS, st>>>(p);
  tda::launched(st, "spa_many_rows");
  return (int)hipGetLastError();
}
template <class Tr>
static int pick(const AttendParams& p, int d, int dv, hipStream_t st) {
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}
int launch_many(const AttendParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 1 ? pick<sda::TrB>(p, d, dv, st) : dtype == 2 ? pick<sda::TrH>(p, d, dv, st) : pick<sda::TrF>(p, d, dv, st);
}

}  // namespace spa
