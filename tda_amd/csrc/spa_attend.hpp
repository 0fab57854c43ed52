// spa_attend.hpp -- softmax differential attention of new positions over pages: one launch for sequences of few rows (a
// decoding step) and of many (a chunk of a prompt), and one that joins the pieces where tiles are cut.
//
// Both forms take the rows of all query heads that share a key head as one, token by token: a chunk of 40 tokens of 4 heads
// fills two tiles of 128 instead of a third of each of four, a tile's positions are few, so little of its last keys
// is hidden, and its keys are read once.  Where the tiles are fewer than the CUs their keys are cut into stretches
// (Deal), so that a batch of unequal conversations, or of tokens and chunks, is even work: a chunk keeps some CUs' matrix
// cores busy while others read the caches of the tokens beside it (a chunk of 700 rows and 23 tokens behind up to 5000, fp16, 16 over 4
// heads of (64, 128): 98 us; as launches of their own for tokens and chunk 132).
#pragma once

#include "spa_common.hpp"

namespace spa {

using sda::f32x16;
using sda::f32x4;
using tda::crow;

// A sum of weighted values by the sum of weights; no weights: zero.
__device__ __forceinline__ float over(float a, float l) { return l > 0.f || l != l ? a / l : 0.f; }

// 8 consecutive values, in memory or by a descriptor.
template <class Tr>
__device__ __forceinline__ typename Tr::frag load8(const typename Tr::T* p) {
  if constexpr (sizeof(typename Tr::T) == 2) {
    return *reinterpret_cast<const typename Tr::frag*>(p);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}
template <class Tr>
__device__ __forceinline__ typename Tr::frag load8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  const sda::u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
  if constexpr (sizeof(typename Tr::T) == 2) {
    return __builtin_bit_cast(typename Tr::frag, a);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 16, 0, 0));
    return {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }
}

// ------------------------------------------------------------------ many rows
// sda_fwd.hip's pass over the keys: 128 rows a workgroup, 8 waves (four groups of 32 rows times the two
// branches), transposed scores, keys and values by direct loads to LDS a stage ahead.  A stage's rows come from pages: one
// load instruction takes 1 KB, 1 to 8 rows that lie in one page (pages are 16 rows or more), whose number a wave has in a
// register of 64 table entries.
// Weights are rounded to the rows' type for their product with the values, in both forms, as sda_fwd.hip rounds them: a product of 32 bits has
// an eighth of the rate or less.  With the output's own rounding that is 2.4e-3 of the output's norm in bf16 (weights in 32 bits: 1.7e-3) and 3.0e-4
// in fp16 (2.1e-4).  Sums of weights are taken before the rounding, in 32 bits.
// Bound by the matrix cores and the exponentials and LDS reads between their products, at the clock that the card's power leaves: 2048 rows
// behind 30000, bf16, 16 over 4 heads of 128: 985 us, 1.06 PFLOP/s, where a large library product reaches 1.23 to 1.32.  128 keys of
// a tile take a CU 3.9 us at (128, 128) and 4.3 at (64, 128), whose exponentials are as many.
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
__device__ __forceinline__ void many_rows(const AttendParams& P, const Job& J, int hk, float* part, char* lds) {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  using S = Shape<Tr, D, DV>;
  using KT = typename S::KT;
  using VT = typename S::VT;
  constexpr int BN = S::BN, NS = BN / 32, NT = D / 16, NO = DV / 32;
  constexpr int KL = KT::LOADS / 8, VL = VT::LOADS / 8;
  constexpr int KR = 1024 / (D * KT::ES), VR = 1024 / (DV * VT::ES);  // rows of a load
  constexpr int G4 = sizeof(T) == 2 ? 4 : 1;  // fragments read ahead; an fp32 one is eight products itself
  const int G = P.H / P.Hk, ps = P.seq.pshift;
  const Seq sq = J.seq;
  const int R = sq.cnt * G;
  const int l = fresh_lane(), n32 = l & 31, g = l >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wv & 3, br = wv >> 2;
  const int r0 = J.tile * kManyRows, r0w = r0 + 32 * rg;
  // positions that the workgroup's, the wave's last rows and the wave's first row see
  const auto sight = [&](int r) { return max(min(sq.len, sq.held + min(r, R - 1) / G + 1), 0); };  // 0 .. 2^30
  int k0p, lim;
  Deal::keys(J, sight(r0 + kManyRows - 1), k0p, lim);
  const int limw = uniform(min(sight(r0w + 31), lim)), clear = uniform(sight(r0w));
  const int nst = (lim - k0p + BN - 1) / BN;
  // This lane's row.  One behind the last is the last again, and not written: loads under a condition of the lanes would
  // be a branch in the middle of the kernel's fullest stretch of registers.
  const int r = min(r0w + n32, R - 1), h = hk * G + r % G, qi = sq.row0 + r / G, see = sight(r);

  uint32_t ko[KL], vo[VL];
#pragma unroll
  for (int u = 0; u < KL; ++u) ko[u] = KT::source(8 * u + wv, D * KT::ES, l) - (uint32_t)((8 * u + wv) * KR * D * KT::ES);
#pragma unroll
  for (int u = 0; u < VL; ++u) vo[u] = VT::source(8 * u + wv, DV * VT::ES, l) - (uint32_t)((8 * u + wv) * VR * DV * VT::ES);
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

  // What registers do not hold of the widest fp32 rows (left to the compiler it went to memory and back in every stage: 1000 rows behind
  // 3000, (16, 4 heads, 128, 256): 1750 us, so 980): the queries, read again in each stage, a few ahead of their products and
  // before the next stage's loads, which they would else wait for; and the reads' addresses, worked out at each read.
  constexpr bool TIGHT = sizeof(T) == 4 && D == 128, AGAIN = sizeof(T) == 4 && DV == 256;
  constexpr int NQ = AGAIN ? 4 : NT;
  frag qf[NQ];
  const T* qr = sda::row_of<T>(P.q[br], sq.qb, h, qi) + 8 * g;
  if constexpr (!AGAIN)
#pragma unroll
    for (int t = 0; t < NT; ++t) qf[t] = load8<Tr>(qr + 16 * t);
  f32x16 o[NO];
  const float none = fresh_zero();
#pragma unroll
  for (int x = 0; x < NO; ++x) o[x] = none;
  float m = sda::kNoMax, sums[4] = {none, none, none, none};

  sda::RowReader<Tr, D> kr;
  sda::ColReader<Tr, DV, true> vr;  // a stage is waited for before its barrier
  const char* kbuf = lds + br * KT::BYTES;
  const char* vbuf = lds + 2 * KT::BYTES;
  kr.init(kbuf, l);
  vr.init(vbuf, l);
  auto step = [&](int j, auto half) {  // stage j, in the half of the buffers that its parity names
    constexpr int AT = half * S::STAGE;
    sda::wait_vm<0>();
    tda::lds_barrier();  // stage j is in place, and every wave is done with stage j - 1
    if (!AGAIN && j + 1 < nst) issue(j + 1);
    const int k0 = k0p + j * BN;
    if (k0 >= limw) {
      if (AGAIN && j + 1 < nst) issue(j + 1);
      prepare(j + 2);
      return;
    }
    // one sequence of NS NT key fragments, then 2 NS NO value fragments, read a group ahead of their use
    frag f[2][G4];
    const int ls = TIGHT ? fresh_lane() : l;
    auto read = [&](int i) {
#pragma unroll
      for (int u = 0; u < G4; ++u) {
        const int e = i * G4 + u, w = e - NS * NT;
        if (e < NS * NT) f[i & 1][u] = kr.read(kbuf, AT + 32 * D * KT::ES * (e % NS), e / NS, ls);
        else f[i & 1][u] = vr.read(vbuf, AT + 32 * DV * VT::ES * (w / (2 * NO)), w / NO % 2, w % NO, ls);
      }
    };
    f32x16 s[NS] = {};
    const T* qs = qr;
    if constexpr (AGAIN) {
      asm volatile("" : "+v"(qs));
#pragma unroll
      for (int t = 0; t < NQ; ++t) qf[t] = load8<Tr>(qs + 16 * t);
    }
    read(0);
#pragma unroll
    for (int i = 0; i < NS * NT / G4; ++i) {
      read(i + 1);
#pragma unroll
      for (int u = 0; u < G4; ++u) {
        const int e = i * G4 + u;
        s[e % NS] = Tr::mma32(f[i & 1][u], qf[e / NS % NQ], s[e % NS]);
        if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
        if (AGAIN && e % NS == NS - 1 && e / NS + NQ < NT) qf[e / NS % NQ] = load8<Tr>(qs + 16 * (e / NS + NQ));
      }
    }
    if (AGAIN && j + 1 < nst) issue(j + 1);
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
        if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  for (int j = 0; j < nst; j += 2) {
    step(j, std::integral_constant<int, 0>());
    if (j + 1 < nst) step(j + 1, std::integral_constant<int, 1>());
  }

  float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  sum += __shfl_xor(sum, 32);
  if (part) {  // its sums as the lanes hold them
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
  if (!br && r0w + n32 < R) {
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

// ------------------------------------------------------------------ few rows
// Tiles of 16 rows, products 16x16: S^T = K Q^T (lane: one query row and 4 of 16 keys), O^T = V^T P^T with the weights
// fed from the registers that hold them (sda_decode.hpp).  Nothing is staged in LDS: each wave takes every WAVES-th tile of 32
// keys.  Keys and values have DEPTH sets of registers each, refilled as soon as the products have taken them: the keys of a
// later tile are on their way during the weights, its values during the next scores.
//
// A launch that has tiles of 16 rows alone takes 4 waves, one a SIMD, whose registers hold two sets for most types.  Beside
// larger tiles 8 waves share the CU with half of the registers each.  Where registers do not hold both branches (SPLIT) half of the waves
// take one branch and half the other, which read the values twice.
// Bound by reading the keys and values: newest tokens of 32 sequences of up to 8192, bf16, 32 over 8 heads of 128: 222 us, 5.5 TB/s
// (two workgroups a CU of one set of registers each: 224 to 230, and 53 instead of 48 for one of 32000).
template <class Tr, int D, int DV, int WAVES>
struct FewRows {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  static constexpr int ES = sizeof(T), NT = D / 32, NO = DV / 16;
  static constexpr int CW = NO < 8 ? NO : 8, NB = NO / CW;  // a lane's columns of a value row stand together, NB blocks of them
  typedef T row __attribute__((ext_vector_type(CW)));
  // 4-byte registers of a lane that holds both branches: a tile's keys and values; queries and sums
  static constexpr int TILE = (D / 2 + DV / 4) * (ES / 2), REST = D / 4 * (ES / 2) + DV / 2;
  static constexpr bool SPLIT = TILE + REST > (WAVES == 8 ? 210 : 420);
  static constexpr int DEPTH = WAVES == 4 && 2 * TILE + REST <= 400 ? 2 : 1;
  static constexpr int NBR = SPLIT ? 1 : 2, SETS = SPLIT ? WAVES / 2 : WAVES;  // branches of a wave, waves that share a branch's keys
  static constexpr int LROW = DV + 4;  // LDS row stride: rows start in different banks
  static constexpr int LDS = (WAVES * kFewRows * LROW + 2 * SETS * 2 * kFewRows) * 4;

  // Output column of value e of product t.
  __device__ __forceinline__ static int column(int t, int e) { return 16 * CW * (t / CW) + CW * e + t % CW; }

  __device__ __forceinline__ static void run(const AttendParams& P, const Job& J, int hk, float* part, float* lds) {
    const int l = fresh_lane(), n = l & 15, kq = l >> 4, ps = P.seq.pshift;
    const int wv = uniform((int)threadIdx.x >> 6), set = wv % SETS, br = SPLIT ? wv / SETS : 0, tid = 64 * wv + l;
    const Seq sq = J.seq;
    const int G = P.H / P.Hk, R = G * sq.cnt, r0 = kFewRows * J.tile, rows = min(kFewRows, R - r0);
    const int at = r0 + min(n, rows - 1), h = hk * G + at % G, i = at / G;  // a row behind the last is the last again, and not written
    int k0, lim;
    Deal::keys(J, max(min(sq.len, sq.held + (r0 + rows - 1) / G + 1), 0), k0, lim);
    const int see = min(max(min(sq.len, sq.held + i + 1), 0), lim);  // keys of this part that the row sees end here

    frag q[NBR][NT], k[DEPTH][NBR][2][NT];
    row v[DEPTH][8][NB];
    f32x4 o[NBR][NO];
    float m[NBR], sum[NBR];
    const float none = fresh_zero();
#pragma unroll
    for (int x = 0; x < NBR; ++x) {
      m[x] = sda::kNoMax;
      sum[x] = none;
#pragma unroll
      for (int y = 0; y < NO; ++y) o[x][y] = none;
    }
    if (k0 < lim) {
      // The page numbers of a tile, one for each half in the lanes by turns, are loaded a tile ahead of its keys: without a
      // branch, so that the loads behind those that a product waits for can stay on their way.
      const int32_t* table = P.seq.table + (int64_t)uniform(J.s) * P.seq.tstride;
      const auto fetch = [&](int t0) { return table[(uint32_t)min((t0 + 16 * (l & 1)) >> ps, P.seq.tlen - 1)]; };
#pragma unroll
      for (int x = 0; x < NBR; ++x) {
        const T* qr = sda::row_of<T>(P.q[SPLIT ? br : x], sq.qb, h, sq.row0 + i);
#pragma unroll
        for (int t = 0; t < NT; ++t) q[x][t] = load8<Tr>(qr + 32 * t + 8 * kq);
      }
      // Rows past the piece's end, and whole tiles, read as zeros by the descriptors' range check: a weight of zero
      // times whatever lies there must stay zero.
      uint64_t prow[2];  // of the tile whose loads are issued next
      int prows[2];
      const auto place = [&](int t0, int entries) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int key = t0 + 16 * y, pg = __builtin_amdgcn_readlane(entries, y);
          const bool is = (uint32_t)pg < (uint32_t)P.seq.pages;
          prow[y] = pool_row(is ? pg : 0, P.Hk, hk, ps, key);
          prows[y] = is ? rows_before(key, 16, lim) : 0;
        }
      };
      const auto load_keys = [&](frag(&k)[NBR][2][NT]) {
#pragma unroll
        for (int x = 0; x < NBR; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const auto r = page_rsrc<D * ES>(P.k[SPLIT ? br : x], uniform(prow[y]), 0, uniform(prows[y]));
#pragma unroll
            for (int t = 0; t < NT; ++t) k[x][y][t] = load8<Tr>(r, (uint32_t)(n * D * ES + (32 * t + 8 * kq) * ES));
          }
      };
      const auto load_values = [&](row(&v)[8][NB]) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const auto r = page_rsrc<DV * ES>(P.v, uniform(prow[y]), 0, uniform(prows[y]));
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int z = 0; z < NB; ++z) {
              const uint32_t off = (uint32_t)((4 * kq + e) * DV * ES + (CW * n + 16 * CW * z) * ES);
              row& to = v[4 * y + e][z];
              if constexpr (CW * ES == 8) to = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
              else if constexpr (CW * ES == 16) to = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
              else to = load8<Tr>(r, off);
            }
        }
      };
      constexpr int STEP = 32 * SETS;
      const int t1 = k0 + 32 * set;
      int next[DEPTH], now[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        now[d] = fetch(t1 + d * STEP);
        next[d] = fetch(t1 + (DEPTH + d) * STEP);
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {  // in the loop's order: a product waits for as many loads as either way to it needs
        place(t1 + d * STEP, now[d]);
        __builtin_amdgcn_sched_barrier(0);
        load_keys(k[d]);
        __builtin_amdgcn_sched_barrier(0);
        load_values(v[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
      for (int t00 = t1; t00 < lim; t00 += DEPTH * STEP)
        sda::times<DEPTH>([&](auto d) {  // a tile behind the last one weighs nothing
          const int t0 = t00 + d * STEP;
          f32x4 s[NBR][2] = {};
#pragma unroll
          for (int x = 0; x < NBR; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int t = 0; t < NT; ++t) s[x][y] = Tr::mma16(k[d][x][y][t], q[x][t], s[x][y]);
          place(t0 + DEPTH * STEP, next[d]);
          next[d] = fetch(t0 + 2 * DEPTH * STEP);
          load_keys(k[d]);
          frag p[NBR];
#pragma unroll
          for (int x = 0; x < NBR; ++x) {
            if (__any(t0 + 31 >= see)) {
#pragma unroll
              for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (t0 + 16 * y + 4 * kq + e >= see) s[x][y][e] = -__builtin_inff();
            }
            float top = fmaxf(fmaxf(fmaxf(s[x][0][0], s[x][0][1]), fmaxf(s[x][0][2], s[x][0][3])),
                              fmaxf(fmaxf(s[x][1][0], s[x][1][1]), fmaxf(s[x][1][2], s[x][1][3]))) * P.c;
            if (__any(top > m[x] + sda::kSlack)) {
              top = fmaxf(top, __shfl_xor(top, 16));
              top = fmaxf(top, __shfl_xor(top, 32));
              const float to = fmaxf(m[x], top), f = sda::exp2_(m[x] - to);
              m[x] = to;
              sum[x] *= f;
#pragma unroll
              for (int y = 0; y < NO; ++y) o[x][y] *= f;
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                s[x][y][e] = sda::exp2_(__builtin_fmaf(s[x][y][e], P.c, -m[x]));
                p[x][4 * y + e] = (T)s[x][y][e];
              }
              sum[x] += (s[x][y][0] + s[x][y][1]) + (s[x][y][2] + s[x][y][3]);
            }
          }
#pragma unroll
          for (int z = 0; z < NB; ++z)
#pragma unroll
            for (int c = 0; c < CW; ++c) {
              frag a;
#pragma unroll
              for (int j = 0; j < 8; ++j) a[j] = v[d][j][z][c];
#pragma unroll
              for (int x = 0; x < NBR; ++x) o[x][CW * z + c] = Tr::mma16(a, p[x], o[x][CW * z + c]);
            }
          load_values(v[d]);
        });
    }
    // the waves' maxima and sums, then their outputs under the branch's common maximum, as many branches at a time as a wave has
    // fewer of
    float* ml = lds + WAVES * kFewRows * LROW;  // [branch][set][m, l][16]
#pragma unroll
    for (int x = 0; x < NBR; ++x) {
      sum[x] += __shfl_xor(sum[x], 16);
      sum[x] += __shfl_xor(sum[x], 32);
      if (kq == 0) {
        float* to = ml + ((SPLIT ? br : x) * SETS + set) * 2 * kFewRows;
        to[n] = m[x];
        to[kFewRows + n] = sum[x];
      }
    }
    const auto joined = [&](int x, int r, float& all, float& tot) {
      const float* from = ml + x * SETS * 2 * kFewRows;
      all = sda::kNoMax;
      tot = 0.f;
#pragma unroll
      for (int w = 0; w < SETS; ++w) all = fmaxf(all, from[w * 2 * kFewRows + r]);
#pragma unroll
      for (int w = 0; w < SETS; ++w)
        tot = __builtin_fmaf(from[(w * 2 + 1) * kFewRows + r], sda::exp2_(from[w * 2 * kFewRows + r] - all), tot);
    };
    constexpr int TH = 64 * WAVES, PER = kFewRows * DV / TH;  // values of a thread: tid + TH u, by row, then column
    float fin[2][PER];
#pragma unroll
    for (int x = 0; x < NBR; ++x) {
      __syncthreads();
      float all, tot;
      joined(SPLIT ? br : x, n, all, tot);
      const float f = sda::exp2_(m[x] - all);
#pragma unroll
      for (int y = 0; y < NO; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) lds[(wv * kFewRows + n) * LROW + column(y, 4 * kq + e)] = o[x][y][e] * f;
      if (part && set == 0 && kq == 0) {
        part[32 * (SPLIT ? br : x) + n] = all;
        part[32 * (SPLIT ? br : x) + 16 + n] = tot;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int e = tid + TH * u;
        const float* a = lds + e / DV * LROW + e % DV;
#pragma unroll
        for (int y = 0; y < 2 / NBR; ++y) {
          float z[SETS];
#pragma unroll
          for (int w = 0; w < SETS; ++w) z[w] = a[(y * SETS + w) * kFewRows * LROW];
#pragma unroll
          for (int d = SETS / 2; d > 0; d /= 2)
#pragma unroll
            for (int w = 0; w < d; ++w) z[w] += z[w + d];
          fin[SPLIT ? y : x][u] = z[0];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = tid + TH * u, r = e / DV, c = e % DV;
      if (r >= rows) break;
      if (part) {
        if (k0 < lim) {  // a piece without keys: not read
          part[64 + r * DV + c] = fin[0][u];
          part[64 + (kFewRows + r) * DV + c] = fin[1][u];
        }
        continue;
      }
      float s1, s2, any;
      joined(0, r, any, s1);
      joined(1, r, any, s2);
      const int row = r0 + r, hh = hk * G + row % G, ii = sq.row0 + row / G;
      const float lam = sda::lambda_of(P.lam, sq.qb, hh, ii);
      sda::row_of<T>(P.out, sq.qb, hh, ii)[c] = (T)__builtin_fmaf(-lam, over(fin[1][u], s2), over(fin[0][u], s1));
    }
  }
};

// What a launch may have: tiles of 16 rows, of 128, or both.
enum { FEW = 1, MANY = 2, BOTH = 3 };
template <class Tr, int D, int DV, int TILES>
struct Kind {
  using Few = FewRows<Tr, D, DV, TILES == FEW ? 4 : 8>;
  static constexpr int THREADS = TILES == FEW ? 256 : 512;
  static constexpr int FEW_LDS = TILES & FEW ? Few::LDS : 0, MANY_LDS = TILES & MANY ? Shape<Tr, D, DV>::LDS : 0;
  static constexpr int LDS = FEW_LDS > MANY_LDS ? FEW_LDS : MANY_LDS;
};

template <class Tr, int D, int DV, int TILES>
__global__ void __launch_bounds__(TILES == FEW ? 256 : 512) attend(AttendParams P) {
  using K = Kind<Tr, D, DV, TILES>;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t bid = tda::grid_bid<K::THREADS>();
  if (bid >= P.grid) return;
  clear_free_rows<typename Tr::T, DV, K::THREADS>(P, bid);
  const int hk = (int)(bid % (uint32_t)P.Hk);
  uint32_t done = 0, all;
  do {  // the tiles of a stretch; each looks at the sequences anew, which costs no registers meanwhile
    const Deal deal(P.seq, P.H / P.Hk, P.bound, P.room, P.cost);
    uint32_t group = bid / (uint32_t)P.Hk;
    const bool many = TILES == MANY || (TILES == BOTH && group < deal.groups[1]);
    if (!many) group -= deal.groups[1];
    if (group >= (many ? deal.groups[1] : deal.groups[0])) return;
    const uint32_t per = many ? deal.per[1] : deal.per[0], begin = group * per, end = min(begin + per, many ? deal.line[1] : deal.line[0]);
    all = end - begin;
    Job J;
    if (many ? !deal.find<1, false>(begin + done, end, J) : !deal.find<0, false>(begin + done, end, J)) return;
    // a stretch has at most two tiles of which it has a part: the one it begins in, and the one it ends in
    const uint64_t place = uniform((uint64_t)(2 * (int64_t)bid + (done != 0)) * (uint64_t)P.stride);
    float* part = uniform(J.count < J.units) ? P.part + place : nullptr;
    if (done) __syncthreads();  // the tile before is done with the LDS
    done += J.count;
    if constexpr (TILES & MANY)
      if (many) many_rows<Tr, D, DV>(P, J, hk, part, lds);
    if constexpr (TILES & FEW)
      if (!many) K::Few::run(P, J, hk, part, reinterpret_cast<float*>(lds));
  } while (done < all);
}

// ------------------------------------------------------------------ joining parts
// One branch of some values: maximum, sum and weighted sums of the parts so far, taken on in order.
template <int N>
struct Joined {
  float m = sda::kNoMax, l = 0.f, a[N] = {};
  // Parts with maxima mm, sums ll (0: no key, its values are not written) and values v.
  template <int B>
  __device__ __forceinline__ void take(const float (&mm)[B], const float (&ll)[B], const float (&v)[B][N]) {
    float top = m;
#pragma unroll
    for (int u = 0; u < B; ++u) top = fmaxf(top, mm[u]);
    const float f = sda::exp2_(m - top);
    l *= f;
    m = top;
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] *= f;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const float w = sda::exp2_(mm[u] - top);
      l = __builtin_fmaf(ll[u], w, l);
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = ll[u] == 0.f ? a[e] : __builtin_fmaf(v[u][e], w, a[e]);
    }
  }
  // Takes on another lane's.
  __device__ __forceinline__ void with(int lanes) {
    const float om = __shfl_xor(m, lanes), top = fmaxf(m, om), f = sda::exp2_(m - top), g = sda::exp2_(om - top);
    m = top;
    const float ol = __shfl_xor(l, lanes);
    l = l * f + ol * g;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float o = __shfl_xor(a[e], lanes);
      a[e] = a[e] * f + o * g;
    }
  }
};

// How a tile is joined.  Of a small one each wave takes a row, four columns a lane; where a row fills a part of the wave only, the
// other lanes take other parts.  Of a large one each wave takes 32 rows, XS times four columns a lane.  The parts' sums and values are loaded
// eight or four parts at a time, all together: a launch of this is a few waits for memory, and little else (4.4 us for one
// token's eight parts, 7.0 for 32 parts of 32000 keys, 9.8 for a chunk's 34 MB).
template <int DV>
struct Join {
  static constexpr int W = DV / 4, SLICES = 64 / W;         // lanes of a row, its parts at a time
  static constexpr int XS = DV >= 128 ? 4 : 2, PB = 8 / XS, RG = kManyRows / 32, COLS = DV / 8 / XS / 4;  // workgroups that 32 rows take
};

// Workgroups of four rows of a small tile each; then of some columns of 32 rows of a large one each.
template <class T, int DV>
__global__ void __launch_bounds__(256) join(AttendParams A) {
  using K = Join<DV>;
  const int G = A.H / A.Hk, l = lane_id(), wv = uniform((int)threadIdx.x >> 6);
  uint32_t bid = tda::grid_bid<256>();
  Deal deal(A.seq, G, A.bound, A.room, A.cost);
  Job J;
  if (!deal.cut) return;
  // the parts of a tile: workgroups first .. first + n - 1 of its form, each in its first place unless the tile is where
  // its stretch ends
  const float *head, *tail;
  int parts;
  const int64_t step = 2 * A.Hk * A.stride;
  const auto parts_of = [&](int form, int hk) {
    const uint32_t per = deal.per[form], first = J.at / per, last = (J.at + J.units - 1) / per;
    parts = (int)(last - first) + 1;
    const uint32_t place = first * per < J.at;  // of the first part; the others begin with this tile
    const uint32_t group = first + (form ? 0 : deal.groups[1]);
    tail = A.part + 2 * ((int64_t)group * A.Hk + hk) * A.stride;
    head = tail + place * A.stride;
  };
  const auto part = [&](int u) { return u ? tail + u * step : head; };
  const uint32_t per = (uint32_t)(A.join_rows + 3) / 4;  // workgroups of a small tile
  if (bid < A.join[0] * per) {
    const uint32_t tile = bid / per;
    const int hk = (int)(tile % (uint32_t)A.Hk), n = 4 * (int)(bid % per) + wv;
    if (!deal.find<0, true>(tile / (uint32_t)A.Hk, 0, J)) return;
    const Seq s = J.seq;
    parts_of(0, hk);
    if (parts < 2 || n >= s.cnt * G - kFewRows * J.tile) return;
    const int q = kFewRows * J.tile + n, h = hk * G + q % G, i = s.row0 + q / G, c = 4 * (l % K::W);
    const float lam = sda::lambda_of(A.lam, s.qb, h, i);
    Joined<4> j[2];
    for (int u0 = l / K::W; u0 < parts; u0 += 8 * K::SLICES) {
      float mm[2][8], ll[2][8], v[2][8][4];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = u0 + u * K::SLICES;
        const float* p = part(min(at, parts - 1));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mm[x][u] = p[32 * x + n];
          ll[x][u] = p[32 * x + 16 + n];
          const f32x4 y = *reinterpret_cast<const f32x4*>(p + 64 + (x * kFewRows + n) * DV + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[x][u][e] = y[e];
          if (at >= parts) ll[x][u] = 0.f;
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) j[x].take(mm[x], ll[x], v[x]);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int d = K::W; d < 64; d *= 2) j[x].with(d);
    if (l >= K::W) return;
    f32x4 z;
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = __builtin_fmaf(-lam, over(j[1].a[e], j[1].l), over(j[0].a[e], j[0].l));
    sda::store4(sda::row_of<T>(A.out, s.qb, h, i) + c, z);
    return;
  }
  bid -= A.join[0] * per;
  if (bid >= A.join[1] * K::COLS) return;
  constexpr int NO = DV / 32;
  const int x0 = (4 * (int)(bid % K::COLS) + wv) * K::XS, rg = (int)(bid / K::COLS % K::RG);
  const uint32_t item = bid / (K::COLS * K::RG);
  const int hk = (int)(item % (uint32_t)A.Hk);
  if (!deal.find<1, true>(item / (uint32_t)A.Hk, 0, J)) return;
  const Seq s = J.seq;
  parts_of(1, hk);
  const int row = 32 * rg + (l & 31), q = kManyRows * J.tile + row;
  if (parts < 2 || q >= s.cnt * G) return;
  const int h = hk * G + q % G, i = s.row0 + q / G;
  const float lam = sda::lambda_of(A.lam, s.qb, h, i);
  Joined<4 * K::XS> j[2];
  for (int u0 = 0; u0 < parts; u0 += K::PB) {
    float mm[2][K::PB], ll[2][K::PB], v[2][K::PB][4 * K::XS];
#pragma unroll
    for (int u = 0; u < K::PB; ++u) {
      const float* p = part(min(u0 + u, parts - 1));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mm[x][u] = p[2 * kManyRows * x + row];
        ll[x][u] = p[2 * kManyRows * x + kManyRows + row];
        if (u0 + u >= parts) ll[x][u] = 0.f;
#pragma unroll
        for (int k = 0; k < K::XS; ++k) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(p + 4 * kManyRows + (int64_t)(((x * K::RG + rg) * NO * 4 + x0 + k) * 64 + l) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[x][u][4 * k + e] = y[e];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) j[x].take(mm[x], ll[x], v[x]);
  }
  T* to = sda::row_of<T>(A.out, s.qb, h, i);
#pragma unroll
  for (int k = 0; k < K::XS; ++k) {
    f32x4 z;
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = __builtin_fmaf(-lam, over(j[1].a[4 * k + e], j[1].l), over(j[0].a[4 * k + e], j[0].l));
    const int x = x0 + k;
    sda::store4(to + 32 * (x / 4) + 8 * (x % 4) + 4 * (l >> 5), z);
  }
}

// ------------------------------------------------------------------ launches
template <class Tr, int D, int DV, int TILES>
static int launch(const AttendParams& p, hipStream_t st) {
  using K = Kind<Tr, D, DV, TILES>;
  if (K::LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&attend<Tr, D, DV, TILES>), hipFuncAttributeMaxDynamicSharedMemorySize, K::LDS);
    if (e != hipSuccess) return (int)e;
  }
  attend<Tr, D, DV, TILES><<<tda::grid_of<K::THREADS>(p.grid), K::THREADS, K::LDS, st>>>(p);
  tda::launched(st, TILES == FEW ? "spa_attend_few" : TILES == MANY ? "spa_attend_many" : "spa_attend");
  return 0;
}
template <class Tr, int D, int DV>
static int run(const AttendParams& p, hipStream_t st) {
  const int e = p.bound == 0 ? launch<Tr, D, DV, MANY>(p, st) : p.bound == 0x7fffffff ? launch<Tr, D, DV, FEW>(p, st) : launch<Tr, D, DV, BOTH>(p, st);
  if (e) return e;
  if (p.room) {
    const int64_t blocks = (int64_t)p.join[0] * ((p.join_rows + 3) / 4) + (int64_t)p.join[1] * Join<DV>::COLS;
    join<typename Tr::T, DV><<<tda::grid_of<256>(blocks), 256, 0, st>>>(p);
    tda::launched(st, "spa_join");
  }
  return (int)hipGetLastError();
}
template <class Tr>
static int pick(const AttendParams& p, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}

}  // namespace spa
