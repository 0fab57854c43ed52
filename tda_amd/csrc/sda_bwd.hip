// sda_bwd.hip -- softmax differential attention, backward.  With P_b the softmax maps, O_b = P_b v,
// dP = dO v^T, r_b = rowsum(dO O_b) and lambda per row:
//   dS_1 = P_1 (dP - r_1),  dS_2 = -lambda P_2 (dP - r_2),  dq_b = s dS_b k_b,  dk_b = s dS_b^T q_b,
//   dv = (P_1 - lambda P_2)^T dO,  dlambda_i = -r_2.
// The outputs' weights were rounded to bf16, so r_b is off by as much; dlambda gets its r_2 from the query pass,
// r_2 + rowsum(P_2 (dP - r_2)) of weights in f32 (bf16 (2, 16 over 4, 4096, 128): 2.4e-3 -> 1.7e-3 off, its
// own rounding).
// One dP and one dv product serve both branches.  r_1 comes from the outputs: dO O = r_1 - lambda r_2.
//
//   bwd_rows   r_1, r_2 and lambda of every row (f32)
//   bwd_keys   key-major: a wave owns 32 keys and walks the query rows that see them
//   bwd_query  query-major: a wave owns 32 query rows and walks the keys they see
//   bwd_sum    adds the key pass' partial sums where several workgroups share a key head
//   bwd_lambda sums dlambda over the axes lambda is broadcast along
// Both passes recompute the weights from the forward's log-sums: no atomics, so results do not depend
// on the order of execution.  Bound by the matrix cores and, for narrow keys, the vector work between the
// products.  bf16: (4, 16, 2048, 64/128) keys 242 us (0.57 PFLOP/s), queries 139 (0.74), rows 29, lambda 9;
// (2, 16 over 4, 4096, 128) keys 493 (0.84), sum 21, queries 392 (0.88), rows 36.  f32 (2, 12, 1111, 64) keys
// 133, queries 109 (0.08 PFLOP/s of 0.15).
#include "sda_common.hpp"

namespace sda {

__device__ __forceinline__ f32x4 load4h(const _Float16* p) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  const half4 v = *reinterpret_cast<const half4*>(p);
  return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <class T>
__device__ __forceinline__ f32x4 load4_(const T* p) {
  if constexpr (std::is_same_v<T, _Float16>) return load4h(p);
  else return tda::load4(p);
}

// ------------------------------------------------------------------ f16's range
// A weight or score gradient in f16 keeps its 11 bits only between 2^-14 and 2^16, so the f16 passes scale
// them by powers of two: score gradients so that the largest possible, |dS| <= 2 max|dO_i| max(1, |lambda_i|)
// max|v_j|, comes to 2^13 .. 2^14, weights by up to 2^8 (1 + max |lambda| leaves room).  peak holds the three
// maxima; bits of floats that are not negative order as integers do, so an atomic maximum has one result.
// Backward of (2, 16, 2048, 64): 236 us, bf16's 204; by f32 products it took 876.
struct Scales {
  float ds, w;  // score gradients by ds, weights by 2^w
};
template <class Tr>
__device__ __forceinline__ Scales scales(const BwdParams& P) {
  if constexpr (std::is_same_v<Tr, TrH>) {
    const float a = P.peak[0] * P.peak[1], l = 1.f + P.peak[2];
    const bool fits = a > 0x1p-100f && a < 0x1p100f;  // else nothing to scale by (zeros, NaN)
    return {fits ? exp2_(floorf(13.f - __builtin_amdgcn_logf(a))) : 1.f,
            l < 0x1p100f ? fminf(8.f, floorf(14.f - __builtin_amdgcn_logf(l))) : 0.f};
  } else {
    return {1.f, 0.f};
  }
}
__device__ __forceinline__ float larger(float a, float b) { return a != a ? a : b > a || b != b ? b : a; }  // a NaN stays
__device__ __forceinline__ void raise(float* to, float x) {  // what an older value exceeds already need not go out
  unsigned* at = reinterpret_cast<unsigned*>(to);
  const unsigned bits = __builtin_bit_cast(unsigned, x);
  if (bits > *const_cast<volatile unsigned*>(at)) atomicMax(at, bits);
}
__global__ void bwd_clear(BwdParams P) {
  if (threadIdx.x < 3) P.peak[threadIdx.x] = 0.f;
}
// max|v_j| over the rows that some row sees.  16 lanes per row, rows in strides of the grid.
template <int DV>
__global__ void __launch_bounds__(256) bwd_peak(BwdParams P) {
  const int64_t rows = (int64_t)P.B * P.Hk * P.Nk;
  const int c = threadIdx.x & 15;
  float top = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); row < rows; row += (int64_t)gridDim.x * 16) {
    const int j = (int)(row % P.Nk), b = (int)(row / P.Nk / P.Hk), h = (int)(row / P.Nk % P.Hk);
    const int len = len_of(P.see, b, P.Nk), lim = P.see.causal ? min(len, off_of(P.see, b) + P.Nq) : len;
    if (j >= lim) continue;  // whole rows: 16 lanes together
    const _Float16* v = row_of<_Float16>(P.v, b, h, j);
    float n = 0.f;
#pragma unroll
    for (int u = 0; u < DV / 64; ++u) {
      const f32x4 x = load4h(v + 64 * u + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) n = __builtin_fmaf(x[e], x[e], n);
    }
    n = tda::group_sum<16>(n);
    top = larger(top, n);
  }
  __shared__ float all[16];
  if (c == 0) all[threadIdx.x >> 4] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int x = 1; x < 16; ++x) top = larger(top, all[x]);
  raise(P.peak + 1, sqrtf(top));
}

// ------------------------------------------------------------------ row sums
// What the passes need of a row, so that it enters their products as a starting value: the log-sums as
// -lse_b / c (score and weight: P = 2^(c (q k - lse / c))), -r_1, r_1 - r_2, -lambda.
// 16 lanes per row, 16 rows per workgroup.
template <class T, int DV>
__global__ void __launch_bounds__(256) bwd_rows(BwdParams P) {
  const int64_t rows = (int64_t)P.B * P.H * P.Nq;
  const int c = threadIdx.x & 15;
  constexpr bool HALF = std::is_same_v<T, _Float16>;
  float top[2] = {0.f, 0.f};  // of this thread's rows
  const int64_t step = HALF ? (int64_t)gridDim.x * 16 : rows;  // f16: a few workgroups, for few atomic maxima
  for (int64_t row = (int64_t)tda::grid_bid<256>() * 16 + (threadIdx.x >> 4); row < rows; row += step) {
    const int i = (int)(row % P.Nq);
    const int64_t bh = row / P.Nq;
    const int b = (int)(bh / P.H), h = (int)(bh % P.H);
    const T* d = row_of<T>(P.dout, b, h, i);
    const T* x = row_of<T>(P.out, b, h, i);
    const float* y = row_of<float>(P.out2, b, h, i);
    const T* z = sizeof(T) == 2 ? row_of<T>(P.low, b, h, i) : nullptr;
    float rx = 0.f, ry = 0.f, n2 = 0.f;
#pragma unroll
    for (int u = 0; u < DV / 64; ++u) {
      const f32x4 dd = load4_(d + 64 * u + 4 * c), yy = load4_(y + 64 * u + 4 * c);
      f32x4 xx = load4_(x + 64 * u + 4 * c);
      if constexpr (sizeof(T) == 2) xx += load4_(z + 64 * u + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (HALF) n2 = __builtin_fmaf(dd[e], dd[e], n2);
        rx = __builtin_fmaf(dd[e], xx[e], rx);
        ry = __builtin_fmaf(dd[e], yy[e], ry);
      }
    }
    rx = tda::group_sum<16>(rx);
    ry = tda::group_sum<16>(ry);
    if constexpr (HALF) n2 = tda::group_sum<16>(n2);
    if (c == 0) {
      const float lam = lambda_of(P.lam, b, h, i), r1 = __builtin_fmaf(lam, ry, rx), inv = 1.0f / P.c;
      P.stat[row] = -P.lse[row] * inv;
      P.stat[rows + row] = -P.lse[rows + row] * inv;
      P.stat[2 * rows + row] = -r1;
      P.stat[3 * rows + row] = r1 - ry;
      P.stat[4 * rows + row] = -lam;
      if constexpr (HALF) {
        const int len = len_of(P.see, b, P.Nk);
        if ((P.see.causal ? min(len, off_of(P.see, b) + i + 1) : len) > 0) {  // a row that sees nothing counts for nothing
          top[0] = larger(top[0], sqrtf(n2) * fmaxf(1.f, fabsf(lam)));
          top[1] = larger(top[1], fabsf(lam));
        }
      }
    }
  }
  if constexpr (HALF) {
    __shared__ float peak[2][16];
    if (c == 0) peak[0][threadIdx.x >> 4] = top[0], peak[1][threadIdx.x >> 4] = top[1];
    __syncthreads();
    if (threadIdx.x < 2) {
      float all = 0.f;
      for (int x = 0; x < 16; ++x) all = larger(all, peak[threadIdx.x][x]);
      raise(P.peak + 2 * threadIdx.x, all);
    }
  }
}

// ------------------------------------------------------------------ key-major pass
// A workgroup has 4 waves: RH = 1 of 32 keys each, which walk the query rows that see them 32 at a time, or
// RH = 2 (few workgroups) pairs of waves on 32 keys, one on every other 32 rows, whose sums meet in LDS.
//
// Two workgroups of the narrowest key pass fit a CU (two waves a SIMD): the whole backward of bf16 (4, 16, 2048,
// 64) 374 -> 343 us.
template <class Tr, int D, int DV>
constexpr bool kKeyTwo = sizeof(typename Tr::T) == 2 && D == 64 && DV == 64;
// The branches one after the other with fewer registers: for two waves a SIMD, and where the sequence of both
// would spill (backward of bf16 (4, 16, 2048, 128/256) 1556 -> 958 us, f32 (2, 16, 2048, 64/128) 1104 -> 1033).
template <class Tr, int D, int DV>
constexpr bool kKeyLean = kKeyTwo<Tr, D, DV> || (sizeof(typename Tr::T) == 2 ? DV == 256 : DV >= 128);

template <class Tr, int D, int DV, int RH>
struct KeyShape {
  using QT = Tile<Tr, 32, D>;
  using OT = Tile<Tr, 32, DV>;
  static constexpr int STAT = 2 * QT::BYTES + OT::BYTES;  // the statistics of the 32 rows
  static constexpr int TILE = STAT + 1024;
  static constexpr int STAGE = RH * TILE;               // of two, one on its way
  static constexpr int XCH = (RH - 1) * 2 * 32 * (2 * D + DV) * 4;  // the second half's sums
  static constexpr int LDS = 2 * STAGE > XCH ? 2 * STAGE : XCH;
  static constexpr int NW = 4, KEYS = 32 * NW / RH;
};

// One wave per SIMD (the three gradients' accumulators and the resident rows fill the registers), so
// the wave hides its own latencies: the LDS operands of a step are one sequence, read a group ahead of their
// use, and the first branch's weights are computed between the second's score products, the second's
// between the first's gradient products.
template <class Tr, int D, int DV, int RH>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu((kKeyTwo<Tr, D, DV> ? 2 : 1)))) bwd_keys(BwdParams P) {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  using S = KeyShape<Tr, D, DV, RH>;
  using QT = typename S::QT;
  using OT = typename S::OT;
  constexpr bool LEAN = kKeyLean<Tr, D, DV>;
  constexpr int NT = D / 16, NV = DV / 16, NW = S::NW, QL = (QT::LOADS + NW - 1) / NW, OL = (OT::LOADS + NW - 1) / NW;
  constexpr int G = sizeof(T) == 4 ? 1 : LEAN ? 2 : 4;  // an fp32 fragment is eight products itself
  // The statistics enter the products as their starting values; f32 adds them after, where a sum that starts
  // far from zero would cost it bits.
  constexpr bool START = sizeof(T) == 2;
  constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1;
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int l = lane_id(), n32 = l & 31, g = l >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rh = RH == 1 ? 0 : wv / (NW / RH);
  const int GQ = P.H / P.Hk, parts = GQ / P.gs, nkt = (P.Nk + S::KEYS - 1) / S::KEYS;
  const uint32_t bid = tda::grid_bid<64 * NW>(), heads = (uint32_t)(P.B * P.Hk) * (uint32_t)parts;
  if (bid >= heads * (uint32_t)nkt) return;
  const Item it = item_of(bid, heads, nkt, false);
  const int part = it.head % parts, bk = it.head / parts, b = bk / P.Hk, hk = bk % P.Hk;
  const int h0 = hk * GQ + part * P.gs;
  const int k0 = it.tile * S::KEYS, k0w = k0 + 32 * (wv % (NW / RH)), key = k0w + n32;
  const int len = len_of(P.see, b, P.Nk), off = off_of(P.see, b);
  const bool live = key < (P.see.causal ? min(len, off + P.Nq) : len);  // some row sees it; others' rows may hold anything
  const int64_t rows = (int64_t)P.B * P.H * P.Nq;

  // query tiles of 32 rows, RH a step: from the first that sees the workgroup's first key on
  const int nqt = (P.Nq + 31) / 32;
  const int first = P.see.causal ? max(k0 - off, 0) >> 5 : 0;
  const int per = k0 < len ? max(nqt - first + RH - 1, 0) / RH : 0;
  const int steps = per * P.gs;

  uint32_t qo[2][QL], oo[OL];
#pragma unroll
  for (int u = 0; u < QL; ++u) {
    qo[0][u] = QT::source(NW * u + wv, (uint32_t)(P.q[0].st * QT::ES));
    qo[1][u] = QT::source(NW * u + wv, (uint32_t)(P.q[1].st * QT::ES));
  }
#pragma unroll
  for (int u = 0; u < OL; ++u) oo[u] = OT::source(NW * u + wv, (uint32_t)(P.dout.st * OT::ES));
  auto issue = [&](char* at, int h, int qt) {  // query tile qt of head h
    const int i0 = 32 * qt, n = max(min(32, P.Nq - i0), 0);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto r = rows_rsrc(row_of<T>(P.q[x], b, h, i0), P.q[x].st * QT::ES, n, D * QT::ES);
#pragma unroll
      for (int u = 0; u < QL; ++u)
        if (QT::LOADS % NW == 0 || NW * u + wv < QT::LOADS) QT::load(r, reinterpret_cast<T*>(at + x * QT::BYTES), NW * u + wv, qo[x][u]);
    }
    const auto r = rows_rsrc(row_of<T>(P.dout, b, h, i0), P.dout.st * OT::ES, n, DV * OT::ES);
#pragma unroll
    for (int u = 0; u < OL; ++u)
      if (OT::LOADS % NW == 0 || NW * u + wv < OT::LOADS) OT::load(r, reinterpret_cast<T*>(at + 2 * QT::BYTES), NW * u + wv, oo[u]);
    // the rows' statistics, two loads a wave (the last three bring the fifth again: every wave's loads of a
    // stage are as many); rows past Nq read as zeros and meet zero rows of q and dO, whose rows do not
    // overlap (sda_validate_bwd)
    const float* src = P.stat + ((int64_t)b * P.H + h) * P.Nq + i0;
#pragma unroll
    for (int z = 0; z < 8; z += NW)
      if (l < 32)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src + min(z + wv, 4) * rows, 4 * n), LDS_PTR(void, at + S::STAT + 128 * (z + wv)), 4, 4 * l, 0, 0, 0);
  };
  int nh = h0, nq = first;  // head and query tile of the next stage to send for
  auto send = [&](int slot) {
#pragma unroll
    for (int s = 0; s < RH; ++s) issue(lds + slot * S::STAGE + s * S::TILE, nh, nq + s);
    nq += RH;
    if (nq >= nqt) nq = first, ++nh;
  };
  if (steps > 0) send(0);

  frag kf[2][NT], vf[NV];
#pragma unroll
  for (int x = 0; x < 2; ++x) load_frags<Tr, NT>(live ? row_of<T>(P.k[x], b, hk, key) : nullptr, g, kf[x]);
  load_frags<Tr, NV>(live ? row_of<T>(P.v, b, hk, key) : nullptr, g, vf);
  const Scales by = scales<Tr>(P);
  constexpr bool HALF = std::is_same_v<Tr, TrH>;
  const float dsw = HALF ? by.ds * exp2_(-by.w) : 1.f;  // from a scaled weight to a scaled score gradient
  f32x16 dk[2][D / 32] = {}, dv[DV / 32] = {};
  pin(dk[0]);
  pin(dk[1]);
  pin(dv);

  RowReader<Tr, D> qr;
  RowReader<Tr, DV> orow;
  ColReader<Tr, D> qc;
  ColReader<Tr, DV> oc;
  char* qb = lds + rh * S::TILE;
  char* ot = qb + 2 * QT::BYTES;
  qr.init(qb);
  qc.init(qb);
  orow.init(ot);
  oc.init(ot);
  auto step = [&](int i0, auto half) {  // the stage in that half of the buffers
    constexpr int AT = half * S::STAGE;
    const bool edge = P.see.causal && off + i0 < k0w + 31;  // some row does not see some key
    const float* st = reinterpret_cast<const float*>(qb + AT + S::STAT);
    // the sequence: dO rows (dP), q1 rows, q2 rows (scores), q1 columns (dk1), q2 columns (dk2), dO columns (dv)
    constexpr int E1 = NV, E2 = E1 + NT, E3 = E2 + NT, E4 = E3 + D / 16, E5 = E4 + D / 16, E6 = E5 + DV / 16;
    frag f[AHEAD + 1][G];
    auto read = [&](auto i) {  // group i of it
      times<G>([&](auto u) {
        constexpr int e = i * G + u;
        frag& to = f[i % (AHEAD + 1)][u];
        if constexpr (e < E1) to = orow.read(ot, AT, e);
        else if constexpr (e < E2) to = qr.read(qb, AT, e - E1);
        else if constexpr (e < E3) to = qr.read(qb, AT + QT::BYTES, e - E2);
        else if constexpr (e < E4) to = qc.read(qb, AT, (e - E3) / (D / 32), (e - E3) % (D / 32));
        else if constexpr (e < E5) to = qc.read(qb, AT + QT::BYTES, (e - E4) / (D / 32), (e - E4) % (D / 32));
        else to = oc.read(ot, AT, (e - E5) / (DV / 32), (e - E5) % (DV / 32));
      });
    };
    auto rowstat = [&](int z) {  // statistic z of the lane's 16 rows
      f32x16 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(st + 32 * z + 8 * r + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * r + e] = w[e];
      }
      return x;
    };
    times<AHEAD>([&](auto i) { read(i); });
    f32x16 dp = START ? rowstat(2) : f32x16{}, s[2], w, dif, lam;
    frag ds[2][2], wf[2];
    auto hide = [&](f32x16& x) {
      if (edge) {
        asm volatile("");  // a branch: few tiles need this
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = key > off + i0 + crow(r, g) ? -__builtin_inff() : x[r];
      }
    };
    auto weight = [&](int x, int r) {
      return HALF ? exp2_(__builtin_fmaf(P.c, s[x][r], by.w)) : START ? exp2_(P.c * s[x][r]) : exp2_(__builtin_fmaf(P.c, s[x][r], P.c * st[32 * x + crow(r, g)]));
    };
    auto first_branch = [&](int r) {
      const float p = weight(0, r);
      w[r] = p;
      s[0][r] = p * (START ? dp[r] : dp[r] + st[64 + crow(r, g)]);
      if constexpr (HALF) s[0][r] *= dsw;
    };
    auto second_branch = [&](int r) {
      const float p = lam[r] * weight(1, r);
      w[r] += p;
      s[1][r] = p * (START ? dp[r] + dif[r] : dp[r] + (dif[r] + st[64 + crow(r, g)]));
      if constexpr (HALF) s[1][r] *= dsw;
    };
    constexpr int NG = E6 / G;
    times<NG>([&](auto i) {
      if constexpr (i + AHEAD < NG) read(std::integral_constant<int, i + AHEAD>());
      if constexpr (i * G == E2) hide(s[0]);
      if constexpr (i * G == E3) hide(s[1]);
      if constexpr (i * G == E1 - G) s[0] = START ? rowstat(0) : f32x16{};
      if constexpr (i * G == E2 - G) s[1] = START ? rowstat(1) : f32x16{};
      if constexpr (i * G == E3 - G) dif = rowstat(3), lam = rowstat(4);
      __builtin_amdgcn_sched_barrier(0);
      times<G>([&](auto u) {
        constexpr int e = i * G + u;
        const frag& a = f[i % (AHEAD + 1)][u];
        if constexpr (e < E1) dp = Tr::mma32(a, vf[e], dp);
        else if constexpr (e < E2) s[0] = Tr::mma32(a, kf[0][e - E1], s[0]);
        else if constexpr (e < E3) s[1] = Tr::mma32(a, kf[1][e - E2], s[1]);
        else if constexpr (e < E4) dk[0][(e - E3) % (D / 32)] = Tr::mma32(a, ds[0][(e - E3) / (D / 32)], dk[0][(e - E3) % (D / 32)]);
        else if constexpr (e < E5) dk[1][(e - E4) % (D / 32)] = Tr::mma32(a, ds[1][(e - E4) / (D / 32)], dk[1][(e - E4) % (D / 32)]);
        else dv[(e - E5) % (DV / 32)] = Tr::mma32(a, wf[(e - E5) / (DV / 32)], dv[(e - E5) % (DV / 32)]);
        // between them, the weights: 16 rows over the segment's products
        if constexpr (e >= E2 && e < E3) {
          constexpr int n = 16 / NT;
          times<n>([&](auto r) { first_branch((e - E2) * n + r); });
          if constexpr (e == E3 - 1) ds[0][0] = pack8<Tr>(s[0], 0), ds[0][1] = pack8<Tr>(s[0], 1);
        }
        if constexpr (e >= E3 && e < E4) {
          constexpr int n = 16 / (D / 16);
          times<n>([&](auto r) { second_branch((e - E3) * n + r); });
          if constexpr (e == E4 - 1) {
            ds[1][0] = pack8<Tr>(s[1], 0), ds[1][1] = pack8<Tr>(s[1], 1);
            wf[0] = pack8<Tr>(w, 0), wf[1] = pack8<Tr>(w, 1);
          }
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // The same with fewer registers: the branches one after the other.
  auto lean = [&](int i0, auto half) {
    constexpr int AT = half * S::STAGE;
    const bool edge = P.see.causal && off + i0 < k0w + 31;
    const float* st = reinterpret_cast<const float*>(qb + AT + S::STAT) + 4 * g;
    constexpr int E1 = NV, E2 = E1 + NT, E3 = E2 + D / 16, E4 = E3 + NT, E5 = E4 + D / 16, E6 = E5 + DV / 16;
    frag f[2][G];
    auto read = [&](auto i) {
      times<G>([&](auto u) {
        constexpr int e = i * G + u;
        frag& to = f[i % 2][u];
        if constexpr (e < E1) to = orow.read(ot, AT, e);
        else if constexpr (e < E2) to = qr.read(qb, AT, e - E1);
        else if constexpr (e < E3) to = qc.read(qb, AT, (e - E2) / (D / 32), (e - E2) % (D / 32));
        else if constexpr (e < E4) to = qr.read(qb, AT + QT::BYTES, e - E3);
        else if constexpr (e < E5) to = qc.read(qb, AT + QT::BYTES, (e - E4) / (D / 32), (e - E4) % (D / 32));
        else to = oc.read(ot, AT, (e - E5) / (DV / 32), (e - E5) % (DV / 32));
      });
    };
    auto rowstat = [&](int z) {
      f32x16 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(st + 32 * z + 8 * r);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * r + e] = y[e];
      }
      return x;
    };
    auto hide = [&](f32x16& x) {
      if (edge) {
        asm volatile("");  // a branch: few tiles need this
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = key > off + i0 + crow(r, g) ? -__builtin_inff() : x[r];
      }
    };
    read(std::integral_constant<int, 0>());
    f32x16 dp = START ? rowstat(2) : f32x16{}, sc, w;
    frag ds[2];
    constexpr int NG = E6 / G;
    times<NG>([&](auto i) {
      if constexpr (i + 1 < NG) read(std::integral_constant<int, i + 1>());
      if constexpr (i * G == E1) sc = START ? rowstat(0) : f32x16{};
      if constexpr (i * G == E3) sc = START ? rowstat(1) : f32x16{};
      if constexpr (i * G == E2) {  // the first branch's weights
        hide(sc);
        if constexpr (!START) dp += rowstat(2), sc += rowstat(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          w[r] = HALF ? exp2_(__builtin_fmaf(P.c, sc[r], by.w)) : exp2_(P.c * sc[r]);
          sc[r] = w[r] * dp[r];
          if constexpr (HALF) sc[r] *= dsw;
        }
        ds[0] = pack8<Tr>(sc, 0), ds[1] = pack8<Tr>(sc, 1);
      }
      if constexpr (i * G == E4) {  // the second's
        hide(sc);
        if constexpr (!START) sc += rowstat(1);
        dp += rowstat(3);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 lam = *reinterpret_cast<const f32x4*>(st + 128 + 8 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * q + e;
            const float p = lam[e] * (HALF ? exp2_(__builtin_fmaf(P.c, sc[r], by.w)) : exp2_(P.c * sc[r]));
            w[r] += p;
            sc[r] = p * dp[r];
            if constexpr (HALF) sc[r] *= dsw;
          }
        }
        ds[0] = pack8<Tr>(sc, 0), ds[1] = pack8<Tr>(sc, 1);
      }
      if constexpr (i * G == E5) ds[0] = pack8<Tr>(w, 0), ds[1] = pack8<Tr>(w, 1);
      __builtin_amdgcn_sched_barrier(0);
      times<G>([&](auto u) {
        constexpr int e = i * G + u;
        const frag& a = f[i % 2][u];
        if constexpr (e < E1) dp = Tr::mma32(a, vf[e], dp);
        else if constexpr (e < E2) sc = Tr::mma32(a, kf[0][e - E1], sc);
        else if constexpr (e < E3) dk[0][(e - E2) % (D / 32)] = Tr::mma32(a, ds[(e - E2) / (D / 32)], dk[0][(e - E2) % (D / 32)]);
        else if constexpr (e < E4) sc = Tr::mma32(a, kf[1][e - E3], sc);
        else if constexpr (e < E5) dk[1][(e - E4) % (D / 32)] = Tr::mma32(a, ds[(e - E4) / (D / 32)], dk[1][(e - E4) % (D / 32)]);
        else dv[(e - E5) % (DV / 32)] = Tr::mma32(a, ds[(e - E5) / (DV / 32)], dv[(e - E5) % (DV / 32)]);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int qt = first;  // of this step
  auto one = [&](int j, auto slot) {
    wait_vm<0>();
    tda::lds_barrier();
    if (j + 1 < steps) send(1 - slot);
    const int i0 = 32 * (qt + rh);
    if (i0 < P.Nq && (!P.see.causal || off + min(i0 + 31, P.Nq - 1) >= k0w)) {
      if constexpr (LEAN) lean(i0, slot);
      else step(i0, slot);
    }
    qt += RH;
    if (qt >= nqt) qt = first;
  };
  for (int j = 0; j < steps; j += 2) {
    one(j, std::integral_constant<int, 0>());
    if (j + 1 < steps) one(j + 1, std::integral_constant<int, 1>());
  }
  wait_vm<0>();

  if constexpr (RH == 2) {  // the second half's sums join the first's
    constexpr int N = (2 * D + DV) / 32 * 4;  // pieces of four values a lane
    f32x4* x4 = reinterpret_cast<f32x4*>(lds) + (wv & 1) * (N * 64) + l;
    __syncthreads();
    if (rh)
      times<N>([&](auto i) {
        constexpr int y = i / 4, r = 4 * (i % 4), W = D / 32;
        const f32x16& a = y < W ? dk[0][y % W] : y < 2 * W ? dk[1][y % W] : dv[y < 2 * W ? 0 : y - 2 * W];
        x4[i * 64] = f32x4{a[r], a[r + 1], a[r + 2], a[r + 3]};
      });
    __syncthreads();
    if (rh) return;
    times<N>([&](auto i) {
      constexpr int y = i / 4, r = 4 * (i % 4), W = D / 32;
      f32x16& a = y < W ? dk[0][y % W] : y < 2 * W ? dk[1][y % W] : dv[y < 2 * W ? 0 : y - 2 * W];
      const f32x4 w = x4[i * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) a[r + e] += w[e];
    });
  }
  if (key >= P.Nk) return;
  const float back = HALF ? P.scale / by.ds : P.scale, backw = HALF ? exp2_(-by.w) : 1.f;
  // a key that no row sees met weights of its own making (of a zero row): its column holds nothing else
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < D / 32; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[x][y][r] = live ? dk[x][y][r] * back : 0.f;
#pragma unroll
  for (int y = 0; y < DV / 32; ++y)
#pragma unroll
    for (int r = 0; r < 16; ++r) dv[y][r] = live ? (HALF ? dv[y][r] * backw : dv[y][r]) : 0.f;
  constexpr int W = 2 * D + DV;
  float* pt = P.part ? P.part + (((int64_t)part * P.B * P.Hk + bk) * P.Nk + key) * W + 4 * g : nullptr;  // dk1, dk2, dv, f32
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    T* to = row_of<T>(P.dk[x], b, hk, key) + 4 * g;
#pragma unroll
    for (int y = 0; y < D / 32; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 z = {dk[x][y][4 * r], dk[x][y][4 * r + 1], dk[x][y][4 * r + 2], dk[x][y][4 * r + 3]};
        if (pt) store4(pt + x * D + 32 * y + 8 * r, z);
        else store4(to + 32 * y + 8 * r, z);
      }
  }
  T* to = row_of<T>(P.dv, b, hk, key) + 4 * g;
#pragma unroll
  for (int y = 0; y < DV / 32; ++y)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 z = {dv[y][4 * r], dv[y][4 * r + 1], dv[y][4 * r + 2], dv[y][4 * r + 3]};
      if (pt) store4(pt + 2 * D + 32 * y + 8 * r, z);
      else store4(to + 32 * y + 8 * r, z);
    }
}

// Sum of the groups' partial rows, in group order.  One thread per 4 values.
template <class T, int D, int DV>
__global__ void __launch_bounds__(256) bwd_sum(BwdParams P, int parts) {
  constexpr int W = 2 * D + DV, C = W / 4;
  const int64_t rows = (int64_t)P.B * P.Hk * P.Nk, id = (int64_t)tda::grid_bid<256>() * 256 + threadIdx.x;
  const int64_t row = id / C;
  const int c = 4 * (int)(id % C);
  if (row >= rows) return;
  f32x4 a = *reinterpret_cast<const f32x4*>(P.part + row * W + c);
  for (int x = 1; x < parts; ++x) a += *reinterpret_cast<const f32x4*>(P.part + (x * rows + row) * W + c);
  const int key = (int)(row % P.Nk), b = (int)(row / P.Nk / P.Hk), h = (int)(row / P.Nk % P.Hk);
  const Rows& to = c < D ? P.dk[0] : c < 2 * D ? P.dk[1] : P.dv;
  store4(row_of<T>(to, b, h, key) + (c < D ? c : c < 2 * D ? c - D : c - 2 * D), a);
}

// ------------------------------------------------------------------ query-major pass
// A workgroup has RG groups of 32 query rows, a wave for each (SPLIT: and for each branch); with RG = 2 (few
// workgroups) two such sets take alternate tiles of 32 keys, and their sums meet in LDS.
template <class Tr, int D, int DV, bool SPLIT, int RG>
struct QueryShape {
  using KT = Tile<Tr, 32, D>;
  using VT = Tile<Tr, 32, DV>;
  static constexpr int WAVES = SPLIT ? 8 : 4;
  static constexpr int KH = 4 / RG, TILE = 2 * KT::BYTES + VT::BYTES, STAGE = KH * TILE;
  static constexpr int LDS = 2 * STAGE;  // a half's sums need less
  static constexpr int KL = (KT::LOADS + WAVES - 1) / WAVES, VL = (VT::LOADS + WAVES - 1) / WAVES;
};

template <class Tr, int D, int DV, bool SPLIT, int RG>
__global__ void __launch_bounds__(SPLIT ? 512 : 256) __attribute__((amdgpu_waves_per_eu(SPLIT || (sizeof(typename Tr::T) == 2 && D == 64) ? 2 : 1))) bwd_query(BwdParams P) {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  using S = QueryShape<Tr, D, DV, SPLIT, RG>;
  using KT = typename S::KT;
  using VT = typename S::VT;
  constexpr int NT = D / 16, NV = DV / 16, KL = S::KL, VL = S::VL, NW = S::WAVES, NB = SPLIT ? 1 : 2, KH = S::KH, ROWS = 32 * RG;
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int l = lane_id(), n32 = l & 31, g = l >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wv % RG;
  const int br = SPLIT ? wv / RG & 1 : 0, kh = RG == 4 ? 0 : wv / (NW / KH);  // kh: which of a stage's key tiles
  const int nqt = (P.Nq + ROWS - 1) / ROWS;
  const uint32_t bid = tda::grid_bid<64 * NW>();
  if (bid >= (uint32_t)(P.B * P.H) * (uint32_t)nqt) return;
  const Item it = item_of(bid, P.B * P.H, nqt, true);
  const int b = it.head / P.H, h = it.head % P.H, hk = h / (P.H / P.Hk);
  const int q0 = it.tile * ROWS, q0w = q0 + 32 * rg, qi = q0w + n32;
  const int len = len_of(P.see, b, P.Nk), off = off_of(P.see, b);
  const int lim = P.see.causal ? min(len, max(off + min(q0 + ROWS, P.Nq), 0)) : len;
  const int limw = P.see.causal ? min(len, max(off + min(q0w + 32, P.Nq), 0)) : len;
  const int clear = P.see.causal ? min(len, max(off + q0w + 1, 0)) : len;
  const int see = P.see.causal ? min(len, off + qi + 1) : len;
  const int nst = (lim + 32 * KH - 1) / (32 * KH);
  const int64_t rows = (int64_t)P.B * P.H * P.Nq;

  uint32_t ko[2][KL], vo[VL];
#pragma unroll
  for (int u = 0; u < KL; ++u) {
    ko[0][u] = KT::source(NW * u + wv, (uint32_t)(P.k[0].st * KT::ES));
    ko[1][u] = KT::source(NW * u + wv, (uint32_t)(P.k[1].st * KT::ES));
  }
#pragma unroll
  for (int u = 0; u < VL; ++u) vo[u] = VT::source(NW * u + wv, (uint32_t)(P.v.st * VT::ES));
  auto tile = [&](char* at, int j) {  // key tile j
    const int n = min(32, lim - 32 * j);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto r = rows_rsrc(row_of<T>(P.k[x], b, hk, 32 * (int64_t)j), P.k[x].st * KT::ES, n, D * KT::ES);
#pragma unroll
      for (int u = 0; u < KL; ++u)
        if (KT::LOADS % NW == 0 || NW * u + wv < KT::LOADS) KT::load(r, reinterpret_cast<T*>(at + x * KT::BYTES), NW * u + wv, ko[x][u]);
    }
    const auto r = rows_rsrc(row_of<T>(P.v, b, hk, 32 * (int64_t)j), P.v.st * VT::ES, n, DV * VT::ES);
#pragma unroll
    for (int u = 0; u < VL; ++u)
      if (VT::LOADS % NW == 0 || NW * u + wv < VT::LOADS) VT::load(r, reinterpret_cast<T*>(at + 2 * KT::BYTES), NW * u + wv, vo[u]);
  };
  auto issue = [&](int j) {
#pragma unroll
    for (int s = 0; s < KH; ++s) tile(lds + (j & 1) * S::STAGE + s * S::TILE, KH * j + s);
  };
  if (nst > 0) issue(0);

  const bool row = qi < P.Nq;
  frag qf[NB][NT], of[NV];
#pragma unroll
  for (int x = 0; x < NB; ++x) load_frags<Tr, NT>(row ? row_of<T>(P.q[SPLIT ? br : x], b, h, qi) : nullptr, g, qf[x]);
  load_frags<Tr, NV>(row ? row_of<T>(P.dout, b, h, qi) : nullptr, g, of);
  const int64_t at0 = (int64_t)it.head * P.Nq + qi;
  float lse[NB], rs[NB], lam = 0.f;
#pragma unroll
  for (int x = 0; x < NB; ++x) {
    const int z = SPLIT ? br : x;
    lse[x] = row ? -P.c * P.stat[z * rows + at0] : 0.f;
    rs[x] = row ? -P.stat[2 * rows + at0] - (z ? P.stat[3 * rows + at0] : 0.f) : 0.f;
  }
  if (row) lam = -P.stat[4 * rows + at0];
  float more = 0.f;  // rowsum(P_2 (dP - r_2))
  const float ds = scales<Tr>(P).ds;
  constexpr bool HALF = std::is_same_v<Tr, TrH>;
  f32x16 dq[NB][D / 32] = {};
  if constexpr (!SPLIT) {
    pin(dq[0]);
    pin(dq[1]);
  }

  RowReader<Tr, D> kr;
  RowReader<Tr, DV> vr;
  ColReader<Tr, D> kc;
  const char* kbuf = lds + kh * S::TILE + (SPLIT ? br * KT::BYTES : 0);  // the wave's own branch of the keys
  const char* vbuf = lds + kh * S::TILE + 2 * KT::BYTES;
  kr.init(kbuf);
  kc.init(kbuf);
  vr.init(vbuf);
  auto step = [&](int j, auto half) {  // stage j, in that half of the buffers
    constexpr int AT = half * S::STAGE;
    wait_vm<0>();
    tda::lds_barrier();
    if (j + 1 < nst) issue(j + 1);
    const int k0 = 32 * (KH * j + kh);
    if (k0 >= limw) return;
    const f32x16 dp = chain<Tr, NV>([&](int t) { return vr.read(vbuf, AT, t); }, of);
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      const int z = SPLIT ? br : x, kt = AT + x * KT::BYTES;
      f32x16 s = chain<Tr, NT>([&](int t) { return kr.read(kbuf, kt, t); }, qf[x]);
      const float f = HALF ? -lam * ds : -lam;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_(__builtin_fmaf(s[r], P.c, -lse[x]));
        s[r] = p * (dp[r] - rs[x]);
      }
      if (k0 + 32 > clear) {
        asm volatile("");  // a branch: few tiles need this
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + crow(r, g) >= see) s[r] = 0.f;
      }
      if (z) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          more += s[r];
          s[r] *= f;
        }
      } else if constexpr (HALF) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= ds;
      }
      const frag e[2] = {pack8<Tr>(s, 0), pack8<Tr>(s, 1)};
      columns<Tr, D / 32>([&](int u, int y) { return kc.read(kbuf, kt, u, y); }, e, dq[x]);
    }
  };
  for (int j = 0; j < nst; j += 2) {
    step(j, std::integral_constant<int, 0>());
    if (j + 1 < nst) step(j + 1, std::integral_constant<int, 1>());
  }
  wait_vm<0>();
  if constexpr (KH == 2) {  // the second half's sums join the first's
    constexpr int N = NB * D / 32 * 4;
    f32x4* x4 = reinterpret_cast<f32x4*>(lds) + wv % (NW / KH) * (N * 64) + l;
    float* xm = reinterpret_cast<float*>(lds + NW / KH * N * 1024) + wv % (NW / KH) * 64 + l;
    static_assert(NW / KH * (N * 1024 + 256) <= S::LDS, "the second half's sums fit");
    __syncthreads();
    if (kh) {
      *xm = more;
      times<N>([&](auto i) {
        constexpr int x = i / 4 / (D / 32), y = i / 4 % (D / 32), r = 4 * (i % 4);
        x4[i * 64] = f32x4{dq[x][y][r], dq[x][y][r + 1], dq[x][y][r + 2], dq[x][y][r + 3]};
      });
    }
    __syncthreads();
    if (kh) return;
    more += *xm;
    times<N>([&](auto i) {
      constexpr int x = i / 4 / (D / 32), y = i / 4 % (D / 32), r = 4 * (i % 4);
      const f32x4 w = x4[i * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) dq[x][y][r + e] += w[e];
    });
  }
  more += __shfl_xor(more, 32);
  if (!row) return;
  if ((!SPLIT || br) && g == 0) P.stat[5 * rows + at0] = rs[NB - 1] + more;
  const float back = HALF ? P.scale / ds : P.scale;
#pragma unroll
  for (int x = 0; x < NB; ++x) {
    T* to = row_of<T>(P.dq[SPLIT ? br : x], b, h, qi) + 4 * g;
#pragma unroll
    for (int y = 0; y < D / 32; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        store4(to + 32 * y + 8 * r, f32x4{dq[x][y][4 * r] * back, dq[x][y][4 * r + 1] * back, dq[x][y][4 * r + 2] * back, dq[x][y][4 * r + 3] * back});
  }
}

// ------------------------------------------------------------------ dlambda
// Minus the sums of r_2 over the axes lambda is broadcast along, each thread's share in order and the
// threads' by a fixed tree.  Where that takes in the rows of a head, each head's are summed first (over
// the first of the row statistics, which no pass reads any more): one workgroup a head.
__global__ void __launch_bounds__(1024) bwd_lambda_heads(BwdParams P) {
  const int64_t bh = tda::grid_bid<1024>(), rows = (int64_t)P.B * P.H * P.Nq;
  if (bh >= (int64_t)P.B * P.H) return;
  const float* r2 = P.stat + 5 * rows + bh * P.Nq;
  __shared__ float part[16];
  float a[4] = {};
  for (int i = threadIdx.x; i < P.Nq; i += 4096) {
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] += i + 1024 * u < P.Nq ? r2[i + 1024 * u] : 0.f;
  }
  const float w = tda::wave_sum((a[0] + a[1]) + (a[2] + a[3]));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x) return;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < 16; ++u) sum += part[u];
  P.stat[bh] = sum;
}
// One thread an element (b, h, i), or a wave where an element has whole heads (HEADS: r_2 is summed by
// head).
template <bool HEADS>
__global__ void __launch_bounds__(256) bwd_lambda(BwdParams P) {
  const int64_t rows = (int64_t)P.B * P.H * P.Nq, all = P.dlam_n[0] * P.dlam_n[1] * P.dlam_n[2];
  const int64_t id = (int64_t)tda::grid_bid<256>() * 256 + threadIdx.x, e = HEADS ? id >> 6 : id;
  if (e >= all) return;
  const float* from = HEADS ? P.stat : P.stat + 5 * rows;
  const int64_t N = HEADS ? 1 : P.Nq;
  const int64_t i0 = HEADS ? 0 : e % P.dlam_n[2], h0 = e / P.dlam_n[2] % P.dlam_n[1], b0 = e / P.dlam_n[2] / P.dlam_n[1];
  const int nb = P.dlam_n[0] == 1 ? P.B : 1, nh = P.dlam_n[1] == 1 ? P.H : 1;
  float a = 0.f;
  for (int x = HEADS ? (int)(id & 63) : 0; x < nb * nh; x += HEADS ? 64 : 1)
    a -= from[((b0 + x / nh) * P.H + h0 + x % nh) * N + i0];
  if constexpr (HEADS) {
    a = tda::wave_sum(a);
    if (id & 63) return;
  }
  if (P.lam.type == 0) static_cast<float*>(P.dlam)[e] = a;
  else if (P.lam.type == 1) static_cast<bf16*>(P.dlam)[e] = (bf16)a;
  else static_cast<_Float16*>(P.dlam)[e] = (_Float16)a;
}

// ------------------------------------------------------------------ launches
template <class F>
static int big_lds(F* fn, int bytes) {
  if (bytes <= 65536) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <class Tr, int D, int DV, int RH>
static int keys(const BwdParams& p, int parts, hipStream_t st) {
  using S = KeyShape<Tr, D, DV, RH>;
  if (const int e = big_lds(&bwd_keys<Tr, D, DV, RH>, S::LDS)) return e;
  bwd_keys<Tr, D, DV, RH><<<tda::grid_of<64 * S::NW>((int64_t)((p.Nk + S::KEYS - 1) / S::KEYS) * p.B * p.Hk * parts), 64 * S::NW, S::LDS, st>>>(p);
  tda::launched(st, "sda_bwd_keys");
  return 0;
}
template <class Tr, int D, int DV, int RG>
static int queries(const BwdParams& p, hipStream_t st) {
  // A wave for each branch where both branches' registers leave no room for the rest: bf16 (128, 128) 297 us
  // against 314 for the whole backward of (2, 16, 2048); (128, 256) 505 against 473, f32 (64, 64) 946 against 880.
  constexpr bool SPLIT = sizeof(typename Tr::T) == 2 && D == 128 && DV == 128;
  using S = QueryShape<Tr, D, DV, SPLIT, RG>;
  if (const int e = big_lds(&bwd_query<Tr, D, DV, SPLIT, RG>, S::LDS)) return e;
  bwd_query<Tr, D, DV, SPLIT, RG><<<tda::grid_of<64 * S::WAVES>((int64_t)((p.Nq + 32 * RG - 1) / (32 * RG)) * p.B * p.H), 64 * S::WAVES, S::LDS, st>>>(p);
  tda::launched(st, "sda_bwd_query");
  return 0;
}
template <class Tr, int D, int DV>
static int run(const BwdParams& p, hipStream_t st) {
  using T = typename Tr::T;
  const int64_t rows = (int64_t)p.B * p.H * p.Nq;
  if constexpr (std::is_same_v<Tr, TrH>) {
    bwd_clear<<<1, 64, 0, st>>>(p);
    const int64_t keys = ((int64_t)p.B * p.Hk * p.Nk + 15) / 16;
    bwd_peak<DV><<<(unsigned)(keys < 1024 ? keys : 1024), 256, 0, st>>>(p);
    tda::launched(st, "sda_bwd_peak");
  }
  const int64_t sets = (rows + 15) / 16;
  bwd_rows<T, DV><<<std::is_same_v<Tr, TrH> ? dim3((unsigned)(sets < 2048 ? sets : 2048)) : tda::grid_of<256>(sets), 256, 0, st>>>(p);
  tda::launched(st, "sda_bwd_rows");
  const int parts = p.H / p.Hk / p.gs;
  int e = -1;
  if constexpr (KeyShape<Tr, D, DV, 2>::LDS <= kLds) {
    if (halve<Tr, D, DV>(p.see, (int64_t)((p.Nk + 127) / 128) * p.B * p.Hk * parts, p.Nq)) e = keys<Tr, D, DV, 2>(p, parts, st);
  }
  if (e < 0) e = keys<Tr, D, DV, 1>(p, parts, st);
  if (e) return e;
  if (p.part) {
    const int64_t n = (int64_t)p.B * p.Hk * p.Nk * ((2 * D + DV) / 4);
    bwd_sum<T, D, DV><<<tda::grid_of<256>((n + 255) / 256), 256, 0, st>>>(p, parts);
    tda::launched(st, "sda_bwd_sum");
  }
  e = -1;
  if constexpr (QueryShape<Tr, D, DV, false, 2>::LDS <= kLds) {
    if (halve<Tr, D, DV>(p.see, (int64_t)((p.Nq + 127) / 128) * p.B * p.H, p.Nq)) e = queries<Tr, D, DV, 2>(p, st);
  }
  if (e < 0) e = queries<Tr, D, DV, 4>(p, st);
  if (e) return e;
  if (p.dlam) {
    const int64_t n = p.dlam_n[0] * p.dlam_n[1] * p.dlam_n[2];
    if (p.dlam_n[2] == 1) {
      bwd_lambda_heads<<<tda::grid_of<1024>((int64_t)p.B * p.H), 1024, 0, st>>>(p);
      tda::launched(st, "sda_bwd_lambda_heads");
      bwd_lambda<true><<<tda::grid_of<256>((n + 3) / 4), 256, 0, st>>>(p);
    } else {
      bwd_lambda<false><<<tda::grid_of<256>((n + 255) / 256), 256, 0, st>>>(p);
    }
    tda::launched(st, "sda_bwd_lambda");
  }
  return (int)hipGetLastError();
}
template <class Tr>
static int pick(const BwdParams& p, int d, int dv, hipStream_t st) {
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}
int launch_bwd(const BwdParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 1 ? pick<TrB>(p, d, dv, st) : dtype == 2 ? pick<TrH>(p, d, dv, st) : pick<TrF>(p, d, dv, st);
}

}  // namespace sda
