// sda_fwd.hip -- softmax differential attention, forward:
//   out = (softmax(s q1 k1^T + M) - lambda softmax(s q2 k2^T + M)) v
//
// One pass over the keys with a running maximum and sum per row and branch.  Workgroup = 128 query
// rows of one head, 8 waves: wave w takes rows 32 (w % 4) .. + 31 of branch w / 4, so that the two
// branches share the value tiles in LDS and the two waves of a SIMD are one of each branch.  Scores are
// computed transposed (S^T = K Q^T): a lane holds one query row (column n = lane % 32) and 16 of a
// tile's 32 keys, so the row maxima and sums need one exchange between the lane's two halves, the
// weights feed the second product (O^T = V^T P^T) from the registers that hold them, and rescaling is
// one factor per lane.  Keys arrive by direct loads to LDS, one stage (64 keys bf16, 32 fp32) ahead.
// Branch 2's normalised result meets branch 1's through LDS at the end.
//
// Grids that would leave CUs idle take 64 query rows a workgroup (RG = 2 row groups): the other four waves
// take the second half of each stage's keys, and the halves' maxima, sums and outputs meet in LDS first.
//
// bf16 (1, 16 over 4, 16384, 128) 1.98 ms (1.93 to 2.18 on several parts), 1.1 PFLOP/s, where a product of 8192^3
// reaches 1.22: bound by the matrix cores.  Narrow keys leave fewer products to an exponential: (4, 16, 2048,
// 64/128), a training forward, 148 us, 0.70 PFLOP/s, bound by both together (a stage's waits cost little: a third
// stage in LDS or waves half a stage apart changed nothing).  f32 (2, 12, 1111, 64) 85 us, 0.09 PFLOP/s of 0.15.
#include "sda_common.hpp"

namespace sda {

template <class Tr, int D, int DV, int RG>
struct FwdShape {
  using T = typename Tr::T;
  static constexpr int BN = (sizeof(T) == 2 && DV <= 128) || RG == 2 ? 64 : 32;  // keys of a stage
  using KT = Tile<Tr, BN, D>;
  using VT = Tile<Tr, BN, DV>;
  static constexpr int STAGE = 2 * KT::BYTES + VT::BYTES;
  static constexpr int XCH = 4 * 32 * DV * 4;          // branch 2's result, f32
  static constexpr int LDS = 2 * STAGE > XCH + 2048 ? 2 * STAGE : XCH + 2048;
  static_assert(KT::LOADS % 8 == 0 && VT::LOADS % 8 == 0, "loads spread evenly over the waves");
};

template <class Tr, int D, int DV, int RG>
__global__ void __launch_bounds__(512) fwd_tiles(FwdParams P) {
  using T = typename Tr::T;
  using frag = typename Tr::frag;
  using S = FwdShape<Tr, D, DV, RG>;
  using KT = typename S::KT;
  using VT = typename S::VT;
  constexpr int BN = S::BN, NS = BN / 32 * RG / 4, NT = D / 16, NO = DV / 32;
  static_assert(NS >= 1, "a wave has whole key tiles");
  constexpr int KL = KT::LOADS / 8, VL = VT::LOADS / 8, ROWS = 32 * RG;
  constexpr int G = sizeof(T) == 2 ? 4 : 1;  // an fp32 fragment is eight products itself
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int l = lane_id(), n32 = l & 31, g = l >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wv % RG, br = wv / RG & 1, kh = wv / (2 * RG);  // kh: which half of a stage's keys
  const uint32_t bid = tda::grid_bid<512>();
  if (bid >= (uint32_t)(P.B * P.H) * (uint32_t)P.nqt) return;
  const Item it = item_of(bid, P.B * P.H, P.nqt, true);
  const int b = it.head / P.H, h = it.head % P.H, hk = h / (P.H / P.Hk);
  const int q0 = it.tile * ROWS, q0w = q0 + 32 * rg;
  const int len = len_of(P.see, b, P.Nk), off = off_of(P.see, b);
  // keys the workgroup / the wave sees at most
  const int qlast = min(q0 + ROWS, P.Nq) - 1;
  const int lim = P.see.causal ? min(len, max(off + qlast + 1, 0)) : len;
  const int limw = P.see.causal ? min(len, max(off + min(q0w + 31, P.Nq - 1) + 1, 0)) : len;
  const int clear = P.see.causal ? min(len, max(off + q0w + 1, 0)) : len;  // every row of the wave sees these
  const int nst = (lim + BN - 1) / BN;
  const int qi = q0w + n32;  // this lane's row
  const int see = P.see.causal ? min(len, off + qi + 1) : len;

  const T* kbase[2] = {row_of<T>(P.k[0], b, hk, 0), row_of<T>(P.k[1], b, hk, 0)};
  const T* vbase = row_of<T>(P.v, b, hk, 0);
  uint32_t ko[2][KL], vo[VL];
#pragma unroll
  for (int u = 0; u < KL; ++u) {
    ko[0][u] = KT::source(8 * u + wv, (uint32_t)(P.k[0].st * KT::ES));
    ko[1][u] = KT::source(8 * u + wv, (uint32_t)(P.k[1].st * KT::ES));
  }
#pragma unroll
  for (int u = 0; u < VL; ++u) vo[u] = VT::source(8 * u + wv, (uint32_t)(P.v.st * VT::ES));
  // Stage j into buffer j % 2; rows behind every row's sight read as zeros (a weight of zero times
  // whatever lies there must stay zero).
  auto issue = [&](int j) {
    char* at = lds + (j & 1) * S::STAGE;
    const int64_t r0 = (int64_t)j * BN;
    const int rows = min(BN, lim - j * BN);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto r = rows_rsrc(kbase[x] + r0 * P.k[x].st, P.k[x].st * KT::ES, rows, D * KT::ES);
#pragma unroll
      for (int u = 0; u < KL; ++u) KT::load(r, reinterpret_cast<T*>(at + x * KT::BYTES), 8 * u + wv, ko[x][u]);
    }
    const auto r = rows_rsrc(vbase + r0 * P.v.st, P.v.st * VT::ES, rows, DV * VT::ES);
#pragma unroll
    for (int u = 0; u < VL; ++u) VT::load(r, reinterpret_cast<T*>(at + 2 * KT::BYTES), 8 * u + wv, vo[u]);
  };
  if (nst > 0) issue(0);

  frag qf[NT];
  load_frags<Tr, NT>(qi < P.Nq ? row_of<T>(P.q[br], b, h, qi) : nullptr, g, qf);
  f32x16 o[NO] = {};
  float m = kNoMax, sums[4] = {};

  RowReader<Tr, D> kr;
  ColReader<Tr, DV> vr;
  const char* kbuf = lds + br * KT::BYTES + 32 * kh * D * KT::ES;
  const char* vbuf = lds + 2 * KT::BYTES + 32 * kh * DV * VT::ES;
  kr.init(kbuf);
  vr.init(vbuf);
  auto step = [&](int j, auto half) {  // stage j, in the half of the buffers that its parity names
    constexpr int AT = half * S::STAGE;
    wait_vm<0>();
    tda::lds_barrier();  // stage j is in place, and every wave is done with stage j - 1
    if (j + 1 < nst) issue(j + 1);
    const int k0 = j * BN + 32 * kh;
    if (k0 >= limw) return;
    // The stage's products take their LDS operands as one sequence, NS NT key fragments then 2 NS NO value
    // fragments, read a group of G ahead of their use: the first value group is on its way before the softmax.
    frag f[2][G];
    auto read = [&](int i) {
#pragma unroll
      for (int u = 0; u < G; ++u) {
        const int e = i * G + u, w = e - NS * NT;
        if (e < NS * NT) f[i & 1][u] = kr.read(kbuf, AT + 32 * D * KT::ES * (e % NS), e / NS);
        else f[i & 1][u] = vr.read(vbuf, AT + 32 * DV * VT::ES * (w / (2 * NO)), w / NO % 2, w % NO);
      }
    };
    f32x16 s[NS] = {};
    read(0);
#pragma unroll
    for (int i = 0; i < NS * NT / G; ++i) {
      read(i + 1);
#pragma unroll
      for (int u = 0; u < G; ++u) {
        const int e = i * G + u;
        s[e % NS] = Tr::mma32(f[i & 1][u], qf[e / NS], s[e % NS]);
      }
    }
    if (k0 + 32 * NS > clear) {
      asm volatile("");  // a branch: few tiles need this
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * x + crow(r, g) >= see) s[x][r] = -__builtin_inff();
    }
    // the maximum and the sum in four chains: one of 32 dependent steps takes longer than the products
    float four[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) four[r % 4] = fmaxf(four[r % 4], s[x][r]);
    float top = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3])) * P.c;
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = fmaxf(m, top), f = exp2_(m - to);
      m = to;
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[r] *= f;
#pragma unroll
      for (int x = 0; x < NO; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[x][r] *= f;
    }
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[x][r] = exp2_(__builtin_fmaf(s[x][r], P.c, -m));
        sums[r % 4] += s[x][r];
      }
    frag p[2 * NS];
#pragma unroll
    for (int x = 0; x < 2 * NS; ++x) p[x] = pack8<Tr>(s[x / 2], x % 2);
    constexpr int first = NS * NT / G, last = first + 2 * NS * NO / G;
#pragma unroll
    for (int i = first; i < last; ++i) {
      if (i + 1 < last) read(i + 1);
#pragma unroll
      for (int u = 0; u < G; ++u) {
        const int w = i * G + u - NS * NT;
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
  if constexpr (RG == 2) {  // the second half's sums join the first's
    __syncthreads();
    float* stat = reinterpret_cast<float*>(lds + 4 * 32 * DV * 4);  // behind the outputs: m, sum by pair and lane
    f32x4* half = reinterpret_cast<f32x4*>(lds) + (wv & 3) * (NO * 4 * 64) + l;
    if (kh) {
      stat[128 * (wv & 3) + l] = m;
      stat[128 * (wv & 3) + 64 + l] = sum;
#pragma unroll
      for (int y = 0; y < NO; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) half[(4 * y + r) * 64] = f32x4{o[y][4 * r], o[y][4 * r + 1], o[y][4 * r + 2], o[y][4 * r + 3]};
    }
    __syncthreads();
    if (!kh) {
      const float m2 = stat[128 * wv + l], all = fmaxf(m, m2), f1 = exp2_(m - all), f2 = exp2_(m2 - all);
      sum = __builtin_fmaf(stat[128 * wv + 64 + l], f2, sum * f1);
      m = all;
#pragma unroll
      for (int y = 0; y < NO; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 w = half[(4 * y + r) * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[y][4 * r + e] = __builtin_fmaf(w[e], f2, o[y][4 * r + e] * f1);
        }
    }
  }
  const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;  // no visible key: zeros
  const bool row = qi < P.Nq;
  if (P.lse && row && g == 0 && !kh)  // a row without keys: +inf, which weighs everything 0
    P.lse[((int64_t)br * P.B * P.H + it.head) * P.Nq + qi] = sum > 0.f || sum != sum ? m + __builtin_amdgcn_logf(sum) : __builtin_inff();
  __syncthreads();  // the stages are read: their place carries branch 2's result
  f32x4* xch = reinterpret_cast<f32x4*>(lds) + rg * (NO * 4 * 64) + l;
  if (br && !kh) {
    float* to = P.out2.p && row ? row_of<float>(P.out2, b, h, qi) : nullptr;
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 w = {o[y][4 * r] * inv, o[y][4 * r + 1] * inv, o[y][4 * r + 2] * inv, o[y][4 * r + 3] * inv};
        xch[(4 * y + r) * 64] = w;
        if (to) store4(to + 32 * y + 8 * r + 4 * g, w);
      }
  }
  __syncthreads();
  if (!br && !kh && row) {
    const float lam = lambda_of(P.lam, b, h, qi);
    T* to = row_of<T>(P.out, b, h, qi);
    T* low = P.out2.p ? row_of<T>(P.low, b, h, qi) : nullptr;  // what rounding leaves out, for the backward's row sums
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 w = xch[(4 * y + r) * 64];
        f32x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = __builtin_fmaf(-lam, w[e], o[y][4 * r + e] * inv);
        store4(to + 32 * y + 8 * r + 4 * g, z);
        if constexpr (sizeof(T) == 2) {
          if (low) {
            f32x4 rest;
#pragma unroll
            for (int e = 0; e < 4; ++e) rest[e] = z[e] - (float)(T)z[e];
            store4(low + 32 * y + 8 * r + 4 * g, rest);
          }
        }
      }
  }
}

template <class Tr, int D, int DV, int RG>
static int launch(FwdParams p, hipStream_t st) {
  using S = FwdShape<Tr, D, DV, RG>;
  const void* fn = reinterpret_cast<const void*>(&fwd_tiles<Tr, D, DV, RG>);
  if (S::LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS);
    if (e != hipSuccess) return (int)e;
  }
  p.nqt = (p.Nq + 32 * RG - 1) / (32 * RG);
  fwd_tiles<Tr, D, DV, RG><<<tda::grid_of<512>((int64_t)p.nqt * p.B * p.H), 512, S::LDS, st>>>(p);
  const hipError_t e = hipGetLastError();
  tda::launched(st, "sda_fwd_tiles");
  return (int)e;
}
template <class Tr, int D, int DV>
static int run(const FwdParams& p, hipStream_t st) {
  if constexpr (FwdShape<Tr, D, DV, 2>::LDS <= kLds) {
    if (halve<Tr, D, DV>(p.see, (int64_t)((p.Nq + 127) / 128) * p.B * p.H, p.Nq)) return launch<Tr, D, DV, 2>(p, st);
  }
  return launch<Tr, D, DV, 4>(p, st);
}
template <class Tr>
static int pick(const FwdParams& p, int d, int dv, hipStream_t st) {
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}
int launch_fwd(const FwdParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 1 ? pick<TrB>(p, d, dv, st) : dtype == 2 ? pick<TrH>(p, d, dv, st) : pick<TrF>(p, d, dv, st);
}

}  // namespace sda
