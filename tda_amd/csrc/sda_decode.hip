// sda_decode.hip -- few query rows over keys and values in the queries' own type (sda_decode.hpp).
#include "sda_decode.hpp"

namespace sda {

template <class Tr, int D_, int DV_>
struct DenseSrc {
  using T = typename Tr::T;
  using Out = T;
  using frag = typename Tr::frag;
  static constexpr int D = D_, DV = DV_, NT = D / 32;
  static constexpr int CW = DV / 16 < 8 ? DV / 16 : 8, NB = DV / (16 * CW);  // columns of a lane, blocks of them
  typedef T row __attribute__((ext_vector_type(CW)));
  static constexpr int NBUF = sizeof(T) == 2 && DV <= 128 ? 2 : 1;
  struct Regs {
    frag k[2][2][NT];
    row v[8][NB];
  };
  frag q[2][NT];
  const T* kp[2];
  const T* vp;
  int64_t ks[2], vs;

  __device__ __forceinline__ static frag load8(const T* p) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const frag*>(p);
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  const FwdParams* F;
  __device__ __forceinline__ void begin(const DecParams& P, int b, int hk, int h, int i, bool live) {
    const int kq = lane_id() >> 4;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      kp[x] = row_of<T>(F->k[x], b, hk, 0);
      ks[x] = F->k[x].st;
      const T* r = row_of<T>(P.q[x], b, h, i);
#pragma unroll
      for (int t = 0; t < NT; ++t) q[x][t] = live ? load8(r + 32 * t + 8 * kq) : frag{};
    }
    vp = row_of<T>(F->v, b, hk, 0);
    vs = F->v.st;
  }
  __device__ __forceinline__ static frag load8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(frag, a);
    } else {
      const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 16, 0, 0));
      return f32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  }
  __device__ __forceinline__ void load(Regs& g, int t0, int lim) {
    const int n = lane_id() & 15, kq = lane_id() >> 4, rows = min(32, lim - t0);
    constexpr int ES = sizeof(T);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto r = rows_rsrc(kp[x] + (int64_t)t0 * ks[x], ks[x] * ES, rows, D * ES);
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int t = 0; t < NT; ++t) g.k[x][y][t] = load8(r, (uint32_t)(16 * y + n) * (uint32_t)(ks[x] * ES) + (32 * t + 8 * kq) * ES);
    }
    const auto r = rows_rsrc(vp + (int64_t)t0 * vs, vs * ES, rows, DV * ES);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        const uint32_t off = (uint32_t)(16 * (j >> 2) + 4 * kq + (j & 3)) * (uint32_t)(vs * ES) + (CW * n + 16 * CW * y) * ES;
        if constexpr (CW * ES == 8) g.v[j][y] = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
        else if constexpr (CW * ES == 16) g.v[j][y] = __builtin_bit_cast(row, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
        else g.v[j][y] = load8(r, off);
      }
  }
  __device__ __forceinline__ void scores(const Regs& g, f32x4 (&s)[2][2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        s[x][y] = f32x4{};
#pragma unroll
        for (int t = 0; t < NT; ++t) s[x][y] = Tr::mma16(g.k[x][y][t], q[x][t], s[x][y]);
      }
  }
  __device__ __forceinline__ void rescale(int, float) {}
  __device__ __forceinline__ void add(const Regs& g, const f32x4 (&s)[2][2], f32x4 (&o)[2][DV / 16]) {
    frag p[2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j) p[x][j] = (T)s[x][j >> 2][j & 3];
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        frag a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = g.v[j][y][c];
#pragma unroll
        for (int x = 0; x < 2; ++x) o[x][CW * y + c] = Tr::mma16(a, p[x], o[x][CW * y + c]);
      }
  }
  __device__ __forceinline__ void finish(f32x4 (&)[2][DV / 16]) {}
  __device__ __forceinline__ static int column(int t, int m) { return 16 * CW * (t / CW) + CW * m + t % CW; }
};

template <class Tr, int D, int DV>
__global__ void __launch_bounds__(256) decode(DecParams P, FwdParams F) {
  extern __shared__ float lds[];
  DenseSrc<Tr, D, DV> src;
  src.F = &F;
  decode_body(P, src, lds);
}

template <class Tr, int D, int DV>
static int run(const FwdParams& f, hipStream_t st) {
  DecParams p{};
  p.q[0] = f.q[0];
  p.q[1] = f.q[1];
  p.out = f.out;
  p.lam = f.lam;
  p.see = f.see;
  p.B = f.B;
  p.H = f.H;
  p.Hk = f.Hk;
  p.Nq = f.Nq;
  p.Nk = f.Nk;
  p.D = D;
  p.DV = DV;
  p.c = f.c;
  p.part = f.part;
  p.nsplit = f.nsplit;
  p.chunk = f.chunk;
  constexpr int LDS = kDecLds<DV>;
  if (LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&decode<Tr, D, DV>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return (int)e;
  }
  const int64_t items = (int64_t)f.B * f.Hk * ((f.H / f.Hk * (int64_t)f.Nq + kDecRows - 1) / kDecRows);
  decode<Tr, D, DV><<<tda::grid_of<256>(items * f.nsplit), 256, LDS, st>>>(p, f);
  tda::launched(st, "sda_decode");
  if (f.nsplit > 1) {
    decode_join<typename Tr::T><<<tda::grid_of<256>(((int64_t)f.B * f.H * f.Nq * DV + 255) / 256), 256, 0, st>>>(p);
    tda::launched(st, "sda_decode_join");
  }
  return (int)hipGetLastError();
}
template <class Tr>
static int pick(const FwdParams& p, int d, int dv, hipStream_t st) {
  if (d == 64) return dv == 64 ? run<Tr, 64, 64>(p, st) : run<Tr, 64, 128>(p, st);
  return dv == 128 ? run<Tr, 128, 128>(p, st) : run<Tr, 128, 256>(p, st);
}
int launch_decode(const FwdParams& p, int dtype, int d, int dv, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 1 ? pick<TrB>(p, d, dv, st) : dtype == 2 ? pick<TrH>(p, d, dv, st) : pick<TrF>(p, d, dv, st);
}

}  // namespace sda
