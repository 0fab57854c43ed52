// sda_decode.hip -- few query rows over keys and values in the queries' own type (sda_decode.hpp).
#include "sda_decode.hpp"

namespace sda {

template <class Tr, int D, int DV>
__global__ void __launch_bounds__(256) decode(DecParams P, FwdParams F) {
  extern __shared__ float lds[];
  DenseSrc<Tr, D, DV> src;
  src.F = &F;
  DecWork W;
  if (dec_work(P, W)) decode_body(P, W, src, lds);
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
