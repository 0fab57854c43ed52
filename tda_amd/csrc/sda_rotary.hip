// sda_rotary.hip -- rotary positions of several axes, for up to four tensors at the same positions.
//
// A workgroup takes a few tokens: their cosines and sines go to LDS once (a table of tokens x pairs),
// then the rows of every head of every tensor at those tokens stream through, each value read and
// written once.  Bound by memory: four tensors of bf16 (4, 16, 4096, 128), 96 values rotated, 120 us for 537 MB
// (4.5 TB/s); all 128 rotated 104 us (5.2 TB/s).  Widths or strides that are no whole pieces of 16 bytes go by single
// values: width 72, all rotated, 131 us for 302 MB (2.3 TB/s), width 80, 40 rotated, 198 us for 336 MB (1.7 TB/s).  The angle is a product of an integer and an f32 frequency taken in
// 64 bits and reduced to a turn there, so far positions keep their accuracy; sine and cosine of the
// reduced angle are f32.
#include "sda_common.hpp"

namespace sda {

__device__ __forceinline__ int64_t position(const RotaryParams& P, int a, int b, int n) {
  const int64_t at = a * P.ps[0] + b * P.ps[1] + n * P.ps[2];
  return P.pos64 ? static_cast<const int64_t*>(P.pos)[at] : static_cast<const int32_t*>(P.pos)[at];
}

// V values a thread moves at a time (V divides the pairs and the copied tail; V-aligned rows).
template <class T, int V>
__global__ void __launch_bounds__(256) rotary(RotaryParams P, int tok) {
  extern __shared__ float2 table[];  // [tok][pairs]
  const uint32_t blocks = (uint32_t)((P.N + tok - 1) / tok), bid = tda::grid_bid<256>();
  if (bid >= (uint32_t)P.B * blocks) return;
  const int b = (int)(bid / blocks), n0 = (int)(bid % blocks) * tok;
  const int nt = min(tok, P.N - n0);
  for (int e = threadIdx.x; e < nt * P.pairs; e += 256) {
    const int t = e / P.pairs, p = e % P.pairs;
    int a = 0;
    while (p >= P.upto[a]) ++a;  // ends: the last section reaches every pair
    const double turns = (double)position(P, a, b, n0 + t) * (double)P.inv_freq[p] * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    table[e] = make_float2(c, s * P.sign);
  }
  __syncthreads();
  typedef T vec __attribute__((ext_vector_type(V)));
  const int pv = P.pairs / V, tail = (P.D - 2 * P.pairs) / V, units = pv + tail;  // a unit: V pairs, or V copied values
  for (int z = 0; z < P.count; ++z) {
    const int64_t total = (int64_t)P.heads[z] * nt * units;
    for (int64_t e = threadIdx.x; e < total; e += 256) {
      const int u = (int)(e % units), t = (int)(e / units % nt), h = (int)(e / units / nt);
      const T* x = row_of<const T>(P.x[z], b, h, n0 + t);
      T* y = row_of<T>(P.y[z], b, h, n0 + t);
      if (u >= pv) {
        const int at = 2 * P.pairs + V * (u - pv);
        *reinterpret_cast<vec*>(y + at) = *reinterpret_cast<const vec*>(x + at);
        continue;
      }
      const int i0 = P.inter ? 2 * V * u : V * u, i1 = P.inter ? i0 + V : P.pairs + V * u;
      const vec p = *reinterpret_cast<const vec*>(x + i0), q = *reinterpret_cast<const vec*>(x + i1);
      vec r, w;
      const float2* cs = table + t * P.pairs + V * u;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float a, c;
        if (P.inter) {
          a = (float)(2 * k < V ? p[2 * k % V] : q[2 * k % V]);
          c = (float)(2 * k < V ? p[(2 * k + 1) % V] : q[(2 * k + 1) % V]);
          if constexpr (V == 1) c = (float)q[0];
        } else {
          a = (float)p[k];
          c = (float)q[k];
        }
        const float f = __builtin_fmaf(a, cs[k].x, -(c * cs[k].y)), d = __builtin_fmaf(c, cs[k].x, a * cs[k].y);
        if (P.inter && V > 1) {
          if (2 * k < V) r[2 * k % V] = (T)f, r[(2 * k + 1) % V] = (T)d;
          else w[2 * k % V] = (T)f, w[(2 * k + 1) % V] = (T)d;
        } else {
          r[k] = (T)f;
          w[k] = (T)d;
        }
      }
      *reinterpret_cast<vec*>(y + i0) = r;
      *reinterpret_cast<vec*>(y + i1) = w;
    }
  }
}

template <class T>
static int run(const RotaryParams& p, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool wide = p.pairs % V == 0 && (p.D - 2 * p.pairs) % V == 0;
  for (int z = 0; z < p.count; ++z)
    for (const Rows* r : {&p.x[z], &p.y[z]})
      wide = wide && (uintptr_t)r->p % 16 == 0 && r->sb % V == 0 && r->sh % V == 0 && r->st % V == 0;
  // one token a workgroup until there are many workgroups anyway: then the heads of four share a fill of the
  // table (four tensors of bf16 (1, 4, 65536, 128): one token 191 us, two 115, four 100, eight 98; (4, 16,
  // 4096, 128): 117, 120, 120, 128)
  int tok = (int64_t)p.B * p.N >= 4096 ? 4 : 1;
  while (tok > 1 && tok * p.pairs * 8 > 65536) tok /= 2;
  const int64_t grid = (int64_t)p.B * ((p.N + tok - 1) / tok);
  const int lds = tok * p.pairs * 8;
  if (wide) rotary<T, V><<<tda::grid_of<256>(grid), 256, lds, st>>>(p, tok);
  else rotary<T, 1><<<tda::grid_of<256>(grid), 256, lds, st>>>(p, tok);
  tda::launched(st, "sda_rotary");
  return (int)hipGetLastError();
}
int launch_rotary(const RotaryParams& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? run<float>(p, st) : dtype == 1 ? run<bf16>(p, st) : run<_Float16>(p, st);
}

}  // namespace sda
