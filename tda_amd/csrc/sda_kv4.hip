// sda_kv4.hip -- a key/value cache held in 4 bits: append, read, and the attention of few query rows.
//
// A row in groups of 64 values x: m = bf16(min), s = bf16((max - m) / 15) in 32 bits,
// code = rint((x - m) / s) clamped to 0 .. 15, value m + s code.  4.5 bits a value.
//
// Codes lie so that the attention's registers need no exchange between lanes and its loads are wide (the
// loads' number is what bounds it next to the memory's rate):
//   keys: word u (32 bits) of a group holds its values 8 u .. 8 u + 7; bits 4 i hold value 2 i and bits
//   16 + 4 i value 2 i + 1, so (word >> 4 i) & 0x000f000f is a pair of neighbours; a row of two groups
//   has words 2 q and 2 q + 1 of both side by side;
//   values: 16-bit units of four neighbouring columns, bits 4 j holding column 4 n + j of group gr in
//   unit (gr, n); the words of a row are its units in order (64 columns), or pair the units (gr, n) and
//   (gr + 1, n) of two groups, by n, then by pair.  Four rows lie together, word by word.
// Behind the codes of all rows: (m, s) of each row's groups, s in the high half of a word.  A head has
// rows for its capacity rounded up to four.
#include "sda_decode.hpp"

namespace sda {

constexpr float kSmallStep = 0x1p-100f;  // a step below this is zero: all codes 0

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ uint32_t bf16_bits(float x) {  // round to nearest even
  const bf16 r = (bf16)x;
  return __builtin_bit_cast(uint16_t, r);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {  // 16-byte aligned
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int u = 0; u < 8 / V; ++u) {
    const vec v = reinterpret_cast<const vec*>(p)[u];
#pragma unroll
    for (int e = 0; e < V; ++e) x[V * u + e] = (float)v[e];
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int u = 0; u < 8 / V; ++u) {
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)x[V * u + e];
    reinterpret_cast<vec*>(p)[u] = v;
  }
}
// x / 15, rounded once: the product by the rounded reciprocal, within a step of it, and its remainder, exact, by
// the reciprocal again (compared with the division for every mantissa; that costs an append 3 % more).
__device__ __forceinline__ float fifteenth(float x) {
  constexpr float inv = 1.0f / 15.0f;
  const float q = x * inv;
  return x < __builtin_inff() ? __builtin_fmaf(__builtin_fmaf(-15.0f, q, x), inv, q) : x;
}
// rint((x - m) / s) with ties to the even code, decided exactly: x - m as an unevaluated sum hi + lo, the
// nearest boundary p = (q + 1/2) s exact (q < 16, s of 8 bits), hi - p exact wherever its sign is in doubt.
__device__ __forceinline__ float exact_code(float x, float m, float s, float inv) {
  const float hi = x - m, z = hi - x, lo = (x - (hi - z)) + (-m - z);
  const float q = floorf(fminf(fmaxf(hi * inv, 0.f), 15.f));
  const float p = (q + 0.5f) * s, a = hi - p;
  const bool up = a > -lo || (a == -lo && ((int)q & 1));
  return fminf(q + (up ? 1.f : 0.f), 15.f);
}
// The same for 8 values: t = (x - m) rcp(s), the reciprocal 2^-23 off, is at most 16 * 4 * 2^-24 = 2^-18 off,
// so its nearest integer is the code unless it lies within 2^-17 of the middle between two; 64 lanes decide
// a value exactly where one of them does (about every seventh for bf16 rows, whose differences often are
// odd multiples of s / 2).
__device__ __forceinline__ void codes_of(const float (&x)[8], float m, float s, bool any, float (&c)[8]) {
  float inv = any ? __builtin_amdgcn_rcpf(s) : 0.f, sure = 0.5f - 0x1p-17f;
  if (__any(any && s > 0x1p120f)) {
    asm volatile("");  // a branch: the reciprocal may have fewer bits
    if (any && s > 0x1p120f) inv = 1.0f / s, sure = -1.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = fminf(fmaxf((x[e] - m) * inv, 0.f), 15.f);
    c[e] = __builtin_rintf(t);
    if (__any(fabsf(t - c[e]) > sure)) {
      asm volatile("");
      c[e] = any ? exact_code(x[e], m, s, inv) : 0.f;
    }
  }
}
// Four codes in 16 bits, the first lowest.
__device__ __forceinline__ uint32_t unit(float a, float b, float c, float d) {
  return (uint32_t)__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(d, 16.f, c), 16.f, b), 16.f, a);
}

// Place of key word u (of W / 8) in its row, and of word w of value row i (L words) of the head whose rows
// start at row0.
__device__ __forceinline__ int key_place(int W, int u) { return W == 64 ? u : 4 * ((u & 7) >> 1) + 2 * (u >> 3) + (u & 1); }
__device__ __forceinline__ int64_t value_word(int64_t row0, int64_t i, int L, int w) {
  return row0 * L + (i >> 2) * (4 * L) + 4 * w + (i & 3);
}

// ------------------------------------------------------------------ append
// 8 lanes per group of 64 values, 8 values a lane; a workgroup has R times 256 / (W / 8) rows of one head,
// `blocks` workgroups the head's.  Bound by the roundings' arithmetic and the memory's rate: bf16 (4, 8, 2048,
// 128) 21 us for 64 MB, (32, 8, 8192, 128) 441 us for 2.06 GB (4.7 TB/s).
template <class T, int R>
__global__ void __launch_bounds__(256) kv4_append(Kv4Params P, int blocks) {
  const int z = blockIdx.z, W = z < 2 ? P.D : P.DV, L = W / 8;  // lanes of a row
  const int shift = W == 64 ? 3 : W == 128 ? 4 : 5;
  const uint32_t wg = tda::grid_bid<256>(), bk = wg / (uint32_t)blocks;
  if (bk >= (uint32_t)P.B * (uint32_t)P.Hk) return;
  const int b = (int)(bk / (uint32_t)P.Hk), hk = (int)(bk % (uint32_t)P.Hk);
  const int u = threadIdx.x & (L - 1), i0 = (int)(wg % (uint32_t)blocks) * R * (256 >> shift) + (threadIdx.x >> shift);
  const int start = P.start ? P.start[b] : max(P.lengths[b], 0);
  const int count = P.counts ? min(max(P.counts[b], 0), P.rows) : P.rows;
  float xs[R][8] = {};
  const int step = 256 >> shift;
  const T* from = row_of<const T>(P.x[z], b, hk, i0) + 8 * u;
#pragma unroll
  for (int y = 0; y < R; ++y) {
    const int i = i0 + y * step;
    const int64_t at = (int64_t)start + i;
    if (i < count && at >= 0 && at < P.cap) load8(from + y * step * P.x[z].st, xs[y]);
  }
  // the head's rows: within them offsets stay in 32 bits; step rows, whole fours, lie between a thread's
  uint32_t* words = reinterpret_cast<uint32_t*>(P.codes[z]) + bk * P.cap4 * L;
  uint32_t* pars = P.pars[z] + bk * P.cap4 * (W / 64);
  const bool second = u & 8;
  const uint32_t at0 = (uint32_t)start + (uint32_t)i0;
  const uint32_t to = z < 2 ? at0 * L + key_place(W, u)
                            : value_word(0, at0, L, W == 64 ? u : 16 * (u >> 4) + 2 * (u & 7) + (second ? 1 : 0));
#pragma unroll
  for (int y = 0; y < R; ++y) {
    const int i = i0 + y * step;
    const int64_t at = (int64_t)start + i;
    const bool put = i < count && at >= 0 && at < P.cap;
    const float (&x)[8] = xs[y];
    float lo = x[0], hi = x[0], zero = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo = fminf(lo, x[e]);
      hi = fmaxf(hi, x[e]);
      zero = __builtin_fmaf(x[e], 0.f, zero);  // NaN where a value is not finite
    }
    if (!(zero == 0.f)) hi = __builtin_inff();  // then s is not finite either
    lo = -tda::group_max<8>(-lo);
    hi = tda::group_max<8>(hi);
    const uint32_t mb = bf16_bits(lo);
    const float m = bf16_lo(mb);
    uint32_t sb = bf16_bits(fifteenth(hi - m));
    float s = bf16_lo(sb);
    if (!(s >= kSmallStep)) s = 0.f, sb = 0;
    const bool bad = !(s < __builtin_inff()) || !(fabsf(m) < __builtin_inff());
    float c[8];
    codes_of(x, bad ? 0.f : m, s, s > 0.f && !bad, c);
    uint32_t word;
    if (z < 2) {
      word = unit(c[0], c[2], c[4], c[6]) | unit(c[1], c[3], c[5], c[7]) << 16;
    } else {
      const uint32_t a = unit(c[0], c[1], c[2], c[3]), d = unit(c[4], c[5], c[6], c[7]);
      if (W == 64) {
        word = a | d << 16;
      } else {  // lanes u and u + 8 (the same columns of two groups) swap a unit
        const uint32_t other = (uint32_t)__shfl_xor((int)(second ? a : d), 8);
        word = second ? other | d << 16 : a | other << 16;
      }
    }
    if (put) {
      words[to + y * step * L] = word;
      if ((u & 7) == 0) pars[((uint32_t)at << (shift - 3)) + (u >> 3)] = bad ? 0x7fc0u : mb | sb << 16;
    }
  }
  if (P.start && P.counts != P.lengths && z == 0 && hk == 0 && i0 == 0 && u == 0)  // else kv4_lengths
    P.lengths[b] = (int)min(max((int64_t)start + count, (int64_t)0), (int64_t)P.cap);
}
__global__ void kv4_lengths(Kv4Params P) {
  const int b = blockIdx.x * 64 + threadIdx.x;
  if (b >= P.B) return;
  const int64_t start = P.start ? P.start[b] : max(P.lengths[b], 0);
  const int count = P.counts ? min(max(P.counts[b], 0), P.rows) : P.rows;
  P.lengths[b] = (int)min(max(start + count, (int64_t)0), (int64_t)P.cap);
}

// ------------------------------------------------------------------ read
// Lanes and workgroups as above.  bf16 (4, 8, 2048, 128): 13 us for 64 MB, the memory's rate.
template <class T, int R>
__global__ void __launch_bounds__(256) kv4_read(Kv4Params P, int blocks) {
  const int z = blockIdx.z, W = z < 2 ? P.D : P.DV, L = W / 8;
  const int shift = W == 64 ? 3 : W == 128 ? 4 : 5;
  const uint32_t wg = tda::grid_bid<256>(), bk = wg / (uint32_t)blocks;
  if (bk >= (uint32_t)P.B * (uint32_t)P.Hk) return;
  const int b = (int)(bk / (uint32_t)P.Hk), hk = (int)(bk % (uint32_t)P.Hk);
  const int u = threadIdx.x & (L - 1), i0 = (int)(wg % (uint32_t)blocks) * R * (256 >> shift) + (threadIdx.x >> shift);
  const int64_t row0 = bk * P.cap4;
  const int held = min(min(P.lengths[b], P.cap), P.rows);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(P.codes[z]);
  uint32_t w0[R] = {}, w1[R] = {}, par[R] = {};
#pragma unroll
  for (int y = 0; y < R; ++y) {
    const int i = i0 + y * (256 >> shift);
    if (i >= held) continue;
    const int64_t row = row0 + i;
    par[y] = P.pars[z][row * (W / 64) + u / 8];
    if (z < 2) {
      w0[y] = words[row * L + key_place(W, u)];
    } else if (W == 64) {
      w0[y] = words[value_word(row0, i, L, u)];
    } else {
      const int place = 16 * (u >> 4) + 2 * (u & 7);
      w0[y] = words[value_word(row0, i, L, place)];
      w1[y] = words[value_word(row0, i, L, place + 1)];
    }
  }
#pragma unroll
  for (int y = 0; y < R; ++y) {
    const int i = i0 + y * (256 >> shift);
    if (i >= P.rows) return;
    const float m = bf16_lo(par[y]), s = bf16_hi(par[y]);  // all zero for a row that is not held
    float x[8];
    if (z < 2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(s, (float)(w0[y] >> (4 * (e >> 1) + 16 * (e & 1)) & 15), m);
    } else {
      // units of columns 8 u' .. + 3 and + 4 .. + 7
      const uint32_t a = W > 64 && (u & 8) ? w0[y] >> 16 : w0[y] & 0xffff;
      const uint32_t d = W == 64 ? w0[y] >> 16 : u & 8 ? w1[y] >> 16 : w1[y] & 0xffff;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __builtin_fmaf(s, (float)(a >> (4 * e) & 15), m);
        x[4 + e] = __builtin_fmaf(s, (float)(d >> (4 * e) & 15), m);
      }
    }
    if constexpr (std::is_same_v<T, _Float16>) {  // the largest float16 instead of infinity
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] > 65504.f ? 65504.f : x[e] < -65504.f ? -65504.f : x[e];
    }
    store8(row_of<T>(P.x[z], b, hk, i) + 8 * u, x);
  }
}

// ------------------------------------------------------------------ attention
// NP: bf16 parts that a query value and a weight are split into: 1 (bf16 queries), 2 (f16: 16 bits), 3
// (f32: 24 bits); a product with a code is exact in each.  Codes become bf16 by setting 0x4300 above
// them (128 + code); the 128 leaves through the sums of the other operand.  f32 and f16 convert the
// codes themselves: 128 times the sum would cost them bits.  Values are taken around their middle, m + 8 s
// + s (code - 8): the rounding of weight * s then counts with |s (code - 8)|, about the value itself, and
// not with s code (bf16 outputs of a short cache: 3.3e-3 off without, 2.3e-3 with).
template <class T, int NP, int D_, int DV_>
struct Kv4Src {
  using Out = T;
  static constexpr int D = D_, DV = DV_, GK = D / 64, GV = DV / 64, WV = DV / 128 ? DV / 128 : 1;
  struct Regs {
    uint32_t k[2][2][GK][2];      // [branch][16 keys][group][word 2 kq + i]
    uint32_t kp[2][2][4][GK];     // [branch][16 keys][key 4 kq + r][group]
    uint32_t v[2][WV][4];         // [16 keys][pair of groups][key 4 kq + r]
    uint32_t vp[8][GV];
  };
  const Kv4Params* C;
  bf16x8 q[2][NP][GK][2];
  float qs[2][GK];                // sum of a group's query values
  float corr[2][GV];              // sum of weight * middle, which every column of a group still gets
  f32x4 used[2][GV];              // sum of the rounded weight * step
  static constexpr int NBUF = 1;
  const uint32_t *kc[2], *kpar[2], *vc, *vpar;  // the head's rows: within them offsets are 32-bit

  uint32_t high;  // 0x43004300 in a vector register: and + or are then one instruction

  __device__ __forceinline__ bf16x8 codes(uint32_t w) const {  // 8 codes of a key word, in value order
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = pair(w >> (4 * i));
    return __builtin_bit_cast(bf16x8, x);
  }
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    if constexpr (NP == 1) {
      return (w & 0x000f000fu) | high;
    } else {
      const float a = (float)(w & 15u), b = (float)(w >> 16 & 15u);  // exact: their low halves are zero
      return __builtin_bit_cast(uint32_t, a) >> 16 | __builtin_bit_cast(uint32_t, b);
    }
  }
  static constexpr float kBias = NP == 1 ? 128.f : 0.f;
  // x as NP bf16 parts
  __device__ __forceinline__ static void split(float x, bf16 (&p)[NP]) {
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      p[e] = (bf16)x;
      x -= (float)p[e];
    }
  }

  __device__ __forceinline__ void begin(const DecParams& P, int b, int hk, int h, int i, bool live) {
    const int kq = lane_id() >> 4;
    const int64_t row0 = ((int64_t)b * P.Hk + hk) * C->cap4;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      kc[x] = reinterpret_cast<const uint32_t*>(C->codes[x]) + row0 * (D / 8);
      kpar[x] = C->pars[x] + row0 * GK;
      const T* r = row_of<const T>(P.q[x], b, h, i);
#pragma unroll
      for (int y = 0; y < GK; ++y) {
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float f[8] = {};
          if (live) load8(r + 64 * y + 16 * kq + 8 * w, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a += f[e];
            bf16 p[NP];
            split(f[e], p);
#pragma unroll
            for (int z = 0; z < NP; ++z) q[x][z][y][w][e] = p[z];
          }
        }
        a += __shfl_xor(a, 16);
        qs[x][y] = a + __shfl_xor(a, 32);
      }
#pragma unroll
      for (int y = 0; y < GV; ++y) corr[x][y] = 0.f, used[x][y] = f32x4{};
    }
    high = 0x43004300u;
    asm volatile("" : "+v"(high));
    vc = reinterpret_cast<const uint32_t*>(C->codes[2]) + row0 * (DV / 8);
    vpar = C->pars[2] + row0 * GV;
  }
  // N words from word `at` on (rows past the descriptor's: zeros).
  template <int N>
  __device__ __forceinline__ static void words(uint32_t* to, __amdgpu_buffer_rsrc_t r, uint32_t at) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (N % 4 == 0) {
        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, 4 * (at + i), 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[i + e] = w[e];
      } else {
        static_assert(N == 2, "2 or a multiple of 4 words");
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, 4 * at, 0, 0);
        to[0] = w[0], to[1] = w[1];
      }
    }
  }
  __device__ __forceinline__ void load(Regs& g, int t0, int lim) {
    const int n = lane_id() & 15, kq = lane_id() >> 4, t = t0 + 4 * kq;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto c = rsrc_of(kc[x], (uint32_t)lim * (D / 2)), p = rsrc_of(kpar[x], (uint32_t)lim * (4 * GK));
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        words<2 * GK>(&g.k[x][y][0][0], c, (uint32_t)(t0 + 16 * y + n) * (D / 8) + 2 * GK * kq);
        words<4 * GK>(&g.kp[x][y][0][0], p, (uint32_t)(t + 16 * y) * GK);
      }
    }
    // codes of rows past the keys may be anything: their steps and minima are zeros
    const auto c = rsrc_of(vc, (uint32_t)((lim + 3) & ~3) * (DV / 2)), p = rsrc_of(vpar, (uint32_t)lim * (4 * GV));
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      words<4 * GV>(&g.vp[4 * y][0], p, (uint32_t)(t + 16 * y) * GV);
#pragma unroll
      for (int z = 0; z < WV; ++z)
        words<4>(&g.v[y][z][0], c, (uint32_t)(t + 16 * y) * (DV / 8) + 4 * (DV == 64 ? n >> 1 : 16 * z + n));
    }
  }
  __device__ __forceinline__ void scores(const Regs& g, f32x4 (&s)[2][2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        s[x][y] = f32x4{};
#pragma unroll
        for (int z = 0; z < GK; ++z) {
          const float start = -kBias * qs[x][z];
          f32x4 a = {start, start, start, start};
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const bf16x8 c = codes(g.k[x][y][z][w]);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) a = TrB::mma16(c, q[x][p][z][w], a);  // small parts first
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float sc = bf16_hi(g.kp[x][y][r][z]), m = bf16_lo(g.kp[x][y][r][z]);
            s[x][y][r] = __builtin_fmaf(sc, a[r], __builtin_fmaf(m, qs[x][z], s[x][y][r]));
          }
        }
      }
  }
  __device__ __forceinline__ void rescale(int x, float f) {
#pragma unroll
    for (int y = 0; y < GV; ++y) {
      corr[x][y] *= f;
      used[x][y] *= f;
    }
  }
  __device__ __forceinline__ void add(const Regs& g, const f32x4 (&s)[2][2], f32x4 (&o)[2][DV / 16]) {
    u32x4 ones;
#pragma unroll
    for (int i = 0; i < 4; ++i) ones[i] = 0x3f803f80u;
#pragma unroll
    for (int z = 0; z < GV; ++z) {
      float step[8], mid[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        step[j] = bf16_hi(g.vp[j][z]);
        mid[j] = __builtin_fmaf(8.f, step[j], bf16_lo(g.vp[j][z]));
      }
      bf16x8 p[2][NP];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = s[x][j >> 2][j & 3];
          bf16 e[NP];
          split(w * step[j], e);
#pragma unroll
          for (int y = 0; y < NP; ++y) p[x][y][j] = e[y];
          corr[x][z] = __builtin_fmaf(w, mid[j], corr[x][z]);
        }
#pragma unroll
        for (int y = NP - 1; y >= 0; --y) used[x][z] = TrB::mma16(__builtin_bit_cast(bf16x8, ones), p[x][y], used[x][z]);
      }
      uint32_t half[4];  // keys 2 i, 2 i + 1: the units of this group, side by side
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = g.v[i / 2][z / 2][2 * i % 4], b = g.v[i / 2][z / 2][2 * i % 4 + 1];
        const bool up = DV == 64 ? lane_id() & 1 : z & 1;
        half[i] = up ? __builtin_amdgcn_perm(b, a, 0x07060302) : __builtin_amdgcn_perm(b, a, 0x05040100);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pair(half[i] >> (4 * c));
        const bf16x8 a = __builtin_bit_cast(bf16x8, w);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = NP - 1; y >= 0; --y) o[x][4 * z + c] = TrB::mma16(a, p[x][y], o[x][4 * z + c]);
      }
    }
  }
  __device__ __forceinline__ void finish(f32x4 (&o)[2][DV / 16]) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int z = 0; z < GV; ++z) {
        float a = corr[x][z];
        a += __shfl_xor(a, 16);
        a += __shfl_xor(a, 32);
        a = __builtin_fmaf(-(kBias + 8.f), used[x][z][0], a);  // every value of the tile is the lane's query's sum
#pragma unroll
        for (int c = 0; c < 4; ++c) o[x][4 * z + c] += a;
      }
  }
  __device__ __forceinline__ static int column(int t, int m) { return 64 * (t / 4) + 4 * m + t % 4; }
};

// One token over (32, 32 over 8, 8192, 128) of unequal lengths, 340 MB of codes: 94 to 104 us (3.3 to 3.6 TB/s), of full
// lengths 107 us (f16 queries 176, f32 262: two and three products a code), bound by the
// instructions that turn codes into operands as much as by reading them; two waves a SIMD cover each other's
// loads (132 us; one, with the next tile's loads on their way, 188 us, both before the unpacking's last steps).
template <class T, int NP, int D, int DV>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu((DV <= 128 ? 2 : 1)))) kv4_attend(DecParams P, Kv4Params C) {
  extern __shared__ float lds[];
  Kv4Src<T, NP, D, DV> src;
  src.C = &C;
  decode_body(P, src, lds);
}

// ------------------------------------------------------------------ launches
// Rows a thread: four where that leaves enough workgroups (bf16 (4, 8, 2048, 128) read 15.7 -> 13.5 us), one for
// the few rows of a decoding step.
template <class F>
static void by_rows(const Kv4Params& p, F&& launch) {
  const int per = 2048 / (p.D > p.DV ? p.D : p.DV);  // rows of the widest a workgroup
  const int64_t heads = (int64_t)p.B * p.Hk;
  const auto go = [&](auto r) {
    const int blocks = (p.rows + per * r - 1) / (per * r);
    dim3 grid = tda::grid_of<256>(heads * blocks);
    grid.z = 3;
    launch(r, grid, blocks);
  };
  if (heads * p.rows >= 4096 * per) go(std::integral_constant<int, 4>());
  else go(std::integral_constant<int, 1>());
}
template <class T>
static void append(const Kv4Params& p, hipStream_t st) {
  by_rows(p, [&](auto r, dim3 grid, int blocks) { kv4_append<T, r><<<grid, 256, 0, st>>>(p, blocks); });
}
template <class T>
static void read(const Kv4Params& p, hipStream_t st) {
  by_rows(p, [&](auto r, dim3 grid, int blocks) { kv4_read<T, r><<<grid, 256, 0, st>>>(p, blocks); });
}
int launch_kv4_append(const Kv4Params& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) append<float>(p, st);
  else if (dtype == 1) append<bf16>(p, st);
  else append<_Float16>(p, st);
  tda::launched(st, "sda_kv4_append");
  if (!p.start || p.counts == p.lengths) {  // every workgroup above reads the lengths
    kv4_lengths<<<dim3((unsigned)((p.B + 63) / 64)), 64, 0, st>>>(p);
    tda::launched(st, "sda_kv4_lengths");
  }
  return (int)hipGetLastError();
}
int launch_kv4_read(const Kv4Params& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) read<float>(p, st);
  else if (dtype == 1) read<bf16>(p, st);
  else read<_Float16>(p, st);
  tda::launched(st, "sda_kv4_read");
  return (int)hipGetLastError();
}
template <class T, int NP, int D, int DV>
static int run(const DecParams& p, const Kv4Params& c, hipStream_t st) {
  constexpr int LDS = kDecLds<DV>;
  if (LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_attend<T, NP, D, DV>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return (int)e;
  }
  const int64_t items = (int64_t)p.B * p.Hk * ((p.H / p.Hk * (int64_t)p.Nq + kDecRows - 1) / kDecRows);
  kv4_attend<T, NP, D, DV><<<tda::grid_of<256>(items * p.nsplit), 256, LDS, st>>>(p, c);
  tda::launched(st, "sda_kv4_attend");
  if (p.nsplit > 1) {
    decode_join<T><<<tda::grid_of<256>(((int64_t)p.B * p.H * p.Nq * DV + 255) / 256), 256, 0, st>>>(p);
    tda::launched(st, "sda_decode_join");
  }
  return (int)hipGetLastError();
}
template <class T, int NP>
static int pick(const DecParams& p, const Kv4Params& c, hipStream_t st) {
  if (p.D == 64) return p.DV == 64 ? run<T, NP, 64, 64>(p, c, st) : run<T, NP, 64, 128>(p, c, st);
  return p.DV == 128 ? run<T, NP, 128, 128>(p, c, st) : run<T, NP, 128, 256>(p, c, st);
}
int launch_kv4_attend(const Kv4Params& c, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  DecParams p{};
  p.q[0] = c.q[0];
  p.q[1] = c.q[1];
  p.out = c.out;
  p.lam = c.lam;
  p.see.lens = c.lengths;
  p.tail = 1;
  p.B = c.B;
  p.H = c.H;
  p.Hk = c.Hk;
  p.Nq = c.Nq;
  p.Nk = c.cap;
  p.D = c.D;
  p.DV = c.DV;
  p.c = c.c;
  p.part = c.part;
  p.nsplit = c.nsplit;
  p.chunk = c.chunk;
  if (dtype == 0) return pick<float, 3>(p, c, st);
  return dtype == 1 ? pick<bf16, 1>(p, c, st) : pick<_Float16, 2>(p, c, st);
}

}  // namespace sda
