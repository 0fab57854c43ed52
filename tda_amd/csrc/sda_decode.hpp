// sda_decode.hpp -- attention of few query rows over a long key axis, shared by the cache forms.
//
// The G Nq query rows of the heads that share a key head form tiles of 16; a workgroup takes one tile
// and one part of the keys, its four waves every fourth tile of 32 keys.  Products are 16x16: S^T =
// K Q^T (lane: one query row and 4 of 16 keys), O^T = V^T P^T with the weights fed from the registers
// that hold them: of a tile of 32 keys the second product takes, from lane quarter kq, keys 4 kq + j
// and 16 + 4 kq + j (j = 0 .. 3), and the value fragments are read in that order.  Nothing is staged:
// every key and value byte is used by one wave alone and goes straight to its registers.  Bound by
// reading the cache.  The waves' sums meet in LDS, the parts' in a second launch.
//
// A source (Src) brings: D, DV, `Regs` (a tile's loads) and NBUF, load, scores, add (O += V^T P^T), finish and column (the output column of value r of tile t in lane
// quarter kq).
#pragma once

#include "sda_common.hpp"

namespace sda {

struct DecParams {
  Rows q[2], out;
  Lambda lam;
  Sight see;
  int tail;      // 1: the rows are the last Nq positions before len (off = len - Nq)
  int B, H, Hk, Nq, Nk, D, DV;
  float c;
  float* part;   // per (b, hk, row tile, split): m, l of 2 branches x 16 rows, then 2 x DV x 16 sums
  int nsplit, chunk;
};
constexpr int kDecRows = 16;
__host__ __device__ constexpr int64_t dec_part_floats(int dv) { return 64 + 2 * 16 * (int64_t)dv; }

template <class Src>
__device__ __forceinline__ void decode_body(const DecParams& P, Src& src, float* lds) {
  constexpr int DV = Src::DV, NO = DV / 16;
  const int l = lane_id(), n = l & 15, kq = l >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = P.H / P.Hk, R = G * P.Nq, tiles = (R + kDecRows - 1) / kDecRows;
  const uint32_t bid = tda::grid_bid<256>();
  const int split = (int)(bid % (uint32_t)P.nsplit), item = (int)(bid / (uint32_t)P.nsplit);
  if (item >= P.B * P.Hk * tiles) return;
  const int rt = item % tiles, bk = item / tiles, b = bk / P.Hk, hk = bk % P.Hk;
  const int row = rt * kDecRows + n;
  const bool live = row < R;
  const int i = live ? row % P.Nq : 0, h = hk * G + (live ? row / P.Nq : 0);
  const int len = len_of(P.see, b, P.Nk);
  const int off = P.tail ? len - P.Nq : off_of(P.see, b);
  const bool causal = P.see.causal || P.tail;
  // rows of the tile are consecutive, so its last position bounds the keys it needs (where the tile
  // spans heads the bound is the last row's)
  const int lim = causal ? max(min(len, off + P.Nq), 0) : len;
  const int see = live && causal ? max(min(len, off + i + 1), 0) : lim;
  const int k0 = split * P.chunk, k1 = min(k0 + P.chunk, lim);

  f32x4 o[2][NO] = {};
  float m[2] = {kNoMax, kNoMax}, sum[2] = {0.f, 0.f};
  if (k0 < k1) {
    src.begin(P, b, hk, h, i, live);
    // NBUF tiles' registers: one in use, the others' loads on their way.  Rows past the part's end, and
    // whole tiles, read as zeros by the buffer descriptors' range check: a weight of zero times whatever lies
    // there must stay zero.  (Skipping such loads would keep the compiler from counting the loads behind
    // the one it waits for.)
    constexpr int NBUF = Src::NBUF;
    typename Src::Regs regs[NBUF];
    const int t1 = k0 + 32 * wv;
    times<NBUF - 1>([&](auto u) { src.load(regs[u], t1 + 128 * u, k1); });
    auto tile = [&](typename Src::Regs& r, int t0) {
      f32x4 w[2][2];
      src.scores(r, w);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        f32x4(&s)[2] = w[x];
        if (__any(t0 + 31 >= see)) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t0 + 16 * y + 4 * kq + e >= min(see, k1)) s[y][e] = -__builtin_inff();
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * P.c;
        if (__any(top > m[x] + kSlack)) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float to = fmaxf(m[x], top), f = exp2_(m[x] - to);
          m[x] = to;
          sum[x] *= f;
          src.rescale(x, f);
#pragma unroll
          for (int y = 0; y < NO; ++y) o[x][y] *= f;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[y][e] = exp2_(__builtin_fmaf(s[y][e], P.c, -m[x]));
          sum[x] += (s[y][0] + s[y][1]) + (s[y][2] + s[y][3]);
        }
      }
      src.add(r, w, o);
    };
    for (int t0 = t1; t0 < k1; t0 += 128 * NBUF)
      times<NBUF>([&](auto u) {
        const int t = t0 + 128 * u;
        src.load(regs[(u + NBUF - 1) % NBUF], t + 128 * (NBUF - 1), k1);
        if (t < k1) tile(regs[u], t);
      });
    src.finish(o);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    sum[x] += __shfl_xor(sum[x], 16);
    sum[x] += __shfl_xor(sum[x], 32);
  }
  // the waves' maxima and sums, then their outputs under the common maximum
  float* ml = lds + 4 * 2 * DV * 16;  // [wave][branch][m, l][16]
  if (kq == 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      ml[((wv * 2 + x) * 2) * 16 + n] = m[x];
      ml[((wv * 2 + x) * 2 + 1) * 16 + n] = sum[x];
    }
  }
  __syncthreads();
  float all[2], tot[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    all[x] = kNoMax;
    tot[x] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) all[x] = fmaxf(all[x], ml[((w * 2 + x) * 2) * 16 + n]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      tot[x] = __builtin_fmaf(ml[((w * 2 + x) * 2 + 1) * 16 + n], exp2_(ml[((w * 2 + x) * 2) * 16 + n] - all[x]), tot[x]);
    const float f = exp2_(m[x] - all[x]);
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        lds[((wv * 2 + x) * DV + Src::column(y, 4 * kq + r)) * 16 + n] = o[x][y][r] * f;
  }
  __syncthreads();
  // thread t: row t % 16, columns t / 16, + 16, ...
  const int tid = threadIdx.x, c0 = tid >> 4;
  if (P.nsplit > 1) {
    float* to = P.part + ((int64_t)item * P.nsplit + split) * dec_part_floats(DV);
    if (tid < 16) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        to[32 * x + n] = all[x];
        to[32 * x + 16 + n] = tot[x];
      }
    }
    if (k0 >= k1) return;  // no sums: the joining launch skips a part without weight
#pragma unroll
    for (int x = 0; x < 2; ++x)
      for (int y = c0; y < DV; y += 16) {
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) a += lds[((w * 2 + x) * DV + y) * 16 + n];
        to[64 + (x * DV + y) * 16 + n] = a;
      }
    return;
  }
  const float lam = live ? lambda_of(P.lam, b, h, i) : 0.f;
  float inv[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) inv[x] = tot[x] > 0.f || tot[x] != tot[x] ? 1.0f / tot[x] : 0.f;
  // the rows' outputs turned in LDS so that a thread stores along a row
  float* turned = lds + 4 * 2 * DV * 16 + 256;  // [16][DV + 1]
  for (int y = c0; y < DV; y += 16) {
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int w = 0; w < 4; ++w) a[x] += lds[((w * 2 + x) * DV + y) * 16 + n];
    turned[n * (DV + 1) + y] = __builtin_fmaf(-lam * inv[1], a[1], a[0] * inv[0]);
  }
  __syncthreads();
  using T = typename Src::Out;
  for (int e = tid; e < 16 * DV; e += 256) {
    const int r = rt * kDecRows + e / DV;
    if (r >= R) break;
    row_of<T>(P.out, b, hk * G + r / P.Nq, r % P.Nq)[e % DV] = (T)turned[(e / DV) * (DV + 1) + e % DV];
  }
}
template <int DV>
constexpr int kDecLds = (4 * 2 * DV * 16 + 256 + 16 * (DV + 1)) * 4;

// Joins the parts of 16 rows: thread per (row, column of a group of 16), parts in order.
template <class T>
__global__ void __launch_bounds__(256) decode_join(DecParams P) {
  const int G = P.H / P.Hk, R = G * P.Nq, tiles = (R + kDecRows - 1) / kDecRows, DV = P.DV;
  const int cols = DV / 16;
  const uint32_t bid = tda::grid_bid<256>();
  const int cb = (int)(bid % (uint32_t)cols), item = (int)(bid / (uint32_t)cols);
  if (item >= P.B * P.Hk * tiles) return;
  const int rt = item % tiles, bk = item / tiles, b = bk / P.Hk, hk = bk % P.Hk;
  const int n = threadIdx.x & 15, y = 16 * cb + (threadIdx.x >> 4);
  const int64_t step = dec_part_floats(DV);
  const float* base = P.part + (int64_t)item * P.nsplit * step;
  // eight parts at a time: their loads are on their way together
  float res[2];
  float all[2] = {kNoMax, kNoMax}, l[2] = {}, a[2] = {};
  for (int s0 = 0; s0 < P.nsplit; s0 += 8) {
    float mm[2][8], ll[2][8], aa[2][8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float* part = base + min(s0 + u, P.nsplit - 1) * step;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mm[x][u] = part[32 * x + n];
        ll[x][u] = s0 + u < P.nsplit ? part[32 * x + 16 + n] : 0.f;
        aa[x][u] = part[64 + (x * DV + y) * 16 + n];
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = all[x];
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, mm[x][u]);
      const float f = exp2_(all[x] - top);
      l[x] *= f;
      a[x] *= f;
      all[x] = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = exp2_(mm[x][u] - top);
        if (ll[x][u] != 0.f) {  // else no key of this part: its sums are not written
          l[x] = __builtin_fmaf(ll[x][u], w, l[x]);
          a[x] = __builtin_fmaf(aa[x][u], w, a[x]);
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) res[x] = l[x] > 0.f || l[x] != l[x] ? a[x] / l[x] : 0.f;
  __shared__ float turned[16][17];
  const int row = rt * kDecRows + n;
  const bool live = row < R;
  const float lam = live ? lambda_of(P.lam, b, hk * G + row / P.Nq, row % P.Nq) : 0.f;
  turned[n][threadIdx.x >> 4] = __builtin_fmaf(-lam, res[1], res[0]);
  __syncthreads();
  const int r = rt * kDecRows + (threadIdx.x >> 4);
  if (r < R) row_of<T>(P.out, b, hk * G + r / P.Nq, r % P.Nq)[16 * cb + n] = (T)turned[threadIdx.x >> 4][n];
}

}  // namespace sda
