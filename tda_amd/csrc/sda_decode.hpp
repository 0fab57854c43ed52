// sda_decode.hpp -- attention of few query rows over a long key axis, shared by the cache forms.
//
// The G Nq query rows of the heads that share a key head form tiles of 16; a workgroup takes one tile
// and one part of the keys, its four waves every fourth tile of 32 keys.  Products are 16x16: S^T =
// K Q^T (lane: one query row and 4 of 16 keys), O^T = V^T P^T with the weights fed from the registers
// that hold them: of a tile of 32 keys the second product takes, from lane quarter kq, keys 4 kq + j
// and 16 + 4 kq + j (j = 0 .. 3), and the value fragments are read in that order.  Nothing is staged:
// every key and value byte is used by one wave alone and goes straight to its registers.  Bound by
// reading the cache: one token over bf16 (32, 32 over 8, 8192, 128) of unequal lengths, 1.22 GB, 256 us and
// 4.8 us for the join (4.7 TB/s; a copy reaches 5.1 to 5.2), of full lengths 5.3 TB/s; f32 (16, 32 over 8, 8192, 128)
// 4.1, (16, 32 over 8, 8192, 64) 5.1.  The waves' sums meet in LDS, the parts' in a second
// launch.
//
// A source (Src) brings: D, DV, `Regs` (a tile's loads) and NBUF, load, scores, rescale (a branch's running
// maximum moved), add (O += V^T P^T), finish and column (the output column of value m of tile t).
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
  float* part;   // per (b, hk, row tile, split): [branch][m, l][16 rows], then sums [branch][row][DV]
  int nsplit, chunk;
};
constexpr int kDecRows = 16;
template <int DV>
constexpr int kDecRow = DV + 4;  // LDS row stride of a wave's sums: rows start in different banks
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
  // the waves' maxima and sums, then their outputs under the common maximum, a branch at a time
  float* ml = lds + 4 * 16 * kDecRow<DV>;  // [wave][branch][m, l][16]
  float* scale = ml + 256;                 // [branch][16]: 1 / l, times -lambda for branch 2
  if (kq == 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      ml[((wv * 2 + x) * 2) * 16 + n] = m[x];
      ml[((wv * 2 + x) * 2 + 1) * 16 + n] = sum[x];
    }
  }
  const int tid = threadIdx.x, rows = min(kDecRows, R - rt * kDecRows);
  float* part = P.nsplit > 1 ? P.part + ((int64_t)item * P.nsplit + split) * dec_part_floats(DV) : nullptr;
  float fin[2][DV / 16];  // this thread's values: tid + 256 k, by row, then column
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    __syncthreads();
    float all = kNoMax, tot = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) all = fmaxf(all, ml[((w * 2 + x) * 2) * 16 + n]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      tot = __builtin_fmaf(ml[((w * 2 + x) * 2 + 1) * 16 + n], exp2_(ml[((w * 2 + x) * 2) * 16 + n] - all), tot);
    const float f = exp2_(m[x] - all);
#pragma unroll
    for (int y = 0; y < NO; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) lds[(wv * 16 + n) * kDecRow<DV> + Src::column(y, 4 * kq + r)] = o[x][y][r] * f;
    if (tid < 16) {
      const float inv = tot > 0.f || tot != tot ? 1.0f / tot : 0.f;
      scale[16 * x + n] = x && live ? -lambda_of(P.lam, b, h, i) * inv : inv;
      if (part) {
        part[32 * x + n] = all;
        part[32 * x + 16 + n] = tot;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < DV / 16; ++k) {
      const int e = tid + 256 * k, r = e / DV, c = e % DV;
      if (r < rows) {
        fin[x][k] = (lds[r * kDecRow<DV> + c] + lds[(16 + r) * kDecRow<DV> + c]) +
                    (lds[(32 + r) * kDecRow<DV> + c] + lds[(48 + r) * kDecRow<DV> + c]);
        if (part && k0 < k1) part[64 + (x * 16 + r) * DV + c] = fin[x][k];  // a part without keys: not read
      }
    }
  }
  if (part) return;
  using T = typename Src::Out;
#pragma unroll
  for (int k = 0; k < DV / 16; ++k) {
    const int e = tid + 256 * k, r = e / DV, c = e % DV;
    if (r >= rows) break;
    const int q = rt * kDecRows + r;
    row_of<T>(P.out, b, hk * G + q / P.Nq, q % P.Nq)[c] = (T)__builtin_fmaf(scale[16 + r], fin[1][k], scale[r] * fin[0][k]);
  }
}
template <int DV>
constexpr int kDecLds = (4 * 16 * kDecRow<DV> + 256 + 32) * 4;

// Joins the parts: a thread per value, the parts in order, eight at a time (their loads are on their way
// together: eight parts of (32, 32, 1, 128) 4.5 us, 11.4 us one at a time).
template <class T>
__global__ void __launch_bounds__(256) decode_join(DecParams P) {
  const int G = P.H / P.Hk, R = G * P.Nq, tiles = (R + kDecRows - 1) / kDecRows, DV = P.DV;
  const int64_t id = (int64_t)tda::grid_bid<256>() * 256 + threadIdx.x;
  const int c = (int)(id % DV);
  const int64_t at = id / DV;  // (b, hk, row)
  if (at >= (int64_t)P.B * P.Hk * R) return;
  const int row = (int)(at % R), bk = (int)(at / R), b = bk / P.Hk, hk = bk % P.Hk;
  const int n = row % kDecRows;
  const int64_t step = dec_part_floats(DV);
  const float* base = P.part + ((int64_t)bk * tiles + row / kDecRows) * P.nsplit * step;
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
        aa[x][u] = part[64 + (x * 16 + n) * DV + c];
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
  float res[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) res[x] = l[x] > 0.f || l[x] != l[x] ? a[x] / l[x] : 0.f;
  const int h = hk * G + row / P.Nq, i = row % P.Nq;
  row_of<T>(P.out, b, h, i)[c] = (T)__builtin_fmaf(-lambda_of(P.lam, b, h, i), res[1], res[0]);
}

}  // namespace sda
