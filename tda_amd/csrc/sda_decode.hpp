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
// What a workgroup computes is a `DecWork`: dec_work deals out the tiles and parts of dense batches.  A source
// (Src) brings: D, DV, `Regs` (a tile's loads) and NBUF, begin, load, scores, rescale (a branch's running
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

// One row tile and part of a workgroup: query rows row0 .. row0 + nq - 1 of batch entry qb over the keys of
// sequence b, row i at position off + i.
struct DecWork {
  int b, hk, rt, qb, row0, nq, len, off, k0, k1;
  bool causal;
  float* part;  // where its sums go; null: its result is the output
};
__device__ __forceinline__ bool dec_work(const DecParams& P, DecWork& W) {
  const int R = P.H / P.Hk * P.Nq, tiles = (R + kDecRows - 1) / kDecRows;
  const uint32_t bid = tda::grid_bid<256>();
  const int split = (int)(bid % (uint32_t)P.nsplit), item = (int)(bid / (uint32_t)P.nsplit);
  if (item >= P.B * P.Hk * tiles) return false;
  const int bk = item / tiles;
  W.rt = item % tiles;
  W.b = W.qb = bk / P.Hk;
  W.hk = bk % P.Hk;
  W.row0 = 0;
  W.nq = P.Nq;
  W.len = len_of(P.see, W.b, P.Nk);
  W.off = P.tail ? W.len - P.Nq : off_of(P.see, W.b);
  W.causal = P.see.causal || P.tail;
  // rows of the tile are consecutive, so its last position bounds the keys it needs (where the tile
  // spans heads the bound is the last row's)
  const int lim = W.causal ? max(min(W.len, W.off + P.Nq), 0) : W.len;
  W.k0 = split * P.chunk;
  W.k1 = min(W.k0 + P.chunk, lim);
  W.part = P.nsplit > 1 ? P.part + ((int64_t)item * P.nsplit + split) * dec_part_floats(P.DV) : nullptr;
  return true;
}

template <class Src>
__device__ __forceinline__ void decode_body(const DecParams& P, const DecWork& W, Src& src, float* lds) {
  constexpr int DV = Src::DV, NO = DV / 16;
  const int l = lane_id(), n = l & 15, kq = l >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = P.H / P.Hk, R = G * W.nq, rt = W.rt, hk = W.hk, k0 = W.k0, k1 = W.k1;
  const int row = rt * kDecRows + n;
  const bool live = row < R;
  const int i = live ? row % W.nq : 0, h = hk * G + (live ? row / W.nq : 0);
  const int lim = W.causal ? max(min(W.len, W.off + W.nq), 0) : W.len;
  const int see = live && W.causal ? max(min(W.len, W.off + i + 1), 0) : lim;

  f32x4 o[2][NO] = {};
  float m[2] = {kNoMax, kNoMax}, sum[2] = {0.f, 0.f};
  if (k0 < k1) {
    src.begin(P, W, h, i, live);
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
  float* part = W.part;
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
      scale[16 * x + n] = x && live ? -lambda_of(P.lam, W.qb, h, W.row0 + i) * inv : inv;
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
    row_of<T>(P.out, W.qb, hk * G + q / W.nq, W.row0 + q % W.nq)[c] = (T)__builtin_fmaf(scale[16 + r], fin[1][k], scale[r] * fin[0][k]);
  }
}
template <int DV>
constexpr int kDecLds = (4 * 16 * kDecRow<DV> + 256 + 32) * 4;

// Keys and values in the queries' own type, at fixed strides.
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
  __device__ __forceinline__ void begin(const DecParams& P, const DecWork& W, int h, int i, bool live) {
    const int kq = lane_id() >> 4;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      kp[x] = row_of<T>(F->k[x], W.b, W.hk, 0);
      ks[x] = F->k[x].st;
      const T* r = row_of<T>(P.q[x], W.qb, h, W.row0 + i);
#pragma unroll
      for (int t = 0; t < NT; ++t) q[x][t] = live ? load8(r + 32 * t + 8 * kq) : frag{};
    }
    vp = row_of<T>(F->v, W.b, W.hk, 0);
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
