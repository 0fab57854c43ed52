// sln.hip -- layer norm over the last axis (RMS norm without `center`), forward and backward.
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  g = dy w;   dw = sum dy xhat,  db = sum dy
//
// A row stays in the registers of the lanes that share it: 8 to 64 lanes of a wave for rows of up to 4 KB, with the
// row's sums by lane moves, and 256 or 1024 threads beyond, whose waves' sums meet in LDS.  A lane's pieces are the same
// columns of every row, so it keeps the sums of dw and db in registers over all its rows; a workgroup leaves one row of
// them, and a second launch adds those up in order (where there are few rows, one workgroup takes them all and writes the
// result).  All sums are 32 bits; the variance is taken around the mean (of a wave, joined by the waves' means).
// Bound by memory, each value read and written once a pass.  bf16, kernels within training steps, one run: 2^18 rows of 128, forward 24 us
// (134 MB, 5.5 TB/s), backward 44 (201 MB, 4.6 TB/s); 16384 rows of 4096, 58 (268 MB, 4.6 TB/s) and 79 (403 MB, 5.1 TB/s).  Another
// part took 31 and 47, 60 and 80.
#include "sda_common.hpp"
#include "sln_params.hpp"

namespace sln {

using sda::lane_id;

// Pieces of V values: whole ones where the width is a number of them (WHOLE), else the last of a row may end
// inside; those behind it are zeros, not read and not written.
template <class T, bool WHOLE>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef vec any __attribute__((aligned(sizeof(T))));  // at any element
  __device__ __forceinline__ static vec load(const T* row, int col, int width) {
    vec x = {};
    if (WHOLE ? col < width : col + V <= width) return *reinterpret_cast<const any*>(row + col);
    if constexpr (!WHOLE) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < width) x[e] = row[col + e];
    }
    return x;
  }
  __device__ __forceinline__ static void store(T* row, int col, int width, vec x) {
    if (WHOLE ? col < width : col + V <= width) {
      *reinterpret_cast<any*>(row + col) = x;
      return;
    }
    if constexpr (!WHOLE) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < width) row[col + e] = x[e];
    }
  }
};
// V weights (of the rows' type or f32) from column col on.
template <class T, bool WHOLE, int V>
__device__ __forceinline__ void weights(const void* p, int type, int64_t row, int col, int width, float (&w)[V]) {
  if (type == 0) {
    using P = Piece<float, WHOLE>;
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const auto x = P::load(static_cast<const float*>(p) + row * width, col + k, width);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[k + e] = x[e];
    }
  } else {
    const auto x = Piece<T, WHOLE>::load(static_cast<const T*>(p) + row * width, col, width);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = (float)x[e];
  }
}

template <class T>
__device__ __forceinline__ void put_sum(void* p, int type, int64_t at, float x) {
  if (type == 0) static_cast<float*>(p)[at] = x;
  else static_cast<T*>(p)[at] = (T)x;
}

// Sum over the L lanes that share a row (of a wave, if they are more).
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
  x = tda::group_sum<(L < 16 ? L : 16)>(x);
  if constexpr (L >= 32) x += __shfl_xor(x, 16);
  if constexpr (L >= 64) x += __shfl_xor(x, 32);
  return x;
}

struct Where { int i0, i1, i2; };
__device__ __forceinline__ Where where(const Params& P, int row) {
  Where w = {0, 0, row};
  if (P.n[2] != P.rows) {
    w.i2 = row % P.n[2];
    const int up = row / P.n[2];
    w.i1 = up % P.n[1];
    w.i0 = up / P.n[1];
  }
  return w;
}
template <class T>
__device__ __forceinline__ T* at(const Tensor& t, int group, const Where& w) {
  return static_cast<T*>(t.p) + group * t.group + w.i0 * t.s[0] + w.i1 * t.s[1] + w.i2 * t.s[2];
}

template <class T, bool WHOLE, int L, int C, int U>
__global__ void __launch_bounds__(L <= 64 ? 256 : L) norm_fwd(Params P, int blocks) {
  using Pc = Piece<T, WHOLE>;
  using vec = typename Pc::vec;
  constexpr int V = Pc::V, TH = L <= 64 ? 256 : L, PER = TH / L * U, WV = L / 64;
  __shared__ float2 lds[2][16];
  const uint32_t bid = tda::grid_bid<TH>();
  const int grp = (int)(bid % (uint32_t)P.groups), blk = (int)(bid / (uint32_t)P.groups);
  if (blk >= blocks) return;
  const int lane = threadIdx.x % L, width = P.width, wv = threadIdx.x >> 6;
  const float inv_n = 1.0f / (float)width;
  constexpr bool KEEP = C <= 2;  // the weights stay in registers
  float w[KEEP ? C : 1][V], b[KEEP ? C : 1][V];
  const auto load_w = [&](int c, float(&ww)[V], float(&bb)[V]) {
    const int col = (lane + L * c) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ww[e] = 1.f, bb[e] = 0.f;
    if (P.weight) weights<T, WHOLE, V>(P.weight, P.weight_type, grp, col, width, ww);
    if (P.bias) weights<T, WHOLE, V>(P.bias, P.weight_type, grp, col, width, bb);
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int c = 0; c < C; ++c) load_w(c, w[c], b[c]);
  }
  // values of this wave's part of a row, for joining the waves' variances
  float part = 0.f;
  if constexpr (L > 64) {
#pragma unroll
    for (int c = 0; c < C; ++c) part += (float)min(max(width - (wv * 64 + L * c) * V, 0), 64 * V);
  }
  int turn = 0;
  for (int64_t r0 = (int64_t)blk * PER; r0 < P.rows; r0 += (int64_t)blocks * PER) {
    vec x[U][C];
    Where at_[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * (TH / L) + threadIdx.x / L;
      live[u] = r < P.rows;
      at_[u] = where(P, (int)(live[u] ? r : r0));
      const T* row = at<const T>(P.x, grp, at_[u]);
#pragma unroll
      for (int c = 0; c < C; ++c) x[u][c] = Pc::load(row, (lane + L * c) * V, width);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float mean = 0.f, m2 = 0.f;
      if (P.center) {
        float s[2] = {};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) s[e & 1] += (float)x[u][c][e];
        mean = lanes_sum<(L < 64 ? L : 64)>(s[0] + s[1]);
      }
      const float sum = mean;
      mean = L <= 64 ? mean / (float)width : part > 0.f ? mean / part : 0.f;  // a quotient: a constant row's is exact
      float s[2] = {};
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = (lane + L * c) * V + e < width ? (float)x[u][c][e] - mean : 0.f;
          s[e & 1] = __builtin_fmaf(d, d, s[e & 1]);
        }
      m2 = lanes_sum<(L < 64 ? L : 64)>(s[0] + s[1]);
      if constexpr (L > 64) {
        // the waves' sums and squares around their own means: M2 = sum of m2 + n (mean of the wave - mean)^2
        float2* put = lds[turn];
        turn ^= 1;
        if (lane_id() == 0) put[wv] = make_float2(sum, m2);
        __syncthreads();  // one a row: the next row's go to the other half
        float all = 0.f;
#pragma unroll
        for (int k = 0; k < WV; ++k) all += put[k].x;
        mean = all / (float)width;
        m2 = 0.f;
#pragma unroll
        for (int k = 0; k < WV; ++k) {
          float nk = 0.f;
#pragma unroll
          for (int c = 0; c < C; ++c) nk += (float)min(max(width - (k * 64 + L * c) * V, 0), 64 * V);
          const float d = P.center && nk > 0.f ? put[k].x / nk - mean : 0.f;
          m2 += __builtin_fmaf(nk * d, d, put[k].y);
        }
      }
      const float rstd = 1.0f / sqrtf(__builtin_fmaf(m2, inv_n, P.eps));
      if (!live[u]) continue;
      if (P.stats.p && lane == 0) {
        *at<float2>(P.stats, grp, at_[u]) = make_float2(mean, rstd);
      }
      T* row = at<T>(P.y, grp, at_[u]);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float ww[V], bb[V];
        if constexpr (!KEEP) load_w(c, ww, bb);
        vec y;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = ((float)x[u][c][e] - mean) * rstd;
          y[e] = (T)__builtin_fmaf(xh, KEEP ? w[KEEP ? c : 0][e] : ww[e], KEEP ? b[KEEP ? c : 0][e] : bb[e]);
        }
        Pc::store(row, (lane + L * c) * V, width, y);
      }
    }
  }
}

template <class T, bool WHOLE, int L, int C, int U>
__global__ void __launch_bounds__(bwd_threads(L)) norm_bwd(Params P) {
  using Pc = Piece<T, WHOLE>;
  using vec = typename Pc::vec;
  constexpr int V = Pc::V, TH = bwd_threads(L), PER = TH / L * U, WV = L / 64;
  extern __shared__ float sums[];  // [dw, db][width], one wave (L > 64: one set of waves) after another
  __shared__ float2 lds[2][16];
  const uint32_t bid = tda::grid_bid<TH>();
  const int grp = (int)(bid % (uint32_t)P.groups), blk = (int)(bid / (uint32_t)P.groups);
  if (blk >= P.blocks) return;
  const int lane = threadIdx.x % L, width = P.width, wv = threadIdx.x >> 6;
  const float inv_n = 1.0f / (float)width;
  constexpr bool KEEP = C <= 2;
  float w[KEEP ? C : 1][V];
  const auto load_w = [&](int c, float(&ww)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) ww[e] = 1.f;
    if (P.weight) weights<T, WHOLE, V>(P.weight, P.weight_type, grp, (lane + L * c) * V, width, ww);
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int c = 0; c < C; ++c) load_w(c, w[c]);
  }
  float dw[C][V] = {}, db[C][V] = {};
  int turn = 0;
  for (int64_t r0 = (int64_t)blk * PER; r0 < P.rows; r0 += (int64_t)P.blocks * PER) {
    vec x[U][C], dy[U][C];
    float2 st[U];
    Where at_[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * (TH / L) + threadIdx.x / L;
      live[u] = r < P.rows;
      at_[u] = where(P, (int)(live[u] ? r : r0));
      const T *px = at<const T>(P.x, grp, at_[u]), *pd = at<const T>(P.dy, grp, at_[u]);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[u][c] = Pc::load(px, (lane + L * c) * V, width);
        dy[u][c] = live[u] ? Pc::load(pd, (lane + L * c) * V, width) : vec{};
      }
      st[u] = *at<const float2>(P.stats, grp, at_[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float mean = st[u].x, rstd = live[u] ? st[u].y : 0.f;
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float ww[V];
        if constexpr (!KEEP) load_w(c, ww);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = (float)dy[u][c][e], xh = ((float)x[u][c][e] - mean) * rstd;
          const float gg = d * (KEEP ? w[KEEP ? c : 0][e] : ww[e]);
          c1 += gg;
          c2 = __builtin_fmaf(gg, xh, c2);
          if (live[u]) {
            dw[c][e] = __builtin_fmaf(d, xh, dw[c][e]);
            db[c][e] += d;
          }
        }
      }
      if (!P.dx.p) continue;  // the same in every thread
      c1 = lanes_sum<(L < 64 ? L : 64)>(c1);
      c2 = lanes_sum<(L < 64 ? L : 64)>(c2);
      if constexpr (L > 64) {
        float2* put = lds[turn];
        turn ^= 1;
        if (lane_id() == 0) put[wv] = make_float2(c1, c2);
        __syncthreads();  // one a row: the next row's go to the other half
        c1 = c2 = 0.f;
#pragma unroll
        for (int k = 0; k < WV; ++k) {
          const float2 z = put[wv / WV * WV + k];
          c1 += z.x;
          c2 += z.y;
        }
      }
      if (!live[u]) continue;
      c1 = P.center ? c1 * inv_n : 0.f;
      c2 *= inv_n;
      T* row = at<T>(P.dx, grp, at_[u]);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float ww[V];
        if constexpr (!KEEP) load_w(c, ww);
        vec z;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = ((float)x[u][c][e] - mean) * rstd;
          const float gg = (float)dy[u][c][e] * (KEEP ? w[KEEP ? c : 0][e] : ww[e]);
          z[e] = (T)(rstd * (gg - __builtin_fmaf(xh, c2, c1)));
        }
        Pc::store(row, (lane + L * c) * V, width, z);
      }
    }
  }
  if (!P.dweight && !P.dbias) return;
  // the rows that a wave has side by side, then the waves, in order
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
      for (int d = L; d < 64; d *= 2) {
        dw[c][e] += __shfl_xor(dw[c][e], d);
        db[c][e] += __shfl_xor(db[c][e], d);
      }
    }
  constexpr int SETS = L < 64 ? TH / 64 : TH / L;
  const int set = threadIdx.x / (L < 64 ? 64 : L);
  for (int s = 0; s < SETS; ++s) {
    if (set == s && (L >= 64 || lane_id() < L)) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int col = (lane + L * c) * V + e;
          if (col < width) {
            sums[col] = s ? sums[col] + dw[c][e] : dw[c][e];
            sums[width + col] = s ? sums[width + col] + db[c][e] : db[c][e];
          }
        }
    }
    __syncthreads();
  }
  if (P.part) {
    float* to = P.part + ((int64_t)grp * P.blocks + blk) * 2 * width;
    for (int e = threadIdx.x; e < 2 * width; e += TH) to[e] = sums[e];
    return;
  }
  for (int e = threadIdx.x; e < width; e += TH) {
    if (P.dweight) put_sum<T>(P.dweight, P.weight_type, (int64_t)grp * width + e, sums[e]);
    if (P.dbias) put_sum<T>(P.dbias, P.weight_type, (int64_t)grp * width + e, sums[width + e]);
  }
}

// Adds up the workgroups' rows of sums: 32 columns a workgroup, every eighth row a thread, then those eight.
template <class T>
__global__ void __launch_bounds__(256) norm_sums(Params P) {
  __shared__ float lds[8][33];
  const int cb = (P.width + 31) / 32;
  uint32_t bid = tda::grid_bid<256>();
  const int blk = (int)(bid % (uint32_t)cb);
  bid /= (uint32_t)cb;
  const int which = (int)(bid & 1), grp = (int)(bid >> 1);
  if (grp >= P.groups) return;
  void* out = which ? P.dbias : P.dweight;
  if (!out) return;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, col = 32 * blk + x;
  float s[4] = {};
  if (col < P.width) {
    const float* p = P.part + ((int64_t)grp * P.blocks * 2 + which) * P.width + col;
    const int64_t step = 2 * (int64_t)P.width;
    int k = y;
    for (; k + 24 < P.blocks; k += 32)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += p[(k + 8 * u) * step];
    for (; k < P.blocks; k += 8) s[0] += p[k * step];
  }
  lds[y][x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (y || col >= P.width) return;
  float all = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) all += lds[k][x];
  put_sum<T>(out, P.weight_type, (int64_t)grp * P.width + col, all);
}

// ------------------------------------------------------------------ launches
template <class T, bool WHOLE, int L, int C, int U>
static int fwd(const Params& p, hipStream_t st) {
  constexpr int TH = L <= 64 ? 256 : L, PER = TH / L * U;
  // Workgroups that each take a few rows: the loads of one are on their way while others sum.  The run of the figures above: 2^18 rows of 128
  // 24.3 us, with 2048 workgroups 25.0; 16384 rows of 4096, whose weights each workgroup reads, 58 with 4096, 56 with half as many, 80 with
  // four times (the other part: 62.6, 65 and 88).
  const int64_t most = ((int64_t)p.rows + PER - 1) / PER, want = ((L <= 64 ? 16384 : 4096 * 256 / TH) + p.groups - 1) / p.groups;
  const int blocks = (int)(most < want ? most : want);
  norm_fwd<T, WHOLE, L, C, U><<<tda::grid_of<TH>((int64_t)blocks * p.groups), TH, 0, st>>>(p, blocks);
  tda::launched(st, "sln_fwd");
  return (int)hipGetLastError();
}
template <class T, bool WHOLE, int L, int C, int U>
static int bwd(const Params& p, hipStream_t st) {
  constexpr int TH = bwd_threads(L);
  const int lds = p.dweight || p.dbias ? 2 * p.width * 4 : 0;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&norm_bwd<T, WHOLE, L, C, U>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
  }
  norm_bwd<T, WHOLE, L, C, U><<<tda::grid_of<TH>((int64_t)p.blocks * p.groups), TH, lds, st>>>(p);
  tda::launched(st, "sln_bwd");
  if (p.part) {
    norm_sums<T><<<tda::grid_of<256>((int64_t)p.groups * 2 * ((p.width + 31) / 32)), 256, 0, st>>>(p);
    tda::launched(st, "sln_sums");
  }
  return (int)hipGetLastError();
}
template <int N>
using Int = std::integral_constant<int, N>;
// go(lanes, pieces, rows in hand at a time): the shorter a lane's part of a row, the more of them it loads at once.
template <class T, class F>
static int by_width(const Params& p, int dtype, F&& go) {
  const Split s = split_of(p.width, dtype);
  if (s.lanes == 8) return go(Int<8>(), Int<1>(), Int<4>());
  if (s.lanes == 16) return go(Int<16>(), Int<1>(), Int<4>());
  if (s.lanes == 32) return go(Int<32>(), Int<1>(), Int<4>());
  if (s.lanes == 64)
    return s.pieces == 1 ? go(Int<64>(), Int<1>(), Int<4>()) : s.pieces == 2 ? go(Int<64>(), Int<2>(), Int<2>()) : go(Int<64>(), Int<4>(), Int<1>());
  if (s.lanes == 256) return s.pieces == 2 ? go(Int<256>(), Int<2>(), Int<1>()) : go(Int<256>(), Int<4>(), Int<1>());
  if constexpr (sizeof(T) == 4) {  // the widest 16-bit row is two pieces for each of 1024 threads
    if (s.pieces == 4) return go(Int<1024>(), Int<4>(), Int<1>());
  }
  return go(Int<1024>(), Int<2>(), Int<1>());
}
template <class T>
static int run_fwd(const Params& p, int dtype, hipStream_t st) {
  if (p.width % (16 / (int)sizeof(T)) == 0) return by_width<T>(p, dtype, [&](auto l, auto c, auto u) { return fwd<T, true, l, c, u>(p, st); });
  return by_width<T>(p, dtype, [&](auto l, auto c, auto u) { return fwd<T, false, l, c, u>(p, st); });
}
template <class T>
static int run_bwd(const Params& p, int dtype, hipStream_t st) {
  if (p.width % (16 / (int)sizeof(T)) == 0) return by_width<T>(p, dtype, [&](auto l, auto c, auto u) { return bwd<T, true, l, c, u>(p, st); });
  return by_width<T>(p, dtype, [&](auto l, auto c, auto u) { return bwd<T, false, l, c, u>(p, st); });
}
int launch_fwd(const Params& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? run_fwd<float>(p, dtype, st) : dtype == 1 ? run_fwd<tda::bf16>(p, dtype, st) : run_fwd<_Float16>(p, dtype, st);
}
int launch_bwd(const Params& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? run_bwd<float>(p, dtype, st) : dtype == 1 ? run_bwd<tda::bf16>(p, dtype, st) : run_bwd<_Float16>(p, dtype, st);
}

}  // namespace sln
