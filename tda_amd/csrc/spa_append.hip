// spa_append.hip -- rows of new positions enter the pages of a cache, queries and keys turned by their rotary
// positions on the way.
//
// A workgroup takes one token, or four: a wave finds its sequence, its place in the pages and its cosines and
// sines (64 bits, reduced to a turn there, as sda_rotary.hip takes them), then the token's rows stream through, each
// value read and written once.  Rows of q1, q2, k1, k2 and of v (one or two rows of D values a head) are alike:
// U units of 2 V values, which are V pairs or are copied.
// Bound by memory: 4 prompts of up to 2048, bf16, 32 over 8 heads of 128: 63 us, 4.8 TB/s of what is read and written; one token of each of 8
// sequences takes 4.1, a launch and its chain of loads (lengths, table, rows).  Four tokens a workgroup share a wave each for their
// angles, where there are enough of them to fill the chip.
#include "spa_common.hpp"

namespace spa {

struct Token {
  int own;      // the row belongs to a sequence
  int page, row;  // where its keys go; page -1: nowhere
  int b, i;     // where its rows are
};

template <class T, int V, int D, int DV>
__global__ void __launch_bounds__(256) append(AppendParams P, int tok, int splits) {
  constexpr int U = D / (2 * V), ROWS = 256 / U, VH = DV / D;  // rows of a pass; rows of D values in one of v
  __shared__ Token token[4];
  __shared__ float2 table[4][D / 2];
  const uint32_t bid = tda::grid_bid<256>();
  const int64_t all = (int64_t)P.lead * P.seq.rows, e0 = (int64_t)(bid / (uint32_t)splits) * tok;
  if (e0 >= all) return;
  const int nt = (int)min((int64_t)tok, all - e0), l = lane_id(), wv = threadIdx.x >> 6;
  if (wv < nt) {
    Token k;
    k.b = (int)((e0 + wv) / P.seq.rows);
    k.i = (int)((e0 + wv) % P.seq.rows);
    int s = k.b;
    if (P.seq.starts) {  // the sequences that end before the row, counted
      s = 0;
      for (int s0 = 1; s0 <= P.seq.S; s0 += 64)
        s += __popcll(__ballot(s0 + l <= P.seq.S && P.seq.starts[min(s0 + l, P.seq.S)] <= k.i));
    }
    k.own = 0;
    k.page = -1;
    int at = 0;
    if (s < P.seq.S) {
      const Seq q = seq_of(P.seq, s);
      k.own = k.i >= q.row0 && k.i < q.row0 + q.cnt;
      at = q.held + k.i - q.row0;
      if (k.own && at >= 0 && at < P.seq.tlen << P.seq.pshift) {
        const int p = P.seq.table[(int64_t)s * P.seq.tstride + (at >> P.seq.pshift)];
        k.page = p >= 0 && p < P.seq.pages ? p : -1;
      }
      k.row = at & ((1 << P.seq.pshift) - 1);
    }
    if (l < P.pairs) {
      int a = 0;
      while (l >= P.upto[a]) ++a;  // ends: the last section reaches every pair
      double pos = at;
      if (P.pos) {
        const int64_t j = a * P.ps[0] + k.b * P.ps[1] + k.i * P.ps[2];
        pos = P.pos64 ? (double)static_cast<const int64_t*>(P.pos)[j] : (double)static_cast<const int32_t*>(P.pos)[j];
      }
      const double turns = pos * (double)P.inv_freq[l] * 0.15915494309189533577;
      float sn, cs;
      sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
      table[wv][l] = make_float2(cs, sn);
    }
    if (l == 0) token[wv] = k;
  }
  __syncthreads();
  typedef T vec __attribute__((ext_vector_type(V)));
  const int per = 2 * P.H + (2 + VH) * P.Hk, u = threadIdx.x % U;
  int t = 0, r = (int)(bid % (uint32_t)splits) * ROWS + (int)threadIdx.x / U;
  for (;; r += ROWS * splits) {
    while (r >= per) r -= per, ++t;
    if (t >= nt) break;
    const Token k = token[t];
    const T* x;
    T* y;
    bool turn = u < P.pairs / V, put = true;
    if (r < 2 * P.H) {
      const int z = r >= P.H, h = r - z * P.H;
      x = sda::row_of<const T>(P.q[z], k.b, h, k.i);
      y = sda::row_of<T>(P.qo[z], k.b, h, k.i);
    } else {
      const int e = r - 2 * P.H, z = e < P.Hk ? 0 : e < 2 * P.Hk ? 1 : 2, f = e - z * P.Hk, h = z == 2 ? f / VH : f;
      const int64_t row = ((((int64_t)max(k.page, 0) * P.Hk + h) << P.seq.pshift) + k.row);
      x = sda::row_of<const T>(P.x[z], k.b, h, k.i) + (z == 2 ? f % VH * D : 0);
      y = static_cast<T*>(P.pool[z]) + (z == 2 ? row * DV + f % VH * D : row * D);
      turn = turn && z < 2;
      put = k.page >= 0;
    }
    if (!put) continue;
    const bool apart = turn && !P.inter;  // the pair's values stand pairs apart
    const int i0 = apart ? V * u : 2 * V * u;
    const int i1 = apart ? P.pairs + V * u : i0 + V;
    vec a = {}, c = {};
    if (k.own) {
      a = *reinterpret_cast<const vec*>(x + i0);
      c = *reinterpret_cast<const vec*>(x + i1);
    }
    if (turn) {
      const float2* cs = table[t] + V * u;
      float p[V], q[V];  // first and second values of the unit's pairs
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = 2 * j;
        p[j] = P.inter && V > 1 ? (float)(e < V ? a[e % V] : c[e % V]) : (float)a[j];
        q[j] = P.inter && V > 1 ? (float)(e < V ? a[(e + 1) % V] : c[(e + 1) % V]) : (float)c[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 w = cs[j];
        const T f = (T)__builtin_fmaf(p[j], w.x, -(q[j] * w.y)), g = (T)__builtin_fmaf(q[j], w.x, p[j] * w.y);
        if (P.inter && V > 1) {
          if (2 * j < V) a[2 * j % V] = f, a[(2 * j + 1) % V] = g;
          else c[2 * j % V] = f, c[(2 * j + 1) % V] = g;
        } else {
          a[j] = f;
          c[j] = g;
        }
      }
    }
    *reinterpret_cast<vec*>(y + i0) = a;
    *reinterpret_cast<vec*>(y + i1) = c;
  }
}

template <class T, int V, int D, int DV>
static int launch(const AppendParams& p, hipStream_t st) {
  const int64_t all = (int64_t)p.lead * p.seq.rows;
  const int tok = all >= 4096 ? 4 : 1;
  constexpr int ROWS = 256 * 2 * V / D;
  const int per = 2 * p.H + (2 + DV / D) * p.Hk;
  int splits = 1;  // workgroups that share a token's rows: about 1024 in all
  while (tok == 1 && 2 * splits * ROWS < 2 * per && all * splits < 1024) splits *= 2;
  append<T, V, D, DV><<<tda::grid_of<256>((all + tok - 1) / tok * splits), 256, 0, st>>>(p, tok, splits);
  tda::launched(st, "spa_append");
  return (int)hipGetLastError();
}
template <class T, int V>
static int pick(const AppendParams& p, hipStream_t st) {
  if (p.D == 64) return p.DV == 64 ? launch<T, V, 64, 64>(p, st) : launch<T, V, 64, 128>(p, st);
  return p.DV == 128 ? launch<T, V, 128, 128>(p, st) : launch<T, V, 128, 256>(p, st);
}
template <class T>
static int run(const AppendParams& p, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  return p.pairs % V == 0 ? pick<T, V>(p, st) : pick<T, 1>(p, st);
}
int launch_append(const AppendParams& p, int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? run<float>(p, st) : dtype == 1 ? run<tda::bf16>(p, st) : run<_Float16>(p, st);
}

}  // namespace spa
