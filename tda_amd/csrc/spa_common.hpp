// spa_common.hpp -- device building blocks of the paged cache: the sequences of a call, the pages of a
// sequence, and how the attention's work is dealt out.
//
// How many rows and keys each sequence has stands in device memory, so no launch knows its work: every
// workgroup reads the sequences' lengths (a wave 64 of them at a time) and finds what falls to its number.
#pragma once

#include "sda_common.hpp"
#include "spa_params.hpp"

namespace spa {

using sda::lane_id;
using sda::rsrc_of;

// A value that every lane has, in a scalar register: descriptors are made of such, and one that the compiler cannot see
// to be the same everywhere, or works out in vector registers (a quotient, a comparison of 64 bits), costs a loop.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return (uint32_t)uniform((int)(uint32_t)x) | ((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

struct Seq {
  int qb, row0, cnt;  // its rows: row0 .. row0 + cnt - 1 of batch entry qb
  int held, len;      // the position of its first row; the positions that it has with its new rows
};
__device__ __forceinline__ Seq seq_of(const Seqs& Q, int s) {
  Seq r;
  if (Q.starts) {
    r.qb = 0;
    r.row0 = min(max(Q.starts[s], 0), Q.rows);
    r.cnt = min(max(Q.starts[s + 1], r.row0), Q.rows) - r.row0;
  } else {
    r.qb = s;
    r.row0 = 0;
    r.cnt = Q.counts ? min(max(Q.counts[s], 0), Q.rows) : Q.rows;
  }
  r.held = min(max(Q.lengths[s], -(1 << 30)), 1 << 30);
  r.len = min(max(r.held + r.cnt, 0), Q.tlen << Q.pshift);
  return r;
}

// The page numbers of 64 consecutive table entries in the lanes of a register, the next 64 on their way:
// page() then costs a few scalar instructions.  Entries behind the table, and numbers that are no page,
// are -1.
struct Pages {
  const int32_t* row;
  int tlen, pages, base;
  int now, next;
  __device__ __forceinline__ int fetch(int at) const {
    const int e = at + lane_id();
    const int p = e < tlen ? row[e] : -1;
    return p < pages ? p : -1;
  }
  __device__ __forceinline__ void begin(const Seqs& Q, int s, int slot) {
    row = Q.table + (int64_t)s * Q.tstride;
    tlen = Q.tlen;
    pages = Q.pages;
    base = slot;
    now = fetch(slot);
    next = fetch(slot + 64);
  }
  // Makes page() know the entries up to `last`, of which the earlier ones asked for so far stay known when they
  // are at most 64 apart.  Slots only grow.
  __device__ __forceinline__ void reach(int first) {
    if (first >= base + 64) {
      base += 64;
      if (first >= base + 64) {  // a jump past what is on its way
        base = first;
        now = fetch(base);
      } else {
        now = next;
      }
      next = fetch(base + 64);
    }
  }
  __device__ __forceinline__ int page(int slot) const {
    const int e = slot - base;
    return e < 64 ? __builtin_amdgcn_readlane(now, e) : __builtin_amdgcn_readlane(next, e - 64);
  }
};
// Row of a pool (of one of its heads, counted over all pages) where position `key` of a page stands.
__device__ __forceinline__ uint64_t pool_row(int page, int Hk, int hk, int pshift, int key) {
  return ((uint64_t)(uint32_t)(max(page, 0) * Hk + hk) << pshift) + (uint32_t)(key & ((1 << pshift) - 1));
}
// How many of the n rows from position `key` on stand before `lim` (a negative number: none).
__device__ __forceinline__ int rows_before(int key, int n, int lim) {
  int rows = min(n, lim - key);
  asm("" : "+s"(rows));  // this minimum and page_rsrc's maximum in one would be a vector instruction
  return rows;
}
// Descriptor over `rows` rows (of WIDTH bytes, at most up to the page's end) from a row of the pool on; rows
// past them, and all rows of no page, read as zeros.
template <int WIDTH>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rsrc(const void* pool, uint64_t row, int page, int rows) {
  return rsrc_of(static_cast<const char*>(pool) + row * WIDTH, page >= 0 ? (uint32_t)(max(rows, 0) * WIDTH) : 0u);
}

// ------------------------------------------------------------------ work
// Running sums over the wave's lanes (lane moves: four within rows of 16 lanes, two from row to row), and their totals.
// Call with every lane active.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t x) {  // 0 where nothing comes from
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ uint32_t running(uint32_t x) {
  x += moved<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x += moved<0x112, 0xF>(x);
  x += moved<0x114, 0xF>(x);
  x += moved<0x118, 0xF>(x);
  x += moved<0x142, 0xA>(x);  // row_bcast 15 into rows 1 and 3
  x += moved<0x143, 0xC>(x);  // row_bcast 31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t wave_total(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)running(x), 63); }
__device__ __forceinline__ uint64_t wave_total(uint64_t x) {  // of values below 2^58
  const uint32_t low = wave_total((uint32_t)(x & 0x3ffffff)), mid = wave_total((uint32_t)(x >> 26) & 0x3ffffff);
  return low + ((uint64_t)mid << 26) + ((uint64_t)wave_total((uint32_t)(x >> 52)) << 52);
}

constexpr int kUnit = 128;  // keys; pieces are whole units

// A tile of RT rows of sequence s (the rows of all heads that share a key head, token by token), and which of
// the `parts` pieces of its keys; `first` is the number of its first piece (of one key head).
struct Job {
  int s, tile, part, parts, units;  // units of keys in a piece
  uint32_t first;
  Seq seq;
};
// The tiles of a form (FEW: sequences of at most `bound` rows), in the order of the sequences, a sequence's last
// tile first: it has the most keys.  With `room` each tile is cut into pieces of the fewest units that leave no more
// than `room` of them: from W / room on, W the sum over N tiles of their units, up to W / (room - N), which always do.
// BY_PIECE: idx counts pieces; else tiles (for the launch that joins them).  False: there is no such one.
template <int RT, bool FEW, bool BY_PIECE>
__device__ __forceinline__ bool find_job(const Seqs& Q, int G, int bound, int room, uint32_t idx, Job& J) {
  const int l = lane_id();
  uint32_t t = 0, u = 0;
  Seq q{};
  const auto sizes = [&](int s0) {
    t = u = 0;
    if (s0 + l < Q.S) {
      q = seq_of(Q, s0 + l);
      const int R = q.cnt * G;
      if ((R <= bound) == FEW) t = (uint32_t)(R + RT - 1) / RT;
      u = (uint32_t)(q.len + kUnit - 1) / kUnit;
    }
  };
  uint32_t units = 0x7fffffffu;
  if (room) {
    uint32_t N = 0;
    uint64_t W = 0;
    for (int s0 = 0; s0 < Q.S; s0 += 64) {
      sizes(s0);
      N += t;
      W += (uint64_t)t * u;
    }
    N = wave_total(N);
    W = wave_total(W);
    if ((uint32_t)room > N) {
      const auto share = [&](uint32_t by) {  // W / by rounded up, of W in 31 bits
        const uint32_t over = (uint32_t)(W >> 31);
        const int shift = (W >> 63) ? 33 : over ? 32 - __builtin_clz(over) : 0;
        const uint32_t w = ((uint32_t)(W >> shift) + (shift ? 1u : 0u) + by - 1) / by;
        return (uint32_t)min(max((uint64_t)w << shift, (uint64_t)1), (uint64_t)0x7fffffff);
      };
      const uint32_t most = share((uint32_t)room - N);  // at most `room` pieces for sure
      units = share((uint32_t)room);                    // the least there could be
      while (units < most) {
        uint32_t n = 0;
        for (int s0 = 0; s0 < Q.S; s0 += 64) {
          if (Q.S > 64) sizes(s0);
          n += t * max((u + units - 1) / units, 1u);
        }
        if (wave_total(n) <= (uint32_t)room) break;
        units = min(units + max(units / 8, 1u), most);
      }
    }
  }
  uint32_t tiles = 0, pieces = 0;  // of the sequences before
  for (int s0 = 0; s0 < Q.S; s0 += 64) {
    if (!room || Q.S > 64) sizes(s0);
    const uint32_t p = t * max((u + units - 1) / units, 1u);
    const uint32_t tu = running(t), pu = running(p), mine = BY_PIECE ? pu : tu, before = BY_PIECE ? pieces : tiles;
    const uint32_t sum = __builtin_amdgcn_readlane(mine, 63);
    if (idx - before < sum) {
      const int x = __builtin_ctzll(__ballot(mine > idx - before));
      const uint32_t nt = __builtin_amdgcn_readlane(t, x), np = __builtin_amdgcn_readlane(p, x);
      const uint32_t first = pieces + __builtin_amdgcn_readlane(pu, x) - np;
      const uint32_t e = idx - before - (__builtin_amdgcn_readlane(mine, x) - (BY_PIECE ? np : nt));
      J.s = s0 + x;
      J.parts = (int)(np / nt);
      const uint32_t at = BY_PIECE ? e / (uint32_t)J.parts : e;
      J.part = BY_PIECE ? (int)(e % (uint32_t)J.parts) : 0;
      J.tile = (int)(nt - 1 - at);
      J.units = (int)units;
      J.first = first + at * (uint32_t)J.parts;
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, x); };
      J.seq = {of(q.qb), of(q.row0), of(q.cnt), of(q.held), of(q.len)};
      return true;
    }
    tiles += __builtin_amdgcn_readlane(tu, 63);
    pieces += __builtin_amdgcn_readlane(pu, 63);
  }
  return false;
}
// A piece's keys within the `lim` that its tile sees.
__device__ __forceinline__ void keys_of(const Job& J, int lim, int& k0, int& k1) {
  const int64_t per = (int64_t)J.units * kUnit;
  k0 = uniform((int)min((int64_t)J.part * per, (int64_t)lim));
  k1 = uniform((int)min((int64_t)k0 + per, (int64_t)lim));
}

// Zeros the rows of no sequence: workgroup `bid` of `blocks`.
template <class T, int DV, int THREADS>
__device__ __forceinline__ void clear_free_rows(const AttendParams& P, uint32_t bid, uint32_t blocks) {
  constexpr int V = 16 / sizeof(T), PER = DV / V;
  if (!P.seq.starts && !P.seq.counts) return;
  const int64_t all = (int64_t)P.lead * P.seq.rows;
  int64_t lo = 0, hi = all;  // where they may be
  int s0 = 0, s1 = 0;        // packed: rows s0 .. s1 - 1 have a sequence
  if (P.seq.starts) {
    s0 = min(max(P.seq.starts[0], 0), P.seq.rows);
    s1 = min(max(P.seq.starts[P.seq.S], s0), P.seq.rows);
    hi = all - (s1 - s0);
  }
  for (int64_t e = lo + bid; e < hi; e += blocks) {
    int b = 0, i;
    if (P.seq.starts) {
      i = (int)(e < s0 ? e : e + (s1 - s0));
    } else {
      b = (int)(e / P.seq.rows);
      i = (int)(e % P.seq.rows);
      if (i < min(max(P.seq.counts[b], 0), P.seq.rows)) continue;
    }
    for (int x = threadIdx.x; x < P.H * PER; x += THREADS)
      *reinterpret_cast<sda::u32x4*>(sda::row_of<T>(P.out, b, x / PER, i) + x % PER * V) = sda::u32x4{};
  }
}

}  // namespace spa
