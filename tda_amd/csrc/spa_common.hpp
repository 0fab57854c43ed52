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

// The lane's number as something new: what a loop's passes make of it is not kept in registers from one to the next.
__device__ __forceinline__ int fresh_lane() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}

// Zero, likewise.
__device__ __forceinline__ float fresh_zero() {
  float z = 0.f;
  asm volatile("" : "+v"(z));
  return z;
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
    // The compiler loads under the first condition and waits for the load there.  Checked in page() instead, every stage would wait for
    // all loads on their way (a chunk among tokens 103 -> 113 us).
    const int p = row[min(e, tlen - 1)];
    return e < tlen && p < pages ? p : -1;
  }
  __device__ __forceinline__ void begin(const Seqs& Q, int s, int slot) {
    row = Q.table + (int64_t)uniform(s) * Q.tstride;
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
constexpr int kUnit = 128;  // keys
// Tiles of 16 rows are cut until there are this many for each workgroup: whole tiles that workgroups take as they come save the joining
// and the second tile's start (newest tokens of 128 sequences of up to 1500, (32 over 8 heads, 128): 171 us, cut 186; of 64 of
// up to 2000: 114, cut 119), while a tile a workgroup leaves the last ones alone (32 of up to 8192: 231, cut 223).
constexpr int kFewCut = 2;
constexpr int kManyCut = 3;

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

// A part of a tile of rows of one sequence (the rows of all heads that share a key head, token by token): units from ..
// from + count - 1 of the tile's `units`.
struct Job {
  int s, tile;
  uint32_t at, from, count, units;  // at: the tile's place on its form's line
  uint32_t per, parts;              // where the tile begins with a stretch: its length, and how many the tile has; else 0
  Seq seq;
};

// How the work of a key head is dealt out.  Sequences of at most `bound` rows have tiles of 16 (form 0), the others of
// 128 (form 1).  The tiles of a form stand on a line, in the order of the sequences, a sequence's last tile first (it has the
// most keys), each as long as its keys in units of 128.  Workgroups take equal stretches of the line: a stretch may
// end in one tile and begin in another, and what it has of either goes to a place of its own, to be joined.  Where stretches
// at most an eighth longer do for every tile to begin with one, tiles are taken to fill their stretches, and shared out evenly among
// them: a workgroup then begins one tile, not two (chunks of 2 x 500 rows behind 3855: 87 -> 84 us).  Two forms share the
// workgroups by their units' costs, `cost` to 1.
// Where the tiles are enough to fill the chip each is one unit, and one workgroup's.
// Everything is whole numbers, so that every workgroup of both launches finds the same.
struct Deal {
  const Seqs& Q;
  int G, bound, l;
  bool cut;
  uint32_t groups[2], per[2], line[2];  // workgroups of a form, units of each, units in all
  bool own[2];                          // each tile begins with a stretch
  uint32_t t, u;                        // this lane's sequence: tiles, units of each
  int form;
  Seq q;

  __device__ __forceinline__ void sizes(int s0) {
    t = u = 0;
    form = 0;
    if (s0 + l < Q.S) {
      q = seq_of(Q, s0 + l);
      const int R = q.cnt * G;
      form = R > bound;
      t = (uint32_t)(R + (form ? kManyRows : kFewRows) - 1) / (form ? kManyRows : kFewRows);
      u = max((uint32_t)(q.len + kUnit - 1) / kUnit, 1u);
    }
  }
  __device__ __forceinline__ static uint32_t fill(uint32_t units, uint32_t per) { return (units + per - 1) / per; }
  __device__ __forceinline__ Deal(const Seqs& Q_, int G_, int bound_, int room, int cost) : Q(Q_), G(G_), bound(bound_), l(lane_id()) {
    // Sums that matter while they are small are held small: a lane's units end at 2^24 (that many keys in fewer tiles than are
    // cut would be 2^31), its stretches at 1023, of two lengths in one number.
    constexpr uint32_t kUnits = 1 << 24, kParts = 1023;
    q = Seq{};
    uint32_t n[2] = {0, 0}, w[2] = {0, 0};
    bool early = false;  // large tiles whose keys are far fewer than their sequence's last one's
    for (int s0 = 0; s0 < Q.S; s0 += 64) {
      sizes(s0);
      const uint32_t x = (uint32_t)min((uint64_t)t * u, (uint64_t)kUnits);
      early |= form && 3 * (int64_t)q.cnt > q.len;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        n[f] += form == f ? t : 0;
        w[f] = min(w[f] + (form == f ? x : 0), kUnits);
      }
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      groups[f] = line[f] = wave_total(n[f]);
      per[f] = 1;
      own[f] = false;
    }
    const uint32_t tiles = line[0] + line[1];
    cut = room && tiles < (uint32_t)(line[1] ? room : kFewCut * room);
    // Two or three rounds of large tiles are cut too where a quarter of the rounds' places would be idle: stretches are then a tile or more and a
    // part (1200 rows behind 3000, 32 over 8 heads of 128: 184 us, whole 203; 2100 behind 8000: 697, 801).  Not among small tiles, nor where
    // tiles have unlike keys: workgroups take these as they come, the longest first (1600 behind 2000: 171, cut 201).
    if (room && !line[0] && !cut && tiles < (uint32_t)(kManyCut * room)) {
      const uint32_t rounds = 1 + (tiles > (uint32_t)room) + (tiles > (uint32_t)(2 * room));
      cut = 4 * tiles < 3 * rounds * (uint32_t)room && !__any(early);
    }
    cut = cut && !__any(w[0] >= kUnits || w[1] >= kUnits);
    if (!cut) return;
    uint32_t all[2] = {0, 0}, to[2] = {(uint32_t)room, (uint32_t)room}, longer[2] = {1, 1};
#pragma unroll
    for (int f = 0; f < 2; ++f)
      if (line[f]) all[f] = wave_total(w[f]);
    if (line[0] && line[1]) {
      const uint64_t a = all[0], b = all[1] * (uint64_t)cost;
      const int shift = max(44 - (int)__builtin_clzll(a + b + 1), 0);  // the sum in 20 bits
      const uint32_t x = (uint32_t)(a >> shift), y = (uint32_t)(b >> shift);
      to[1] = min(max(((uint32_t)room * y + (x + y) / 2) / max(x + y, 1u), 1u), (uint32_t)room - 1);
      to[0] = (uint32_t)room - to[1];
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
      if (line[f]) {
        per[f] = max((all[f] + to[f] - 1) / to[f], 1u);
        longer[f] = per[f] + (per[f] + 7) / 8;
      }
    uint32_t m[2] = {0, 0};  // stretches that tiles of their own take, of either length
    for (int s0 = 0; s0 < Q.S; s0 += 64) {
      if (Q.S > 64) sizes(s0);
      const uint32_t a = min(t * fill(u, form ? per[1] : per[0]), kParts), b = min(t * fill(u, form ? longer[1] : longer[0]), kParts);
#pragma unroll
      for (int f = 0; f < 2; ++f)
        if (form == f) m[f] = min((m[f] & 0xffff) + a, kParts) | min((m[f] >> 16) + b, kParts) << 16;
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
      if (line[f]) {
        const uint32_t both = wave_total(m[f]), a = both & 0xffff, b = both >> 16;
        own[f] = min(a, b) <= to[f];
        if (own[f]) {
          if (a > to[f]) per[f] = longer[f];
          groups[f] = a > to[f] ? b : a;
          line[f] = groups[f] * per[f];
        } else {
          line[f] = all[f];
          groups[f] = (all[f] + per[f] - 1) / per[f];
        }
      }
  }
  // What stands at unit `at` of a form's line, or with TILE the tile number `at`; up to `end` or the tile's end.  False:
  // nothing.
  template <int FORM, bool TILE>
  __device__ __forceinline__ bool find(uint32_t at, uint32_t end, Job& J) const {
    Deal d = *this;
    return d.look<FORM, TILE>(at, end, J);
  }
  template <int FORM, bool TILE>
  __device__ __forceinline__ bool look(uint32_t at, uint32_t end, Job& J) {
    uint32_t tiles = 0, units = 0;  // of the sequences before
    for (int s0 = 0; s0 < Q.S; s0 += 64) {
      if (Q.S > 64) sizes(s0);
      uint32_t each = cut ? u : 1u, parts = 0;
      if (own[FORM]) {
        parts = fill(u, per[FORM]);
        each = parts * per[FORM];
      }
      const uint32_t n = form == FORM ? t : 0, w = n * each;
      const uint32_t nu = running(n), wu = running(w);
      const auto lane = [&](uint32_t v, int x) { return (uint32_t)__builtin_amdgcn_readlane((int)v, x); };
      const uint32_t sum = lane(TILE ? nu : wu, 63), rest = at - (TILE ? tiles : units);
      if (rest < sum) {
        const int x = __builtin_ctzll(__ballot((TILE ? nu : wu) > rest));
        const uint32_t e = rest - (lane(TILE ? nu : wu, x) - lane(TILE ? n : w, x));  // within the sequence
        J.units = lane(each, x);
        const uint32_t tile = TILE ? e : e / J.units;
        J.s = s0 + x;
        J.tile = (int)(lane(n, x) - 1 - tile);
        J.at = units + lane(wu, x) - lane(w, x) + tile * J.units;
        J.from = TILE ? 0 : at - J.at;
        J.count = TILE ? J.units : min(J.units - J.from, end - at);
        J.per = own[FORM] ? per[FORM] : 0;
        J.parts = lane(parts, x);
        const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, x); };
        J.seq = {of(q.qb), of(q.row0), of(q.cnt), of(q.held), of(q.len)};
        return true;
      }
      tiles += lane(nu, 63);
      units += lane(wu, 63);
    }
    return false;
  }
  // A part's keys within the `lim` that its tile sees.
  __device__ __forceinline__ static void keys(const Job& J, int lim, int& k0, int& k1) {
    uint32_t from = J.from, to = J.from + J.count;
    if (J.per) {
      const uint32_t part = from / J.per, units = (uint32_t)(lim + kUnit - 1) / kUnit, each = units / J.parts, more = units - each * J.parts;
      from = part * each + min(part, more);
      to = from + each + (part < more);
    }
    const bool whole = J.count == J.units;
    k0 = uniform(whole ? 0 : min((int)(from * kUnit), lim));
    k1 = uniform(whole ? lim : min((int)(to * kUnit), lim));
  }
};

// Zeros the rows of no sequence, each workgroup some.
template <class T, int DV, int THREADS>
__device__ __forceinline__ void clear_free_rows(const AttendParams& P, uint32_t bid) {
  const uint32_t blocks = P.grid;
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
