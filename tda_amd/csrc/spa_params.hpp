// spa_params.hpp -- kernel argument blocks of the paged cache, passed by value from the host entry points
// (spa_host.cpp), and the launchers each kernel file exports.
#pragma once

#include "sda_params.hpp"

namespace spa {

using sda::Lambda;
using sda::Rows;

struct Seqs {            // whose rows a call has (spa_rows of include/spa.h)
  const int32_t *table, *lengths, *starts, *counts;  // starts, counts: may be null
  int64_t tstride;
  int tlen, S, rows, pshift, pages;                  // pshift: log2 of the page size
};

struct AppendParams {
  Seqs seq;
  void* pool[3];
  Rows x[3];             // k1, k2, v
  Rows q[2], qo[2];
  int Hk, H, D, DV, lead;
  int pairs, inter, axes;
  int upto[4];           // first pair past each axis' section
  const void* pos;       // may be null
  int64_t ps[3];
  int pos64;
  const float* inv_freq;
};

// The attention takes sequences of at most `bound` rows (a row: a query row of one of the heads that share a key head)
// in tiles of 16 rows, the others in tiles of 128.
constexpr int kFewRows = 16, kManyRows = 128;
struct AttendParams {
  Seqs seq;
  const void* k[2];
  const void* v;
  Rows q[2], out;
  Lambda lam;
  int H, Hk, lead, bound;
  float c;               // scale * log2(e)
  int cost;              // what 128 keys of a large tile cost next to those of a small one
  int room;              // workgroups that may share a key head's tiles; 0: whole tiles only
  uint32_t grid;         // workgroups of all key heads, at most
  uint32_t join[2];      // what the joining launch may have to join: small tiles; groups of 32 rows of large ones
  int join_rows;         // rows of a small tile, at most
  float* part;           // two places for each of room workgroups of every key head, `stride` floats each
  int64_t stride;
};

// The sums of a part of a tile.  Few rows: [branch][m, l][16], then [branch][row][dv].  Many: [branch][m, l][128], then
// [branch][32 rows][4 of a lane's values][lane][4].
constexpr int64_t few_floats(int64_t dv) { return 64 + 2 * kFewRows * dv; }
constexpr int64_t many_floats(int64_t dv) { return 4 * kManyRows + 2 * kManyRows * dv; }

int launch_append(const AppendParams& p, int dtype, void* stream);
int launch_attend(const AttendParams& p, int dtype, int d, int dv, void* stream);
// one type to a file, so that they compile side by side
int launch_attend_f32(const AttendParams& p, int d, int dv, void* stream);
int launch_attend_bf16(const AttendParams& p, int d, int dv, void* stream);
int launch_attend_f16(const AttendParams& p, int d, int dv, void* stream);

}  // namespace spa
