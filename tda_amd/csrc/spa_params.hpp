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

// One of the two forms of the attention: `few` takes the sequences of at most `bound` rows (a row: a query
// row of one of the heads that share a key head), `many` the others.
struct Form {
  uint32_t grid;         // workgroups; 0: not launched
  uint32_t join;         // workgroups of its joining launch; 0: none
  int room;              // pieces a key head may be cut into; 0: whole tiles only
  float* part;           // grid pieces' sums, when room is not 0
};
struct AttendParams {
  Seqs seq;
  const void* k[2];
  const void* v;
  Rows q[2], out;
  Lambda lam;
  int H, Hk, lead, bound;
  float c;               // scale * log2(e)
  Form few, many;
};

constexpr int kFewRows = 16, kManyRows = 128;  // rows of a tile of each form
constexpr int64_t few_floats(int dv) { return 64 + 2 * kFewRows * (int64_t)dv; }     // a piece's sums
constexpr int64_t many_floats(int dv) { return 4 * kManyRows + 2 * kManyRows * (int64_t)dv; }

int launch_append(const AppendParams& p, int dtype, void* stream);
int launch_attend(const AttendParams& p, int dtype, int d, int dv, void* stream);
// the two forms, one to a file so that they compile side by side
int launch_few(const AttendParams& p, int dtype, int d, int dv, void* stream);
int launch_many(const AttendParams& p, int dtype, int d, int dv, void* stream);

}  // namespace spa
