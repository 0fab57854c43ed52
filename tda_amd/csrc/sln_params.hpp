// sln_params.hpp -- kernel argument blocks of the layer norm, passed by value from the host entry points
// (sln_host.cpp), and its launchers.
#pragma once

#include "sda_params.hpp"

namespace sln {

// Rows in groups that share a weight row (one group, or one a head), within a group along three axes with the
// smallest stride last, merged where the tensors allow it.
struct Tensor {
  void* p;
  int64_t group, s[3];  // element strides
};
struct Params {
  Tensor x, y, dy, dx, stats;  // stats: pairs of floats
  const void *weight, *bias;
  void *dweight, *dbias;
  int weight_type;             // 0 f32, else as the rows
  int groups, n[3], rows;      // rows of a group: n[0] n[1] n[2]
  int width, center;
  float eps;
  float* part;                 // backward: [group][blocks][dw, db][width]
  int blocks;                  // workgroups of a group
};

int launch_fwd(const Params& p, int dtype, void* stream);
int launch_bwd(const Params& p, int dtype, void* stream);

// How a row is shared out: `lanes` threads with pieces of 16 bytes `lanes` apart, `pieces` each.
struct Split { int lanes, pieces; };
inline Split split_of(int width, int dtype) {
  const int c = (width * (dtype == 0 ? 4 : 2) + 15) / 16;
  for (int l = 8; l <= 64; l *= 2)
    if (c <= l) return {l, 1};
  for (int l = 64; l <= 256; l *= 4)
    for (int k = 2; k <= 4; k *= 2)
      if (c <= l * k) return {l, k};
  return {1024, c <= 2048 ? 2 : 4};
}
constexpr int bwd_threads(int lanes) { return lanes == 1024 ? 1024 : 512; }
// Workgroups of a group of rows in the backward: each leaves a row of sums, so no more than fill the chip.
inline int bwd_blocks(int width, int dtype, int groups, int rows) {
  const Split s = split_of(width, dtype);
  const int at_once = bwd_threads(s.lanes) / s.lanes, chip = s.pieces == 1 ? 1024 : s.lanes == 1024 ? 256 : 512;
  const int most = (rows + at_once - 1) / at_once, want = (chip + groups - 1) / groups;
  if (most <= 8) return 1;  // a workgroup's few rounds cost less than the second launch
  return most < want ? most : want;
}

}  // namespace sln
