// sda_params.hpp -- kernel argument blocks of the softmax differential attention operators, passed by
// value from the host entry points (sda_host.cpp), and the launchers each kernel file exports.
#pragma once

#include <stdint.h>

namespace sda {

struct Rows {     // a (B, H, N, width) tensor: element strides of the batch, head and sequence axes
  void* p;
  int64_t sb, sh, st;
};

struct Lambda {   // element (b, h, i)
  const void* p;
  int64_t sb, sh, si;
  int type;       // 0 f32, 1 bf16, 2 f16
};

// Who sees what: row i of sequence b stands at off(b) + i and sees key j when j < len(b) and
// (causal) j <= off(b) + i.
struct Sight {
  int causal, qoff;
  const int32_t* qoffs;  // may be null
  const int32_t* lens;   // may be null
};

struct FwdParams {
  Rows q[2], k[2], v, out, out2, low;  // out2.p (f32) may be null; low: with it, not for f32
  Lambda lam;
  Sight see;
  int B, H, Hk, Nq, Nk, nqt;      // nqt: query tiles (set by launch_fwd)
  float c;                        // scale * log2(e)
  float* lse;                     // may be null
  // decode kernels: the keys cut into nsplit parts of `chunk` keys; per (row, part) the partial sums
  float* part;
  int nsplit, chunk;
};

struct BwdParams {
  Rows q[2], k[2], v, out, out2, low, dout, dq[2], dk[2], dv;
  Lambda lam;
  Sight see;
  int B, H, Hk, Nq, Nk;
  float c, scale;
  const float* lse;  // [2][B*H*Nq]
  float* stat;       // [6][B*H*Nq]: what the passes need of a row (bwd_rows), and r_2 (bwd_query)
  float* peak;       // f16: [3], what its range has to hold (bwd_rows, bwd_peak); else null
  float* part;       // may be null: dk1, dk2, dv of each group of gs query heads, f32
  int gs;            // query heads a workgroup of the key pass sums over
  void* dlam;        // may be null
  int64_t dlam_n[3]; // extents of the distinct elements (1 along a broadcast axis)
};

struct RotaryParams {
  Rows x[4], y[4];
  int heads[4];
  int count, B, N, D, pairs, inter, axes;
  int upto[4];                     // first pair past each axis' section
  const void* pos;
  int64_t ps[3];
  int pos64;
  const float* inv_freq;
  float sign;
};

struct Kv4Params {
  // cache
  uint8_t* codes[3];
  uint32_t* pars[3];               // (m, s) bf16 pairs: s in the high half
  int32_t* lengths;
  int B, Hk, cap, D, DV;
  int64_t cap4;                    // rows of a head: cap rounded up to four
  // append / read
  Rows x[3];
  int rows;
  const int32_t* start;
  const int32_t* counts;
  // attend
  Rows q[2], out;
  Lambda lam;
  int H, Nq;
  float c;
  float* part;
  int nsplit, chunk;
};

// launchers return a hipError_t value; dtype 0 f32, 1 bf16, 2 f16
int launch_fwd(const FwdParams& p, int dtype, int d, int dv, void* stream);
int launch_decode(const FwdParams& p, int dtype, int d, int dv, void* stream);
int launch_bwd(const BwdParams& p, int dtype, int d, int dv, void* stream);
int launch_rotary(const RotaryParams& p, int dtype, void* stream);
int launch_kv4_append(const Kv4Params& p, int dtype, void* stream);
int launch_kv4_read(const Kv4Params& p, int dtype, void* stream);
int launch_kv4_attend(const Kv4Params& p, int dtype, void* stream);

}  // namespace sda

namespace tda {  // tda_host.cpp, tda_timing.cpp
void record_hip_error(int e);
void timing_begin(void* stream);
void launched(void* stream, const char* name);
int timing_end();
}  // namespace tda
