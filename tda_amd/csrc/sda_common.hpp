// sda_common.hpp -- device building blocks of the softmax differential attention kernels.
//
// Matrix-core layouts are those of tda_common.hpp.  A fragment here is always 8 contraction
// elements per lane (16 per 32x32 product, 32 per 16x16 product); fp32 computes it as 8 steps of one
// element, so that both types share every index below.
#pragma once

#include <type_traits>
#include <utility>

#include "sda_params.hpp"
#include "tda_common.hpp"

namespace sda {

using tda::bf16;
using tda::bf16x2;
using tda::bf16x4;
using tda::bf16x8;
using tda::crow;
using tda::f32x16;
using tda::f32x4;
using tda::lane_id;
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Running maxima start here instead of at -inf: a masked score (-inf) then weighs exp2(-inf) = 0
// before the first visible one too.
constexpr float kNoMax = -1e37f;
// A running maximum moves only when a new score passes it by this much (log2): the sums then hold
// weights up to 2^8 instead of 1, which costs 32-bit sums nothing and saves rescaling them.
constexpr float kSlack = 8.0f;

// f(0), .., f(N - 1) with constant arguments: an unrolled loop of any length.
template <class F, int... I>
__device__ __forceinline__ void times_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void times(F&& f) {
  times_(f, std::make_integer_sequence<int, N>());
}

struct TrB {
  using T = bf16;
  using frag = bf16x8;
  __device__ __forceinline__ static f32x16 mma32(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 mma16(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct TrH {
  using T = _Float16;
  using frag = f16x8;
  __device__ __forceinline__ static f32x16 mma32(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 mma16(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
struct TrF {
  using T = float;
  using frag = f32x8;
  __device__ __forceinline__ static f32x16 mma32(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 mma16(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Values 8 s .. 8 s + 7 of a score tile as the B operand of the next product (round to nearest
// even; bf16 holds a weight to 2^-9, as it would hold the output, f16 one of a running maximum's part to 2^-12,
// and to 2^-25 of the maximum's below 2^-14).
template <class Tr>
__device__ __forceinline__ typename Tr::frag pack8(const f32x16& c, int s) {
  typename Tr::frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (typename Tr::T)c[8 * s + j];
  return f;
}

template <class T>
__device__ __forceinline__ T* row_of(const Rows& r, int b, int h, int64_t i) {
  return static_cast<T*>(r.p) + (int64_t)b * r.sb + (int64_t)h * r.sh + i * r.st;
}
__device__ __forceinline__ float lambda_of(const Lambda& l, int b, int h, int i) {
  const int64_t at = (int64_t)b * l.sb + (int64_t)h * l.sh + (int64_t)i * l.si;
  return l.type == 0   ? static_cast<const float*>(l.p)[at]
         : l.type == 1 ? (float)static_cast<const bf16*>(l.p)[at]
                       : (float)static_cast<const _Float16*>(l.p)[at];
}
__device__ __forceinline__ int len_of(const Sight& s, int b, int Nk) {
  return s.lens ? min(max(s.lens[b], 0), Nk) : Nk;
}
__device__ __forceinline__ int off_of(const Sight& s, int b) {
  // a position beyond +-2^30 sees all or nothing already
  return s.qoffs ? min(max(s.qoffs[b], -(1 << 30)), 1 << 30) : s.qoff;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
// Descriptor over `rows` rows of `width` bytes, `stride` bytes apart: rows past them read as zeros, or, where rows
// overlap (stride < width, 0 for a broadcast one), as bytes of the rows before: then they need weights of zero.
// rows * stride stays below 2^32 (tiles of up to 64 rows, strides of at most 2^25 bytes).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int64_t stride, int rows, int width) {
  return rsrc_of(base, rows > 0 ? (uint32_t)((int64_t)(rows - 1) * stride + width) : 0u);
}
template <int N>
__device__ __forceinline__ void wait_vm() {  // vmcnt(N) with the other counters left alone
  static_assert(N >= 0 && N < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}

// ------------------------------------------------------------------ tiles in LDS
// ROWS x W values, row-major, filled by direct buffer -> LDS loads of 16 bytes a lane: the load of
// instruction u puts chunk 64 u + lane of the tile in place, so the bank swizzle is applied to the
// source address: place (row, chunk) holds the row's chunk (chunk ^ swz(row)).
template <class Tr, int ROWS, int W>
struct Tile {
  using T = typename Tr::T;
  static constexpr int ES = sizeof(T);
  static constexpr int CPR = W * ES / 16;          // 16-byte chunks of a row
  static constexpr int BYTES = ROWS * W * ES;
  static constexpr int LOADS = BYTES / 1024;       // load instructions (64 lanes x 16 bytes)
  static constexpr int PER = 16 / ES;              // values of a chunk

  __device__ __forceinline__ static int swz(int r) {
    if constexpr (ES == 2) return tda::bswz<W>(r);
    else return r & 15;
  }
  // Byte offset (from the tile's first row in memory) that this lane loads in instruction u.
  __device__ __forceinline__ static uint32_t source(int u, uint32_t stride) {
    const int ci = 64 * u + lane_id(), r = ci / CPR, c = ci % CPR;
    return (uint32_t)r * stride + 16u * (uint32_t)(c ^ swz(r));
  }
  __device__ __forceinline__ static void load(__amdgpu_buffer_rsrc_t r, T* lds, int u, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, LDS_PTR(void, reinterpret_cast<char*>(lds) + 1024 * u), 16, off, 0, 0, 0);
  }
  // Row fragment step t: lane (m, g) gets row r0 + m, values 16 t + 8 g + [0, 8).
  __device__ __forceinline__ static typename Tr::frag row(const T* lds, int r0, int t) {
    const int l = lane_id(), r = r0 + (l & 31), g = l >> 5;
    static_assert(ES == 4, "16-bit types: RowReader");
    const int c = 4 * t + 2 * g;
    const f32x4 a = *reinterpret_cast<const f32x4*>(lds + r * W + 4 * (c ^ swz(r)));
    const f32x4 b = *reinterpret_cast<const f32x4*>(lds + r * W + 4 * ((c + 1) ^ swz(r)));
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  // Transposed fragment, step s (16 rows from r0 + 16 s): lane (n, g) gets column 32 cs + n at rows
  // r0 + crow(8 s + j, g), j = 0 .. 7, which is the order of a score tile's values.
  __device__ __forceinline__ static typename Tr::frag col(const T* lds, int r0, int s, int cs) {
    static_assert(ES == 4, "16-bit types: ColReader");
    const int l = lane_id(), g = l >> 5, n = 32 * cs + (l & 31);
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = r0 + crow(8 * s + j, g);
      f[j] = lds[r * W + 4 * ((n >> 2) ^ swz(r)) + (n & 3)];
    }
    return f;
  }
};

// The same fragments by way of LDS addresses that a lane keeps (16-bit types): the swizzle makes the address of each
// step another one, which the compiler would work out again for every read (a third of a pass' vector
// instructions).  `at` of a read is a constant offset: the tile's place, and rows 32 apart.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
template <class Tr, int W>
struct RowReader {
  static constexpr int NT = W / 16;
  uint32_t a[NT];
  __device__ __forceinline__ void init(const void* lds) {
    const int r = lane_id() & 31, g = lane_id() >> 5;
    const uint32_t base = lds_address(lds);
    if constexpr (sizeof(typename Tr::T) == 2) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        a[t] = base + r * W * 2 + 16 * ((2 * t + g) ^ Tile<Tr, 32, W>::swz(r));
        asm volatile("" : "+v"(a[t]));
      }
    }
  }
  __device__ __forceinline__ typename Tr::frag read(const void* lds, int at, int t) const {
    if constexpr (sizeof(typename Tr::T) == 2)
      return *reinterpret_cast<const __attribute__((address_space(3))) typename Tr::frag*>(a[t] + at);
    else
      return Tile<Tr, 32, W>::row(reinterpret_cast<const float*>(static_cast<const char*>(lds) + at), 0, t);
  }
};
template <class Tr, int W>
struct ColReader {
  static constexpr int NY = W / 32;
  uint32_t a[2][NY];
  __device__ __forceinline__ void init(const void* lds) {
    const int l = lane_id(), bk = l >> 4, j = l & 15;
    const uint32_t base = lds_address(lds);
    if constexpr (sizeof(typename Tr::T) == 2) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int y = 0; y < NY; ++y) {
          const int r = 8 * hh + 4 * (bk >> 1) + (j >> 2), d = 32 * y + 16 * (bk & 1) + 4 * (j & 3);
          a[hh][y] = base + r * W * 2 + 16 * ((d >> 3) ^ Tile<Tr, 32, W>::swz(r)) + 2 * (d & 7);
          asm volatile("" : "+v"(a[hh][y]));
        }
    }
  }
  // Step s (16 rows) of the tile at `at`, column block y.
  __device__ __forceinline__ typename Tr::frag read(const void* lds, int at, int s, int y) const {
    if constexpr (sizeof(typename Tr::T) == 2) {
      typedef __attribute__((address_space(3))) tda::s16x4 quad;
      typedef typename Tr::T half4 __attribute__((ext_vector_type(4)));
      typename Tr::frag f;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const half4 w = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<quad*>(a[hh][y] + at + 32 * W * s)));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * hh + e] = w[e];
      }
      return f;
    } else {
      return Tile<Tr, 32, W>::col(reinterpret_cast<const float*>(static_cast<const char*>(lds) + at), 0, s, y);
    }
  }
};

// Row fragments of one row in memory (null: zeros), lane half g.
template <class Tr, int NT>
__device__ __forceinline__ void load_frags(const typename Tr::T* row, int g, typename Tr::frag (&f)[NT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (row) {
      if constexpr (sizeof(typename Tr::T) == 2) {
        f[t] = *reinterpret_cast<const typename Tr::frag*>(row + 16 * t + 8 * g);
      } else {
        const f32x4 a = *reinterpret_cast<const f32x4*>(row + 16 * t + 8 * g);
        const f32x4 b = *reinterpret_cast<const f32x4*>(row + 16 * t + 8 * g + 4);
        f[t] = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      }
    } else {
      f[t] = typename Tr::frag{};
    }
  }
}

// acc += a(t) b(t) over NT steps, the operands a read from LDS a group of four steps ahead of their use
// and no further (see tda::mma_chain): left to itself the compiler waits for every read by itself.
template <class Tr, int NT, class FA>
__device__ __forceinline__ f32x16 chain(FA&& a, const typename Tr::frag (&b)[NT]) {
  constexpr int G = sizeof(typename Tr::T) == 2 ? 4 : 1;  // an fp32 step is eight products itself
  static_assert(NT % G == 0, "whole groups");
  typename Tr::frag f[2][G];
  f32x16 acc = {};
#pragma unroll
  for (int t0 = -G; t0 < NT; t0 += G) {
    if (t0 + G < NT) {
#pragma unroll
      for (int u = 0; u < G; ++u) f[(t0 / G + 1) & 1][u] = a(t0 + G + u);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 >= 0) {
#pragma unroll
      for (int u = 0; u < G; ++u) acc = Tr::mma32(f[(t0 / G) & 1][u], b[t0 + u], acc);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return acc;
}
// acc[y] += col(u, y) b[u] for a transposed tile of 32 rows and NY blocks of 32 columns, the operands read
// four ahead in the same way.
template <class Tr, int NY, class FA>
__device__ __forceinline__ void columns(FA&& col, const typename Tr::frag (&b)[2], f32x16 (&acc)[NY]) {
  constexpr int G = sizeof(typename Tr::T) == 2 ? 4 : 1, N = 2 * NY;
  typename Tr::frag f[2][G];
#pragma unroll
  for (int t0 = -G; t0 < N; t0 += G) {
    if (t0 + G < N) {
#pragma unroll
      for (int u = 0; u < G; ++u) f[(t0 / G + 1) & 1][u] = col((t0 + G + u) / NY, (t0 + G + u) % NY);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 >= 0) {
#pragma unroll
      for (int u = 0; u < G; ++u) acc[(t0 + u) % NY] = Tr::mma32(f[(t0 / G) & 1][u], b[(t0 + u) / NY], acc[(t0 + u) % NY]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Accumulators that a loop carries stay whole in accumulation registers: known to start at zero, they
// would be taken apart into 16 floats each, which are moved there and back in every iteration.
template <int N>
__device__ __forceinline__ void pin(f32x16 (&acc)[N]) {
#pragma unroll
  for (int y = 0; y < N; ++y) asm("" : "+a"(acc[y]));
}

// Store 4 consecutive values.
__device__ __forceinline__ void store4(bf16* p, f32x4 v) { tda::store4(p, v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(_Float16* p, f32x4 v) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<half4*>(p) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}
__device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }

// Workgroup ids over (heads x tiles) with the heaviest tiles first: consecutive ids go to the 8 XCDs
// in turn, so where the heads divide evenly an XCD keeps to its own heads, whose rows its L2 then
// serves; `late`: tile 0 is the lightest.
struct Item { int head, tile; };
__device__ __forceinline__ Item item_of(uint32_t bid, uint32_t heads, int tiles, bool late) {
  Item it;
  uint32_t t;
  if (heads % 8 == 0) {
    const uint32_t per = heads / 8, x = bid & 7, i = bid >> 3;
    it.head = x * per + i % per;
    t = i / per;
  } else {
    it.head = bid % heads;
    t = bid / heads;
  }
  it.tile = late ? tiles - 1 - (int)t : (int)t;
  return it;
}

constexpr int kLds = 160 * 1024;  // of a CU

// Whether a launch of n workgroups of 128 rows (or keys) takes workgroups of 64 instead, whose waves share
// the other axis out: where the 128s leave half of the 256 CUs' places idle, or, under a causal mask that
// gives some of them far more work than others, where all of them are placed at once and the longest decides.
// A CU holds one workgroup, two of 16-bit (64, 64).  Forward and backward, us, whole : halved:
//   bf16 (128, 128), 500 rows of 4355 keys, 128 workgroups   127 : 103
//   bf16 (64, 128), (1, 8, 1024) causal, 64                   33 : 25 and 98 : 64
//   bf16 (64, 128), (2, 16, 1024) causal, 256                 40 : 37 and 109 : 88;  all seen 43 : 50, 113 : 122
//   bf16 (64, 128), (2, 16, 1500) causal, 384                 54 : 63 and 155 : 157
//   bf16 (64, 64), (2, 16, 2048) causal, 512                  62 : 59 and 236 : 212;  1024: 95 : 109, 339 : 379
//   f32 (64, 64), (2, 12, 1111) causal, 216                  157 : 94 and 455 : 274;  all seen 156 : 159, 453 : 480
//   f32 (64, 64), (2, 16, 2048) causal, 512                  291 : 296 and 876 : 903
template <class Tr, int D, int DV>
inline bool halve(const Sight& see, int64_t n, int Nq) {
  const int64_t places = sizeof(typename Tr::T) == 2 && D == 64 && DV == 64 ? 512 : 256;
  const bool unequal = see.causal && !see.qoffs && see.qoff < Nq / 2;
  return n <= (unequal ? places : places / 2);
}

}  // namespace sda
