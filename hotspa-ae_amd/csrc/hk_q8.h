// Activations kept in 8 bits for the backward pass: rows as blocks of 32 columns that share one power of two (the MXINT8
// format of the OCP microscaling specification).  Of a block with the largest magnitude a, E = the exponent field of a as
// fp32 (at least 7), a column holds q = rint(x 2^(133 - E)), cut to [-127, 127], and stands for q 2^(E - 133): off by at
// most half a step of 2^(E - 133), by less than a whole one past 127.5 steps.  A block with an infinity or a NaN has E = 255
// and stands for NaN.  The scale is a power of two, so that both directions are exact but for the one rounding to q.
#pragma once

#include "hk_common.h"

#include <type_traits>

namespace hk {

constexpr int kQ8Block = 32;
inline int64_t q8_blocks(int64_t cols) { return (cols + kQ8Block - 1) / kQ8Block; }

// A row's columns [c, c + N) of R as floats, c a multiple of N; 0 past the row's end: one load of 16 bytes, or of 8 where a
// 16-bit operand goes along with an fp32 one (neighbouring lanes then read neighbouring memory in both: a residual stream in
// fp32 beside bf16 rows, read as two 16-byte loads 32 bytes apart: the forward norm of 32768 x 4096 in 430 us instead of
// 284).  kTail: the row may end before or inside a vector, which is then loaded as the row's last N elements and moved down, so that every load is a whole vector
// inside the row and none sits in a branch; kWhole: every vector lies inside; kShort: the row may be shorter than a load, a
// variant of its own, since the branch for it makes the compiler wait for loads that are under way.  kOdd: as kTail, and rows of
// 16-bit elements may begin on an odd element, where a load of 16 bytes takes a multiple of its time: those load from one
// column on, and the first column of a lane's vector comes from the lane before it, or for the wavefront's first lane (of a
// row) from a load of its own.  raw is the load, floats() what comes of it.
typedef u32x2 u32x2_on2 __attribute__((aligned(2)));
constexpr int kWhole = 0, kTail = 1, kShort = 2, kOdd = 3;
template <typename R, int N, int TAIL>
struct RowVec {
  static constexpr int kWords = N * int(sizeof(R)) / 4;
  static_assert(kWords == 4 || kWords == 2, "one load of 16 or 8 bytes");
  u32x4 raw;
  static constexpr bool kOddRows = TAIL == kOdd && sizeof(R) == 2;
  struct Nothing {};
  typename std::conditional<kOddRows, uint32_t, Nothing>::type first;   // kOddRows: the wavefront's first element
  typename std::conditional<kOddRows, bool, Nothing>::type odd;
  // row: any element boundary; one of cols elements, cols >= 1
  template <bool KEEP = false>   // KEEP: read by many workgroups
  __device__ __forceinline__ void load(const R* row, int c, int cols, [[maybe_unused]] int lane_in_row = 0) {
    if (TAIL == kShort && cols < N) {   // uniform
      float f[8] = {};
      if (c == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < cols) f[j] = Cvt<R>::load(row + j);
      }
      raw = VecIO<R>::pack(f);
      return;
    }
    int from = c;
    if constexpr (kOddRows) {
      odd = (reinterpret_cast<uintptr_t>(row) & 2u) != 0;
      from += odd ? 1 : 0;
      first = *reinterpret_cast<const uint16_t*>(row + min(c - (lane_in_row & 63) * N, cols - 1));
    }
    // (a scalar base and 32 bits of offset)
    const R* p = reinterpret_cast<const R*>(reinterpret_cast<const char*>(row) + uint32_t(TAIL ? min(from, cols - N) : c) * uint32_t(sizeof(R)));
    if constexpr (kWords == 4) {
      if constexpr (KEEP) raw = ld16_any_keep<R>(p);
      else raw = ld16_any<R>(p);
    } else {
      u32x2 w;
      if constexpr (KEEP) w = *reinterpret_cast<const u32x2_on2*>(p);
      else w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_on2*>(p));
      raw = u32x4{w.x, w.y, 0, 0};
    }
  }
  // full (uniform): every lane's vector lies inside the row
  __device__ __forceinline__ void floats(float* f, int c, int cols, bool full = false, [[maybe_unused]] int lane_in_row = 0) const {
    u32x4 r = raw;
    if constexpr (kOddRows) {
      constexpr int kWaveShr1 = 0x138;
      uint32_t before = uint32_t(__builtin_amdgcn_update_dpp(0, int(raw[kWords - 1]), kWaveShr1, 0xf, 0xf, false));
      before = (lane_in_row & 63) == 0 ? first << 16 : before;
      const bool shifted = odd && c < cols - N;
#pragma unroll
      for (int k = 0; k < kWords; ++k) r[k] = shifted ? __builtin_amdgcn_alignbit(raw[k], k ? raw[k - 1] : before, 16) : raw[k];
    }
    if constexpr (TAIL) {
      if (!full && (TAIL != kShort || cols >= N)) {   // uniform
        const int bits = (c - min(c, cols - N)) * int(sizeof(R)) * 8;
        const uint64_t lo = uint64_t(r.y) << 32 | r.x;
        if constexpr (kWords == 2) {
          const uint64_t l = bits < 64 ? lo >> (bits & 63) : 0;
          r = u32x4{uint32_t(l), uint32_t(l >> 32), 0, 0};
        } else {
          const uint64_t hi = uint64_t(r.w) << 32 | r.z, in = bits & 63 ? hi << (64 - (bits & 63)) : 0;
          uint64_t l = bits >= 64 ? hi >> (bits & 63) : (lo >> (bits & 63)) | in, h = bits >= 64 ? 0 : hi >> (bits & 63);
          if (bits >= 128) l = 0;
          r = u32x4{uint32_t(l), uint32_t(l >> 32), uint32_t(h), uint32_t(h >> 32)};
        }
      }
    }
    if constexpr (kWords == 4) {
      VecIO<R>::unpack(r, f);
    } else {
      float e[8];
      VecIO<R>::unpack(r, e);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = e[j];
    }
  }
};

// stores N floats as R at columns [c, c + N) of a row, those inside it
template <typename R, int N, int TAIL>
__device__ __forceinline__ void store_row_floats(R* row, int c, int cols, const float* f) {
  constexpr int kWords = N * int(sizeof(R)) / 4;
  float e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = j < N ? f[j] : 0.f;
  const u32x4 r = VecIO<R>::pack(e);
  const int left = cols - c;
  R* p = reinterpret_cast<R*>(reinterpret_cast<char*>(row) + uint32_t(c) * uint32_t(sizeof(R)));
  if (!TAIL || left >= N) {
    if constexpr (kWords == 4) st16_any(p, r);
    else __builtin_nontemporal_store(u32x2{r.x, r.y}, reinterpret_cast<u32x2_on2*>(p));
  } else if (left > 0) {
    typedef uint32_t word __attribute__((aligned(2)));
    const int words = left * int(sizeof(R)) / 4;
#pragma unroll
    for (int i = 0; i < kWords - 1; ++i)
      if (i < words) reinterpret_cast<word*>(p)[i] = r[i];
    if (sizeof(R) == 2 && (left & 1)) {
      const uint32_t last = words == 0 ? r.x : words == 1 ? r.y : words == 2 ? r.z : r.w;
      reinterpret_cast<uint16_t*>(p)[left - 1] = uint16_t(last);
    }
  }
}

// The exponent field of the block that this lane's N elements belong to: the 32 / N lanes of a block are neighbours and
// start at a multiple of their number.  Infinities and NaN have the largest field, 255.  ANY: a NaN may be among them (a
// maximum of floats passes it over; integers see it, for an instruction more per element).
__device__ __forceinline__ float max3_abs(float a, float b, float c) {   // max(|a|, |b|, c)
  float r;
  asm("v_max3_f32 %0, |%1|, |%2|, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <int N, bool ANY = true>
__device__ __forceinline__ uint32_t q8_exponent(const float* f) {
  static_assert(N == 4 || N == 8, "a block is 8 or 4 lanes");
  uint32_t m = 0;
  if constexpr (ANY) {
#pragma unroll
    for (int j = 0; j < N; ++j) m = max(m, f2u(f[j]) & 0x7fffffffu);
  } else {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < N; j += 2) x = max3_abs(f[j], f[j + 1], x);
    m = f2u(x);
  }
  m = max(m, f2u(dpp_perm<kDppXor1>(u2f(m))));
  m = max(m, f2u(dpp_perm<kDppXor2>(u2f(m))));
  if constexpr (N == 4) m = max(m, f2u(dpp_perm<kDppHalfMirror>(u2f(m))));
  return max(m >> 23, 7u);
}
// q of 4 elements in the bytes of a word; factor = 2^(133 - E).  Added to 1.5 * 2^23 a float of that size is rounded to a
// whole number, ties to even, whose two's complement stands in its lowest bits.
__device__ __forceinline__ float q8_factor(uint32_t exponent) { return u2f((260u - exponent) << 23); }
__device__ __forceinline__ uint32_t q8_encode4(const float* f, float factor) {
  constexpr float kMagic = 12582912.f;
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = f2u(__builtin_amdgcn_fmed3f(fmaf(f[j], factor, kMagic), kMagic - 127.f, kMagic + 127.f));
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return lo | hi;
}
// 2^(E - 133), NaN for E = 255; E below 7 (which q8_exponent never gives) is a subnormal step
__device__ __forceinline__ float q8_step(uint32_t exponent) {
  const uint32_t bits = exponent >= 7 ? (exponent - 6) << 23 : 1u << (exponent + 16);
  return u2f(exponent == 255 ? 0x7fc00000u : bits);
}
// the whole numbers of 4 bytes
__device__ __forceinline__ void q8_numbers4(uint32_t bytes, float* f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = float(int8_t(bytes >> (8 * j)));
}

// the words of N elements, N = 4 or 8
template <int N> struct Q8Words;
template <> struct Q8Words<8> {
  typedef u32x2 type;
  static __device__ __forceinline__ type encode(const float* f, float factor) {
    return u32x2{q8_encode4(f, factor), q8_encode4(f + 4, factor)};
  }
  static __device__ __forceinline__ void numbers(type w, float* f) {
    q8_numbers4(w.x, f);
    q8_numbers4(w.y, f + 4);
  }
};
template <> struct Q8Words<4> {
  typedef uint32_t type;
  static __device__ __forceinline__ type encode(const float* f, float factor) { return q8_encode4(f, factor); }
  static __device__ __forceinline__ void numbers(type w, float* f) { q8_numbers4(w, f); }
};

// ---------------------------------------------------------------------------
// what the norm calls are given
// ---------------------------------------------------------------------------
struct Q8FwdArgs {
  const void *x0, *residual, *gamma, *beta;
  void *z, *x_out;
  int8_t* q;
  uint8_t* scale;
  float *mu, *rs;
  int64_t x0_pitch, res_pitch, z_pitch, xout_pitch;
  float eps, inv_cols;
  int rows, cols, blocks;   // blocks: of 32 columns in a row
  uint16_t threads;
};
struct Q8BwdArgs {
  const void *dz, *dx_in, *gamma;
  const int8_t* q;
  const uint8_t* scale;
  const float *mu, *rs;
  void *dx0, *dres;
  float *part_dgamma, *part_dbeta;
  int64_t dz_pitch, dxin_pitch, dx_pitch, dres_pitch;
  float inv_cols;
  int rows, cols, blocks, grid;
  uint16_t threads;
  uint8_t few;              // 1, 2: without partial rows, in one launch or two; part_dgamma / part_dbeta are then dgamma / dbeta
};

constexpr int kQ8MaxCols = 32768;

// rows of a launch that gives each `threads` threads: a launch's threads fit 32 bits
inline int64_t rows_of_a_launch(int64_t threads) { return (int64_t(1) << 31) / threads; }

// columns of a lane's vector: see RowVec
template <typename T, typename RT>
constexpr int q8_vec() { return sizeof(T) == 2 && sizeof(RT) == 2 ? 8 : 4; }

// Lanes that hold a row and vectors per lane: lanes of a wavefront (8, 16, 32, 64) or, above 64, a workgroup's threads.
struct Q8Shape {
  int lanes, nv;
};
Q8Shape q8_fwd_shape(int64_t cols, int vec);
Q8Shape q8_bwd_shape(int64_t cols, int vec);
// workgroups of the backward kernel
int q8_bwd_grid(int64_t rows, const Q8Shape& shape, bool extra);

template <typename T> int q8_norm_fwd_typed(const Q8FwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, hipStream_t s);
template <typename T> int q8_norm_bwd_typed(const Q8BwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, void* dgamma,
                                            void* dbeta, hipStream_t s);

} // namespace hk
