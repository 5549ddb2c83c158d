// The norm of a pre-norm block whose input is kept in 8 bits: forward and backward kernels, included by the per-type files.
//
//   x = x0 + residual (fp32);  mu = mean x;  rs = 1 / sqrt(mean (x - mu)^2 + eps), RMSNorm 1 / sqrt(mean x^2 + eps)
//   z = gamma rs (x - [mu]) + beta;  (q, scale) = x in 8 bits (hk_q8.h)
// and with x^ = rs (x8 - [mu]) of the kept values x8, u = dz gamma:
//   dx = rs (u - [mean u] - x^ mean(u x^)) + dx_in;   dgamma = sum over rows dz x^,  dbeta = sum over rows dz
// ([..]: LayerNorm only).
#pragma once

#include "hk_q8.h"

namespace hk {

// how a thread group holds a row: LPR lanes of a wavefront, or a workgroup (LPR == 0)
template <int LPR>
struct Q8Group {
  static __device__ __forceinline__ int count(int threads) { return LPR ? LPR : threads; }
  static __device__ __forceinline__ int lane() { return LPR ? int(threadIdx.x) & (LPR - 1) : int(threadIdx.x); }
  static __device__ __forceinline__ int group() {
    return LPR == 0 ? 0 : LPR == kWave ? wave_index() : int(threadIdx.x) / LPR;
  }
  static constexpr int kRows = LPR ? 256 / (LPR ? LPR : 1) : 1;   // rows of a workgroup
  template <typename P>
  static __device__ __forceinline__ P allreduce(P p, float* red, int threads) {
    if constexpr (LPR == 0) return group_allreduce_tuple(p, red, 0, threads >> 6);
    else return lanes_allreduce_tuple<LPR>(p);
  }
};

// One pass: the row stays in registers, two reductions (one for RMSNorm), then z.  The sum goes out after the first
// reduction: it may lie over the residual, and every lane has read its part of the row by then.
template <typename T, typename RT, int NV, int LPR, bool HAS_RES, bool IS_RMS, bool TAIL>
__global__ __launch_bounds__(LPR ? 256 : 1024)
void q8_norm_fwd_kernel(Q8FwdArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Group = Q8Group<LPR>;
  using Words = Q8Words<VEC>;
  __shared__ float red[2][kMaxWaves * 2];
  const int tpr = Group::count(a.threads), t = Group::lane();
  const int64_t row = int64_t(blockIdx.x) * Group::kRows + Group::group();
  if (LPR && row >= a.rows) return;   // no barrier in this mode
  const int cols = a.cols;
  auto column = [&](int i) { return (i * tpr + t) * VEC; };

  float v[NV][VEC];
  {
    RowVec<T, VEC, TAIL> x[NV];
    [[maybe_unused]] RowVec<RT, VEC, TAIL> r[NV];
    const T* xr = static_cast<const T*>(a.x0) + row * a.x0_pitch;
    const RT* rr = HAS_RES ? static_cast<const RT*>(a.residual) + row * a.res_pitch : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].load(xr, column(i), cols, false);
      if constexpr (HAS_RES) r[i].load(rr, column(i), cols, false);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].floats(v[i], column(i), cols);
      if constexpr (HAS_RES) {
        float f[VEC];
        r[i].floats(f, column(i), cols);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += f[j];
      }
    }
  }
  auto store_sum = [&] {
    if (a.x_out) {   // uniform
      RT* xo = static_cast<RT*>(a.x_out) + row * a.xout_pitch;
#pragma unroll
      for (int i = 0; i < NV; ++i) store_row_floats<RT, VEC, TAIL>(xo, column(i), cols, v[i]);
    }
  };
  float mu, rs;
  if constexpr (IS_RMS) {
    SumTuple<2> s = SumTuple<2>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) { s.v[0] = fmaf(v[i][j], v[i][j], s.v[0]); s.v[1] += v[i][j]; }
    s = Group::allreduce(s, red[0], tpr);
    mu = s.v[1] * a.inv_cols;
    rs = 1.0f / sqrtf(s.v[0] * a.inv_cols + a.eps);
    store_sum();
  } else {
    SumTuple<1> s = SumTuple<1>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.v[0] += v[i][j];
    s = Group::allreduce(s, red[0], tpr);
    mu = s.v[0] * a.inv_cols;
    store_sum();
    s = SumTuple<1>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = cols - column(i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = j < left ? v[i][j] - mu : 0.f;
        s.v[0] = fmaf(d, d, s.v[0]);
      }
    }
    s = Group::allreduce(s, red[1], tpr);
    rs = 1.0f / sqrtf(s.v[0] * a.inv_cols + a.eps);
  }
  if (t == 0) {
    a.mu[row] = mu;
    a.rs[row] = rs;
  }
  // the input in 8 bits; zeros behind the row's end up to the block's
  int8_t* qr = a.q + row * int64_t(a.blocks) * kQ8Block;
  uint8_t* sr = a.scale + row * int64_t(a.blocks);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t e = q8_exponent<VEC>(v[i]);
    const typename Words::type w = Words::encode(v[i], q8_factor(e));
    const int c = column(i);
    if (c < a.blocks * kQ8Block) {
      *reinterpret_cast<typename Words::type*>(qr + c) = w;
      if (t % LPB == 0) sr[c / kQ8Block] = uint8_t(e);
    }
  }
  T* zr = static_cast<T*>(a.z) + row * a.z_pitch;
  const T* gp = static_cast<const T*>(a.gamma);
  const T* bp = static_cast<const T*>(a.beta);
  const float shift = IS_RMS ? 0.f : mu;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column(i);
    float g[VEC], b[VEC], f[VEC];
    RowVec<T, VEC, TAIL> p;
    if (gp) { p.load(gp, c, cols, true); p.floats(g, c, cols); }   // uniform
    if (bp) { p.load(bp, c, cols, true); p.floats(b, c, cols); }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float n = rs * (v[i][j] - shift);
      f[j] = gp ? (bp ? fmaf(g[j], n, b[j]) : g[j] * n) : (bp ? n + b[j] : n);
    }
    store_row_floats<T, VEC, TAIL>(zr, c, cols, f);
  }
}

// A persistent grid walks the rows; a thread keeps its columns' sums of dz x^ and dz, and the workgroup leaves one fp32
// partial row of each.  The next row's loads are under way while a row is worked on.
// MAXT: the most threads of a workgroup; above 512 the register budget is half of what the widest rows would take.
template <typename T, typename RT, int NV, int LPR, int MAXT, bool EXTRA, bool IS_RMS, bool TAIL>
__global__ __launch_bounds__(MAXT)
void q8_norm_bwd_kernel(Q8BwdArgs a) {
  constexpr int VEC = VecIO<T>::N, NE = NV * VEC;
  using Group = Q8Group<LPR>;
  using Words = Q8Words<VEC>;
  constexpr int KS = IS_RMS ? 1 : 2;
  extern __shared__ __align__(16) float lds[];   // LPR: [kRows, pitch] staging of the column sums
  __shared__ float red[2][kMaxWaves * KS];
  const int tpr = Group::count(a.threads), t = Group::lane(), group = Group::group();
  const int cols = a.cols, pitch = a.blocks * kQ8Block;
  auto column = [&](int i) { return (i * tpr + t) * VEC; };

  float gm[NE], dg[NE];
  [[maybe_unused]] float db[IS_RMS ? 1 : NE];
  const T* gp = static_cast<const T*>(a.gamma);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) gm[i * VEC + j] = 1.f;
    if (gp) {
      RowVec<T, VEC, TAIL> p;
      p.load(gp, column(i), cols, true);
      p.floats(&gm[i * VEC], column(i), cols);
    }
  }
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    dg[e] = 0.f;
    if constexpr (!IS_RMS) db[e] = 0.f;
  }
  struct Slot {
    RowVec<T, VEC, TAIL> dz[NV];
    RowVec<RT, VEC, TAIL> up[EXTRA ? NV : 1];
    typename Words::type q[NV];
    uint8_t e[NV];
    float mu, rs;
  } next;
  const int64_t last = a.rows - 1;
  auto issue = [&](int64_t r) {
    const int64_t rc = r < last ? r : last;
    next.rs = a.rs[rc];
    if constexpr (!IS_RMS) next.mu = a.mu[rc];
    const T* dr = static_cast<const T*>(a.dz) + rc * a.dz_pitch;
    const int8_t* qr = a.q + rc * int64_t(pitch);
    const uint8_t* sr = a.scale + rc * int64_t(a.blocks);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = min(column(i), pitch - VEC);
      next.dz[i].load(dr, column(i), cols, false);
      next.q[i] = __builtin_nontemporal_load(reinterpret_cast<const typename Words::type*>(qr + c));
      next.e[i] = sr[c / kQ8Block];
      if constexpr (EXTRA) {
        if (a.dx_in) next.up[i].load(static_cast<const RT*>(a.dx_in) + rc * a.dxin_pitch, column(i), cols, false);
      }
    }
  };
  const int64_t stride = int64_t(a.grid) * Group::kRows;
  int64_t base = int64_t(blockIdx.x) * Group::kRows;
  int parity = 0;
  issue(base + group);
#pragma nounroll
  for (; base < a.rows; base += stride) {   // uniform over the workgroup
    const int64_t row = base + group;
    const bool valid = LPR == 0 || row < a.rows;
    float x[NE], u[NE];
    [[maybe_unused]] float up[EXTRA ? NE : 1];
    const float rs = next.rs;
    const float mu = IS_RMS ? 0.f : next.mu;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = column(i);
      next.dz[i].floats(&u[i * VEC], c, cols);
      Words::decode(next.q[i], next.e[i], &x[i * VEC]);
      if constexpr (EXTRA) {
        if (a.dx_in) next.up[i].floats(&up[i * VEC], c, cols);
      }
    }
    issue(row + stride);
    SumTuple<KS> s = SumTuple<KS>::identity();
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const float dz = valid ? u[e] : 0.f;           // 0 past the row's end
      // (nothing past the row's end, where another column's value or a NaN block's may stand)
      x[e] = column(e / VEC) + (TAIL ? e % VEC : 0) < cols ? rs * (x[e] - mu) : 0.f;
      dg[e] = fmaf(dz, x[e], dg[e]);
      if constexpr (!IS_RMS) db[e] += dz;
      u[e] = dz * gm[e];
      s.v[KS - 1] = fmaf(u[e], x[e], s.v[KS - 1]);
      if constexpr (!IS_RMS) s.v[0] += u[e];
    }
    s = Group::allreduce(s, red[parity], tpr);
    parity ^= 1;
    if (valid) {
      const float k1 = IS_RMS ? 0.f : s.v[0] * a.inv_cols, k2 = s.v[KS - 1] * a.inv_cols;
      T* dxr = static_cast<T*>(a.dx0) + row * a.dx_pitch;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = i * VEC + j;
          o[j] = rs * fmaf(-x[e], k2, u[e] - k1);
          if constexpr (EXTRA) {
            if (a.dx_in) o[j] += up[e];
          }
        }
        store_row_floats<T, VEC, TAIL>(dxr, column(i), cols, o);
        if constexpr (EXTRA) {
          if (a.dres) store_row_floats<RT, VEC, TAIL>(static_cast<RT*>(a.dres) + row * a.dres_pitch, column(i), cols, o);
        }
      }
    }
  }
  auto put = [&](float* dst, const float* acc) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (column(i) < pitch) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          st16(dst + column(i) + j, u32x4{f2u(acc[i * VEC + j]), f2u(acc[i * VEC + j + 1]), f2u(acc[i * VEC + j + 2]),
                                          f2u(acc[i * VEC + j + 3])});
      }
    }
  };
  auto leave = [&](float* part, const float* acc) {
    if (part == nullptr) return;   // uniform
    float* dst = part + int64_t(blockIdx.x) * pitch;
    if constexpr (LPR == 0) {
      put(dst, acc);
    } else {
      __syncthreads();
      put(lds + group * pitch, acc);
      __syncthreads();
      for (int c = int(threadIdx.x) * 4; c < pitch; c += 256 * 4) {
        float r[4] = {0.f, 0.f, 0.f, 0.f};
        for (int g = 0; g < Group::kRows; ++g) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(lds + g * pitch + c);
          r[0] += u2f(w.x); r[1] += u2f(w.y); r[2] += u2f(w.z); r[3] += u2f(w.w);
        }
        st16(dst + c, u32x4{f2u(r[0]), f2u(r[1]), f2u(r[2]), f2u(r[3])});
      }
    }
  };
  leave(a.part_dgamma, dg);
  if constexpr (!IS_RMS) leave(a.part_dbeta, db);
}

// the partial rows folded into dgamma / dbeta (blockIdx.y picks which)
template <typename T, int LANES>
__global__ __launch_bounds__(fold_threads(LANES))
void q8_norm_fold_kernel(const float* part0, const float* part1, T* out0, T* out1, int nparts, int cols, int pitch) {
  const float s = fold_partial_rows<LANES>(blockIdx.y == 0 ? part0 : part1, nparts, pitch, int(blockIdx.x));
  const int c = int(blockIdx.x) * (4 * LANES) + int(threadIdx.x);
  if (int(threadIdx.x) < 4 * LANES && c < cols) Cvt<T>::store((blockIdx.y == 0 ? out0 : out1) + c, s);
}

template <typename T, typename RT, int NV, int LPR, bool TAIL>
static void launch_q8_norm_fwd(const Q8FwdArgs& a, bool is_rms, hipStream_t s) {
  const dim3 grid{unsigned((a.rows + Q8Group<LPR>::kRows - 1) / Q8Group<LPR>::kRows)}, block{LPR ? 256u : unsigned(a.threads)};
  profile_before(s);
  if (a.residual) {
    if (is_rms) HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, true, true, TAIL>), grid, block, 0, s, a);
    else HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, true, false, TAIL>), grid, block, 0, s, a);
  } else {
    if (is_rms) HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, false, true, TAIL>), grid, block, 0, s, a);
    else HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, false, false, TAIL>), grid, block, 0, s, a);
  }
  profile_after(s);
}
template <typename T, typename RT, int NV, int LPR, int MAXT, bool TAIL>
static void launch_q8_norm_bwd(const Q8BwdArgs& a, bool is_rms, hipStream_t s) {
  const dim3 grid{unsigned(a.grid)}, block{LPR ? 256u : unsigned(a.threads)};
  const size_t lds = LPR ? size_t(Q8Group<LPR>::kRows) * a.blocks * kQ8Block * sizeof(float) : 0;
  profile_before(s);
  if (a.dx_in || a.dres) {
    if (is_rms) HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, true, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, true, false, TAIL>), grid, block, lds, s, a);
  } else {
    if (is_rms) HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, false, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, false, false, TAIL>), grid, block, lds, s, a);
  }
  profile_after(s);
}

// WHAT: 0 forward, 1 backward
template <typename T, typename RT, int WHAT, typename A>
static int launch_q8_norm(const A& a, bool is_rms, const Q8Shape& shape, hipStream_t s) {
  const bool tail = a.cols % VecIO<T>::N != 0;
#define HK_Q8(NV, LPR)                                                                               \
  do {                                                                                               \
    if constexpr (WHAT == 0) {                                                                       \
      if (tail) launch_q8_norm_fwd<T, RT, NV, LPR, true>(a, is_rms, s);                              \
      else launch_q8_norm_fwd<T, RT, NV, LPR, false>(a, is_rms, s);                                  \
    } else {                                                                                         \
      constexpr int kMost = LPR ? 256 : 512;                                                         \
      if (LPR == 0 && NV >= 4 && a.threads > kMost) {                                                \
        if (tail) launch_q8_norm_bwd<T, RT, NV, LPR, LPR || NV < 4 ? kMost : 1024, true>(a, is_rms, s);  \
        else launch_q8_norm_bwd<T, RT, NV, LPR, LPR || NV < 4 ? kMost : 1024, false>(a, is_rms, s);  \
      } else if (tail) launch_q8_norm_bwd<T, RT, NV, LPR, kMost, true>(a, is_rms, s);                \
      else launch_q8_norm_bwd<T, RT, NV, LPR, kMost, false>(a, is_rms, s);                           \
    }                                                                                                \
  } while (0)
  switch (shape.lanes) {
    case 8: HK_Q8(1, 8); break;
    case 16: HK_Q8(1, 16); break;
    case 32: HK_Q8(1, 32); break;
    case 64:
      switch (shape.nv) {
        case 1: HK_Q8(1, 64); break;
        case 2: HK_Q8(2, 64); break;
        default: HK_Q8(4, 64); break;
      }
      break;
    default:
      switch (shape.nv) {
        case 1: HK_Q8(1, 0); break;
        case 2: HK_Q8(2, 0); break;
        case 4: HK_Q8(4, 0); break;
        default:
          HK_REQUIRE(sizeof(T) == 4 && shape.nv == 8, HK_ERR_UNSUPPORTED, "q8_norm: no kernel for %d vectors a thread", shape.nv);
          if constexpr (sizeof(T) == 4) HK_Q8(8, 0);
          break;
      }
  }
#undef HK_Q8
  return launch_check(WHAT == 0 ? "q8_norm_fwd_kernel" : "q8_norm_bwd_kernel");
}

template <typename T>
int q8_norm_fwd_typed(const Q8FwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (rtype == HK_FLOAT32) return launch_q8_norm<T, float, 0>(a, is_rms, shape, s);
  }
  return launch_q8_norm<T, T, 0>(a, is_rms, shape, s);
}
template <typename T>
int q8_norm_bwd_typed(const Q8BwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, void* dgamma, void* dbeta,
                      hipStream_t s) {
  int rc;
  if (sizeof(T) == 2 && rtype == HK_FLOAT32) {
    if constexpr (sizeof(T) == 2) rc = launch_q8_norm<T, float, 1>(a, is_rms, shape, s);
  } else {
    rc = launch_q8_norm<T, T, 1>(a, is_rms, shape, s);
  }
  if (rc != HK_OK || (dgamma == nullptr && dbeta == nullptr)) return rc;
  const int pitch = a.blocks * kQ8Block, sums = (dgamma != nullptr) + (dbeta != nullptr);
  const float* p0 = dgamma ? a.part_dgamma : a.part_dbeta;
  T* o0 = static_cast<T*>(dgamma ? dgamma : dbeta);
#define HK_Q8_FOLD(LANES)                                                                                              \
  HK_LAUNCH((q8_norm_fold_kernel<T, LANES>), dim3(unsigned((pitch + 4 * LANES - 1) / (4 * LANES)), unsigned(sums)),    \
            dim3(fold_threads(LANES)), 0, s, p0, a.part_dbeta, o0, static_cast<T*>(dbeta), a.grid, a.cols, pitch)
  if (fold_lanes(pitch, sums) == 8) HK_Q8_FOLD(8);
  else HK_Q8_FOLD(32);
#undef HK_Q8_FOLD
  return launch_check("q8_norm_fold_kernel");
}

} // namespace hk
