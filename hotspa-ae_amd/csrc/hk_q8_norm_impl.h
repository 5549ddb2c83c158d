// The norm of a pre-norm block whose input is kept in 8 bits: forward and backward kernels, included by the per-type files.
//
//   x = x0 + residual (fp32);  mu = mean x;  rs = 1 / sqrt(mean (x - mu)^2 + eps), RMSNorm 1 / sqrt(mean x^2 + eps)
//   z = gamma rs (x - [mu]) + beta;  (q, scale) = x in 8 bits (hk_q8.h)
// and with x^ = rs (x8 - [mu]) of the kept values x8, u = dz gamma:
//   dx = rs (u - [mean u] - x^ mean(u x^)) + dx_in;   dgamma = sum over rows dz x^,  dbeta = sum over rows dz
// ([..]: LayerNorm only).
#pragma once

#include "hk_q8.h"

#include <algorithm>

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
  // the first column behind the i-th vectors of this wavefront's lanes (uniform)
  template <int VEC>
  static __device__ __forceinline__ int wave_end(int i, int threads) {
    if constexpr (LPR) return (i + 1) * LPR * VEC;
    else return (i * threads + (wave_index() + 1) * kWave) * VEC;
  }
  template <typename P>
  static __device__ __forceinline__ P allreduce(P p, float* red, int threads) {
    if constexpr (LPR == 0) return group_allreduce_tuple(p, red, 0, threads >> 6);
    else return lanes_allreduce_tuple<LPR>(p);
  }
};

// One pass: the row stays in registers, two reductions (one for RMSNorm), then z.  The sum goes out after the first
// reduction: it may lie over the residual, and every lane has read its part of the row by then.  The 8 bits go out before it:
// they need no statistics, and nothing waits for them.  Bound by memory (32768 x 4096 bf16, us here / what the bytes take:
// RMSNorm 102 / 99, with a bf16 residual 182 / 178, with one in fp32 274 / 257; LayerNorm of 16384 x 5120 68 / 62); odd widths
// pay for loads and stores that begin on any element (LayerNorm of 9000 rows bf16: 29.5 at 3584 columns, 33.0 at 3579; 30.0 at
// 3579 with the rows on 16-byte boundaries).
template <typename T, typename RT, int NV, int LPR, bool HAS_RES, bool IS_RMS, int TAIL>
__global__ __launch_bounds__(LPR ? 256 : 1024)
void q8_norm_fwd_kernel(Q8FwdArgs a) {
  constexpr int VEC = q8_vec<T, RT>(), LPB = kQ8Block / VEC;
  using Group = Q8Group<LPR>;
  using Words = Q8Words<VEC>;
  __shared__ float red[2][kMaxWaves * 2];
  const int tpr = Group::count(a.threads), t = Group::lane();
  const int64_t row = int64_t(blockIdx.x) * Group::kRows + Group::group();
  if (LPR && row >= a.rows) return;   // no barrier in this mode
  const int cols = a.cols;
  auto column = [&](int i) { return (i * tpr + t) * VEC; };

  // whether vector i of the wavefront's lanes lies inside the row (without TAIL all do)
  auto full = [&](int i) { return !TAIL || Group::template wave_end<VEC>(i, tpr) <= cols; };

  const T* gp = static_cast<const T*>(a.gamma);
  const T* bp = static_cast<const T*>(a.beta);
  RowVec<T, VEC, TAIL == kOdd ? kTail : TAIL> g[NV], b[NV];
  float v[NV][VEC];
  {
    RowVec<T, VEC, TAIL> x[NV];
    [[maybe_unused]] RowVec<RT, VEC, TAIL> r[NV];
    const T* xr = static_cast<const T*>(a.x0) + row * a.x0_pitch;
    const RT* rr = HAS_RES ? static_cast<const RT*>(a.residual) + row * a.res_pitch : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].load(xr, column(i), cols, t);
      if constexpr (HAS_RES) r[i].load(rr, column(i), cols, t);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].floats(v[i], column(i), cols, full(i), t);
      if constexpr (HAS_RES) {
        float f[VEC];
        r[i].floats(f, column(i), cols, full(i), t);
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
  // the input in 8 bits, zeros behind the row's end up to the block's; before LayerNorm centres the row in place
  auto keep = [&](float sum) {   // sum of this thread's elements: a NaN where one of them is
    const bool nan = __builtin_expect(__builtin_amdgcn_ballot_w64(sum != sum) != 0, 0);   // uniform in a wavefront
    int8_t* qr = a.q + row * int64_t(a.blocks) * kQ8Block;
    uint8_t* sr = a.scale + row * int64_t(a.blocks);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t e = q8_exponent<VEC, false>(v[i]);
      if (nan) e = q8_exponent<VEC, true>(v[i]);
      const typename Words::type w = Words::encode(v[i], q8_factor(e));
      const uint32_t c = uint32_t(column(i));
      if (!TAIL || int(c) < a.blocks * kQ8Block) {
        *reinterpret_cast<typename Words::type*>(qr + c) = w;
        if (t % LPB == 0) sr[c / kQ8Block] = uint8_t(e);
      }
    }
  };
  auto parameters = [&] {
    if (gp)   // uniform
#pragma unroll
      for (int i = 0; i < NV; ++i) g[i].template load<true>(gp, column(i), cols);
    if (bp)
#pragma unroll
      for (int i = 0; i < NV; ++i) b[i].template load<true>(bp, column(i), cols);
  };
  float mu, rs;
  if constexpr (IS_RMS) {
    SumTuple<2> s = SumTuple<2>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) { s.v[0] = fmaf(v[i][j], v[i][j], s.v[0]); s.v[1] += v[i][j]; }
    keep(s.v[0]);
    s = Group::allreduce(s, red[0], tpr);
    parameters();
    mu = s.v[1] * a.inv_cols;
    rs = 1.0f / sqrtf(s.v[0] * a.inv_cols + a.eps);
    store_sum();
  } else {
    SumTuple<1> s = SumTuple<1>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.v[0] += v[i][j];
    keep(s.v[0]);
    s = Group::allreduce(s, red[0], tpr);
    parameters();
    mu = s.v[0] * a.inv_cols;
    store_sum();
    // centred in place: the second sum and z take the same values
    s = SumTuple<1>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (full(i)) {   // uniform
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] -= mu;
          s.v[0] = fmaf(v[i][j], v[i][j], s.v[0]);
        }
      } else {
        const int left = cols - column(i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] = j < left ? v[i][j] - mu : 0.f;
          s.v[0] = fmaf(v[i][j], v[i][j], s.v[0]);
        }
      }
    }
    s = Group::allreduce(s, red[1], tpr);
    rs = 1.0f / sqrtf(s.v[0] * a.inv_cols + a.eps);
  }
  if (t == 0) {
    a.mu[row] = mu;
    a.rs[row] = rs;
  }
  T* zr = static_cast<T*>(a.z) + row * a.z_pitch;
  auto finish = [&](auto has_g, auto has_b) {
    constexpr bool HG = decltype(has_g)::value, HB = decltype(has_b)::value;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      [[maybe_unused]] float gf[VEC], bf[VEC];
      float f[VEC];
      if constexpr (HG) g[i].floats(gf, column(i), cols, full(i));
      if constexpr (HB) b[i].floats(bf, column(i), cols, full(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float n = rs * v[i][j];
        f[j] = HG ? (HB ? fmaf(gf[j], n, bf[j]) : gf[j] * n) : (HB ? n + bf[j] : n);
      }
      store_row_floats<T, VEC, TAIL>(zr, column(i), cols, f);
    }
  };
  if (gp && bp) finish(std::true_type{}, std::true_type{});   // uniform
  else if (gp) finish(std::true_type{}, std::false_type{});
  else if (bp) finish(std::false_type{}, std::true_type{});
  else finish(std::false_type{}, std::false_type{});
}

// A persistent grid walks the rows; a thread keeps its columns' sums of dz x^ and dz, and the workgroup leaves one fp32
// partial row of each.  The next row's loads are under way while a row is worked on, and none sits in a branch (two and three
// rows ahead, RMSNorm of 32768 x 4096 bf16 with an upstream gradient: 200 and 204 us instead of 196).  Bound by memory: 178 us is
// what the bytes take.  EXTRA: an upstream gradient comes in.  MAXT: the most threads of a workgroup; above 512 the register
// budget is half of what the widest rows would take.
template <typename T, typename RT, int NV, int LPR, int MAXT, bool EXTRA, bool IS_RMS, int TAIL>
__global__ __launch_bounds__(MAXT)
void q8_norm_bwd_kernel(Q8BwdArgs a) {
  constexpr int VEC = q8_vec<T, RT>(), NE = NV * VEC;
  using Group = Q8Group<LPR>;
  using Words = Q8Words<VEC>;
  constexpr int KS = IS_RMS ? 1 : 2;
  extern __shared__ __align__(16) float lds[];   // LPR: [kRows, pitch] staging of the column sums
  __shared__ float red[2][kMaxWaves * KS];
  const int tpr = Group::count(a.threads), t = Group::lane(), group = Group::group();
  const int cols = a.cols, pitch = a.blocks * kQ8Block;
  auto column = [&](int i) { return (i * tpr + t) * VEC; };
  auto full = [&](int i) { return !TAIL || Group::template wave_end<VEC>(i, tpr) <= cols; };

  float dg[NE];
  [[maybe_unused]] float db[IS_RMS ? 1 : NE];
  const T* gp = static_cast<const T*>(a.gamma);
  // gamma as fp32, packed where that is more registers than there are
  constexpr bool kPacked = NE > 16 && sizeof(T) == 2;
  RowVec<T, VEC, TAIL == kOdd ? kTail : TAIL> gm[NV];
  [[maybe_unused]] float gf[kPacked ? 1 : NE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (gp) {   // uniform
      gm[i].template load<true>(gp, column(i), cols);
    } else {
      float one[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) one[j] = 1.f;
      gm[i].raw = VecIO<T>::pack(one);
    }
    if constexpr (!kPacked) gm[i].floats(&gf[i * VEC], gp ? column(i) : 0, gp ? cols : VEC);   // (ones need no moving)
  }
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    dg[e] = 0.f;
    if constexpr (!IS_RMS) db[e] = 0.f;
  }
  struct {
    RowVec<T, VEC, TAIL> dz[NV];
    RowVec<RT, VEC, TAIL> up[EXTRA ? NV : 1];
    typename Words::type q[NV];
    uint8_t e[NV];
    float mu, rs;
  } next;
  const int64_t last = a.rows - 1;
  auto issue = [&](int64_t r) {   // a row past the end reads the last one, which is then not used
    const int64_t rc = r < last ? r : last;
    next.rs = a.rs[rc];
    if constexpr (!IS_RMS) next.mu = a.mu[rc];
    const T* dr = static_cast<const T*>(a.dz) + rc * a.dz_pitch;
    const int8_t* qr = a.q + rc * int64_t(pitch);
    const uint8_t* sr = a.scale + rc * int64_t(a.blocks);
    const RT* ur = EXTRA ? static_cast<const RT*>(a.dx_in) + rc * a.dxin_pitch : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = uint32_t(TAIL ? min(column(i), pitch - VEC) : column(i));
      next.dz[i].load(dr, column(i), cols, t);
      next.q[i] = __builtin_nontemporal_load(reinterpret_cast<const typename Words::type*>(qr + c));
      next.e[i] = sr[c / kQ8Block];
      if constexpr (EXTRA) next.up[i].load(ur, column(i), cols, t);
    }
  };
  const int64_t stride = int64_t(a.grid) * Group::kRows;
  int64_t base = int64_t(blockIdx.x) * Group::kRows;
  int parity = 0;
  issue(base + group);
  // guarded: the row may not exist (the tail)
  auto step = [&](auto guarded) {
    constexpr bool GUARD = decltype(guarded)::value;
    const int64_t row = base + group;
    const bool valid = !GUARD || row < a.rows;
    float x[NE], u[NE];
    [[maybe_unused]] RowVec<RT, VEC, TAIL> up[EXTRA ? NV : 1];   // (packed until it is added)
    const float rs = next.rs;
    [[maybe_unused]] const float shift = IS_RMS ? 0.f : -rs * next.mu;
    float step_of[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next.dz[i].floats(&u[i * VEC], column(i), cols, full(i), t);
      Words::numbers(next.q[i], &x[i * VEC]);
      step_of[i] = rs * q8_step(next.e[i]);   // (a power of two: exact)
      if constexpr (EXTRA) up[i] = next.up[i];
      // (here before the reduction: the gradient may be written over it, and a vector may reach into another wavefront's columns)
      if constexpr (EXTRA && TAIL != kWhole && LPR == 0) asm volatile("" ::"v"(up[i].raw));
    }
    issue(row + stride);
    SumTuple<KS> s = SumTuple<KS>::identity();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float g[VEC];
      if constexpr (kPacked) gm[i].floats(g, gp ? column(i) : 0, gp ? cols : VEC, full(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (!kPacked) g[j] = gf[i * VEC + j];
        x[i * VEC + j] = IS_RMS ? x[i * VEC + j] * step_of[i] : fmaf(x[i * VEC + j], step_of[i], shift);
      }
      // (nothing past the row's end, where another column's value or a NaN block's may stand)
      if (!full(i))   // uniform
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i * VEC + j] = column(i) + j < cols ? x[i * VEC + j] : 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = i * VEC + j;
        const float dz = valid ? u[e] : 0.f;           // 0 past the row's end
        dg[e] = fmaf(dz, x[e], dg[e]);
        if constexpr (!IS_RMS) db[e] += dz;
        u[e] = dz * g[j];
        s.v[KS - 1] = fmaf(u[e], x[e], s.v[KS - 1]);
        if constexpr (!IS_RMS) s.v[0] += u[e];
      }
    }
    s = Group::allreduce(s, red[parity], tpr);
    parity ^= 1;
    if (valid) {
      const float k1 = IS_RMS ? 0.f : -rs * (s.v[0] * a.inv_cols), k2 = -rs * (s.v[KS - 1] * a.inv_cols);
      T* dxr = static_cast<T*>(a.dx0) + row * a.dx_pitch;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float o[VEC];
        [[maybe_unused]] float add[VEC];
        if constexpr (EXTRA) up[i].floats(add, column(i), cols, full(i), t);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = i * VEC + j;
          o[j] = fmaf(x[e], k2, IS_RMS ? u[e] * rs : fmaf(u[e], rs, k1));
          if constexpr (EXTRA) o[j] += add[j];
        }
        store_row_floats<T, VEC, TAIL>(dxr, column(i), cols, o);
        if (a.dres) store_row_floats<RT, VEC, TAIL>(static_cast<RT*>(a.dres) + row * a.dres_pitch, column(i), cols, o);   // uniform
      }
    }
  };
  // (the loops' bounds are the same for the whole workgroup, so every thread reaches the reductions' barriers)
#pragma nounroll
  for (; base + Group::kRows <= a.rows; base += stride) step(std::false_type{});
  if (base < a.rows) step(std::true_type{});
  auto put = [&](float* dst, const float* acc) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!TAIL || column(i) < pitch) {
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

// The whole backward without partial rows, of few rows in one launch (of wide ones in two: the sums, then dx): the first `sums` workgroups form the column sums of 8 vectors of columns each,
// from all rows, the others dx, rows side by side in a workgroup.  The partial rows that the kernel above would leave are as
// many bytes as the rows themselves by then (LayerNorm of 512 x 4096 bf16: 16.8 us with them and their fold, 5.2 so).  Only
// where nothing that is written lies over what is read, or in two launches.
template <typename T, typename RT, int NV, bool EXTRA, bool IS_RMS, int TAIL>
__global__ __launch_bounds__(kSmallThreads)
void q8_norm_bwd_few_kernel(Q8BwdArgs a, int sums) {
  constexpr int VEC = q8_vec<T, RT>(), KS = IS_RMS ? 1 : 2, LANES = 8;
  using Words = Q8Words<VEC>;
  __shared__ __align__(16) float red[kMaxWaves * KS];
  const int cols = a.cols, pitch = a.blocks * kQ8Block, rows = a.rows;
  const T* const dz = static_cast<const T*>(a.dz);
  if (int(blockIdx.x) < sums) {
    struct Fetched {
      RowVec<T, VEC, kTail> dz;   // (the last workgroup's columns may lie past the row's end)
      typename Words::type q;
      uint8_t e;
      float mu, rs;
    };
    const int first = int(blockIdx.x) * LANES * VEC, col = first + (int(threadIdx.x) & (LANES - 1)) * VEC;
    const uint32_t c = uint32_t(min(col, pitch - VEC));
    column_sums_of_few_rows<KS, VEC, LANES>(
        rows,
        [&](int64_t r) {
          Fetched f;
          f.dz.template load<true>(dz + r * a.dz_pitch, col, cols);
          f.q = *reinterpret_cast<const typename Words::type*>(a.q + r * pitch + c);
          f.e = a.scale[r * a.blocks + c / kQ8Block];
          f.mu = IS_RMS ? 0.f : a.mu[r];
          f.rs = a.rs[r];
          return f;
        },
        [&](const Fetched& f, bool in, float (&acc)[KS][VEC]) {
          float x[VEC], d[VEC];
          f.dz.floats(d, col, cols);
          Words::numbers(f.q, x);
          const float step = f.rs * q8_step(f.e), shift = IS_RMS ? 0.f : -f.rs * f.mu;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float xh = IS_RMS ? x[j] * step : fmaf(x[j], step, shift);
            const float more = fmaf(d[j], xh, acc[0][j]);
            acc[0][j] = in ? more : acc[0][j];
            if constexpr (KS == 2) acc[1][j] += in ? d[j] : 0.f;
          }
        },
        [&](int k, int j, float sum) {
          T* out = reinterpret_cast<T*>(k == 0 ? a.part_dgamma : a.part_dbeta);
          if (out != nullptr && first + j < cols) Cvt<T>::store(out + first + j, sum);
        });
    return;
  }
  const int tpr = a.threads, rpb = kSmallThreads / tpr;
  const int group = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / tpr), t = int(threadIdx.x) - group * tpr;
  // (wavefronts that no row is left for work on the last one too and store nothing)
  const bool idle = group >= rpb;
  const int64_t wanted = idle ? rows : int64_t(int(blockIdx.x) - sums) * rpb + group, row = wanted < rows ? wanted : rows - 1;
  auto column = [&](int i) { return (i * tpr + t) * VEC; };
  auto full = [&](int i) { return !TAIL || (i * tpr + (__builtin_amdgcn_readfirstlane(t) | 63) + 1) * VEC <= cols; };   // as above
  const T* gp = static_cast<const T*>(a.gamma);
  RowVec<T, VEC, TAIL> rd[NV], rg[NV];
  [[maybe_unused]] RowVec<RT, VEC, TAIL> up[EXTRA ? NV : 1];
  typename Words::type q[NV];
  uint8_t e[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = uint32_t(TAIL ? min(column(i), pitch - VEC) : column(i));
    rd[i].template load<true>(dz + row * a.dz_pitch, column(i), cols);
    q[i] = *reinterpret_cast<const typename Words::type*>(a.q + row * pitch + c);
    e[i] = a.scale[row * a.blocks + c / kQ8Block];
    if (gp) rg[i].template load<true>(gp, column(i), cols);   // uniform
    if constexpr (EXTRA) up[i].load(static_cast<const RT*>(a.dx_in) + row * a.dxin_pitch, column(i), cols);
  }
  if constexpr (EXTRA && TAIL != kWhole)   // as above
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" ::"v"(up[i].raw));
  const float rs = a.rs[row];
  [[maybe_unused]] const float shift = IS_RMS ? 0.f : -rs * a.mu[row];
  float x[NV][VEC], u[NV][VEC];
  SumTuple<KS> s = SumTuple<KS>::identity();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float g[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = 1.f;
    if (gp) rg[i].floats(g, column(i), cols, full(i));
    rd[i].floats(u[i], column(i), cols, full(i));
    Words::numbers(q[i], x[i]);
    const float step = rs * q8_step(e[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {   // as in the kernel above, to the same bits
      x[i][j] = IS_RMS ? x[i][j] * step : fmaf(x[i][j], step, shift);
      if (TAIL && !full(i)) x[i][j] = column(i) + j < cols ? x[i][j] : 0.f;
      u[i][j] *= g[j];
      s.v[KS - 1] = fmaf(u[i][j], x[i][j], s.v[KS - 1]);
      if constexpr (!IS_RMS) s.v[0] += u[i][j];
    }
  }
  s = group_allreduce_tuple(s, red, idle ? 0 : group * (tpr >> 6), tpr >> 6);
  if (wanted >= rows) return;
  const float k1 = IS_RMS ? 0.f : -rs * (s.v[0] * a.inv_cols), k2 = -rs * (s.v[KS - 1] * a.inv_cols);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float o[VEC];
    [[maybe_unused]] float add[VEC];
    if constexpr (EXTRA) up[i].floats(add, column(i), cols, full(i));
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      o[j] = fmaf(x[i][j], k2, IS_RMS ? u[i][j] * rs : fmaf(u[i][j], rs, k1));
      if constexpr (EXTRA) o[j] += add[j];
    }
    store_row_floats<T, VEC, TAIL>(static_cast<T*>(a.dx0) + row * a.dx_pitch, column(i), cols, o);
    if (a.dres) store_row_floats<RT, VEC, TAIL>(static_cast<RT*>(a.dres) + row * a.dres_pitch, column(i), cols, o);
  }
}

template <typename T, typename RT, int NV, bool EXTRA, int TAIL>
static void launch_q8_norm_few(const Q8BwdArgs& a, bool is_rms, dim3 grid, int sums, hipStream_t s) {
  profile_before(s);
  if (is_rms) HK_LAUNCH((q8_norm_bwd_few_kernel<T, RT, NV, EXTRA, true, TAIL>), grid, dim3(kSmallThreads), 0, s, a, sums);
  else HK_LAUNCH((q8_norm_bwd_few_kernel<T, RT, NV, EXTRA, false, TAIL>), grid, dim3(kSmallThreads), 0, s, a, sums);
  profile_after(s);
}
template <typename T, typename RT>
static int launch_q8_norm_few_shape(const Q8BwdArgs& a, bool is_rms, const Q8Shape& shape, bool tail, dim3 grid, int sums, hipStream_t s) {
#define HK_Q8_FEW(NV)                                                                                                \
  do {                                                                                                               \
    if (a.dx_in) {                                                                                                   \
      if (tail) launch_q8_norm_few<T, RT, NV, true, kTail>(a, is_rms, grid, sums, s);                                \
      else launch_q8_norm_few<T, RT, NV, true, kWhole>(a, is_rms, grid, sums, s);                                    \
    } else {                                                                                                         \
      if (tail) launch_q8_norm_few<T, RT, NV, false, kTail>(a, is_rms, grid, sums, s);                               \
      else launch_q8_norm_few<T, RT, NV, false, kWhole>(a, is_rms, grid, sums, s);                                   \
    }                                                                                                                \
  } while (0)
  switch (shape.nv) {
    case 1: HK_Q8_FEW(1); break;
    case 2: HK_Q8_FEW(2); break;
    case 4: HK_Q8_FEW(4); break;
    default:
      if constexpr (q8_vec<T, RT>() == 4) HK_Q8_FEW(8);
      else HK_REQUIRE(false, HK_ERR_UNSUPPORTED, "q8_norm: no kernel for %d vectors a thread", shape.nv);
      break;
  }
#undef HK_Q8_FEW
  return launch_check("q8_norm_bwd_few_kernel");
}
template <typename T, typename RT>
static int q8_norm_few(Q8BwdArgs a, bool is_rms, const Q8Shape& shape, void* dgamma, void* dbeta, hipStream_t s) {
  constexpr int VEC = q8_vec<T, RT>();
  a.part_dgamma = static_cast<float*>(dgamma);
  a.part_dbeta = static_cast<float*>(dbeta);
  const bool tail = a.cols != shape.nv * shape.lanes * VEC;
  const int strips = (a.blocks * kQ8Block + 8 * VEC - 1) / (8 * VEC), rpb = kSmallThreads / shape.lanes;
  if (a.few == 2) {   // the sums first: dx may lie over what they are made of
    if (dgamma || dbeta) {
      const int rc = launch_q8_norm_few_shape<T, RT>(a, is_rms, shape, tail, dim3(unsigned(strips)), strips, s);
      if (rc != HK_OK) return rc;
    }
    const int64_t at_once = rows_of_a_launch(kSmallThreads) * rpb;
    for (int64_t r = 0; r < a.rows; r += at_once) {
      Q8BwdArgs b = a;
      b.rows = int(std::min<int64_t>(at_once, a.rows - r));
      b.dz = static_cast<const T*>(a.dz) + r * a.dz_pitch;
      b.dx0 = static_cast<T*>(a.dx0) + r * a.dx_pitch;
      if (b.dx_in) b.dx_in = static_cast<const RT*>(a.dx_in) + r * a.dxin_pitch;
      if (b.dres) b.dres = static_cast<RT*>(a.dres) + r * a.dres_pitch;
      b.q = a.q + r * int64_t(a.blocks) * kQ8Block;
      b.scale = a.scale + r * a.blocks;
      b.rs = a.rs + r;
      if (b.mu) b.mu = a.mu + r;
      const int rc = launch_q8_norm_few_shape<T, RT>(b, is_rms, shape, tail, dim3(unsigned((b.rows + rpb - 1) / rpb)), 0, s);
      if (rc != HK_OK) return rc;
    }
    return HK_OK;
  }
  return launch_q8_norm_few_shape<T, RT>(a, is_rms, shape, tail, dim3(unsigned(strips + (a.rows + rpb - 1) / rpb)), strips, s);
}

// the partial rows folded into dgamma / dbeta (blockIdx.y picks which)
template <typename T, int LANES>
__global__ __launch_bounds__(fold_threads(LANES))
void q8_norm_fold_kernel(const float* part0, const float* part1, T* out0, T* out1, int nparts, int cols, int pitch) {
  const float s = fold_partial_rows<LANES>(blockIdx.y == 0 ? part0 : part1, nparts, pitch, int(blockIdx.x));
  const int c = int(blockIdx.x) * (4 * LANES) + int(threadIdx.x);
  if (int(threadIdx.x) < 4 * LANES && c < cols) Cvt<T>::store((blockIdx.y == 0 ? out0 : out1) + c, s);
}

template <typename T, typename RT, int NV, int LPR, int TAIL>
static void launch_q8_norm_fwd(const Q8FwdArgs& a, bool is_rms, hipStream_t s) {
  const dim3 grid{unsigned((a.rows + Q8Group<LPR>::kRows - 1) / Q8Group<LPR>::kRows)}, block{LPR ? 256u : unsigned(a.threads)};
  // four workgroups of 256 threads to a compute unit where a 16-bit residual comes along: more of them read and write more rows
  // at once than memory takes well (RMSNorm of 32768 x 4096 bf16: 202 us without the limit, 191 with it)
  size_t lds = 0;
  if (a.residual && LPR == 0 && a.threads == 256 && q8_vec<T, RT>() == 8) lds_bytes_for_residency(4, 256, &lds);
  profile_before(s);
  if (a.residual) {
    if (is_rms) HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, true, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, true, false, TAIL>), grid, block, lds, s, a);
  } else {
    if (is_rms) HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, false, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_fwd_kernel<T, RT, NV, LPR, false, false, TAIL>), grid, block, lds, s, a);
  }
  profile_after(s);
}
template <typename T, typename RT, int NV, int LPR, int MAXT, int TAIL>
static void launch_q8_norm_bwd(const Q8BwdArgs& a, bool is_rms, hipStream_t s) {
  const dim3 grid{unsigned(a.grid)}, block{LPR ? 256u : unsigned(a.threads)};
  const size_t lds = LPR ? size_t(Q8Group<LPR>::kRows) * a.blocks * kQ8Block * sizeof(float) : 0;
  profile_before(s);
  if (a.dx_in) {
    if (is_rms) HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, true, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, true, false, TAIL>), grid, block, lds, s, a);
  } else {
    if (is_rms) HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, false, true, TAIL>), grid, block, lds, s, a);
    else HK_LAUNCH((q8_norm_bwd_kernel<T, RT, NV, LPR, MAXT, false, false, TAIL>), grid, block, lds, s, a);
  }
  profile_after(s);
}

// whether rows begin on odd elements of 16 bits
static inline bool odd_rows(const void* rows, int64_t pitch) {
  return rows && ((pitch & 1) || (reinterpret_cast<uintptr_t>(rows) & 2u));
}
// WHAT: 0 forward, 1 backward
template <typename T, typename RT, int WHAT, typename A>
static int launch_q8_norm(const A& a, bool is_rms, const Q8Shape& shape, hipStream_t s) {
  const bool tail = a.cols != shape.nv * shape.lanes * q8_vec<T, RT>();   // a lane's vector may lie outside the row
  // rows that begin on odd elements of 16 bits, where a workgroup holds a row (us as any row / so: LayerNorm of 9000 x 3579 bf16,
  // forward 34.5 / 33.0, with a residual 63.3 / 58.2, backward with an upstream gradient 69.6 / 61.2; not where a wavefront holds
  // it, 8192 x 1021 fp16 forward 9.7 / 10.4, nor at 8-byte loads beside fp32, 9000 x 3579 72.4 / 73.3)
  bool odd = false;
  if constexpr (q8_vec<T, RT>() == 8) {
    if constexpr (WHAT == 0) odd = odd_rows(a.x0, a.x0_pitch) || odd_rows(a.residual, a.res_pitch);
    else odd = odd_rows(a.dz, a.dz_pitch) || odd_rows(a.dx_in, a.dxin_pitch);
  }
#define HK_Q8_TAIL(NV, LPR, TAIL)                                                                    \
  do {                                                                                               \
    constexpr int kMost = LPR ? 256 : 512;                                                           \
    if constexpr (WHAT == 0) launch_q8_norm_fwd<T, RT, NV, LPR, TAIL>(a, is_rms, s);                 \
    else if (LPR == 0 && a.threads > kMost) launch_q8_norm_bwd<T, RT, NV, LPR, LPR ? kMost : 1024, TAIL>(a, is_rms, s); \
    else launch_q8_norm_bwd<T, RT, NV, LPR, kMost, TAIL>(a, is_rms, s);                              \
  } while (0)
#define HK_Q8(NV, LPR)                                                                               \
  do {                                                                                               \
    if (odd && LPR == 0) {                                                                           \
      if constexpr (LPR == 0 && q8_vec<T, RT>() == 8) HK_Q8_TAIL(NV, LPR, kOdd);                     \
    } else if (tail) HK_Q8_TAIL(NV, LPR, kTail);                                                            \
    else HK_Q8_TAIL(NV, LPR, kWhole);                                                                \
  } while (0)
  switch (shape.lanes) {
    case 8:
      if (a.cols < q8_vec<T, RT>()) HK_Q8_TAIL(1, 8, kShort);
      else HK_Q8(1, 8);
      break;
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
        case 1:   // (where the shapes' rules give one)
          if constexpr (WHAT == 1 && q8_vec<T, RT>() == 8) HK_Q8(1, 0);
          else HK_REQUIRE(false, HK_ERR_UNSUPPORTED, "q8_norm: no kernel for %d vectors a thread", shape.nv);
          break;
        case 2: HK_Q8(2, 0); break;
        case 4:   // (the backward of wider rows takes another way)
          if constexpr (WHAT == 0 || q8_vec<T, RT>() == 4) HK_Q8(4, 0);
          else HK_REQUIRE(false, HK_ERR_UNSUPPORTED, "q8_norm: no kernel for %d vectors a thread", shape.nv);
          break;
        default:
          if constexpr (WHAT == 0 && q8_vec<T, RT>() == 4) HK_Q8(8, 0);
          else HK_REQUIRE(false, HK_ERR_UNSUPPORTED, "q8_norm: no kernel for %d vectors a thread", shape.nv);
          break;
      }
  }
#undef HK_Q8
#undef HK_Q8_TAIL
  return launch_check(WHAT == 0 ? "q8_norm_fwd_kernel" : "q8_norm_bwd_kernel");
}

template <typename T, typename RT>
static int q8_norm_fwd_runs(const Q8FwdArgs& a, bool is_rms, const Q8Shape& shape, hipStream_t s) {
  const int64_t at_once = rows_of_a_launch(shape.lanes);
  for (int64_t r = 0; r < a.rows; r += at_once) {
    Q8FwdArgs b = a;
    b.rows = int(std::min<int64_t>(at_once, a.rows - r));
    b.x0 = static_cast<const T*>(a.x0) + r * a.x0_pitch;
    b.z = static_cast<T*>(a.z) + r * a.z_pitch;
    if (b.residual) b.residual = static_cast<const RT*>(a.residual) + r * a.res_pitch;
    if (b.x_out) b.x_out = static_cast<RT*>(a.x_out) + r * a.xout_pitch;
    b.q = a.q + r * int64_t(a.blocks) * kQ8Block;
    b.scale = a.scale + r * a.blocks;
    b.mu = a.mu + r;
    b.rs = a.rs + r;
    const int rc = launch_q8_norm<T, RT, 0>(b, is_rms, shape, s);
    if (rc != HK_OK) return rc;
  }
  return HK_OK;
}
template <typename T>
int q8_norm_fwd_typed(const Q8FwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (rtype == HK_FLOAT32) return q8_norm_fwd_runs<T, float>(a, is_rms, shape, s);
  }
  return q8_norm_fwd_runs<T, T>(a, is_rms, shape, s);
}
template <typename T>
int q8_norm_bwd_typed(const Q8BwdArgs& a, int rtype, bool is_rms, const Q8Shape& shape, void* dgamma, void* dbeta,
                      hipStream_t s) {
  int rc;
  if (a.few) {
    if constexpr (sizeof(T) == 2) {
      if (rtype == HK_FLOAT32) return q8_norm_few<T, float>(a, is_rms, shape, dgamma, dbeta, s);
    }
    return q8_norm_few<T, T>(a, is_rms, shape, dgamma, dbeta, s);
  }
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
