// Activations kept in 8 bits (hk_q8.h): packing, unpacking, a norm's output from its kept input, and the entry points of
// the norm whose kernels the per-type files hold.
#include "hk_q8.h"

#include <algorithm>

namespace hk {

// ---------------------------------------------------------------------------
// Element-wise kernels: a thread takes one vector of VEC columns; vectors are counted over all rows, whole blocks of 32
// columns a row.
// ---------------------------------------------------------------------------
struct Q8FlatArgs {
  const void* x;         // pack: the rows; unpack: unused
  void* out;             // unpack: the rows
  int8_t* q;
  uint8_t* scale;
  const void *gamma, *beta;
  const float *mu, *rs;  // of a norm's output; rs == null: the values themselves
  int64_t pitch;
  uint32_t nvec, row_vecs, magic;   // v / row_vecs == (v * magic) >> (32 + shift)
  uint32_t rows;
  int cols;
  uint16_t threads;
  uint8_t shift, is_rms;
};
static_assert(sizeof(Q8FlatArgs) <= kCheapArgs, "");

struct Q8Place {
  uint32_t row;
  int col;
};
__device__ __forceinline__ Q8Place q8_place(const Q8FlatArgs& a, uint32_t v, int vec) {
  const uint32_t row = __umulhi(v, a.magic) >> a.shift;
  return {row, int(v - row * a.row_vecs) * vec};
}

// Packing and unpacking, two vectors a thread in workgroups of 256; bound by memory.  One vector and 64 threads / so, us (one set
// of arrays, in part from a cache), of what
// the bytes take: packing 32768 x 4096 bf16 67 / 58.6 of 59.8, 14549 x 3579 fp32 45 / 38 of 38.5; unpacking the same 62.5 / 64
// and 52 / 44.
template <typename T, int TAIL, int U>
__global__ __launch_bounds__(256)
void q8_pack_kernel(Q8FlatArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Words = Q8Words<VEC>;
  // (a block's lanes are all there or none: rows are whole blocks)
  const uint32_t v0 = blockIdx.x * uint32_t(U * a.threads) + threadIdx.x;
  Q8Place at[U];
  RowVec<T, VEC, TAIL> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t v = v0 + u * a.threads;
    at[u] = q8_place(a, v < a.nvec ? v : a.nvec - 1, VEC);
    x[u].load(static_cast<const T*>(a.x) + int64_t(at[u].row) * a.pitch, at[u].col, a.cols);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t v = v0 + u * a.threads;
    float f[VEC];
    x[u].floats(f, at[u].col, a.cols);
    const uint32_t e = q8_exponent<VEC>(f);
    if (v < a.nvec) {
      __builtin_nontemporal_store(Words::encode(f, q8_factor(e)), reinterpret_cast<typename Words::type*>(a.q) + v);
      if (v % LPB == 0) a.scale[v / LPB] = uint8_t(e);
    }
  }
}

template <typename T, int TAIL, int U>
__global__ __launch_bounds__(256)
void q8_unpack_kernel(Q8FlatArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Words = Q8Words<VEC>;
  const uint32_t v0 = blockIdx.x * uint32_t(U * a.threads) + threadIdx.x;
  typename Words::type w[U];
  uint32_t e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t v = min(v0 + u * a.threads, a.nvec - 1);
    w[u] = __builtin_nontemporal_load(reinterpret_cast<const typename Words::type*>(a.q) + v);
    e[u] = a.scale[v / LPB];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t v = v0 + u * a.threads;
    if (v >= a.nvec) return;
    const Q8Place at = q8_place(a, v, VEC);
    float f[VEC];
    Words::numbers(w[u], f);
    const float step = q8_step(e[u]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] *= step;
    store_row_floats<T, VEC, TAIL>(static_cast<T*>(a.out) + int64_t(at.row) * a.pitch, at.col, a.cols, f);
  }
}

// A norm's output from its kept input, gamma rs (x8 - [mu]) + beta: a thread takes the same columns of U rows, for which it
// reads gamma and beta once (LayerNorm of 32768 x 4096 bf16, of 59.8 us that the bytes take: one row a thread 93, four
// neighbouring vectors of a row 82, four rows 69).
template <typename T, int TAIL, int U>
__global__ __launch_bounds__(256)
void q8_norm_out_kernel(Q8FlatArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Words = Q8Words<VEC>;
  const uint32_t v = blockIdx.x * uint32_t(a.threads) + threadIdx.x;
  const Q8Place at = q8_place(a, v, VEC);
  const uint32_t row0 = at.row * U, c = uint32_t(at.col) / VEC;
  if (row0 >= a.rows) return;
  typename Words::type w[U];
  uint32_t e[U];
  float rs[U], mu[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = min(row0 + u, a.rows - 1);
    const int64_t i = int64_t(r) * a.row_vecs + c;
    w[u] = __builtin_nontemporal_load(reinterpret_cast<const typename Words::type*>(a.q) + i);
    e[u] = a.scale[i / LPB];
    rs[u] = a.rs[r];
    mu[u] = a.is_rms ? 0.f : a.mu[r];
  }
  float g[VEC], b[VEC];
  RowVec<T, VEC, TAIL> p;
  if (a.gamma) { p.template load<true>(static_cast<const T*>(a.gamma), at.col, a.cols); p.floats(g, at.col, a.cols); }   // uniform
  if (a.beta) { p.template load<true>(static_cast<const T*>(a.beta), at.col, a.cols); p.floats(b, at.col, a.cols); }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row0 + u >= a.rows) return;
    float f[VEC];
    Words::numbers(w[u], f);
    const float scale = rs[u] * q8_step(e[u]), shift = a.is_rms ? 0.f : -rs[u] * mu[u];   // (a power of two: exact)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float n = fmaf(f[j], scale, shift);
      f[j] = a.gamma ? (a.beta ? fmaf(g[j], n, b[j]) : g[j] * n) : (a.beta ? n + b[j] : n);
    }
    store_row_floats<T, VEC, TAIL>(static_cast<T*>(a.out) + int64_t(row0 + u) * a.pitch, at.col, a.cols, f);
  }
}

// f(args) for runs of rows whose vectors fit 31 bits
template <typename F>
static int each_q8_run(Q8FlatArgs a, int64_t rows, int64_t cols, size_t es, int per_thread, bool down, F&& f) {
  const int vec = int(16 / es);
  const int64_t blocks = q8_blocks(cols), row_vecs = blocks * (kQ8Block / vec);
  a.row_vecs = uint32_t(row_vecs);
  a.cols = int(cols);
  // 2^s >= d: with m = floor(2^(31 + s) / d) + 1, v m exceeds v 2^(31 + s) / d by less than 2^(31 + s) / d for v < 2^31
  int s = 0;
  while ((int64_t(1) << s) < row_vecs) ++s;   // (row_vecs >= 4)
  a.magic = uint32_t((uint64_t(1) << (31 + s)) / uint64_t(row_vecs) + 1);
  a.shift = uint8_t(s - 1);
  const int64_t at_once = std::max<int64_t>(1, 0x7fffff00LL / row_vecs);
  for (int64_t r = 0; r < rows; r += at_once) {
    const int64_t n = std::min(at_once, rows - r);
    Q8FlatArgs b = a;
    b.nvec = uint32_t(n * row_vecs);
    b.rows = uint32_t(n);
    if (b.x) b.x = static_cast<const char*>(a.x) + r * a.pitch * int64_t(es);
    if (b.out) b.out = static_cast<char*>(a.out) + r * a.pitch * int64_t(es);
    b.q = a.q + r * blocks * kQ8Block;
    b.scale = a.scale + r * blocks;
    if (b.mu) b.mu = a.mu + r;
    if (b.rs) b.rs = a.rs + r;
    // per_thread vectors of neighbouring columns or, `down`, of neighbouring rows
    const int64_t vecs = down ? (n + per_thread - 1) / per_thread * row_vecs : n * row_vecs;
    const int64_t per = (down ? 1 : per_thread) * int64_t(a.threads);
    const int rc = f(b, dim3(unsigned((vecs + per - 1) / per)));
    if (rc != HK_OK) return rc;
  }
  return HK_OK;
}

// f(args, rows, cols) for all rows at once, or for runs of whole blocks of each row where the offsets inside one pass 32 bits
template <typename F>
static int each_q8_piece(const Q8FlatArgs& a, int64_t rows, int64_t cols, size_t es, F&& f) {
  constexpr int64_t kRun = int64_t(1) << 28;
  if (cols <= kRun) return f(a, rows, cols);
  for (int64_t r = 0; r < rows; ++r) {
    for (int64_t c = 0; c < cols; c += kRun) {
      Q8FlatArgs b = a;
      if (b.x) b.x = static_cast<const char*>(a.x) + (r * a.pitch + c) * int64_t(es);
      if (b.out) b.out = static_cast<char*>(a.out) + (r * a.pitch + c) * int64_t(es);
      b.q = a.q + r * q8_blocks(cols) * kQ8Block + c;
      b.scale = a.scale + r * q8_blocks(cols) + c / kQ8Block;
      const int rc = f(b, 1, std::min(kRun, cols - c));
      if (rc != HK_OK) return rc;
    }
  }
  return HK_OK;
}

#define HK_Q8_LAUNCH(KERNEL)                                                                          \
  do {                                                                                                \
    profile_before(s);                                                                                \
    if (cols % kQ8Block == 0) HK_LAUNCH((KERNEL<T, kWhole, U>), grid, dim3(b.threads), 0, s, b);      \
    else if (cols >= VecIO<T>::N) HK_LAUNCH((KERNEL<T, kTail, U>), grid, dim3(b.threads), 0, s, b);   \
    else HK_LAUNCH((KERNEL<T, kShort, U>), grid, dim3(b.threads), 0, s, b);                           \
    profile_after(s);                                                                                 \
  } while (0)
template <typename T>
static int q8_pack_typed(Q8FlatArgs a, int64_t rows, int64_t cols, hipStream_t s) {
  constexpr int U = 2;
  a.threads = 256;
  return each_q8_run(a, rows, cols, sizeof(T), U, false, [&](const Q8FlatArgs& b, dim3 grid) {
    HK_Q8_LAUNCH(q8_pack_kernel);
    return launch_check("q8_pack_kernel");
  });
}
template <typename T>
static int q8_unpack_typed(Q8FlatArgs a, int64_t rows, int64_t cols, hipStream_t s) {
  constexpr int U = 2;
  a.threads = 256;
  return each_q8_run(a, rows, cols, sizeof(T), U, false, [&](const Q8FlatArgs& b, dim3 grid) {
    HK_Q8_LAUNCH(q8_unpack_kernel);
    return launch_check("q8_unpack_kernel");
  });
}
template <typename T>
static int q8_norm_out_typed(Q8FlatArgs a, int64_t rows, int64_t cols, hipStream_t s) {
  constexpr int U = 4;
  a.threads = 256;
  return each_q8_run(a, rows, cols, sizeof(T), U, true, [&](const Q8FlatArgs& b, dim3 grid) {
    HK_Q8_LAUNCH(q8_norm_out_kernel);
    return launch_check("q8_norm_out_kernel");
  });
}
#undef HK_Q8_LAUNCH

// the fewest lanes of a wavefront up to one vector each, up to four vectors in a wavefront of their own
static bool q8_wave_shape(int64_t n, Q8Shape* s) {
  if (n <= 32) *s = {n <= 8 ? 8 : n <= 16 ? 16 : 32, 1};
  else if (n <= 256) *s = {64, n <= 64 ? 1 : n <= 128 ? 2 : 4};
  else return false;
  return true;
}
// a workgroup of at most `threads` threads with one of 2, 4, 8 vectors each, or of 1024
static Q8Shape q8_group_shape(int64_t n, int max_nv, int threads) {
  for (int nv = 2; nv < max_nv; nv *= 2) {
    const int64_t t = ((n + nv - 1) / nv + 63) / 64 * 64;
    if (t <= threads) return {int(t), nv};
  }
  return {int(((n + max_nv - 1) / max_nv + 63) / 64 * 64), max_nv};
}
Q8Shape q8_fwd_shape(int64_t cols, int vec) {
  const int64_t n = q8_blocks(cols) * (kQ8Block / vec);   // vectors of a row, whole blocks
  Q8Shape s;
  return q8_wave_shape(n, &s) ? s : q8_group_shape(n, vec == 4 ? 8 : 4, 512);
}
// One vector a thread where 1024 threads hold the row in 16-byte vectors of 16-bit elements: twice the wavefronts, whose
// loads and reductions hide one another (LayerNorm of 16384 x 5120 bf16, 320 threads x 2 / 640 x 1: 88.4 / 79.9 us; RMSNorm of
// 32768 x 4096 with an upstream gradient, 256 x 2 / 512 x 1: 200 / 196).  Of more, up to 1024 threads before a thread takes twice
// as many columns (RMSNorm of 4096 x 10240 bf16 with an upstream gradient, 320 x 4 / 640 x 2: 100 / 79, without 47 / 44, of 12289
// 277 / 174 and 96 / 71; LayerNorm without one 69 / 77).
Q8Shape q8_bwd_shape(int64_t cols, int vec) {
  const int64_t n = q8_blocks(cols) * (kQ8Block / vec);
  Q8Shape s;
  if (q8_wave_shape(n, &s)) return s;
  if (vec == 8 && n <= 1024) return {int((n + 63) / 64 * 64), 1};
  return q8_group_shape(n, vec == 4 ? 8 : 4, 1024);
}
// As many workgroups as fill a compute unit to 1024 threads; to 512 where an upstream gradient comes in and the rows' loads are
// half as many again (RMSNorm of 32768 x 4096 bf16, one / two / four workgroups of 512 threads to a compute unit: with it 196 /
// 205 / 208 us, without 125 / 115 / 130), and where a workgroup would have fewer than 16 rows, whose partial sums then weigh
// more than what is gained.
int q8_bwd_grid(int64_t rows, const Q8Shape& shape, bool extra) {
  const int64_t per = shape.lanes <= kWave ? 256 / shape.lanes : 1;
  const int64_t threads = shape.lanes <= kWave ? 256 : shape.lanes, cus = device_cu_count();
  int64_t most = cus * std::max<int64_t>(1, 1024 / threads);
  if ((extra && shape.lanes > kWave) || rows < 16 * most * per) most = cus * std::max<int64_t>(1, 512 / threads);
  return int(std::min((rows + per - 1) / per, most));
}

// Up to how many rows the column sums are formed from the rows themselves, in the launch that forms dx (us, so / with partial
// rows and a fold: LayerNorm of 768 x 4096 bf16 6.4 / 17.4, 1024 8.0 / 18.5, of 1024 x 1024 6.9 / 6.8; with an upstream gradient in
// fp32 768 x 4096 11.6 / 12.7, 1024 16.1 / 14.9).
static int64_t q8_few_rows(bool extra) { return extra ? 768 : 1024; }
// Rows whose backward is two launches, the column sums from the rows themselves, then dx: where a thread would keep the sums of
// more than 16 columns, which spill, or of 16 beside an upstream gradient, in the half of the registers that more than 512
// threads leave (persistent / two launches, us, 4096 rows: 20480 bf16 508 / 169, with an upstream gradient 785 / 208; 12288
// fp32 with one 224 / 207, bf16 with one in fp32 203 / 164, LayerNorm bf16 with one 130 / 119; but RMSNorm 89 / 117 and without
// one 52 / 96).
static bool q8_wide(const Q8Shape& shape, int vec, bool extra, bool is_rms) {
  const int columns = shape.nv * vec;
  return shape.lanes > kWave && (columns > 16 || (columns == 16 && shape.lanes > 512 && extra && (vec == 4 || !is_rms)));
}
// nothing that is written may lie over what is read there
static bool q8_apart(const Q8BwdArgs& a, const void* dgamma, const void* dbeta, size_t es, size_t rs) {
  const int64_t rows = a.rows, cols = a.cols;
  auto rows_of = [&](const void* p, int64_t pitch, size_t size) { return Span{p, ((rows - 1) * pitch + cols) * int64_t(size)}; };
  return apart({rows_of(a.dx0, a.dx_pitch, es), rows_of(a.dres, a.dres_pitch, rs), Span{dgamma, cols * int64_t(es)},
                Span{dbeta, cols * int64_t(es)}},
               {rows_of(a.dz, a.dz_pitch, es), rows_of(a.dx_in, a.dxin_pitch, rs), Span{a.gamma, cols * int64_t(es)},
                Span{a.q, rows * a.blocks * kQ8Block}, Span{a.scale, rows * a.blocks}, Span{a.mu, rows * 4}, Span{a.rs, rows * 4}});
}

constexpr int64_t kQ8MaxRow = int64_t(1) << 40;   // columns of a row to pack
static bool q8_dtype(int dtype) { return dtype == HK_FLOAT32 || dtype == HK_BFLOAT16 || dtype == HK_FLOAT16; }

#define HK_Q8_TYPED(dtype, call)                      \
  ((dtype) == HK_FLOAT32 ? call(float) : (dtype) == HK_BFLOAT16 ? call(bf16) : call(fp16))

} // namespace hk

using namespace hk;

extern "C" {

int hk_q8_pack(int dtype, const void* x, int64_t x_pitch, int8_t* q, uint8_t* scale, int64_t rows, int64_t cols,
               hkStream_t stream) {
  HK_REQUIRE(q8_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_q8_pack: not implemented for dtype %d", dtype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && cols <= kQ8MaxRow, HK_ERR_INVALID, "hk_q8_pack: bad shape");
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(x && q && scale, HK_ERR_INVALID, "hk_q8_pack: null input/output");
  HK_REQUIRE(x_pitch >= cols, HK_ERR_INVALID, "hk_q8_pack: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_q8_pack: q must lie on an 8-byte boundary");
  Q8FlatArgs a{};
  a.x = x; a.pitch = x_pitch; a.q = q; a.scale = scale;
#define HK_CALL_PACK(T) q8_pack_typed<T>(b, n, m, as_hip(stream))
  return each_q8_piece(a, rows, cols, dtype_size(dtype), [&](const Q8FlatArgs& b, int64_t n, int64_t m) {
    return HK_Q8_TYPED(dtype, HK_CALL_PACK);
  });
#undef HK_CALL_PACK
}

int hk_q8_unpack(int dtype, const int8_t* q, const uint8_t* scale, void* out, int64_t out_pitch, int64_t rows, int64_t cols,
                 hkStream_t stream) {
  HK_REQUIRE(q8_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_q8_unpack: not implemented for dtype %d", dtype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && cols <= kQ8MaxRow, HK_ERR_INVALID, "hk_q8_unpack: bad shape");
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(out && q && scale, HK_ERR_INVALID, "hk_q8_unpack: null input/output");
  HK_REQUIRE(out_pitch >= cols, HK_ERR_INVALID, "hk_q8_unpack: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_q8_unpack: q must lie on an 8-byte boundary");
  Q8FlatArgs a{};
  a.out = out; a.pitch = out_pitch; a.q = const_cast<int8_t*>(q); a.scale = const_cast<uint8_t*>(scale);
#define HK_CALL_UNPACK(T) q8_unpack_typed<T>(b, n, m, as_hip(stream))
  return each_q8_piece(a, rows, cols, dtype_size(dtype), [&](const Q8FlatArgs& b, int64_t n, int64_t m) {
    return HK_Q8_TYPED(dtype, HK_CALL_UNPACK);
  });
#undef HK_CALL_UNPACK
}

int hk_add_ln_q8_out(int itype, const int8_t* q, const uint8_t* scale, const float* mu, const float* rsigma, const void* gamma,
                     const void* beta, void* z, int64_t z_pitch, int64_t rows, int64_t cols, int is_rms_norm,
                     hkStream_t stream) {
  HK_REQUIRE(q8_dtype(itype), HK_ERR_UNSUPPORTED, "hk_add_ln_q8_out: not implemented for dtype %d", itype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && cols <= kQ8MaxCols, HK_ERR_INVALID, "hk_add_ln_q8_out: bad shape (at most %d columns)",
             kQ8MaxCols);
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(z && q && scale && rsigma && (mu || is_rms_norm), HK_ERR_INVALID, "hk_add_ln_q8_out: null input/output");
  HK_REQUIRE(z_pitch >= cols, HK_ERR_INVALID, "hk_add_ln_q8_out: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_add_ln_q8_out: q must lie on an 8-byte boundary");
  Q8FlatArgs a{};
  a.out = z; a.pitch = z_pitch; a.q = const_cast<int8_t*>(q); a.scale = const_cast<uint8_t*>(scale);
  a.gamma = gamma; a.beta = beta; a.mu = mu; a.rs = rsigma; a.is_rms = uint8_t(is_rms_norm != 0);
#define HK_CALL_OUT(T) q8_norm_out_typed<T>(a, rows, cols, as_hip(stream))
  return HK_Q8_TYPED(itype, HK_CALL_OUT);
#undef HK_CALL_OUT
}

int hk_add_ln_q8_fwd(int itype, int rtype, const void* x0, int64_t x0_pitch, const void* residual, int64_t residual_pitch,
                     const void* gamma, const void* beta, void* z, int64_t z_pitch, void* x_out, int64_t x_out_pitch,
                     int8_t* q, uint8_t* scale, float* mu, float* rsigma, int64_t rows, int64_t cols, float eps,
                     int is_rms_norm, hkStream_t stream) {
  HK_REQUIRE(q8_dtype(itype) && (rtype == itype || rtype == HK_FLOAT32), HK_ERR_UNSUPPORTED,
             "hk_add_ln_q8_fwd: not implemented for dtype %d with residual dtype %d", itype, rtype);
  HK_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && cols >= 0 && cols <= kQ8MaxCols, HK_ERR_INVALID,
             "hk_add_ln_q8_fwd: bad shape (at most %d columns)", kQ8MaxCols);
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(x0 && z && q && scale && mu && rsigma, HK_ERR_INVALID, "hk_add_ln_q8_fwd: null input/output");
  HK_REQUIRE(x0_pitch >= cols && z_pitch >= cols && (!residual || residual_pitch >= cols) && (!x_out || x_out_pitch >= cols),
             HK_ERR_INVALID, "hk_add_ln_q8_fwd: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_add_ln_q8_fwd: q must lie on an 8-byte boundary");
  Q8FwdArgs a{};
  a.x0 = x0; a.x0_pitch = x0_pitch; a.residual = residual; a.res_pitch = residual_pitch; a.gamma = gamma; a.beta = beta;
  a.z = z; a.z_pitch = z_pitch; a.x_out = x_out; a.xout_pitch = x_out_pitch; a.q = q; a.scale = scale; a.mu = mu; a.rs = rsigma;
  a.rows = int(rows); a.cols = int(cols); a.blocks = int(q8_blocks(cols)); a.eps = eps; a.inv_cols = 1.0f / float(cols);
  if (!residual && !x_out) rtype = itype;
  const Q8Shape shape = q8_fwd_shape(cols, rtype == HK_FLOAT32 ? 4 : 8);
  a.threads = uint16_t(shape.lanes);
#define HK_CALL_FWD(T) q8_norm_fwd_typed<T>(a, rtype, is_rms_norm != 0, shape, as_hip(stream))
  return HK_Q8_TYPED(itype, HK_CALL_FWD);
#undef HK_CALL_FWD
}

int hk_add_ln_q8_bwd_workspace_bytes(int64_t rows, int64_t cols, size_t* bytes) {
  HK_REQUIRE(bytes && rows >= 0 && rows <= 0x7fffffffLL && cols >= 0 && cols <= kQ8MaxCols, HK_ERR_INVALID,
             "hk_add_ln_q8_bwd_workspace_bytes: bad argument");
  *bytes = 0;
  if (rows == 0 || cols == 0) return HK_OK;
  // (an upstream gradient never asks for more)
  const int parts = std::max(q8_bwd_grid(rows, q8_bwd_shape(cols, 8), false), q8_bwd_grid(rows, q8_bwd_shape(cols, 4), false));
  *bytes = 2 * size_t(parts) * size_t(q8_blocks(cols)) * kQ8Block * sizeof(float);
  return HK_OK;
}

int hk_add_ln_q8_bwd(int itype, int rtype, const void* dz, int64_t dz_pitch, const void* dx_in, int64_t dx_in_pitch,
                     const int8_t* q, const uint8_t* scale, const float* mu, const float* rsigma, const void* gamma, void* dx0,
                     int64_t dx0_pitch, void* dresidual, int64_t dresidual_pitch, void* dgamma, void* dbeta, int64_t rows,
                     int64_t cols, int is_rms_norm, void* workspace, size_t workspace_bytes, hkStream_t stream) {
  HK_REQUIRE(q8_dtype(itype) && (rtype == itype || rtype == HK_FLOAT32), HK_ERR_UNSUPPORTED,
             "hk_add_ln_q8_bwd: not implemented for dtype %d with residual dtype %d", itype, rtype);
  HK_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && cols >= 0 && cols <= kQ8MaxCols, HK_ERR_INVALID,
             "hk_add_ln_q8_bwd: bad shape (at most %d columns)", kQ8MaxCols);
  HK_REQUIRE(!is_rms_norm || !dbeta, HK_ERR_INVALID, "hk_add_ln_q8_bwd: an RMSNorm has no beta");
  if (cols == 0) return HK_OK;
  hipStream_t s = as_hip(stream);
  if (rows == 0) {   // the empty sums
    for (void* out : {dgamma, dbeta}) {
      const int rc = out ? hk_memset(out, 0, size_t(cols) * dtype_size(itype), stream) : HK_OK;
      if (rc != HK_OK) return rc;
    }
    return HK_OK;
  }
  HK_REQUIRE(dz && q && scale && rsigma && dx0 && (mu || is_rms_norm), HK_ERR_INVALID, "hk_add_ln_q8_bwd: null input/output");
  HK_REQUIRE(dz_pitch >= cols && dx0_pitch >= cols && (!dx_in || dx_in_pitch >= cols) &&
             (!dresidual || dresidual_pitch >= cols), HK_ERR_INVALID, "hk_add_ln_q8_bwd: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_add_ln_q8_bwd: q must lie on an 8-byte boundary");
  if (!dx_in && !dresidual) rtype = itype;
  const int vec = rtype == HK_FLOAT32 ? 4 : 8;
  const Q8Shape shape = q8_bwd_shape(cols, vec);
  Q8BwdArgs a{};
  a.blocks = int(q8_blocks(cols));
  a.grid = q8_bwd_grid(rows, shape, dx_in != nullptr);
  const size_t part = size_t(a.grid) * size_t(a.blocks) * kQ8Block;   // floats
  const size_t need = part * sizeof(float) * ((dgamma != nullptr) + (dbeta != nullptr));
  HK_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), HK_ERR_WORKSPACE,
             "hk_add_ln_q8_bwd: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  HK_REQUIRE(need == 0 || aligned16(workspace), HK_ERR_INVALID, "hk_add_ln_q8_bwd: the workspace must lie on a 16-byte boundary");
  float* ws = static_cast<float*>(workspace);
  a.part_dgamma = dgamma ? ws : nullptr;
  a.part_dbeta = dbeta ? ws + (dgamma ? part : 0) : nullptr;
  a.dz = dz; a.dz_pitch = dz_pitch; a.dx_in = dx_in; a.dxin_pitch = dx_in_pitch; a.gamma = gamma; a.q = q; a.scale = scale;
  a.mu = mu; a.rs = rsigma; a.dx0 = dx0; a.dx_pitch = dx0_pitch; a.dres = dresidual; a.dres_pitch = dresidual_pitch;
  a.rows = int(rows); a.cols = int(cols); a.inv_cols = 1.0f / float(cols); a.threads = uint16_t(shape.lanes);
  a.few = rows <= q8_few_rows(dx_in != nullptr) && shape.lanes >= kWave && shape.lanes <= kSmallThreads && (dgamma || dbeta) &&
          q8_apart(a, dgamma, dbeta, dtype_size(itype), dtype_size(rtype));
  if (!a.few && q8_wide(shape, vec, dx_in != nullptr, is_rms_norm != 0)) a.few = 2;
#define HK_CALL_BWD(T) q8_norm_bwd_typed<T>(a, rtype, is_rms_norm != 0, shape, dgamma, dbeta, s)
  return HK_Q8_TYPED(itype, HK_CALL_BWD);
#undef HK_CALL_BWD
}

} // extern "C"
