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
  uint32_t nvec, row_vecs;
  int cols;
  int is_rms;
};
static_assert(sizeof(Q8FlatArgs) <= kCheapArgs, "");

template <typename T, bool TAIL>
__global__ __launch_bounds__(kStreamThreads)
void q8_pack_kernel(Q8FlatArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Words = Q8Words<VEC>;
  // (a block's lanes all exist: rows are whole blocks)
  const uint32_t v = blockIdx.x * uint32_t(kStreamThreads) + threadIdx.x;
  if (v >= a.nvec) return;
  const uint32_t row = v / a.row_vecs;
  const int c = int(v - row * a.row_vecs) * VEC;
  float f[VEC];
  RowVec<T, VEC, TAIL> x;
  x.load(static_cast<const T*>(a.x) + int64_t(row) * a.pitch, c, a.cols, false);
  x.floats(f, c, a.cols);
  const uint32_t e = q8_exponent<VEC>(f);
  __builtin_nontemporal_store(Words::encode(f, q8_factor(e)), reinterpret_cast<typename Words::type*>(a.q) + v);
  if (v % LPB == 0) a.scale[v / LPB] = uint8_t(e);
}

// NORM: gamma rs (x8 - [mu]) + beta
template <typename T, bool TAIL, bool NORM>
__global__ __launch_bounds__(kStreamThreads)
void q8_unpack_kernel(Q8FlatArgs a) {
  constexpr int VEC = VecIO<T>::N, LPB = kQ8Block / VEC;
  using Words = Q8Words<VEC>;
  const uint32_t v = blockIdx.x * uint32_t(kStreamThreads) + threadIdx.x;
  if (v >= a.nvec) return;
  const uint32_t row = v / a.row_vecs;
  const int c = int(v - row * a.row_vecs) * VEC;
  const typename Words::type w = __builtin_nontemporal_load(reinterpret_cast<const typename Words::type*>(a.q) + v);
  const uint32_t e = a.scale[v / LPB];
  float f[VEC];
  Words::decode(w, e, f);
  if constexpr (NORM) {
    const float rs = a.rs[row], shift = a.is_rms ? 0.f : a.mu[row];
    float g[VEC], b[VEC];
    RowVec<T, VEC, TAIL> p;
    if (a.gamma) { p.load(static_cast<const T*>(a.gamma), c, a.cols, true); p.floats(g, c, a.cols); }   // uniform
    if (a.beta) { p.load(static_cast<const T*>(a.beta), c, a.cols, true); p.floats(b, c, a.cols); }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float n = rs * (f[j] - shift);
      f[j] = a.gamma ? (a.beta ? fmaf(g[j], n, b[j]) : g[j] * n) : (a.beta ? n + b[j] : n);
    }
  }
  store_row_floats<T, VEC, TAIL>(static_cast<T*>(a.out) + int64_t(row) * a.pitch, c, a.cols, f);
}

// f(args) for runs of rows whose vectors fit 31 bits
template <typename F>
static int each_q8_run(Q8FlatArgs a, int64_t rows, int64_t cols, size_t es, F&& f) {
  const int vec = int(16 / es);
  const int64_t blocks = q8_blocks(cols), row_vecs = blocks * (kQ8Block / vec);
  a.row_vecs = uint32_t(row_vecs);
  a.cols = int(cols);
  const int64_t at_once = std::max<int64_t>(1, 0x7fffff00LL / row_vecs);
  for (int64_t r = 0; r < rows; r += at_once) {
    const int64_t n = std::min(at_once, rows - r);
    Q8FlatArgs b = a;
    b.nvec = uint32_t(n * row_vecs);
    if (b.x) b.x = static_cast<const char*>(a.x) + r * a.pitch * int64_t(es);
    if (b.out) b.out = static_cast<char*>(a.out) + r * a.pitch * int64_t(es);
    b.q = a.q + r * blocks * kQ8Block;
    b.scale = a.scale + r * blocks;
    if (b.mu) b.mu = a.mu + r;
    if (b.rs) b.rs = a.rs + r;
    const int rc = f(b, dim3(unsigned((b.nvec + kStreamThreads - 1) / kStreamThreads)));
    if (rc != HK_OK) return rc;
  }
  return HK_OK;
}

template <typename T>
static int q8_pack_typed(const Q8FlatArgs& a, int64_t rows, int64_t cols, hipStream_t s) {
  return each_q8_run(a, rows, cols, sizeof(T), [&](const Q8FlatArgs& b, dim3 grid) {
    profile_before(s);
    if (cols % VecIO<T>::N) HK_LAUNCH((q8_pack_kernel<T, true>), grid, dim3(kStreamThreads), 0, s, b);
    else HK_LAUNCH((q8_pack_kernel<T, false>), grid, dim3(kStreamThreads), 0, s, b);
    profile_after(s);
    return launch_check("q8_pack_kernel");
  });
}
template <typename T, bool NORM>
static int q8_unpack_typed(const Q8FlatArgs& a, int64_t rows, int64_t cols, hipStream_t s) {
  return each_q8_run(a, rows, cols, sizeof(T), [&](const Q8FlatArgs& b, dim3 grid) {
    profile_before(s);
    if (cols % VecIO<T>::N) HK_LAUNCH((q8_unpack_kernel<T, true, NORM>), grid, dim3(kStreamThreads), 0, s, b);
    else HK_LAUNCH((q8_unpack_kernel<T, false, NORM>), grid, dim3(kStreamThreads), 0, s, b);
    profile_after(s);
    return launch_check("q8_unpack_kernel");
  });
}

static Q8Shape wave_or_group(int64_t cols, int vec, int wave_nv, int max_nv, int threads) {
  const int64_t n = q8_blocks(cols) * (kQ8Block / vec);   // vectors of a row, whole blocks
  if (n <= 32) return {n <= 8 ? 8 : n <= 16 ? 16 : 32, 1};
  if (n <= 64 * wave_nv) return {64, n <= 64 ? 1 : n <= 128 ? 2 : 4};
  for (int nv = 2; nv < max_nv; nv *= 2) {
    const int64_t t = ((n + nv - 1) / nv + 63) / 64 * 64;
    if (t <= threads) return {int(t), nv};
  }
  return {int(((n + max_nv - 1) / max_nv + 63) / 64 * 64), max_nv};
}
Q8Shape q8_fwd_shape(int64_t cols, int vec) { return wave_or_group(cols, vec, 4, vec == 4 ? 8 : 4, 512); }
Q8Shape q8_bwd_shape(int64_t cols, int vec) { return wave_or_group(cols, vec, 4, vec == 4 ? 8 : 4, 512); }
int q8_bwd_grid(int64_t rows, const Q8Shape& shape) {
  const int64_t per = shape.lanes <= kWave ? 256 / shape.lanes : 1;
  const int64_t threads = shape.lanes <= kWave ? 256 : shape.lanes;
  const int64_t most = device_cu_count() * std::max<int64_t>(1, 1024 / threads);
  return int(std::min((rows + per - 1) / per, most));
}

static bool q8_dtype(int dtype) { return dtype == HK_FLOAT32 || dtype == HK_BFLOAT16 || dtype == HK_FLOAT16; }

#define HK_Q8_TYPED(dtype, call)                      \
  ((dtype) == HK_FLOAT32 ? call(float) : (dtype) == HK_BFLOAT16 ? call(bf16) : call(fp16))

} // namespace hk

using namespace hk;

extern "C" {

int hk_q8_pack(int dtype, const void* x, int64_t x_pitch, int8_t* q, uint8_t* scale, int64_t rows, int64_t cols,
               hkStream_t stream) {
  HK_REQUIRE(q8_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_q8_pack: not implemented for dtype %d", dtype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && cols <= 0x7fffff00LL, HK_ERR_INVALID, "hk_q8_pack: bad shape");
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(x && q && scale, HK_ERR_INVALID, "hk_q8_pack: null input/output");
  HK_REQUIRE(x_pitch >= cols, HK_ERR_INVALID, "hk_q8_pack: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_q8_pack: q must lie on an 8-byte boundary");
  Q8FlatArgs a{};
  a.x = x; a.pitch = x_pitch; a.q = q; a.scale = scale;
#define HK_CALL_PACK(T) q8_pack_typed<T>(a, rows, cols, as_hip(stream))
  return HK_Q8_TYPED(dtype, HK_CALL_PACK);
#undef HK_CALL_PACK
}

int hk_q8_unpack(int dtype, const int8_t* q, const uint8_t* scale, void* out, int64_t out_pitch, int64_t rows, int64_t cols,
                 hkStream_t stream) {
  HK_REQUIRE(q8_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_q8_unpack: not implemented for dtype %d", dtype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && cols <= 0x7fffff00LL, HK_ERR_INVALID, "hk_q8_unpack: bad shape");
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(out && q && scale, HK_ERR_INVALID, "hk_q8_unpack: null input/output");
  HK_REQUIRE(out_pitch >= cols, HK_ERR_INVALID, "hk_q8_unpack: row pitch below the columns");
  HK_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7u) == 0, HK_ERR_INVALID, "hk_q8_unpack: q must lie on an 8-byte boundary");
  Q8FlatArgs a{};
  a.out = out; a.pitch = out_pitch; a.q = const_cast<int8_t*>(q); a.scale = const_cast<uint8_t*>(scale);
#define HK_CALL_UNPACK(T) q8_unpack_typed<T, false>(a, rows, cols, as_hip(stream))
  return HK_Q8_TYPED(dtype, HK_CALL_UNPACK);
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
  a.gamma = gamma; a.beta = beta; a.mu = mu; a.rs = rsigma; a.is_rms = is_rms_norm;
#define HK_CALL_OUT(T) q8_unpack_typed<T, true>(a, rows, cols, as_hip(stream))
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
  const Q8Shape shape = q8_fwd_shape(cols, int(16 / dtype_size(itype)));
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
  const int parts = std::max(q8_bwd_grid(rows, q8_bwd_shape(cols, 8)), q8_bwd_grid(rows, q8_bwd_shape(cols, 4)));
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
  const Q8Shape shape = q8_bwd_shape(cols, int(16 / dtype_size(itype)));
  Q8BwdArgs a{};
  a.blocks = int(q8_blocks(cols));
  a.grid = q8_bwd_grid(rows, shape);
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
#define HK_CALL_BWD(T) q8_norm_bwd_typed<T>(a, rtype, is_rms_norm != 0, shape, dgamma, dbeta, s)
  return HK_Q8_TYPED(itype, HK_CALL_BWD);
#undef HK_CALL_BWD
}

} // extern "C"
