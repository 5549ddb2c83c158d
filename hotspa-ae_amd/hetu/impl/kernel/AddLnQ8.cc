// Activations kept in 8 bits (blocks of 32 columns with a power of two each) and the pre-norm block's norm that keeps its
// input that way: Q8PackCuda, Q8UnpackCuda, AddLnQ8FwdCuda, AddLnQ8OutCuda, AddLnQ8BwdCuda.  No counterpart in the reference,
// whose norm keeps its input in the residual stream's type (hetu/impl/kernel/RMSNorm.cu:91-470).
#include "hetu/graph/ops/kernel_links.h"
#include "hetu/impl/kernel/kernel_utils.h"

#include <memory>

namespace hetu {
namespace impl {

namespace {
void RowsCols(const NDArray& a, int64_t& rows, int64_t& cols) {
  HT_ASSERT(a->ndim() >= 1) << "rows need at least one dimension";
  rows = 1;
  for (size_t i = 0; i + 1 < a->ndim(); ++i) rows *= a->shape(i);
  cols = a->shape(a->ndim() - 1);
}

void CheckKept(const NDArray& ref, const NDArray& q, const NDArray& scale, int64_t rows, int64_t cols) {
  const int64_t blocks = (cols + HK_Q8_BLOCK - 1) / HK_Q8_BLOCK;
  HT_ASSERT(q.is_defined() && scale.is_defined()) << "the kept values and their exponents are missing";
  HT_ASSERT_SAME_DEVICE(ref, q);
  HT_ASSERT_SAME_DEVICE(ref, scale);
  HT_ASSERT(q->dtype() == kInt8 && scale->dtype() == kUInt8)
    << "kept values are int8 with uint8 exponents, got " << q->dtype() << " and " << scale->dtype();
  HT_ASSERT(int64_t(q->numel()) == rows * blocks * HK_Q8_BLOCK && int64_t(scale->numel()) == rows * blocks)
    << "[" << rows << ", " << cols << "] values are kept in " << blocks << " blocks a row, got " << q->shape() << " and "
    << scale->shape();
  HT_ASSERT(q->is_contiguous() && scale->is_contiguous()) << "kept values must be dense";
}

void CheckValues(const NDArray& a, const NDArray& ref, DataType dtype, int64_t count, const char* what) {
  if (!a.is_defined()) return;
  HT_ASSERT_SAME_DEVICE(ref, a);
  HT_ASSERT(a->dtype() == dtype) << what << " must be " << dtype << ", got " << a->dtype();
  HT_ASSERT(int64_t(a->numel()) == count) << what << " must hold " << count << " values, got " << a->shape();
  HT_ASSERT(a->is_contiguous()) << what << " must be dense";
}

void CheckRows(const NDArray& a, const NDArray& ref, DataType dtype, const char* what) {
  if (!a.is_defined()) return;
  HT_ASSERT_SAME_DEVICE(ref, a);
  HT_ASSERT_SAME_SHAPE(ref, a);
  HT_ASSERT(a->dtype() == dtype) << what << " must be " << dtype << ", got " << a->dtype();
}

// an optional row operand: its pitch, or none
NDArray OptionalRows(const NDArray& a, const Stream& stream, int64_t* pitch) {
  return a.is_defined() ? RowOperand(a, 1, stream, pitch) : a;
}

// an optional row output
struct OptionalOutput {
  std::unique_ptr<RowOutput> out;
  OptionalOutput(NDArray& a, const Stream& stream) {
    if (a.is_defined()) out.reset(new RowOutput(a, 1, stream));
  }
  void* ptr() { return out ? out->ptr() : nullptr; }
  int64_t pitch() const { return out ? out->pitch() : 0; }
  NDArray array() { return out ? out->array() : NDArray(); }
  void Commit() { if (out) out->Commit(); }
};

int8_t* Bytes(const NDArray& q) { return static_cast<int8_t*>(q->raw_data_ptr()); }
uint8_t* Exponents(const NDArray& scale) { return static_cast<uint8_t*>(scale->raw_data_ptr()); }
float* Floats(const NDArray& a) { return a.is_defined() ? static_cast<float*>(a->raw_data_ptr()) : nullptr; }
} // namespace

void Q8PackCuda(const NDArray& input, NDArray& q, NDArray& scale, const Stream& stream) {
  HT_ASSERT(input.is_defined()) << "an input is missing";
  HT_ASSERT_CUDA_DEVICE(input);
  int64_t rows, cols, pitch = 0;
  RowsCols(input, rows, cols);
  CheckKept(input, q, scale, rows, cols);
  if (rows == 0 || cols == 0) return;
  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  NDArray x = RowOperand(input, 1, stream, &pitch);
  HK_CALL(hk_q8_pack(int(x->dtype()), x->raw_data_ptr(), pitch, Bytes(q), Exponents(scale), rows, cols, hip_stream));
  NDArray::MarkUsedBy({x, q, scale}, stream);
}

void Q8UnpackCuda(const NDArray& q, const NDArray& scale, NDArray& output, const Stream& stream) {
  HT_ASSERT(output.is_defined()) << "the output is missing";
  HT_ASSERT_CUDA_DEVICE(output);
  int64_t rows, cols;
  RowsCols(output, rows, cols);
  CheckKept(output, q, scale, rows, cols);
  if (rows == 0 || cols == 0) return;
  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  RowOutput out(output, 1, stream);
  HK_CALL(hk_q8_unpack(int(output->dtype()), Bytes(q), Exponents(scale), out.ptr(), out.pitch(), rows, cols, hip_stream));
  out.Commit();
  NDArray::MarkUsedBy({q, scale, out.array()}, stream);
}

void AddLnQ8FwdCuda(const NDArray& x0, const NDArray& residual_, const NDArray& gamma_, const NDArray& beta_, NDArray& z,
                    NDArray& x, NDArray& q, NDArray& scale, NDArray& mu, NDArray& rsigma, const float epsilon,
                    bool is_rms_norm, const Stream& stream) {
  HT_ASSERT(x0.is_defined() && z.is_defined() && mu.is_defined() && rsigma.is_defined()) << "a required array is missing";
  HT_ASSERT_CUDA_DEVICE(x0);
  int64_t rows, cols, x0_pitch = 0, residual_pitch = 0;
  RowsCols(x0, rows, cols);
  const auto itype = x0->dtype();
  const auto rtype = residual_.is_defined() ? residual_->dtype() : x.is_defined() ? x->dtype() : itype;
  CheckRows(residual_, x0, rtype, "residual");
  CheckRows(x, x0, rtype, "x");
  CheckRows(z, x0, itype, "z");
  CheckValues(gamma_, x0, itype, cols, "gamma");
  CheckValues(beta_, x0, itype, cols, "beta");
  CheckValues(mu, x0, kFloat32, rows, "mu");
  CheckValues(rsigma, x0, kFloat32, rows, "rsigma");
  CheckKept(x0, q, scale, rows, cols);
  if (rows == 0 || cols == 0) return;
  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  NDArray in = RowOperand(x0, 1, stream, &x0_pitch), res = OptionalRows(residual_, stream, &residual_pitch);
  RowOutput zo(z, 1, stream);
  OptionalOutput xo(x, stream);
  HK_CALL(hk_add_ln_q8_fwd(int(itype), int(rtype), in->raw_data_ptr(), x0_pitch, PtrOrNull(res), residual_pitch,
                           PtrOrNull(gamma_), PtrOrNull(beta_), zo.ptr(), zo.pitch(), xo.ptr(), xo.pitch(), Bytes(q),
                           Exponents(scale), Floats(mu), Floats(rsigma), rows, cols, epsilon, is_rms_norm ? 1 : 0, hip_stream));
  zo.Commit();
  xo.Commit();
  NDArray::MarkUsedBy({in, res, gamma_, beta_, zo.array(), xo.array(), q, scale, mu, rsigma}, stream);
}

void AddLnQ8OutCuda(const NDArray& q, const NDArray& scale, const NDArray& mu_, const NDArray& rsigma, const NDArray& gamma_,
                    const NDArray& beta_, NDArray& z, bool is_rms_norm, const Stream& stream) {
  HT_ASSERT(z.is_defined() && rsigma.is_defined() && (mu_.is_defined() || is_rms_norm)) << "a required array is missing";
  HT_ASSERT_CUDA_DEVICE(z);
  int64_t rows, cols;
  RowsCols(z, rows, cols);
  CheckValues(gamma_, z, z->dtype(), cols, "gamma");
  CheckValues(beta_, z, z->dtype(), cols, "beta");
  CheckValues(mu_, z, kFloat32, rows, "mu");
  CheckValues(rsigma, z, kFloat32, rows, "rsigma");
  CheckKept(z, q, scale, rows, cols);
  if (rows == 0 || cols == 0) return;
  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  RowOutput zo(z, 1, stream);
  HK_CALL(hk_add_ln_q8_out(int(z->dtype()), Bytes(q), Exponents(scale), Floats(mu_), Floats(rsigma), PtrOrNull(gamma_),
                           PtrOrNull(beta_), zo.ptr(), zo.pitch(), rows, cols, is_rms_norm ? 1 : 0, hip_stream));
  zo.Commit();
  NDArray::MarkUsedBy({q, scale, mu_, rsigma, gamma_, beta_, zo.array()}, stream);
}

void AddLnQ8BwdCuda(const NDArray& dz, const NDArray& dx_, const NDArray& q, const NDArray& scale, const NDArray& mu_,
                    const NDArray& rsigma, const NDArray& gamma_, NDArray& dx0, NDArray& dresidual, NDArray& dgamma,
                    NDArray& dbeta, bool is_rms_norm, const Stream& stream) {
  HT_ASSERT(dz.is_defined() && dx0.is_defined() && rsigma.is_defined() && (mu_.is_defined() || is_rms_norm))
    << "a required array is missing";
  HT_ASSERT(!is_rms_norm || !dbeta.is_defined()) << "an RMSNorm has no beta";
  HT_ASSERT_CUDA_DEVICE(dz);
  int64_t rows, cols, dz_pitch = 0, dx_pitch = 0;
  RowsCols(dz, rows, cols);
  const auto itype = dz->dtype();
  const auto rtype = dx_.is_defined() ? dx_->dtype() : dresidual.is_defined() ? dresidual->dtype() : itype;
  CheckRows(dx_, dz, rtype, "dx");
  CheckRows(dresidual, dz, rtype, "dresidual");
  CheckRows(dx0, dz, itype, "dx0");
  CheckValues(gamma_, dz, itype, cols, "gamma");
  CheckValues(dgamma, dz, itype, cols, "dgamma");
  CheckValues(dbeta, dz, itype, cols, "dbeta");
  CheckValues(mu_, dz, kFloat32, rows, "mu");
  CheckValues(rsigma, dz, kFloat32, rows, "rsigma");
  CheckKept(dz, q, scale, rows, cols);
  if (cols == 0) return;
  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  NDArray in = rows ? RowOperand(dz, 1, stream, &dz_pitch) : dz, up = rows ? OptionalRows(dx_, stream, &dx_pitch) : dx_;
  RowOutput dxo(dx0, 1, stream);
  OptionalOutput dro(dresidual, stream);
  size_t ws_bytes = 0;
  if (dgamma.is_defined() || dbeta.is_defined()) HK_CALL(hk_add_ln_q8_bwd_workspace_bytes(rows, cols, &ws_bytes));
  NDArray ws = Scratch(ws_bytes, dz->device(), stream);
  HK_CALL(hk_add_ln_q8_bwd(int(itype), int(rtype), in->raw_data_ptr(), dz_pitch, PtrOrNull(up), dx_pitch, Bytes(q),
                           Exponents(scale), Floats(mu_), Floats(rsigma), PtrOrNull(gamma_), dxo.ptr(), dxo.pitch(), dro.ptr(),
                           dro.pitch(), MutPtrOrNull(dgamma), MutPtrOrNull(dbeta), rows, cols, is_rms_norm ? 1 : 0,
                           MutPtrOrNull(ws), ws_bytes, hip_stream));
  dxo.Commit();
  dro.Commit();
  NDArray::MarkUsedBy({in, up, q, scale, mu_, rsigma, gamma_, dxo.array(), dro.array(), dgamma, dbeta, ws}, stream);
}

} // namespace impl
} // namespace hetu
