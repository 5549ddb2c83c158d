// TokenLogProbCuda / TokenLogProbGradientCuda and their vocabulary-parallel halves: log probabilities of given tokens with
// the rows' entropy and most likely alternatives, beside the sparse cross-entropy.  No counterpart in the reference, whose
// loss gives the negated log probability alone (hetu/impl/kernel/SoftmaxCrossEntropySparse.cu:239-318).
#include "hetu/graph/ops/kernel_links.h"
#include "hetu/impl/kernel/kernel_utils.h"

namespace hetu {
namespace impl {

namespace {
void RowsCols(const NDArray& pred, int64_t& rows, int64_t& cols) {
  HT_ASSERT(pred->ndim() >= 1) << "logits need at least one dimension";
  rows = 1;
  for (size_t i = 0; i + 1 < pred->ndim(); ++i) rows *= pred->shape(i);
  cols = pred->shape(pred->ndim() - 1);
}

// `count` dense values of a type on the logits' device; an undefined array is an output left out
void CheckValues(const NDArray& a, const NDArray& pred, DataType dtype, int64_t count, const char* what) {
  if (!a.is_defined()) return;
  HT_ASSERT_SAME_DEVICE(pred, a);
  HT_ASSERT(a->dtype() == dtype) << what << " must be " << dtype << ", got " << a->dtype();
  HT_ASSERT(int64_t(a->numel()) == count) << what << " must hold " << count << " values, got " << a->shape();
  HT_ASSERT(a->is_contiguous()) << what << " must be dense";
}

// how many alternatives a row has room for in a pair of arrays (both or none)
int64_t Alternatives(const NDArray& value, const NDArray& token) {
  HT_ASSERT(value.is_defined() == token.is_defined()) << "values and tokens of the alternatives come together";
  if (!value.is_defined()) return 0;
  HT_ASSERT(value->ndim() >= 1 && value->shape() == token->shape())
    << "values and tokens of the alternatives differ in shape: " << value->shape() << ", " << token->shape();
  return value->shape(value->ndim() - 1);
}

float* Floats(NDArray& a) { return static_cast<float*>(MutPtrOrNull(a)); }
const float* Floats(const NDArray& a) { return static_cast<const float*>(PtrOrNull(a)); }
int64_t* Tokens(NDArray& a) { return static_cast<int64_t*>(MutPtrOrNull(a)); }
const int64_t* Tokens(const NDArray& a) { return static_cast<const int64_t*>(PtrOrNull(a)); }
} // namespace

void TokenLogProbCuda(const NDArray& pred, const NDArray& token, NDArray& logprob, NDArray& entropy, NDArray& lse,
                      NDArray& top_logprob, NDArray& top_token, const int64_t ignored_index, const Stream& stream) {
  HT_ASSERT(pred.is_defined() && token.is_defined()) << "logits or tokens are missing";
  HT_ASSERT_CUDA_DEVICE(pred);
  int64_t rows, cols;
  RowsCols(pred, rows, cols);
  const int64_t top = Alternatives(top_logprob, top_token);
  CheckValues(token, pred, kInt64, rows, "tokens");
  CheckValues(logprob, pred, kFloat32, rows, "log probabilities");
  CheckValues(entropy, pred, kFloat32, rows, "entropy");
  CheckValues(lse, pred, kFloat32, rows, "log-sum-exp");
  CheckValues(top_logprob, pred, kFloat32, rows * top, "alternatives' log probabilities");
  CheckValues(top_token, pred, kInt64, rows * top, "alternatives' tokens");
  if (rows == 0) return;
  HT_VALUE_ERROR_IF(cols == 0) << "log probabilities over zero tokens";

  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  int64_t pitch = 0;
  NDArray x = RowOperand(pred, 1, stream, &pitch);
  size_t ws_bytes = 0;
  HK_CALL(hk_token_logprob_workspace_bytes(int(x->dtype()), rows, cols, top, &ws_bytes));
  NDArray ws = Scratch(ws_bytes, x->device(), stream);
  HK_CALL(hk_token_logprob_fwd(int(x->dtype()), x->raw_data_ptr(), pitch, Tokens(token), Floats(logprob), Floats(entropy),
                               Floats(lse), Floats(top_logprob), Tokens(top_token), top, rows, cols, ignored_index,
                               MutPtrOrNull(ws), ws_bytes, hip_stream));
  NDArray::MarkUsedBy({x, token, logprob, entropy, lse, top_logprob, top_token, ws}, stream);
}

void TokenLogProbGradientCuda(const NDArray& pred, const NDArray& token, const NDArray& lse, const NDArray& entropy_,
                              const NDArray& grad_logprob_, const NDArray& grad_entropy_, NDArray& output,
                              const int64_t vocab_start_index, const int64_t ignored_index, const Stream& stream) {
  HT_ASSERT(pred.is_defined() && token.is_defined() && lse.is_defined() && output.is_defined()) << "a required array is missing";
  HT_ASSERT_CUDA_DEVICE(pred);
  HT_ASSERT_SAME_DEVICE(pred, output);
  HT_ASSERT_SAME_SHAPE(pred, output);
  HT_ASSERT_SAME_DTYPE(pred, output);
  int64_t rows, cols;
  RowsCols(pred, rows, cols);
  CheckValues(token, pred, kInt64, rows, "tokens");
  CheckValues(lse, pred, kFloat32, rows, "log-sum-exp");
  CheckValues(entropy_, pred, kFloat32, rows, "entropy");
  CheckValues(grad_logprob_, pred, kFloat32, rows, "gradient of the log probabilities");
  CheckValues(grad_entropy_, pred, kFloat32, rows, "gradient of the entropy");
  HT_ASSERT(grad_logprob_.is_defined() || grad_entropy_.is_defined()) << "neither output has a gradient";
  HT_ASSERT(!grad_entropy_.is_defined() || entropy_.is_defined()) << "the entropy's gradient needs the entropy";
  if (rows == 0 || cols == 0) return;

  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  int64_t pitch = 0;
  NDArray x = RowOperand(pred, 1, stream, &pitch);
  RowOutput out(output, 1, stream);
  HK_CALL(hk_token_logprob_bwd(int(x->dtype()), x->raw_data_ptr(), pitch, Tokens(token), Floats(lse), Floats(entropy_),
                               Floats(grad_logprob_), Floats(grad_entropy_), out.ptr(), out.pitch(), rows, cols,
                               vocab_start_index, ignored_index, hip_stream));
  out.Commit();
  NDArray::MarkUsedBy({x, token, lse, entropy_, grad_logprob_, grad_entropy_, out.array()}, stream);
}

void VocabParallelLogProbStatsCuda(const NDArray& vocab_parallel_logits, const NDArray& token, NDArray& stats,
                                   NDArray& top_value, NDArray& top_token, const int64_t vocab_start_index,
                                   const int64_t ignored_index, const Stream& stream) {
  HT_ASSERT(vocab_parallel_logits.is_defined() && token.is_defined()) << "logits or tokens are missing";
  HT_ASSERT_CUDA_DEVICE(vocab_parallel_logits);
  int64_t rows, cols;
  RowsCols(vocab_parallel_logits, rows, cols);
  const int64_t top = Alternatives(top_value, top_token);
  HT_ASSERT(stats.is_defined()) << "the shard's statistics need an array";
  CheckValues(token, vocab_parallel_logits, kInt64, rows, "tokens");
  CheckValues(stats, vocab_parallel_logits, kFloat32, 4 * rows, "statistics");
  CheckValues(top_value, vocab_parallel_logits, kFloat32, rows * top, "alternatives' logits");
  CheckValues(top_token, vocab_parallel_logits, kInt64, rows * top, "alternatives' tokens");
  if (rows == 0) return;
  HT_VALUE_ERROR_IF(cols == 0) << "a shard without tokens";

  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  int64_t pitch = 0;
  NDArray x = RowOperand(vocab_parallel_logits, 1, stream, &pitch);
  size_t ws_bytes = 0;
  HK_CALL(hk_token_logprob_workspace_bytes(int(x->dtype()), rows, cols, top, &ws_bytes));
  NDArray ws = Scratch(ws_bytes, x->device(), stream);
  HK_CALL(hk_vocab_parallel_logprob_stats(int(x->dtype()), x->raw_data_ptr(), pitch, Tokens(token), Floats(stats),
                                          Floats(top_value), Tokens(top_token), top, rows, cols, vocab_start_index,
                                          ignored_index, MutPtrOrNull(ws), ws_bytes, hip_stream));
  NDArray::MarkUsedBy({x, token, stats, top_value, top_token, ws}, stream);
}

void VocabParallelLogProbCombineCuda(const NDArray& stats, const NDArray& top_values, const NDArray& top_tokens,
                                     const NDArray& token, const int64_t ignored_index, const int64_t vocab_size,
                                     NDArray& logprob, NDArray& entropy, NDArray& lse, NDArray& top_logprob,
                                     NDArray& top_token, const Stream& stream) {
  HT_ASSERT(stats.is_defined() && token.is_defined()) << "statistics or tokens are missing";
  HT_ASSERT_CUDA_DEVICE(stats);
  HT_ASSERT(stats->ndim() == 3 && stats->shape(1) == 4) << "statistics must be [shards, 4, rows], got " << stats->shape();
  const int64_t shards = stats->shape(0), rows = stats->shape(2);
  const int64_t top = Alternatives(top_logprob, top_token);
  HT_ASSERT(Alternatives(top_values, top_tokens) == top) << "the shards hold another number of alternatives than asked for";
  CheckValues(stats, stats, kFloat32, shards * 4 * rows, "statistics");
  CheckValues(top_values, stats, kFloat32, shards * rows * top, "the shards' alternatives");
  CheckValues(top_tokens, stats, kInt64, shards * rows * top, "the shards' alternatives' tokens");
  CheckValues(token, stats, kInt64, rows, "tokens");
  CheckValues(logprob, stats, kFloat32, rows, "log probabilities");
  CheckValues(entropy, stats, kFloat32, rows, "entropy");
  CheckValues(lse, stats, kFloat32, rows, "log-sum-exp");
  CheckValues(top_logprob, stats, kFloat32, rows * top, "alternatives' log probabilities");
  CheckValues(top_token, stats, kInt64, rows * top, "alternatives' tokens");
  if (rows == 0) return;

  HIPStream hip_stream(stream);
  hip::DeviceGuard guard(hip_stream.device_id());
  HK_CALL(hk_vocab_parallel_logprob_combine(Floats(stats), Floats(top_values), Tokens(top_tokens), shards, Tokens(token),
                                            ignored_index, vocab_size, Floats(logprob), Floats(entropy), Floats(lse),
                                            Floats(top_logprob), Tokens(top_token), top, rows, hip_stream));
  NDArray::MarkUsedBy({stats, top_values, top_tokens, token, logprob, entropy, lse, top_logprob, top_token}, stream);
}

} // namespace impl
} // namespace hetu
