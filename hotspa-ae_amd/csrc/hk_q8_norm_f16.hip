// The norm with an 8-bit checkpoint for fp16 rows.
#include "hk_q8_norm_impl.h"

namespace hk {
template int q8_norm_fwd_typed<fp16>(const Q8FwdArgs&, int, bool, const Q8Shape&, hipStream_t);
template int q8_norm_bwd_typed<fp16>(const Q8BwdArgs&, int, bool, const Q8Shape&, void*, void*, hipStream_t);
} // namespace hk
