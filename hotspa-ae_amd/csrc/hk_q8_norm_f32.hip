// The norm with an 8-bit checkpoint for fp32 rows.
#include "hk_q8_norm_impl.h"

namespace hk {
template int q8_norm_fwd_typed<float>(const Q8FwdArgs&, int, bool, const Q8Shape&, hipStream_t);
template int q8_norm_bwd_typed<float>(const Q8BwdArgs&, int, bool, const Q8Shape&, void*, void*, hipStream_t);
} // namespace hk
