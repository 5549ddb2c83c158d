// The norm with an 8-bit checkpoint for bf16 rows.
#include "hk_q8_norm_impl.h"

namespace hk {
template int q8_norm_fwd_typed<bf16>(const Q8FwdArgs&, int, bool, const Q8Shape&, hipStream_t);
template int q8_norm_bwd_typed<bf16>(const Q8BwdArgs&, int, bool, const Q8Shape&, void*, void*, hipStream_t);
} // namespace hk
