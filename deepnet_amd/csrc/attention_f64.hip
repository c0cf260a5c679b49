// Double-precision instantiations of the cross-attention kernels.
#include "attention_kernels.h"

namespace dnh {
template <> int32_t attention_forward<double>(AttArgs<double>& p, void* scratch, size_t scratch_bytes, hipStream_t s) { return attention_forward_impl<double>(p, scratch, scratch_bytes, s); }
template <> int32_t attention_backward<double>(AttArgs<double>& p, void* scratch, size_t scratch_bytes, hipStream_t s) { return attention_backward_impl<double>(p, scratch, scratch_bytes, s); }
}  // namespace dnh
