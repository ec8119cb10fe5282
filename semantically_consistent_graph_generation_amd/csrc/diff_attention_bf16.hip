// Differential attention for __bf16 tensors: the kernels of diff_attention_fwd.h and diff_attention_bwd.h.
#include "diff_attention_bwd.h"

namespace scgg {
namespace diffattn {
template int run_forward<__bf16>(const Args&, hipStream_t);
template int run_split<__bf16>(const Args&, hipStream_t);
template int run_backward<__bf16>(const Args&, hipStream_t);
}  // namespace diffattn
}  // namespace scgg
