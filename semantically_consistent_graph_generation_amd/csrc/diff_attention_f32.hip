// Differential attention for float tensors: the kernels of diff_attention_fwd.h and diff_attention_bwd.h.
#include "diff_attention_bwd.h"

namespace scgg {
namespace diffattn {
template int run_forward<float>(const Args&, hipStream_t);
template int run_split<float>(const Args&, hipStream_t);
template int run_backward<float>(const Args&, hipStream_t);
}  // namespace diffattn
}  // namespace scgg
