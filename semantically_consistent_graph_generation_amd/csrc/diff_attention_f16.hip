// Differential attention for _Float16 tensors: the kernels of diff_attention_fwd.h and diff_attention_bwd.h.
#include "diff_attention_bwd.h"

namespace scgg {
namespace diffattn {
template int run_forward<_Float16>(const Args&, hipStream_t);
template int run_split<_Float16>(const Args&, hipStream_t);
template int run_backward<_Float16>(const Args&, hipStream_t);
}  // namespace diffattn
}  // namespace scgg
