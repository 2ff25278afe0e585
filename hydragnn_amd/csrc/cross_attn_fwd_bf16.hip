// The kernels of cross_attn_fwd.h for bfloat16.
#include "cross_attn_fwd.h"

namespace hy {
namespace xa {
template void forward_rows<__bf16>(const Args&, at::ScalarType, int, hipStream_t);
}
}  // namespace hy
