// The kernels of cross_attn_bwd.h for bfloat16.
#include "cross_attn_bwd.h"

namespace hy {
namespace xa {
template void backward_rows<__bf16>(const Args&, at::ScalarType, int, float*, hipStream_t);
}
}  // namespace hy
