// The kernels of cross_attn_bwd.h for float16.
#include "cross_attn_bwd.h"

namespace hy {
namespace xa {
template void backward_rows<_Float16>(const Args&, at::ScalarType, int, float*, hipStream_t);
}
}  // namespace hy
