// The kernels of cross_attn_fwd.h for float16.
#include "cross_attn_fwd.h"

namespace hy {
namespace xa {
template void forward_rows<_Float16>(const Args&, at::ScalarType, int, hipStream_t);
}
}  // namespace hy
