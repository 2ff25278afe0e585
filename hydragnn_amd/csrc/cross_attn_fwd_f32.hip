// The kernels of cross_attn_fwd.h for float.
#include "cross_attn_fwd.h"

namespace hy {
namespace xa {
template void forward_rows<float>(const Args&, at::ScalarType, int, hipStream_t);
}
}  // namespace hy
