// The attention kernels in float16.
#include "attention_bwd.h"
#include "attention_fwd.h"

namespace s2cnn {
namespace attn {
template void forward<F16>(const Args&, const Plans&, hipStream_t);
template void backward<F16>(Args, const Plans&, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace s2cnn
