// The attention kernels in float32.
#include "attention_bwd.h"
#include "attention_fwd.h"

namespace s2cnn {
namespace attn {
template void forward<F32>(const Args&, const Plans&, hipStream_t);
template void backward<F32>(Args, const Plans&, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace s2cnn
