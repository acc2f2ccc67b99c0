// The attention kernels in bfloat16.
#include "attention_bwd.h"
#include "attention_fwd.h"

namespace s2cnn {
namespace attn {
template void forward<BF16>(const Args&, const Plans&, hipStream_t);
template void backward<BF16>(Args, const Plans&, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace s2cnn
