// Attention with gradients over float16 rows in 8-byte chunks (attention_train_kernel.h).
#include "attention_train_kernel.h"

namespace nori {
namespace attn_train {

int launch_f16_narrow(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    return launch_width<NORI_F16, 4>(kind, p, blocks, stream);
}

}  // namespace attn_train
}  // namespace nori
