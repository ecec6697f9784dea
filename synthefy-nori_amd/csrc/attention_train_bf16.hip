// Attention with gradients over bfloat16 rows in 16-byte chunks (attention_train_kernel.h).
#include "attention_train_kernel.h"

namespace nori {
namespace attn_train {

int launch_bf16(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    return launch_width<NORI_BF16, 8>(kind, p, blocks, stream);
}

}  // namespace attn_train
}  // namespace nori
