// Attention with gradients over float32 rows (attention_train_kernel.h).
#include "attention_train_kernel.h"

namespace nori {
namespace attn_train {

int launch_f32(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    return launch_width<NORI_F32, 4>(kind, p, blocks, stream);
}

}  // namespace attn_train
}  // namespace nori
