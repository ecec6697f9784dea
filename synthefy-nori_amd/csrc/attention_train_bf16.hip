// Attention with gradients over bfloat16 rows (attention_train_kernel.h).
#include "attention_train_kernel.h"

namespace nori {
namespace attn_train {

int launch_bf16(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) { return launch_chunks<NORI_BF16>(kind, p, blocks, stream); }

}  // namespace attn_train
}  // namespace nori
