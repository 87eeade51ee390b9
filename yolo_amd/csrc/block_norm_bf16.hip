// The kernels of block_norm.h for bf16 rows (residual stream bf16 or fp32).
#include "block_norm.h"

namespace yolo_amd {

void block_norm_launch_bf16(const NormArgs& a, bool stream_f32, int blocks, bool backward, hipStream_t s) {
    if (stream_f32) norm_launch<__bf16, float>(a, blocks, backward, s);
    else norm_launch<__bf16, __bf16>(a, blocks, backward, s);
}

}  // namespace yolo_amd
