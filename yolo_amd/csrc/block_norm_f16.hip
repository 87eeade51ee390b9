// The kernels of block_norm.h for f16 rows (residual stream f16 or fp32).
#include "block_norm.h"

namespace yolo_amd {

void block_norm_launch_f16(const NormArgs& a, bool stream_f32, int blocks, bool backward, hipStream_t s) {
    if (stream_f32) norm_launch<_Float16, float>(a, blocks, backward, s);
    else norm_launch<_Float16, _Float16>(a, blocks, backward, s);
}

}  // namespace yolo_amd
