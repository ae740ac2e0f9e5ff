// The attention kernels for fp32 tensors over 4-bit codes (their instances compile apart).
#include "kv_attention.cuh"

namespace nnrcu {
namespace attn {
int launch_f32_b4(const Args& p, bool own, cudaStream_t st) { return launch_for<2, 2, 4>(p, own, st); }
}  // namespace attn
}  // namespace nnrcu
