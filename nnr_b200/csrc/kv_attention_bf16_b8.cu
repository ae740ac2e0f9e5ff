// The attention kernels for bf16 tensors over 8-bit codes (their instances compile apart).
#include "kv_attention.cuh"

namespace nnrcu {
namespace attn {
int launch_bf16_b8(const Args& p, bool own, cudaStream_t st) { return launch_for<1, 1, 8>(p, own, st); }
}  // namespace attn
}  // namespace nnrcu
