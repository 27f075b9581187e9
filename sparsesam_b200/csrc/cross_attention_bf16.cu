// The bf16 instance of the tensor-core cross attention.
#include "cross_attention_mma.cuh"

namespace ssam {

int xattn_bf16(const XAttn& a, bool backward, cudaStream_t stream) { return xattn_mma<__nv_bfloat16>(a, backward, stream); }

}  // namespace ssam
