// The fp16 instance of the tensor-core cross attention.
#include "cross_attention_mma.cuh"

namespace ssam {

int xattn_fp16(const XAttn& a, bool backward, cudaStream_t stream) { return xattn_mma<__half>(a, backward, stream); }

}  // namespace ssam
