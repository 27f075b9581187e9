// The encoder's translation unit of libsparsesam_b200.so: its kernels share the device
// error flag and the host caches without relocatable device code. The decoder's
// operators, which use neither, are compiled beside it (build.py, UNITS).
#include "host_util.cu"
#include "gemm.cu"
#include "perm.cu"
#include "rows.cu"
#include "attention.cu"
#include "cross_attention_tc.cu"
#include "capi.cu"
#include "noalloc.cu"
