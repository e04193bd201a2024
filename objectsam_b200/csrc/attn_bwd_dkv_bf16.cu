#include "attn_bwd.cuh"
namespace osam {
template cudaError_t launch_attn_bwd<__nv_bfloat16, true>(const AttnBwdLaunch&, cudaStream_t);
}
