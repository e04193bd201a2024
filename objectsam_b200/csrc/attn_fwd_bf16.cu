#include "attn_fwd.cuh"
namespace osam {
template cudaError_t launch_attn_fwd<__nv_bfloat16>(const AttnFwdLaunch&, cudaStream_t);
}
