#include "attn_bwd.cuh"
namespace osam {
template cudaError_t launch_attn_bwd<__half, false>(const AttnBwdLaunch&, cudaStream_t);
}
