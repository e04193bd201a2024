#include "attn_fwd.cuh"
namespace osam {
template cudaError_t launch_attn_fwd<__half>(const AttnFwdLaunch&, cudaStream_t);
}
