#include "latent_common.cuh"
namespace el {
bool attention_tc_takes(const el_attention_t&, bool) { return false; }
int launch_attention_tc(const el_attention_t&, cudaStream_t) { return EL_ERR_UNSUPPORTED_SHAPE; }
int launch_attention_backward_tc(const el_attention_t&, const float*, float*, cudaStream_t) { return EL_ERR_UNSUPPORTED_SHAPE; }
}
