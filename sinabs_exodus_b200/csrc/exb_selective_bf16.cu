// The selective scan on bfloat16 tensors.
#include "exb_selective_kernels.cuh"

namespace exb {

template cudaError_t selective_forward_typed<__nv_bfloat16>(const SelArgs &, const SelPlan &, cudaStream_t);
template cudaError_t selective_backward_typed<__nv_bfloat16>(const SelArgs &, const SelPlan &, void *, void *, cudaStream_t);

}  // namespace exb
