// The selective scan on float32 tensors.
#include "exb_selective_kernels.cuh"

namespace exb {

template cudaError_t selective_forward_typed<float>(const SelArgs &, const SelPlan &, cudaStream_t);
template cudaError_t selective_backward_typed<float>(const SelArgs &, const SelPlan &, void *, void *, cudaStream_t);

}  // namespace exb
