// The kernels of fa_paged_kernels.h with capped and biased scores and windows.
// (Kernels of their own: the plain ones keep their registers and their code.)
#include "fa_paged_kernels.h"

namespace fa {

hipError_t launch_paged_scored(const PagedFwdArgs& args, const PagedPlan& plan, int head_dim, bool bf16,
                               void* workspace, hipStream_t stream) {
  return launch_as<true>(args, plan, head_dim, bf16, workspace, stream);
}

}  // namespace fa
