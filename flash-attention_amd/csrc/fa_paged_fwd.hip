// The kernels of fa_paged_kernels.h with plain scores, scale q.k.
#include "fa_paged_kernels.h"

namespace fa {

hipError_t launch_paged_fwd(const PagedFwdArgs& args, const PagedPlan& plan, int head_dim, bool bf16,
                            void* workspace, hipStream_t stream) {
  return launch_as<false>(args, plan, head_dim, bf16, workspace, stream);
}

}  // namespace fa
