// Products of rows sorted by expert with 4-bit weights.
#include "tab_experts_launch.h"

namespace tab {

hipError_t launch_experts4(int out, const ExpertsPlan &plan, const ExpertsArgs &a, void *workspace, hipStream_t stream)
{
    if (plan.few)
        return out == 0 ? launch_expert_rows<3, 0, 0, 4>(plan, a, a.N, stream)
                        : out == 1 ? launch_expert_rows<3, 0, 1, 4>(plan, a, a.N, stream) : launch_expert_rows<3, 0, 2, 4>(plan, a, a.N, stream);
    return launch_expert_product<0, 4>(out, true, plan, a, a.N, workspace, stream);
}

hipError_t launch_experts4_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, hipStream_t stream) { return launch_expert_few<4>(dtype, plan, a, a.N, stream); }

}  // namespace tab
