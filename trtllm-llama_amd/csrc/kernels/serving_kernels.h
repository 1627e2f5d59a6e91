// Host-side launch interface of the kernels behind include/tllm_serving_api.h (paged_plan.hip, paged_append.hip, paged_attn.hip,
// group_gemm.hip).  The parameters have been checked by the caller (plugins/serving_api.cpp); launchers enqueue on `stream` and return 0, or -1
// with set_error when the launch itself is refused.
#pragma once
#include "../../../include/tllm_serving_api.h"
#include "kernels.h"

namespace tllm
{
namespace kernels
{

constexpr int kPlanMaxSeqs = 4096;

int launch_paged_plan(const tllm_paged_plan_params_t& p, hipStream_t stream);
int launch_paged_append(const tllm_paged_append_params_t& p, hipStream_t stream);
size_t paged_attention_workspace(const tllm_paged_attention_params_t& p);
int launch_paged_attention(const tllm_paged_attention_params_t& p, void* workspace, hipStream_t stream);
int launch_group_matmul(const tllm_group_matmul_params_t& p, hipStream_t stream);

inline int launched(const char* what)
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess)
        return 0;
    set_error("%s: %s", what, hipGetErrorString(e));
    return -1;
}

} // namespace kernels
} // namespace tllm
