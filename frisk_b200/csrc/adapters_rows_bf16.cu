// adapters.cu's kernel for bf16.
#include "adapters_rows.cuh"

namespace fb {

cudaError_t launch_adapter_rows_bf16(frisk_b200_ctx* ctx, const adapter::AdapterParams& p, bool f32, cudaStream_t s) {
  return f32 ? launch_types<__nv_bfloat16, float>(ctx, p, s) : launch_types<__nv_bfloat16, __nv_bfloat16>(ctx, p, s);
}

}  // namespace fb
