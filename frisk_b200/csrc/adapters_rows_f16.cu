// adapters.cu's kernel for fp16.
#include "adapters_rows.cuh"

namespace fb {

cudaError_t launch_adapter_rows_f16(frisk_b200_ctx* ctx, const adapter::AdapterParams& p, bool f32, cudaStream_t s) {
  return f32 ? launch_types<__half, float>(ctx, p, s) : launch_types<__half, __half>(ctx, p, s);
}

}  // namespace fb
