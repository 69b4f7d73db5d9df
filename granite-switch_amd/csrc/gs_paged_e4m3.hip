// The row form of attention over a quantised paged cache: gs_paged_rows.h's kernels with
// e4m3 rows, which become bf16 (fp32) operands in registers.
#include "gs_paged_rows.h"

namespace gs {

void launch_rows_e4m3(const PagedArgs& a, bool bf16, int DT, int64_t workgroups, hipStream_t st) {
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(workgroups)), dim3(256), 0, st, a); };
  switch (DT) {
    case 64: bf16 ? go(paged_attention_kernel<true, 64, true>) : go(paged_attention_kernel<false, 64, true>); break;
    case 128: bf16 ? go(paged_attention_kernel<true, 128, true>) : go(paged_attention_kernel<false, 128, true>); break;
    default: bf16 ? go(paged_attention_kernel<true, 256, true>) : go(paged_attention_kernel<false, 256, true>); break;
  }
}

}  // namespace gs
