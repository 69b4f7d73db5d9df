// The row form of attention over a quantised paged cache: gs_paged_rows.h's kernels with
// e4m3 rows, which become bf16 (fp32) operands in registers.
//
// 256 sequences of 16 .. 2047 keys, 8 key/value heads of 128, bf16 queries: 68 us, 3.9 TB/s
// (a bf16 cache: 109); one of 131071 keys: 61 us, 4.4 TB/s (105).  With probabilities as one
// bf16 number, 67 and 61 us, the loads and the schedule alone took 62, the arithmetic alone 54 and
// 41; a start, a join and parts of uneven length, which 270 MB hide less than 540 do, are the
// rest.  Against those 67 and 61 no gain: two blocks ahead instead of one (74 and 64 us), three
// workgroups to a compute unit (78 and 77: registers spill), parts drawn first come, first
// served (68.5 and 61), a part's first loads before the results of the one ahead (69.6 and 63),
// half the keys to a part (76 and 68).
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
