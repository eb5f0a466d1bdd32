// Attention over packed texts (tms_train_attn_kernel.h): the bf16 kernels.
#include "tms_train_attn_kernel.h"

namespace tms {

int attn_run_bf16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st) { return attn_run<TMS_DTYPE_BF16>(a, D, pass, st); }

}  // namespace tms
