// Attention over packed texts (tms_train_attn_kernel.h): the f16 kernels.
#include "tms_train_attn_kernel.h"

namespace tms {

int attn_run_f16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st) { return attn_run<TMS_DTYPE_F16>(a, D, pass, st); }

}  // namespace tms
