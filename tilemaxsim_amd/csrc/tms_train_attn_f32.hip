// Attention over packed texts (tms_train_attn_kernel.h): the f32 kernels.
#include "tms_train_attn_kernel.h"

namespace tms {

int attn_run_f32(const AttnArgs& a, int D, AttnPass pass, hipStream_t st) { return attn_run<TMS_DTYPE_F32>(a, D, pass, st); }

}  // namespace tms
