// The training operators' rules on sizes, for ctypes.
#include "tms_train_rules.h"

extern "C" int gemm_size_of(int64_t m, int64_t n, int64_t steps) { return tms::gemm_size(m, n, steps); }

extern "C" double gemm_time(int size, int64_t m, int64_t n, int64_t steps, int64_t splits) { return tms::gemm_us(size, m, n, steps, splits); }

extern "C" void lce_plan_of(int64_t N, int64_t V, int64_t d, int planes, int64_t* out) {
  const tms::LcePlan p = tms::lce_plan(N, V, d, planes);
  const int64_t all[] = {p.dp, p.rows_p, p.piece, p.splits, p.size_p, p.size_h, p.size_w};
  for (int i = 0; i < 7; i++) out[i] = all[i];
}
