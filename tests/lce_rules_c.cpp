// The times that cross entropy's tiles are picked by (tms_train_rules.h), for test_training_times.py.
#include "tms_train_rules.h"

using namespace tms;

extern "C" int logits_size_of(int64_t N, int64_t V, int64_t dp, int planes) { return terms_size(V, N, dp, planes, gemm_largest(planes)); }
extern "C" double terms_time(int size, int64_t m, int64_t n, int64_t k, int planes, int64_t splits) { return terms_us(size, m, n, k, planes, splits); }
extern "C" double product_time(int size, int64_t m, int64_t n, int64_t k, int planes, int64_t splits) { return product_us(size, m, n, k, planes, splits); }
extern "C" void plan_of(int64_t N, int64_t V, int64_t d, int planes, int64_t* out) {
  const LcePlan p = lce_plan(N, V, d, planes);
  const int64_t all[] = {p.dp, p.rows_p, p.piece, p.splits, p.size_p, p.size_h, p.size_w};
  for (int i = 0; i < 7; i++) out[i] = all[i];
}
