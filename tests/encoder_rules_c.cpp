// The rules of attention, of few tokens and of split products (tms_train_rules.h), for test_encoder_host.py.
#include "tms_train_rules.h"

using namespace tms;

extern "C" int64_t attn_slots_of(int64_t T, int64_t B, int64_t rows) { return attn_slots(T, B, rows); }
extern "C" int attn_wide_of(int64_t T, int64_t B, int64_t heads) { return attn_wide(T, B, heads); }
extern "C" int64_t attn_parts_of(int64_t T, int64_t B, int64_t kv, int64_t many) { return attn_parts(T, B, kv, many); }
extern "C" void gemm_split_of(int64_t m, int64_t n, int64_t k, int planes, int64_t* out) {
  const GemmSplit s = gemm_split(m, n, k, planes);
  out[0] = s.size;
  out[1] = s.splits;
}
extern "C" int gated_few_of(int64_t N, int64_t d, int64_t F, int f32) { return gated_few(N, d, F, f32 != 0); }
