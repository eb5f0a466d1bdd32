// Attention over packed texts: the C entry points. The kernels are in tms_train_attn_kernel.h.
#include "tms_train_attn_kernel.h"

namespace tms {

// Workgroups of 256 threads that one axis of a launch holds (2^31 threads of them).
constexpr int64_t kAttnMostTiles = 1 << 23;

constexpr int64_t kAttnMostStride = 1 << 22;

static int check_attention(const char* fn, const tms_attention* p, AttnArgs& a) {
  if (!p) return fail(TMS_ERR_INVALID, "%s: NULL description", fn);
  if (p->texts < 0 || p->tokens < 0 || p->heads < 0 || p->kv_heads < 0 || p->width < 0) return fail(TMS_ERR_INVALID, "%s: negative size", fn);
  if (p->dtype != TMS_DTYPE_F16 && p->dtype != TMS_DTYPE_BF16 && p->dtype != TMS_DTYPE_F32)
    return fail(TMS_ERR_UNSUPPORTED, "%s: dtype must be fp16, bf16 or fp32", fn);
  if (p->width != 32 && p->width != 64 && p->width != 96 && p->width != 128)
    return fail(TMS_ERR_UNSUPPORTED, "%s: heads of 32, 64, 96 or 128 elements (got %lld)", fn, (long long)p->width);
  if (p->heads == 0 || p->kv_heads == 0 || p->heads % p->kv_heads)
    return fail(TMS_ERR_INVALID, "%s: %lld heads do not share %lld", fn, (long long)p->heads, (long long)p->kv_heads);
  if (!(p->scale >= 1e-15) || !(p->scale <= 1e15)) return fail(TMS_ERR_INVALID, "%s: scale must be from 1e-15 to 1e15", fn);
  if (p->cap != 0 && (!(p->cap >= 1e-15) || !(p->cap <= 1e15))) return fail(TMS_ERR_INVALID, "%s: cap must be from 1e-15 to 1e15, or 0 for none", fn);
  if (p->tokens > ((int64_t)1 << 31) - (1 << 16) || p->texts > ((int64_t)1 << 31) - (1 << 16) || p->heads > (1 << 16) ||
      attn_grid(attn_slots(p->tokens, p->texts, 64), p->heads) >= kAttnMostTiles)
    return fail(TMS_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads in %lld texts are too many", fn, (long long)p->tokens, (long long)p->heads, (long long)p->texts);
  if (p->tokens == 0) return TMS_OK;
  if (!p->q || !p->k || !p->v || !p->offsets) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v) % 16) return fail(TMS_ERR_INVALID, "%s: q, k and v must be 16-byte aligned", fn);
  const int64_t whole = p->dtype == TMS_DTYPE_F32 ? 4 : 8;
  if ((p->q_token | p->q_head | p->k_token | p->k_head | p->v_token | p->v_head) % whole)
    return fail(TMS_ERR_INVALID, "%s: strides must be whole 16 bytes", fn);
  const int64_t strides[] = {p->q_token, p->k_token, p->v_token, p->heads * p->width};
  for (int64_t x : strides)  // a tile's rows are reached by 32-bit offsets
    if (x < 0 || x > kAttnMostStride) return fail(TMS_ERR_UNSUPPORTED, "%s: tokens of 0 to %lld elements apart (got %lld)", fn, (long long)kAttnMostStride, (long long)x);
  a = {};
  a.q = p->q, a.k = p->k, a.v = p->v;
  a.qt = p->q_token, a.qh = p->q_head, a.kt = p->k_token, a.kh = p->k_head, a.vt = p->v_token, a.vh = p->v_head;
  a.offsets = p->offsets, a.prefix = p->prefix, a.slopes = p->slopes;
  a.T = p->tokens;
  a.B = (int32_t)p->texts, a.H = (int32_t)p->heads, a.KV = (int32_t)p->kv_heads;
  a.many = a.H / a.KV;
  a.parts = 1;
  a.scale = (float)p->scale, a.cap = (float)p->cap;
  return TMS_OK;
}

static int run_attention(const tms_attention* p, const AttnArgs& a, AttnPass pass, hipStream_t st) {
  if (p->dtype == TMS_DTYPE_F16) return attn_run_f16(a, (int)p->width, pass, st);
  if (p->dtype == TMS_DTYPE_BF16) return attn_run_bf16(a, (int)p->width, pass, st);
  return attn_run_f32(a, (int)p->width, pass, st);
}

}  // namespace tms

using namespace tms;

extern "C" int64_t tms_attention_stats(int64_t tokens, int64_t heads, int64_t kv_heads) {
  return tokens <= 0 || heads <= 0 || kv_heads <= 0 ? 0 : up_to(heads * tokens, 4) + (heads + kv_heads) * kAttnNorms;
}

// Bytes of delta, and of the parts' sums.
static int64_t delta_bytes(int64_t tokens, int64_t heads) { return up_to(tokens * heads * 4, 256); }
extern "C" int64_t tms_attention_workspace_size(int64_t texts, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t width) {
  if (texts < 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || width <= 0) return 0;
  const int64_t parts = attn_parts(tokens, texts, kv_heads, heads / kv_heads);
  return delta_bytes(tokens, heads) + (parts > 1 ? parts * 2 * tokens * kv_heads * width * 4 : 0);
}

static float* norms_of(const AttnArgs& a, float* stats) {
  return stats && a.slopes && a.cap == 0.f && attn_reaches(a.T, a.B) ? stats + up_to((int64_t)a.H * a.T, 4) : nullptr;
}

extern "C" int tms_packed_attention(const tms_attention* attention, void* out, void* low, float* stats, void* stream) {
  const char* fn = "tms_packed_attention";
  AttnArgs a;
  const int rc = check_attention(fn, attention, a);
  if (rc || attention->tokens == 0) return rc;
  if (!out) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)out | (uintptr_t)low | (uintptr_t)stats) % 16) return fail(TMS_ERR_INVALID, "%s: out, low and stats must be 16-byte aligned", fn);
  a.out = out, a.low = low, a.lse = stats;
  a.norms = norms_of(a, stats);
  return run_attention(attention, a, kAttnForward, (hipStream_t)stream);
}

extern "C" int tms_packed_attention_grad(const tms_attention* attention, const void* out, const void* low, const float* stats, const void* grad,
                                         void* workspace, int64_t workspace_bytes, void* dq, void* dk, void* dv, void* stream) {
  const char* fn = "tms_packed_attention_grad";
  AttnArgs a;
  int rc = check_attention(fn, attention, a);
  if (rc || attention->tokens == 0 || (!dq && !dk && !dv)) return rc;
  if (!out || !stats || !grad || (!low && attention->dtype != TMS_DTYPE_F32)) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)out | (uintptr_t)low | (uintptr_t)stats | (uintptr_t)grad | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16)
    return fail(TMS_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  const int64_t bytes = tms_attention_workspace_size(attention->texts, attention->tokens, attention->heads, attention->kv_heads, attention->width);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < bytes)
    return fail(TMS_ERR_INVALID, "%s: a workspace of %lld bytes is needed, 256-byte aligned", fn, (long long)bytes);
  a.out = const_cast<void*>(out), a.low = const_cast<void*>(low), a.lse = const_cast<float*>(stats);
  a.norms = norms_of(a, a.lse);
  a.grad = grad, a.delta = (float*)workspace;
  a.parts = (int32_t)attn_parts(a.T, a.B, a.KV, a.many);
  a.sums = (float*)((uint8_t*)workspace + delta_bytes(a.T, a.H));
  a.dq = dq, a.dk = dk, a.dv = dv;
  if ((rc = run_attention(attention, a, kAttnDq, (hipStream_t)stream)) || (!dk && !dv)) return rc;  // it leaves delta, too
  return run_attention(attention, a, kAttnDkv, (hipStream_t)stream);
}
