// ec_attn_ops.cu -- causal grouped-head attention over packed queries, with
// the keys in packed rows (ec_attn_prompt) or in the pages of a cache
// (ec_attn_cached).
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "ec_ops.h"

namespace ec {
namespace {

struct AttnOpArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  int64_t qt, qh, kt, kh, vt, vh, ot, oh;
  int64_t tokens;
  int q_heads, group, head_dim, nseq;
  const int32_t *cu, *slots;
  float scale;
  KvCache c;  // c.k nullptr: packed keys
  int layer;
};

template <typename T>
__device__ __forceinline__ float ld(const T* p);
template <>
__device__ __forceinline__ float ld(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float ld(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void st(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void st(__half* p, float v) { *p = __float2half_rn(v); }

// One warp per (token, query head): the keys one after the other, running
// maximum and sum, four elements of the head per lane.
template <typename T>
__global__ void attn_rows_kernel(const AttnOpArgs a) {
  const int64_t w = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= a.tokens * a.q_heads) return;
  const int64_t t = w / a.q_heads;
  const int h = static_cast<int>(w % a.q_heads), kvh = h / a.group;
  int lo = 0, hi = a.nseq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  const int64_t begin = max(a.cu[lo], 0), end = a.cu[lo + 1];
  if (t < begin || t >= end) return;  // behind the last sequence
  int64_t last;                       // keys [0, last) are seen
  const int32_t* table = nullptr;
  if (a.c.k) {
    const int s = a.slots ? a.slots[lo] : lo;
    if (s < 0 || s >= a.c.slots) last = 0;
    else {
      const int64_t len = min(max(int64_t(a.c.lens[s]), int64_t(0)), int64_t(a.c.width) * a.c.page_size);
      last = len - (end - t) + 1;
      table = a.c.tables + static_cast<int64_t>(s) * a.c.width;
    }
  } else {
    last = t - begin + 1;
  }
  const T* q = static_cast<const T*>(a.q) + t * a.qt + h * a.qh;
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = lane + 32 * i < a.head_dim ? ld(q + lane + 32 * i) : 0.f;
  for (int64_t j = 0; j < last; ++j) {
    const T *k, *v;
    if (table) {
      const int page = table[j / a.c.page_size];
      const int64_t row = a.c.heads * static_cast<int64_t>(a.head_dim);
      const bool there = page >= 0 && page < a.c.pages;
      const int64_t at = ((static_cast<int64_t>(a.layer) * a.c.pages + page) * a.c.page_size + j % a.c.page_size) * row +
                         kvh * a.head_dim;
      k = there ? static_cast<const T*>(a.c.k) + at : nullptr;
      v = there ? static_cast<const T*>(a.c.v) + at : nullptr;
    } else {
      k = static_cast<const T*>(a.k) + (begin + j) * a.kt + kvh * a.kh;
      v = static_cast<const T*>(a.v) + (begin + j) * a.vt + kvh * a.vh;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k && lane + 32 * i < a.head_dim) s += qv[i] * ld(k + lane + 32 * i);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale;
    const float mn = fmaxf(m, s);
    const float c = m == -INFINITY ? 0.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = v && lane + 32 * i < a.head_dim ? ld(v + lane + 32 * i) : 0.f;
      o[i] = o[i] * c + p * x;
    }
    m = mn;
  }
  T* out = static_cast<T*>(a.out) + t * a.ot + h * a.oh;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.head_dim) st(out + lane + 32 * i, l > 0.f ? o[i] / l : l == 0.f ? 0.f : NAN);
  if (a.lse && lane == 0) a.lse[t * a.q_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t attention_work_bytes(const KvCache&, int64_t, int, int, int) { return 256; }

int run_attention(const AttnOp& op, int, cudaStream_t st) {
  AttnOpArgs a{};
  a.q = op.q.p, a.qt = op.q.token, a.qh = op.q.head;
  a.k = op.k.p, a.kt = op.k.token, a.kh = op.k.head;
  a.v = op.v.p, a.vt = op.v.token, a.vh = op.v.head;
  a.out = const_cast<void*>(op.out.p), a.ot = op.out.token, a.oh = op.out.head;
  a.lse = op.lse;
  a.tokens = op.tokens, a.q_heads = op.q_heads, a.group = op.q_heads / op.kv_heads, a.head_dim = op.head_dim;
  a.nseq = op.nseq, a.cu = op.cu, a.slots = op.slots, a.scale = op.scale, a.layer = op.layer;
  if (op.cache) a.c = *op.cache;
  const int64_t warps = op.tokens * op.q_heads;
  const unsigned grid = static_cast<unsigned>((warps + 7) / 8);
  if (op.dtype == EC_BF16) attn_rows_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  else attn_rows_kernel<__half><<<grid, 256, 0, st>>>(a);
  return check_cuda(cudaGetLastError(), "attention");
}

namespace {

int check_attention(const AttnOp& op, int64_t tokens, int nseq, float scale) {
  if (op.dtype != EC_BF16 && op.dtype != EC_F16)
    return set_error(EC_EINVAL, "attention takes bf16 or f16, not dtype %d", op.dtype);
  if (tokens < 0 || tokens > INT32_MAX || nseq < 0) return set_error(EC_EINVAL, "bad token or sequence count");
  if (op.head_dim < 8 || op.head_dim > 128 || op.head_dim % 8)
    return set_error(EC_EINVAL, "head_dim %d (supported: multiples of 8 up to 128)", op.head_dim);
  if (op.q_heads < 1 || op.kv_heads < 1 || op.q_heads > 1024 || op.q_heads % op.kv_heads || op.q_heads / op.kv_heads > 128)
    return set_error(EC_EINVAL, "%d query heads over %d key heads (a multiple of at most 128)", op.q_heads, op.kv_heads);
  if (!std::isfinite(scale) || scale < 0.f) return set_error(EC_EINVAL, "scale must be finite and >= 0 (0: 1 / sqrt(head_dim))");
  if (int rc = op_check_rows("q", op.q, tokens, op.q_heads, op.head_dim)) return rc;
  if (int rc = op_check_rows("out", op.out, tokens, op.q_heads, op.head_dim)) return rc;
  if (!op.cu && tokens && nseq) return set_error(EC_EINVAL, "cu is NULL");
  if (!op_aligned(op.cu, 4) || !op_aligned(op.slots, 4) || !op_aligned(op.lse, 4))
    return set_error(EC_EINVAL, "cu, slots and lse must be 4-byte aligned");
  return EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" int ec_op_status(void) {
  clear_error();
  if (int rc = check_cuda(cudaDeviceSynchronize(), "operators")) return rc;
  return EC_OK;
}

extern "C" int ec_attn_prompt(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                              int64_t k_head, const void* v, int64_t v_token, int64_t v_head, void* out,
                              int64_t o_token, int64_t o_head, float* lse, int dtype, int64_t tokens, int q_heads,
                              int kv_heads, int head_dim, const int32_t* cu, int nseq, float scale, void* stream) {
  clear_error();
  AttnOp op{};
  op.dtype = dtype, op.head_dim = head_dim, op.q_heads = q_heads, op.kv_heads = kv_heads;
  op.q = {q, q_token, q_head}, op.k = {k, k_token, k_head}, op.v = {v, v_token, v_head};
  op.out = {out, o_token, o_head}, op.lse = lse;
  op.tokens = tokens, op.cu = cu, op.nseq = nseq;
  if (int rc = check_attention(op, tokens, nseq, scale)) return rc;
  if (int rc = op_check_rows("k", op.k, tokens, kv_heads, head_dim)) return rc;
  if (int rc = op_check_rows("v", op.v, tokens, kv_heads, head_dim)) return rc;
  if (tokens == 0 || nseq == 0) return EC_OK;
  op.scale = scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(head_dim));
  OpDevice dev;
  if (int rc = dev.enter({q, k, v, out, lse, cu})) return rc;
  return run_attention(op, dev.num_sms(), static_cast<cudaStream_t>(stream));
}

extern "C" int64_t ec_attn_cached_work_size(int handle, int64_t tokens, int q_heads, int nseq, int max_new) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (tokens < 0 || tokens > INT32_MAX || nseq < 0 || max_new < 0 || q_heads < 1 || q_heads % c->heads)
    return set_error(EC_EINVAL, "bad attention shape");
  return static_cast<int64_t>(attention_work_bytes(*c, tokens, q_heads, nseq, max_new));
}

extern "C" int ec_attn_cached(int handle, int layer, const void* q, int64_t q_token, int64_t q_head, void* out,
                              int64_t o_token, int64_t o_head, float* lse, int64_t tokens, int q_heads,
                              const int32_t* cu, const int32_t* slots, int nseq, int max_new, float scale, void* work,
                              int64_t work_bytes, void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (layer < 0 || layer >= c->layers) return set_error(EC_EINVAL, "layer %d of %d", layer, c->layers);
  AttnOp op{};
  op.dtype = c->dtype, op.head_dim = c->head_dim, op.q_heads = q_heads, op.kv_heads = c->heads;
  op.q = {q, q_token, q_head}, op.out = {out, o_token, o_head}, op.lse = lse;
  op.tokens = tokens, op.cu = cu, op.nseq = nseq, op.slots = slots, op.max_new = max_new;
  op.cache = c.get(), op.layer = layer;
  if (int rc = check_attention(op, tokens, nseq, scale)) return rc;
  if (max_new < 0) return set_error(EC_EINVAL, "max_new is negative");
  const int64_t need = static_cast<int64_t>(attention_work_bytes(*c, tokens, q_heads, nseq, max_new));
  if (!work || !op_aligned(work, 16) || work_bytes < need)
    return set_error(EC_EINVAL, "work must be 16-byte aligned and hold %lld bytes", static_cast<long long>(need));
  if (!slots && nseq > c->slots) return set_error(EC_EINVAL, "%d sequences, the cache has %d slots", nseq, c->slots);
  if (tokens == 0 || nseq == 0) return EC_OK;
  op.work = work, op.work_bytes = static_cast<size_t>(work_bytes);
  op.scale = scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(c->head_dim));
  OpDevice dev;
  if (int rc = dev.enter({c->refs, q, out, lse, cu, slots, work})) return rc;
  return run_attention(op, dev.num_sms(), static_cast<cudaStream_t>(stream));
}
