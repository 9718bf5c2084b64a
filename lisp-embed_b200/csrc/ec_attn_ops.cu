// ec_attn_ops.cu -- causal grouped-head attention over packed queries, with
// the keys in packed rows (ec_attn_prompt) or in the pages of a cache
// (ec_attn_cached).
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "ec_attn_ops.cuh"

namespace ec {

PFN_cuTensorMapEncodeTiled_v12000 gemm_encode_fn();  // ec_gemm.cu

namespace {

// tensor map of 16-bit rows: dims and strides (bytes) outermost last, box of
// 64 columns by `box` of the outer dimensions
bool encode(CUtensorMap* tm, int dtype, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  auto enc = gemm_init_driver() ? gemm_encode_fn() : nullptr;  // no ec_init needed
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc && enc(tm, dtype == EC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                    const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_rows(CUtensorMap* tm, int dtype, const OpRows& r, int head_dim, int heads, int64_t tokens, int box_heads,
                 int box_tokens) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(tokens)};
  // the stride of a single head or token is never used, but has to be valid
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? r.head : head_dim) * 2,
                                 static_cast<cuuint64_t>(tokens > 1 ? r.token : head_dim) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  return encode(tm, dtype, r.p, 3, dims, strides, box);
}

using FlashFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, FlashArgs);

// Lists of pairs of tiles by sequence are launched plainly.  A CTA that starts
// early, while the kernel before still runs, gets the SM that came free first;
// then CTAs that read the same keys no longer run side by side.  One call after
// the other on the same buffers, 256 prompts of 320 tokens take 255 us (with early
// starts 1.2), 1024 of 130 553 (1.11), 96 texts behind 650 cached tokens 133
// (1.05).  The other launches gain by it (one token 11.3 us, without it 1.2; 8
// prompts of 512 24 us, 1.06; one of 4096 72 us, 1.04).
class PlainLaunch {
 public:
  explicit PlainLaunch(bool plain) : before_(pdl_enabled()), plain_(plain) {
    if (plain_) pdl_set_thread(false);
  }
  ~PlainLaunch() {
    if (plain_) pdl_set_thread(before_);
  }

 private:
  bool before_, plain_;
};

// kernel `id` on device `dev` (its shared memory is set once per device)
int launch_one(int dev, int id, FlashFn fn, int threads, size_t smem, const CUtensorMap& q, const CUtensorMap& k,
               const CUtensorMap& v, const FlashArgs& a, int grid, cudaStream_t st) {
  static std::mutex mu;
  static uint32_t set[64] = {};
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!(set[dev] >> id & 1)) {
      if (int rc = check_cuda(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(smem)),
                              "attention shared memory"))
        return rc;
      set[dev] |= 1u << id;
    }
  }
  return check_cuda(launch_pdl(fn, dim3(grid), dim3(threads), smem, st, q, k, v, a), "attention");
}

// tile sets of 256 rows (kHalves: of short sequences), tiles of 128 rows, tiles of at most 32 .. 4 rows
enum FlashKind { kPairs, kHalves, kTiles, kFew32, kFew16, kFew8, kFew4 };

template <int HD, int NP, typename T>
int launch_token(int dev, int id, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FlashArgs& a, int grid,
                 cudaStream_t st) {
  using Cfg = TokenCfg<HD, NP>;
  return launch_one(dev, id, flash_token_kernel<HD, NP, T>, Cfg::THREADS, Cfg::SMEM, q, k, v, a, grid, st);
}

template <int HD, typename T>
int launch_flash(int dev, FlashKind kind, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FlashArgs& a,
                 int grid, cudaStream_t st) {
  const int id = (HD == 64 ? 0 : 16) + (std::is_same<T, __half>::value ? 8 : 0) + kind;
  int rc;
  switch (kind) {
    case kPairs:
      rc = launch_one(dev, id, flash_kernel<HD, 2, false, T>, FlashCfg<HD, 2>::THREADS, FlashCfg<HD, 2>::SMEM, q, k, v, a, grid, st);
      break;
    case kHalves:
      rc = launch_one(dev, id, flash_kernel<HD, 2, true, T>, FlashCfg<HD, 2>::THREADS, FlashCfg<HD, 2>::SMEM, q, k, v, a, grid, st);
      break;
    case kTiles:
      rc = launch_one(dev, id, flash_kernel<HD, 1, true, T>, FlashCfg<HD, 1>::THREADS, FlashCfg<HD, 1>::SMEM, q, k, v, a, grid, st);
      break;
    case kFew32: rc = launch_token<HD, 32, T>(dev, id, q, k, v, a, grid, st); break;
    case kFew16: rc = launch_token<HD, 16, T>(dev, id, q, k, v, a, grid, st); break;
    case kFew8: rc = launch_token<HD, 8, T>(dev, id, q, k, v, a, grid, st); break;
    default: rc = launch_token<HD, 4, T>(dev, id, q, k, v, a, grid, st);
  }
  return rc;
}

// packed prompts below this many tokens on average run the kernel that leaves
// out halves of blocks (measured beside it)
constexpr int kHalvesBelow = 1024;
// How a call is cut up, from what the host knows
struct FlashPlan {
  FlashKind kind;
  int even, rows_tok;  // tokens of a tile
  int part_rows;
};
// Few rows (a sequence's new tokens and their heads in at most 32 rows): the
// kernels with the operands turned round, in the smallest size that holds them;
// always an even split (64 sequences of up to 8192 tokens 94 us; in 32 rows
// whatever they need 1.1, in tiles of 128 rows 1.23).  More rows in fewer tiles
// than SMs: an even split, which leaves whole what is not worth cutting.  Else
// whole tiles, in pairs where every SM has a pair (one prompt of 16384 tokens 477
// us, in single tiles 1.2); one tile at a time is better for fewer, and where no
// sequence fills more than a tile.
//
// The kind goes by the call's longest sequence and their count.  One call after
// the other, 64 single tokens behind up to 8192 keys take 108 us, with a text of 9 tokens or more among them 160 to
// 170 (its rows pass 32: tiles of 128 rows for all), of 8 tokens 236 (32 rows for
// all); 2048 single tokens behind 500 keys 664, 2049 837 (more than the even
// split's prefix sums hold).  Heads other than 64 and 128 run padded to those, in
// MMAs and shared memory (the bytes from memory are their own): 256 prompts of
// 128 to 512 tokens take 217, 217 and 219 us with heads of 16, 32 and 64, 242
// with 80 and 96, 246 with 128.
FlashPlan flash_plan(const KvCache* c, int64_t tokens, int q_heads, int kv_heads, int nseq, int max_new, int num_sms) {
  const int group = q_heads / kv_heads;
  FlashPlan p{kTiles, 0, 128 / group, 128};
  if (c && nseq <= FlashCfg<128, 1>::MAX_SEQS) {
    const int64_t tiles = (tokens / p.rows_tok + nseq) * kv_heads;
    const int64_t few = static_cast<int64_t>(std::max(1, max_new)) * group;  // rows of a sequence's new tokens
    // unit counts of the split are 32-bit
    const int64_t most = (static_cast<int64_t>(c->width) * c->page_size + 127) / 128 + 8;
    const bool fits = (tokens + nseq) * kv_heads * most < (int64_t(1) << 30);
    if (fits && few <= 32) {
      p.kind = few <= 4 ? kFew4 : few <= 8 ? kFew8 : few <= 16 ? kFew16 : kFew32;
      p.part_rows = few <= 4 ? 4 : few <= 8 ? 8 : few <= 16 ? 16 : 32;
      p.rows_tok = p.part_rows / group;
      p.even = 1;
    } else if (fits && tiles <= num_sms) {
      p.even = 1;
    }
  }
  if (!p.even && tokens > static_cast<int64_t>(nseq) * p.rows_tok &&
      (tokens / (2 * p.rows_tok) + nseq) * kv_heads >= num_sms)
    p.kind = !c && tokens < static_cast<int64_t>(nseq) * kHalvesBelow ? kHalves : kPairs;
  return p;
}

size_t part_bytes(int rows, int hd) { return static_cast<size_t>(2) * kMaxCtas * rows * hd * 4; }

}  // namespace

size_t attention_work_bytes(const KvCache& c, int64_t tokens, int q_heads, int nseq, int max_new) {
  const FlashPlan p = flash_plan(&c, tokens, q_heads, c.heads, nseq, max_new, kMaxCtas);
  if (!p.even) return 256;
  return part_bytes(p.part_rows, c.head_dim <= 64 ? 64 : 128) + part_bytes(p.part_rows, 1) + kMaxCtas * 4;
}

namespace {
thread_local unsigned* t_status_word = nullptr;

// the word that ec_op_status asks on device `dev`, the current one
int caller_status_word(int dev, unsigned** word) {
  static std::atomic<unsigned*> words[64] = {};
  *word = words[dev].load(std::memory_order_relaxed);
  if (*word) return EC_OK;
  void* p = nullptr;
  if (int rc = check_cuda(cudaGetSymbolAddress(&p, g_op_status), "operator status")) return rc;
  words[dev].store(*word = static_cast<unsigned*>(p), std::memory_order_relaxed);
  return EC_OK;
}
}  // namespace
OpStatusWord::OpStatusWord(unsigned* word) { t_status_word = word; }
OpStatusWord::~OpStatusWord() { t_status_word = nullptr; }

int op_status_mark(unsigned code) {
  return check_cuda(cudaMemcpyToSymbol(g_op_status, &code, sizeof code), "operator status");
}

size_t attention_work_most(int head_dim) {
  return part_bytes(128, head_dim <= 64 ? 64 : 128) + part_bytes(128, 1) + kMaxCtas * 4;
}

int attention_counts() { return kMaxCtas; }

int run_attention(const AttnOp& op, cudaStream_t st) {
  const KvCache* c = op.cache;
  const int num_sms = std::min(op.num_sms, kMaxCtas);
  const FlashPlan p = flash_plan(c, op.tokens, op.q_heads, op.kv_heads, op.nseq, op.max_new, num_sms);
  const int group = op.q_heads / op.kv_heads, hd = op.head_dim <= 64 ? 64 : 128;
  CUtensorMap tq, tk, tv;
  bool ok = encode_rows(&tq, op.dtype, op.q, op.head_dim, op.q_heads, op.tokens, group, p.rows_tok);
  if (c) {
    const cuuint64_t row = static_cast<cuuint64_t>(c->heads) * c->head_dim * 2;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->head_dim), static_cast<cuuint64_t>(c->heads),
                                static_cast<cuuint64_t>(c->page_size),
                                static_cast<cuuint64_t>(c->layers) * static_cast<cuuint64_t>(c->pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c->head_dim) * 2, row, row * c->page_size};
    const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(c->page_size), 1};
    ok = ok && encode(&tk, c->dtype, c->k, 4, dims, strides, box) && encode(&tv, c->dtype, c->v, 4, dims, strides, box);
  } else {
    ok = ok && encode_rows(&tk, op.dtype, op.k, op.head_dim, op.kv_heads, op.tokens, 1, 128) &&
         encode_rows(&tv, op.dtype, op.v, op.head_dim, op.kv_heads, op.tokens, 1, 128);
  }
  if (!ok) return set_error(EC_EINVAL, "the attention's strides cannot be described to the TMA");
  FlashArgs a{};
  a.out = const_cast<void*>(op.out.p), a.ot = op.out.token, a.oh = op.out.head;
  a.wide = op_aligned(a.out, 32) && a.ot % 16 == 0 && a.oh % 16 == 0 && op.head_dim % 16 == 0;
  a.q = op.q.p, a.qt = op.q.token, a.qh = op.q.head;
  a.k = c ? c->k : op.k.p, a.kt = op.k.token, a.kh = op.k.head;
  a.v = c ? c->v : op.v.p, a.vt = op.v.token, a.vh = op.v.head;
  a.lse = op.lse;
  a.status = t_status_word;
  if (!a.status)
    if (int rc = caller_status_word(op.device, &a.status)) return rc;
  a.cu = op.cu, a.slots = op.slots;
  a.tokens = static_cast<int>(op.tokens), a.nseq = op.nseq;
  a.group = group, a.rows_tok = p.rows_tok, a.q_heads = op.q_heads, a.kv_heads = op.kv_heads;
  a.head_dim = op.head_dim;
  a.scale_log2 = op.scale * 1.4426950408889634f;
  if (c) {
    a.paged = 1;
    a.lens = c->lens, a.tables = c->tables, a.width = c->width, a.nslots = c->slots;
    a.pages = c->pages, a.page_size = c->page_size;
    a.page0 = op.layer * c->pages, a.page_end = c->layers * c->pages;
  }
  const int sets = p.rows_tok * (p.kind == kPairs || p.kind == kHalves ? 2 : 1);
  int64_t grid = (op.tokens / sets + op.nseq) * op.kv_heads;
  if (grid >= INT32_MAX / 2)
    return set_error(EC_EINVAL, "%lld tokens of %d sequences and %d key heads: too many for one call",
                     static_cast<long long>(op.tokens), op.nseq, op.kv_heads);
  if (p.even) {
    char* w = static_cast<char*>(op.work);
    a.even = 1;
    a.min_chunk = 4;
    a.over = 1;
    a.part_rows = p.part_rows;
    // the counts, which have to be zero, lie in the same place for every kind
    // of call that shares the workspace
    a.arrived = reinterpret_cast<int*>(w);
    a.part_o = reinterpret_cast<float*>(w + kMaxCtas * 4);
    a.part_l = reinterpret_cast<float*>(w + kMaxCtas * 4 + part_bytes(p.part_rows, hd));
    static_assert(kMaxCtas * 4 % 32 == 0, "parts are written 32 bytes at a time");
    grid = num_sms;
  }
  const int ctas = static_cast<int>(std::min<int64_t>(grid, num_sms));
  const PlainLaunch launch((p.kind == kPairs || p.kind == kHalves) && op.nseq > kFlashFew);
  if (op.dtype == EC_BF16)
    return hd == 64 ? launch_flash<64, __nv_bfloat16>(op.device, p.kind, tq, tk, tv, a, ctas, st)
                    : launch_flash<128, __nv_bfloat16>(op.device, p.kind, tq, tk, tv, a, ctas, st);
  return hd == 64 ? launch_flash<64, __half>(op.device, p.kind, tq, tk, tv, a, ctas, st)
                  : launch_flash<128, __half>(op.device, p.kind, tq, tk, tv, a, ctas, st);
}

namespace {

int check_heads(int q_heads, int kv_heads) {
  if (q_heads < 1 || kv_heads < 1 || q_heads > 1024 || q_heads % kv_heads || q_heads / kv_heads > 128)
    return set_error(EC_EINVAL, "%d query heads over %d key heads (a multiple of at most 128)", q_heads, kv_heads);
  return EC_OK;
}

int check_attention(AttnOp& op, int64_t tokens, int nseq, float scale) {
  if (op.dtype != EC_BF16 && op.dtype != EC_F16)
    return set_error(EC_EINVAL, "attention takes bf16 or f16, not dtype %d", op.dtype);
  if (tokens < 0 || tokens > (1 << 30) || nseq < 0 || nseq > (1 << 24))
    return set_error(EC_EINVAL, "bad token or sequence count");
  if (op.head_dim < 8 || op.head_dim > 128 || op.head_dim % 8)
    return set_error(EC_EINVAL, "head_dim %d (supported: multiples of 8 up to 128)", op.head_dim);
  if (int rc = check_heads(op.q_heads, op.kv_heads)) return rc;
  if (!std::isfinite(scale) || scale < 0.f) return set_error(EC_EINVAL, "scale must be finite and >= 0 (0: 1 / sqrt(head_dim))");
  if (int rc = op_check_rows("q", op.q, tokens, op.q_heads, op.head_dim)) return rc;
  if (int rc = op_check_rows("out", op.out, tokens, op.q_heads, op.head_dim)) return rc;
  if (!op_rows_apart(op.out.token, op.out.head, tokens, op.q_heads, op.head_dim))
    return set_error(EC_EINVAL, "out's tokens overlap (strides %lld / %lld)", static_cast<long long>(op.out.token),
                     static_cast<long long>(op.out.head));
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
  unsigned v = 0;
  if (int rc = check_cuda(cudaMemcpyFromSymbol(&v, g_op_status, sizeof v), "operator status")) return rc;
  if (v == 0) return EC_OK;
  const unsigned zero = 0;
  if (int rc = check_cuda(cudaMemcpyToSymbol(g_op_status, &zero, sizeof zero), "operator status")) return rc;
  return set_error(v == kDevBadArg ? EC_ECUDA : EC_ETIMEOUT, "a wait inside an attention kernel gave up (code %u)", v);
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
  op.device = dev.ordinal(), op.num_sms = dev.num_sms();
  return run_attention(op, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t ec_attn_cached_work_size(int handle, int64_t tokens, int q_heads, int nseq, int max_new) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (tokens < 0 || tokens > (1 << 30) || nseq < 0 || nseq > (1 << 24) || max_new < 0)
    return set_error(EC_EINVAL, "bad attention shape");
  if (int rc = check_heads(q_heads, c->heads)) return rc;
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
  if (!work || !op_aligned(work, 32) || work_bytes < need)
    return set_error(EC_EINVAL, "work must be 32-byte aligned and hold %lld bytes", static_cast<long long>(need));
  if (!slots && nseq > c->slots) return set_error(EC_EINVAL, "%d sequences, the cache has %d slots", nseq, c->slots);
  if (tokens == 0 || nseq == 0) return EC_OK;
  op.work = work, op.work_bytes = static_cast<size_t>(work_bytes);
  op.scale = scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(c->head_dim));
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {q, out, lse, cu, slots, work})) return rc;
  op.device = dev.ordinal(), op.num_sms = dev.num_sms();
  return run_attention(op, static_cast<cudaStream_t>(stream));
}
