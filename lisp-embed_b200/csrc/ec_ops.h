// ec_ops.h -- what the operators over caller-owned device buffers (rotary
// positions, prompt and cached attention, the paged cache) share: argument
// checks, the device of a call, and the description behind a cache handle.
//
// Like ec_flat_search_noalloc they need no ec_init, allocate no device memory
// and only enqueue work on the caller's stream.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>
#include <memory>
#include <new>

#include "ec_state.h"

namespace ec {

// Makes the device that holds `p` current for one call and puts the caller's
// device back afterwards: a host that drives several GPUs passes buffers of a
// device other than the current one.
class OpDevice {
 public:
  // EC_OK, or an error when one of the non-null pointers is not device memory
  // or lies on another device than the first (or than `dev`)
  int enter(std::initializer_list<const void*> ptrs, int dev = -1);
  ~OpDevice();
  int num_sms() const { return sms_; }
  int ordinal() const { return dev_; }

 private:
  int prev_ = -1, dev_ = -1, sms_ = 0;
};

// No C++ exception leaves the C ABI: a host allocation that fails is EC_ENOMEM.
template <class F>
int guarded(const char* what, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return set_error(EC_ENOMEM, "%s: out of host memory", what);
  } catch (const std::exception& e) {
    return set_error(EC_EINVAL, "%s: %s", what, e.what());
  }
}

// element size of EC_F32 / EC_BF16 / EC_F16, 0 for another code
inline int op_elem_size(int dtype) {
  return dtype == EC_F32 ? 4 : dtype == EC_BF16 || dtype == EC_F16 ? 2 : 0;
}
inline bool op_aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Heads of a packed row: element (token, head, i) lies at
// p[token * token_stride + head * head_stride + i].
struct OpRows {
  const void* p;
  int64_t token, head;
};
// checks pointer, 16-byte base and strides (in elements of 2 bytes), and that
// heads do not overlap; the stride of a single token or head, which is never
// used, becomes 0
int op_check_rows(const char* name, OpRows& r, int64_t tokens, int heads, int head_dim);
// rows that are written: no two heads of any tokens may overlap either
bool op_rows_apart(int64_t token, int64_t head, int64_t tokens, int heads, int head_dim);

// a cache as ec_kv_open describes it; the memory is the caller's
struct KvCache {
  void *k, *v;         // [layers][pages][page_size][heads][head_dim]
  int dtype, layers, pages, page_size, heads, head_dim;
  int32_t* tables;     // [slots][width]
  int slots, width;
  int32_t* lens;       // [slots]
  int32_t* refs;       // [pages]
  int32_t* work;       // scratch of the page operations
};
struct KvOpen : KvCache {
  explicit KvOpen(const KvCache& c) : KvCache(c) {}
  // the device that all its buffers were found on, by the first call that
  // launches anything (a handle's pointers never change); -1: not looked at
  mutable std::atomic<int> device{-1};
};
// the cache behind a handle (held until the pointer goes away), or nullptr
// with the error set
std::shared_ptr<const KvOpen> kv_find(int handle);
// dev.enter for a call on cache c with these buffers
int kv_enter(OpDevice& dev, const KvOpen& c, std::initializer_list<const void*> ptrs);

// ---- attention over packed queries (ec_attn_ops.cu) --------------------------
struct AttnOp {
  int dtype, head_dim, q_heads, kv_heads;
  OpRows q, k, v, out;  // k and v unused with a cache
  float* lse;           // [tokens][q_heads] or nullptr
  int64_t tokens;
  const int32_t* cu;    // [nseq + 1]
  int nseq;
  float scale;
  // keys in a cache (nullptr: the packed rows k and v)
  const KvCache* cache;
  int layer;
  const int32_t* slots;  // [nseq] or nullptr (sequence s is slot s)
  int max_new;
  void* work;
  size_t work_bytes;
  int device, num_sms;  // of the call (OpDevice)
};
int run_attention(const AttnOp& op, cudaStream_t st);
size_t attention_work_bytes(const KvCache& c, int64_t tokens, int q_heads, int nseq, int max_new);
// While one lives, this thread's attention calls mark `word` (of the call's
// device) when a wait gives up, not the word that ec_op_status asks: a forward
// of the library and a caller's own calls do not hear of each other's.
class OpStatusWord {
 public:
  explicit OpStatusWord(unsigned* word);
  ~OpStatusWord();
};
// marks the word that ec_op_status asks, on the current device (for tests)
int op_status_mark(unsigned code);
// enough for every call on a cache of this head size
size_t attention_work_most(int head_dim);
// the int32 counts at the start of a workspace, zero between calls
int attention_counts();

}  // namespace ec
