// ec_prefix.cu -- texts behind a shared prefix.
//
// llama::embed (llama.lisp:296-344) computes every text from its first token.
// With causal attention the keys and values of a common prefix do not depend
// on what follows, so they are computed once (ec_prefix_open), stay in the
// pages of a cache, and each text's forward runs over its own tokens alone:
// P + L tokens of GEMMs become L.  The texts share the prefix's whole pages by
// count and copy its last partly filled one (ec_kv_fork).
#include "ec_prefix.h"

#include <algorithm>
#include <vector>

#include "../../include/embedcuda.h"
#include "ec_ops.h"

namespace ec {

static size_t up256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int prefix_grow(Device& d) {
  if (d.prefixes) return EC_OK;
  const ModelW& m = d.model;
  const int width = (m.max_pos + kPrefixPage - 1) / kPrefixPage, nslots = kPrefixes + kPrefixSeqs;
  // every prefix and text may end inside a page, and a text copies one
  const int pages = kPrefixes * width + kPrefixTokens / kPrefixPage + 2 * kPrefixSeqs;
  const size_t half = static_cast<size_t>(m.layers) * pages * kPrefixPage * m.kv_heads * m.hd * 2;
  const int64_t kv_work = ec_kv_work_size(pages, nslots);
  if (kv_work < 0) return static_cast<int>(kv_work);
  const size_t att = attention_work_most(m.hd);
  size_t o = 0;
  auto take = [&](size_t n) { const size_t at = o; o += up256(n); return at; };
  const size_t at_k = take(half), at_v = take(half);
  const size_t zero = o;  // from here on all zero at first
  const size_t at_tab = take(static_cast<size_t>(nslots) * width * 4), at_len = take(nslots * 4),
               at_ref = take(static_cast<size_t>(pages) * 4), at_kw = take(static_cast<size_t>(kv_work)),
               at_att = take(att), at_add = take(kPrefixSeqs * 4), at_st = take(3 * 8);
  const size_t at_slots = take((kPrefixes + 1) * kPrefixSeqs * 4);
  PrefixPool* p = new PrefixPool();
  p->bytes = o;
  int rc = dev_alloc(d, &p->mem, o, "prefix cache");
  if (rc) {
    delete p;
    return rc;
  }
  d.prefixes = p;  // prefix_drop takes it back from here on
  char* b = static_cast<char*>(p->mem);
  std::vector<int32_t> slots((kPrefixes + 1) * kPrefixSeqs);
  for (int r = 0; r <= kPrefixes; ++r)
    for (int i = 0; i < kPrefixSeqs; ++i) slots[r * kPrefixSeqs + i] = r < kPrefixes ? r : kPrefixes + i;
  if (cudaHostAlloc(reinterpret_cast<void**>(&p->status_host), 64, cudaHostAllocPortable) != cudaSuccess) {
    cudaGetLastError();
    p->status_host = nullptr;
    rc = set_error(EC_ENOMEM, "pinned staging of the prefix cache failed");
  }
  if (!rc) rc = check_cuda(cudaMemsetAsync(b + zero, 0, o - zero, d.stream), "prefix cache");
  if (!rc)
    rc = check_cuda(cudaMemcpyAsync(b + at_slots, slots.data(), slots.size() * 4, cudaMemcpyHostToDevice, d.stream),
                    "prefix cache");
  if (!rc) rc = check_cuda(cudaStreamSynchronize(d.stream), "prefix cache");
  p->work = b + at_att;
  p->work_bytes = att;
  p->slots = reinterpret_cast<int32_t*>(b + at_slots);
  p->add = reinterpret_cast<int32_t*>(b + at_add);
  p->status = reinterpret_cast<int32_t*>(b + at_st);
  if (!rc)
    rc = ec_kv_open(b + at_k, b + at_v, EC_BF16, m.layers, pages, kPrefixPage, m.kv_heads, m.hd,
                    reinterpret_cast<int32_t*>(b + at_tab), nslots, width, reinterpret_cast<int32_t*>(b + at_len),
                    reinterpret_cast<int32_t*>(b + at_ref), b + at_kw, kv_work, &p->handle);
  if (rc) prefix_drop(d);
  return rc;
}

void prefix_drop(Device& d) {
  PrefixPool* p = d.prefixes;
  if (!p) return;
  graphs_clear(d);  // captured forwards point into it
  cudaStreamSynchronize(d.stream);
  if (p->handle) ec_kv_close(p->handle);
  if (p->status_host) cudaFreeHost(p->status_host);
  dev_free(d, p->mem, p->bytes);
  delete p;
  d.prefixes = nullptr;
}

PrefixRun prefix_run(const PrefixPool& p, int slot, bool fill, int longest) {
  PrefixRun r;
  r.handle = p.handle;
  r.first = fill ? 0 : p.len[slot];
  r.longest = longest;
  r.slots = p.slots + (fill ? slot : kPrefixes) * kPrefixSeqs;
  r.work = p.work;
  r.work_bytes = p.work_bytes;
  return r;
}

int prefix_plan(Device& d, PrefixPool& p, int slot, bool fill, const int* lens, int nseq) {
  const int32_t* texts = p.slots + kPrefixes * kPrefixSeqs;
  const int32_t* own = p.slots + slot * kPrefixSeqs;
  int rc = check_cuda(cudaMemcpyAsync(p.add, lens, static_cast<size_t>(nseq) * 4, cudaMemcpyHostToDevice, d.stream),
                      "length upload");
  // also after a forward that failed: the texts' slots are emptied here, not
  // at its end
  if (!rc) rc = ec_kv_free(p.handle, texts, kPrefixSeqs, p.status, d.stream);
  if (!rc) rc = fill ? ec_kv_free(p.handle, own, 1, p.status + 2, d.stream)
                     : ec_kv_fork(p.handle, own, texts, nseq, p.status + 2, d.stream);
  if (!rc) rc = ec_kv_reserve(p.handle, fill ? own : texts, p.add, nseq, p.status + 4, d.stream);
  return rc;
}

int prefix_fetch(Device& d, PrefixPool& p) {
  return check_cuda(cudaMemcpyAsync(p.status_host, p.status, 24, cudaMemcpyDeviceToHost, d.stream), "status download");
}

int prefix_check(const PrefixPool& p) {
  for (int i = 0; i < 3; ++i)
    if (p.status_host[2 * i] != EC_KV_OK)
      return set_error(EC_ECUDA, "prefix cache: page operation %d failed (%d, %d pages)", i, p.status_host[2 * i],
                       p.status_host[2 * i + 1]);
  return EC_OK;
}

// A wait that gave up may have left tiles of the cached attention half counted:
// the next forward would join their parts too early, or never.
void prefix_failed(Device& d, PrefixPool& p) {
  cudaMemsetAsync(p.work, 0, p.work_bytes, d.stream);
  cudaStreamSynchronize(d.stream);
}

// the slot of a prefix id, or -1 with the error set
static int prefix_slot(int id) {
  const PrefixPool* p = G().devs[0]->prefixes;
  for (int s = 0; p && s < kPrefixes; ++s)
    if (p->len[s] && p->id[s] == id) return s;
  set_error(EC_EINVAL, "prefix %d is not open", id);
  return -1;
}

static void prefix_forget(int slot) {
  for (Device* d : G().devs) {
    PrefixPool* p = d->prefixes;
    if (!p) continue;
    cudaSetDevice(d->ordinal);
    graphs_clear(*d);  // captured forwards hold its length
    p->len[slot] = 0;
    if (std::all_of(p->len, p->len + kPrefixes, [](int n) { return n == 0; }))
      prefix_drop(*d);
    else
      ec_kv_free(p->handle, p->slots + slot * kPrefixSeqs, 1, p->status, d->stream);
  }
}

}  // namespace ec

using namespace ec;

static int prefix_open(const int32_t* ids, int n, int* prefix) {
  if (!G().inited) return set_error(EC_ESTATE, "ec_init first");
  if (!ids || !prefix) return set_error(EC_EINVAL, "ids and prefix must not be NULL");
  const ModelW& m = G().devs[0]->model;
  if (!m.family) return set_error(EC_ESTATE, "no model loaded");
  if (m.family != EC_FAMILY_LLAMA)
    return set_error(EC_EUNSUPPORTED, "a shared prefix needs causal attention (the llama family)");
  if (n < 1 || n >= m.max_pos)
    return set_error(EC_EINVAL, "a prefix of %d tokens (1 to %d leave room for a text)", n, m.max_pos - 1);
  int slot = 0;
  for (const PrefixPool* p = G().devs[0]->prefixes; p && slot < kPrefixes && p->len[slot];) ++slot;
  if (slot == kPrefixes) return set_error(EC_ENOMEM, "%d prefixes are open", kPrefixes);
  static int ids_given = 0;
  const int id = ++ids_given;
  const int64_t offsets[2] = {0, n};
  std::vector<float> out(m.out_dim);
  for (Device* d : G().devs) {
    int rc = check_cuda(cudaSetDevice(d->ordinal), "set device");
    if (!rc) rc = prefix_grow(*d);
    if (!rc) rc = embed_on_device(*d, ids, nullptr, {0}, offsets, out.data(), m.out_dim, nullptr, slot, true);
    if (rc) {
      const std::string why = ec_last_error();
      prefix_forget(slot);
      return set_error(rc, "%s", why.c_str());
    }
    graphs_clear(*d);  // captured forwards of the slot's earlier prefix
    d->prefixes->len[slot] = n;
    d->prefixes->id[slot] = id;
  }
  *prefix = id;
  return EC_OK;
}

extern "C" int ec_prefix_open(const int32_t* ids, int n, int* prefix) {
  std::lock_guard<std::mutex> lk(G().mu);
  clear_error();
  return guarded("prefix", [&] { return prefix_open(ids, n, prefix); });
}

extern "C" int ec_prefix_close(int prefix) {
  std::lock_guard<std::mutex> lk(G().mu);
  clear_error();
  if (!G().inited) return set_error(EC_ESTATE, "ec_init first");
  const int slot = prefix_slot(prefix);
  if (slot < 0) return EC_EINVAL;
  prefix_forget(slot);
  return EC_OK;
}

extern "C" int ec_embed_batch_prefix(int prefix, const int32_t* ids, const int64_t* offsets, int nseq, float* out,
                                     int out_stride) {
  std::lock_guard<std::mutex> lk(G().mu);
  clear_error();
  if (!G().inited) return set_error(EC_ESTATE, "ec_init first");
  const int slot = prefix_slot(prefix);
  if (slot < 0) return EC_EINVAL;
  return guarded("batch", [&] { return embed_batch_split(ids, offsets, nseq, out, out_stride, slot); });
}
