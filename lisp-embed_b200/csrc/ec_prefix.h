// ec_prefix.h -- keys and values of prefixes that many texts share (the
// instruction in front of every query), kept on a device in a paged cache.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ec_state.h"

namespace ec {

constexpr int kPrefixes = 8;        // open at a time
constexpr int kPrefixSeqs = 512;    // texts of one forward
constexpr int kPrefixTokens = 32768;  // their tokens
constexpr int kPrefixPage = 32;

// The cache of one device: slot p < kPrefixes holds prefix p, slot kPrefixes +
// i text i of the running forward.  One device block, laid out by prefix_grow.
struct PrefixPool {
  void* mem = nullptr;
  size_t bytes = 0;
  int handle = 0;                 // of ec_kv_open
  void* work = nullptr;           // of ec_attn_cached
  size_t work_bytes = 0;
  int32_t* slots = nullptr;       // [kPrefixes + 1][kPrefixSeqs]: row p is all p, the last row the texts' slots
  int32_t* add = nullptr;         // [kPrefixSeqs] lengths of the running forward
  int32_t* status = nullptr;      // [3][2] of its page operations
  int32_t* status_host = nullptr;
  int len[kPrefixes] = {};        // tokens of an open prefix, 0: closed
  int id[kPrefixes] = {};         // what ec_prefix_open returned
};

// what the forward's attention needs
struct PrefixRun {
  int handle, first, longest;     // position of the first token, longest sequence
  const int32_t* slots;
  void* work;
  size_t work_bytes;
};

// the pool of d's model, made at the first prefix
int prefix_grow(Device& d);
// no prefix is open any more, or the model goes away
void prefix_drop(Device& d);
PrefixRun prefix_run(const PrefixPool& p, int slot, bool fill, int longest);
// enqueue the pages of a forward: the last one's texts leave, nseq texts of
// lens[] (pinned) tokens come in behind the prefix; `fill`: the prefix itself
int prefix_plan(Device& d, PrefixPool& p, int slot, bool fill, const int* lens, int nseq);
int prefix_fetch(Device& d, PrefixPool& p);  // enqueue the download of the page operations' status
int prefix_check(const PrefixPool& p);       // after the stream was waited for
void prefix_failed(Device& d, PrefixPool& p);  // after a forward that gave up

}  // namespace ec
