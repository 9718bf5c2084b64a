// ec_attn_ops.cuh -- causal grouped-head attention on the 5th-generation
// tensor cores, keys in packed rows or in the pages of a cache.
//
//   o_r = sum_j softmax_j(scale * q_r . k_j) v_j over the keys that row r sees
//
// A tile is 128 query rows of one key head: R = 128 / G tokens with their G
// query heads (row = token * G + head), so that the heads of a group share
// every key and value that is read.  A CTA takes NT tiles of consecutive
// tokens through the 128-key blocks that they see:
//
//   S = Q K^T      tcgen05.mma, Q and K from shared memory  -> TMEM
//   P = exp2(..)   one thread per row: 128 scores to registers, running
//                  maximum and sum without any exchange; P (16 bits) goes
//                  back to TMEM over S's first 64 columns
//   O += P V       tcgen05.mma, P from TMEM, V from shared memory -> TMEM
//
// NT = 2: while one tile's rows go through the exponential, the tensor core
// works on the other tile's P V and next S.  NT = 1 (few queries): S is
// double-buffered instead, so the next block's scores are there when the
// current block's exponentials are done.
//
// O is rescaled only when a row's maximum grows by more than 2^8 (P stays
// below 2^8 in its 16 bits; sums are fp32).
//
// Warps: 4 per tile softmax, then one each for the loads, the MMAs and the
// work list.  NT = 2 has four more that divide O by the row sums and write it,
// and the MMA warp issues a tile's first scores of the next tile set as soon as
// the tile is through: a softmax warp has nothing to wait for between two sets
// (a trace had shown 35% of its time between its last exponentials and the next
// scores).  All waits are bounded.
//
// Times here are of one pass by itself with cold caches (a graph replayed after a
// write larger than L2) where nothing else is said.  "The corpus" is 256 prompts
// of 128 to 512 tokens (71060 in all) of 16 query and 8 key heads of 128; what an
// alternative cost is said as a factor of the time without it.
//
// What bounds it: the chain of a block.  16384 tokens of 8 heads of 128 take 477
// us; the MMAs alone took 344 (the peak rate 328), the softmax warps alone 426,
// and no unit is full then (tensor pipe 53%, special functions 40%, issue 42%).
// A block costs a warp 128 exponentials (three of four on the special-function
// unit, 16 a cycle and SM, every fourth on the FMA units; all on the former
// 1.10, every third on the FMA units 1.04), the scale, sum and packing two
// values an instruction, the maximum three, two reads of the scores from TMEM,
// which keep a thread within 168 registers, and the rescaling of O.  In short
// tile sets (the corpus 252 us, 134 for its bytes) each set's start counts: its
// queries have one buffer and are asked for within the key stream, once the last
// scores of the set before are done; and a set of one tile runs its scores,
// exponentials and P V one after the other.
#pragma once

#include <cuda_fp16.h>

#include <climits>

#include "ec_fa.cuh"
#include "ec_ops.h"
#include "ec_ptx.cuh"

namespace ec {

// CTAs that an even split can have: one per SM (148 on a B200)
constexpr int kMaxCtas = 160;

struct FlashArgs {
  const void *q, *k, *v;   // rows, or the cache's pools: for rows that are computed again
  int64_t qt, qh, kt, kh, vt, vh;  // their strides in elements
  void* out;
  float* lse;
  int64_t ot, oh;          // out strides in elements
  const int32_t *cu, *slots, *lens, *tables;
  int width, nslots;       // of the cache's tables
  int pages, page_size, page0, page_end;  // page0: first page of the layer, page_end: pages of all layers
  int tokens, nseq;
  int group, rows_tok;     // G, R
  int q_heads, kv_heads, head_dim;
  float scale_log2;
  int paged;
  int wide;                // out rows in 32-byte pieces
  int even;                // 1: the blocks are split evenly over the CTAs
  int min_chunk;           // units a CTA takes at least
  int over;                // units of a tile besides its blocks
  int part_rows;
  float* part_o;           // [2 * CTAs][part_rows][HD] partial results of cut tiles
  float* part_l;           // [2 * CTAs][part_rows] their log2-sum-exp2
  int* arrived;            // [CTAs] parts done of the tile whose first part is the CTA's; 0 between calls
  unsigned* status;        // marked by a wait that gives up
};

// a tile set that one CTA works on
struct FlashEntry {
  int valid;
  int tok0, qv;   // first token, tokens
  int kvh;
  int pos0;       // position of tok0 in its sequence
  int kv_len;
  int kbase;      // packed keys: first token of the sequence; cache: its slot
  int kb0;        // first key block
  int nb[2];      // end block of each tile
  int part;       // partial result, -1: the whole of the tile's keys
  int c0, parts;  // CTA of the tile's first part, their number
};
struct FlashItem : FlashEntry {
  int pages[32];  // cache: the first 32 pages from block kb0 on
};

// one of this many pairs of exponentials goes to the FMA units instead of the
// special-function unit
constexpr int kFmaEvery = 4;

// work-list entries in flight
constexpr int kFlashRing = 3;

// a list of whole tiles counts its sets in this many groups of sequences, up
// to kFlashCounted sequences
constexpr int kFlashGroups = 128, kFlashCounted = 4096;
// up to this many sequences go by set (one to a lane)
constexpr int kFlashFew = 32;

template <int HD, int NT>
struct FlashCfg {
  static constexpr int AT = HD / 64;                 // 64-column atoms
  static constexpr uint32_t ATOM = 16384;            // 128 rows x 128 B
  static constexpr uint32_t TILE = AT * ATOM;
  static constexpr int STAGES = HD == 128 ? 5 : 8;   // K and V tiles in flight
  static constexpr int MAX_SEQS = 2048;              // prefix sums of an even split
  // NT 1: four softmax warps, loads, MMAs, list.  NT 2: eight, loads, MMAs,
  // list, none, and four that write the results.
  static constexpr int WARPS = NT == 2 ? 16 : 7;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr uint32_t TAIL = 1536 + (NT == 1 ? 8 * MAX_SEQS : 1024 + 4 * kFlashGroups);
  static constexpr size_t SMEM = NT * TILE + STAGES * TILE + TAIL;
  static constexpr uint32_t O_COL = 256;
  static_assert(SMEM <= 232448, "shared memory");
};

// first wait of a caller's own call that gave up on this device since
// ec_op_status last asked
static __device__ unsigned g_op_status;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^x for two values on the FMA units: x = n + f with n the nearest integer,
// 2^f by a minimax polynomial of degree 5 on [-1/2, 1/2] (Remez; with its
// coefficients rounded to fp32 1.6e-7 from the truth, 2.4e-7 with the roundings
// of its evaluation, both relative), 2^n put together as
// an exponent.  x <= -127 gives 0; NaN stays NaN.  For x < 128.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  const float2 magic = make_float2(12582912.f + 127.f, 12582912.f + 127.f);  // 1.5 * 2^23: n + 127 in the low bits
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  const float2 t = __fadd2_rn(x, magic);
  const float2 n = __fadd2_rn(t, make_float2(-magic.x, -magic.y));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  auto c = [](float v) { return make_float2(v, v); };
  float2 p = __ffma2_rn(f, c(0.0013276472454890609f), c(0.009675540961325169f));
  p = __ffma2_rn(f, p, c(0.05550713092088699f));
  p = __ffma2_rn(f, p, c(0.24022120237350464f));
  p = __ffma2_rn(f, p, c(0.6931469440460205f));
  p = __ffma2_rn(f, p, c(1.0000001192092896f));
  return __fmul2_rn(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23),
                                   __uint_as_float(__float_as_uint(t.y) << 23)));
}

// acc + 0 * v, both halves: NaN once a value is not finite
template <typename T>
__device__ __forceinline__ uint32_t times_zero(uint32_t v, uint32_t acc) {
  if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0));
  return acc;
}

// 32 bytes to a 32-byte aligned address
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// key blocks that the first n tokens of a sequence's queries see
__device__ __forceinline__ int blocks_seen(int pos0, int n, int kv_len) {
  const int seen = min(kv_len, pos0 + n);
  return seen > 0 ? (seen + 127) >> 7 : 0;
}

// sequence s: its queries [begin, end) within the rows of the call, and keys
struct FlashSeq {
  int begin, end, kv_len, kbase;
};
__device__ __forceinline__ FlashSeq flash_seq(const FlashArgs& a, int s) {
  FlashSeq q;
  q.begin = min(max(a.cu[s], 0), a.tokens);
  q.end = min(max(a.cu[s + 1], q.begin), a.tokens);
  if (a.paged) {
    const int slot = a.slots ? a.slots[s] : s;
    const bool ok = slot >= 0 && slot < a.nslots;
    const int most = a.width * a.page_size;  // fits 31 bits (checked when the cache is opened)
    q.kv_len = ok ? min(max(a.lens[slot], 0), most) : 0;
    q.kbase = ok ? slot : 0;
  } else {
    q.kv_len = q.end - q.begin;
    q.kbase = q.begin;
  }
  return q;
}

// ------------------------------------------------------------- work lists --
// Without a split: the tile sets of all sequences, the last one first, and of
// each the key heads.  flash_count leaves the number of sets of every group of
// sequences; a set's group is found by bisection, its sequence from there, 32
// sets at a time.  The key heads of a set and the sets of a sequence follow
// each other, so that the CTAs read the same keys at about the same time (a run
// of the list for every CTA, of equal work: the corpus 1.41).  With more
// sequences than are counted, slot u is set i of sequence s for f(s) + i = u,
// f(s) = cu[s] / BT + s (BT tokens per set): f leaves at least ceil(len / BT)
// slots to every sequence and needs no sums, but its empty slots make the turns
// uneven (96 texts behind 650 cached tokens 1.13, 64 prompts of 300 1.16).  Slots
// times key heads fit 31 bits, checked on the host.
//
// Up to 32 sequences go by set, the latest sets of all of them first (slot u:
// set u / nseq of sequence u % nseq), so that a CTA's few turns cost the same:
// 4 prompts of 2048 tokens 86 us (by sequence 1.6).  With more sequences that
// costs the keys' reuse: 96 texts behind 650 cached tokens 1.29.
//
// Sums over the sequences are bounded by the tokens of the call as long as the
// offsets ascend.  flash_count and flash_measure mark where they do not; then
// the list stays empty (the sums could pass 32 bits, and what is laid out by
// them the buffers).  The mark lies in shared memory: in a register it cost the
// pairs' kernels spills (the corpus 1.05).
template <int NT>
__device__ __forceinline__ void flash_count(const FlashArgs& a, int* groups, volatile int* descend) {
  const int size = (a.nseq + kFlashGroups - 1) / kFlashGroups, BT = NT * a.rows_tok;
  for (int s = threadIdx.x; s < a.nseq; s += blockDim.x) {
    const int c0 = a.cu[s], c1 = a.cu[s + 1];
    const int begin = min(max(c0, 0), a.tokens), end = min(max(c1, begin), a.tokens);
    if (c1 < c0) *descend = 1;
    if (end > begin) atomicAdd(&groups[s / size], (end - begin + BT - 1) / BT);
  }
}
// (`summed`: the groups' sums are there already, their total in *sets)
template <int NT, typename Publish>
__device__ __noinline__ bool flash_slots(const FlashArgs& a, int lane, int* groups, int* sets, bool summed,
                                         const Publish& publish) {
  const int R = a.rows_tok, BT = NT * R;
  uint32_t slots = a.tokens / BT + a.nseq;
  const uint32_t step = gridDim.x;
  bool few = a.nseq <= kFlashFew;
  if (few) {
    const FlashSeq q = flash_seq(a, min(lane, a.nseq - 1));
    const uint32_t most = __reduce_max_sync(0xffffffffu, (q.end - q.begin + BT - 1) / BT);
    few = static_cast<uint64_t>(most) * a.nseq * a.kv_heads < (1u << 30);
    if (few) slots = most * a.nseq;
  }
  const bool counted = a.nseq > kFlashFew && a.nseq <= kFlashCounted;
  const int size = (a.nseq + kFlashGroups - 1) / kFlashGroups;
  if (counted && summed) {
    slots = *sets;
  } else if (counted) {
    int total = 0;
#pragma unroll 1
    for (int g = lane; g < kFlashGroups; g += 32) {  // sets before each group
      const int v = groups[g];
      int x = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      groups[g] = total + x - v;
      total += __shfl_sync(0xffffffffu, x, 31);
    }
    __syncwarp();
    slots = *sets = total;
  }
  const uint32_t all = slots * a.kv_heads;
  bool ok = true;
#pragma unroll 1
  for (uint32_t t0 = 0; ok && t0 < all; t0 += 32 * step) {
    // late (long) tile sets first; the order turns round every pass, so that
    // no CTA gets the longest of each
    const uint32_t t = t0 + lane * step + ((lane & 1) ? step - 1 - blockIdx.x : blockIdx.x);
    FlashEntry it{};
    if (t < all) {
      const int u = static_cast<int>(slots - 1 - t / a.kv_heads);
      int lo = few ? u % a.nseq : 0, i = few ? u / a.nseq : 0;  // sequence, set
      int hi = few ? 0 : counted ? kFlashGroups : a.nseq;
      while (hi - lo > 1) {  // last group that begins by u, or sequence with f <= u
        const int mid = (lo + hi) >> 1;
        if ((counted ? groups[mid] : min(max(a.cu[mid], 0), a.tokens) / BT + mid) <= u) lo = mid;
        else hi = mid;
      }
      if (counted) {
        i = u - groups[lo];
        lo *= size;
        int begin = min(max(a.cu[lo], 0), a.tokens);
        while (lo + 1 < a.nseq) {
          const int end = min(max(a.cu[lo + 1], begin), a.tokens), sets = (end - begin + BT - 1) / BT;
          if (i < sets) break;
          i -= sets;
          ++lo;
          begin = min(max(a.cu[lo], 0), a.tokens);
        }
      }
      const FlashSeq q = flash_seq(a, lo);
      const int len = q.end - q.begin;
      if (!few && !counted) i = u - (q.begin / BT + lo);
      if (i >= 0 && i < (len + BT - 1) / BT) {
        const int q0 = i * BT;
        it.valid = 1;
        it.tok0 = q.begin + q0;
        it.qv = min(BT, len - q0);
        it.kvh = static_cast<int>(t % a.kv_heads);
        it.pos0 = q.kv_len - len + q0;
        it.kv_len = q.kv_len;
        it.kbase = q.kbase;
        it.nb[0] = blocks_seen(it.pos0, min(R, it.qv), q.kv_len);
        it.nb[1] = NT == 2 && it.qv > R ? blocks_seen(it.pos0, it.qv, q.kv_len) : 0;
        it.part = -1;
      }
    }
    __syncwarp();
    for (unsigned m = __ballot_sync(0xffffffffu, it.valid); ok && m; m &= m - 1) ok = publish(it, __ffs(m) - 1);
  }
  return ok;
}

// The longest tile that flash_measure has bits for (4.19 million keys); it stands
// for all longer ones, too, so nothing is laid out by it
constexpr int kLongestMost = 0x7fff;

// Even split: every CTA takes the same share of the key blocks, in the order
// (sequence, tile, key head, block).  A tile costs its blocks and `over` units
// more, for its start and end, which come first.  Where there are fewer tiles
// than CTAs and the longest would not gain what a join costs (8 units, 20 with
// 128 rows: 25 us), every tile has a CTA of its own instead: 4 texts of 200
// tokens behind 4000 59 us (cut 1.4), 4 of 40 behind 2000 35 (cut 1.3); cut are
// one of 40 behind 20000, 98 us (whole 2.1), and 8 of 64 behind 8000, 96 us
// (whole 1.02).
//
// Each thread of the CTA first looks at some sequences (the loads are far
// away, and the CTA has nothing else to do yet): units[s] (-1: its offsets
// descend), and tiles | longest tile << 16, with the sign bit where a tile sees
// no key.
__device__ __forceinline__ void flash_measure(const FlashArgs& a, int* units, int* about) {
  for (int s = threadIdx.x; s < a.nseq; s += blockDim.x) {
    const FlashSeq q = flash_seq(a, s);
    const int len = q.end - q.begin, R = a.rows_tok;
    int v = 0, n = 0, most = 0, none = 0;
#pragma unroll 1
    for (int i = 0; i < len; i += R) {
      const int nb = blocks_seen(q.kv_len - len + i, min(R, len - i), q.kv_len);
      if (nb) v += nb + a.over, ++n, most = nb + a.over;
      else none = 1;
    }
    units[s] = a.cu[s + 1] < a.cu[s] ? -1 : v * a.kv_heads;
    about[s] = min(n * a.kv_heads, 0xffff) | min(most, kLongestMost) << 16 | none << 31;
  }
}
// (Kept out of line, as the list above: inlined into the kernels, the
// optimiser dropped an iteration of the sequence loop.)
template <typename Publish>
__device__ __noinline__ bool flash_even(const FlashArgs& a, int lane, int* prefix, const int* about, Publish publish) {
  const int R = a.rows_tok, ctas = gridDim.x, me = blockIdx.x;
  int tiles = 0, most = 0, work = 0;
  for (int s = lane; s < a.nseq; s += 32) {
    work += prefix[s];
    tiles += about[s] & 0xffff;
    most = max(most, prefix[s] < 0 ? INT_MAX : about[s] >> 16 & kLongestMost);
  }
  tiles = __reduce_add_sync(0xffffffffu, min(tiles, 1 << 20));
  most = __reduce_max_sync(0xffffffffu, most);
  work = __reduce_add_sync(0xffffffffu, work);
  if (most == INT_MAX) return true;  // offsets that descend
  // every tile, padded to the longest, its own CTA
  const bool alone = tiles <= ctas && most < kLongestMost && most <= work / ctas + 8 + a.part_rows / 10;
  int total = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.nseq; s0 += 32) {
    int v = 0;
    if (s0 + lane < a.nseq) v = alone ? (about[s0 + lane] & 0xffff) * most : prefix[s0 + lane];
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (s0 + lane < a.nseq) prefix[s0 + lane] = total + x - v;
    total += __shfl_sync(0xffffffffu, x, 31);
  }
  __syncwarp();
  const int chunk = alone ? max(most, 1) : max(a.min_chunk, (total + ctas - 1) / ctas);
  const int64_t w64 = static_cast<int64_t>(me) * chunk;
  const int begin = static_cast<int>(min(w64, static_cast<int64_t>(total)));
  const int end = static_cast<int>(min(w64 + chunk, static_cast<int64_t>(total)));
  // last sequence with prefix <= begin (those without blocks are skipped)
  int lo = 0, hi = a.nseq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= begin) lo = mid;
    else hi = mid;
  }
  FlashEntry it{};
  it.valid = 1;
  bool ok = true;
#pragma unroll 1
  for (int s = lo; ok && s < a.nseq; ++s) {
    int at = prefix[s];
    if (at >= end) break;
    const FlashSeq q = flash_seq(a, s);
    const int len = q.end - q.begin;
    it.kv_len = q.kv_len;
    it.kbase = q.kbase;
#pragma unroll 1
    for (int i = 0; ok && i < len; i += R) {
      it.tok0 = q.begin + i;
      it.qv = min(R, len - i);
      it.pos0 = q.kv_len - len + i;
      const int nb = blocks_seen(it.pos0, it.qv, q.kv_len);
      const int cost = nb == 0 ? 0 : alone ? most : nb + a.over;
      // key heads that end before this CTA's share are skipped
      int h = nb && at < begin ? min(a.kv_heads, (begin - at) / cost) : 0;
#pragma unroll 1
      for (; ok && h < a.kv_heads; ++h) {
        const int block0 = at + h * cost + a.over;  // unit of the tile's first block
        const int from = max(0, begin - block0), to = min(nb, end - block0);
        if (from < to) {
          it.kvh = h;
          it.kb0 = from;
          it.nb[0] = to;
          // a CTA has at most one part that goes on from another CTA and one
          // that another CTA goes on with
          it.part = from == 0 && to == nb ? -1 : 2 * me + (from == 0);
          it.c0 = block0 / chunk;
          it.parts = (block0 + nb - 1) / chunk - it.c0 + 1;
          ok = publish(it);
        }
      }
      at += a.kv_heads * cost;
    }
  }
  // tiles that see no key: entries without blocks, whose rows are cleared
#pragma unroll 1
  for (int s = me; ok && s < a.nseq; s += ctas) {
    if (about[s] >= 0) continue;
    const FlashSeq q = flash_seq(a, s);
    const int len = q.end - q.begin;
    it.kv_len = q.kv_len;
    it.kbase = q.kbase;
    it.kb0 = it.nb[0] = 0;
    it.part = -1;
#pragma unroll 1
    for (int i = 0; ok && i < len; i += R) {
      it.tok0 = q.begin + i;
      it.qv = min(R, len - i);
      it.pos0 = q.kv_len - len + i;
      if (blocks_seen(it.pos0, it.qv, q.kv_len)) break;
#pragma unroll 1
      for (int h = 0; ok && h < a.kv_heads; ++h) {
        it.kvh = h;
        ok = publish(it);
      }
    }
  }
  return ok;
}

// The CTA that finishes a cut tile's last part joins the parts, in the order of
// the keys.  A warp has a quarter of the rows: their weights first, a row to a
// lane, then the rows themselves, eight at a time, so that many loads are under
// way (a row after the other, each waiting for its loads: 4 texts of 200 tokens
// behind 4000, two parts to a tile, 1.44).
template <int HD, typename T>
__device__ __noinline__ void flash_join(const FlashArgs& a, int tok0, int qv, int kvh, int c0, int parts, int warp,
                                        int lane) {
  const int rows = qv * a.group, each = (rows + 3) / 4, base = warp * each, mine = min(each, rows - base);
  if (mine <= 0) return;
  const int row = base + min(lane, mine - 1);
  auto part = [&](int i) { return static_cast<int64_t>(2 * (c0 + i) + (i == 0)) * a.part_rows; };
  float m = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) m = fmaxf(m, __ldcg(&a.part_l[part(i) + row]));
  auto weight = [&](int i) {
    const float l2 = __ldcg(&a.part_l[part(i) + row]);
    return l2 == -INFINITY ? 0.f : fa_exp2(l2 - m);
  };
#pragma unroll 4
  for (int i = 0; i < parts; ++i) sum += weight(i);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane < mine && a.lse)
    a.lse[static_cast<int64_t>(tok0 + row / a.group) * a.q_heads + kvh * a.group + row % a.group] =
        sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945309f;
  auto store = [&](int at, const float* o) {
    uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(tok0 + at / a.group) * a.ot +
                    (kvh * a.group + at % a.group) * a.oh;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e)
      if (lane + 32 * e < a.head_dim) out[lane + 32 * e] = static_cast<uint16_t>(pack2<T>(o[e], 0.f));
  };
  if (mine < 8) {  // the parts under way together instead
#pragma unroll 1
    for (int r = 0; r < mine; ++r) {
      float o[HD / 32] = {};
#pragma unroll 4
      for (int i = 0; i < parts; ++i) {
        const float x = __shfl_sync(0xffffffffu, weight(i) * inv, r);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) o[e] += x * __ldcg(&a.part_o[(part(i) + base + r) * HD + lane + 32 * e]);
      }
      store(base + r, o);
    }
    return;
  }
#pragma unroll 1
  for (int r0 = 0; r0 < mine; r0 += 8) {
    float o[8][HD / 32] = {};
#pragma unroll 1
    for (int i = 0; i < parts; ++i) {
      const float w = weight(i) * inv;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int at = min(r0 + r, mine - 1);
        const float x = __shfl_sync(0xffffffffu, w, at);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) o[r][e] += x * __ldcg(&a.part_o[(part(i) + base + at) * HD + lane + 32 * e]);
      }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r0 + r < mine) store(base + r0 + r, o[r]);
  }
}

// -------------------------------------------------- rows computed again --
// A key that a row does not see has the probability 0, and 0 times an infinity
// or a NaN among its values is NaN.  It can only lie in the blocks that the
// row's tile cuts, at most 255 keys behind the row.  So a row whose result is
// not finite, although its sum is, looks there; if such a value is found, the
// row is computed again from the keys that it sees alone, by one warp, in fp32.
// Finite inputs cost the look at the result, which no time shows.

// row j of the keys (kv 0) or values (kv 1) of a packed sequence that starts at
// kbase or of slot kbase; nullptr: a page that is none, which reads as zeros
template <typename T>
__device__ __forceinline__ const T* flash_key(const FlashArgs& a, int kv, int kbase, int kvh, int j) {
  const T* base = static_cast<const T*>(kv ? a.v : a.k);
  if (!a.paged) return base + static_cast<int64_t>(kbase + j) * (kv ? a.vt : a.kt) + kvh * (kv ? a.vh : a.kh);
  const int p = a.tables[static_cast<int64_t>(kbase) * a.width + j / a.page_size];
  if (p < 0 || p >= a.pages) return nullptr;
  return base + ((static_cast<int64_t>(a.page0 + p) * a.page_size + j % a.page_size) * a.kv_heads + kvh) * a.head_dim;
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16, uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ float2 unpack2(__half, uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Row of token `tok` and query head `head` over the keys [first, vis): elements
// d0 + 32 e + lane, e < E, divided by the sum, to out (this lane's addresses
// for e = 0 are out and part; part: a part of a cut tile).
template <int E, typename T>
__device__ __noinline__ void flash_row(const FlashArgs& a, int tok, int head, int kvh, int kbase, int first, int vis,
                                       int d0, int lane, T* out, float* part) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + tok * a.qt + head * a.qh);
  float m = -INFINITY, l = 0.f, o[E] = {};
#pragma unroll 1
  for (int j0 = first; j0 < vis; j0 += 32) {
    float s = -INFINITY;
    if (j0 + lane < vis) {
      const uint4* k = reinterpret_cast<const uint4*>(flash_key<T>(a, 0, kbase, kvh, j0 + lane));
      s = 0.f;
#pragma unroll 1
      for (int i = 0; k && i < a.head_dim / 8; ++i) {
        const uint4 x = q[i], y = k[i];
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float2 f = unpack2(T(), xs[c]), g = unpack2(T(), ys[c]);
          s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
        }
      }
      s *= a.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - base);
    float p = exp2f(s - base), sum = p;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    l = l * corr + sum;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= corr;
#pragma unroll 4
    for (int i = 0; i < min(32, vis - j0); ++i) {
      const T* v = flash_key<T>(a, 1, kbase, kvh, j0 + i);
      const float w = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v && d0 + 32 * e + lane < a.head_dim) o[e] = fmaf(w, static_cast<float>(v[d0 + 32 * e + lane]), o[e]);
    }
    bool any = false;  // a row of which nothing is finite stays so
#pragma unroll
    for (int e = 0; e < E; ++e) any |= d0 + 32 * e + lane < a.head_dim && !isnan(o[e]);
    if (!__any_sync(0xffffffffu, any)) break;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float v = l == 0.f ? 0.f : o[e] / l;
    if (part) part[32 * e] = v;
    else if (d0 + 32 * e + lane < a.head_dim) out[32 * e] = static_cast<T>(v);
  }
}

// the last of the keys [from, to) with a value that is not finite, or -1
template <typename T>
__device__ __forceinline__ int flash_last_odd(const FlashArgs& a, int kbase, int kvh, int from, int to, int lane) {
  constexpr uint32_t EXP = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  int last = -1;
#pragma unroll 1
  for (int j = from + lane; j < to; j += 32) {
    const uint4* v = reinterpret_cast<const uint4*>(flash_key<T>(a, 1, kbase, kvh, j));
#pragma unroll 1
    for (int i = 0; v && i < a.head_dim / 8; ++i) {
      const uint4 x = v[i];
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if ((xs[c] & EXP) == EXP || (xs[c] >> 16 & EXP) == EXP) last = j;
    }
  }
  return __reduce_max_sync(0xffffffffu, last);
}

// Rows base .. base + 31 of a tile of rows (token, head) whose first token is
// tok0, at position pos: those of the lanes with `odd` are looked at, by the
// whole warp.  Keys [first, end) of the slot or sequence; part: of a cut tile,
// -1: whole.  Elements from d0 on, 32 E of them.
template <int HD, int E, typename T>
__device__ __noinline__ void flash_again(const FlashArgs& a, int tok0, int pos, int kvh, int kbase, int first, int end,
                                         int base, bool odd, int part, int d0, int lane) {
  const int vis = min(end, pos + (base + lane) / a.group + 1);
  odd &= vis < end;
  if (!__any_sync(0xffffffffu, odd)) return;
  const int from = __reduce_min_sync(0xffffffffu, odd ? vis : end);
  odd &= flash_last_odd<T>(a, kbase, kvh, from, end, lane) >= vis;
  __syncwarp();  // the rows have been written
#pragma unroll 1
  for (unsigned rest = __ballot_sync(0xffffffffu, odd); rest; rest &= rest - 1) {
    const int i = __ffs(rest) - 1, r = base + i, tok = tok0 + r / a.group, head = kvh * a.group + r % a.group;
    T* out = static_cast<T*>(a.out) + tok * a.ot + head * a.oh + d0 + lane;
    float* po = part < 0 ? nullptr : a.part_o + (static_cast<int64_t>(part) * a.part_rows + r) * HD + d0 + lane;
    flash_row<E, T>(a, tok, head, kvh, kbase, first, __shfl_sync(0xffffffffu, vis, i), d0, lane, out, po);
  }
}

// The list of pairs of tiles.  `finish` ends it and waits for the results; where
// it says that one of them is not finite, the list's warp goes through the list
// again and looks at them.  (The closures that go into functions out of line hold
// copies: kernel variables that they held by reference lay in local memory for
// all warps: the corpus 1.13, one token of one sequence 1.04.)
template <int HD, typename T, typename Publish, typename Finish>
__device__ __forceinline__ bool flash_pairs(const FlashArgs& a, int lane, int* groups, int* sets, bool empty,
                                            const Publish& publish, Finish finish) {
  bool ok = empty || flash_slots<2>(a, lane, groups, sets, false, publish);
  if (!finish(ok)) return ok;
  const int R = a.rows_tok;
  return flash_slots<2>(a, lane, groups, sets, true, [&](const FlashEntry& mine, int from) -> bool {
    auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
    const int tok0 = of(mine.tok0), qv = of(mine.qv), kvh = of(mine.kvh), pos0 = of(mine.pos0), kv_len = of(mine.kv_len);
    const int kbase = of(mine.kbase), nb0 = of(mine.nb[0]), nb1 = of(mine.nb[1]);
#pragma unroll 1
    for (int r = 0; r < qv * a.group; ++r) {
      const int tok = r / a.group, end = min(kv_len, (tok < R ? nb0 : nb1) * 128), vis = min(end, pos0 + tok + 1);
      if (vis >= end) continue;
      const int head = kvh * a.group + r % a.group;
      T* out = static_cast<T*>(a.out) + (tok0 + tok) * a.ot + head * a.oh + lane;
      bool odd = false;
#pragma unroll
      for (int e = 0; e < HD / 32; ++e)
        if (32 * e + lane < a.head_dim) odd |= !(fabsf(static_cast<float>(out[32 * e])) < INFINITY);
      if (__any_sync(0xffffffffu, odd) && flash_last_odd<T>(a, kbase, kvh, vis, end, lane) >= 0)
        flash_row<HD / 32, T>(a, tok0 + tok, head, kvh, kbase, 0, vis, 0, lane, out, nullptr);
    }
    return true;
  });
}

// Counts a finished part; true in the CTA that finished the last one, which
// leaves the count at 0 for the next call.  By one thread, once it has met all
// threads that wrote the part: its fence between the meeting and the count
// releases what they wrote.
__device__ __forceinline__ bool flash_arrive(const FlashArgs& a, const FlashEntry& it) {
  __threadfence();
  const bool last = atomicAdd(&a.arrived[it.c0], 1) == it.parts - 1;
  if (last) a.arrived[it.c0] = 0;
  __threadfence();
  return last;
}

// The end of the results (NT 2): the four warps that write them arrive, whether a
// wait of theirs gave up or not, and the list's warp waits (in hardware: a warp
// that polls takes turns from the softmax warps, 16384 tokens 1.01).
__device__ __forceinline__ void results_done(bool wait) {
  __syncwarp();
  if (wait) asm volatile("barrier.cta.sync 1, 160;" ::: "memory");
  else asm volatile("barrier.cta.arrive 1, 160;" ::: "memory");
}

template <int HD, int NT, bool HALF, typename T>
__global__ void __launch_bounds__(FlashCfg<HD, NT>::THREADS, 1)
    flash_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FlashArgs a) {
  using Cfg = FlashCfg<HD, NT>;
  constexpr int AT = Cfg::AT, ST = Cfg::STAGES;
  constexpr int FMT = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0 : 1;
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, 128), IDESC_S64 = make_idesc(FMT, 128, 64);
  constexpr uint32_t IDESC_PV = make_idesc(FMT, 128, HD) | (1u << 16);  // B MN-major
  constexpr int W_LOAD = 4 * NT, W_MMA = 4 * NT + 1, W_LIST = 4 * NT + 2;
  constexpr int W_EPI = 12;                         // NT 2: warps 12 .. 15
  constexpr int READERS = NT == 2 ? 14 : 6;         // warps that read a list entry

  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) report(a.status, kDevBadArg);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + NT * Cfg::TILE;
  uint8_t* tail = sKV + ST * Cfg::TILE;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(tail);
  uint64_t* q_empty = q_full + 1;
  uint64_t* kv_full = q_empty + 1;
  uint64_t* kv_empty = kv_full + ST;
  uint64_t* s_full = kv_empty + ST;   // [2] tile (NT 2) or buffer (NT 1)
  uint64_t* p_full = s_full + 2;      // [2]
  uint64_t* p_half = p_full + 2;      // [2] the first 64 keys' P
  uint64_t* o_full = p_half + 2;      // [2] tile (NT 2), or even / odd blocks (NT 1)
  uint64_t* x_bar = o_full + 2;       // [2] the softmax warps of NT 1
  uint64_t* r_full = x_bar + 2;       // [2] a tile's sums (NT 2)
  uint64_t* o_free = r_full + 2;      // [2] a tile's O has been read (NT 2)
  uint64_t* i_full = o_free + 2;      // [kFlashRing]
  uint64_t* i_empty = i_full + kFlashRing;
  FlashItem* items = reinterpret_cast<FlashItem*>(i_empty + kFlashRing);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + kFlashRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_part = abort_flag + 1;
  volatile int* descend = last_part + 1;
  volatile int* odd_rows = descend + 1;  // some result is not finite (NT 2)
  int* sets = reinterpret_cast<int*>(tmem_slot + 5);  // of a counted list
  int* prefix = reinterpret_cast<int*>(tail + 1536);  // [MAX_SEQS] of an even split
  float* inverse = reinterpret_cast<float*>(tail + 1536);  // [2][128] 1 / l (NT 2)
  int* groups = reinterpret_cast<int*>(tail + 1536 + (NT == 1 ? 0 : 1024));  // [kFlashGroups] of a list
  static_assert(8 * (2 + 2 * ST + 14 + 2 * kFlashRing) + kFlashRing * sizeof(FlashItem) + 24 <= 1536, "tail");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&x_bar[i], 4);
      mbar_init(&r_full[i], 4);
      mbar_init(&o_free[i], 4);
    }
    for (int i = 0; i < kFlashRing; ++i) {
      mbar_init(&i_full[i], 1);
      mbar_init(&i_empty[i], READERS);
    }
    *abort_flag = 0;
    *descend = 0;
    *odd_rows = 0;
    fence_barrier_init();
  }
  if (warp == W_LOAD && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == W_MMA) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  const bool count = !a.even && a.nseq > kFlashFew && a.nseq <= kFlashCounted;
  if (count) {
    for (int i = threadIdx.x; i < kFlashGroups; i += blockDim.x) groups[i] = 0;
    __syncthreads();
  }
  pdl_wait();  // what comes before may still be running up to here
  pdl_trigger();
  if (count) flash_count<NT>(a, groups, descend);
  if (NT == 1 && a.even) flash_measure(a, prefix, prefix + Cfg::MAX_SEQS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int R = a.rows_tok, G = a.group;
  bool ok = true;
  unsigned code = kDevTimeoutOther;

  // the next entry of the list for the reading warps; it stays readable until
  // done_item
  int it_n = 0;
  auto next_item = [&]() -> const FlashItem* {
    const int b = it_n % kFlashRing;
    if (!mbar_wait_warp(&i_full[b], (it_n / kFlashRing) & 1, abort_flag)) return nullptr;
    return &items[b];
  };
  auto done_item = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[it_n % kFlashRing]);
    ++it_n;
  };
  // Keys that the last query of tile t sees, from the block `at` on.  HALF: in
  // a block where that is 64 or less, the other half takes no part in anything.
  // It pays with short sequences, whose last blocks are many (1024 prompts of
  // 130 tokens 559 us, without it 1.08; 256 of 320 262 us, 1.02); elsewhere the
  // loops of one or two halves slow the others down (one of 16384 with it 1.03,
  // of 4096 1.05, 32 of 1024 0.99).
  auto tile_sees = [&](const FlashEntry& it, int t, int at) {
    return HALF ? min(it.kv_len, it.pos0 + min((t + 1) * R, it.qv)) - at * 128 : 128;
  };
  auto one_half = [&](int sees, int j) { return HALF && sees - j * 128 <= 64; };
  const int ppb = a.paged ? 128 / a.page_size : 1;  // pages per key block
  // page of table entry e of a slot with `in_use` pages; one that is none
  // reads past the pages, which fills the tile with zeros
  auto fetch = [&](int slot, int e, int in_use) -> int {
    int p = -1;
    if (e < in_use) p = a.tables[static_cast<int64_t>(slot) * a.width + e];
    return p >= 0 && p < a.pages ? a.page0 + p : a.page_end;
  };
  auto pages_in_use = [&](int kv_len) { return (kv_len + a.page_size - 1) / a.page_size; };

  // writes this warp's rows of tile t: O / l, or 0 where inv is 0 (a row that
  // sees nothing)
  auto write_rows = [&](const FlashEntry& it, int t, int n, bool live, float inv, uint32_t o_addr) {
    const int r = (warp & 3) * 32 + lane, tok = r / G;
    const int64_t row = it.tok0 + t * R + tok;
    T* o = static_cast<T*>(a.out) + row * a.ot + (it.kvh * G + r - tok * G) * a.oh;
    float* po = a.part_o + (static_cast<int64_t>(max(it.part, 0)) * a.part_rows + r) * HD;
    float2 sum = make_float2(0.f, 0.f);  // finite if the row is (NT 1)
    uint32_t zero = 0;                   // 0 if it is (NT 2)
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t v[32];
      if (n > 0) {
        tmem_ld_32x32b_x32(o_addr + c * 32, v);
        tmem_wait_ld();
      }
      if (NT == 2 && n > 0 && c == HD / 32 - 1) {  // the next P V may overwrite it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[t]);
      }
      if (live) {
        if constexpr (NT == 1) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            sum = __fadd2_rn(sum, make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = inv == 0.f ? 0u : __float_as_uint(__uint_as_float(v[i]) * inv);
        if (NT == 1 && it.part >= 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) store32(po + c * 32 + 8 * i, v + 8 * i);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
          if constexpr (NT == 2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) zero = times_zero<T>(v[i], zero);
          }
          if (a.wide) {
            if (c * 32 < a.head_dim) store32(o + c * 32, v);
            if (c * 32 + 16 < a.head_dim) store32(o + c * 32 + 16, v + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c * 32 + 8 * i < a.head_dim)
                *reinterpret_cast<uint4*>(o + c * 32 + 8 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      }
      __syncwarp();  // the loads from TMEM are the whole warp's
    }
    if constexpr (NT == 2) {
      if (zero & 0x7fff7fffu) *odd_rows = 1;  // looked at by the list's warp, at the end
    } else {
      const bool odd = live && n > 0 && !(fabsf(sum.x + sum.y) < INFINITY);
      if (__any_sync(0xffffffffu, odd))
        flash_again<HD, HD / 32, T>(a, it.tok0, it.pos0, it.kvh, it.kbase, it.kb0 * 128, min(it.kv_len, it.nb[0] * 128),
                                    (warp & 3) * 32, odd, it.part, 0, lane);
    }
  };

  if constexpr (NT == 2) {
    // 512 threads of 128 registers: 168 for the softmax, 88 for the rest
    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  }
  if (warp == W_LIST) {
    using Entry = FlashEntry;
    // ------------------------------------------------------------ work list
    int n = 0;
    auto publish = [=, &a, &n](const Entry& it, int from) -> bool {  // lane `from`'s entry
      const int b = n % kFlashRing;
      if (!mbar_wait_warp(&i_empty[b], ((n / kFlashRing) & 1) ^ 1, abort_flag)) return false;
      if (a.paged && __shfl_sync(0xffffffffu, it.valid, from)) {
        // looked up here, ahead of the loads: the table is far away
        const int slot = __shfl_sync(0xffffffffu, it.kbase, from), kv_len = __shfl_sync(0xffffffffu, it.kv_len, from);
        items[b].pages[lane] = fetch(slot, __shfl_sync(0xffffffffu, it.kb0, from) * ppb + lane, pages_in_use(kv_len));
      }
      if (lane == from) *static_cast<Entry*>(&items[b]) = it;
      __syncwarp();
      if (lane == 0) mbar_arrive(&i_full[b]);
      ++n;
      return true;
    };
    if constexpr (NT == 2) {
      ok = flash_pairs<HD, T>(a, lane, groups, sets, *descend, publish, [=](bool& fine) -> bool {
        fine = fine && publish(Entry{}, 0);
        results_done(true);
        return fine && *odd_rows && !*abort_flag;
      });
    } else {
      if (a.even)
        ok = flash_even(a, lane, prefix, prefix + Cfg::MAX_SEQS, [=](const Entry& e) { return publish(e, 0); });
      else if (!*descend) ok = flash_slots<NT>(a, lane, groups, sets, false, publish);
      if (ok) ok = publish(Entry{}, 0);
    }
  } else if (warp == W_LOAD) {
    // ---------------------------------------------------------------- loads
    code = kDevTimeoutProducer;
    int st = 0, qi = 0;
    uint32_t ph = 0;
    while (true) {
      const FlashItem* it = next_item();
      if (!(ok = it != nullptr) || !it->valid) break;
      const int kb0 = it->kb0, nb = max(it->nb[0], NT == 2 ? it->nb[1] : 0);
      const int kvh = it->kvh, kbase = it->kbase, tok0 = it->tok0, in_use = a.paged ? pages_in_use(it->kv_len) : 0;
      int page = a.paged ? it->pages[lane] : 0, ahead = 0;
      done_item();
      if (nb <= kb0) continue;
      int first = kb0 * ppb;  // table entry of lane 0's page
      if (a.paged && nb * ppb > first + 32) ahead = fetch(kbase, first + 32 + lane, in_use);
#pragma unroll 1
      for (int j = kb0; ok && j < nb; ++j) {
        if (a.paged && j * ppb - first == 32) {
          first += 32;
          page = ahead;
          ahead = fetch(kbase, first + 32 + lane, in_use);
        }
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (!(ok = mbar_wait_warp(&kv_empty[st], ph ^ 1, abort_flag))) break;
          const uint32_t dst = smem_u32(sKV + st * Cfg::TILE), bar = smem_u32(&kv_full[st]);
          const uint64_t map = reinterpret_cast<uint64_t>(kv ? &tm_v : &tm_k);
          if (elect_one()) mbar_arrive_expect_tx(&kv_full[st], Cfg::TILE);
          __syncwarp();
          if (a.paged) {
            int p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __shfl_sync(0xffffffffu, page, (j * ppb - first + i) & 31);
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < AT; ++c)
                  if (i < ppb)
                    asm volatile(
                        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                        "[%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst + c * Cfg::ATOM + i * a.page_size * 128),
                        "l"(map), "r"(bar), "r"(c * 64), "r"(kvh), "r"(0), "r"(p[i])
                        : "memory");
            }
          } else if (elect_one()) {
#pragma unroll
            for (int c = 0; c < AT; ++c)
              asm volatile(
                  "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                  "[%1, {%3, %4, %5}], [%2];" ::"r"(dst + c * Cfg::ATOM),
                  "l"(map), "r"(bar), "r"(c * 64), "r"(kvh), "r"(kbase + j * 128)
                  : "memory");
          }
          __syncwarp();
          if (++st == ST) {
            st = 0;
            ph ^= 1;
          }
          if (j == kb0 && kv == 0) {
            // the queries, once the tiles before have no more use for theirs;
            // rows past the tokens of the call are filled with zeros
            if (!(ok = mbar_wait_warp(q_empty, (qi & 1) ^ 1, abort_flag))) break;
            ++qi;
            if (elect_one()) {
              mbar_arrive_expect_tx(q_full, NT * AT * static_cast<uint32_t>(G * R) * 128u);
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int c = 0; c < AT; ++c)
                  asm volatile(
                      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                      "[%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(sQ + t * Cfg::TILE + c * Cfg::ATOM)),
                      "l"(reinterpret_cast<uint64_t>(&tm_q)), "r"(smem_u32(q_full)), "r"(c * 64), "r"(kvh * G),
                      "r"(tok0 + t * R)
                      : "memory");
            }
            __syncwarp();
          }
        }
      }
      if (!ok) break;
    }
  } else if (warp == W_MMA) {
    // ----------------------------------------------------------------- MMAs
    // one thread: operands of tcgen05 instructions are warp-uniform, which the
    // compiler knows of the elected thread only
    code = kDevTimeoutMma;
    if (elect_one()) {
      int st = 0;            // stage of the next K / V tile
      uint32_t ph = 0;       // its phase
      int qi = 0;            // items so far
      uint32_t pf[2] = {0, 0};  // P's waited for, per tile
      uint32_t of[2] = {0, 0};  // results begun, per tile (NT 2)
      uint32_t g = 0;           // blocks (NT 1)
      const uint64_t dq = desc_sw128_kmajor(smem_u32(sQ));
      const uint64_t dk = desc_sw128_kmajor(smem_u32(sKV));
      const uint64_t dv = desc_mnmajor<false>(smem_u32(sKV), Cfg::ATOM);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool fine = mbar_wait(bar, parity, abort_flag);
        tc_fence_after();
        return fine;
      };
      auto advance = [&] {
        if (++st == ST) {
          st = 0;
          ph ^= 1;
        }
      };
      auto mma_s = [&](int t, int stage, uint32_t d, bool half) {
        const uint64_t q = dq + t * (Cfg::TILE >> 4), k = dk + stage * (Cfg::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * Cfg::ATOM + (kk & 3) * 32) >> 4;
          umma_f16(d, q + off, k + off, half ? IDESC_S64 : IDESC_S, kk > 0);
        }
      };
      auto mma_pv = [&](uint32_t d, uint32_t p, int stage, bool first, int half) {
        const uint64_t v = dv + stage * (Cfg::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f16_ts(d, p + (4 * half + kk) * 8, v + (4 * half + kk) * (2048 >> 4), IDESC_PV,
                      kk > 0 || half > 0 || !first);
      };
      int n0 = 0, n1 = 0;  // key blocks of the tiles of the item that `take` found
      int k0 = 0, k1 = 0;  // and keys that they see of them
      bool more = true;    // there was one
      auto take = [&]() -> bool {
        while (true) {
          const int b = it_n % kFlashRing;
          if (!mbar_wait(&i_full[b], (it_n / kFlashRing) & 1, abort_flag)) return false;
          const int kb0 = items[b].kb0;
          more = items[b].valid;
          n0 = items[b].nb[0] - kb0, n1 = NT == 2 ? items[b].nb[1] - kb0 : 0;
          k0 = tile_sees(items[b], 0, kb0), k1 = NT == 2 ? tile_sees(items[b], 1, kb0) : 0;
          mbar_arrive(&i_empty[b]);
          ++it_n;
          if (!more || max(n0, n1) > 0) return true;
        }
      };
      if constexpr (NT == 2) {
        // the first scores of the item taken last, tile t
        auto begin = [&](int t) -> bool {
          if (t == 0) {
            if (!wait(q_full, qi & 1) || !wait(&kv_full[st], ph)) return false;
            ++qi;
          }
          if ((t ? n1 : n0) > 0) {
            mma_s(t, st, tmem + t * 128, one_half(t ? k1 : k0, 0));
            umma_commit(&s_full[t]);
          }
          if (t == 1) {
            umma_commit(&kv_empty[st]);
            if (max(n0, n1) == 1) umma_commit(q_empty);
            advance();
          }
          return true;
        };
        ok = take();
        if (ok && more) ok = begin(0) && begin(1);
        while (ok && more) {
          const int c0 = n0, c1 = n1, n = max(c0, c1), e0 = k0, e1 = k1;
#pragma unroll 1
          for (int j = 0; ok && j < n; ++j) {
            const int sv = st;
            const uint32_t phv = ph;
            advance();
            bool have_v = false, have_k = false;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int nt = t ? c1 : c0;
              if (!ok) continue;
              if (j < nt) {
                if (!have_v && !(ok = wait(&kv_full[sv], phv))) continue;
                have_v = true;
                if (!(ok = wait(&p_half[t], pf[t] & 1))) continue;
                if (j == 0) {
                  if (of[t] > 0 && !(ok = wait(&o_free[t], (of[t] - 1) & 1))) continue;
                  ++of[t];
                }
                mma_pv(tmem + Cfg::O_COL + t * HD, tmem + t * 128, sv, j == 0, 0);
                if (!(ok = wait(&p_full[t], pf[t] & 1))) continue;
                ++pf[t];
                if (!one_half(t ? e1 : e0, j)) mma_pv(tmem + Cfg::O_COL + t * HD, tmem + t * 128, sv, false, 1);
              }
              if (j + 1 == nt) umma_commit(&o_full[t]);
              if (t == 1) umma_commit(&kv_empty[sv]);
              if (j + 1 < nt) {
                if (!have_k && !(ok = wait(&kv_full[st], ph))) continue;
                have_k = true;
                mma_s(t, st, tmem + t * 128, one_half(t ? e1 : e0, j + 1));
                umma_commit(&s_full[t]);
              }
              if (j + 1 == n) {
                // this tile is done: the next item's scores do not wait for
                // the other tile's last block
                if (t == 0) ok = take();
                if (ok && more) ok = begin(t);
              }
            }
            if (!ok) break;
            if (j + 1 < n) {
              umma_commit(&kv_empty[st]);
              if (j + 2 == n) umma_commit(q_empty);
              advance();
            }
          }
        }
      }
      while (NT == 1) {
        if (!(ok = take()) || !more) break;
        const int n = n0;
        if (!(ok = wait(q_full, qi & 1)) || !(ok = wait(&kv_full[st], ph))) break;
        ++qi;
        {
          mma_s(0, st, tmem + (g & 1) * 128, one_half(k0, 0));
          umma_commit(&s_full[g & 1]);
          umma_commit(&kv_empty[st]);
          if (n == 1) umma_commit(q_empty);
          advance();
#pragma unroll 1
          for (int j = 0; j < n; ++j, ++g) {
            const int sv = st;
            const uint32_t phv = ph;
            advance();
            if (j + 1 < n) {
              if (!(ok = wait(&kv_full[st], ph))) break;
              mma_s(0, st, tmem + ((g + 1) & 1) * 128, one_half(k0, j + 1));
              umma_commit(&s_full[(g + 1) & 1]);
              umma_commit(&kv_empty[st]);
              if (j + 2 == n) umma_commit(q_empty);
              advance();
            }
            if (!(ok = wait(&kv_full[sv], phv)) || !(ok = wait(&p_half[g & 1], (g >> 1) & 1))) break;
            mma_pv(tmem + Cfg::O_COL, tmem + (g & 1) * 128, sv, j == 0, 0);
            if (!(ok = wait(&p_full[g & 1], (g >> 1) & 1))) break;
            if (!one_half(k0, j)) mma_pv(tmem + Cfg::O_COL, tmem + (g & 1) * 128, sv, false, 1);
            umma_commit(&o_full[g & 1]);
            umma_commit(&kv_empty[sv]);
          }
        }
        if (!ok) break;
      }
      if (!ok) {
        report(a.status, code);
        *abort_flag = 1;
      }
    }
    __syncwarp();
  } else if (NT == 2 && warp >= 8) {
    // -------------------------------------------------------------- results
    code = kDevTimeoutEpilogue;
    uint32_t done[2] = {0, 0};
    while (warp >= W_EPI) {
      const FlashItem* ip = next_item();
      if (!(ok = ip != nullptr) || !ip->valid) break;
      const FlashEntry it = *ip;
      done_item();
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = (warp & 3) * 32 + lane, tok = r / G;
        const bool live = tok < R && t * R + tok < it.qv;
        const int n = it.nb[t] - it.kb0;
        float inv = 0.f;
        if (n > 0) {
          if (!(ok = mbar_wait_warp(&r_full[t], done[t] & 1, abort_flag)) ||
              !(ok = mbar_wait_warp(&o_full[t], done[t] & 1, abort_flag)))
            break;
          ++done[t];
          tc_fence_after();
          inv = inverse[t * 128 + r];
        }
        if (n > 0 || __any_sync(0xffffffffu, live))
          write_rows(it, t, n, live, inv, tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + Cfg::O_COL + t * HD);
      }
      if (!ok) break;
    }
    if (warp >= W_EPI) results_done(false);
  } else {
    // -------------------------------------------------------------- softmax
    if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    code = kDevTimeoutEpilogue;
    const int t = warp >> 2;               // tile (0 for NT 1)
    const int r = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
    const int tok = r / G, head = r - tok * G;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_addr = t_lane + Cfg::O_COL + t * HD;
    const float sc = a.scale_log2;
    int g = 0;       // blocks so far (of this tile)
    int e = 0;       // K / V tiles before this item's
    int done = 0;    // results handed on (NT 2)
    int x = 0;       // meetings of the four warps (NT 1)
    while (true) {
      const FlashItem* ip = next_item();
      if (!(ok = ip != nullptr) || !ip->valid) break;
      const FlashEntry it = *ip;
      done_item();
      const int qt = t * R + tok;          // token within the tile set
      const bool live = tok < R && qt < it.qv;
      const bool warp_live = __any_sync(0xffffffffu, live);
      // keys [0, vis) are seen by this row
      const int vis = live ? min(it.kv_len, it.pos0 + qt + 1) : 0;
      const int n = (t ? it.nb[1] : it.nb[0]) - it.kb0;
      float m = -INFINITY, l = 0.f;  // maximum (raw score) that O and l are relative to
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++g) {
        const int buf = NT == 2 ? t : g & 1;
        const uint32_t s_addr = t_lane + buf * 128;
        if (!(ok = mbar_wait_warp(&s_full[buf], NT == 2 ? g & 1 : (g >> 1) & 1, abort_flag))) break;
        tc_fence_after();
        // V rows behind the sequence's keys are another sequence's, or what a
        // page held before: their probabilities are 0, and 0 * NaN would not
        // be.  Cleared by the tile's own warps before its P V.
        const int rows = it.kv_len - (it.kb0 + j) * 128;
        if (rows < 128) {
          // the tile has landed: these writes come after the copy's
          const int entry = e + 2 * j + 1;
          if (!(ok = mbar_wait_warp(&kv_full[entry % ST], (entry / ST) & 1, abort_flag))) break;
          if (r >= rows) {
            uint8_t* v = sKV + (entry % ST) * Cfg::TILE + r * 128;
#pragma unroll 1
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int c = 0; c < AT; ++c) *reinterpret_cast<uint4*>(v + c * Cfg::ATOM + i * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (warp_live) {
          // The scores are read twice, 64 at a time (first their maximum, then
          // P): half the code and a third of the registers of holding all 128
          const int left = vis - (it.kb0 + j) * 128;
          const bool cut = __any_sync(0xffffffffu, live && left < 128);
          const int halves = HALF && tile_sees(it, t, it.kb0 + j) <= 64 ? 1 : 2;
          uint32_t s[2][32];
          auto scores = [&](int h) {
            tmem_ld_32x32b_x32(s_addr + h * 64, s[0]);
            tmem_ld_32x32b_x32(s_addr + h * 64 + 32, s[1]);
            tmem_wait_ld();
            if (cut) {
              const int see = left - h * 64;
              const uint32_t w0 = see >= 32 ? 0xffffffffu : see <= 0 ? 0u : (1u << see) - 1u;
              const uint32_t w1 = see >= 64 ? 0xffffffffu : see <= 32 ? 0u : (1u << (see - 32)) - 1u;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (!(w0 & (1u << i))) s[0][i] = 0xff800000u;  // -infinity
                if (!(w1 & (1u << i))) s[1][i] = 0xff800000u;
              }
            }
          };
          float top = -INFINITY;
#pragma unroll 1
          for (int h = 0; h < halves; ++h) {
            scores(h);
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              mx[c] = __uint_as_float(s[c >> 1][(c & 1) * 16]);
#pragma unroll
              for (int i = 1; i < 15; i += 2)
                asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[c]) : "f"(__uint_as_float(s[c >> 1][(c & 1) * 16 + i])), "f"(__uint_as_float(s[c >> 1][(c & 1) * 16 + i + 1])));
              mx[c] = fmaxf(mx[c], __uint_as_float(s[c >> 1][(c & 1) * 16 + 15]));
            }
            top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          }
          // keep the older maximum unless the new one is 2^8 above it
          const bool grow = live && ((top - m) * sc > 8.f || (m == -INFINITY && top > m));
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? top : m;
            const float corr = mn == -INFINITY ? 1.f : fa_exp2((m - mn) * sc);
            if (j > 0) {
              // O holds the blocks before: their last P V has to be done (with
              // NT 2 this block's S came after it)
              if (NT == 1 && !(ok = mbar_wait_warp(&o_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag))) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(o_addr + c * 32, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
                tmem_st_32x32b_x32(o_addr + c * 32, v);
              }
              tmem_wait_st();
            }
            l *= corr;
            m = mn;
          }
          const float nm = m == -INFINITY ? 0.f : -m * sc;
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
#pragma unroll 1
          for (int h = 0; h < halves; ++h) {
            scores(h);
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const uint32_t* x = s[i >> 4] + 2 * (i & 15);
              const float2 y = __ffma2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), sc2, nm2);
              const float2 w = (i % kFmaEvery) == kFmaEvery - 1 ? exp2_fma(y) : make_float2(fa_exp2(y.x), fa_exp2(y.y));
              sum[i & 1] = __fadd2_rn(sum[i & 1], w);
              p[i] = pack2<T>(w.x, w.y);
            }
            tmem_st_32x32b_x32(s_addr + h * 32, p);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(h ? &p_full[buf] : &p_half[buf]);
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          if (halves == 1 && lane == 0) mbar_arrive(&p_full[buf]);
        } else {
          tc_fence_before();
          if (lane == 0) {
            mbar_arrive(&p_half[buf]);
            mbar_arrive(&p_full[buf]);
          }
        }
      }
      if (!ok) break;
      e += 2 * max(0, max(it.nb[0], NT == 2 ? it.nb[1] : 0) - it.kb0);
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
      const float l2 = l == 0.f ? -INFINITY : m * sc + log2f(l);
      if (live && it.part < 0 && a.lse)
        a.lse[static_cast<int64_t>(it.tok0 + qt) * a.q_heads + it.kvh * G + head] = l2 * 0.693147180559945309f;
      if constexpr (NT == 2) {
        if (n > 0) {
          // the warps that write the results take it from here, once they
          // are done with the tile's last ones
          if (done > 0 && !(ok = mbar_wait_warp(&o_free[t], (done - 1) & 1, abort_flag))) break;
          ++done;
          inverse[t * 128 + r] = inv;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&r_full[t]);
        }
        continue;
      } else {
        if (n > 0) {
          // the last P V.  Two barriers alternate: the scores of block g came
          // after P V of g - 2, so a wait for g - 1 is never two phases from
          // its barrier's
          if (!(ok = mbar_wait_warp(&o_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag))) break;
          tc_fence_after();
        }
        if (warp_live) {
          write_rows(it, t, n, live, inv, o_addr);
          if (live && it.part >= 0) a.part_l[it.part * a.part_rows + r] = l2;
        }
        __syncwarp();
      }
      if (NT == 1 && it.part >= 0) {
        auto meet = [&]() -> bool {  // the four warps
          __syncwarp();
          if (lane == 0) mbar_arrive(&x_bar[x & 1]);
          const bool fine = mbar_wait_warp(&x_bar[x & 1], (x >> 1) & 1, abort_flag);
          ++x;
          return fine;
        };
        if (!(ok = meet())) break;  // every warp has written its rows
        if (warp == 0 && lane == 0) *last_part = flash_arrive(a, it);
        if (!(ok = meet())) break;
        if (*last_part) flash_join<HD, T>(a, it.tok0, it.qv, it.kvh, it.c0, it.parts, warp, lane);
        __syncwarp();
      }
      tc_fence_before();
    }
  }
  if (!ok) {
    report(a.status, code);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // let copies and MMAs in flight land before the memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) {
    }
  }
  if (warp == W_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------- few rows --
// The same for tiles of at most NP rows (single tokens and their query heads),
// with the operands the other way round: S^T = K Q^T has a key per TMEM lane
// and a row per column, so that the four softmax warps share a block's keys
// and every lane has work, and O^T += V^T P^T has an element of the head per
// lane.  What bounds it then is reading K and V.  The warps agree on a block's
// row maxima through shared memory.  One warp runs per scheduler, so a block
// takes as long as its instructions do, one after the other: NP = 4, 8, 16 and
// 32 rows each have their own kernel (the MMA's N is 16 at least; what the
// columns behind NP hold reaches nothing).  One call after the other, three
// contexts of 100000 to 131000 tokens take 223 us, at the copy rate; 64 sequences
// of up to 8192 tokens, grouped by four, 74 us at 79% of it (tiles of 128 rows
// 1.5): there the starts and joins of about two tiles a CTA count; one token of
// one sequence 11 us, most of them between launch and first key.
template <int HD, int NP>
struct TokenCfg {
  static constexpr int NR = NP < 16 ? 16 : NP;         // columns of the MMAs
  static constexpr int AT = HD / 64;
  static constexpr uint32_t ATOM = 16384;
  static constexpr uint32_t TILE = AT * ATOM;          // 128 keys
  static constexpr int STAGES = (NR == 16 ? 6 : 5) * (HD == 128 ? 1 : 2);
  static constexpr uint32_t QATOM = NR * 128;          // 64 columns of the queries
  static constexpr uint32_t QBUF = AT * QATOM;
  static constexpr uint32_t PBUF = 2 * NR * 128;       // P^T: NR rows x 128 keys
  static constexpr int MAX_SEQS = FlashCfg<HD, 1>::MAX_SEQS;
  static constexpr int THREADS = 7 * 32;
  static constexpr uint32_t XCH = 2 * 4 * NP * 4;      // row maxima of the warps
  static constexpr uint32_t TAIL = 1536 + XCH + 8 * MAX_SEQS;
  static constexpr size_t SMEM = STAGES * TILE + 2 * QBUF + 2 * PBUF + TAIL;
  static constexpr uint32_t COLS = NR == 16 ? 64 : 128;  // two S^T, one O^T
  static_assert(SMEM <= 232448, "shared memory");
};

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// NP 32-bit columns of this thread's TMEM lane
template <int NP>
__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&r)[NP]) {
  if constexpr (NP == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  } else if constexpr (NP == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
  } else if constexpr (NP == 16) {
    tmem_ld_32x32b_x16(addr, r);
  } else {
    tmem_ld_32x32b_x32(addr, r);
  }
}
template <int NP>
__device__ __forceinline__ void tmem_st_rows(uint32_t addr, const uint32_t (&r)[NP]) {
  if constexpr (NP == 4) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
  } else if constexpr (NP == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else if constexpr (NP == 16) {
    tmem_st_32x32b_x16(addr, r);
  } else {
    tmem_st_32x32b_x32(addr, r);
  }
}

template <int HD, int NP, typename T>
__global__ void __launch_bounds__(TokenCfg<HD, NP>::THREADS, 1)
    flash_token_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FlashArgs a) {
  using Cfg = TokenCfg<HD, NP>;
  constexpr int AT = Cfg::AT, ST = Cfg::STAGES, NR = Cfg::NR;
  constexpr int FMT = std::is_same<T, __half>::value ? 0 : 1;
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, NR);
  constexpr uint32_t IDESC_PV = make_idesc(FMT, 128, NR) | (1u << 15);  // A (V^T) MN-major
  constexpr int W_LOAD = 4, W_MMA = 5, W_LIST = 6, READERS = 6;

  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) report(a.status, kDevBadArg);
    return;
  }
  uint8_t* sKV = smem;
  uint8_t* sQ = sKV + ST * Cfg::TILE;
  uint8_t* sP = sQ + 2 * Cfg::QBUF;
  uint8_t* tail = sP + 2 * Cfg::PBUF;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(tail);  // [2]
  uint64_t* q_empty = q_full + 2;
  uint64_t* kv_full = q_empty + 2;
  uint64_t* kv_empty = kv_full + ST;
  uint64_t* s_full = kv_empty + ST;  // [2] even / odd blocks, as the next two
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* x_bar = o_full + 2;      // [2] the four softmax warps
  uint64_t* i_full = x_bar + 2;
  uint64_t* i_empty = i_full + kFlashRing;
  FlashItem* items = reinterpret_cast<FlashItem*>(i_empty + kFlashRing);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + kFlashRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(8 * (4 + 2 * ST + 8 + 2 * kFlashRing) + kFlashRing * sizeof(FlashItem) + 8 <= 1536, "tail");
  float* xch = reinterpret_cast<float*>(tail + 1536);  // [2][4][NP]
  int* prefix = reinterpret_cast<int*>(tail + 1536 + Cfg::XCH);  // [MAX_SEQS]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&x_bar[i], 4);
    }
    for (int i = 0; i < kFlashRing; ++i) {
      mbar_init(&i_full[i], 1);
      mbar_init(&i_empty[i], READERS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == W_LOAD && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == W_MMA) {
    tmem_alloc(tmem_slot, Cfg::COLS);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  flash_measure(a, prefix, prefix + Cfg::MAX_SEQS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int R = a.rows_tok, G = a.group;
  bool ok = true;
  unsigned code = kDevTimeoutOther;
  int it_n = 0;
  auto next_item = [&]() -> const FlashItem* {
    const int b = it_n % kFlashRing;
    if (!mbar_wait_warp(&i_full[b], (it_n / kFlashRing) & 1, abort_flag)) return nullptr;
    return &items[b];
  };
  auto done_item = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[it_n % kFlashRing]);
    ++it_n;
  };
  const int ppb = 128 / a.page_size;
  auto fetch = [&](int slot, int e, int in_use) -> int {
    int p = -1;
    if (e < in_use) p = a.tables[static_cast<int64_t>(slot) * a.width + e];
    return p >= 0 && p < a.pages ? a.page0 + p : a.page_end;
  };

  if (warp == W_LIST) {
    int n = 0;
    auto publish = [=, &a, &n](const FlashEntry& it) -> bool {
      const int b = n % kFlashRing;
      if (!mbar_wait_warp(&i_empty[b], ((n / kFlashRing) & 1) ^ 1, abort_flag)) return false;
      if (it.valid)
        items[b].pages[lane] = fetch(it.kbase, it.kb0 * ppb + lane, (it.kv_len + a.page_size - 1) / a.page_size);
      if (lane == 0) *static_cast<FlashEntry*>(&items[b]) = it;
      __syncwarp();
      if (lane == 0) mbar_arrive(&i_full[b]);
      ++n;
      return true;
    };
    ok = flash_even(a, lane, prefix, prefix + Cfg::MAX_SEQS, publish);
    FlashEntry end{};
    if (ok) ok = publish(end);
  } else if (warp == W_LOAD) {
    code = kDevTimeoutProducer;
    int st = 0, qi = 0;
    uint32_t ph = 0;
    while (true) {
      const FlashItem* it = next_item();
      if (!(ok = it != nullptr) || !it->valid) break;
      const int kb0 = it->kb0, nb = it->nb[0], kvh = it->kvh, kbase = it->kbase, tok0 = it->tok0;
      const int in_use = (it->kv_len + a.page_size - 1) / a.page_size;
      int page = it->pages[lane], ahead = 0;
      done_item();
      if (nb <= kb0) continue;
      int first = kb0 * ppb;
      if (nb * ppb > first + 32) ahead = fetch(kbase, first + 32 + lane, in_use);
#pragma unroll 1
      for (int j = kb0; ok && j < nb; ++j) {
        if (j * ppb - first == 32) {
          first += 32;
          page = ahead;
          ahead = fetch(kbase, first + 32 + lane, in_use);
        }
        int p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __shfl_sync(0xffffffffu, page, (j * ppb - first + i) & 31);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (!(ok = mbar_wait_warp(&kv_empty[st], ph ^ 1, abort_flag))) break;
          const uint32_t dst = smem_u32(sKV + st * Cfg::TILE), bar = smem_u32(&kv_full[st]);
          const uint64_t map = reinterpret_cast<uint64_t>(kv ? &tm_v : &tm_k);
          if (elect_one()) {
            mbar_arrive_expect_tx(&kv_full[st], Cfg::TILE);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int c = 0; c < AT; ++c)
                if (i < ppb)
                  asm volatile(
                      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                      "[%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst + c * Cfg::ATOM + i * a.page_size * 128),
                      "l"(map), "r"(bar), "r"(c * 64), "r"(kvh), "r"(0), "r"(p[i])
                      : "memory");
          }
          __syncwarp();
          if (++st == ST) {
            st = 0;
            ph ^= 1;
          }
          if (j == kb0 && kv == 0) {
            const int qb = qi & 1;
            const uint32_t qp = (qi >> 1) & 1;
            ++qi;
            if (!(ok = mbar_wait_warp(&q_empty[qb], qp ^ 1, abort_flag))) break;
            if (elect_one()) {
              mbar_arrive_expect_tx(&q_full[qb], AT * static_cast<uint32_t>(G * R) * 128u);
#pragma unroll
              for (int c = 0; c < AT; ++c)
                asm volatile(
                    "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                    "[%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(sQ + qb * Cfg::QBUF + c * Cfg::QATOM)),
                    "l"(reinterpret_cast<uint64_t>(&tm_q)), "r"(smem_u32(&q_full[qb])), "r"(c * 64), "r"(kvh * G),
                    "r"(tok0)
                    : "memory");
            }
            __syncwarp();
          }
        }
      }
      if (!ok) break;
    }
  } else if (warp == W_MMA) {
    code = kDevTimeoutMma;
    if (elect_one()) {
      int st = 0, qi = 0;
      uint32_t ph = 0, g = 0;
      const uint64_t dq = desc_sw128_kmajor(smem_u32(sQ));
      const uint64_t dk = desc_sw128_kmajor(smem_u32(sKV));
      const uint64_t dp = desc_sw128_kmajor(smem_u32(sP));
      // a 64-wide head has one atom: rows 64 .. 127 of O^T repeat the first
      const uint64_t dv = desc_mnmajor<false>(smem_u32(sKV), AT == 2 ? Cfg::ATOM : 0);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool fine = mbar_wait(bar, parity, abort_flag);
        tc_fence_after();
        return fine;
      };
      auto advance = [&] {
        if (++st == ST) {
          st = 0;
          ph ^= 1;
        }
      };
      auto mma_s = [&](int qb, int stage, uint32_t d) {
        const uint64_t q = dq + qb * (Cfg::QBUF >> 4), k = dk + stage * (Cfg::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_f16(d, k + (((kk >> 2) * Cfg::ATOM + (kk & 3) * 32) >> 4),
                   q + (((kk >> 2) * Cfg::QATOM + (kk & 3) * 32) >> 4), IDESC_S, kk > 0);
      };
      while (true) {
        const int b = it_n % kFlashRing;
        if (!(ok = mbar_wait(&i_full[b], (it_n / kFlashRing) & 1, abort_flag))) break;
        const int valid = items[b].valid, n = items[b].nb[0] - items[b].kb0;
        mbar_arrive(&i_empty[b]);
        ++it_n;
        if (!valid) break;
        if (n <= 0) continue;
        const int qb = qi & 1;
        if (!(ok = wait(&q_full[qb], (qi >> 1) & 1)) || !(ok = wait(&kv_full[st], ph))) break;
        ++qi;
        mma_s(qb, st, tmem + (g & 1) * NR);
        umma_commit(&s_full[g & 1]);
        umma_commit(&kv_empty[st]);
        if (n == 1) umma_commit(&q_empty[qb]);
        advance();
#pragma unroll 1
        for (int j = 0; j < n; ++j, ++g) {
          const int sv = st;
          const uint32_t phv = ph;
          advance();
          if (j + 1 < n) {
            if (!(ok = wait(&kv_full[st], ph))) break;
            mma_s(qb, st, tmem + ((g + 1) & 1) * NR);
            umma_commit(&s_full[(g + 1) & 1]);
            umma_commit(&kv_empty[st]);
            if (j + 2 == n) umma_commit(&q_empty[qb]);
            advance();
          }
          if (!(ok = wait(&kv_full[sv], phv)) || !(ok = wait(&p_full[g & 1], (g >> 1) & 1))) break;
          const uint64_t v = dv + sv * (Cfg::TILE >> 4), p = dp + (g & 1) * (Cfg::PBUF >> 4);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_f16(tmem + 2 * NR, v + kk * (2048 >> 4), p + (((kk >> 2) * (NR * 128) + (kk & 3) * 32) >> 4), IDESC_PV,
                     j > 0 || kk > 0);
          umma_commit(&o_full[g & 1]);
          umma_commit(&kv_empty[sv]);
        }
        if (!ok) break;
      }
      if (!ok) {
        report(a.status, code);
        *abort_flag = 1;
      }
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- softmax
    code = kDevTimeoutEpilogue;
    const int key = warp * 32 + lane;  // TMEM lane: key of the block / element of the head
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t o_addr = t_lane + 2 * NR;
    const float sc = a.scale_log2;
    const int nr = G * R;  // rows in use
    int g = 0, e = 0, x = 0;
    // every warp's values of the rows (lane i: row i), from all four warps
    auto exchange = [&](float mine, float (&all)[4][NP]) {
      float* slot = xch + (x & 1) * 4 * NP;
      if (lane < NP) slot[warp * NP + lane] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_bar[x & 1]);
      ok = mbar_wait_warp(&x_bar[x & 1], (x >> 1) & 1, abort_flag);
      ++x;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NP; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(slot + c * NP + i);
          all[c][i] = v.x, all[c][i + 1] = v.y, all[c][i + 2] = v.z, all[c][i + 3] = v.w;
        }
    };
    while (true) {
      const FlashItem* ip = next_item();
      if (!(ok = ip != nullptr) || !ip->valid) break;
      const FlashEntry it = *ip;
      done_item();
      const int n = it.nb[0] - it.kb0, rows = min(nr, it.qv * G);
      float m[NP], l[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++g) {
        const int buf = g & 1;
        if (!(ok = mbar_wait_warp(&s_full[buf], (g >> 1) & 1, abort_flag))) break;
        tc_fence_after();
        const int at = (it.kb0 + j) * 128 + key;  // this lane's key
        if (it.kv_len - (it.kb0 + j) * 128 < 128) {
          // what a page holds behind the sequence: 0 * NaN would not be 0
          const int entry = e + 2 * j + 1;
          if (!(ok = mbar_wait_warp(&kv_full[entry % ST], (entry / ST) & 1, abort_flag))) break;
          if (at >= it.kv_len) {
            uint8_t* v = sKV + (entry % ST) * Cfg::TILE + key * 128;
#pragma unroll 1
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int c = 0; c < AT; ++c) *reinterpret_cast<uint4*>(v + c * Cfg::ATOM + i * 16) = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
        }
        uint32_t s[NP];
        tmem_ld_rows<NP>(t_lane + buf * NR, s);
        tmem_wait_ld();
        float mine = -INFINITY;
        int own = it.pos0, head = 0;  // position of row i's token: the last key that it sees
        // (all NP rows: what lies in those without a query reaches nothing)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (at >= it.kv_len || at > own) s[i] = 0xff800000u;
          if (++head == G) head = 0, ++own;
          const float v = warp_max(__uint_as_float(s[i]));
          mine = lane == i ? v : mine;
        }
        float all[4][NP];
        exchange(mine, all);
        if (!ok) break;
        float corr[NP];
        bool grown = false;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float top = fmaxf(fmaxf(all[0][i], all[1][i]), fmaxf(all[2][i], all[3][i]));
          // keep the older maximum unless the new one is 2^8 above it
          const bool grow = i < rows && ((top - m[i]) * sc > 8.f || (m[i] == -INFINITY && top > m[i]));
          corr[i] = grow ? fa_exp2((m[i] - top) * sc) : 1.f;
          l[i] *= corr[i];
          m[i] = grow ? top : m[i];
          grown |= grow;
        }
        if (grown && j > 0) {  // the same in every thread
          if (!(ok = mbar_wait_warp(&o_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag))) break;
          tc_fence_after();
          uint32_t o[NP];
          tmem_ld_rows<NP>(o_addr, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < NP; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr[i]);
          tmem_st_rows<NP>(o_addr, o);
          tmem_wait_st();
        }
        uint8_t* prow = sP + buf * Cfg::PBUF + (key >> 6) * (NR * 128) + (key & 7) * 2;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float nm = m[i] == -INFINITY ? 0.f : -m[i] * sc;
          const float p = fa_exp2(fmaf(__uint_as_float(s[i]), sc, nm));
          l[i] += p;
          *reinterpret_cast<uint16_t*>(prow + i * 128 + ((((key & 63) >> 3) ^ (i & 7)) << 4)) =
              static_cast<uint16_t>(pack2<T>(p, 0.f));
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      if (!ok) break;
      e += 2 * n;
      // the rows' sums over the lanes, then over the warps
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float v = l[i];
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        mine = lane == i ? v : mine;
      }
      float all[4][NP];
      exchange(mine, all);
      if (!ok) break;
      uint32_t o[NP];
      if (n > 0) {
        if (!(ok = mbar_wait_warp(&o_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag))) break;
        tc_fence_after();
        tmem_ld_rows<NP>(o_addr, o);
        tmem_wait_ld();
        tc_fence_before();
      }
      // the row of this lane's statistics, and its element of every row
      float mine_l = 0.f, mine_m = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        mine_l = lane == i ? (all[0][i] + all[1][i]) + (all[2][i] + all[3][i]) : mine_l;
        mine_m = lane == i ? m[i] : mine_m;
      }
      if (warp == 0 && lane < rows) {
        const float l2 = mine_l == 0.f ? -INFINITY : mine_m * sc + log2f(mine_l);
        if (it.part >= 0) a.part_l[it.part * a.part_rows + lane] = l2;
        else if (a.lse)
          a.lse[static_cast<int64_t>(it.tok0 + lane / G) * a.q_heads + it.kvh * G + lane % G] = l2 * 0.693147180559945309f;
      }
      const float mine_inv = mine_l > 0.f ? 1.f / mine_l : mine_l;  // 0 stays 0, NaN NaN
      int64_t to = it.tok0 * a.ot + static_cast<int64_t>(it.kvh) * G * a.oh + key;
      int head = 0;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float inv = __shfl_sync(0xffffffffu, mine_inv, i);
        const float v = inv == 0.f ? 0.f : __uint_as_float(o[i]) * inv;
        if (it.part >= 0) {
          if (key < HD && i < rows) a.part_o[(static_cast<int64_t>(it.part) * a.part_rows + i) * HD + key] = v;
        } else if (key < a.head_dim && i < rows) {
          reinterpret_cast<uint16_t*>(a.out)[to] = static_cast<uint16_t>(pack2<T>(v, 0.f));
        }
        to += a.oh;
        if (++head == G) head = 0, to += a.ot - G * a.oh;
      }
      const int keys = min(it.kv_len, it.nb[0] * 128);
      if (it.pos0 + 1 < keys) {  // some keys are not seen by some rows
        unsigned odd = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
          if (!(fabsf(__uint_as_float(o[i])) < INFINITY)) odd |= 1u << i;
        odd = __reduce_or_sync(0xffffffffu, key < HD && n > 0 ? odd : 0u);
        if (rows < 32) odd &= (1u << rows) - 1u;
        if (odd)
          flash_again<HD, 1, T>(a, it.tok0, it.pos0, it.kvh, it.kbase, it.kb0 * 128, keys, 0, odd >> lane & 1, it.part,
                                warp * 32, lane);
      }
      __syncwarp();
      if (it.part >= 0) {
        exchange(0.f, all);  // every warp has written its share
        if (!ok) break;
        exchange(warp == 0 && lane == 0 && flash_arrive(a, it) ? 1.f : 0.f, all);
        if (!ok) break;
        if (all[0][0] != 0.f) flash_join<HD, T>(a, it.tok0, it.qv, it.kvh, it.c0, it.parts, warp, lane);
        __syncwarp();
      }
    }
  }
  if (!ok) {
    report(a.status, code);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) {
    }
  }
  if (warp == W_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::COLS);
  }
}

}  // namespace ec
