// ec_kv.cu -- pages of a key / value cache: reserve, fork, free, compact and
// write, on caller-owned device buffers.
//
// A slot's tokens lie in pages of page_size rows; tables[slot][j] is the page
// of its tokens [j * page_size, (j + 1) * page_size), lens[slot] its length
// and refs[page] the number of slots that hold a page (0: free).  Whole pages
// can be shared; a partly filled last page belongs to one slot, so writing
// behind lens[slot] never touches another slot's rows.
//
// Every request is planned by one CTA (its lists are short and pages are given
// out in a fixed order, the lowest free page first, so the state after a call
// does not depend on timing); what moves many bytes runs on a grid that reads
// the plan.  A request either happens as a whole or changes nothing: status[0]
// says which, and every index read from the device is checked before use.
//
// What bounds them: the plans are chains of loads that wait for one another
// (lengths, counts, lists, tables: about 1 us each out of L2), 7 to 11 us a
// plan, so a plan reads ahead what it will need and gives a request to a warp.
// Reserve and fork pass over their lists more than once (claims, checks, sums,
// hand-out) and read lists and lengths again each time, which makes part of that
// chain.  Free, fork, reserve and write for 96 texts (8 layers copied) take 41 us
// together, 12 of them for the bytes.  The copies run near the memory's rate:
// 4096 pages compacted in 51 us, 36 for the bytes.
#include <algorithm>
#include <map>
#include <mutex>

#include "ec_ops.h"

namespace ec {

namespace {
std::mutex g_kv_mu;
std::map<int, std::shared_ptr<const KvOpen>> g_kv;
int g_kv_next = 1;
}  // namespace

std::shared_ptr<const KvOpen> kv_find(int handle) {
  std::lock_guard<std::mutex> lk(g_kv_mu);
  auto it = g_kv.find(handle);
  if (it == g_kv.end()) {
    set_error(EC_EINVAL, "unknown cache handle %d", handle);
    return nullptr;
  }
  return it->second;
}

namespace {

constexpr int kPlanThreads = 1024;

// scratch: the plan's scalars, then per slot a copy (from, to, rows) and a
// claim, then pages handed out or holes, then the new page of a moved page
constexpr int kPlanScalars = 16;
struct Plan {
  int32_t* scalars;
  int4* copies;
  int32_t *claim, *list, *map;
  __host__ __device__ explicit Plan(const KvCache& c)
      : scalars(c.work), copies(reinterpret_cast<int4*>(c.work + kPlanScalars)),
        claim(c.work + kPlanScalars + 4 * static_cast<int64_t>(c.slots)), list(claim + c.slots), map(list + c.pages) {}
};

__device__ __forceinline__ int pages_of(int len, int page) { return (len + page - 1) / page; }

// exclusive prefix sums of x and y over the CTA (kPlanThreads threads), totals
// in sum
__device__ __forceinline__ int2 block_scan2(int x, int y, int2& sum) {
  __shared__ int2 part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 v = make_int2(x, y);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int px = __shfl_up_sync(0xffffffffu, v.x, d), py = __shfl_up_sync(0xffffffffu, v.y, d);
    if (lane >= d) v.x += px, v.y += py;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int2 p = part[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int px = __shfl_up_sync(0xffffffffu, p.x, d), py = __shfl_up_sync(0xffffffffu, p.y, d);
      if (lane >= d) p.x += px, p.y += py;
    }
    part[lane] = p;
  }
  __syncthreads();
  sum = part[31];
  const int2 before = warp ? part[warp - 1] : make_int2(0, 0);
  __syncthreads();
  return make_int2(before.x + v.x - x, before.y + v.y - y);
}
__device__ __forceinline__ int block_scan(int v, int& sum) {
  int2 s2;
  const int before = block_scan2(v, 0, s2).x;
  sum = s2.x;
  return before;
}

// The first pages' counts, read at the start of a plan so that they are there
// when it gets to the free pages: bit i, page 4 * thread + i is free
__device__ __forceinline__ int free_ahead(const KvCache& c) {
  int f = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = threadIdx.x * 4 + i;
    f |= (p < c.pages && c.refs[p] == 0) << i;
  }
  return f;
}

// The `need` lowest free pages into list; false if there are fewer.
__device__ bool find_free(const KvCache& c, int32_t* list, int64_t need, int ahead) {
  int64_t got = 0;
  for (int p0 = 0; p0 < c.pages && got < need; p0 += kPlanThreads * 4) {
    int f = ahead;
    if (p0) {
      f = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + threadIdx.x * 4 + i;
        f |= (p < c.pages && c.refs[p] == 0) << i;
      }
    }
    int sum;
    int64_t r = got + block_scan(__popc(f), sum);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f >> i & 1) {
        if (r < need) list[r] = p0 + threadIdx.x * 4 + i;
        ++r;
      }
    got += sum;
  }
  __syncthreads();
  return got >= need;
}

// Whether slots[0..n) are slots and no two are the same.  A slot is claimed by
// the index that names it; whoever does not find its own claim is a second.  A
// list longer than the cache has slots names one twice, and is not read.
__device__ bool claim_slots(const KvCache& c, int32_t* claim, const int32_t* slots, int n) {
  if (n > c.slots) return false;
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = slots[i];
    if (s < 0 || s >= c.slots) bad = true;
    else claim[s] = i;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = slots[i];
    if (s >= 0 && s < c.slots && claim[s] != i) bad = true;
  }
  return !__syncthreads_or(bad);
}

__device__ __forceinline__ bool bad_len(const KvCache& c, int len) {
  return len < 0 || len > static_cast<int64_t>(c.width) * c.page_size;
}

// ---------------------------------------------------------------- reserve --
__global__ void __launch_bounds__(kPlanThreads) kv_reserve_kernel(const KvCache c, const int32_t* slots,
                                                                  const int32_t* add, int n, int32_t* status) {
  __shared__ int4 request[kPlanThreads];  // slot, pages it has, pages more, their place in the list
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  const int ahead = free_ahead(c);
  const bool ok = claim_slots(c, plan.claim, slots, n);
  bool bad = false;
  if (ok)
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
      const int len = c.lens[slots[i]], more = add[i];
      bad |= bad_len(c, len) || more < 0 || static_cast<int64_t>(len) + more > static_cast<int64_t>(c.width) * c.page_size;
    }
  if (__syncthreads_or(bad || !ok)) {
    if (threadIdx.x == 0) status[0] = EC_KV_BAD, status[1] = 0;
    return;
  }
  int64_t need = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int v = 0;
    if (i < n) {
      const int len = c.lens[slots[i]];
      v = pages_of(len + add[i], c.page_size) - pages_of(len, c.page_size);
      v = min(v, c.pages + 1);  // at most 2^20 + 1: the sum over a CTA fits 32 bits
    }
    int sum;
    block_scan(v, sum);
    need += sum;
  }
  if (need > c.pages || !find_free(c, plan.list, need, ahead)) {
    if (threadIdx.x == 0) status[0] = EC_KV_FULL, status[1] = static_cast<int32_t>(min(need, int64_t(INT32_MAX)));
    return;
  }
  const int lane = threadIdx.x & 31;
  int at = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int have = 0, v = 0, s = 0;
    if (i < n) {
      s = slots[i];
      const int len = c.lens[s], more = add[i];
      have = pages_of(len, c.page_size);
      v = pages_of(len + more, c.page_size) - have;
      c.lens[s] = len + more;
    }
    int sum;
    const int off = at + block_scan(v, sum);
    request[threadIdx.x] = make_int4(s, have, v, off);
    __syncthreads();
    // a warp per request
    for (int k = threadIdx.x >> 5; k < min(n - i0, kPlanThreads); k += kPlanThreads / 32) {
      const int4 q = request[k];
      for (int j = lane; j < q.z; j += 32) {
        const int p = plan.list[q.w + j];
        c.tables[static_cast<int64_t>(q.x) * c.width + q.y + j] = p;
        c.refs[p] = 1;
      }
    }
    __syncthreads();
    at += sum;
  }
  if (threadIdx.x == 0) status[0] = EC_KV_OK, status[1] = static_cast<int32_t>(need);
}

// ------------------------------------------------------------------- fork --
// the copy of every source's partly filled page goes to list[rank]
__global__ void __launch_bounds__(kPlanThreads) kv_fork_plan_kernel(const KvCache c, const int32_t* src,
                                                                    const int32_t* dst, int n, int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  const int ahead = free_ahead(c);
  const bool ok = claim_slots(c, plan.claim, dst, n);
  bool bad = false;
  if (ok)
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
      const int s = src[i];
      if (s < 0 || s >= c.slots) {
        bad = true;
        continue;
      }
      // a source that is itself filled by this call
      const int by = plan.claim[s];
      bad |= by >= 0 && by < n && dst[by] == s;
      bad |= bad_len(c, c.lens[s]) || c.lens[dst[i]] != 0;
    }
  if (__syncthreads_or(bad || !ok)) {
    if (threadIdx.x == 0) status[0] = EC_KV_BAD, status[1] = 0, plan.scalars[0] = 0;
    return;
  }
  int need = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int sum;
    block_scan(i < n && c.lens[src[i]] % c.page_size ? 1 : 0, sum);
    need += sum;
  }
  if (need > c.pages || !find_free(c, plan.list, need, ahead)) {
    if (threadIdx.x == 0) status[0] = EC_KV_FULL, status[1] = need, plan.scalars[0] = 0;
    return;
  }
  // the copy's page is the destination's last one; the rest follows
  int at = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    const int s = i < n ? src[i] : 0, len = i < n ? c.lens[s] : 0;
    const int v = len % c.page_size ? 1 : 0;
    int sum;
    const int off = at + block_scan(v, sum);
    if (i < n) {
      int4 copy = make_int4(-1, -1, 0, len);
      if (v) {
        const int p = plan.list[off], from = c.tables[static_cast<int64_t>(s) * c.width + len / c.page_size];
        c.tables[static_cast<int64_t>(dst[i]) * c.width + len / c.page_size] = p;
        c.refs[p] = 1;
        if (from >= 0 && from < c.pages) copy = make_int4(from, p, len % c.page_size, len);
      }
      plan.copies[i] = copy;
    }
    at += sum;
  }
  if (threadIdx.x == 0) status[0] = EC_KV_OK, status[1] = need, plan.scalars[0] = 1;
}

// rows [0, rows) of page `from` to page `to`, in layer l of the keys (kv 0)
// or values (kv 1)
__device__ __forceinline__ void copy_rows(const KvCache& c, int l, int kv, int from, int to, int rows) {
  const int64_t row = static_cast<int64_t>(c.heads) * c.head_dim / 8;  // 16-byte pieces
  uint4* base = static_cast<uint4*>(kv ? c.v : c.k) + static_cast<int64_t>(l) * c.pages * c.page_size * row;
  const uint4* s = base + static_cast<int64_t>(from) * c.page_size * row;
  uint4* d = base + static_cast<int64_t>(to) * c.page_size * row;
  const int n = static_cast<int>(rows * row);  // at most 128 x 1024 x 16
  constexpr int B = 8;  // pieces under way per thread
  for (int i0 = threadIdx.x; i0 < n; i0 += B * blockDim.x) {
    uint4 v[B];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (i0 + b * blockDim.x < n) v[b] = s[i0 + b * blockDim.x];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (i0 + b * blockDim.x < n) d[i0 + b * blockDim.x] = v[b];
  }
}

// block (i, piece): piece 0 also shares the whole pages of request i
__global__ void kv_fork_copy_kernel(const KvCache c, const int32_t* src, const int32_t* dst) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  const int i = blockIdx.x;
  const int4 copy = plan.copies[i];  // there is one for every slot, and no more blocks than that
  if (plan.scalars[0] == 0) return;
  if (blockIdx.y == 0) {
    const int full = copy.w / c.page_size;
    const int32_t* from = c.tables + static_cast<int64_t>(src[i]) * c.width;
    int32_t* to = c.tables + static_cast<int64_t>(dst[i]) * c.width;
    for (int j = threadIdx.x; j < full; j += blockDim.x) {
      const int p = from[j];
      to[j] = p;
      if (p >= 0 && p < c.pages) atomicAdd(&c.refs[p], 1);
    }
    if (threadIdx.x == 0) c.lens[dst[i]] = copy.w;
  }
  for (int l = blockIdx.y; copy.z && l < 2 * c.layers; l += gridDim.y) copy_rows(c, l >> 1, l & 1, copy.x, copy.y, copy.z);
}

// ------------------------------------------------------------------- free --
// kFreeAlone table entries or fewer: this CTA does it all; else it plans for
// kv_free_kernel
constexpr int kFreeAlone = 16384;
__global__ void __launch_bounds__(kPlanThreads) kv_free_plan_kernel(const KvCache c, const int32_t* slots, int n,
                                                                    int32_t* status, int alone) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  const bool ok = claim_slots(c, plan.claim, slots, n);
  bool bad = false;
  if (ok)
    for (int i = threadIdx.x; i < n; i += kPlanThreads) bad |= bad_len(c, c.lens[slots[i]]);
  bad = __syncthreads_or(bad || !ok);
  int gone = 0;
  if (alone && !bad) {
    // four table entries under way per thread; the lengths go last
    constexpr int B = 4;
    const int all = n * c.width;
    for (int e0 = threadIdx.x; e0 < all; e0 += B * kPlanThreads) {
      int32_t* at[B];
      int page[B], held[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int e = e0 + b * kPlanThreads, s = e < all ? slots[e / c.width] : 0;
        at[b] = c.tables + static_cast<int64_t>(s) * c.width + e % c.width;
        page[b] = e < all ? *at[b] : -1;
        held[b] = e < all && e % c.width < pages_of(c.lens[s], c.page_size);
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (e0 + b * kPlanThreads < all) *at[b] = -1;
        if (held[b] && page[b] >= 0 && page[b] < c.pages) gone += atomicSub(&c.refs[page[b]], 1) == 1;
      }
    }
    int sum;
    block_scan(gone, sum);  // also: every length has been read
    gone = sum;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) c.lens[slots[i]] = 0;
  }
  if (threadIdx.x == 0) status[0] = bad ? EC_KV_BAD : EC_KV_OK, status[1] = gone, plan.scalars[0] = !bad;
}

// block per slot: its pages let go, its row of the table cleared
__global__ void kv_free_kernel(const KvCache c, const int32_t* slots, int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  if (plan.scalars[0] == 0) return;
  const int s = slots[blockIdx.x];
  const int np = pages_of(c.lens[s], c.page_size);
  __syncthreads();
  int32_t* row = c.tables + static_cast<int64_t>(s) * c.width;
  int gone = 0;
  for (int j = threadIdx.x; j < c.width; j += blockDim.x) {
    const int p = row[j];
    if (j < np && p >= 0 && p < c.pages) gone += atomicSub(&c.refs[p], 1) == 1;
    row[j] = -1;
  }
  gone = __reduce_add_sync(0xffffffffu, gone);
  if ((threadIdx.x & 31) == 0 && gone) atomicAdd(&status[1], gone);
  if (threadIdx.x == 0) c.lens[s] = 0;
}

// ---------------------------------------------------------------- compact --
// list[r]: the r-th hole below the number of live pages; map[p]: the hole
// that live page p above it moves to; scalars: {live, moves}
__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(const KvCache c, int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  int live = 0;
  for (int p0 = 0; p0 < c.pages; p0 += kPlanThreads * 4) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + threadIdx.x * 4 + i;
      n += p < c.pages && c.refs[p] > 0;
    }
    int sum;
    block_scan(n, sum);
    live += sum;
  }
  int holes = 0;
  for (int p0 = 0; p0 < live; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const int v = p < live && c.refs[p] <= 0;
    int sum;
    const int r = holes + block_scan(v, sum);
    if (v) plan.list[r] = p;
    holes += sum;
  }
  __syncthreads();
  int moves = 0;
  for (int p0 = live; p0 < c.pages && moves < holes; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const int v = p < c.pages && c.refs[p] > 0;
    int sum;
    const int r = moves + block_scan(v, sum);
    if (v) {
      const int to = plan.list[r];
      plan.map[p] = to;
      plan.map[r] = p;  // r < holes <= live <= p: the page that fills hole r
      c.refs[to] = c.refs[p];
      c.refs[p] = 0;
    }
    moves += sum;
  }
  if (threadIdx.x == 0) {
    plan.scalars[0] = live;
    plan.scalars[1] = moves;
    status[0] = EC_KV_OK;
    status[1] = moves;
  }
}

__global__ void kv_compact_copy_kernel(const KvCache c) {
  pdl_wait();
  pdl_trigger();
  const Plan plan(c);
  const int live = plan.scalars[0], moves = plan.scalars[1];
  if (moves == 0) return;
  const int per = 2 * c.layers;
  for (int64_t w = blockIdx.x; w < static_cast<int64_t>(moves) * per; w += gridDim.x) {
    const int r = static_cast<int>(w / per), l = static_cast<int>(w % per);
    copy_rows(c, l >> 1, l & 1, plan.map[r], plan.list[r], c.page_size);
  }
  // the tables of the slots in use
  const int64_t n = static_cast<int64_t>(c.slots) * c.width;
  for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int p = c.tables[e];
    if (p < live || p >= c.pages) continue;
    if (static_cast<int>(e % c.width) < pages_of(c.lens[e / c.width], c.page_size)) c.tables[e] = plan.map[p];
  }
}

// ------------------------------------------------------------------ write --
struct WriteArgs {
  const uint4 *k, *v;
  int64_t kt, kh, vt, vh;  // strides in 16-byte pieces
  int64_t tokens;
  const int32_t *cu, *slots;
  int nseq, layer;
};

// A block takes kWriteTokens tokens: a warp finds each one's sequence (32 ways
// at a time) and place in the cache, then all copy 16-byte pieces, four of the
// keys and four of the values under way per thread.
constexpr int kWriteTokens = 8;
__global__ void __launch_bounds__(kWriteTokens * 32) kv_write_kernel(const KvCache c, const WriteArgs a) {
  __shared__ int64_t at[kWriteTokens];  // row in the pool, -1: none
  pdl_wait();
  pdl_trigger();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kWriteTokens;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    const int64_t t = t0 + warp;
    int64_t row = -1;
    if (t < a.tokens) {
      // last sequence that starts at or before t
      int lo = 0, hi = a.nseq;
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, s = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, s < hi && a.cu[s] <= t);
        const int k = m ? 31 - __clz(m) : 0;
        hi = min(hi, lo + (k + 1) * step);
        lo = lo + k * step;
      }
      const int64_t begin = a.cu[lo], end = a.cu[lo + 1];
      const int s = a.slots ? a.slots[lo] : lo;
      if (begin <= t && t < end && s >= 0 && s < c.slots) {
        const int64_t p = c.lens[s] - (end - t);
        if (p >= 0 && p < static_cast<int64_t>(c.width) * c.page_size) {
          const int page = c.tables[static_cast<int64_t>(s) * c.width + p / c.page_size];
          if (page >= 0 && page < c.pages) row = static_cast<int64_t>(page) * c.page_size + p % c.page_size;
        }
      }
    }
    if (lane == 0) at[warp] = row;
  }
  __syncthreads();
  const int piece = c.head_dim / 8, row = c.heads * piece, n = kWriteTokens * row;
  const int64_t pool = static_cast<int64_t>(a.layer) * c.pages * c.page_size * row;
  uint4 *dk = static_cast<uint4*>(c.k) + pool, *dv = static_cast<uint4*>(c.v) + pool;
  constexpr int B = 4;
  for (int e0 = threadIdx.x; e0 < n; e0 += B * blockDim.x) {
    uint4 k[B], v[B];
    int64_t to[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int e = e0 + b * blockDim.x;
      to[b] = -1;
      if (e >= n) continue;
      const int i = e / row, r = e % row, h = r / piece, x = r % piece;
      if (at[i] < 0) continue;
      to[b] = at[i] * row + r;
      k[b] = a.k[(t0 + i) * a.kt + h * a.kh + x];
      v[b] = a.v[(t0 + i) * a.vt + h * a.vh + x];
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (to[b] >= 0) {
        dk[to[b]] = k[b];
        dv[to[b]] = v[b];
      }
  }
}

int check_lists(const void* a, const void* b, int n, const void* status) {
  if (n < 0) return set_error(EC_EINVAL, "negative count");
  if (!status || (n > 0 && (!a || !b))) return set_error(EC_EINVAL, "a list or the status is NULL");
  if (!op_aligned(a, 4) || !op_aligned(b, 4) || !op_aligned(status, 4))
    return set_error(EC_EINVAL, "lists and status must be 4-byte aligned");
  return EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" int64_t ec_kv_work_size(int pages, int slots) {
  clear_error();
  if (pages < 1 || slots < 1) return set_error(EC_EINVAL, "pages and slots must be positive");
  return 4 * (2 * static_cast<int64_t>(pages) + 5 * static_cast<int64_t>(slots) + kPlanScalars);
}

extern "C" int ec_kv_open(void* k, void* v, int dtype, int layers, int pages, int page_size, int heads, int head_dim,
                          int32_t* tables, int slots, int table_width, int32_t* lens, int32_t* refs, void* work,
                          int64_t work_bytes, int* handle) {
  clear_error();
  if (!k || !v || !tables || !lens || !refs || !work || !handle) return set_error(EC_EINVAL, "a cache buffer is NULL");
  if (dtype != EC_BF16 && dtype != EC_F16) return set_error(EC_EINVAL, "a cache holds bf16 or f16, not dtype %d", dtype);
  if (layers < 1 || layers > 65536 || pages < 1 || pages > (1 << 20) || slots < 1 || slots > (1 << 24) ||
      table_width < 1 || table_width > (1 << 24) || heads < 1 || heads > 1024)
    return set_error(EC_EINVAL, "bad cache shape: %d layers of %d pages, %d heads, %d slots of %d pages", layers, pages,
                     heads, slots, table_width);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return set_error(EC_EINVAL, "page_size %d (supported: 16, 32, 64, 128)", page_size);
  if (head_dim < 8 || head_dim > 128 || head_dim % 8)
    return set_error(EC_EINVAL, "head_dim %d (supported: multiples of 8 up to 128)", head_dim);
  if (static_cast<int64_t>(table_width) * page_size > (1 << 30))
    return set_error(EC_EINVAL, "a table row of %d pages passes 2^30 tokens", table_width);
  if (static_cast<int64_t>(layers) * pages > (1 << 30))
    return set_error(EC_EINVAL, "%d layers of %d pages pass 2^30 pages", layers, pages);
  if (!op_aligned(k, 16) || !op_aligned(v, 16) || !op_aligned(work, 16))
    return set_error(EC_EINVAL, "pages and work must be 16-byte aligned");
  if (!op_aligned(tables, 4) || !op_aligned(lens, 4) || !op_aligned(refs, 4))
    return set_error(EC_EINVAL, "tables, lens and refs must be 4-byte aligned");
  if (work_bytes < ec_kv_work_size(pages, slots))
    return set_error(EC_EINVAL, "work holds %lld bytes, the cache needs %lld", static_cast<long long>(work_bytes),
                     static_cast<long long>(ec_kv_work_size(pages, slots)));
  return guarded("kv open", [&] {
    auto c = std::make_shared<KvOpen>(KvCache{k, v, dtype, layers, pages, page_size, heads, head_dim, tables, slots,
                                              table_width, lens, refs, static_cast<int32_t*>(work)});
    std::lock_guard<std::mutex> lk(g_kv_mu);
    g_kv.emplace(g_kv_next, std::move(c));
    *handle = g_kv_next++;
    return EC_OK;
  });
}

extern "C" int ec_kv_close(int handle) {
  clear_error();
  if (!kv_find(handle)) return EC_EINVAL;
  std::lock_guard<std::mutex> lk(g_kv_mu);
  g_kv.erase(handle);
  return EC_OK;
}

extern "C" int ec_kv_reserve(int handle, const int32_t* slots, const int32_t* add, int n, int32_t* status,
                             void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (int rc = check_lists(slots, add, n, status)) return rc;
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {slots, add, status})) return rc;
  return check_cuda(launch_pdl(kv_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), *c,
                               slots, add, n, status),
                    "kv reserve");
}

extern "C" int ec_kv_fork(int handle, const int32_t* src, const int32_t* dst, int n, int32_t* status, void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (int rc = check_lists(src, dst, n, status)) return rc;
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {src, dst, status})) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = check_cuda(launch_pdl(kv_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, *c, src, dst, n, status),
                          "kv fork"))
    return rc;
  if (n == 0 || n > c->slots) return EC_OK;  // the plan refuses the latter; its scratch has `slots` copies
  return check_cuda(launch_pdl(kv_fork_copy_kernel, dim3(n, std::min(2 * c->layers, 65535)), dim3(256), 0, st, *c, src,
                               dst),
                    "kv fork copy");
}

extern "C" int ec_kv_free(int handle, const int32_t* slots, int n, int32_t* status, void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (int rc = check_lists(slots, slots, n, status)) return rc;
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {slots, status})) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int alone = static_cast<int64_t>(n) * c->width <= kFreeAlone;
  if (int rc = check_cuda(launch_pdl(kv_free_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, *c, slots, n, status, alone),
                          "kv free"))
    return rc;
  if (alone || n > c->slots) return EC_OK;
  return check_cuda(launch_pdl(kv_free_kernel, dim3(n), dim3(128), 0, st, *c, slots, status), "kv free");
}

extern "C" int ec_kv_compact(int handle, int32_t* status, void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (int rc = check_lists(status, status, 0, status)) return rc;
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {status})) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = check_cuda(launch_pdl(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, *c, status), "kv compact"))
    return rc;
  return check_cuda(launch_pdl(kv_compact_copy_kernel, dim3(dev.num_sms() * 8), dim3(256), 0, st, *c), "kv compact copy");
}

extern "C" int ec_kv_write(int handle, int layer, const void* k, int64_t k_token, int64_t k_head, const void* v,
                           int64_t v_token, int64_t v_head, int64_t tokens, const int32_t* cu, const int32_t* slots,
                           int nseq, void* stream) {
  clear_error();
  auto c = kv_find(handle);
  if (!c) return EC_EINVAL;
  if (layer < 0 || layer >= c->layers) return set_error(EC_EINVAL, "layer %d of %d", layer, c->layers);
  // (more sequences than any cache has slots; the search adds such counts)
  if (tokens < 0 || tokens > INT32_MAX || nseq < 0 || nseq > (1 << 30)) return set_error(EC_EINVAL, "bad token or sequence count");
  OpRows kr{k, k_token, k_head}, vr{v, v_token, v_head};
  if (int rc = op_check_rows("k", kr, tokens, c->heads, c->head_dim)) return rc;
  if (int rc = op_check_rows("v", vr, tokens, c->heads, c->head_dim)) return rc;
  if (tokens == 0 || nseq == 0) return EC_OK;
  if (!cu || !op_aligned(cu, 4) || !op_aligned(slots, 4)) return set_error(EC_EINVAL, "cu is NULL or a list misaligned");
  OpDevice dev;
  if (int rc = kv_enter(dev, *c, {k, v, cu, slots})) return rc;
  const WriteArgs a{static_cast<const uint4*>(k), static_cast<const uint4*>(v), kr.token / 8, kr.head / 8, vr.token / 8,
                    vr.head / 8, tokens, cu, slots, nseq, layer};
  const int64_t grid = (tokens + kWriteTokens - 1) / kWriteTokens;
  return check_cuda(launch_pdl(kv_write_kernel, dim3(static_cast<unsigned>(grid)), dim3(kWriteTokens * 32), 0,
                               static_cast<cudaStream_t>(stream), *c, a),
                    "kv write");
}
