// kv8_pages_kernels.cuh -- moving sequences and pages of the 8-bit cache about:
// sequences that share pages (fork, free), pages for the tokens to come
// (reserve), and pages in use brought together (compact).
//
// refs[page] counts the page table's entries that hold the page; a page with none is
// free.  A full block is never written again, so sequences with a common
// beginning hold the same pages for it, and a fork copies no codes: only the open block's
// rows, which lie in the sequence's own tail.
//
// All is decided on the device, from lengths and tables as they are there: nothing is read
// back, and the calls go into a captured graph.  Every result is a function of the state
// before the call: pages are given out lowest first, in the order of rows and blocks, and
// counts are integers, so the order in which CTAs run changes nothing.  One call at a time
// works on a cache's pages.
//
// What bounds them, in a graph: the small calls are chains of trips to memory (fork of 4 of 8 slots 4.5 us; free and reserve
// for 2 of 32 slots 9.8, two launches).  Fork of 8 prompts to 128 samples (4 layers of 8 heads of 128): 66 MB written in
// 22.6 us, 2.9 TB/s, the sources out of L2 (written once, with 3 MB read, 10.6 us at the copy rate); issue 43 %, barriers
// between an item's reads and writes.  Free and reserve for 64 of 128 long sequences (62000 entries, 200000 pages): 25 us,
// 16 SMs in step, barriers.  Compaction that moves 336 MB: 123 us, 5.5 TB/s of the measured 6.55.
#pragma once

#include "kv8_cache_kernels.cuh"

namespace b200tx {

struct Kv8Pool {
  uint8_t* codes;       // [layers, pages, 2, kv_heads, 64, D]
  float* scales;        // [layers, pages, 2, kv_heads]
  uint4* tail;          // [layers, slots, 2 (block parity), 2, kv_heads, 64, D] bf16
  int32_t* page_table;  // [slots, max_blocks]
  int32_t* lengths;     // [slots]
  int32_t* refs;        // [pages]
  int32_t* scratch;     // counters (kPoolCounters), then two lists of pages
  int64_t pages;
  int slots, max_blocks, kv_heads, dim, layers;
};

constexpr int kPoolCounters = 64;  // [0] arrivals of a fork's CTAs, [1] moves of a compaction
constexpr int kPoolRows = 2048;    // sequences of a call

// ------------------------------------------------------------------ which rows count
// Of rows that name the same slot one counts: the last (fork) or the first (reserve).  A table of
// twice as many places, in shared memory: the slot, and the row that counts.
struct SlotOwners {
  int* slots;
  int* rows;
  int mask;

  __device__ __forceinline__ int place(int slot) const {
    int at = static_cast<int>((static_cast<uint32_t>(slot) * 2654435761u) >> 8) & mask;
    while (true) {
      const int found = atomicCAS(slots + at, -1, slot);
      if (found == -1 || found == slot) return at;
      at = (at + 1) & mask;
    }
  }
};

// ------------------------------------------------------------------ fork and free
constexpr int kForkThreads = 256;
constexpr int kForkCtas = 3;                                 // of an SM
constexpr int kForkHeld = 8;                                 // 16-byte pieces a thread holds
constexpr int kForkPieces = kForkThreads * kForkHeld;        // of all pairs of an item
static_assert(kForkPieces >= kPoolRows, "an item holds a piece of every pair");

struct Kv8ForkArgs {
  Kv8Pool pool;
  const int32_t* source;  // [pairs], or null: from nothing
  const int32_t* target;  // [pairs]
  int pairs;
  int owners;             // places of the table of slots, a power of two
  int region_log2;        // log2 of the pieces of a head's block
  int piece_shift;        // log2 of the pieces of a pair in a tail item
  int column_shift;       // log2 of the columns in a table item
  int tail_items, table_items;
};

struct __align__(16) ForkPair {
  uint32_t from, to;  // the block's place in the source's and in the target's tail: 16-byte pieces from the layer's first slot
  int pieces;         // of the open block in a head, 0: there is nothing to copy
  int target;         // -1: the pair does nothing
  int source;         // -1: from nothing
  int full;           // full blocks of the source
  int held;           // tokens of the source
  int unused;
};

// All pairs at once: every target becomes what its source was before the call.  An item is
// a place in the tails (or some columns of the table) for all pairs: its values
// are read for every pair before any is written, so a slot may be the source of one pair and the
// target of another (beams that are put in a new order).
__global__ void __launch_bounds__(kForkThreads, kForkCtas) kv8_fork_kernel(const __grid_constant__ Kv8ForkArgs a) {
  extern __shared__ __align__(16) uint8_t fork_smem[];
  __shared__ int s_last, s_most;
  ForkPair* const pair = reinterpret_cast<ForkPair*>(fork_smem);
  SlotOwners owners;
  owners.slots = reinterpret_cast<int*>(pair + a.pairs);
  owners.rows = owners.slots + a.owners;
  owners.mask = a.owners - 1;
  const Kv8Pool& p = a.pool;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();

  for (int i = tid; i < a.owners; i += kForkThreads) owners.slots[i] = owners.rows[i] = -1;
  __syncthreads();
  for (int i = tid; i < a.pairs; i += kForkThreads) {
    const int target = a.target[i];
    if (target >= 0 && target < p.slots) atomicMax(owners.rows + owners.place(target), i);
  }
  __syncthreads();
  const int row = p.dim / 8;           // 16-byte pieces of a token's head
  const int region = kKv8Block * row;  // of a head's block
  const int heads = 2 * p.kv_heads;
  const uint32_t of_parity = static_cast<uint32_t>(heads) * region;  // of a slot's blocks of one parity
  int most = 0;  // pieces of the longest open block
  for (int i = tid; i < a.pairs; i += kForkThreads) {
    ForkPair f = {};
    f.source = a.source == nullptr ? -1 : a.source[i];
    f.target = a.target[i];
    const bool known = f.target >= 0 && f.target < p.slots && f.source < p.slots;
    // a sequence that becomes itself stays as it is, with the pages that are reserved for it
    if (!known || f.source == f.target || owners.rows[owners.place(f.target)] != i) {
      f.target = -1;
    } else if (f.source >= 0) {
      f.held = max(0, p.lengths[f.source]);
      f.full = min(f.held / kKv8Block, p.max_blocks);
      const uint32_t parity = f.held / kKv8Block & 1;
      f.from = (2u * f.source + parity) * of_parity;
      f.to = (2u * f.target + parity) * of_parity;
      f.pieces = f.held % kKv8Block * row;
    } else {
      f.source = -1;
    }
    pair[i] = f;
    most = max(most, f.pieces);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (tid == 0) s_most = 0;
  __syncthreads();
  if (tid % 32 == 0) atomicMax(&s_most, most);
  __syncthreads();
  most = s_most;

  const int each = 1 << a.piece_shift, pieces_log2 = a.region_log2 - a.piece_shift;
  for (int item = blockIdx.x; item < a.tail_items + a.table_items; item += gridDim.x) {
    if (item < a.tail_items) {
      const int part = (item & ((1 << pieces_log2) - 1)) << a.piece_shift;
      if (part >= most) continue;  // past every open block
      const int rest = item >> pieces_log2, layer = rest / heads, head = rest - layer * heads;
      uint4* const base = p.tail + static_cast<int64_t>(layer) * p.slots * 2 * of_parity + static_cast<int64_t>(head) * region;
      uint4 v[kForkHeld];
      uint32_t to[kForkHeld];
#pragma unroll
      for (int j = 0; j < kForkHeld; ++j) {
        const int e = j * kForkThreads + tid, i = e >> a.piece_shift, at = part + (e & (each - 1));
        to[j] = 0xffffffffu;
        if (i >= a.pairs) continue;
        const int4 f = *reinterpret_cast<const int4*>(pair + i);
        if (at >= f.z) continue;
        v[j] = base[static_cast<uint32_t>(f.x) + at];
        to[j] = static_cast<uint32_t>(f.y) + at;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kForkHeld; ++j)
        if (to[j] != 0xffffffffu) base[to[j]] = v[j];
    } else {
      const int columns = 1 << a.column_shift, from = (item - a.tail_items) << a.column_shift;
      int now[kForkHeld], before[kForkHeld];
      int32_t* entry[kForkHeld];
#pragma unroll
      for (int j = 0; j < kForkHeld; ++j) {
        const int e = j * kForkThreads + tid, i = e >> a.column_shift, block = from + (e & (columns - 1));
        now[j] = before[j] = -1;
        entry[j] = nullptr;
        if (i >= a.pairs || block >= p.max_blocks || pair[i].target < 0) continue;
        entry[j] = p.page_table + static_cast<int64_t>(pair[i].target) * p.max_blocks + block;
        before[j] = __ldcg(entry[j]);
        if (block < pair[i].full) now[j] = __ldcg(p.page_table + static_cast<int64_t>(pair[i].source) * p.max_blocks + block);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kForkHeld; ++j) {
        if (entry[j] == nullptr) continue;
        if (now[j] < 0 || now[j] >= p.pages) now[j] = -1;
        if (before[j] == now[j]) continue;
        if (before[j] >= 0 && before[j] < p.pages) atomicSub(p.refs + before[j], 1);
        if (now[j] >= 0) atomicAdd(p.refs + now[j], 1);
        *entry[j] = now[j];
      }
    }
  }

  // The lengths change when every CTA has read them: the last to arrive writes them.
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s_last = atomicInc(reinterpret_cast<unsigned int*>(p.scratch), gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  for (int i = tid; i < a.pairs; i += kForkThreads)
    if (pair[i].target >= 0) p.lengths[pair[i].target] = pair[i].held;
}

// ------------------------------------------------------------------ order over a cluster
// One CTA, or a cluster of them for many pages or entries, does what needs an order over all: each
// takes a stretch, and the stretches' counts go round through (distributed) shared memory.
constexpr int kPoolCtas = 16;  // (more than 8: the most that this GPU allows)
constexpr int kPoolThreads = 1024;
constexpr int kPoolWarps = kPoolThreads / 32;

__device__ __forceinline__ int pool_ctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return static_cast<int>(n);
}

__device__ __forceinline__ void pool_sync(int ctas) {
  if (ctas > 1)
    cluster_sync();
  else
    __syncthreads();
}

struct PoolShared {
  int warp[2][kPoolWarps];
  int cta[2][2][kPoolCtas];  // [exchange's parity][which count][CTA]
};

// N counts that the warps before this one hold, and of all, over the cluster.  All
// threads call it; the counts are a warp's (the same in its lanes).
template <int N>
__device__ __forceinline__ void pool_order(PoolShared& s, int ctas, int& turn, const int (&count)[N], int (&before)[N], int (&all)[N]) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, me = static_cast<int>(cluster_ctarank());
  const int parity = turn++ & 1;
  __syncthreads();
  if (lane < N) s.warp[lane][warp] = lane == 0 ? count[0] : count[N - 1];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int mine = s.warp[k][lane];
    all[k] = __reduce_add_sync(0xffffffffu, mine);
    before[k] = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
    if (ctas > 1 && warp == 0 && lane < ctas)
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(peer_smem_addr(&s.cta[parity][k][me], lane)), "r"(all[k]) : "memory");
  }
  if (ctas == 1) return;
  cluster_sync();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    all[k] = 0;
    for (int i = 0; i < ctas; ++i) {
      if (i < me) before[k] += s.cta[parity][k][i];
      all[k] += s.cta[parity][k][i];
    }
  }
}

// Calls f(page, refs[4]) for this warp's stretch of the pages: four neighbours a lane, 128 a warp, all lanes
// together; refs past the end is -1.
template <typename F>
__device__ __forceinline__ void pool_pages(const Kv8Pool& p, int ctas, F f) {
  const int pages = static_cast<int>(p.pages), warps = ctas * kPoolWarps;
  const int each = ((pages + 127) / 128 + warps - 1) / warps * 128;
  const int64_t warp = cluster_ctarank() * kPoolWarps + threadIdx.x / 32;
  const int from = static_cast<int>(min(static_cast<int64_t>(pages), each * warp));
  const int to = min(pages, from + each);
  constexpr int U = 4;
  for (int at = from; at < to; at += U * 128) {
    int4 refs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int page = at + u * 128 + threadIdx.x % 32 * 4;
      refs[u] = make_int4(-1, -1, -1, -1);
      if (page + 4 <= to) {
        refs[u] = __ldcg(reinterpret_cast<const int4*>(p.refs + page));
      } else {
        if (page < to) refs[u].x = __ldcg(p.refs + page);
        if (page + 1 < to) refs[u].y = __ldcg(p.refs + page + 1);
        if (page + 2 < to) refs[u].z = __ldcg(p.refs + page + 2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at + u * 128 >= to) break;
      const int page = at + u * 128 + threadIdx.x % 32 * 4;
      int four[4] = {refs[u].x, refs[u].y, refs[u].z, refs[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) four[i] = page + i < to ? max(0, four[i]) : -1;
      f(page, four);
    }
  }
}

// The sum of the lanes' counts before this one; `total` of all.
__device__ __forceinline__ int lanes_before(int count, int& total) {
  const int lane = threadIdx.x % 32;
  int sum = count;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  total = __shfl_sync(0xffffffffu, sum, 31);
  return sum - count;
}

// ------------------------------------------------------------------ reserve
struct Kv8ReserveArgs {
  Kv8Pool pool;
  const int32_t* slot_ids;  // [rows] or null = identity
  const int32_t* counts;    // [rows] tokens, or null = tokens
  int32_t* missing;         // [rows]
  int tokens, rows;
  int owners;
};

// The blocks that the next tokens may fill get pages of their own: an entry without a page, or with one
// that another entry holds too, takes the lowest free page.  Entries are in the order
// of rows and blocks; the pages that all entries give back are free for all.
__global__ void __launch_bounds__(kPoolThreads, 1) kv8_reserve_kernel(const __grid_constant__ Kv8ReserveArgs a) {
  extern __shared__ __align__(16) uint8_t reserve_smem[];
  __shared__ PoolShared s;
  int* const slot_of = reinterpret_cast<int*>(reserve_smem);  // [rows]
  int* const begin = slot_of + a.rows;                        // [rows] first block
  int* const upto = begin + a.rows;                           // [rows] entries of the rows up to this one
  SlotOwners owners;
  owners.slots = upto + a.rows;
  owners.rows = owners.slots + a.owners;
  owners.mask = a.owners - 1;
  const Kv8Pool& p = a.pool;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, me = static_cast<int>(cluster_ctarank());
  int turn = 0;
  const int ctas = pool_ctas();
  if (ctas > 1) cluster_sync();
  griddep_wait();
  griddep_launch_dependents();

  if (a.slot_ids != nullptr) {
    for (int i = tid; i < a.owners; i += kPoolThreads) {
      owners.slots[i] = -1;
      owners.rows[i] = kPoolRows;
    }
    __syncthreads();
    for (int b = tid; b < a.rows; b += kPoolThreads) {
      const int slot = a.slot_ids[b];
      slot_of[b] = slot;
      if (slot >= 0 && slot < p.slots) atomicMin(owners.rows + owners.place(slot), b);
    }
    __syncthreads();
  } else {
    for (int b = tid; b < a.rows; b += kPoolThreads) slot_of[b] = b;
  }
  int running = 0;
  for (int base = 0; base < a.rows; base += kPoolThreads) {
    const int b = base + tid;
    int entries = 0;
    if (b < a.rows) {
      const int slot = slot_of[b];
      int past = 0;
      if (slot >= 0 && slot < p.slots && (a.slot_ids == nullptr || owners.rows[owners.place(slot)] == b)) {
        const int64_t held = max(0, p.lengths[slot]), n = a.counts == nullptr ? a.tokens : min(max(a.counts[b], 0), a.tokens);
        const int64_t from = held / kKv8Block, to = (held + n) / kKv8Block;
        begin[b] = static_cast<int>(from);
        entries = static_cast<int>(max(static_cast<int64_t>(0), min(to, static_cast<int64_t>(p.max_blocks)) - from));
        past = static_cast<int>(to - from) - entries;
      }
      if (me == 0) a.missing[b] = past;  // blocks that the table has no place for
    }
    // entries up to and with this row
    int sum = entries;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    __syncthreads();
    if (lane == 31) s.warp[0][warp] = sum;
    __syncthreads();
    const int of_warp = s.warp[0][lane];
    const int warps_before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0);
    if (b < a.rows) upto[b] = running + warps_before + sum;
    running += __reduce_add_sync(0xffffffffu, of_warp);
  }
  __syncthreads();
  const int all_entries = running;

  // this warp's stretch of the entries, 32 neighbours at a time, several of these with their loads in flight
  const int warps = ctas * kPoolWarps;
  const int each = ((all_entries + 31) / 32 + warps - 1) / warps * 32;
  const int first = each * (me * kPoolWarps + warp), last = min(first + each, all_entries);
  constexpr int U = 4;
  // f(page, entry, row, whether there is one) for each entry with its page, all lanes
  auto row_of = [&](int entry, int lo, int hi) {
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (upto[mid] > entry)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  };
  // the rows of this warp's first and last entry: mostly one, or two
  const int row0 = first < last ? row_of(first, 0, a.rows - 1) : 0;
  const int row1 = first < last ? row_of(last - 1, row0, a.rows - 1) : 0;
  auto entries = [&](auto f) {
    int near = row0;
    for (int at = first; at < last; at += 32 * U) {
      int row[U], page[U];
      int32_t* entry[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = at + u * 32 + lane;
        entry[u] = nullptr;
        row[u] = page[u] = 0;
        if (e >= last) continue;
        near = row_of(e, near, row1);
        row[u] = near;
        entry[u] = p.page_table + static_cast<int64_t>(slot_of[near]) * p.max_blocks + begin[near] + (e - (near == 0 ? 0 : upto[near - 1]));
        page[u] = *entry[u];
      }
      f(page, entry, row);
    }
  };
  // A page that another entry holds too: the entry is marked with it, and given back when all are marked.
  int wanted = 0, shared = 0;
  entries([&](int (&page)[U], int32_t* (&entry)[U], int (&)[U]) {
    int refs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool known = entry[u] != nullptr && page[u] >= 0 && page[u] < p.pages;
      refs[u] = known ? p.refs[page[u]] : 0;
      if (!known) page[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool twice = refs[u] > 1, want = entry[u] != nullptr && (page[u] < 0 || twice);
      if (want) *entry[u] = twice ? -2 - page[u] : -1;
      wanted += __popc(__ballot_sync(0xffffffffu, want));
      shared += __popc(__ballot_sync(0xffffffffu, twice));
    }
  });
  int before[2], all[2];
  pool_order(s, ctas, turn, {wanted, shared}, before, all);
  if (all[0] == 0) return;
  if (all[1] != 0) {
    entries([&](int (&page)[U], int32_t* (&)[U], int (&)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (page[u] <= -2) atomicSub(p.refs + (-2 - page[u]), 1);
    });
    pool_sync(ctas);
  }

  int free_pages = 0;
  pool_pages(p, ctas, [&](int, int (&refs)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) free_pages += refs[i] == 0;
  });
  free_pages = __reduce_add_sync(0xffffffffu, free_pages);
  int free_before[1], free_all[1];
  pool_order(s, ctas, turn, {free_pages}, free_before, free_all);
  int32_t* const list = p.scratch + kPoolCounters;
  int at_free = free_before[0];
  if (at_free < all[0]) {
    pool_pages(p, ctas, [&](int page, int (&refs)[4]) {
      int total, k = at_free + lanes_before((refs[0] == 0) + (refs[1] == 0) + (refs[2] == 0) + (refs[3] == 0), total);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (refs[i] != 0) continue;
        if (k < all[0]) list[k] = page + i;
        ++k;
      }
      at_free += total;
    });
  }
  pool_sync(ctas);
  int at_want = before[0];
  entries([&](int (&page)[U], int32_t* (&entry)[U], int (&row)[U]) {
    int given[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool want = entry[u] != nullptr && page[u] < 0;
      const uint32_t bits = __ballot_sync(0xffffffffu, want);
      const int k = at_want + __popc(bits & ((1u << lane) - 1));
      if (!want) entry[u] = nullptr;
      given[u] = want && k < free_all[0] ? __ldcg(list + k) : -1;
      at_want += __popc(bits);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (entry[u] == nullptr) continue;
      *entry[u] = given[u];
      if (given[u] >= 0)
        p.refs[given[u]] = 1;
      else
        atomicAdd(a.missing + row[u], 1);
    }
  });
}

// ------------------------------------------------------------------ compact
struct Kv8CompactArgs {
  Kv8Pool pool;
  int32_t* used;  // [1]
  int64_t page_bytes;
  int piece;      // bytes of a page that a CTA copies at a time
  int pieces;     // of a page
};

// With n pages in use: the k-th page in use from n on goes to the k-th free one below n.
// scratch: the number of moves; where[page], -1 for a free page; the pages that move.
__global__ void __launch_bounds__(kPoolThreads, 1) kv8_compact_plan_kernel(const __grid_constant__ Kv8CompactArgs a) {
  __shared__ PoolShared s;
  const Kv8Pool& p = a.pool;
  int32_t* const where = p.scratch + kPoolCounters;
  int32_t* const list = where + p.pages;  // holes from the front, movers from the back: not more than the pages
  int turn = 0;
  const int ctas = pool_ctas();
  if (ctas > 1) cluster_sync();
  griddep_wait();
  griddep_launch_dependents();
  int held = 0;
  pool_pages(p, ctas, [&](int, int (&refs)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) held += refs[i] > 0;
  });
  held = __reduce_add_sync(0xffffffffu, held);
  int before[2], all[2], none[1], in_use[1];
  pool_order(s, ctas, turn, {held}, none, in_use);
  const int used = in_use[0];
  auto hole_at = [&](int page, int refs) { return refs == 0 && page < used; };
  auto mover_at = [&](int page, int refs) { return refs > 0 && page >= used; };
  int holes = 0, movers = 0;
  pool_pages(p, ctas, [&](int page, int (&refs)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      holes += hole_at(page + i, refs[i]);
      movers += mover_at(page + i, refs[i]);
    }
  });
  pool_order(s, ctas, turn, {__reduce_add_sync(0xffffffffu, holes), __reduce_add_sync(0xffffffffu, movers)}, before, all);
  int hole = before[0], mover = before[1];
  pool_pages(p, ctas, [&](int page, int (&refs)[4]) {
    int to = 0, of = 0, all_to, all_of;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      to += hole_at(page + i, refs[i]);
      of += mover_at(page + i, refs[i]);
    }
    to = hole + lanes_before(to, all_to);
    of = mover + lanes_before(of, all_of);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (refs[i] < 0) continue;
      if (hole_at(page + i, refs[i])) list[to++] = page + i;
      if (mover_at(page + i, refs[i])) list[p.pages - 1 - of++] = page + i;
      where[page + i] = refs[i] > 0 && page + i < used ? page + i : -1;
    }
    hole += all_to;
    mover += all_of;
  });
  pool_sync(ctas);
  const int moves = all[1];
  for (int k = static_cast<int>(cluster_ctarank()) * kPoolThreads + threadIdx.x; k < moves; k += ctas * kPoolThreads) {
    const int to = __ldcg(list + k), of = __ldcg(list + p.pages - 1 - k);
    where[of] = to;
    p.refs[to] = __ldcg(p.refs + of);
    p.refs[of] = 0;
  }
  if (cluster_ctarank() == 0 && threadIdx.x == 0) {
    p.scratch[1] = moves;
    *a.used = used;
  }
}

constexpr int kCompactThreads = 256;
constexpr int kCompactHeld = 8;

__global__ void __launch_bounds__(kCompactThreads) kv8_compact_move_kernel(const __grid_constant__ Kv8CompactArgs a) {
  const Kv8Pool& p = a.pool;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  const int32_t* const where = p.scratch + kPoolCounters;
  const int32_t* const list = where + p.pages;
  const int64_t moves = p.scratch[1], items = moves * p.layers * a.pieces;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int piece = static_cast<int>(item % a.pieces);
    const int64_t rest = item / a.pieces;
    const int layer = static_cast<int>(rest % p.layers);
    const int64_t k = rest / p.layers;
    const int64_t first = layer * p.pages, to = first + list[k], of = first + list[p.pages - 1 - k];
    const uint4* const src = reinterpret_cast<const uint4*>(p.codes + of * a.page_bytes);
    uint4* const dst = reinterpret_cast<uint4*>(p.codes + to * a.page_bytes);
    const int begin = piece * (a.piece / 16), end = min(begin + a.piece / 16, static_cast<int>(a.page_bytes / 16));
    for (int at = begin + tid; at < end; at += kCompactThreads * kCompactHeld) {
      uint4 v[kCompactHeld];
#pragma unroll
      for (int j = 0; j < kCompactHeld; ++j)
        if (at + j * kCompactThreads < end) v[j] = __ldcs(src + at + j * kCompactThreads);
#pragma unroll
      for (int j = 0; j < kCompactHeld; ++j)
        if (at + j * kCompactThreads < end) __stcs(dst + at + j * kCompactThreads, v[j]);
    }
    if (piece == 0)
      for (int i = tid; i < 2 * p.kv_heads; i += kCompactThreads) p.scales[to * 2 * p.kv_heads + i] = p.scales[of * 2 * p.kv_heads + i];
  }
  const int64_t entries = static_cast<int64_t>(p.slots) * p.max_blocks;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kCompactThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCompactThreads + tid; i < entries; i += threads) {
    const int page = p.page_table[i];
    const int now = page >= 0 && page < p.pages ? where[page] : -1;
    if (now != page) p.page_table[i] = now;
  }
}

}  // namespace b200tx
