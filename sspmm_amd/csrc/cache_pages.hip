// Pages of the cache: which are free is what their reference counts say, and the lowest free ones are taken first, so that a
// run of calls gives the same tables every time.
#include "cache_pages.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr size_t kPlanLds = 15 * 1024;  // integers of a plan that stay in LDS

// Sum of v over the threads before this one, and over all of them.  Two barriers; `share` holds kPlanWaves values.
__device__ __forceinline__ uint32_t block_exclusive_sum(uint32_t v, uint32_t *share, uint32_t *all) {
  const int wave = threadIdx.x >> 6;
  const uint32_t upto = wave_inclusive_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) share[wave] = upto;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const uint32_t x = share[w];
    before += w < wave ? x : 0u;
    total += x;
  }
  *all = total;
  return before + upto - v;
}

// The lowest free pages, up to `need` of them, into list, each with one reference from now on.  Returns how many there were.
__device__ uint32_t take_free_pages(int32_t *refs, int pages, uint32_t need, int32_t *list, uint32_t *share) {
  uint32_t found = 0;
  for (int p0 = 0; p0 < pages && found < need; p0 += 4 * kPlanThreads) {
    const int p = p0 + 4 * (int)threadIdx.x;
    bool is_free[4];
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      is_free[i] = p + i < pages && refs[p + i] <= 0;
      count += is_free[i];
    }
    uint32_t all;
    uint32_t rank = found + block_exclusive_sum(count, share, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (is_free[i]) {
        if (rank < need) {
          list[rank] = p + i;
          refs[p + i] = 1;
        }
        ++rank;
      }
    found += all;
  }
  __syncthreads();
  return min(found, need);
}

// The slots of row b that begin with one of the new tokens, at positions starts[b] ..: first .. end - 1.  (A slot that they go on in has its page, or has lost the
// tokens in front of them: a page given to it now would show what was in it before as theirs.)
__device__ __forceinline__ void new_slots(const int32_t *starts, const int32_t *offsets, int b, int page_size, int slots, int *first, int *end) {
  const int start = starts[b];
  const long long n = (long long)offsets[b + 1] - offsets[b];
  *first = 0;
  *end = 0;
  if (start < 0 || n <= 0) return;
  *first = start / page_size + (start % page_size != 0);
  *end = (int)min((long long)slots, (start + n + page_size - 1) / page_size);
}

// Chains of loads and barriers, one workgroup, whose waves take their rows one after the other: 48 rows of one new token 3.0 us where all pages are there and 6.0
// where one is given, five prompts 2.0 and 5.0 (127 pages); 256 rows 9.6 and 21, 4096 rows 138 and 275, and 356 where a quarter of a million pages in use come first.
// A wave counts a row's slots without a page, ranks follow in the order of rows and slots, the list of free pages is made, and
// the slots take theirs.  workspace: the ranks, then the list; null: in LDS.
__global__ __launch_bounds__(kPlanThreads) void reserve_pages_kernel(const PageTable t, const int32_t *starts, const int32_t *offsets, int page_size,
                                                                     int32_t *workspace) {
  __shared__ uint32_t share[kPlanWaves];
  extern __shared__ int32_t plan_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (!workspace) workspace = plan_lds;
  uint32_t *const ranks = reinterpret_cast<uint32_t *>(workspace);
  int32_t *const list = workspace + t.rows;
  for (int b = wave; b < t.rows; b += kPlanWaves) {
    int first, end;
    new_slots(starts, offsets, b, page_size, t.slots, &first, &end);
    uint32_t missing = 0;
    for (int s0 = first; s0 < end; s0 += 64) {
      const int s = s0 + lane;
      missing += __popcll(__ballot(s < end && t.table[(long long)b * t.slots + s] < 0));
    }
    if (lane == 0) ranks[b] = missing;
  }
  __syncthreads();
  uint32_t need = 0;
  for (int b0 = 0; b0 < t.rows; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const uint32_t v = b < t.rows ? ranks[b] : 0u;
    uint32_t all;
    const uint32_t before = block_exclusive_sum(v, share, &all);
    if (b < t.rows) ranks[b] = need + before;
    need += all;
  }
  if (need == 0) return;
  const uint32_t found = take_free_pages(t.refs, t.pages, need, list, share);
  for (int b = wave; b < t.rows; b += kPlanWaves) {
    int first, end;
    new_slots(starts, offsets, b, page_size, t.slots, &first, &end);
    uint32_t rank = ranks[b];
    for (int s0 = first; s0 < end; s0 += 64) {
      const int s = s0 + lane;
      int32_t *const at = t.table + (long long)b * t.slots + s;
      const bool is = s < end && *at < 0;
      const unsigned long long which = __ballot(is);
      const uint32_t mine = rank + __popcll(which & ((1ull << lane) - 1));
      if (is && mine < found) *at = list[mine];
      rank += __popcll(which);
    }
  }
}

// A workgroup a named row.  An entry is taken out of the table by whoever comes first, so a row named twice is given back once.
__global__ __launch_bounds__(256) void release_pages_kernel(const PageTable t, int32_t *lengths, const int32_t *named) {
  const int row = named[blockIdx.x];
  if (row < 0 || row >= t.rows) return;
  if (threadIdx.x == 0) lengths[row] = 0;
  for (int s = threadIdx.x; s < t.slots; s += 256) {
    const int page = atomicExch(&t.table[(long long)row * t.slots + s], -1);
    if (page >= 0 && page < t.pages) atomicSub(&t.refs[page], 1);
  }
}

// What becomes of a child: the page that is copied for it (or -1) and to which, the slots that it shares.
struct Fork {
  int32_t child, parent, source, target, shared;  // child -1: nothing
};

// 4.7 us: six barriers and the loads between them.  One workgroup.  Per row the last naming as a child holds; a row that becomes another's copy in the call cannot be a
// parent in it; a row that is named its own parent stays as it is.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(const PageTable t, int32_t *lengths, const int32_t *parents, const int32_t *children, int count,
                                                                 int page_size, int32_t *workspace) {
  __shared__ uint32_t share[kPlanWaves];
  const int tid = threadIdx.x;
  int32_t *const mark = workspace, *const list = workspace + t.rows;
  Fork *const forks = reinterpret_cast<Fork *>(list + count);
  for (int r = tid; r < t.rows; r += kPlanThreads) mark[r] = -1;
  __syncthreads();
  for (int i = tid; i < count; i += kPlanThreads)
    if (children[i] >= 0 && children[i] < t.rows) atomicMax(&mark[children[i]], i);
  __syncthreads();
  uint32_t need = 0;
  for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
    const int i = i0 + tid;
    Fork f = {-1, -1, -1, -1, 0};
    if (i < count && children[i] >= 0 && children[i] < t.rows && mark[children[i]] == i && parents[i] != children[i]) {
      f.child = children[i];
      const int parent = parents[i];
      if (parent >= 0 && parent < t.rows && (mark[parent] < 0 || parents[mark[parent]] == parent)) {
        const int length = (int)max(0ll, min((long long)lengths[parent], (long long)t.slots * page_size));
        f.parent = parent;
        f.shared = length / page_size;
        if (length % page_size > 0) {
          f.source = t.table[(long long)parent * t.slots + f.shared];
          if (f.source < 0 || f.source >= t.pages) f.source = f.parent = -1;  // (its last tokens are nowhere)
        }
      }
    }
    uint32_t all;
    const uint32_t rank = need + block_exclusive_sum(f.source >= 0 ? 1u : 0u, share, &all);
    if (f.source >= 0) f.target = (int)rank;  // its rank, for now
    if (i < count) forks[i] = f;
    need += all;
  }
  const uint32_t found = need > 0 ? take_free_pages(t.refs, t.pages, need, list, share) : 0;
  __syncthreads();
  for (int i = tid; i < count; i += kPlanThreads) {
    Fork f = forks[i];
    if (f.child < 0) continue;
    if (f.source >= 0) {
      if ((uint32_t)f.target < found) {
        f.target = list[f.target];
      } else {
        f.source = f.parent = -1;
      }
    }
    if (f.source < 0) f.target = -1;
    if (f.parent < 0) f.shared = 0;
    lengths[f.child] = f.parent < 0 ? 0 : max(0, lengths[f.parent]);  // (tokens behind the table count, as they do for the parent)
    forks[i] = f;
  }
}

// A part of page `source` to page `target`.  Bound by memory: 131 MB of pages 65.7 us a call as one piece of 16 bytes of either side after the other, 63.3 with
// four of them on their way and twice as many workgroups (the plan before it is 5 of these; 42 us and 6.3 TB/s where the last-level cache has the pool).
__device__ __forceinline__ void copy_page(const PagePool &pool, int source, int target, int part, int parts) {
  const long long pieces = pool.block_bytes / 16;
  const long long from = pieces * part / parts, upto = pieces * (part + 1) / parts;
  const uintx4 *const k0 = reinterpret_cast<const uintx4 *>(pool.keys + source * pool.block_bytes), *const v0 = reinterpret_cast<const uintx4 *>(pool.values + source * pool.block_bytes);
  uintx4 *const k1 = reinterpret_cast<uintx4 *>(pool.keys + target * pool.block_bytes), *const v1 = reinterpret_cast<uintx4 *>(pool.values + target * pool.block_bytes);
  long long i = from + threadIdx.x;
  for (; i + 3 * 256 < upto; i += 4 * 256) {
    uintx4 k[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k[j] = k0[i + 256 * j];
      v[j] = v0[i + 256 * j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k1[i + 256 * j] = k[j];
      v1[i + 256 * j] = v[j];
    }
  }
  for (; i < upto; i += 256) {
    k1[i] = k0[i];
    v1[i] = v0[i];
  }
  if (part == 0)
    for (int i = threadIdx.x; i < pool.scale_floats; i += 256)
      pool.scales[(long long)target * pool.scale_floats + i] = pool.scales[(long long)source * pool.scale_floats + i];
}

__global__ __launch_bounds__(256) void fork_copy_kernel(const PageTable t, const PagePool pool, const Fork *forks) {
  const Fork f = forks[blockIdx.x];
  if (f.child < 0) return;
  if (f.source >= 0) copy_page(pool, f.source, f.target, blockIdx.y, gridDim.y);
  if (blockIdx.y != 0) return;
  for (int s = threadIdx.x; s < t.slots; s += 256) {
    int page = -1;
    if (s < f.shared) {
      page = t.table[(long long)f.parent * t.slots + s];
      if (page >= 0 && page < t.pages) atomicAdd(&t.refs[page], 1);
      else page = -1;
    } else if (s == f.shared && f.source >= 0) {
      page = f.target;
    }
    int32_t *const at = t.table + (long long)f.child * t.slots + s;
    const int before = *at;
    if (before >= 0 && before < t.pages) atomicSub(&t.refs[before], 1);  // (while the plan was made its pages were in use)
    *at = page;
  }
}

constexpr int kPer = 4, kChunk = kPer * kPlanThreads;  // pages that a thread and a workgroup of the compaction look at

__global__ __launch_bounds__(kPlanThreads) void compact_count_kernel(const int32_t *refs, int pages, int32_t *counts) {
  __shared__ uint32_t share[kPlanWaves];
  uint32_t used = 0, all;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int p = blockIdx.x * kChunk + i * kPlanThreads + threadIdx.x;
    used += p < pages && refs[p] > 0;
  }
  block_exclusive_sum(used, share, &all);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)all;
}

// With U pages in use, those at U and behind move, in their order, to the free ones below U, in theirs.  rank_of[p] = its place among the
// movers (-1: it stays), hole[i] / mover[i] = the i-th of either, counts[chunks] = how many.  counted: counts[] are there.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const int32_t *refs, int pages, int32_t *counts, int chunks, bool counted,
                                                                    int32_t *rank_of, int32_t *hole, int32_t *mover) {
  __shared__ uint32_t share[kPlanWaves];
  const int tid = threadIdx.x, p0 = blockIdx.x * kChunk + tid * kPer;
  bool used[kPer];
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    used[i] = p0 + i < pages && refs[p0 + i] > 0;
    count += used[i];
  }
  uint32_t in_chunk;
  uint32_t ahead = block_exclusive_sum(count, share, &in_chunk);  // pages in use before the thread's, for now of the chunk
  uint32_t in_use = 0, before = 0, below = 0;  // pages in use: all of them, in the chunks before this one, below U
  int boundary;
  if (chunks == 1) {
    in_use = in_chunk;
    boundary = (int)in_use;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) n += used[i] && p0 + i < boundary;
    block_exclusive_sum(n, share, &below);
  } else if (counted) {
    for (int i0 = 0; i0 < chunks; i0 += kPlanThreads) {
      const int i = i0 + tid;
      const uint32_t v = i < chunks ? (uint32_t)counts[i] : 0u;
      uint32_t all, part;
      block_exclusive_sum(v, share, &all);
      block_exclusive_sum(i < (int)blockIdx.x ? v : 0u, share, &part);
      in_use += all;
      before += part;
    }
    boundary = (int)in_use;
    const int its = boundary / kChunk;  // the chunk that U lies in: those before it, and its own pages up to U
    for (int i0 = 0; i0 < chunks; i0 += kPlanThreads) {
      const int i = i0 + tid;
      uint32_t all;
      block_exclusive_sum(i < its && i < chunks ? (uint32_t)counts[i] : 0u, share, &all);
      below += all;
    }
    uint32_t n = 0, all;
    for (int p = its * kChunk + tid; p < min(boundary, pages); p += kPlanThreads) n += refs[p] > 0;
    block_exclusive_sum(n, share, &all);
    below += all;
  } else {
    uint32_t n = 0, m = 0;
    for (int p = tid; p < pages; p += kPlanThreads) {
      const bool is = refs[p] > 0;
      n += is;
      m += is && p < (int)blockIdx.x * kChunk;
    }
    block_exclusive_sum(n, share, &in_use);
    block_exclusive_sum(m, share, &before);
    boundary = (int)in_use;
    n = 0;
    for (int p = tid; p < boundary; p += kPlanThreads) n += refs[p] > 0;
    block_exclusive_sum(n, share, &below);
  }
  if (blockIdx.x == 0 && tid == 0) counts[chunks] = boundary - (int)below;
  ahead += before;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int p = p0 + i;
    if (p >= pages) break;
    int rank = -1;
    if (used[i] && p >= boundary) {
      rank = (int)(ahead - below);
      mover[rank] = p;
    } else if (!used[i] && p < boundary) {
      hole[p - (int)ahead] = p;
    }
    rank_of[p] = rank;
    ahead += used[i];
  }
}

__global__ __launch_bounds__(256) void compact_move_kernel(const PageTable t, const PagePool pool, const int32_t *moves, const int32_t *rank_of, const int32_t *hole,
                                                           const int32_t *mover, int parts) {
  const int count = *moves;
  for (long long i = blockIdx.x; i < (long long)count * parts; i += gridDim.x) {
    const int move = (int)(i / parts), part = (int)(i % parts), source = mover[move], target = hole[move];
    copy_page(pool, source, target, part, parts);
    if (part == 0 && threadIdx.x == 0) {
      t.refs[target] = t.refs[source];
      t.refs[source] = 0;
    }
  }
  const long long entries = (long long)t.rows * t.slots;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long long)gridDim.x * 256) {
    const int page = t.table[i];
    if (page < 0 || page >= t.pages) continue;
    const int rank = rank_of[page];
    if (rank >= 0) t.table[i] = hole[rank];
  }
}

}  // namespace

// a rank a row, and the pages taken
static size_t reserve_ints(int pages, int rows, int slots) { return (size_t)rows + (size_t)min((long long)pages, (long long)rows * slots); }
size_t reserve_workspace_ints(int pages, int rows, int slots) {
  const size_t n = reserve_ints(pages, rows, slots);
  return n <= kPlanLds ? 0 : n;
}
// a mark a row, the pages taken, what becomes of each child
size_t fork_workspace_ints(int rows, int count) { return (size_t)rows + (size_t)count * (1 + sizeof(Fork) / 4); }
// the chunks' counts and the moves', and three lists
size_t compact_workspace_ints(int pages) { return ((size_t)pages + kChunk - 1) / kChunk + 1 + 3 * (size_t)pages; }

hipError_t launch_reserve_pages(const PageTable &t, const int32_t *starts, const int32_t *offsets, int page_size, int32_t *workspace, hipStream_t stream) {
  const size_t ints = reserve_ints(t.pages, t.rows, t.slots);
  const bool inside = ints <= kPlanLds;
  hipLaunchKernelGGL(reserve_pages_kernel, dim3(1), dim3(kPlanThreads), inside ? ints * 4 : 0, stream, t, starts, offsets, page_size, inside ? nullptr : workspace);
  return hipGetLastError();
}

hipError_t launch_release_pages(const PageTable &t, int32_t *lengths, const int32_t *named, int count, hipStream_t stream) {
  hipLaunchKernelGGL(release_pages_kernel, dim3(count), dim3(256), 0, stream, t, lengths, named);
  return hipGetLastError();
}

hipError_t launch_fork_pages(const PageTable &t, const PagePool &pool, int32_t *lengths, const int32_t *parents, const int32_t *children, int count, int page_size,
                             int32_t *workspace, hipStream_t stream) {
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, t, lengths, parents, children, count, page_size, workspace);
  const int parts = (int)max(1ll, min(pool.block_bytes / 16384, 16ll));
  hipLaunchKernelGGL(fork_copy_kernel, dim3(count, parts), dim3(256), 0, stream, t, pool, reinterpret_cast<const Fork *>(workspace + t.rows + count));
  return hipGetLastError();
}

hipError_t launch_compact_pages(const PageTable &t, const PagePool &pool, int32_t *workspace, hipStream_t stream) {
  const int chunks = (t.pages + kChunk - 1) / kChunk;
  int32_t *const counts = workspace, *const rank_of = counts + chunks + 1, *const hole = rank_of + t.pages, *const mover = hole + t.pages;
  // (a few chunks are counted by the plan itself, in each of its workgroups: a launch less)
  const bool counted = chunks > 4;
  if (counted) hipLaunchKernelGGL(compact_count_kernel, dim3(chunks), dim3(kPlanThreads), 0, stream, t.refs, t.pages, counts);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(chunks), dim3(kPlanThreads), 0, stream, t.refs, t.pages, counts, chunks, counted, rank_of, hole, mover);
  const int parts = (int)max(1ll, min(pool.block_bytes / 16384, 16ll));
  const unsigned grid = (unsigned)max(1ll, min(4096ll, (long long)t.pages * parts));
  hipLaunchKernelGGL(compact_move_kernel, dim3(grid), dim3(256), 0, stream, t, pool, counts + chunks, rank_of, hole, mover, parts);
  return hipGetLastError();
}

}  // namespace sspmm
