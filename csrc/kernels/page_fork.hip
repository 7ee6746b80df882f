// Forks of paged sequences: slot s goes on with the pages that slot parents[s] holds.  Full pages are shared (refs counts a page's
// holders, 0 = free); the page that a slot's next token goes to becomes its own.  Three launches, or two where the tables are
// small enough for the workgroup of the second:
//
//   tables  every workgroup takes a strip of 4 columns of the tables, reads what the slots give up and take over, counts holders
//           down and up where the two differ (integer atomics: the order does not matter), and writes the strip after its last read.
//   pages   one workgroup: who needs a page of its own, the lowest free ones in slot order, counts, lengths, the list of copies.
//   copies  the listed pages of every pool and layer, 64 bytes a lane in flight; workgroups walk the list, whose length only the
//           device knows.
//
// Beams of a request have the same pages but for the last few, so the first launch is two reads of the tables and few atomics; the
// copies are what costs, two passes over each page: 64x8 slots behind 4000 tokens 5.0 + 7.9 us for tables and pages, 16.4 to 17.7 for
// 89 MB of copies (5.0 TB/s); 16x4 slots over 32 layers of keys and values 9.6 in one launch and 49 for 252 MB (5.1 TB/s).  The free pages
// are searched from page 0, 4096 a step: where 90000 of 100000 pages are held from the low end, the second launch takes 33 us.
#include "api_beams.h"

namespace dsse {

constexpr int kStrip = 4;           // columns of a workgroup of the first launch
constexpr int kForkThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnits = 4;       // 16-byte units of a lane

constexpr int kSmall = 2;           // table entries of a thread of the second launch where it does without the first

DEV bool goes_on(int parent, int slots) { return (unsigned)parent < (unsigned)slots; }
// Counts are read past L1, which does not see the atomics of the same launch
DEV int holders(const PageForkParams& p, int page) {
  return __hip_atomic_load(&p.refs[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A workgroup's part of the tables, whole columns of it, N entries of a thread; place(n, s, j): whether entry n is one, and which.  A
// column's entries come from the same column, so no other workgroup reads what this one writes.
template <int N, typename P>
DEV void move_entries(const PageForkParams& p, P place) {
  int next[N], old[N];
  bool given[N];  // the parent holds the entry, whatever its number: a slot never keeps a page that it has given up
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int s, j;
    next[n] = old[n] = -1;
    given[n] = false;
    if (!place(n, s, j)) continue;
    const int q = p.parents[s];
    if (q == s) continue;
    if (j < p.held[s]) old[n] = p.tables[(size_t)s * p.max_blocks + j];
    if (goes_on(q, p.slots) && j < p.held[q]) next[n] = p.tables[(size_t)q * p.max_blocks + j], given[n] = true;
  }
  __syncthreads();  // the part is read: it may change
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int s, j;
    if (!place(n, s, j) || (old[n] == next[n] && old[n] >= 0)) continue;  // most of the pages that beams of a request hold
    if ((unsigned)old[n] < (unsigned)p.pages) atomicSub(&p.refs[old[n]], 1);
    if ((unsigned)next[n] < (unsigned)p.pages) atomicAdd(&p.refs[next[n]], 1);
    if (given[n]) p.tables[(size_t)s * p.max_blocks + j] = next[n];
  }
}

template <int N>
__global__ void __launch_bounds__(kForkThreads) fork_tables_kernel(PageForkParams p) {
  move_entries<N>(p, [&](int n, int& s, int& j) {
    s = threadIdx.x / kStrip + n * (kForkThreads / kStrip);
    j = blockIdx.x * kStrip + threadIdx.x % kStrip;
    return s < p.slots && j < p.max_blocks;
  });
}

// exclusive prefix sum over the workgroup; total: the sum
DEV int block_scan(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kForkThreads / 64; ++w) {
    if (w < wave) before += sh[w];
    total += sh[w];
  }
  return before + x - v;
}

template <bool TABLES>
__global__ void __launch_bounds__(kForkThreads) fork_pages_kernel(PageForkParams p) {
  __shared__ int follow[kForkSlots], last[kForkSlots], fresh[kForkSlots], goes_to[kForkSlots], scan[kForkThreads / 64];
  constexpr int kPer = kForkSlots / kForkThreads;  // neighbouring slots of a thread
  const int s0 = threadIdx.x * kPer;
  if constexpr (TABLES) {
    move_entries<kSmall>(p, [&](int n, int& s, int& j) {
      const int e = n * kForkThreads + threadIdx.x;
      s = e / p.max_blocks, j = e % p.max_blocks;
      return s < p.slots;
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's counts have reached L2, where holders() reads
    __syncthreads();
  }
  // counts of four neighbouring pages, on their way while the slots are looked at
  int count[4];
  auto look = [&](int base) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = base + threadIdx.x * 4 + k;
      count[k] = i < p.pages ? holders(p, i) : 1;
    }
  };
  look(0);
  for (int i = threadIdx.x; i < kForkSlots; i += kForkThreads) follow[i] = 0, last[i] = -1;
  __syncthreads();
  int parent[kPer], len[kPer], held[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = s0 + i, q = s < p.slots ? p.parents[s] : -1;
    parent[i] = goes_on(q, p.slots) ? q : -1;
    len[i] = held[i] = 0;
    if (parent[i] >= 0) {
      len[i] = p.lens[q], held[i] = min(max(p.held[q], 0), p.max_blocks);
      atomicAdd(&follow[q], 1);
      atomicMax(&last[q], s);
    }
  }
  __syncthreads();  // lengths and page counts are read: they may change
  int page[kPer], shared_by[kPer], mask = 0, ask = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    page[i] = shared_by[i] = goes_to[s0 + i] = -1;
    const int s = s0 + i, q = parent[i], j = len[i] / kBS;
    if (q < 0 || len[i] < 0 || j >= p.max_blocks) continue;
    if (j < held[i]) {
      page[i] = p.tables[(size_t)s * p.max_blocks + j];
      if ((unsigned)page[i] >= (unsigned)p.pages) { page[i] = -1; continue; }
      goes_to[s] = page[i];
      const int held_by = holders(p, page[i]);
      if (held_by == follow[q]) {  // its followers alone hold it: the last one keeps it
        if (last[q] == s) continue;
      } else {
        shared_by[i] = held_by, ask = 1;
      }
    }
    mask |= 1 << i;
  }
  int wanted, rank = block_scan(__popc(mask) | ask << 16, scan, wanted);  // of up to 2048 slots; above them, whether any asks
  // Slots of several parents go on in one page where an earlier call found no free one.  That is rare, so all slots are looked through
  // then: if they alone hold it, the last of them keeps it.
  if (wanted >> 16) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (shared_by[i] < 0) continue;
      int n = 0, end = -1;
      for (int t = 0; t < p.slots; ++t)
        if (goes_to[t] == page[i]) ++n, end = t;
      if (n == shared_by[i] && end == s0 + i) mask &= ~(1 << i);
    }
    rank = block_scan(__popc(mask), scan, wanted);
  }
  // the lowest free pages, as many as are wanted
  int found = 0;
  for (int base = 0; base < p.pages && found < wanted; base += kForkThreads * 4) {
    int at[4], n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      at[k] = count[k] == 0 ? 1 : 0;
      n += at[k];
    }
    look(base + kForkThreads * 4);
    int all, to = block_scan(n, scan, all) + found;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at[k]) {
        if (to < wanted) fresh[to] = base + threadIdx.x * 4 + k;
        ++to;
      }
    found += all;
  }
  __syncthreads();  // free pages are chosen: the counts may change
  const int had = found < wanted ? found : wanted;
  int copied = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = s0 + i;
    if (s >= p.slots) continue;
    int src = -1, dst = -1;
    if (mask >> i & 1) {
      if (rank < had) {
        const int j = len[i] / kBS, to = fresh[rank];
        p.tables[(size_t)s * p.max_blocks + j] = to;
        p.refs[to] = 1;
        if (page[i] >= 0) {
          atomicSub(&p.refs[page[i]], 1);
          if (len[i] % kBS) src = page[i], dst = to;
        }
        if (held[i] <= j) held[i] = j + 1;
      }
      ++rank;
    }
    p.held[s] = held[i];
    p.lens[s] = len[i];
    p.copies[2 * s] = src;
    p.copies[2 * s + 1] = dst;
    if (src >= 0) copied |= 1 << i;
  }
  int copies, at = block_scan(__popc(copied), scan, copies);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (copied >> i & 1) p.list[1 + at++] = s0 + i;
  if (threadIdx.x == 0) {
    p.starved[0] = wanted - had;
    p.list[0] = copies;
  }
}

// Work item: 16 KB of a page of a pool's layer, for one of the listed slots; up to 2^31 - 1 of them, and a workgroup's step further
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(PageCopyParams p) {
  const unsigned blocks = p.blocks, total = p.list[0] * blocks;
  for (unsigned w = blockIdx.x; w < total; w += gridDim.x) {
    const int slot = p.list[1 + w / blocks], b = w % blocks;
    const int src = p.copies[2 * slot], dst = p.copies[2 * slot + 1];
    int i = 0;
    while (i + 1 < p.npools && b >= p.pool[i + 1].first) ++i;
    const auto o = p.pool[i];
    const int layer = (b - o.first) / o.per, e0 = (b - o.first) % o.per * kCopyThreads * kCopyUnits * 16 + threadIdx.x * 16;
    const char* from = o.base + layer * o.layer + (int64_t)src * o.bytes;
    char* to = o.base + layer * o.layer + (int64_t)dst * o.bytes;
    u32x4 v[kCopyUnits];
#pragma unroll
    for (int u = 0; u < kCopyUnits; ++u) v[u] = ld_global<u32x4>(from + min(e0 + u * kCopyThreads * 16, o.bytes - 16));
#pragma unroll
    for (int u = 0; u < kCopyUnits; ++u)
      if (e0 + u * kCopyThreads * 16 < o.bytes) *reinterpret_cast<u32x4*>(to + e0 + u * kCopyThreads * 16) = v[u];
  }
}

}  // namespace dsse

extern "C" hipError_t dsse_page_fork(const dsse::PageForkParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->slots < 1 || p->slots > kForkSlots || p->max_blocks < 1 || p->pages < 1) return hipErrorInvalidValue;
  const dim3 block(kForkThreads);
  // One launch of both against two, us without the gap between: 104 entries 6.3 / 8.0, 1536 9.8 / 10.8, 3264 and 7680 11.5 / 8.5 and 19.8 / 17
  if ((int64_t)p->slots * p->max_blocks <= kSmall * kForkThreads) {
    hipLaunchKernelGGL(fork_pages_kernel<true>, dim3(1), block, 0, st, *p);
    return hipGetLastError();
  }
  const dim3 grid((p->max_blocks + kStrip - 1) / kStrip);
  constexpr int kStep = kForkThreads / kStrip;
  if (p->slots <= kStep) hipLaunchKernelGGL(fork_tables_kernel<1>, grid, block, 0, st, *p);
  else hipLaunchKernelGGL(fork_tables_kernel<kForkSlots / kStep>, grid, block, 0, st, *p);
  hipLaunchKernelGGL(fork_pages_kernel<false>, dim3(1), block, 0, st, *p);
  return hipGetLastError();
}

extern "C" hipError_t dsse_page_copy(const dsse::PageCopyParams* in, hipStream_t st) {
  using namespace dsse;
  if (in->slots < 1 || in->slots > kForkSlots || in->npools < 1 || in->npools > kCopyPools) return hipErrorInvalidValue;
  PageCopyParams p = *in;
  static_assert(kCopyThreads * kCopyUnits * 16 == kCopyPiece, "a work item is a piece");
  int64_t blocks = 0;
  for (int i = 0; i < p.npools; ++i) {
    p.pool[i].per = (p.pool[i].bytes + kCopyPiece - 1) / kCopyPiece;
    p.pool[i].first = (int)blocks;
    blocks += (int64_t)p.pool[i].per * p.pool[i].layers;
    if (blocks * p.slots > kCopyPieces) return hipErrorInvalidValue;
  }
  p.blocks = (int)blocks;
  const int64_t most = blocks * p.slots;  // all slots copy
  hipLaunchKernelGGL(page_copy_kernel, dim3((unsigned)(most < 2048 ? most : 2048)), dim3(kCopyThreads), 0, st, p);
  return hipGetLastError();
}
