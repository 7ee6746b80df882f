// Forks of paged sequences: slot s goes on with the pages that slot parents[s] holds.  Full pages are shared (refs counts a page's
// holders, 0 = free); the page that a slot's next token goes to becomes its own.  Three launches:
//
//   tables  every workgroup takes a strip of 16 columns of the tables, reads what the slots give up and take over, counts holders
//           down and up where the two differ (integer atomics: the order does not matter), and writes the strip after its last read.
//   pages   one workgroup: who needs a page of its own, the lowest free ones in slot order, counts, lengths, the list of copies.
//   copies  the listed pages of every pool and layer, 16 bytes a lane.
//
// Beams of a request have the same pages but for the last few, so the first launch is two reads of the tables and few atomics; the
// copies are what costs, two passes over each page.
#include "api_beams.h"

namespace dsse {

constexpr int kStrip = 16;          // columns of a workgroup of the first launch
constexpr int kForkThreads = 1024;
constexpr int kCopyThreads = 256;

DEV bool goes_on(int parent, int slots) { return (unsigned)parent < (unsigned)slots; }

// N: table entries of a thread
template <int N>
__global__ void __launch_bounds__(kForkThreads) fork_tables_kernel(PageForkParams p) {
  const int j = blockIdx.x * kStrip + threadIdx.x % kStrip;
  const int s0 = threadIdx.x / kStrip;
  constexpr int kStep = kForkThreads / kStrip;  // slots of a pass
  int next[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int s = s0 + n * kStep;
    next[n] = -1;
    if (s >= p.slots || j >= p.max_blocks) continue;
    const int q = p.parents[s];
    if (q == s) continue;
    const bool on = goes_on(q, p.slots);
    const int old = j < p.held[s] ? p.tables[(size_t)s * p.max_blocks + j] : -1;
    if (on && j < p.held[q]) next[n] = p.tables[(size_t)q * p.max_blocks + j];
    if (old != next[n]) {
      if ((unsigned)old < (unsigned)p.pages) atomicSub(&p.refs[old], 1);
      if ((unsigned)next[n] < (unsigned)p.pages) atomicAdd(&p.refs[next[n]], 1);
    }
  }
  __syncthreads();  // the strip is read: it may change
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (next[n] >= 0) p.tables[(size_t)(s0 + n * kStep) * p.max_blocks + j] = next[n];
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

__global__ void __launch_bounds__(kForkThreads) fork_pages_kernel(PageForkParams p) {
  __shared__ int follow[kForkSlots], last[kForkSlots], fresh[kForkSlots], scan[kForkThreads / 64];
  constexpr int kPer = kForkSlots / kForkThreads;  // neighbouring slots of a thread
  const int s0 = threadIdx.x * kPer;
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
  int page[kPer], need = 0, mask = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    page[i] = -1;
    const int s = s0 + i, q = parent[i], j = len[i] / kBS;
    if (q < 0 || len[i] < 0 || j >= p.max_blocks) continue;
    if (j < held[i]) {
      page[i] = p.tables[(size_t)s * p.max_blocks + j];
      if ((unsigned)page[i] >= (unsigned)p.pages) { page[i] = -1; continue; }
      if (last[q] == s && p.refs[page[i]] == follow[q]) continue;  // its followers alone hold it: the last one keeps it
    }
    mask |= 1 << i;
    ++need;
  }
  int wanted;
  int rank = block_scan(need, scan, wanted);
  // the lowest free pages, as many as are wanted
  int found = 0;
  for (int base = 0; base < p.pages && found < wanted; base += kForkThreads * 4) {
    int at[4], n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = base + threadIdx.x * 4 + k;
      at[k] = i < p.pages && p.refs[i] == 0 ? 1 : 0;
      n += at[k];
    }
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
  }
  if (threadIdx.x == 0) p.starved[0] = wanted - had;
}

// grid (pieces of a page, slots): the workgroups of a slot walk the layers of all pools
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(PageCopyParams p) {
  const int src = p.copies[2 * blockIdx.y], dst = p.copies[2 * blockIdx.y + 1];
  if ((unsigned)src >= (unsigned)p.pages || (unsigned)dst >= (unsigned)p.pages) return;
  for (int i = 0; i < p.npools; ++i) {
    const auto o = p.pool[i];
    const int units = o.bytes / 16;
    for (int64_t u = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; u < (int64_t)units * o.layers; u += (int64_t)gridDim.x * kCopyThreads) {
      const int l = (int)(u / units), e = (int)(u % units);
      char* base = o.base + l * o.layer + (int64_t)e * 16;
      *reinterpret_cast<u32x4*>(base + (int64_t)dst * o.bytes) = *reinterpret_cast<const u32x4*>(base + (int64_t)src * o.bytes);
    }
  }
}

}  // namespace dsse

extern "C" hipError_t dsse_page_fork(const dsse::PageForkParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->slots < 1 || p->slots > kForkSlots || p->max_blocks < 1 || p->pages < 1) return hipErrorInvalidValue;
  const dim3 grid((p->max_blocks + kStrip - 1) / kStrip), block(kForkThreads);
  constexpr int kStep = kForkThreads / kStrip;
  const int per = (p->slots + kStep - 1) / kStep;
  if (per <= 1) hipLaunchKernelGGL((fork_tables_kernel<1>), grid, block, 0, st, *p);
  else if (per <= 8) hipLaunchKernelGGL((fork_tables_kernel<8>), grid, block, 0, st, *p);
  else hipLaunchKernelGGL((fork_tables_kernel<kForkSlots / kStep>), grid, block, 0, st, *p);
  hipLaunchKernelGGL(fork_pages_kernel, dim3(1), block, 0, st, *p);
  return hipGetLastError();
}

extern "C" hipError_t dsse_page_copy(const dsse::PageCopyParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->slots < 1 || p->slots > 65535 || p->npools < 1 || p->npools > kCopyPools) return hipErrorInvalidValue;
  hipLaunchKernelGGL(page_copy_kernel, dim3(64, p->slots), dim3(kCopyThreads), 0, st, *p);
  return hipGetLastError();
}
