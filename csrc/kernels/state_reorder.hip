// Recurrent states that follow their beams: slot s of every tensor takes what slot parents[s] held, in place, over all tensors in
// one launch.
//
// In place without a copy on the side: a thread owns the same bytes of every slot of a group.  It loads what the group's slots
// take, all loads before its first store, so it has read a slot before anyone overwrites it (only it touches these bytes).  A slot
// that keeps its own state is neither read nor written; a source that several slots take is read from memory once, the further
// loads hit the cache.  Bound by memory: each source read once, each changed slot written once.
#include "api_beams.h"

namespace dsse {

constexpr int kReorderThreads = 256;

// U: unit of a thread (16, 4 or 2 bytes); N: slots of a group that the registers hold
template <typename U, int N>
__global__ void __launch_bounds__(kReorderThreads) state_reorder_kernel(StateReorderParams p) {
  int i = 0;
  while (i + 1 < p.ntensors && (int)blockIdx.x >= p.t[i + 1].first) ++i;
  const auto t = p.t[i];
  const int64_t at = ((int64_t)(blockIdx.x - t.first) * kReorderThreads + threadIdx.x) * sizeof(U);
  if (at >= t.bytes) return;
  const int first = blockIdx.y * p.width;
  U u[N];
  int from[N];
#pragma unroll
  for (int w = 0; w < N; ++w) {
    from[w] = -1;
    if (w < p.width) {
      const int q = p.parents[first + w];
      if (q != first + w && q >= first && q < first + p.width) from[w] = q;
    }
  }
#pragma unroll
  for (int w = 0; w < N; ++w)
    if (from[w] >= 0) u[w] = *reinterpret_cast<const U*>(t.base + from[w] * t.stride + at);
#pragma unroll
  for (int w = 0; w < N; ++w)
    if (from[w] >= 0) *reinterpret_cast<U*>(t.base + (first + w) * t.stride + at) = u[w];
}

template <typename U>
void launch_reorder(const StateReorderParams& p, int blocks, hipStream_t st) {
  const dim3 grid(blocks, p.slots / p.width);
  if (p.width <= 4) hipLaunchKernelGGL((state_reorder_kernel<U, 4>), grid, dim3(kReorderThreads), 0, st, p);
  else if (p.width <= 8) hipLaunchKernelGGL((state_reorder_kernel<U, 8>), grid, dim3(kReorderThreads), 0, st, p);
  else if (p.width <= 16) hipLaunchKernelGGL((state_reorder_kernel<U, 16>), grid, dim3(kReorderThreads), 0, st, p);
  else hipLaunchKernelGGL((state_reorder_kernel<U, 32>), grid, dim3(kReorderThreads), 0, st, p);
}

}  // namespace dsse

// The widest unit that every slot of every tensor starts and ends at: 16 bytes, or 4 or 2
extern "C" hipError_t dsse_state_reorder(const dsse::StateReorderParams* in, hipStream_t st) {
  using namespace dsse;
  if (in->width < 1 || in->width > kBeamWidth || in->slots % in->width || in->slots / in->width > 65535 || in->ntensors > kReorderLists)
    return hipErrorInvalidValue;
  if (in->slots == 0 || in->ntensors == 0) return hipSuccess;
  StateReorderParams p = *in;
  uintptr_t bits = 0;
  for (int i = 0; i < p.ntensors; ++i) bits |= reinterpret_cast<uintptr_t>(p.t[i].base) | (uintptr_t)p.t[i].stride | (uintptr_t)p.t[i].bytes;
  const int unit = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : (bits % 2 == 0 ? 2 : 0));
  if (unit == 0) return hipErrorInvalidValue;
  int64_t blocks = 0;
  for (int i = 0; i < p.ntensors; ++i) {
    p.t[i].first = (int)blocks;
    blocks += (p.t[i].bytes + unit * kReorderThreads - 1) / (unit * kReorderThreads);
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  }
  if (unit == 16) launch_reorder<u32x4>(p, (int)blocks, st);
  else if (unit == 4) launch_reorder<uint32_t>(p, (int)blocks, st);
  else launch_reorder<uint16_t>(p, (int)blocks, st);
  return hipGetLastError();
}
