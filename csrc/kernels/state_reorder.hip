// Recurrent states that follow their beams: slot s of every tensor takes what slot parents[s] held, in place, over all tensors in
// one launch.
//
// In place without a copy on the side: a thread owns the same bytes of every slot of a group.  It loads what the group's slots
// take, all loads before its first store, so it has read a slot before anyone overwrites it (only it touches these bytes).  A slot
// that keeps its own state is neither read nor written; a source that several slots take is read from memory once, the further
// loads hit the cache.  Bound by memory: each source read once, each changed slot written once (64 slots of 6 x 1 MB 100 us, 5.3 TB/s).
// 16 bytes a thread whatever the slots' alignment: 128 slots with tails of 9612 bytes beside 1 MB 298 us by words, 186 so.
#include "api_beams.h"

namespace dsse {

constexpr int kReorderThreads = 256;
// Global accesses may begin anywhere; a slot's part begins at two bytes
typedef u32x4 unit16 __attribute__((aligned(2)));
typedef uint32_t word __attribute__((aligned(2)));
DEV void take(u32x4& v, const char* p) { v = *reinterpret_cast<const unit16*>(p); }
DEV void take(uint32_t& v, const char* p) { v = *reinterpret_cast<const word*>(p); }
DEV void take(uint16_t& v, const char* p) { v = *reinterpret_cast<const uint16_t*>(p); }
DEV void give(char* p, const u32x4& v) { *reinterpret_cast<unit16*>(p) = v; }
DEV void give(char* p, uint32_t v) { *reinterpret_cast<word*>(p) = v; }
DEV void give(char* p, uint16_t v) { *reinterpret_cast<uint16_t*>(p) = v; }

// N: slots of a group that the registers hold
template <int N>
__global__ void __launch_bounds__(kReorderThreads) state_reorder_kernel(StateReorderParams p) {
  int i = 0;
  while (i + 1 < p.ntensors && (int)blockIdx.x >= p.t[i + 1].first) ++i;
  const auto t = p.t[i];
  const int units = t.bytes / 16, words = t.bytes % 16 / 4, item = (int)(blockIdx.x - t.first) * kReorderThreads + (int)threadIdx.x;
  const int first = blockIdx.y * p.width;
  int from[N];
#pragma unroll
  for (int w = 0; w < N; ++w) {
    from[w] = -1;
    if (w < p.width) {
      const int q = p.parents[first + w];
      if (q != first + w && q >= first && q < first + p.width) from[w] = q;
    }
  }
  auto move = [&](auto unit, int64_t at) {
    using U = decltype(unit);
    U u[N];
#pragma unroll
    for (int w = 0; w < N; ++w)
      if (from[w] >= 0) take(u[w], t.base + from[w] * t.stride + at);
#pragma unroll
    for (int w = 0; w < N; ++w)
      if (from[w] >= 0) give(t.base + (first + w) * t.stride + at, u[w]);
  };
  // whole units, then the last few bytes of a slot: a word, or half a one, per thread
  if (item < units) move(u32x4{}, (int64_t)item * 16);
  else if (item < units + words) move(uint32_t{}, (int64_t)units * 16 + 4 * (item - units));
  else if (item == units + words && t.bytes % 4) move(uint16_t{}, t.bytes - 2);
}

}  // namespace dsse

extern "C" hipError_t dsse_state_reorder(const dsse::StateReorderParams* in, hipStream_t st) {
  using namespace dsse;
  if (in->width < 1 || in->width > kBeamWidth || in->slots % in->width || in->slots / in->width > 65535 || in->ntensors > kReorderLists)
    return hipErrorInvalidValue;
  if (in->slots == 0 || in->ntensors == 0) return hipSuccess;
  StateReorderParams p = *in;
  int64_t bytes = 0;
  int blocks = 0;
  for (int i = 0; i < p.ntensors; ++i) {
    if ((reinterpret_cast<uintptr_t>(p.t[i].base) | (uintptr_t)p.t[i].stride | (uintptr_t)p.t[i].bytes) % 2) return hipErrorInvalidValue;
    bytes += p.t[i].bytes;
    if (bytes > kReorderBytes) return hipErrorInvalidValue;
    p.t[i].first = blocks;
    const int items = p.t[i].bytes / 16 + p.t[i].bytes % 16 / 4 + (p.t[i].bytes % 4 ? 1 : 0);
    blocks += (items + kReorderThreads - 1) / kReorderThreads;
  }
  const dim3 grid(blocks, p.slots / p.width), block(kReorderThreads);
  if (p.width <= 4) hipLaunchKernelGGL(state_reorder_kernel<4>, grid, block, 0, st, p);
  else if (p.width <= 8) hipLaunchKernelGGL(state_reorder_kernel<8>, grid, block, 0, st, p);
  else if (p.width <= 16) hipLaunchKernelGGL(state_reorder_kernel<16>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(state_reorder_kernel<32>, grid, block, 0, st, p);
  return hipGetLastError();
}
