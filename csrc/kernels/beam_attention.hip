// Attention of one new token per beam over the paged cache, for requests whose beams share pages (layouts of attention.hip).
//
// A group's leading `shared` pages are the same in all of its tables.  They are read once for the group: the columns of the score
// tile Sᵀ = K Qᵀ are (beam, q head) pairs, so a page's K and V feed every beam.  The pages behind them are read per slot.  Both walks
// are cut over their length, and a second launch joins the parts of a (slot, q head):
//
//   work items  x < groups * col_blocks * ns: the shared keys of a group, a block of columns, one of ns parts
//               else                        : a slot's own keys, one of no parts
//
// for every key/value head, heads first, parts last: workgroups go to the XCDs and CUs in turn, so the long walks have to be
// neighbours, and so have the first parts of short walks, whose last ones are empty (16x4 beams of 512 + 100 tokens with 32 parts in
// place of 4: 54 us with the part as the fastest index, 26 as it is; 2x16 of 31077 tokens 29.7, with the heads last 36).
//
// T = 1 (up to 16 columns): four waves take the pages in turn, straight to registers, and join their sums in LDS; a slot's own pages
// go to two waves in the same way, several slots to a workgroup.
// T = 2, 4, 8: a wave per column tile; the pages pass through LDS once for all waves, filled by LDS-DMA kRing - 1 pages ahead.  A
// page costs 16 KB from memory and T tiles' products, so what bounds it is memory.  A ring of 5 pages lets fewer workgroups on a CU
// than one of 3, which lets three of T = 2 or 4: 2x16 beams of 31077 tokens 36 -> 28.6 us.  T = 8 has one by its registers, 142 in each
// of eight waves, and two pages on their way: 19x16 beams of 32 heads over 4 and some 985 tokens 56 + 7 us (2.9 TB/s in the walks).
//
// Measured, walks + join: 8x8 beams of 32 heads over 8 and some 8300 tokens 60 + 5 us (5.6 TB/s in the walks), 2x16 of 16 over 4 and
// 31077 29 to 33 + 5, 16x4 of 612 17 + 4.5.  Each beam's pages read by themselves are 6 times the bytes in the first case, 15 in the second.
//
// Pages are read by non-temporal loads: a step reads every layer's pages and weights before it comes back to a layer's, so nothing of
// them is left in the caches.  Over 32 layers in turn 16x4 beams of 612 tokens take 19.0 to 19.7 us so, 20.5 to 21.0 by default loads,
// 8x8 of 8300 65 to 69 and 72 to 74, 2x16 of 31077 36 and 38; of one layer read again and again the first 20.8 and 19.3.
//
// Statistics and sums in fp32; scores in base 2 with the scale folded in; weights rounded to bf16 for the second product, as in
// paged_attention.
#include "api_beams.h"
#include "lds_dma.h"

#include <atomic>

namespace dsse {
namespace {

constexpr int kPg = 32;
constexpr int kDim = 128;
constexpr int kHalf = kPg * kDim * 2;  // bytes of a page's keys, or of its values
constexpr int kRing = 3;               // pages in LDS: three workgroups of a CU (T = 8: one) keep two pages each on their way
constexpr int kOwnWaves = 2;           // waves that split a slot's own pages
constexpr float kLow = -3.4028234663852886e38f;  // a finite start, below any score: fully masked columns stay finite and sum to zero

constexpr int waves_of(int T) { return T == 1 ? 4 : T; }

// Shared pages of a group that every live beam has whole; live: the first live slot, -1 if none
DEV int group_pages(const BeamAttnParams& p, int g, int& live) {
  const int w = threadIdx.x & 63;
  const int n = w < p.width ? p.ctx_len[g * p.width + w] : 0;
  const unsigned long long mask = __ballot(n > 0);
  int pages = n > 0 ? n / kPg : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < kBeamWidth; o <<= 1) pages = min(pages, __shfl_xor(pages, o));
  pages = __builtin_amdgcn_readfirstlane(pages);
  live = __builtin_amdgcn_readfirstlane(mask ? g * p.width + __ffsll(mask) - 1 : -1);
  return __builtin_amdgcn_readfirstlane(mask ? max(0, min(min(pages, p.shared[g]), p.max_blocks)) : 0);
}

// Entry `pg` of a table row: a wave-uniform scalar load, which does not wait for the vector loads in flight.  (The tables are
// read-only for the kernel.)
DEV int entry(const int* bt, int pg) {
  return ((const __attribute__((address_space(4))) int*)bt)[__builtin_amdgcn_readfirstlane(pg)];
}
// An entry that is no page reads page 0, not past the cache
DEV int page_of(const BeamAttnParams& p, int entry) { return (unsigned)entry < (unsigned)p.num_blocks ? entry : 0; }

struct Column {  // 16 columns' running sums of a wave: lane (r, g) holds head dims 16 dt + 4 g + i of column r
  f32x4 o[8];
  float m, l;
  DEV void clear() {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = kLow;
    l = 0.f;
  }
  // The weights of a page's scores (keys 4g + i and 16 + 4g + i of column r), as the second product's operand
  DEV bf16x8 weigh(const f32x4& s0, const f32x4& s1, float scale, int left) {
    float s[8], top = -INFINITY;
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = (i < 4 ? s0[i] : s1[i - 4]) * scale;
    if (left < kPg) {  // keys of the page past the sequence
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = (i < 4 ? 4 * g + i : 12 + 4 * g + i) < left ? s[i] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i]);
    const float now = fmaxf(m, rows4_max(top));
    if (__any(now > m)) {  // after the first pages a maximum moves rarely
      const float by = __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= by;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= by;
    }
    bf16x8 w;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(s[i] - m);
      sum += e;
      w[i] = f2bf(e);
    }
    l += sum;
    return w;
  }
};

// What a page holds past the sequence is not read as a number: 0 * NaN would reach the sums
DEV void blank_values(bf16x8 (&vf)[8], int left) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = (j < 4 ? 4 * g + j : 12 + 4 * g + j) < left;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) vf[dt][j] = in ? vf[dt][j] : (bf16)0.f;
  }
}

// Keys of pages [pb, pe) up to `limit`, for 16 columns, pages in turn to NW waves
template <int NW>
DEV void walk(const BeamAttnParams& p, const int* bt, int h, int pb, int pe, int limit, int row, Column& c) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW;
  bf16x8 qf[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) qf[k] = row >= 0 ? ld_bf16x8(p.q + (size_t)row * kDim + 32 * k + 8 * g) : zero_bf16x8();
  c.clear();
  if (pb + kw >= pe) return;
  int id = entry(bt, pb + kw);
  for (int pg = pb + kw; pg < pe; pg += NW) {
    const size_t at = ((size_t)page_of(p, id) * p.hkv + h) * kPg * kDim;
    id = entry(bt, min(pg + NW, pe - 1));  // the next one is on its way while this page is computed
    const bf16 *kp = p.k_cache + at, *vp = p.v_cache + at;
    bf16x8 k0[4], k1[4], vf[8];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      k0[s] = ld_once<bf16x8>(kp + r * kDim + 32 * s + 8 * g);
      k1[s] = ld_once<bf16x8>(kp + (16 + r) * kDim + 32 * s + 8 * g);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) vf[dt] = ld_once<bf16x8>(vp + (16 * dt + r) * kPg + 8 * g);
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      s0 = mfma16x16x32(k0[s], qf[s], s0);
      s1 = mfma16x16x32(k1[s], qf[s], s1);
    }
    const int left = limit - pg * kPg;
    const bf16x8 w = c.weigh(s0, s1, p.scale_log2, left);
    if (left < kPg) blank_values(vf, left);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) c.o[dt] = mfma16x16x32(vf[dt], w, c.o[dt]);
  }
}

// The same for T column tiles, one per wave: whole pages [pb, pe) through LDS
template <int T>
DEV void walk_tiles(const BeamAttnParams& p, const int* bt, int h, int pb, int pe, int row, Column& c, char* smem) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // head dims of a k-step: 32 g + 8 s .. + 7 of both operands
  bf16x8 qf[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) qf[s] = row >= 0 ? ld_bf16x8(p.q + (size_t)row * kDim + 32 * g + 8 * s) : zero_bf16x8();
#pragma unroll
  for (int s = 0; s < 4; ++s) asm volatile("" ::"v"(qf[s]));  // their wait is here, not behind the DMAs of the loop
  c.clear();
  // A page is 16 instructions of 1 KiB, a wave's all keys or all values.  Keys: 4 rows of 16 pieces, piece ^ swz(row); values: 16
  // rows d of 4 pieces, piece ^ vswz(row): the swizzles sit on the source address and make the fragment reads free of conflicts.
  constexpr int IPW = 16 / T;
  auto vswz = [](int row) { return (4 - (row >> 2)) & 3; };
  const bool keys = wave * IPW < 8;
  uint32_t from[IPW];
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int n = (wave * IPW + i) & 7;
    from[i] = n * 1024 + (keys ? (lane >> 4) * 256 + (((lane & 15) ^ swz(4 * (n & 3) + (lane >> 4))) << 4)
                               : (lane >> 2) * 64 + (((lane & 3) ^ vswz(lane >> 2)) << 4));
  }
  const bf16* mine = (keys ? p.k_cache : p.v_cache) + (size_t)h * kPg * kDim;
  int id = entry(bt, pb), next = pb, slot_in = 0;
  auto issue = [&]() {  // a page past the last lands as zeros, without traffic, so that every step issues as many
    const __amdgpu_buffer_rsrc_t src = make_rsrc(mine + (size_t)page_of(p, id) * p.hkv * kPg * kDim, next < pe ? kHalf : 0);
    ++next;
    id = entry(bt, min(next, pe - 1));
    char* to = smem + slot_in * 2 * kHalf + wave * IPW * 1024;
    slot_in = slot_in + 1 == kRing ? 0 : slot_in + 1;
#pragma unroll
    for (int i = 0; i < IPW; ++i) lds_dma<kAuxNT>(src, to + i * 1024, from[i]);
  };
  int kofs[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) kofs[s] = r * 256 + (((4 * g + s) ^ swz(r)) << 4);
  const int vofs = kHalf + r * 64 + ((g ^ vswz(r)) << 4);
  for (int i = 0; i < kRing - 1; ++i) issue();
  int slot = 0;
  for (int pg = pb; pg < pe; ++pg) {
    // this page has landed in every wave's share, and every wave has read the page whose slot is filled next
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kRing - 2) * IPW) : "memory");
    issue();
    const char* at = smem + slot * 2 * kHalf;
    slot = slot + 1 == kRing ? 0 : slot + 1;
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
    bf16x8 k0[4], k1[4], vf[8];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      k0[s] = *reinterpret_cast<const bf16x8*>(at + kofs[s]);
      k1[s] = *reinterpret_cast<const bf16x8*>(at + 4096 + kofs[s]);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) vf[dt] = *reinterpret_cast<const bf16x8*>(at + dt * 1024 + vofs);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      s0 = mfma16x16x32(k0[s], qf[s], s0);
      s1 = mfma16x16x32(k1[s], qf[s], s1);
    }
    const bf16x8 w = c.weigh(s0, s1, p.scale_log2, kPg);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) c.o[dt] = mfma16x16x32(vf[dt], w, c.o[dt]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way into LDS when the workgroup ends
}

// A column tile's sums as part z of the columns' rows (slot * hq + head, -1: no column)
DEV void leave(const BeamAttnParams& p, const Column& c, int row, int z) {
  const int g = (threadIdx.x & 63) >> 4, np = p.ns + p.no;
  const float l = rows4_sum(c.l);
  if (row < 0) return;
  float* po = p.part_o + ((size_t)row * np + z) * kDim + 4 * g;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt) = c.o[dt];
  if (g == 0) p.part_ml[(size_t)row * np + z] = make_float2(c.m, l);
}

// The same for groups of NW waves that split the keys of one column tile: joined in LDS, wave kw of a group the head dims
// 128 kw / NW ..  Every wave of the workgroup comes here.
constexpr int join_bytes(int waves) { return waves * (32 * 64 + 32) * 4; }
template <int NW>
DEV void leave_joined(const BeamAttnParams& p, const Column& c, int row, int z, char* smem) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6, kw = wave % NW, np = p.ns + p.no;
  float* o = reinterpret_cast<float*>(smem + wave / NW * join_bytes(NW));  // [NW][32][64]
  float* ms = o + NW * 32 * 64;                // [NW][16]
  float* ls = ms + NW * 16;
  const float own = rows4_sum(c.l);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[(kw * 32 + dt * 4 + i) * 64 + lane] = c.o[dt][i];
  if (g == 0) ms[kw * 16 + r] = c.m, ls[kw * 16 + r] = own;
  __syncthreads();
  float top = ms[r];
#pragma unroll
  for (int v = 1; v < NW; ++v) top = fmaxf(top, ms[v * 16 + r]);
  float w[NW], sum = 0.f;
#pragma unroll
  for (int v = 0; v < NW; ++v) {
    w[v] = __builtin_amdgcn_exp2f(ms[v * 16 + r] - top);
    sum += ls[v * 16 + r] * w[v];
  }
  if (row < 0) return;
  float* po = p.part_o + ((size_t)row * np + z) * kDim + 4 * g;
#pragma unroll
  for (int t = 0; t < 8 / NW; ++t) {
    const int dt = kw * (8 / NW) + t;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] += o[(v * 32 + dt * 4 + i) * 64 + lane] * w[v];
    *reinterpret_cast<f32x4*>(po + 16 * dt) = a;
  }
  if (kw == 0 && g == 0) p.part_ml[(size_t)row * np + z] = make_float2(top, sum);
}

// Pages [first, second) of part z of n: at least `least` pages a part, the rest empty
DEV int2 part_of(int pages, int n, int z, int least) {
  const int per = max((pages + n - 1) / n, least), pb = min(pages, z * per);
  return make_int2(pb, min(pages, pb + per));
}

template <int T>
__global__ void __launch_bounds__(64 * waves_of(T), 2) beam_attention_kernel(BeamAttnParams p) {
  constexpr int NW = waves_of(T);
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15;
  const int h = blockIdx.x % p.hkv, x = blockIdx.x / p.hkv, np = p.ns + p.no;
  const int groups = p.slots / p.width, nshared = groups * p.col_blocks * p.ns;
  int live;
  Column c;
  if (x < nshared) {
    const int cb = x % p.col_blocks, gr = x / p.col_blocks % groups, z = x / (p.col_blocks * groups);
    const int2 part = part_of(group_pages(p, gr, live), p.ns, z, 4);
    const int at = (cb * T + (T == 1 ? 0 : threadIdx.x >> 6)) * 16 + r, w = at / p.group, s = gr * p.width + w;
    const int row = w < p.width && p.ctx_len[s] > 0 ? s * p.hq + h * p.group + at % p.group : -1;
    if (part.x >= part.y) {  // nothing to read: the part says so
      if (lane < 16 && row >= 0) p.part_ml[(size_t)row * np + z] = make_float2(kLow, 0.f);
      return;
    }
    const int* bt = p.block_tables + (size_t)live * p.max_blocks;
    if constexpr (T == 1) {
      walk<NW>(p, bt, h, part.x, part.y, part.y * kPg, row, c);
      leave_joined<NW>(p, c, row, z, smem);
    } else {
      walk_tiles<T>(p, bt, h, part.x, part.y, row, c, smem);
      leave(p, c, row, z);
    }
  } else {
    constexpr int kGroups = NW / kOwnWaves;
    const int item = (x - nshared) * kGroups + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kOwnWaves;
    const int s = item % p.slots, z = item / p.slots, n = z < p.no ? p.ctx_len[s] : 0;
    const int row = n > 0 && r < p.group ? s * p.hq + h * p.group + r : -1;
    const int skip = group_pages(p, s / p.width, live);
    const int2 part = part_of(n > 0 ? min((n + kPg - 1) / kPg, p.max_blocks) - skip : 0, p.no, z, 2 * kOwnWaves);
    if (!__syncthreads_or(part.x < part.y)) {
      if (lane < 16 && row >= 0) p.part_ml[(size_t)row * np + p.ns + z] = make_float2(kLow, 0.f);
      return;
    }
    walk<kOwnWaves>(p, p.block_tables + (size_t)s * p.max_blocks, h, skip + part.x, skip + part.y, n, row, c);
    leave_joined<kOwnWaves>(p, c, row, p.ns + z, smem);
  }
}

// One wave per (slot, q head): lane z holds part z's statistics; then the parts that have keys, two at a time (a half wave each, four
// head dims a lane), as many in flight as the loop is unrolled
__global__ void __launch_bounds__(256) beam_join_kernel(BeamAttnParams p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.slots * p.hq || p.ctx_len[row / p.hq] <= 0) return;
  const int np = p.ns + p.no;
  float2 ml = make_float2(kLow, 0.f);
  if (lane < np) ml = p.part_ml[(size_t)row * np + lane];
  const float top = wave_max(ml.x), w = __builtin_amdgcn_exp2f(ml.x - top);
  const float sum = wave_sum(ml.y * w);
  unsigned long long mask = __ballot(ml.x > kLow);  // a part without keys has left no sums
  const float* po = p.part_o + (size_t)row * np * kDim + 4 * (lane & 31);
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  while (mask) {
    f32x4 v[4];
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int z0 = mask ? __ffsll(mask) - 1 : 64;
      mask &= mask - 1;
      const int z1 = mask ? __ffsll(mask) - 1 : 64;
      mask &= mask - 1;
      const int z = lane < 32 ? z0 : z1;
      const float by = __shfl(w, z & 63);
      f[i] = z < 64 ? by : 0.f;
      v[i] = z < 64 ? *reinterpret_cast<const f32x4*>(po + (size_t)z * kDim) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) a += v[i] * f[i];
  }
  const float inv = 1.f / sum;
  bf16x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = f2bf((a[i] + __shfl_xor(a[i], 32)) * inv);
  if (lane < 32) *reinterpret_cast<bf16x4*>(p.out + (size_t)row * kDim + 4 * lane) = out;
}

// one wave per group: leading table columns, whole pages of every live beam, that are the same in all of them
__global__ void __launch_bounds__(64) beam_shared_kernel(const int* tables, const int* ctx_len, int* shared, int width, int max_blocks) {
  const int g = blockIdx.x, lane = threadIdx.x;
  int live = -1, pages = max_blocks;
  for (int w = 0; w < width; ++w) {
    const int n = ctx_len[g * width + w];
    if (n <= 0) continue;
    if (live < 0) live = g * width + w;
    pages = min(pages, n / kPg);
  }
  int found = live < 0 ? 0 : pages;
  for (int base = 0; base < found; base += 64) {
    const int j = base + lane;
    bool same = true;
    if (j < found) {
      const int a = tables[(size_t)live * max_blocks + j];
      for (int w = 0; w < width; ++w) {
        const int s = g * width + w;
        if (ctx_len[s] > 0) same = same && tables[(size_t)s * max_blocks + j] == a;
      }
    }
    const unsigned long long other = __ballot(!same);
    if (other) { found = base + __ffsll(other) - 1; break; }
  }
  if (lane == 0) shared[g] = found;
}

template <int T>
hipError_t launch_attention(dim3 grid, const BeamAttnParams& p, hipStream_t st) {
  constexpr int NW = waves_of(T), ring = T > 1 ? kRing * 2 * kHalf : 0, lds = ring > join_bytes(NW) ? ring : join_bytes(NW);
  if (lds > 64 * 1024) {  // once per device
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == hipSuccess && !(set.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(&beam_attention_kernel<T>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e == hipSuccess) set.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((beam_attention_kernel<T>), grid, dim3(64 * NW), lds, st, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace dsse

// Column tiles of a workgroup and cuts of the walks, from what the host knows: the lengths are on the device, so the tables' width
// stands for them.  Shared walks: a workgroup per CU where it holds four tiles or more (4x16 beams of 16 heads and 16077 tokens
// 28.9 us with 16 parts, 35 with 32), two where it holds fewer.  Own walks: four waves per CU, two a walk.  Tables of 1025 columns in
// place of the sequences' own cost 2 to 5 % of short walks (1x4 beams of 700 tokens 10.1 -> 10.4 us) and nothing of long ones.
extern "C" void dsse_beam_plan(dsse::BeamAttnParams* p) {
  using namespace dsse;
  const int cols = p->width * p->group, groups = p->slots / p->width;
  p->tiles = cols <= 16 ? 1 : (cols <= 32 ? 2 : (cols <= 64 ? 4 : 8));
  p->col_blocks = (cols + 16 * p->tiles - 1) / (16 * p->tiles);
  auto cut = [](int64_t want, int64_t items, int most) {
    const int64_t n = (want + items - 1) / items;
    return (int)(n < most ? n : most);
  };
  const int by4 = (p->max_blocks + 3) / 4;
  p->ns = cut(p->tiles >= 4 ? 256 : 512, (int64_t)groups * p->col_blocks * p->hkv, by4 < 48 ? by4 : 48);
  p->no = cut(512, (int64_t)p->slots * p->hkv, by4 < 16 ? by4 : 16);
}

extern "C" hipError_t dsse_beam_attention(const dsse::BeamAttnParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->slots < 1 || p->width < 1 || p->width > kBeamWidth || p->slots % p->width || p->group < 1 || p->group > 16 || p->ns < 1 || p->no < 1 ||
      p->ns + p->no > 64 || (int64_t)p->slots * p->hq > kBeamRows)
    return hipErrorInvalidValue;
  const int groups = p->slots / p->width;
  const int per = waves_of(p->tiles) / kOwnWaves;  // own walks of a workgroup
  const dim3 grid((groups * p->col_blocks * p->ns + (p->slots * p->no + per - 1) / per) * p->hkv);
  hipError_t e = hipErrorInvalidValue;
  if (p->tiles == 1) e = launch_attention<1>(grid, *p, st);
  else if (p->tiles == 2) e = launch_attention<2>(grid, *p, st);
  else if (p->tiles == 4) e = launch_attention<4>(grid, *p, st);
  else if (p->tiles == 8) e = launch_attention<8>(grid, *p, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(beam_join_kernel, dim3((p->slots * p->hq + 3) / 4), dim3(256), 0, st, *p);
  return hipGetLastError();
}

extern "C" hipError_t dsse_beam_shared(const int* tables, const int* ctx_len, int* shared, int groups, int width, int max_blocks,
                                       hipStream_t st) {
  if (groups < 1 || width < 1 || width > dsse::kBeamWidth) return hipErrorInvalidValue;
  hipLaunchKernelGGL(dsse::beam_shared_kernel, dim3(groups), dim3(64), 0, st, tables, ctx_len, shared, width, max_blocks);
  return hipGetLastError();
}
