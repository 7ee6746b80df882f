// Attention of one new token per beam over the paged cache, for requests whose beams share pages (layouts of attention.hip).
//
// A group's leading `shared` pages are the same in all of its tables.  They are read once for the group: the columns of the score
// tile Sᵀ = K Qᵀ are (beam, q head) pairs, so a page's K and V fragments feed every beam.  The pages behind them are read per
// slot.  Both walks are cut over their length, and a second launch joins the parts of a (slot, q head):
//
//   work items  x < col_blocks * ns: the shared keys of group z, part x % ns, columns of block x / ns
//               else               : a slot's own keys, part (x - col_blocks * ns) % no
//
// Statistics and sums in fp32; scores in base 2 with the scale folded in; bf16 products as in paged_attention.
#include "api_beams.h"

namespace dsse {
namespace {

constexpr int kPg = 32;
constexpr int kDim = 128;
constexpr int kBeamWaves = 4;
constexpr float kLow = -1e30f;  // a finite start: fully masked columns stay finite and sum to zero

// shared pages of a group that every live beam has whole; live: the first live slot, -1 if none
DEV int group_pages(const BeamAttnParams& p, int g, int& live) {
  int pages = min(p.shared[g], p.max_blocks);
  live = -1;
  for (int w = 0; w < p.width; ++w) {
    const int s = g * p.width + w, n = p.ctx_len[s];
    if (n <= 0) continue;
    if (live < 0) live = s;
    pages = min(pages, n / kPg);
  }
  return live < 0 ? 0 : max(pages, 0);
}

// Keys [kPg pb, min(kPg pe, limit)) of a table row for CT tiles of 16 columns, by the waves of a workgroup; leaves a wave's sums
template <int CT>
DEV void walk(const BeamAttnParams& p, const int* bt, int h, int pb, int pe, int limit, const bf16x8 (&qf)[CT][4], f32x4 (&o)[CT][8],
              float (&m)[CT], float (&l)[CT]) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, kw = threadIdx.x >> 6;
  for (int pg = pb + kw; pg < pe; pg += kBeamWaves) {
    int page = __builtin_amdgcn_readfirstlane(bt[pg]);
    page = (unsigned)page < (unsigned)p.num_blocks ? page : 0;  // an id that is no page reads page 0, not past the cache
    const bf16* kp = p.k_cache + ((size_t)page * p.hkv + h) * kPg * kDim;
    const bf16* vp = p.v_cache + ((size_t)page * p.hkv + h) * kDim * kPg;
    bf16x8 k0[4], k1[4], vf[8];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      k0[s] = ld_once<bf16x8>(kp + (size_t)r * kDim + 32 * s + 8 * g);
      k1[s] = ld_once<bf16x8>(kp + (size_t)(16 + r) * kDim + 32 * s + 8 * g);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) vf[dt] = ld_once<bf16x8>(vp + (size_t)(16 * dt + r) * kPg + 8 * g);
    const int kb = pg * kPg;
    const bool part = kb + kPg > limit;
    if (part) {  // what a page holds past the sequence is not read as a number: 0 * NaN would reach the sums
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = kb + (j < 4 ? 4 * g + j : 12 + 4 * g + j) < limit;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) vf[dt][j] = in ? vf[dt][j] : (bf16)0.f;
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        s0 = mfma16x16x32(k0[s], qf[ct][s], s0);
        s1 = mfma16x16x32(k1[s], qf[ct][s], s1);
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // keys kb + 4g + i and kb + 16 + 4g + i
        s0[i] = !part || kb + 4 * g + i < limit ? s0[i] * p.scale_log2 : -INFINITY;
        s1[i] = !part || kb + 16 + 4 * g + i < limit ? s1[i] * p.scale_log2 : -INFINITY;
        top = fmaxf(top, fmaxf(s0[i], s1[i]));
      }
      top = rows4_max(top);
      const float now = fmaxf(m[ct], top), alpha = exp2f(m[ct] - now);
      m[ct] = now;
      bf16x8 pf;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = exp2f(s0[i] - now), e1 = exp2f(s1[i] - now);
        sum += e0 + e1;
        pf[i] = f2bf(e0);  // bf16 weights, as the values they meet; the sum above keeps 32 bits
        pf[4 + i] = f2bf(e1);
      }
      l[ct] = l[ct] * alpha + sum;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[ct][dt] = mfma16x16x32(vf[dt], pf, o[ct][dt] * alpha);
    }
  }
}

struct MergeLds {
  float o[kBeamWaves][32][64];
  float m[kBeamWaves][16], l[kBeamWaves][16];
};

// Joins the waves' sums of one column tile and leaves them as part z of the columns' (slot, head).  row: column r's
// slot * hq + head, or -1.  Wave kw writes the head dims 32 kw .. 32 kw + 31.
DEV void leave(const BeamAttnParams& p, MergeLds& lds, const f32x4 (&o)[8], float m, float l, int row, int z) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, kw = threadIdx.x >> 6;
  l = rows4_sum(l);
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < 8; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) lds.o[kw][dt * 4 + i][lane] = o[dt][i];
  if (g == 0) lds.m[kw][r] = m, lds.l[kw][r] = l;
  __syncthreads();
  float top = lds.m[0][r];
#pragma unroll
  for (int v = 1; v < kBeamWaves; ++v) top = fmaxf(top, lds.m[v][r]);
  float w[kBeamWaves], sum = 0.f;
#pragma unroll
  for (int v = 0; v < kBeamWaves; ++v) {
    w[v] = exp2f(lds.m[v][r] - top);
    sum += lds.l[v][r] * w[v];
  }
  if (row < 0) return;
  const int np = p.ns + p.no;
  float* po = p.part_o + ((size_t)row * np + z) * kDim;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int dt = 2 * kw + t;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kBeamWaves; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] += lds.o[v][dt * 4 + i][lane] * w[v];
    *reinterpret_cast<f32x4*>(po + 16 * dt + 4 * g) = a;
  }
  if (kw == 0 && g == 0) p.part_ml[(size_t)row * np + z] = make_float2(top, sum);
}

template <int CT>
__global__ void __launch_bounds__(64 * kBeamWaves) beam_attention_kernel(BeamAttnParams p) {
  __shared__ MergeLds lds;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, np = p.ns + p.no;
  const int groups = p.slots / p.width, nshared = groups * p.col_blocks * p.ns;
  if ((int)blockIdx.x < nshared) {
    const int z = blockIdx.x % p.ns, cb = blockIdx.x / p.ns % p.col_blocks, gr = blockIdx.x / (p.ns * p.col_blocks);
    int live;
    const int pages = group_pages(p, gr, live);
    int row[CT];
    bf16x8 qf[CT][4];
    f32x4 o[CT][8];
    float m[CT], l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = (cb * CT + ct) * 16 + r, w = c / p.group, s = gr * p.width + w;
      const bool in = w < p.width && p.ctx_len[s] > 0;
      row[ct] = in ? s * p.hq + h * p.group + c % p.group : -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) qf[ct][k] = in ? ld_bf16x8(p.q + (size_t)row[ct] * kDim + 32 * k + 8 * g) : zero_bf16x8();
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[ct] = kLow;
      l[ct] = 0.f;
    }
    const int per = (pages + p.ns - 1) / p.ns, pb = min(pages, z * per), pe = min(pages, pb + per);
    if (pb >= pe) {  // nothing to read: the parts say so
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        if (threadIdx.x < 16 && row[ct] >= 0) p.part_ml[(size_t)row[ct] * np + z] = make_float2(kLow, 0.f);
      return;
    }
    walk<CT>(p, p.block_tables + (size_t)live * p.max_blocks, h, pb, pe, pe * kPg, qf, o, m, l);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) leave(p, lds, o[ct], m[ct], l[ct], row[ct], z);
  } else {
    const int x = blockIdx.x - nshared, z = x % p.no, s = x / p.no;
    const int n = p.ctx_len[s];
    if (n <= 0) return;
    int live;
    const int skip = group_pages(p, s / p.width, live);
    const int pages = min((n + kPg - 1) / kPg, p.max_blocks) - skip;
    const int row = r < p.group ? s * p.hq + h * p.group + r : -1;
    const int per = (pages + p.no - 1) / p.no, pb = min(pages, z * per), pe = min(pages, pb + per);
    if (pb >= pe) {
      if (threadIdx.x < 16 && row >= 0) p.part_ml[(size_t)row * np + p.ns + z] = make_float2(kLow, 0.f);
      return;
    }
    bf16x8 qf[1][4];
    f32x4 o[1][8];
    float m[1] = {kLow}, l[1] = {0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) qf[0][k] = row >= 0 ? ld_bf16x8(p.q + (size_t)row * kDim + 32 * k + 8 * g) : zero_bf16x8();
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[0][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    walk<1>(p, p.block_tables + (size_t)s * p.max_blocks, h, skip + pb, skip + pe, n, qf, o, m, l);
    leave(p, lds, o[0], m[0], l[0], row, p.ns + z);
  }
}

// one wave per (slot, q head): lane z holds part z's statistics, then every lane two head dims
__global__ void __launch_bounds__(256) beam_join_kernel(BeamAttnParams p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.slots * p.hq || p.ctx_len[row / p.hq] <= 0) return;
  const int np = p.ns + p.no;
  float2 ml = make_float2(kLow, 0.f);
  if (lane < np) ml = p.part_ml[(size_t)row * np + lane];
  const float top = wave_max(ml.x), w = exp2f(ml.x - top);
  const float sum = wave_sum(ml.y * w);
  const float* po = p.part_o + (size_t)row * np * kDim + 2 * lane;
  float a = 0.f, b = 0.f;
  for (int z = 0; z < np; ++z) {
    if (__shfl(ml.y, z) == 0.f) continue;  // a part without keys has left no sums
    const float wz = __shfl(w, z);
    const f32x2 v = *reinterpret_cast<const f32x2*>(po + (size_t)z * kDim);
    a += v[0] * wz;
    b += v[1] * wz;
  }
  const float inv = 1.f / sum;
  bf16* op = p.out + (size_t)row * kDim + 2 * lane;
  op[0] = f2bf(a * inv);
  op[1] = f2bf(b * inv);
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

}  // namespace
}  // namespace dsse

// Column tiles of a workgroup and cuts of the walks, from what the host knows: the lengths are on the device, so the tables' width
// stands for them.
extern "C" void dsse_beam_plan(dsse::BeamAttnParams* p) {
  const int cols = p->width * p->group, groups = p->slots / p->width;
  p->tiles = cols <= 16 ? 1 : (cols <= 32 ? 2 : 4);
  p->col_blocks = (cols + 16 * p->tiles - 1) / (16 * p->tiles);
  auto cut = [&](int64_t items, int most) {
    const int64_t n = items >= 512 ? 1 : (512 + items - 1) / items;
    return (int)(n < most ? n : most);
  };
  const int by4 = (p->max_blocks + 3) / 4;  // a page per wave
  p->ns = cut((int64_t)groups * p->col_blocks * p->hkv, by4 < 32 ? by4 : 32);
  p->no = cut((int64_t)p->slots * p->hkv, by4 < 8 ? by4 : 8);
}

extern "C" hipError_t dsse_beam_attention(const dsse::BeamAttnParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->slots < 1 || p->width < 1 || p->width > kBeamWidth || p->slots % p->width || p->group < 1 || p->group > 16 || p->ns < 1 || p->no < 1 ||
      p->ns + p->no > 64 || p->hkv > 65535)
    return hipErrorInvalidValue;
  const int groups = p->slots / p->width;
  const dim3 grid(groups * p->col_blocks * p->ns + p->slots * p->no, p->hkv), block(64 * kBeamWaves);
  if (p->tiles == 1) hipLaunchKernelGGL((beam_attention_kernel<1>), grid, block, 0, st, *p);
  else if (p->tiles == 2) hipLaunchKernelGGL((beam_attention_kernel<2>), grid, block, 0, st, *p);
  else if (p->tiles == 4) hipLaunchKernelGGL((beam_attention_kernel<4>), grid, block, 0, st, *p);
  else return hipErrorInvalidValue;
  hipLaunchKernelGGL(beam_join_kernel, dim3((p->slots * p->hq + 3) / 4), dim3(256), 0, st, *p);
  return hipGetLastError();
}

extern "C" hipError_t dsse_beam_shared(const int* tables, const int* ctx_len, int* shared, int groups, int width, int max_blocks,
                                       hipStream_t st) {
  if (groups < 1 || width < 1 || width > dsse::kBeamWidth) return hipErrorInvalidValue;
  hipLaunchKernelGGL(dsse::beam_shared_kernel, dim3(groups), dim3(64), 0, st, tables, ctx_len, shared, width, max_blocks);
  return hipGetLastError();
}
