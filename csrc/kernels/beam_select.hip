// Beam search's choice: the K best continuations of a group over its beams' rows of logits and the vocabulary,
//   score(row, token) = scores[row] + logits[row, token] - log sum_t exp logits[row, t],
// by (score descending, row ascending, token ascending), in two launches.
//
// rows   one workgroup per (row, chunk of the vocabulary).  A chunk stays in registers: its maximum, the sum of exponentials about
//        it, then its K best logits (within a row the order of the logits is the order of the scores).  The K-th best of 64
//        buckets' maxima (bucket = lane) bounds the chunk's K-th best from below; what reaches it (1.2 K values where they fall at
//        random) is gathered in LDS, and a value's place is the number of gathered ones before it.  No sort, no second read.
// merge  one workgroup per group: the chunks' sums joined into each row's log-sum, the same selection over the rows' candidates.
//
// Two candidates of different rows may be nearer to each other than 32 bits of a score of tens tell, so scores are compared in 64
// bits, and the exponentials' argument carries the error of log2(e): a row's log-sum is off by some 1e-8, not 1e-6.
#include "api_beams.h"

namespace dsse {
namespace {

constexpr int kSelThreads = 256;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kMergeCap = 2048;  // gathered candidates of a group that LDS holds

DEV bool before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }

// e^(x - m) for x <= m, by 2^y with y = (x - m) log2(e) in two parts
DEV float exp_below(float x, float m) {
  const float d = x - m;
  return __builtin_amdgcn_exp2f(fmaf(d, 1.4426950216293335f, d * 1.9259629911266175e-8f));
}

template <typename T> struct Quad;
template <> struct Quad<float> {
  static constexpr int N = 4;
  f32x4 v;
  DEV float at(int i) const { return v[i]; }
  DEV void put(int i, float x) { v[i] = x; }
};
template <> struct Quad<bf16> {
  static constexpr int N = 8;
  bf16x8 v;
  DEV float at(int i) const { return (float)v[i]; }
  DEV void put(int i, float x) { v[i] = (bf16)x; }
};

// Q: 16-byte pieces of a thread
template <typename T, int Q>
__global__ void __launch_bounds__(kSelThreads) beam_rows_kernel(BeamSelectParams p) {
  constexpr int N = Quad<T>::N;
  __shared__ float s_max[kSelWaves], s_sum[kSelWaves];
  __shared__ float b_val[kSelWaves][64];
  __shared__ int b_idx[kSelWaves][64];
  __shared__ float t_val;
  __shared__ int t_idx, count;
  __shared__ float g_val[kSelThreads * Q * N];
  __shared__ int g_idx[kSelThreads * Q * N];
  const int row = blockIdx.y, c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const int lo = c * p.chunk, hi = min(p.V, lo + p.chunk);
  // pieces of 16 bytes at 16-byte addresses; `skew` elements of the first one belong to what is before the chunk
  const int skew = (int)(reinterpret_cast<uintptr_t>(x + lo) % 16 / sizeof(T));
  const int first = lo - skew;
  Quad<T> q[Q];
  if (threadIdx.x == 0) count = 0;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const int e = first + (k * kSelThreads + threadIdx.x) * N;
    if (e >= lo && e + N <= hi) {
      q[k].v = ld_global<decltype(q[k].v)>(x + e);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) q[k].put(i, e + i >= lo && e + i < hi ? (float)x[e + i] : -INFINITY);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, q[k].at(i));
  }
  m = wave_max(m);
  if (lane == 0) s_max[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) m = fmaxf(m, s_max[w]);
  const float ref = fmaxf(m, -3.4028234663852886e38f);  // a chunk of -inf alone sums to zero
  float sum = 0.f;
  float best = -INFINITY;
  int bidx = 0x7fffffff - lane;  // lanes without a value keep places of their own
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const int e = first + (k * kSelThreads + threadIdx.x) * N;
    if (p.eos >= e && p.eos < e + N && p.eos >= lo && p.eos < hi) {  // the end token counts in the sum and is no candidate
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e + i == p.eos) {
          if (p.end_scores) p.end_logit[row] = q[k].at(i);
          sum += exp_below(q[k].at(i), ref);
          q[k].put(i, -INFINITY);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = q[k].at(i);
      sum += exp_below(v, ref);
      if (v > best) best = v, bidx = e + i;
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) s_sum[wave] = sum;
  b_val[wave][lane] = best;
  b_idx[wave][lane] = bidx;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kSelWaves; ++w)
      if (before(b_val[w][lane], b_idx[w][lane], best, bidx)) best = b_val[w][lane], bidx = b_idx[w][lane];
    int rank = 0;
    for (int l = 0; l < 64; ++l) {
      const float v = __shfl(best, l);
      const int i = __shfl(bidx, l);
      rank += before(v, i, best, bidx) ? 1 : 0;
    }
    if (rank == p.K - 1) t_val = best, t_idx = bidx;
    if (lane == 0) {
      float all = 0.f;
      for (int w = 0; w < kSelWaves; ++w) all += s_sum[w];
      p.stat[(size_t)row * p.chunks + c] = make_float2(ref, all);
    }
  }
  __syncthreads();
  const float tv = t_val;
  const int ti = t_idx;
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const int e = first + (k * kSelThreads + threadIdx.x) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = q[k].at(i);
      if (v > -INFINITY && (v > tv || (v == tv && e + i <= ti))) {
        const int at = atomicAdd(&count, 1);
        g_val[at] = v;
        g_idx[at] = e + i;
      }
    }
  }
  __syncthreads();
  const int n = count;
  float2* cand = p.cand + ((size_t)row * p.chunks + c) * p.K;
  for (int a = threadIdx.x; a < n; a += kSelThreads) {
    const float v = g_val[a];
    const int i = g_idx[a];
    int rank = 0;
    for (int b = 0; b < n; ++b) rank += before(g_val[b], g_idx[b], v, i) ? 1 : 0;
    if (rank < p.K) cand[rank] = make_float2(v, __int_as_float(i));
  }
  for (int a = n + threadIdx.x; a < p.K; a += kSelThreads) cand[a] = make_float2(-INFINITY, __int_as_float(-1));
}

struct Pick {
  double s;
  int row, token;  // row: beam of the group
};
DEV bool before(const Pick& a, const Pick& b) {
  return a.s > b.s || (a.s == b.s && (a.row < b.row || (a.row == b.row && a.token < b.token)));
}
DEV Pick shfl_pick(const Pick& a, int lane) { return Pick{__shfl(a.s, lane), __shfl(a.row, lane), __shfl(a.token, lane)}; }
DEV Pick shfl_xor_pick(const Pick& a, int o) { return Pick{__shfl_xor(a.s, o), __shfl_xor(a.row, o), __shfl_xor(a.token, o)}; }

__global__ void __launch_bounds__(kSelThreads) beam_merge_kernel(BeamSelectParams p) {
  __shared__ double base[kBeamWidth], top[kBeamWidth];  // scores[row] - log(sum about `top`); NaN: the row offers nothing
  __shared__ Pick bucket[kSelWaves][64], thr, got[kMergeCap];
  __shared__ int count;
  const int g = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) count = 0;
  for (int w = wave; w < p.width; w += kSelWaves) {
    const float2* st = p.stat + (size_t)(g * p.width + w) * p.chunks;
    float m = -INFINITY;
    for (int c = lane; c < p.chunks; c += 64) m = fmaxf(m, st[c].x);
    m = wave_max(m);
    double sum = 0;
    for (int c = lane; c < p.chunks; c += 64) sum += (double)st[c].y * exp((double)st[c].x - (double)m);
    sum = wave_sum(sum);
    if (lane == 0) {
      const float s = p.scores[g * p.width + w];
      const bool ok = s - s == 0.f && m - m == 0.f && sum - sum == 0. && sum > 0.;
      base[w] = ok ? (double)s - log(sum) : __builtin_nan("");
      top[w] = m;
      if (p.end_scores) {
        const float e = p.end_logit[g * p.width + w];
        p.end_scores[g * p.width + w] = ok ? (float)(base[w] + ((double)e - (double)m)) : -INFINITY;
      }
    }
  }
  __syncthreads();
  const int lists = p.width * p.chunks, total = lists * p.K;
  const float2* cand = p.cand + (size_t)g * total;
  // candidate e: list e % lists, place e / lists -- neighbouring threads look at different lists
  auto pick_of = [&](int e) {
    const int l = e % lists, w = l / p.chunks;
    const float2 c = cand[(size_t)l * p.K + e / lists];
    const double b = base[w];
    Pick r{-INFINITY, 0x7fffffff, e};
    if (c.x > -INFINITY && b == b) r = Pick{b + ((double)c.x - top[w]), w, __float_as_int(c.y)};
    return r;
  };
  Pick best{-INFINITY, 0x7fffffff, 0x7fffffff - (int)threadIdx.x};
  for (int e = threadIdx.x; e < total; e += kSelThreads) {
    const Pick c = pick_of(e);
    if (before(c, best)) best = c;
  }
  bucket[wave][lane] = best;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kSelWaves; ++w)
      if (before(bucket[w][lane], best)) best = bucket[w][lane];
    int rank = 0;
    for (int l = 0; l < 64; ++l) rank += before(shfl_pick(best, l), best) ? 1 : 0;
    if (rank == p.K - 1) thr = best;
  }
  __syncthreads();
  const Pick t = thr;
  for (int e = threadIdx.x; e < total; e += kSelThreads) {
    const Pick c = pick_of(e);
    if (c.s > -INFINITY && !before(t, c)) {
      const int at = atomicAdd(&count, 1);
      if (at < kMergeCap) got[at] = c;
    }
  }
  __syncthreads();
  const int n = count;
  auto put = [&](int at, const Pick& c) {
    p.out_scores[(size_t)g * p.K + at] = (float)c.s;
    p.out_rows[(size_t)g * p.K + at] = g * p.width + c.row;
    p.out_tokens[(size_t)g * p.K + at] = c.token;
  };
  if (n <= kMergeCap) {
    for (int a = threadIdx.x; a < n; a += kSelThreads) {
      const Pick c = got[a];
      int rank = 0;
      for (int b = 0; b < n; ++b) rank += before(got[b], c) ? 1 : 0;
      if (rank < p.K) put(rank, c);
    }
  } else {
    // more than LDS holds (the best ones all in a few lanes' lists): one place after another
    Pick prev{INFINITY, -1, -1};
    for (int at = 0; at < p.K; ++at) {
      Pick b{-INFINITY, 0x7fffffff, 0x7fffffff};
      for (int e = threadIdx.x; e < total; e += kSelThreads) {
        const Pick c = pick_of(e);
        if (before(prev, c) && before(c, b)) b = c;
      }
      for (int o = 32; o >= 1; o >>= 1) {
        const Pick c = shfl_xor_pick(b, o);
        if (before(c, b)) b = c;
      }
      __syncthreads();
      if (lane == 0) bucket[wave][0] = b;
      __syncthreads();
      b = bucket[0][0];
      for (int w = 1; w < kSelWaves; ++w)
        if (before(bucket[w][0], b)) b = bucket[w][0];
      if (threadIdx.x == 0) put(at, b);
      prev = b;
    }
  }
  for (int a = n + threadIdx.x; a < p.K; a += kSelThreads) {
    p.out_scores[(size_t)g * p.K + a] = -INFINITY;
    p.out_rows[(size_t)g * p.K + a] = -1;
    p.out_tokens[(size_t)g * p.K + a] = -1;
  }
}

template <typename T>
hipError_t launch_rows(const BeamSelectParams& p, hipStream_t st) {
  const dim3 grid(p.chunks, p.rows), block(kSelThreads);
  constexpr int N = Quad<T>::N, kPiece = kSelThreads * N;
  const bool whole = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld % N == 0 && p.chunk % N == 0;
  const int q = (p.chunk + (whole ? 0 : N - 1) + kPiece - 1) / kPiece;  // a chunk that begins inside a piece needs one more
  if (q <= 1) hipLaunchKernelGGL((beam_rows_kernel<T, 1>), grid, block, 0, st, p);
  else if (q <= 2) hipLaunchKernelGGL((beam_rows_kernel<T, 2>), grid, block, 0, st, p);
  else if (q <= 4 && N == 4) hipLaunchKernelGGL((beam_rows_kernel<T, 4>), grid, block, 0, st, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace
}  // namespace dsse

// Vocabulary of a workgroup: as much as its registers hold, less while that leaves CUs empty
extern "C" int dsse_beam_chunk(int rows, int V, int f32, int whole) {
  const int n = f32 ? 4 : 8;
  for (int q = f32 ? 4 : 2; q >= 1; q /= 2) {
    const int chunk = q * dsse::kSelThreads * n - (whole ? 0 : n);
    if (q == 1 || (int64_t)rows * ((V + chunk - 1) / chunk) >= 512) return chunk;
  }
  return 1;
}

extern "C" hipError_t dsse_beam_select(const dsse::BeamSelectParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->width < 1 || p->width > kBeamWidth || p->K < 1 || p->K > kBeamKeep || p->rows % p->width || p->rows > 65535 || p->V < 1 ||
      p->chunk < 1 || (int64_t)p->chunk * p->chunks < p->V)
    return hipErrorInvalidValue;
  if (p->rows == 0) return hipSuccess;
  const hipError_t e = p->f32 ? launch_rows<float>(*p, st) : launch_rows<bf16>(*p, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(p->rows / p->width), dim3(kSelThreads), 0, st, *p);
  return hipGetLastError();
}
