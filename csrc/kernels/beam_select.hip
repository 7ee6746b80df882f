// Beam search's choice: the K best continuations of a group over its beams' rows of logits and the vocabulary,
//   score(row, token) = scores[row] + logits[row, token] - log sum_t exp logits[row, t],
// by (score descending, row ascending, token ascending), in two launches.
//
// rows   one workgroup per (row, chunk of the vocabulary).  A chunk stays in registers: its maximum, the sum of exponentials about
//        it, then its K best logits (within a row the order of the logits is the order of the scores).  The K-th best of some
//        buckets' maxima bounds the chunk's K-th best from below; what reaches it (1.2 K values where they fall at random) is gathered
//        in LDS, and a value's place is the number of gathered ones before it.  No sort, no second read.
// merge  one workgroup per group: the chunks' sums joined into each row's log-sum, the same selection over the rows' candidates.
//
// Two candidates of different rows may be nearer to each other than 32 bits of a score of tens tell, so scores are compared in 64
// bits, the exponentials' argument carries the error of log2(e), and sums are joined in 64 bits from the wave on.  A row's log-sum is
// off by 1e-8 to 3e-8 rms for 32768 tokens and more (by 1.2e-7 with every sum in 32 bits), 5e-8 for 1000; where all of a row's terms
// are the same, by the rounding of their exponential, 1.2e-7.
//
// 64 groups of 8 rows of 131072 bf16 logits, 16 candidates: 35 us (3.8 TB/s; 31 of logits that the caches still hold in part), 29 without
// the selection, which the exponentials share the vector units with; the merge 7.4 to 7.9.  One group of 4 rows of 32768 (fp32): 4.4 and
// 4.6 to 5.0 us, all latency.
#include "api_beams.h"

namespace dsse {
namespace {

constexpr int kSelThreads = 512;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kGather = 1024;  // candidates that LDS holds; a chunk or group with more that reach the bound (the best ones all in a few
                               // threads) is walked K times instead
// Where more buckets than this are as good as the K-th one, the bound lies among equals, as in a row that a finite value masks: it then
// goes by their places too, or all of them would be gathered.  64x8 rows of 131072 bf16 with five tokens left: 38 us, 451 by a walk per
// candidate; rows without equals 31 either way.
constexpr int kTies = 16;

// e^(x - m) for x <= m, by 2^y with y = (x - m) log2(e) in two parts
DEV float exp_below(float x, float m) {
  const float d = x - m;
  return __builtin_amdgcn_exp2f(fmaf(d, 1.4426950216293335f, d * 1.9259629911266175e-8f));
}

// 16 bytes of logits, from any element on: global accesses may begin anywhere
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  u32x4 v;
  typedef u32x4 unit __attribute__((aligned(4)));
  DEV void load(const float* p) { v = *reinterpret_cast<const unit*>(p); }
  DEV float at(int i) const { return __uint_as_float(v[i]); }
  DEV void drop(int i, bool yes) { v[i] = yes ? kNone : v[i]; }
};
template <> struct Piece<bf16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;
  u32x4 v;
  typedef u32x4 unit __attribute__((aligned(2)));
  DEV void load(const bf16* p) { v = *reinterpret_cast<const unit*>(p); }
  DEV float at(int i) const { return __uint_as_float(i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16); }
  DEV void drop(int i, bool yes) { v[i / 2] = yes ? (v[i / 2] & (i % 2 ? 0xffffu : 0xffff0000u)) | (kNone & (i % 2 ? 0xffff0000u : 0xffffu)) : v[i / 2]; }
};

// (value descending, token ascending) as the order of one number; -0 counts as 0
DEV uint64_t logit_key(float v, int token) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~token;
}
DEV float key_logit(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

template <typename V>
DEV V lane_value(V v, int lane) {  // a wave-uniform lane's value, without LDS
  static_assert(sizeof(V) % 4 == 0, "whole words");
  uint32_t w[sizeof(V) / 4];
  __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) w[i] = __builtin_amdgcn_readlane(w[i], lane);
  __builtin_memcpy(&v, w, sizeof(V));
  return v;
}

// The K-th largest of 64 buckets' maxima, the same for every thread; mine: this thread's maximum, bucket = lane.  Of the chunk's values
// some 64 (H(64) - H(64 - K)) reach it: 1.1 K of them for K = 8, 1.4 K for 32, but 4.7 K for 64.  ties: buckets that equal it.
template <typename V>
DEV V bound_of_lanes(V mine, int K, V* all, int* rank, int& ties) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  all[threadIdx.x] = mine;
  if (wave == 0) rank[lane] = 0;
  __syncthreads();
  V v = all[lane];
#pragma unroll
  for (int w = 1; w < kSelWaves; ++w) v = all[w * 64 + lane] > v ? all[w * 64 + lane] : v;
  int n = 0;  // buckets before this one, some of them per wave; of equal ones the lower lane is before
#pragma unroll
  for (int i = 0; i < 64 / kSelWaves; ++i) {
    const int l = wave * (64 / kSelWaves) + i;
    const V u = lane_value(v, l);
    n += u > v || (u == v && l < lane) ? 1 : 0;
  }
  atomicAdd(&rank[lane], n);
  __syncthreads();
  const unsigned long long who = __ballot(rank[lane] == K - 1);
  const V bound = lane_value(v, __ffsll(who) - 1);
  ties = __popcll(__ballot(v == bound));
  return bound;
}
// The same with 128 buckets, where 64 would let too much through: 1.4 K for K = 64
template <typename V>
DEV V bound_of_many(V mine, int K, V* all, int* rank, int& ties) {
  constexpr int kBuckets = 128, kParts = kSelThreads / kBuckets, kEach = kBuckets / kParts;
  const int b = threadIdx.x % kBuckets, part = threadIdx.x / kBuckets;
  all[threadIdx.x] = mine;
  if (part == 0) rank[b] = 0;
  __syncthreads();
  V v = all[b];
#pragma unroll
  for (int k = 1; k < kParts; ++k) v = all[b + k * kBuckets] > v ? all[b + k * kBuckets] : v;
  __syncthreads();
  if (part == 0) all[b] = v;
  __syncthreads();
  int n = 0;  // buckets before this one, a part of them per thread; of equal ones the lower is before
#pragma unroll 8
  for (int i = part * kEach; i < part * kEach + kEach; ++i) n += all[i] > v || (all[i] == v && i < b) ? 1 : 0;
  atomicAdd(&rank[b], n);
  __syncthreads();
  if (part == 0 && rank[b] == K - 1) all[kBuckets] = v;
  __syncthreads();
  const V bound = all[kBuckets];
  ties = __popcll(__ballot(all[threadIdx.x & 63] == bound)) + __popcll(__ballot(all[64 + (threadIdx.x & 63)] == bound));
  return bound;
}
template <typename V>
DEV V bound_of(V mine, int K, V* all, int* rank, int& ties) {
  return K <= 32 ? bound_of_lanes(mine, K, all, rank, ties) : bound_of_many(mine, K, all, rank, ties);
}
// The place that the equals of such a bound count up to.  above, equal: whether this thread's maximum is above the bound or equals it;
// place: of the first of this thread's values that equals it.  Called by every thread.
DEV int last_place(bool above, bool equal, int place, int K, int* all, int* rank) {
  int ties;
  __syncthreads();  // everyone has read what the bound left in `all` and `rank`
  return 0x7ffffffe - bound_of(above ? 0x7fffffff : (equal ? 0x7ffffffe - place : -1), K, all, rank, ties);
}

// Q: 16-byte pieces of a thread.  A row is whole pieces from its first element on, whatever address that has, and the few elements
// behind them, which go to the first threads of its first workgroup, one each.  So the token alone says who adds what, and rows of
// the same logits have the same log-sum, bit for bit: their candidates tie, as they should.  64x8 rows of 131071 bf16 take 43.5 us so,
// 38 with pieces at 16-byte addresses, whose sums differ with the address; of 50001 and 131069 fp32 as long either way.
template <typename T, int Q>
__global__ void __launch_bounds__(kSelThreads, 6) beam_rows_kernel(BeamSelectParams p) {
  constexpr int N = Piece<T>::N;
  __shared__ float s_max[kSelWaves];
  __shared__ double s_sum[kSelWaves];
  __shared__ float bucket[kSelThreads];
  __shared__ int rank[128], count;
  __shared__ uint64_t got[kGather];
  const int row = blockIdx.y, c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const int pieces = p.V / N;
  const int place = c * Q * kSelThreads + (int)threadIdx.x;  // of this thread's first piece; the others kSelThreads apart
  Piece<T> q[Q];
  float extra = -INFINITY;
  int extra_at = -1;
  if (threadIdx.x == 0) count = 0;
  if (pieces > 0) {  // all requested before the first is used
#pragma unroll
    for (int k = 0; k < Q; ++k) q[k].load(x + min(place + k * kSelThreads, pieces - 1) * N);
  }
  if (c == 0 && (int)threadIdx.x < p.V - pieces * N) {
    extra_at = pieces * N + threadIdx.x;
    extra = (float)x[extra_at];
  }
  if ((c + 1) * Q * kSelThreads > pieces) {  // what is past the row
#pragma unroll
    for (int k = 0; k < Q; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) q[k].v[i] = place + k * kSelThreads < pieces ? q[k].v[i] : Piece<T>::kNone;
  }
  // the end token counts in the sum and is no candidate
  float end = -INFINITY;
  const int ahead = p.eos - place * N;  // elements from this thread's first one to it
  if (p.eos >= 0) {
    bool mine = extra_at == p.eos;
    if (mine) extra = -INFINITY;
    if (__any(ahead >= 0 && ahead < Q * kSelThreads * N)) {
#pragma unroll
      for (int k = 0; k < Q; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool here = ahead == k * kSelThreads * N + i && place + k * kSelThreads < pieces;
          mine = mine || here;
          q[k].drop(i, here);
        }
    }
    if (mine) {
      end = (float)x[p.eos];
      if (p.end_scores) p.end_logit[row] = end;
    }
  }
  float most[Q], m = extra;
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    most[k] = q[k].at(0);
#pragma unroll
    for (int i = 1; i < N; ++i) most[k] = fmaxf(most[k], q[k].at(i));
    m = fmaxf(m, most[k]);
  }
  const float ref = fmaxf(fmaxf(m, end), -3.4028234663852886e38f);  // -inf alone sums to zero
  // a piece's sum, then the thread's, in 32 bits, everything behind it in 64: a likely token, beside which the others are rounded, is added
  // to 7 + Q times, not to all of the thread's and then the wave's
  float own = 0.f;
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    float part = exp_below(q[k].at(0), ref);
#pragma unroll
    for (int i = 1; i < N; ++i) part += exp_below(q[k].at(i), ref);
    own += part;
  }
  double sum = (double)own + ((double)exp_below(extra, ref) + exp_below(end, ref));
  const float top = wave_max(ref);
  sum *= exp_below(ref, top);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) s_max[wave] = top, s_sum[wave] = sum;
  int ties;
  const float bound = bound_of(m, p.K, bucket, rank, ties);
  if (threadIdx.x == 0) {
    float all = s_max[0];
    double s = 0;
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w) all = fmaxf(all, s_max[w]);
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) s += s_sum[w] * exp_below(s_max[w], all);
    p.most[(size_t)row * p.chunks + c] = all;
    p.sum[(size_t)row * p.chunks + c] = s;
  }
  // pieces that reach the bound are few: they are read again (from the caches), so that the registers need no index
  int last = 0x7fffffff;  // piece that the bound's equals count up to; what is behind the whole pieces counts as the next one
  if (ties > kTies && bound > -INFINITY) {
    int first = pieces;
#pragma unroll
    for (int k = Q - 1; k >= 0; --k) first = most[k] == m ? place + k * kSelThreads : first;
    last = last_place(m > bound, m == bound, first, p.K, reinterpret_cast<int*>(bucket), rank);
  }
  auto reaches = [&](float v, int piece) { return v >= bound && v > -INFINITY && (v > bound || piece <= last); };
  auto gather = [&](float v, int piece, int token) {
    if (reaches(v, piece) && token != p.eos) {
      const int at = atomicAdd(&count, 1);
      if (at < kGather) got[at] = logit_key(v, token);
    }
  };
  uint32_t hits = 0;
#pragma unroll
  for (int k = 0; k < Q; ++k) hits |= reaches(most[k], place + k * kSelThreads) ? 1u << k : 0u;
  if (extra_at >= 0) gather(extra, pieces, extra_at);
  while (hits) {
    const int piece = place + (__ffs(hits) - 1) * kSelThreads, token = piece * N;
    hits &= hits - 1;
    Piece<T> h;
    h.load(x + token);
#pragma unroll
    for (int i = 0; i < N; ++i) gather(h.at(i), piece, token + i);
  }
  __syncthreads();
  const int n = count;
  float2* cand = p.cand + ((size_t)row * p.chunks + c) * p.K;
  auto put = [&](int at, uint64_t key) { cand[at] = make_float2(key_logit(key), __int_as_float(~(int)(uint32_t)key)); };
  if (n <= kGather) {
    for (int a = threadIdx.x; a < n; a += kSelThreads) {
      const uint64_t key = got[a];
      int before = 0;
#pragma unroll 8
      for (int b = 0; b < n; ++b) before += got[b] > key ? 1 : 0;
      if (before < p.K) put(before, key);
    }
  } else {
    uint64_t prev = ~0ull;
    for (int at = 0; at < p.K; ++at) {
      uint64_t best = 0;
      auto next = [&](float v, int token) {
        const uint64_t key = logit_key(v, token);
        if (v > -INFINITY && token != p.eos && key < prev && key > best) best = key;
      };
      if (extra_at >= 0) next(extra, extra_at);
      for (int e = place; e < min(place + Q * kSelThreads, pieces); e += kSelThreads)
        for (int i = 0; i < N; ++i) next((float)x[e * N + i], e * N + i);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) got[wave + kSelWaves * (at & 1)] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSelWaves; ++w) best = max(best, got[w + kSelWaves * (at & 1)]);
      if (threadIdx.x == 0) put(at, best);
      prev = best;
    }
  }
  for (int a = n + threadIdx.x; a < p.K; a += kSelThreads) cand[a] = make_float2(-INFINITY, __int_as_float(-1));
}

struct Pick {
  double s;
  int id;  // beam of the group * V + token
};
DEV bool before(const Pick& a, const Pick& b) { return a.s > b.s || (a.s == b.s && a.id < b.id); }
// n / d for whole numbers below 2^21, inv = 1 / d in 32 bits: half of one away from the next, where the product is off by 2^-22
DEV int quotient(int n, float inv) { return (int)(((float)n + 0.5f) * inv); }

__global__ void __launch_bounds__(kSelThreads) beam_merge_kernel(BeamSelectParams p) {
  constexpr int kHeld = 8;             // candidates of a thread that its registers hold
  constexpr int kNoted = kHeld * kSelThreads;  // lists that can be noted
  __shared__ double base[kBeamWidth];  // scores[row] - log(sum about `top`); NaN: the row offers nothing
  __shared__ float top[kBeamWidth];
  __shared__ double bucket[kSelThreads];
  __shared__ Pick got[kGather];
  __shared__ int rank[128], count, open[kNoted], nopen;
  const int g = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) count = nopen = 0;
  // The chunks' lists are in order: their first `deep` places are looked at, the others only where the last of those reaches the
  // bound.  Neighbouring threads look at a list's places, each list from another one on: a row far ahead has its best in few lists, and
  // they have to fall into different buckets.
  const int lists = p.width * p.chunks, deep = min(p.K, max(1, kHeld * kSelThreads / lists)), total = lists * deep;
  const float by_deep = 1.f / (float)deep, by_chunks = 1.f / (float)p.chunks;
  const float2* cand = p.cand + (size_t)g * lists * p.K;
  auto spot = [&](int e, int& list) {  // candidate e's list and place
    list = quotient(e, by_deep);
    const int at = e - list * deep + 5 * list;
    return at - quotient(at, by_deep) * deep;
  };
  auto load = [&](int e) {
    int list;
    const int at = spot(e, list);
    return cand[(size_t)list * p.K + at];
  };
  float2 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (i == 0 || i * kSelThreads < total) held[i] = load(min((int)threadIdx.x + i * kSelThreads, total - 1));
  for (int w = threadIdx.x >> 4; w < p.width; w += kSelThreads / 16) {  // 16 lanes per row
    const size_t at = (size_t)(g * p.width + w) * p.chunks;
    const int l = threadIdx.x & 15;
    float m = -INFINITY;
    for (int c = l; c < p.chunks; c += 16) m = fmaxf(m, p.most[at + c]);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    double sum = 0;
    for (int c = l; c < p.chunks; c += 16) sum += p.sum[at + c] * exp((double)p.most[at + c] - (double)m);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    if (l == 0) {
      const float s = p.scores[g * p.width + w];
      const bool ok = s - s == 0.f && m - m == 0.f && sum - sum == 0. && sum > 0.;
      const double b = ok ? (double)s - log(sum) : __builtin_nan("");
      base[w] = b;
      top[w] = m;
      if (p.end_scores) p.end_scores[g * p.width + w] = ok ? (float)(b + ((double)p.end_logit[g * p.width + w] - (double)m)) : -INFINITY;
    }
  }
  __syncthreads();
  auto pick_of = [&](int list, float2 c) {
    const int w = quotient(list, by_chunks);
    const double b = base[w];
    Pick r{-INFINITY, 0x7fffffff};
    if (c.x > -INFINITY && b == b) r = Pick{b + ((double)c.x - (double)top[w]), w * p.V + __float_as_int(c.y)};
    return r;
  };
  // the looked-at candidates of this thread, those in registers first
  auto each = [&](auto f) {
    int list;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int e = threadIdx.x + i * kSelThreads;
      if (e >= total) return;
      const int at = spot(e, list);
      f(pick_of(list, held[i]), list, at);
    }
    for (int e = threadIdx.x + kHeld * kSelThreads; e < total; e += kSelThreads) {
      const int at = spot(e, list);
      f(pick_of(list, load(e)), list, at);
    }
  };
  double best = -INFINITY;
  each([&](const Pick& c, int, int) { best = c.s > best ? c.s : best; });
  int ties;
  const double bound = bound_of(best, p.K, bucket, rank, ties);
  int last = 0x7fffffff;  // id that the bound's equals count up to
  if (ties > kTies && bound > -INFINITY) {
    int first = 0x7ffffffe;
    each([&](const Pick& c, int, int) { first = c.s == bound ? min(first, c.id) : first; });
    last = last_place(best > bound, best == bound, first, p.K, reinterpret_cast<int*>(bucket), rank);
  }
  auto gather = [&](const Pick& c) {
    if (c.s >= bound && c.s > -INFINITY && (c.s > bound || c.id <= last)) {
      const int at = atomicAdd(&count, 1);
      if (at < kGather) got[at] = c;
    }
  };
  if (best >= bound)
    each([&](const Pick& c, int list, int at) {
      gather(c);
      // by the score alone: of logits whose scores are equal the later one in a list may be the lower token
      if (at == deep - 1 && deep < p.K && c.s >= bound && c.s > -INFINITY) {
        const int o = atomicAdd(&nopen, 1);
        if (o < kNoted) open[o] = list;
        else atomicAdd(&count, kGather + 1);  // place by place, below
      }
    });
  __syncthreads();
  const int opened = count <= kGather ? nopen : 0;
  __syncthreads();  // every thread has read the counts: they may change
  if (opened > 0) {  // the other places of the lists that go on, all at once
    const int left = p.K - deep;
    const float by_left = 1.f / (float)left;
    for (int e = threadIdx.x; e < opened * left; e += kSelThreads) {
      const int o = quotient(e, by_left), list = open[o];
      gather(pick_of(list, cand[(size_t)list * p.K + deep + e - o * left]));
    }
    __syncthreads();
  }
  const int n = count;
  auto put = [&](int at, const Pick& c) {
    p.out_scores[(size_t)g * p.K + at] = (float)c.s;
    p.out_rows[(size_t)g * p.K + at] = g * p.width + c.id / p.V;
    p.out_tokens[(size_t)g * p.K + at] = c.id % p.V;
  };
  if (n <= kGather) {
    for (int a = threadIdx.x; a < n; a += kSelThreads) {
      const Pick c = got[a];
      int at = 0;
#pragma unroll 8
      for (int b = 0; b < n; ++b) at += before(got[b], c) ? 1 : 0;
      if (at < p.K) put(at, c);
    }
  } else {
    Pick prev{INFINITY, -1};
    for (int at = 0; at < p.K; ++at) {
      Pick b{-INFINITY, 0x7fffffff};
      for (int e = threadIdx.x; e < lists * p.K; e += kSelThreads) {
        const Pick c = pick_of(e / p.K, cand[e]);
        if (before(prev, c) && before(c, b)) b = c;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const Pick c{__shfl_xor(b.s, o), __shfl_xor(b.id, o)};
        if (before(c, b)) b = c;
      }
      if (lane == 0) got[wave + kSelWaves * (at & 1)] = b;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSelWaves; ++w)
        if (before(got[w + kSelWaves * (at & 1)], b)) b = got[w + kSelWaves * (at & 1)];
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
  if (p.pieces == 1) hipLaunchKernelGGL((beam_rows_kernel<T, 1>), grid, block, 0, st, p);
  else if (p.pieces == 2) hipLaunchKernelGGL((beam_rows_kernel<T, 2>), grid, block, 0, st, p);
  else if (p.pieces == 4) hipLaunchKernelGGL((beam_rows_kernel<T, 4>), grid, block, 0, st, p);
  else if (p.pieces == 8) hipLaunchKernelGGL((beam_rows_kernel<T, 8>), grid, block, 0, st, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace
}  // namespace dsse

// Pieces of a thread: as many as a row has and its registers hold, fewer while that leaves CUs empty
extern "C" void dsse_beam_plan_rows(dsse::BeamSelectParams* p) {
  const int n = p->f32 ? 4 : 8, row = (p->V + n - 1) / n, threads = dsse::kSelThreads;
  p->pieces = 1;
  while (p->pieces < 8 && p->pieces * threads < row) p->pieces *= 2;
  auto chunks = [&] { return (row + p->pieces * threads - 1) / (p->pieces * threads); };
  while (p->pieces > 1 && (int64_t)p->rows * chunks() < 512) p->pieces /= 2;
  p->chunks = chunks();
}

extern "C" hipError_t dsse_beam_select(const dsse::BeamSelectParams* p, hipStream_t st) {
  using namespace dsse;
  if (p->width < 1 || p->width > kBeamWidth || p->K < 1 || p->K > kBeamKeep || p->rows % p->width || p->rows > 65535 || p->V < 1 ||
      (int64_t)p->pieces * kSelThreads * p->chunks * (p->f32 ? 4 : 8) < p->V)
    return hipErrorInvalidValue;
  if (p->rows == 0) return hipSuccess;
  const hipError_t e = p->f32 ? launch_rows<float>(*p, st) : launch_rows<bf16>(*p, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(p->rows / p->width), dim3(kSelThreads), 0, st, *p);
  return hipGetLastError();
}
