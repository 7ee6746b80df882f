// torch operator registrations (namespace torch.ops.dsse) of the kernels in api_beams.h: selection over beams and vocabulary,
// attention over pages that beams share, forks of block tables, states that change slots.
//
// As in the other binding files, every op validates device, dtype and the shapes and strides its kernel's indexing assumes before
// launching, and launches on torch's current HIP stream of the tensors' device (graph-capturable).  Work areas come from torch's
// allocator within the call: on that stream, and inside a captured graph from the graph's own pool, so no two graphs share one.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "api_beams.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

#define DSSE_CHECK_HIP(expr)                                                             \
  do {                                                                                   \
    hipError_t _e = (expr);                                                              \
    TORCH_CHECK(_e == hipSuccess, "dsse kernel launch failed: ", hipGetErrorString(_e)); \
  } while (0)

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void on(const Tensor& t, const Tensor& first, const char* name, bool contiguous = true) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.device() == first.device(), name, " must be on the device of the other tensors");
  if (contiguous) TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void typed(const Tensor& t, const Tensor& first, at::ScalarType type, const char* name) {
  on(t, first, name);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", c10::toString(type));
}
int beams(int64_t slots, int64_t width) {
  TORCH_CHECK(width >= 1 && width <= dsse::kBeamWidth, "a group has 1 to ", dsse::kBeamWidth, " beams");
  TORCH_CHECK(slots % width == 0, "slots must be whole groups of `width` beams");
  return (int)(slots / width);
}
// whether the dimensions from `first` on are one contiguous run
bool packed(const Tensor& t, int64_t first) {
  int64_t run = 1;
  for (int64_t d = t.dim() - 1; d >= first; --d) {
    if (t.size(d) != 1 && t.stride(d) != run) return false;
    run *= t.size(d);
  }
  return true;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

void beam_select(const Tensor& logits, const Tensor& scores, Tensor& out_scores, Tensor& out_rows, Tensor& out_tokens, int64_t eos_id,
                 const OptTensor& end_scores) {
  on(logits, logits, "logits", false);
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16, "logits must be fp32 or bf16");
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) == 1 || logits.stride(1) == 1) && (logits.size(0) == 1 || logits.stride(0) >= logits.size(1)),
              "logits must be [rows, V] with a unit innermost stride");
  typed(scores, logits, at::kFloat, "scores");
  typed(out_scores, logits, at::kFloat, "out_scores");
  typed(out_rows, logits, at::kInt, "out_rows");
  typed(out_tokens, logits, at::kInt, "out_tokens");
  TORCH_CHECK(scores.dim() == 2 && scores.numel() == logits.size(0), "scores must be [groups, width], a number per row of logits");
  const int groups = beams(logits.size(0), scores.size(1));
  const int64_t V = logits.size(1), K = out_scores.dim() == 2 ? out_scores.size(1) : 0;
  TORCH_CHECK(out_scores.dim() == 2 && out_scores.size(0) == groups && K >= 1 && K <= dsse::kBeamKeep, "out_scores must be [groups, 1 to ",
              dsse::kBeamKeep, "]");
  TORCH_CHECK(out_rows.sizes() == out_scores.sizes() && out_tokens.sizes() == out_scores.sizes(), "outputs differ in shape");
  TORCH_CHECK(V >= 1 && V <= (1 << 24) && logits.size(0) <= 65535, "1 to 2^24 tokens, at most 65535 rows");
  TORCH_CHECK(eos_id >= -1 && eos_id < V, "eos_id must be a token or -1");
  if (end_scores.has_value()) {
    typed(*end_scores, logits, at::kFloat, "end_scores");
    TORCH_CHECK(end_scores->sizes() == scores.sizes(), "end_scores must match scores");
    TORCH_CHECK(eos_id >= 0, "end_scores needs an eos_id");
  }
  if (logits.size(0) == 0) return;
  const c10::DeviceGuard guard(logits.device());
  dsse::BeamSelectParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.size(0) == 1 ? V : logits.stride(0);
  p.f32 = logits.scalar_type() == at::kFloat ? 1 : 0;
  p.rows = (int)logits.size(0), p.width = (int)scores.size(1), p.V = (int)V, p.K = (int)K, p.eos = (int)eos_id;
  dsse_beam_plan_rows(&p);
  // [sums | candidates | maxima | end logits]
  const int64_t parts = (int64_t)p.rows * p.chunks;
  Tensor work = at::empty({parts * (3 + 2 * K) + p.rows}, scores.options());
  p.sum = reinterpret_cast<double*>(work.data_ptr<float>());
  p.cand = reinterpret_cast<float2*>(p.sum + parts);
  p.most = reinterpret_cast<float*>(p.cand + parts * K);
  p.end_logit = p.most + parts;
  p.scores = scores.data_ptr<float>();
  p.out_scores = out_scores.data_ptr<float>();
  p.out_rows = out_rows.data_ptr<int>();
  p.out_tokens = out_tokens.data_ptr<int>();
  p.end_scores = end_scores.has_value() ? end_scores->data_ptr<float>() : nullptr;
  DSSE_CHECK_HIP(dsse_beam_select(&p, stream_of(logits)));
}

void beam_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_tables, const Tensor& ctx_len,
                    const Tensor& shared, Tensor& out, int64_t width) {
  typed(q, q, at::kBFloat16, "q");
  typed(k_cache, q, at::kBFloat16, "k_cache");
  typed(v_cache, q, at::kBFloat16, "v_cache");
  typed(out, q, at::kBFloat16, "out");
  typed(block_tables, q, at::kInt, "block_tables");
  typed(ctx_len, q, at::kInt, "ctx_len");
  typed(shared, q, at::kInt, "shared");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128, "q must be [slots, Hq, 128]");
  TORCH_CHECK(out.sizes() == q.sizes(), "out must match q");
  const int64_t S = q.size(0), hq = q.size(1);
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(2) == dsse::kBS && k_cache.size(3) == 128 && k_cache.size(0) >= 1 && k_cache.size(0) < INT_MAX,
              "k_cache must be [blocks, Hkv, 32, 128]");
  const int64_t hkv = k_cache.size(1);
  TORCH_CHECK(v_cache.sizes() == at::IntArrayRef({k_cache.size(0), hkv, 128, dsse::kBS}), "v_cache must be [blocks, Hkv, 128, 32]");
  TORCH_CHECK(hkv >= 1 && hq >= 1 && hq % hkv == 0 && hq / hkv <= 16, "up to 16 q heads per key/value head, the same for each");
  const int groups = beams(S, width);
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == S && block_tables.size(1) >= 1 && block_tables.size(1) < (1 << 26),
              "block_tables must be [slots, max_blocks]");
  TORCH_CHECK(ctx_len.numel() == S && shared.numel() == groups, "ctx_len must be [slots], shared [groups]");
  TORCH_CHECK(S * hq <= dsse::kBeamRows, "at most ", dsse::kBeamRows, " slots times q heads");
  if (S == 0) return;
  TORCH_CHECK(aligned16(q.data_ptr()) && aligned16(k_cache.data_ptr()) && aligned16(v_cache.data_ptr()) && aligned16(out.data_ptr()),
              "q, caches and out must start at 16 bytes");
  const c10::DeviceGuard guard(q.device());
  dsse::BeamAttnParams p{};
  p.q = reinterpret_cast<const bf16*>(q.data_ptr());
  p.k_cache = reinterpret_cast<const bf16*>(k_cache.data_ptr());
  p.v_cache = reinterpret_cast<const bf16*>(v_cache.data_ptr());
  p.block_tables = block_tables.data_ptr<int>();
  p.ctx_len = ctx_len.data_ptr<int>();
  p.shared = shared.data_ptr<int>();
  p.out = reinterpret_cast<bf16*>(out.data_ptr());
  p.slots = (int)S, p.width = (int)width, p.hq = (int)hq, p.hkv = (int)hkv, p.group = (int)(hq / hkv);
  p.max_blocks = (int)block_tables.size(1), p.num_blocks = (int)k_cache.size(0);
  p.scale_log2 = 1.4426950408889634f / sqrtf(128.f);
  dsse_beam_plan(&p);
  const int64_t parts = S * hq * (p.ns + p.no);
  Tensor work = at::empty({parts * 130}, q.options().dtype(at::kFloat));
  p.part_o = work.data_ptr<float>();
  p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * 128);
  DSSE_CHECK_HIP(dsse_beam_attention(&p, stream_of(q)));
}

void beam_shared(const Tensor& block_tables, const Tensor& ctx_len, int64_t width, Tensor& shared) {
  typed(block_tables, block_tables, at::kInt, "block_tables");
  typed(ctx_len, block_tables, at::kInt, "ctx_len");
  typed(shared, block_tables, at::kInt, "shared");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(1) >= 1 && block_tables.size(1) < (1 << 26), "block_tables must be [slots, max_blocks]");
  TORCH_CHECK(block_tables.size(0) <= dsse::kSharedSlots, "at most ", dsse::kSharedSlots, " slots");
  const int groups = beams(block_tables.size(0), width);
  TORCH_CHECK(ctx_len.numel() == block_tables.size(0) && shared.numel() == groups, "ctx_len must be [slots], shared [groups]");
  if (groups == 0) return;
  const c10::DeviceGuard guard(block_tables.device());
  DSSE_CHECK_HIP(dsse_beam_shared(block_tables.data_ptr<int>(), ctx_len.data_ptr<int>(), shared.data_ptr<int>(), groups, (int)width,
                                  (int)block_tables.size(1), stream_of(block_tables)));
}

void page_fork(Tensor& block_tables, Tensor& held, Tensor& lens, const Tensor& parents, Tensor& refs, Tensor& copies, Tensor& starved,
               at::TensorList pools) {
  typed(block_tables, block_tables, at::kInt, "block_tables");
  typed(held, block_tables, at::kInt, "held");
  typed(lens, block_tables, at::kInt, "lens");
  typed(parents, block_tables, at::kInt, "parents");
  typed(refs, block_tables, at::kInt, "refs");
  typed(copies, block_tables, at::kInt, "copies");
  typed(starved, block_tables, at::kInt, "starved");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(1) >= 1 && block_tables.size(1) < (1 << 26), "block_tables must be [slots, max_blocks]");
  const int64_t S = block_tables.size(0), pages = refs.numel();
  TORCH_CHECK(S <= dsse::kForkSlots, "at most ", dsse::kForkSlots, " slots");
  TORCH_CHECK(held.numel() == S && lens.numel() == S && parents.numel() == S, "held, lens and parents must be [slots]");
  TORCH_CHECK(copies.dim() == 2 && copies.size(0) == S && copies.size(1) == 2 && starved.numel() == 1, "copies must be [slots, 2], starved [1]");
  TORCH_CHECK(pages >= 1 && pages < (1 << 30), "refs must have a count per page");
  int64_t pieces = 0;  // of a slot
  for (const Tensor& t : pools) {
    on(t, block_tables, "pool", false);
    TORCH_CHECK(t.dim() >= 3 && t.size(1) == pages, "a pool must be [layers, pages, ..]");
    if (t.numel() == 0) continue;
    TORCH_CHECK(packed(t, 1) && (t.size(0) == 1 || t.stride(0) >= t.numel() / t.size(0)), "a pool's pages must be contiguous");
    const int64_t bytes = t.numel() / t.size(0) / pages * t.element_size();
    TORCH_CHECK(bytes % 16 == 0 && aligned16(t.data_ptr()) && (t.size(0) == 1 || t.stride(0) * t.element_size() % 16 == 0),
                "a pool's pages must start and end at 16 bytes");
    TORCH_CHECK(bytes <= dsse::kCopyPage, "a page of a pool's layer is at most 1 GiB");  // 32-bit offsets
    pieces += t.size(0) * ((bytes + dsse::kCopyPiece - 1) / dsse::kCopyPiece);
    TORCH_CHECK(pieces <= dsse::kCopyPieces / std::max<int64_t>(S, 1), "pages of all slots, pools and layers are at most 2^31 - 1 pieces of 16 KiB");
  }
  if (S == 0) return;
  const c10::DeviceGuard guard(block_tables.device());
  const hipStream_t st = stream_of(block_tables);
  Tensor list = at::empty({S + 1}, block_tables.options());
  dsse::PageForkParams p{block_tables.data_ptr<int>(), held.data_ptr<int>(), lens.data_ptr<int>(), parents.data_ptr<int>(), refs.data_ptr<int>(),
                         copies.data_ptr<int>(), starved.data_ptr<int>(), list.data_ptr<int>(), (int)S, (int)block_tables.size(1), (int)pages};
  DSSE_CHECK_HIP(dsse_page_fork(&p, st));
  dsse::PageCopyParams c{};
  c.copies = p.copies, c.list = p.list, c.slots = p.slots;
  for (size_t i = 0; i < pools.size(); ++i) {
    const Tensor& t = pools[i];
    if (t.numel() > 0)
      c.pool[c.npools++] = {reinterpret_cast<char*>(t.data_ptr()), t.size(0) == 1 ? 0 : t.stride(0) * (int64_t)t.element_size(), (int)t.size(0),
                            (int)(t.numel() / t.size(0) / pages * t.element_size()), 0, 0};
    if (c.npools == dsse::kCopyPools || (i + 1 == pools.size() && c.npools > 0)) {
      DSSE_CHECK_HIP(dsse_page_copy(&c, st));
      c.npools = 0;
    }
  }
}

void state_reorder(at::TensorList states, const Tensor& parents, int64_t width) {
  typed(parents, parents, at::kInt, "parents");
  const int64_t S = parents.numel();
  const int groups = beams(S, width);
  TORCH_CHECK(groups <= 65535, "at most 65535 groups");
  int64_t bytes = 0;
  for (const Tensor& t : states) {
    on(t, parents, "state", false);
    TORCH_CHECK(t.dim() >= 1 && t.size(0) == S, "a state must be [slots, ..]");
    if (t.numel() == 0) continue;
    const int64_t row = t.numel() / S;
    TORCH_CHECK(packed(t, 1) && (S == 1 || t.stride(0) >= row), "a slot's state must be contiguous");
    TORCH_CHECK(row * t.element_size() % 2 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 2 == 0 &&
                    (S == 1 || t.stride(0) * t.element_size() % 2 == 0) && row * t.element_size() < INT_MAX - (1 << 16),
                "a slot's state must have an even number of bytes, under 2 GiB");
    bytes += row * t.element_size();
    for (const Tensor& u : states) TORCH_CHECK(&u == &t || u.data_ptr() != t.data_ptr() || u.numel() == 0, "a state is listed twice");
  }
  TORCH_CHECK(bytes <= dsse::kReorderBytes, "at most 32 GiB of a slot in all");
  if (S == 0) return;
  const c10::DeviceGuard guard(parents.device());
  const hipStream_t st = stream_of(parents);
  dsse::StateReorderParams p{};
  p.parents = parents.data_ptr<int>(), p.slots = (int)S, p.width = (int)width;
  for (size_t i = 0; i < states.size(); ++i) {
    const Tensor& t = states[i];
    if (t.numel() > 0)
      p.t[p.ntensors++] = {reinterpret_cast<char*>(t.data_ptr()), S == 1 ? 0 : t.stride(0) * (int64_t)t.element_size(),
                           (int)(t.numel() / S * t.element_size()), 0};
    if (p.ntensors == dsse::kReorderLists || (i + 1 == states.size() && p.ntensors > 0)) {
      DSSE_CHECK_HIP(dsse_state_reorder(&p, st));
      p.ntensors = 0;
    }
  }
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dsse, m) {
  m.def("beam_select(Tensor logits, Tensor scores, Tensor(a!) out_scores, Tensor(b!) out_rows, Tensor(c!) out_tokens, int eos_id=-1, "
        "Tensor(d!)? end_scores=None) -> ()");
  m.def("beam_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor ctx_len, Tensor shared, Tensor(a!) out, "
        "int width) -> ()");
  m.def("beam_shared(Tensor block_tables, Tensor ctx_len, int width, Tensor(a!) shared) -> ()");
  m.def("page_fork(Tensor(a!) block_tables, Tensor(b!) held, Tensor(c!) lens, Tensor parents, Tensor(d!) refs, Tensor(e!) copies, "
        "Tensor(f!) starved, Tensor(g!)[] pools) -> ()");
  m.def("state_reorder(Tensor(a!)[] states, Tensor parents, int width) -> ()");
}

TORCH_LIBRARY_IMPL(dsse, CUDA, m) {
  m.impl("beam_select", &beam_select);
  m.impl("beam_attention", &beam_attention);
  m.impl("beam_shared", &beam_shared);
  m.impl("page_fork", &page_fork);
  m.impl("state_reorder", &state_reorder);
}
