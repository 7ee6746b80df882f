// Host-visible API of the kernels of a beam search over the paged cache: selection over beams and vocabulary, attention of
// beams that share pages, forks of block tables with the copies of half-written pages, states that change slots.
//
// A request is a group of `width` neighbouring slots: slot g * width + w is beam w of group g.
#pragma once
#include "api.h"

namespace dsse {

constexpr int kBeamWidth = 32;  // beams of a group
constexpr int kBeamKeep = 64;   // candidates of a group
constexpr int kForkSlots = 2048;
constexpr int kSharedSlots = (1 << 26) - 1;  // slots whose common pages are counted: a grid's threads, 64 a group, stay in 32 bits
constexpr int kReorderLists = 96;  // tensors of one launch (24 bytes each of a kernel's arguments)
constexpr int kCopyPools = 64;     // (32 bytes each)
constexpr int kCopyPage = 1 << 30;     // bytes of a page in a layer: offsets past its end, of whole work items, stay in 32 bits
constexpr int kCopyPiece = 1 << 14;    // bytes of a page that a workgroup copies at a time
constexpr int kCopyPieces = 0x7fffffff;  // pieces of a fork's slots over all pools and layers: a launch counts them in 32 bits
constexpr int kBeamRows = 1 << 22;     // (slot, q head) pairs of an attention: a grid's threads stay in 32 bits
constexpr int64_t kReorderBytes = int64_t{1} << 35;  // bytes of a slot over all tensors: so do those of a launch

struct BeamSelectParams {
  const void* logits;   // [rows, V] rows ld apart
  const float* scores;  // [rows]
  float* out_scores;    // [groups, K]
  int* out_rows;        // [groups, K] absolute rows, -1 where nothing is left
  int* out_tokens;      // [groups, K]
  float* end_scores;    // [rows] or null
  double* sum;          // [rows, chunks] sum of exponentials about the maximum
  float* most;          // [rows, chunks] maximum
  float2* cand;         // [rows, chunks, K] logit, token (bits); best first
  float* end_logit;     // [rows]
  int64_t ld;
  int rows, width, V, K, eos, pieces, chunks, f32;  // pieces of 16 bytes per thread; workgroups of a row
};

struct BeamAttnParams {
  const bf16* q;            // [slots, hq, 128]
  const bf16* k_cache;      // [blocks, hkv, kBS, 128]
  const bf16* v_cache;      // [blocks, hkv, 128, kBS] (token-permuted inside a page)
  const int* block_tables;  // [slots, max_blocks]
  const int* ctx_len;       // [slots], 0 = idle
  const int* shared;        // [groups] leading pages that the group's tables have in common
  bf16* out;                // [slots, hq, 128]
  float* part_o;            // [slots, hq, ns + no, 128]
  float2* part_ml;          // [slots, hq, ns + no] running maximum (log2 units), sum
  int slots, width, hq, hkv, group, max_blocks, num_blocks, ns, no, tiles, col_blocks;
  float scale_log2;
};

struct PageForkParams {
  int* tables;         // [slots, max_blocks]
  int* held;           // [slots] pages of each slot
  int* lens;           // [slots] tokens of each slot
  const int* parents;  // [slots]
  int* refs;           // [pages] holders of each page
  int* copies;         // [slots, 2] source, destination; -1 without a copy
  int* starved;        // [1] slots that found no free page
  int* list;           // [1 + slots] how many slots copy, which
  int slots, max_blocks, pages;
};

struct PageCopyParams {
  const int* copies;  // [slots, 2]
  const int* list;    // [1 + slots]
  int slots, npools, blocks;  // blocks: of a slot, over all pools
  struct Pool {
    char* base;
    int64_t layer;      // bytes from a layer to the next
    int layers, bytes;  // bytes of a page
    int per, first;     // workgroups of a layer's page, the pool's first one (set by the launcher)
  } pool[kCopyPools];
};

struct StateReorderParams {
  const int* parents;  // [slots]
  int slots, width, ntensors;
  struct List {
    char* base;
    int64_t stride;  // bytes from a slot to the next
    int bytes;       // of a slot
    int first;       // first workgroup (in x) of this tensor
  } t[kReorderLists];
};

}  // namespace dsse

extern "C" {
void dsse_beam_plan_rows(dsse::BeamSelectParams* p);  // pieces and chunks of the other fields
hipError_t dsse_beam_select(const dsse::BeamSelectParams* p, hipStream_t st);
void dsse_beam_plan(dsse::BeamAttnParams* p);  // tiles, col_blocks, ns, no of the other fields
hipError_t dsse_beam_attention(const dsse::BeamAttnParams* p, hipStream_t st);
hipError_t dsse_beam_shared(const int* tables, const int* ctx_len, int* shared, int groups, int width, int max_blocks, hipStream_t st);
hipError_t dsse_page_fork(const dsse::PageForkParams* p, hipStream_t st);
hipError_t dsse_page_copy(const dsse::PageCopyParams* p, hipStream_t st);
hipError_t dsse_state_reorder(const dsse::StateReorderParams* p, hipStream_t st);
}
