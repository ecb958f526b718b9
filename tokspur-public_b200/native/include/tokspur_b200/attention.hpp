// Attention sub-layer of a verify / decode step, the half of a layer that stands before encode_moe / encode_verify_nax_moe on the same rows:
// head norm and rotation, the paged key / value cache, attention of the drafted tokens. The encoders have the batch rules of the MoE encoders: nothing
// is allocated or read back inside a batch, host-side mismatches throw FormatError before anything is launched.
#pragma once

#include "tokspur_b200/graph.hpp"

namespace tokspur_b200 {

struct KvShape { uint32_t kv_heads, head_dim, page_tokens, type; };   // type: TSP_TYPE_Q8_0 or TSP_TYPE_F16
// The page table is the host's: u32 [sequences x pages_per_sequence], written between batches with CudaGraph::write.
struct KvCache {
    GpuView pages, page_table;
    KvShape shape{};
    uint32_t sequences = 0, page_count = 0, pages_per_sequence = 0;
};
// The rows of one step (tsp_kv_batch): u32 row_offsets [sequences + 1], u32 lengths [sequences], and how many rows the buffers hold.
struct KvStep { GpuView row_offsets, lengths; uint32_t rows = 0; };
// FP32 weights; a view of no bytes: no norm / no rotation
struct AttentionWeights {
    GpuView q_norm, k_norm, inv_freq;
    uint32_t rotary_dim = 0;
    bool pairs = false;        // rotation of neighbouring dims instead of halves
    float eps = 1e-6f, magnitude = 1.f;
};
struct AttentionScratch { GpuView join; };

[[nodiscard]] KvCache allocate_kv_cache(CudaGraph& graph, KvShape shape, uint32_t sequences, uint32_t pages, uint32_t pages_per_sequence);
void release_kv_cache(CudaGraph& graph, const KvCache& cache);
[[nodiscard]] AttentionScratch allocate_attention_scratch(CudaGraph& graph);
void release_attention_scratch(CudaGraph& graph, const AttentionScratch& scratch);

// Norm and rotation of q in place, of k on its way into the cache beside v, then the attention of every row over its sequence's context and the step's own
// tokens (`tree`: u64 words as tsp_tree_attention has them; a view of no bytes: a chain). q, out: rows of q_heads * head_dim values; k, v: of
// kv_heads * head_dim. most_rows: the most rows of a sequence in the step, 1 .. 64. Two launches.
void encode_verify_attention(CudaGraph& graph, const AttentionWeights& weights, const KvCache& cache, const KvStep& step, const AttentionScratch& scratch, GpuRowsF32 q,
                             GpuRowsF32 k, GpuRowsF32 v, GpuView positions, GpuView tree, uint32_t most_rows, float scale, GpuRowsF32 out);
inline uint32_t verify_attention_dispatches() { return 2; }
// After the verify: the accepted tokens' slots to the front of the step's (tsp_kv_cache_keep). accepted: u32 [rows], counts: u32 [sequences]
void encode_kv_keep(CudaGraph& graph, const KvCache& cache, const KvStep& step, GpuView accepted, GpuView counts);
// Rows into the step's slots as they are (prompt rows that were normed elsewhere), and the slots back as FP32 rows
void encode_kv_append(CudaGraph& graph, const KvCache& cache, const KvStep& step, GpuRowsF32 k, GpuRowsF32 v);
void encode_kv_read(CudaGraph& graph, const KvCache& cache, const KvStep& step, GpuRowsF32 k, GpuRowsF32 v);

}  // namespace tokspur_b200
