// Encoders of the attention sub-layer: view checks, then the C ABI entries.
#include "tokspur_b200/attention.hpp"

namespace tokspur_b200 {
namespace {
void check(int rc) { if (rc != TSP_OK) throw FormatError(tsp_last_error()); }

void require_rows(const GpuRowsF32& r, uint32_t rows, uint64_t columns, const char* what) {
    if (!rows || r.rows < rows || r.columns != columns || r.stride_bytes % 16 || r.stride_bytes < columns * 4 ||
        r.view.bytes < (rows - 1) * r.stride_bytes + columns * 4)
        throw FormatError(std::string(what) + " rows shape mismatch");
}

tsp_kv_cache cache_of(const CudaGraph& g, const KvCache& c, bool for_write) {
    const uint64_t page = tsp_kv_page_bytes(c.shape.type, c.shape.page_tokens, c.shape.kv_heads, c.shape.head_dim);
    if (!page || !c.page_count || c.pages.bytes != page * c.page_count || c.page_table.bytes != uint64_t(c.sequences) * c.pages_per_sequence * 4)
        throw FormatError("kv cache shape mismatch");
    tsp_kv_cache k{};
    k.d_pages = g.device_pointer(c.pages, for_write);
    k.page_stride_bytes = page;
    k.d_page_table = static_cast<const uint32_t*>(g.device_pointer(c.page_table));
    k.table_stride = c.pages_per_sequence;
    k.pages = c.page_count;
    k.page_tokens = c.shape.page_tokens;
    k.kv_heads = c.shape.kv_heads;
    k.head_dim = c.shape.head_dim;
    k.type = c.shape.type;
    return k;
}

tsp_kv_batch step_of(const CudaGraph& g, const KvCache& c, const KvStep& s) {
    const uint64_t sequences = s.lengths.bytes / 4;
    if (!sequences || s.lengths.bytes % 4 || sequences > c.sequences || s.row_offsets.bytes != (sequences + 1) * 4) throw FormatError("kv step shape mismatch");
    return {static_cast<const uint32_t*>(g.device_pointer(s.row_offsets)), static_cast<const uint32_t*>(g.device_pointer(s.lengths)), uint32_t(sequences), s.rows};
}

const float* weight(const CudaGraph& g, GpuView v, uint64_t values, const char* what) {
    if (!v.bytes) return nullptr;
    if (v.bytes != values * 4) throw FormatError(std::string(what) + " shape mismatch");
    return static_cast<const float*>(g.device_pointer(v));
}
}  // namespace

KvCache allocate_kv_cache(CudaGraph& g, KvShape shape, uint32_t sequences, uint32_t pages, uint32_t pages_per_sequence) {
    const uint64_t page = tsp_kv_page_bytes(shape.type, shape.page_tokens, shape.kv_heads, shape.head_dim);
    if (!page || !sequences || !pages || !pages_per_sequence) throw FormatError("kv cache shape without a kernel");
    KvCache c;
    c.shape = shape;
    c.sequences = sequences; c.page_count = pages; c.pages_per_sequence = pages_per_sequence;
    c.pages = g.zeros(page * pages, "kv cache pages");
    c.page_table = g.zeros(uint64_t(sequences) * pages_per_sequence * 4, "kv cache page table");
    return c;
}
void release_kv_cache(CudaGraph& g, const KvCache& c) { g.release(c.pages); g.release(c.page_table); }

AttentionScratch allocate_attention_scratch(CudaGraph& g) { return {g.zeros(tsp_tree_attention_scratch_bytes(), "attention scratch")}; }
void release_attention_scratch(CudaGraph& g, const AttentionScratch& s) { g.release(s.join); }

void encode_verify_attention(CudaGraph& g, const AttentionWeights& w, const KvCache& cache, const KvStep& step, const AttentionScratch& scratch, GpuRowsF32 q, GpuRowsF32 k,
                             GpuRowsF32 v, GpuView positions, GpuView tree, uint32_t most_rows, float scale, GpuRowsF32 out) {
    g.require_batch();
    const uint32_t dim = cache.shape.head_dim, rows = step.rows;
    if (!dim || q.columns % dim) throw FormatError("query rows shape mismatch");
    require_rows(q, rows, q.columns, "query");
    require_rows(out, rows, q.columns, "attention output");
    require_rows(k, rows, uint64_t(cache.shape.kv_heads) * dim, "key");
    require_rows(v, rows, uint64_t(cache.shape.kv_heads) * dim, "value");
    if (positions.bytes < uint64_t(rows) * 4) throw FormatError("fewer positions than rows");
    if (tree.bytes && tree.bytes < uint64_t(rows) * 8) throw FormatError("fewer tree words than rows");
    const tsp_kv_cache kc = cache_of(g, cache, true);
    const tsp_kv_batch kb = step_of(g, cache, step);
    const tsp_qk_norm_rope_args a{weight(g, w.q_norm, dim, "query norm"), weight(g, w.k_norm, dim, "key norm"), weight(g, w.inv_freq, w.rotary_dim / 2, "frequencies"),
                                  dim, w.rotary_dim, w.pairs ? TSP_ROPE_PAIRS : TSP_ROPE_HALVES, w.eps, w.magnitude};
    const uint32_t q_heads = q.columns / dim;
    void *qp = g.device_pointer(q.view, true), *op = g.device_pointer(out.view, true), *sp = g.device_pointer(scratch.join, true);
    const void *kp = g.device_pointer(k.view), *vp = g.device_pointer(v.view);
    const auto* words = tree.bytes ? static_cast<const uint64_t*>(g.device_pointer(tree)) : nullptr;
    // what the second launch would refuse is refused before the first, which turns the query rows in place
    check(tsp_tree_attention_check(&kc, &kb, qp, q.stride_bytes, words, q_heads, most_rows, scale, op, out.stride_bytes, 0, sp, scratch.join.bytes));
    check(tsp_qk_norm_rope_append(&a, &kc, &kb, qp, q.stride_bytes, kp, k.stride_bytes, vp, v.stride_bytes, 0, static_cast<const uint32_t*>(g.device_pointer(positions)), q_heads, qp,
                                  q.stride_bytes, 0, g.error_word(), g.stream()));
    check(tsp_tree_attention(&kc, &kb, qp, q.stride_bytes, words, q_heads, most_rows, scale, op, out.stride_bytes, 0, sp, scratch.join.bytes, g.error_word(), g.stream()));
    g.count_dispatches(verify_attention_dispatches());
}

void encode_kv_keep(CudaGraph& g, const KvCache& cache, const KvStep& step, GpuView accepted, GpuView counts) {
    g.require_batch();
    const tsp_kv_cache kc = cache_of(g, cache, true);
    const tsp_kv_batch kb = step_of(g, cache, step);
    if (accepted.bytes < uint64_t(step.rows) * 4 || counts.bytes < uint64_t(kb.sequences) * 4) throw FormatError("accepted indices or counts too short");
    check(tsp_kv_cache_keep(&kc, &kb, static_cast<const uint32_t*>(g.device_pointer(accepted)), static_cast<const uint32_t*>(g.device_pointer(counts)), g.error_word(), g.stream()));
    g.count_dispatches(1);
}

void encode_kv_append(CudaGraph& g, const KvCache& cache, const KvStep& step, GpuRowsF32 k, GpuRowsF32 v) {
    g.require_batch();
    const uint64_t columns = uint64_t(cache.shape.kv_heads) * cache.shape.head_dim;
    require_rows(k, step.rows, columns, "key");
    require_rows(v, step.rows, columns, "value");
    const tsp_kv_cache kc = cache_of(g, cache, true);
    const tsp_kv_batch kb = step_of(g, cache, step);
    check(tsp_kv_cache_append(&kc, &kb, g.device_pointer(k.view), k.stride_bytes, g.device_pointer(v.view), v.stride_bytes, 0, g.error_word(), g.stream()));
    g.count_dispatches(1);
}

void encode_kv_read(CudaGraph& g, const KvCache& cache, const KvStep& step, GpuRowsF32 k, GpuRowsF32 v) {
    g.require_batch();
    const uint64_t columns = uint64_t(cache.shape.kv_heads) * cache.shape.head_dim;
    require_rows(k, step.rows, columns, "key");
    require_rows(v, step.rows, columns, "value");
    const tsp_kv_cache kc = cache_of(g, cache, false);
    const tsp_kv_batch kb = step_of(g, cache, step);
    check(tsp_kv_cache_read(&kc, &kb, g.device_pointer(k.view, true), k.stride_bytes, g.device_pointer(v.view, true), v.stride_bytes, 0, g.error_word(), g.stream()));
    g.count_dispatches(1);
}

}  // namespace tokspur_b200
