// C ABI of the attention operators: argument validation (refused before any launch), then the launches.
#include <cmath>
#include <initializer_list>

#include "tsp_kv.cuh"

namespace tsp {

int launch_head_rows(const tsp_qk_norm_rope_args&, const void*, uint64_t, const void*, uint64_t, const void*, uint64_t, uint32_t, const uint32_t*, uint32_t, uint32_t,
                     uint32_t, void*, uint64_t, void*, uint64_t, uint32_t, const tsp_kv_cache*, const tsp_kv_batch*, uint32_t*, cudaStream_t);
int launch_cache_read(const tsp_kv_cache&, const tsp_kv_batch&, void*, uint64_t, void*, uint64_t, uint32_t, uint32_t*, cudaStream_t);
int launch_cache_keep(const tsp_kv_cache&, const tsp_kv_batch&, const uint32_t*, const uint32_t*, uint32_t*, cudaStream_t);
int launch_tree_attention(const tsp_kv_cache&, const tsp_kv_batch&, const void*, uint64_t, const uint64_t*, uint32_t, uint32_t, float, void*, uint64_t, uint32_t, void*,
                          uint32_t*, cudaStream_t);
uint64_t tree_attention_scratch_bytes();

static bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

static int check_cache(const tsp_kv_cache* c, const tsp_kv_batch* b) {
    TSP_REQUIRE(c && b, "kv cache: null cache or batch");
    if (c->type != TSP_TYPE_Q8_0 && c->type != TSP_TYPE_F16) return fail(TSP_E_TYPE, "kv cache: encoding %u has no kernel", c->type);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return fail(TSP_E_TYPE, "kv cache: head_dim %u has no kernel", c->head_dim);
    TSP_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 256, "kv cache: kv_heads out of range");
    TSP_REQUIRE(c->page_tokens >= 16 && c->page_tokens <= 256 && (c->page_tokens & (c->page_tokens - 1)) == 0, "kv cache: page_tokens must be 16, 32, 64, 128 or 256");
    TSP_REQUIRE(c->d_pages && aligned16(c->d_pages) && c->d_page_table && aligned4(c->d_page_table), "kv cache: null or unaligned pages or page table");
    TSP_REQUIRE(c->page_stride_bytes % 16 == 0 && c->page_stride_bytes >= tsp_kv_page_bytes(c->type, c->page_tokens, c->kv_heads, c->head_dim) &&
                c->page_stride_bytes <= (1ull << 40), "kv cache: page stride must cover a page and be a multiple of 16");
    TSP_REQUIRE(c->pages >= 1 && c->pages < (1u << 31) && c->table_stride >= 1 && static_cast<uint64_t>(c->table_stride) * c->page_tokens < (1u << 31),
                "kv cache: pages or table stride out of range");
    TSP_REQUIRE(b->d_row_offsets && b->d_lengths && aligned4(b->d_row_offsets) && aligned4(b->d_lengths), "kv batch: null or unaligned offsets or lengths");
    TSP_REQUIRE(b->sequences >= 1 && b->sequences <= TSP_KV_MAX_SEQUENCES && b->rows >= 1 && b->rows <= (1u << 20), "kv batch: sequences or rows out of range");
    return TSP_OK;
}

static int check_head_rows(const void* p, uint64_t stride, uint32_t heads, uint32_t dim, uint32_t dtype, const char* name) {
    TSP_REQUIRE(dtype <= 1, "%s: dtype must be 0 (FP32) or 1 (binary16)", name);
    TSP_REQUIRE(heads >= 1 && heads <= 4096, "%s: heads out of range", name);
    TSP_REQUIRE(p && aligned16(p), "%s: rows must be 16-byte aligned", name);
    TSP_REQUIRE(stride >= static_cast<uint64_t>(heads) * dim * (dtype ? 2 : 4) && stride % 16 == 0 && stride <= (1ull << 32), "%s: row stride must cover the row and be a multiple of 16",
                name);
    return TSP_OK;
}

static int check_turn(const tsp_qk_norm_rope_args* a) {
    TSP_REQUIRE(a != nullptr, "norm and rotation: null arguments");
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return fail(TSP_E_TYPE, "norm and rotation: head_dim %u has no kernel", a->head_dim);
    TSP_REQUIRE(a->rotary_dim % 8 == 0 && a->rotary_dim <= a->head_dim, "norm and rotation: rotary_dim must be a multiple of 8 within the head");
    TSP_REQUIRE(a->style == TSP_ROPE_HALVES || a->style == TSP_ROPE_PAIRS, "norm and rotation: unknown pairing");
    TSP_REQUIRE(a->eps >= 0.f && std::isfinite(a->eps) && std::isfinite(a->magnitude), "norm and rotation: eps or magnitude out of range");
    TSP_REQUIRE(a->rotary_dim == 0 || a->d_inv_freq, "norm and rotation: no frequencies");
    TSP_REQUIRE(aligned4(a->d_inv_freq) && aligned16(a->d_q_norm) && aligned16(a->d_k_norm), "norm and rotation: unaligned weights or frequencies");
    return TSP_OK;
}

struct Rows { const void* p; uint64_t stride, bytes; };
static bool meet(const Rows& a, const Rows& b, uint64_t rows) { return a.p && b.p && rows_overlap(a.p, a.stride, a.bytes, b.p, b.stride, b.bytes, rows); }
static uint64_t pool_bytes(const tsp_kv_cache& c) {
    return (c.pages - 1) * c.page_stride_bytes + tsp_kv_page_bytes(c.type, c.page_tokens, c.kv_heads, c.head_dim);
}
// Arrays that a kernel reads, some of them again and again, while its other blocks write rows or pages
struct Array { const void* p; uint64_t bytes; };
static bool over(const Rows& w, uint64_t rows, std::initializer_list<Array> read) {
    for (const Array& a : read) {
        if (!w.p || !a.p || !a.bytes || !overlap(w.p, (rows - 1) * w.stride + w.bytes, a.p, a.bytes)) continue;
        const uintptr_t x = reinterpret_cast<uintptr_t>(w.p), y = reinterpret_cast<uintptr_t>(a.p);
        if (y < x) return true;
        const uint64_t in = (y - x) % w.stride;   // an array may lie between two rows
        if (in < w.bytes || in + a.bytes > w.stride) return true;
    }
    return false;
}
static bool over_step(const Rows& w, uint64_t rows, const tsp_kv_cache& c, const tsp_kv_batch& b) {
    return over(w, rows, {{b.d_row_offsets, (b.sequences + 1) * 4ull}, {b.d_lengths, b.sequences * 4ull}, {c.d_page_table, static_cast<uint64_t>(b.sequences) * c.table_stride * 4}});
}
static bool over_turn(const Rows& w, uint64_t rows, const tsp_qk_norm_rope_args& a, const uint32_t* positions, uint64_t tokens) {
    return over(w, rows, {{positions, a.rotary_dim ? tokens * 4 : 0}, {a.d_q_norm, a.head_dim * 4ull}, {a.d_k_norm, a.head_dim * 4ull}, {a.d_inv_freq, a.rotary_dim / 2 * 4ull}});
}
static Rows pool(const tsp_kv_cache& c) { return {c.d_pages, c.page_stride_bytes, tsp_kv_page_bytes(c.type, c.page_tokens, c.kv_heads, c.head_dim)}; }
static bool meets_pages(const Rows& a, const tsp_kv_cache& c, uint64_t rows) {
    return a.p && overlap(a.p, (rows - 1) * a.stride + a.bytes, c.d_pages, pool_bytes(c));
}

}  // namespace tsp

using namespace tsp;

extern "C" {

uint64_t tsp_kv_page_bytes(uint32_t type, uint32_t page_tokens, uint32_t kv_heads, uint32_t head_dim) {
    if ((type != TSP_TYPE_Q8_0 && type != TSP_TYPE_F16) || (head_dim != 64 && head_dim != 128 && head_dim != 256) || page_tokens < 16 || page_tokens > 256 ||
        (page_tokens & (page_tokens - 1)) || !kv_heads || kv_heads > 256)
        return 0;
    return static_cast<uint64_t>(kv_heads) * (page_tokens / kKvGroup) * kv_group_bytes(head_dim, type == TSP_TYPE_Q8_0);
}

int tsp_qk_norm_rope(const tsp_qk_norm_rope_args* a, const void* d_q, uint64_t q_stride, const void* d_k, uint64_t k_stride, uint32_t in_dtype,
                     const uint32_t* d_positions, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, void* d_q_out, uint64_t q_out_stride, void* d_k_out,
                     uint64_t k_out_stride, uint32_t out_dtype, uint32_t* d_error, void* stream) {
    if (int rc = check_turn(a)) return rc;
    TSP_REQUIRE(rows >= 1 && rows <= (1u << 20) && q_heads + static_cast<uint64_t>(kv_heads) >= 1, "norm and rotation: rows or heads out of range");
    TSP_REQUIRE(a->rotary_dim == 0 || (d_positions && aligned4(d_positions)), "norm and rotation: null or unaligned positions");
    const uint32_t in = in_dtype ? 2 : 4, out = out_dtype ? 2 : 4, dim = a->head_dim;
    if (q_heads) {
        if (int rc = check_head_rows(d_q, q_stride, q_heads, dim, in_dtype, "q")) return rc;
        if (int rc = check_head_rows(d_q_out, q_out_stride, q_heads, dim, out_dtype, "q out")) return rc;
    }
    if (kv_heads) {
        if (int rc = check_head_rows(d_k, k_stride, kv_heads, dim, in_dtype, "k")) return rc;
        if (int rc = check_head_rows(d_k_out, k_out_stride, kv_heads, dim, out_dtype, "k out")) return rc;
    }
    const Rows q{q_heads ? d_q : nullptr, q_stride, static_cast<uint64_t>(q_heads) * dim * in}, k{kv_heads ? d_k : nullptr, k_stride, static_cast<uint64_t>(kv_heads) * dim * in};
    const Rows qo{q_heads ? d_q_out : nullptr, q_out_stride, static_cast<uint64_t>(q_heads) * dim * out}, ko{kv_heads ? d_k_out : nullptr, k_out_stride, static_cast<uint64_t>(kv_heads) * dim * out};
    const bool q_in_place = qo.p == q.p && q_stride == q_out_stride && in == out, k_in_place = ko.p == k.p && k_stride == k_out_stride && in == out;
    TSP_REQUIRE((q_in_place || !meet(qo, q, rows)) && (k_in_place || !meet(ko, k, rows)) && !meet(qo, k, rows) && !meet(ko, q, rows) && !meet(qo, ko, rows),
                "norm and rotation: output rows overlap other rows");
    TSP_REQUIRE(!over_turn(qo, rows, *a, d_positions, rows) && !over_turn(ko, rows, *a, d_positions, rows), "norm and rotation: output rows overlap positions, weights or frequencies");
    return launch_head_rows(*a, d_q, q_stride, d_k, k_stride, nullptr, 0, in_dtype, d_positions, rows, q_heads, kv_heads, d_q_out, q_out_stride, d_k_out, k_out_stride,
                            out_dtype, nullptr, nullptr, d_error, static_cast<cudaStream_t>(stream));
}

int tsp_qk_norm_rope_append(const tsp_qk_norm_rope_args* a, const tsp_kv_cache* cache, const tsp_kv_batch* batch, const void* d_q, uint64_t q_stride,
                            const void* d_k, uint64_t k_stride, const void* d_v, uint64_t v_stride, uint32_t in_dtype, const uint32_t* d_positions, uint32_t q_heads,
                            void* d_q_out, uint64_t q_out_stride, uint32_t out_dtype, uint32_t* d_error, void* stream) {
    if (int rc = check_turn(a)) return rc;
    if (int rc = check_cache(cache, batch)) return rc;
    TSP_REQUIRE(a->head_dim == cache->head_dim, "norm and rotation: head_dim differs from the cache's");
    TSP_REQUIRE(a->rotary_dim == 0 || (d_positions && aligned4(d_positions)), "norm and rotation: null or unaligned positions");
    const uint32_t in = in_dtype ? 2 : 4, out = out_dtype ? 2 : 4, dim = a->head_dim, rows = batch->rows;
    if (int rc = check_head_rows(d_q, q_stride, q_heads, dim, in_dtype, "q")) return rc;
    if (int rc = check_head_rows(d_q_out, q_out_stride, q_heads, dim, out_dtype, "q out")) return rc;
    if (int rc = check_head_rows(d_k, k_stride, cache->kv_heads, dim, in_dtype, "k")) return rc;
    if (int rc = check_head_rows(d_v, v_stride, cache->kv_heads, dim, in_dtype, "v")) return rc;
    const uint64_t kv_bytes = static_cast<uint64_t>(cache->kv_heads) * dim * in;
    const Rows q{d_q, q_stride, static_cast<uint64_t>(q_heads) * dim * in}, k{d_k, k_stride, kv_bytes}, v{d_v, v_stride, kv_bytes};
    const Rows qo{d_q_out, q_out_stride, static_cast<uint64_t>(q_heads) * dim * out};
    const bool in_place = qo.p == q.p && q_stride == q_out_stride && in == out;
    TSP_REQUIRE((in_place || !meet(qo, q, rows)) && !meet(qo, k, rows) && !meet(qo, v, rows), "norm and rotation: output rows overlap other rows");
    TSP_REQUIRE(!meets_pages(q, *cache, rows) && !meets_pages(k, *cache, rows) && !meets_pages(v, *cache, rows) && !meets_pages(qo, *cache, rows), "kv cache: rows overlap the pages");
    TSP_REQUIRE(!over_turn(qo, rows, *a, d_positions, rows) && !over_step(qo, rows, *cache, *batch) && !over_turn(pool(*cache), cache->pages, *a, d_positions, rows) &&
                !over_step(pool(*cache), cache->pages, *cache, *batch), "kv cache: output rows or pages overlap the arrays that describe the step");
    return launch_head_rows(*a, d_q, q_stride, d_k, k_stride, d_v, v_stride, in_dtype, d_positions, rows, q_heads, 0, d_q_out, q_out_stride, nullptr, 0, out_dtype, cache,
                            batch, d_error, static_cast<cudaStream_t>(stream));
}

int tsp_kv_cache_append(const tsp_kv_cache* cache, const tsp_kv_batch* batch, const void* d_k, uint64_t k_stride, const void* d_v, uint64_t v_stride, uint32_t dtype,
                        uint32_t* d_error, void* stream) {
    if (int rc = check_cache(cache, batch)) return rc;
    if (int rc = check_head_rows(d_k, k_stride, cache->kv_heads, cache->head_dim, dtype, "k")) return rc;
    if (int rc = check_head_rows(d_v, v_stride, cache->kv_heads, cache->head_dim, dtype, "v")) return rc;
    const uint64_t bytes = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim * (dtype ? 2 : 4);
    TSP_REQUIRE(!meets_pages({d_k, k_stride, bytes}, *cache, batch->rows) && !meets_pages({d_v, v_stride, bytes}, *cache, batch->rows), "kv cache: rows overlap the pages");
    TSP_REQUIRE(!over_step(pool(*cache), cache->pages, *cache, *batch), "kv cache: the pages overlap the arrays that describe the step");
    tsp_qk_norm_rope_args a = {};
    a.head_dim = cache->head_dim;
    a.magnitude = 1.f;
    return launch_head_rows(a, nullptr, 0, d_k, k_stride, d_v, v_stride, dtype, nullptr, batch->rows, 0, 0, nullptr, 0, nullptr, 0, dtype, cache, batch, d_error,
                            static_cast<cudaStream_t>(stream));
}

int tsp_kv_cache_read(const tsp_kv_cache* cache, const tsp_kv_batch* batch, void* d_k, uint64_t k_stride, void* d_v, uint64_t v_stride, uint32_t dtype, uint32_t* d_error,
                      void* stream) {
    if (int rc = check_cache(cache, batch)) return rc;
    TSP_REQUIRE(d_k || d_v, "kv cache: no rows to read into");
    if (d_k) if (int rc = check_head_rows(d_k, k_stride, cache->kv_heads, cache->head_dim, dtype, "k")) return rc;
    if (d_v) if (int rc = check_head_rows(d_v, v_stride, cache->kv_heads, cache->head_dim, dtype, "v")) return rc;
    const uint64_t bytes = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim * (dtype ? 2 : 4);
    const Rows k{d_k, k_stride, bytes}, v{d_v, v_stride, bytes};
    TSP_REQUIRE(!meet(k, v, batch->rows) && !meets_pages(k, *cache, batch->rows) && !meets_pages(v, *cache, batch->rows), "kv cache: output rows overlap each other or the pages");
    TSP_REQUIRE(!over_step(k, batch->rows, *cache, *batch) && !over_step(v, batch->rows, *cache, *batch), "kv cache: output rows overlap the arrays that describe the step");
    return launch_cache_read(*cache, *batch, d_k, k_stride, d_v, v_stride, dtype, d_error, static_cast<cudaStream_t>(stream));
}

int tsp_kv_cache_keep(const tsp_kv_cache* cache, const tsp_kv_batch* batch, const uint32_t* d_accepted, const uint32_t* d_counts, uint32_t* d_error, void* stream) {
    if (int rc = check_cache(cache, batch)) return rc;
    TSP_REQUIRE(d_accepted && d_counts && aligned4(d_accepted) && aligned4(d_counts), "kv cache: null or unaligned accepted indices or counts");
    TSP_REQUIRE(!over_step(pool(*cache), cache->pages, *cache, *batch) && !over(pool(*cache), cache->pages, {{d_accepted, batch->rows * 4ull}, {d_counts, batch->sequences * 4ull}}),
                "kv cache: the pages overlap the arrays that describe the step");
    return launch_cache_keep(*cache, *batch, d_accepted, d_counts, d_error, static_cast<cudaStream_t>(stream));
}

uint64_t tsp_tree_attention_scratch_bytes(void) { return tree_attention_scratch_bytes(); }

int tsp_tree_attention(const tsp_kv_cache* cache, const tsp_kv_batch* batch, const void* d_q, uint64_t q_stride, const uint64_t* d_tree_mask, uint32_t q_heads,
                       uint32_t max_rows, float scale, void* d_out, uint64_t out_stride, uint32_t dtype, void* d_scratch, uint64_t scratch_bytes, uint32_t* d_error,
                       void* stream) {
    if (int rc = check_cache(cache, batch)) return rc;
    if (int rc = check_head_rows(d_q, q_stride, q_heads, cache->head_dim, dtype, "q")) return rc;
    if (int rc = check_head_rows(d_out, out_stride, q_heads, cache->head_dim, dtype, "out")) return rc;
    TSP_REQUIRE(q_heads % cache->kv_heads == 0 && q_heads / cache->kv_heads <= 64, "attention: q_heads must be a multiple of kv_heads, at most 64 times");
    TSP_REQUIRE(max_rows >= 1 && max_rows <= TSP_KV_MAX_DRAFT, "attention: max_rows out of range");
    TSP_REQUIRE(std::isfinite(scale), "attention: scale is not finite");
    TSP_REQUIRE((reinterpret_cast<uintptr_t>(d_tree_mask) & 7u) == 0, "attention: unaligned tree words");
    TSP_REQUIRE(d_scratch && aligned16(d_scratch) && scratch_bytes >= tree_attention_scratch_bytes(), "attention: scratch too small or unaligned");
    const uint64_t bytes = static_cast<uint64_t>(q_heads) * cache->head_dim * (dtype ? 2 : 4);
    const Rows q{d_q, q_stride, bytes}, out{d_out, out_stride, bytes};
    TSP_REQUIRE(!meet(q, out, batch->rows) && !meets_pages(out, *cache, batch->rows), "attention: output rows overlap the query rows or the pages");
    TSP_REQUIRE(!overlap(d_scratch, scratch_bytes, d_out, (batch->rows - 1) * out_stride + bytes) && !overlap(d_scratch, scratch_bytes, d_q, (batch->rows - 1) * q_stride + bytes) &&
                !overlap(d_scratch, scratch_bytes, cache->d_pages, pool_bytes(*cache)), "attention: scratch overlaps other buffers");
    const Rows scratch{d_scratch, scratch_bytes, scratch_bytes};
    TSP_REQUIRE(!over_step(out, batch->rows, *cache, *batch) && !over_step(scratch, 1, *cache, *batch) && !over(out, batch->rows, {{d_tree_mask, batch->rows * 8ull}}) &&
                !over(scratch, 1, {{d_tree_mask, batch->rows * 8ull}}), "attention: output rows or scratch overlap the arrays that describe the step");
    return launch_tree_attention(*cache, *batch, d_q, q_stride, d_tree_mask, q_heads, max_rows, scale, d_out, out_stride, dtype, d_scratch, d_error,
                                 static_cast<cudaStream_t>(stream));
}

int tsp_tree_attention_check(const tsp_kv_cache* cache, const tsp_kv_batch* batch, const void* d_q, uint64_t q_stride, const uint64_t* d_tree_mask, uint32_t q_heads,
                             uint32_t max_rows, float scale, const void* d_out, uint64_t out_stride, uint32_t dtype, const void* d_scratch, uint64_t scratch_bytes) {
    LaunchCount& count = launch_count();
    const LaunchCount before = count;
    count.dry = true;
    const int rc = tsp_tree_attention(cache, batch, d_q, q_stride, d_tree_mask, q_heads, max_rows, scale, const_cast<void*>(d_out), out_stride, dtype,
                                      const_cast<void*>(d_scratch), scratch_bytes, nullptr, nullptr);
    count = before;
    return rc;
}

}  // extern "C"
