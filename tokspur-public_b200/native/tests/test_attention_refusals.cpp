// encode_verify_attention refuses what either of its two launches would refuse before the first of them: the query rows, which that launch turns in place,
// and the cache are as they were, whatever view the caller got wrong.
#include <cmath>
#include <cstring>
#include <functional>
#include <iostream>
#include <stdexcept>
#include <vector>

#include "tokspur_b200/attention.hpp"

using namespace tokspur_b200;
namespace {
size_t checks = 0;
void require(bool v, const std::string& message) { ++checks; if (!v) throw std::runtime_error(message); }
template <class T> std::span<const std::byte> bytes(const std::vector<T>& v) { return std::as_bytes(std::span(v)); }

constexpr uint32_t D = 64, HQ = 4, HK = 2, ROWS = 5, PAGE = 16, PAGES = 2;

void run() {
    CudaGraph g(0, uint64_t(1) << 30);
    KvCache cache = allocate_kv_cache(g, {HK, D, PAGE, TSP_TYPE_Q8_0}, 1, PAGES, PAGES);
    g.write(cache.page_table, bytes(std::vector<uint32_t>{0, 1}));
    const AttentionScratch scratch = allocate_attention_scratch(g);
    std::vector<float> freq(D / 2);
    for (uint32_t i = 0; i < D / 2; ++i) freq[i] = std::pow(10000.f, -float(i) / (D / 2));
    const AttentionWeights w{{}, {}, g.upload(bytes(freq), "frequencies"), D, false};
    const KvStep step{g.upload(bytes(std::vector<uint32_t>{0, ROWS}), "offsets"), g.zeros(4, "lengths"), ROWS};
    // query rows and a join scratch that may overlap them in one buffer
    const uint64_t q_bytes = uint64_t(ROWS) * HQ * D * 4, scratch_bytes = tsp_tree_attention_scratch_bytes();
    const GpuView wide = g.zeros(q_bytes + scratch_bytes, "query rows and scratch");
    std::vector<float> hq((q_bytes + scratch_bytes) / 4), hkv(uint64_t(ROWS) * HK * D);
    for (size_t i = 0; i < q_bytes / 4; ++i) hq[i] = float(i % 17) - 8;
    for (size_t i = 0; i < hkv.size(); ++i) hkv[i] = float(i % 13) - 6;
    g.write(wide, bytes(hq));
    auto rows = [](GpuView v, uint32_t columns) { return GpuRowsF32{v, ROWS, columns, columns * 4ull}; };
    const GpuRowsF32 q = rows(g.slice(wide, 0, q_bytes), HQ * D), k = rows(g.upload(bytes(hkv), "k"), HK * D);
    const GpuView out = g.zeros(q_bytes + 16, "out"), tree = g.zeros(ROWS * 8 + 8, "tree"), join = g.zeros(scratch_bytes + 16, "join");
    std::vector<uint32_t> pos(ROWS);
    for (uint32_t i = 0; i < ROWS; ++i) pos[i] = 3 + i;
    const GpuView positions = g.upload(bytes(pos), "positions");
    const GpuRowsF32 good_out = rows(g.slice(out, 0, q_bytes), HQ * D);
    const GpuView good_tree = g.slice(tree, 0, ROWS * 8);
    const auto q_before = g.read(q.view), pages_before = g.read(cache.pages);

    auto refused = [&](const char* what, const GpuRowsF32& o, GpuView words, AttentionScratch s, uint32_t most, float scale) {
        g.begin();
        bool thrown = false;
        try { encode_verify_attention(g, w, cache, step, s, q, k, k, positions, words, most, scale, o); } catch (const FormatError&) { thrown = true; }
        const uint64_t dispatches = g.submit().dispatches;
        require(thrown, std::string(what) + ": accepted");
        require(dispatches == 0, std::string(what) + ": counted");
        require(g.read(q.view) == q_before, std::string(what) + ": query rows changed");
        require(g.read(cache.pages) == pages_before, std::string(what) + ": cache changed");
    };
    refused("output rows off their alignment", rows(g.slice(out, 4, q_bytes), HQ * D), good_tree, scratch, ROWS, 0.125f);
    refused("tree words off theirs", good_out, g.slice(tree, 4, ROWS * 8), scratch, ROWS, 0.125f);
    refused("scratch off its own", good_out, good_tree, {g.slice(join, 8, scratch_bytes)}, ROWS, 0.125f);
    refused("scratch over the query rows", good_out, good_tree, {g.slice(wide, q_bytes - 512, scratch_bytes)}, ROWS, 0.125f);
    refused("scratch over the output rows", rows(g.slice(join, 0, q_bytes), HQ * D), good_tree, {g.slice(join, 0, scratch_bytes)}, ROWS, 0.125f);
    refused("output rows over the query rows", rows(g.slice(wide, 16, q_bytes), HQ * D), good_tree, scratch, ROWS, 0.125f);
    require(cache.pages.bytes >= q_bytes, "pages hold output rows");
    refused("output rows over the pages", rows(g.slice(cache.pages, 0, q_bytes), HQ * D), good_tree, scratch, ROWS, 0.125f);
    refused("short scratch", good_out, good_tree, {g.slice(join, 0, 1024)}, ROWS, 0.125f);
    refused("too many rows", good_out, good_tree, scratch, 65, 0.125f);
    refused("a scale that is not finite", good_out, good_tree, scratch, ROWS, INFINITY);

    // and the same call with nothing wrong
    g.begin();
    encode_verify_attention(g, w, cache, step, scratch, q, k, k, positions, {}, ROWS, 0.125f, good_out);
    require(g.submit().dispatches == verify_attention_dispatches(), "dispatch count");
    require(g.read(q.view) != q_before && g.read(cache.pages) != pages_before, "the step has run");
}
}  // namespace

int main() {
    try { run(); } catch (const std::exception& e) {
        std::cerr << "attention refusal check failed after " << checks << " checks: " << e.what() << '\n';
        return 1;
    }
    std::cout << "attention refusal checks passed: " << checks << '\n';
    return 0;
}
