// The attention encoders of the host layer: two verify steps of two sequences, drafted trees, the accepted paths kept in between, against sums in
// double over what the cache says it holds; then the refusals.
#include <algorithm>
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
void require(bool v, const char* message) { ++checks; if (!v) throw std::runtime_error(message); }
void refuses(const std::function<void()>& action, const char* message) {
    ++checks;
    try { action(); } catch (const FormatError&) { return; }
    throw std::runtime_error(message);
}
template <class T> std::span<const std::byte> bytes(const std::vector<T>& v) { return std::as_bytes(std::span(v)); }
template <class T> std::vector<T> read(CudaGraph& g, GpuView v) {
    const auto b = g.read(v);
    std::vector<T> out(b.size() / sizeof(T));
    std::memcpy(out.data(), b.data(), b.size());
    return out;
}
uint32_t rng = 1;
float noise() { rng = rng * 1664525u + 1013904223u; return (float(rng >> 8) / float(1u << 24) - 0.5f) * 3.4f; }
std::vector<float> noise(size_t n) { std::vector<float> v(n); for (auto& x : v) x = noise(); return v; }

constexpr uint32_t D = 64, HQ = 4, HK = 2, T = 5, S = 2, PAGE = 16, PAGES = 4;

struct Sequence { std::vector<std::vector<double>> k, v; };   // kept slots, [HK * D] each

void steps(uint32_t type) {
    CudaGraph g(0, uint64_t(1) << 30);
    KvCache cache = allocate_kv_cache(g, {HK, D, PAGE, type}, S, S * PAGES + 1, PAGES);
    const AttentionScratch scratch = allocate_attention_scratch(g);
    std::vector<uint32_t> table(S * PAGES);
    for (uint32_t i = 0; i < table.size(); ++i) table[i] = uint32_t(table.size()) - i;   // any order, page 0 unused
    g.write(cache.page_table, bytes(table));
    std::vector<float> qn(D), kn(D), freq(D / 2);
    for (uint32_t i = 0; i < D; ++i) { qn[i] = 1 + 0.1f * noise(); kn[i] = 1 + 0.1f * noise(); }
    for (uint32_t i = 0; i < D / 2; ++i) freq[i] = std::pow(10000.f, -float(i) / (D / 2));
    AttentionWeights w{g.upload(bytes(qn), "q norm"), g.upload(bytes(kn), "k norm"), g.upload(bytes(freq), "frequencies"), D, false};
    const uint32_t rows = S * T;
    KvStep step{g.upload(bytes(std::vector<uint32_t>{0, T, 2 * T}), "offsets"), g.zeros(S * 4, "lengths"), rows};
    auto rows_of = [&](uint32_t columns, const char* label) { return GpuRowsF32{g.zeros(uint64_t(rows) * columns * 4, label), rows, columns, columns * 4ull}; };
    GpuRowsF32 q = rows_of(HQ * D, "q"), k = rows_of(HK * D, "k"), v = rows_of(HK * D, "v"), out = rows_of(HQ * D, "out"), kr = rows_of(HK * D, "k read"), vr = rows_of(HK * D, "v read");
    const GpuView positions = g.zeros(rows * 4, "positions"), tree = g.zeros(rows * 8, "tree"), accepted = g.zeros(rows * 4, "accepted"), counts = g.zeros(S * 4, "counts");
    const float scale = 1.f / std::sqrt(float(D));
    // a tree: 0 - 1 - 3, 0 - 2 - 4
    const uint64_t words[T] = {1, 3, 5, 11, 21};
    const uint32_t depth[T] = {0, 1, 1, 2, 2};
    const std::vector<std::vector<uint32_t>> paths[3] = {{{0, 2, 4}, {0}}, {{}, {0, 1, 3}}, {{0, 1}, {0, 2}}};
    Sequence kept[S];
    std::vector<uint32_t> length(S, 0);
    const uint64_t allocations = g.allocations();
    for (const auto& path : paths) {
        const auto hq = noise(rows * HQ * D), hk = noise(rows * HK * D), hv = noise(rows * HK * D);
        std::vector<uint32_t> pos(rows), acc(rows, 0), cnt(S);
        std::vector<uint64_t> tw(rows);
        for (uint32_t s = 0; s < S; ++s) {
            for (uint32_t j = 0; j < T; ++j) { pos[s * T + j] = length[s] + depth[j]; tw[s * T + j] = words[j]; }
            cnt[s] = uint32_t(path[s].size());
            std::copy(path[s].begin(), path[s].end(), acc.begin() + s * T);
        }
        g.write(q.view, bytes(hq)); g.write(k.view, bytes(hk)); g.write(v.view, bytes(hv)); g.write(positions, bytes(pos)); g.write(tree, bytes(tw));
        g.write(accepted, bytes(acc)); g.write(counts, bytes(cnt)); g.write(step.lengths, bytes(length));
        g.begin();
        encode_verify_attention(g, w, cache, step, scratch, q, k, v, positions, tree, T, scale, out);
        encode_kv_read(g, cache, step, kr, vr);
        encode_kv_keep(g, cache, step, accepted, counts);
        require(g.submit().dispatches == verify_attention_dispatches() + 2, "dispatch count");
        const auto gq = read<float>(g, q.view), go = read<float>(g, out.view), gk = read<float>(g, kr.view), gv = read<float>(g, vr.view);
        // norm and rotation, FP32
        for (uint32_t r = 0; r < rows; ++r)
            for (uint32_t h = 0; h < HQ + HK; ++h) {
                const bool is_k = h >= HQ;
                const float* x = is_k ? &hk[(r * HK + h - HQ) * D] : &hq[(r * HQ + h) * D];
                const auto& wn = is_k ? kn : qn;
                double ss = 0, top = 0, y[D];
                for (uint32_t i = 0; i < D; ++i) ss += double(x[i]) * x[i];
                for (uint32_t i = 0; i < D; ++i) y[i] = x[i] / std::sqrt(ss / D + double(1e-6f)) * wn[i];
                for (uint32_t i = 0; i < D / 2; ++i) {
                    const double a = double(pos[r]) * freq[i], u = y[i], z = y[i + D / 2];
                    y[i] = u * std::cos(a) - z * std::sin(a); y[i + D / 2] = z * std::cos(a) + u * std::sin(a);
                    top = std::max({top, std::abs(y[i]), std::abs(y[i + D / 2])});
                }
                for (uint32_t i = 0; i < D; ++i) {
                    // keys come back from the cache: half a step of the block's scale (or of binary16) away, and the scale's own rounding
                    const double got = is_k ? gk[(r * HK + h - HQ) * D + i] : gq[(r * HQ + h) * D + i], tol = is_k ? top * (type == TSP_TYPE_F16 ? 1.0 / 1024 : 0.51 / 127 + 1.0 / 2048) : top / 524288;
                    require(std::abs(got - y[i]) <= tol, is_k ? "key in the cache" : "query norm and rotation");
                }
            }
        // attention over what the cache holds
        for (uint32_t s = 0; s < S; ++s)
            for (uint32_t j = 0; j < T; ++j)
                for (uint32_t h = 0; h < HQ; ++h) {
                    std::vector<double> e;
                    std::vector<const double*> val;
                    std::vector<std::vector<double>> own;
                    own.reserve(2 * T);
                    double top = -1e300;
                    const uint32_t r = s * T + j, kh = h / (HQ / HK);
                    auto add = [&](const double* kk, const double* vv) {
                        double x = 0;
                        for (uint32_t i = 0; i < D; ++i) x += double(gq[(r * HQ + h) * D + i]) * kk[kh * D + i];
                        e.push_back(x * scale); val.push_back(vv + kh * D); top = std::max(top, x * scale);
                    };
                    for (size_t i = 0; i < kept[s].k.size(); ++i) add(kept[s].k[i].data(), kept[s].v[i].data());
                    for (uint32_t i = 0; i < T; ++i)
                        if (words[j] >> i & 1) {
                            own.emplace_back(&gk[(s * T + i) * HK * D], &gk[(s * T + i + 1) * HK * D]);
                            const auto& kk = own.back();
                            own.emplace_back(&gv[(s * T + i) * HK * D], &gv[(s * T + i + 1) * HK * D]);
                            add(kk.data(), own.back().data());
                        }
                    double sum = 0, o[D] = {};
                    for (size_t i = 0; i < e.size(); ++i) {
                        const double p = std::exp(e[i] - top);
                        sum += p;
                        for (uint32_t d = 0; d < D; ++d) o[d] += p * val[i][d];
                    }
                    for (uint32_t d = 0; d < D; ++d) require(std::abs(go[(r * HQ + h) * D + d] - o[d] / sum) <= 2e-5, "attention row");
                }
        for (uint32_t s = 0; s < S; ++s) {
            for (uint32_t a : path[s]) {
                kept[s].k.emplace_back(&gk[(s * T + a) * HK * D], &gk[(s * T + a + 1) * HK * D]);
                kept[s].v.emplace_back(&gv[(s * T + a) * HK * D], &gv[(s * T + a + 1) * HK * D]);
            }
            length[s] += cnt[s];
        }
    }
    require(g.allocations() == allocations, "a step allocated");
    // the kept slots, read as whole sequences
    const uint32_t all = length[0] + length[1];
    KvStep whole{g.upload(bytes(std::vector<uint32_t>{0, length[0], all}), "offsets"), g.zeros(S * 4, "zero lengths"), all};
    auto whole_of = [&](const char* label) { return GpuRowsF32{g.zeros(uint64_t(all) * HK * D * 4, label), all, HK * D, HK * D * 4ull}; };
    GpuRowsF32 ka = whole_of("whole k"), va = whole_of("whole v"), kb = whole_of("whole k again"), vb = whole_of("whole v again");
    g.begin();
    encode_kv_read(g, cache, whole, ka, va);
    // what the cache holds is written as it is and comes back as it was
    encode_kv_append(g, cache, whole, ka, va);
    encode_kv_read(g, cache, whole, kb, vb);
    (void)g.submit();
    const auto gk = read<float>(g, ka.view), gv = read<float>(g, va.view);
    for (uint32_t s = 0, at = 0; s < S; ++s)
        for (uint32_t i = 0; i < length[s]; ++i, ++at)
            for (uint32_t d = 0; d < HK * D; ++d)
                require(gk[at * HK * D + d] == kept[s].k[i][d] && gv[at * HK * D + d] == kept[s].v[i][d], "kept slot");
    require(read<float>(g, kb.view) == gk && read<float>(g, vb.view) == gv, "values of the cache written again");

    // refusals, and a batch whose page table names no page
    refuses([&] { encode_kv_read(g, cache, whole, ka, va); }, "encode outside a batch accepted");
    g.begin();
    GpuRowsF32 narrow = k;
    narrow.columns = D;
    refuses([&] { encode_verify_attention(g, w, cache, step, scratch, q, narrow, v, positions, tree, T, scale, out); }, "narrow key rows accepted");
    refuses([&] { encode_verify_attention(g, w, cache, step, scratch, q, k, v, positions, tree, 65, scale, out); }, "too many drafted rows accepted");
    refuses([&] { encode_verify_attention(g, w, cache, step, scratch, q, k, v, positions, tree, T, scale, q); }, "output over the query rows accepted");
    refuses([&] { encode_verify_attention(g, w, cache, step, {g.slice(scratch.join, 0, 1024)}, q, k, v, positions, tree, T, scale, out); }, "short scratch accepted");
    refuses([&] { encode_verify_attention(g, w, cache, step, scratch, q, k, v, g.slice(positions, 0, 16), tree, T, scale, out); }, "short positions accepted");
    refuses([&] { encode_kv_keep(g, cache, step, g.slice(accepted, 0, 16), counts); }, "short accepted indices accepted");
    KvCache other = cache;
    other.shape.page_tokens = 32;
    refuses([&] { encode_kv_keep(g, other, step, accepted, counts); }, "foreign page shape accepted");
    require(g.submit().dispatches == 0, "a refused call was counted");
    std::fill(table.begin(), table.end(), 0xffffffffu);
    g.write(cache.page_table, bytes(table));
    g.begin();
    encode_verify_attention(g, w, cache, step, scratch, q, k, v, positions, tree, T, scale, out);
    refuses([&] { (void)g.submit(); }, "pages out of range were not reported");
    release_attention_scratch(g, scratch);
    release_kv_cache(g, cache);
    refuses([&] { (void)allocate_kv_cache(g, {HK, 96, PAGE, type}, S, 4, 2); }, "head of 96 dims accepted");
}
}  // namespace

int main() {
    for (const uint32_t type : {TSP_TYPE_Q8_0, TSP_TYPE_F16}) {
        try { steps(type); } catch (const std::exception& e) {
            std::cerr << "attention check failed (type " << type << ") after " << checks << " checks: " << e.what() << '\n';
            return 1;
        }
    }
    std::cout << "attention encode checks passed: " << checks << '\n';
    return 0;
}
