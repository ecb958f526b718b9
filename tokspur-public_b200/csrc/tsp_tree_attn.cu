// Attention of the drafted tokens of every sequence over its paged cache (tsp_tree_attention).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(f q.k_j - m), f = scale log2(e), in one pass over the cache with the running maximum m and sum of every row.
//
// The query rows of one kv head (drafted tokens x heads of the group) share the head's keys and values: tiles of 16 such rows are the M of
// m16n8k16 MMAs, the slots of the cache their N (scores) and K (values). Work is cut into units of `kUnit` slots of one (sequence, head, row tile)
// item; the units of the whole batch, item after item, are dealt to the blocks in equal runs, so that one long context fills the GPU as a ragged
// batch does. A block is a producer warp (bulk copies of whole groups of 16 slots into a ring) and eight warps that take the units in
// turn, each with its own maximum, sum and accumulators; they join in shared memory when the item or the run ends. An item that spans blocks is
// joined by the last of them to arrive, from the partial results in the scratch, in block order: the same bits every time.
#include "tsp_kv.cuh"

namespace tsp {

constexpr uint32_t kWarps = 8, kProducers = 4, kRows = 16, kAttnThreads = 32 * (kWarps + kProducers);
// Registers after the hand-over between the warpgroups (setmaxnreg): the consumers' request waits for what the producers give back, so
// kWarps * (kConsumerRegs - launch) <= kProducers * (launch - kProducerRegs) must hold for the count at launch (168); the launcher checks it.
constexpr int kConsumerRegs = 224, kProducerRegs = 56;
constexpr uint32_t kAttnMaxBlocks = 192;     // blocks (one per SM) that the scratch has room for
constexpr uint32_t kLeastUnits = 4;          // units of a block's run at least

struct AttnScratch {   // one per launch; counters are zero between calls
    uint32_t counters[kAttnMaxBlocks];
};
// partial result of a run's first or last item: 16 maxima, 16 sums, a flag, then the rows
constexpr uint32_t kPartHead = 48;
__host__ __device__ constexpr uint64_t part_floats() { return kPartHead + kRows * 256; }

struct AttnParams {
    tsp_kv_cache cache;
    tsp_kv_batch batch;
    const uint8_t* q; uint64_t q_stride;
    const uint64_t* mask;
    uint8_t* out; uint64_t out_stride;
    uint32_t group, max_rows;
    float scale;
    uint32_t* counters;
    float* parts;
    uint32_t* error;
};

template <uint32_t D, bool Q8>
struct AttnShape {
    static constexpr uint32_t kGroupBytes = kv_group_bytes(D, Q8), kHalf = kv_half_bytes(D, Q8);
    static constexpr uint32_t kGroups = kGroupBytes * 2 <= 17408 ? 2 : 1, kUnit = kGroups * kKvGroup, kStage = kGroups * kGroupBytes;
    // A multiple of the warps: a stage then always has the same consumer (and producer), so that nobody waits for a phase while the one before
    // it is open, which a wait by parity would take for done.
    static constexpr uint32_t kStages = 16 * kStage <= 139264 ? 16 : 8;
    static_assert(kStages % kWarps == 0 && kStages % kProducers == 0, "a stage has one consumer and one producer");
    static constexpr uint32_t kSlots = D == 256 ? 4 : 8;   // accumulators that meet in shared memory at once
};
template <uint32_t D, bool Q8, bool F16>
struct AttnSmem {
    using S = AttnShape<D, Q8>;
    alignas(128) uint8_t ring[S::kStages][S::kStage];
    alignas(16) uint32_t q[F16 ? 1 : 2][D / 16][32][4];     // A fragments of the item's rows; binary16 high and low parts of FP32 rows
    float o[S::kSlots][kRows][D];
    float m[kWarps][kRows], l[kWarps][kRows];
    float qscale[kRows];
    uint64_t words[kRows];
    uint64_t full[S::kStages], empty[S::kStages];
    uint64_t cum[TSP_KV_MAX_SEQUENCES + 1];
    uint64_t warp_sums[kWarps + kProducers];
    uint32_t bad_stage[S::kStages];
    uint32_t row_bad[kRows];
    uint32_t failed, dead, last;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
// four codes + 128 -> two pairs of binary16 integers: 0x64 in front of a byte is 1024 + byte
__device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    const __half2 bias = bits_h2(0x64806480u);   // 1152
    a = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4140)), bias));
    b = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4342)), bias));
}

static_assert(kAttnMaxBlocks * kRows <= 6 * kRows * 64 && kAttnMaxBlocks * kRows <= 2 * kRows * 256, "the join's weights lie in accumulators 2 and up");

struct AttnItem {
    uint64_t start, end;     // units of the item
    uint64_t length, total;  // slots of the context, and with the step's own
    uint32_t seq, head, tile, row0, drafted, rows;   // rows: of this tile
    bool dead;               // out of range: zeros
};

// Geometry of a sequence: units of an item, row tiles
template <uint32_t UNIT>
__device__ __forceinline__ void sequence_shape(const AttnParams& p, uint32_t s, uint32_t& row0, uint32_t& drafted, uint64_t& length, uint64_t& units, uint32_t& tiles, bool& dead) {
    row0 = p.batch.d_row_offsets[s];
    const uint32_t end = p.batch.d_row_offsets[s + 1];
    drafted = end >= row0 && end <= p.batch.rows ? end - row0 : 0;
    length = p.batch.d_lengths[s];
    const uint64_t total = length + drafted;
    dead = drafted > p.max_rows || total > static_cast<uint64_t>(p.cache.table_stride) * p.cache.page_tokens;
    units = dead ? 1 : (total + UNIT - 1) / UNIT;
    tiles = static_cast<uint32_t>((static_cast<uint64_t>(drafted) * p.group + kRows - 1) / kRows);
}

template <uint32_t UNIT>
__device__ __forceinline__ AttnItem item_of(const AttnParams& p, const uint64_t* cum, uint64_t u) {
    uint32_t lo = 0, hi = p.batch.sequences;    // cum[lo] <= u < cum[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (cum[mid] <= u) lo = mid; else hi = mid;
    }
    AttnItem i;
    uint64_t units;
    uint32_t tiles;
    i.seq = lo;
    sequence_shape<UNIT>(p, lo, i.row0, i.drafted, i.length, units, tiles, i.dead);
    i.total = i.length + i.drafted;
    const uint64_t rest = u - cum[lo];
    const uint32_t n = rest >> 32 ? static_cast<uint32_t>(rest / units) : static_cast<uint32_t>(rest) / static_cast<uint32_t>(units);
    i.start = cum[lo] + n * units;
    i.end = i.start + units;
    i.head = n / tiles;
    i.tile = n - i.head * tiles;
    i.rows = min(kRows, i.drafted * p.group - i.tile * kRows);
    return i;
}

template <uint32_t D, bool Q8, bool F16>
__global__ void __launch_bounds__(kAttnThreads, 1)
tree_attention_kernel(const AttnParams p) {
    using S = AttnShape<D, Q8>;
    constexpr uint32_t UNIT = S::kUnit, NB = D / 32;
    extern __shared__ uint8_t raw[];
    AttnSmem<D, Q8, F16>& sm = *reinterpret_cast<AttnSmem<D, Q8, F16>*>(raw);
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;
    pdl_launch_dependents();
    if (tid == 0) {
        for (uint32_t i = 0; i < S::kStages; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
        mbar_fence_init();
        sm.failed = sm.dead = 0;
    }
    pdl_wait();
    // units before every sequence
    {
        uint64_t mine[4], sum = 0;
        const uint32_t per = (p.batch.sequences + kAttnThreads - 1) / kAttnThreads;   // <= 4
        bool bad = false;
        for (uint32_t k = 0; k < per; ++k) {
            const uint32_t s = tid * per + k;
            mine[k] = sum;
            if (s < p.batch.sequences) {
                uint32_t row0, drafted, tiles;
                uint64_t length, units;
                bool dead;
                sequence_shape<UNIT>(p, s, row0, drafted, length, units, tiles, dead);
                bad |= dead && drafted;
                sum += static_cast<uint64_t>(p.cache.kv_heads) * tiles * units;
            }
        }
        if (bad && blockIdx.x == 0) raise_error(p.error, TSP_ERR_INDEX);
        uint64_t run = sum;
#pragma unroll
        for (uint32_t o = 1; o < 32; o *= 2) {
            const uint64_t below = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += below;
        }
        if (lane == 31) sm.warp_sums[warp] = run;
        __syncthreads();
        uint64_t base = run - sum;
        for (uint32_t w = 0; w < warp; ++w) base += sm.warp_sums[w];
        for (uint32_t k = 0; k < per; ++k) {
            const uint32_t s = tid * per + k;
            if (s < p.batch.sequences) sm.cum[s] = base + mine[k];
        }
        if (tid == kAttnThreads - 1) sm.cum[p.batch.sequences] = base + sum;
        if (blockIdx.x == 0) kv_check_offsets(p.batch, p.error);
        __syncthreads();
    }
    const uint64_t units = sm.cum[p.batch.sequences];
    const uint64_t quota = max(static_cast<uint64_t>(kLeastUnits), (units + gridDim.x - 1) / gridDim.x);
    const uint64_t u0 = min(units, blockIdx.x * quota), u1 = min(units, u0 + quota);
    if (u0 >= u1) return;

    if (warp >= kWarps) {   // producers, every fourth unit each: the lanes look up the sources of 32 units, then the copies go out one after another
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
        const uint32_t mine = static_cast<uint32_t>(u1 - u0);
        for (uint32_t base = warp - kWarps; base < mine; base += 32 * kProducers) {
            const uint32_t ahead = base + lane * kProducers;
            const uint8_t* src[S::kGroups] = {};
            uint32_t groups = 0, bad = 0;
            if (ahead < mine) {
                const AttnItem it = item_of<UNIT>(p, sm.cum, u0 + ahead);
                if (it.dead) bad = 1;
                else {
                    const uint64_t slot = (u0 + ahead - it.start) * UNIT;
#pragma unroll
                    for (uint32_t k = 0; k < S::kGroups; ++k)
                        if (slot + k * kKvGroup < it.total) {
                            src[k] = kv_group(p.cache, it.seq, slot + k * kKvGroup, it.head, p.error);
                            if (!src[k]) bad = 1;
                            ++groups;
                        }
                }
                if (bad) groups = 0;
            }
            for (uint32_t k = 0; k < 32 && base + k * kProducers < mine; ++k) {
                const uint32_t li = base + k * kProducers, st = li % S::kStages, round = li / S::kStages;
                const uint32_t gs = __shfl_sync(0xffffffffu, groups, k), b = __shfl_sync(0xffffffffu, bad, k);
                const uint8_t* from[S::kGroups];
#pragma unroll
                for (uint32_t j = 0; j < S::kGroups; ++j)
                    from[j] = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src[j]), k));
                if (round && !mbar_wait(&sm.empty[st], (round - 1) & 1)) {
                    raise_error(p.error, TSP_ERR_TIMEOUT);
                    return;   // the consumers' own waits run out
                }
                if (elect_one()) {
                    sm.bad_stage[st] = b;
                    mbar_arrive_expect_tx(&sm.full[st], gs * S::kGroupBytes);
                    if (gs == 2 && from[1 % S::kGroups] == from[0] + S::kGroupBytes) bulk_g2s(sm.ring[st], from[0], 2 * S::kGroupBytes, &sm.full[st]);
                    else {
#pragma unroll
                        for (uint32_t j = 0; j < S::kGroups; ++j)
                            if (j < gs) bulk_g2s(sm.ring[st] + j * S::kGroupBytes, from[j], S::kGroupBytes, &sm.full[st]);
                    }
                }
                __syncwarp();
            }
        }
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));

    for (uint64_t at = u0; at < u1;) {
        const AttnItem it = item_of<UNIT>(p, sm.cum, at);
        const uint64_t stop = min(it.end, u1);
        // ---- the item's rows as A fragments: step x / 32 * 2 + x % 8 / 4, lane (row % 8, x % 32 / 8), the order in which a lane holds the keys
        named_bar_sync(1, kWarps * 32);
        for (uint32_t r = warp; r < kRows; r += kWarps) {
            const uint32_t flat = it.tile * kRows + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
            float v[NB];
            float top = 0.f;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                v[b] = 0.f;
                if (r < it.rows) {
                    const uint8_t* src = p.q + static_cast<uint64_t>(it.row0 + node) * p.q_stride + (head * D + b * 32 + lane) * (F16 ? 2 : 4);
                    v[b] = F16 ? __half2float(*reinterpret_cast<const __half*>(src)) : *reinterpret_cast<const float*>(src);
                }
                top = fmaxf(top, fabsf(v[b]));
            }
            float up = 1.f;
            if constexpr (!F16) {   // the row times a power of two that puts its largest value at 2^14: both parts keep their 11 bits
#pragma unroll
                for (uint32_t o = 16; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
                const int shift = top > 0.f && e < 128 ? max(-100, min(100, 14 - e)) : 0;
                up = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23);
                if (lane == 0) sm.qscale[r] = p.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
            } else if (lane == 0) sm.qscale[r] = p.scale * 1.4426950408889634f;
            const uint32_t y = lane, tt = y / 8, s = y % 8 / 4, e = y % 4;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t step = 2 * b + s, reg = (r >= 8) + 2 * (e >= 2), dst = (r % 8) * 4 + tt;
                const float x = v[b] * up;
                const __half hi = __float2half_rn(x);
                reinterpret_cast<__half*>(&sm.q[0][step][dst][reg])[e & 1] = hi;
                if constexpr (!F16) reinterpret_cast<__half*>(&sm.q[1][step][dst][reg])[e & 1] = __float2half_rn(x - __half2float(hi));
            }
            if (lane == 0) {
                sm.words[r] = r >= it.rows ? 0 : p.mask ? p.mask[it.row0 + node] : ~0ull >> (63 - min(node, 63u));
                sm.row_bad[r] = 0;
            }
        }
        named_bar_sync(1, kWarps * 32);
        const float f0 = sm.qscale[g], f1 = sm.qscale[g + 8];
        const uint64_t word0 = sm.words[g], word1 = sm.words[g + 8];

        float o[NB][4][4];   // [32 dims][n tile][c]: rows g, g + 8; dims 32 b + 8 i + 2 t, + 1
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) o[b][i][c] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        [[maybe_unused]] float vup = 0.f;   // FP32 rows of a Q8_0 cache: power of two that the weights times the value scales are held at
        bool dead = false;

        const uint32_t first = static_cast<uint32_t>(at - u0);
        for (uint32_t li = first + (warp + kWarps - first % kWarps) % kWarps; li < static_cast<uint32_t>(stop - u0); li += kWarps) {
            const uint32_t st = li % S::kStages;
            const uint64_t slot0 = (u0 + li - it.start) * UNIT;
            bool ok = *reinterpret_cast<volatile uint32_t*>(&sm.failed) == 0 && mbar_wait(&sm.full[st], (li / S::kStages) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) { sm.failed = 1; raise_error(p.error, TSP_ERR_TIMEOUT); }
                dead = true;
                continue;
            }
            if (sm.bad_stage[st]) dead = true;
            else {
                const bool edge = slot0 + UNIT > it.length;
                const uint8_t* stage = sm.ring[st];
                float s[S::kGroups][2][4];
#pragma unroll
                for (uint32_t k = 0; k < S::kGroups; ++k)
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n) {
                        const uint8_t* keys = stage + k * S::kGroupBytes;
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) s[k][n][c] = 0.f;
#pragma unroll
                        for (uint32_t b = 0; b < NB; ++b) {   // 32 dims: two steps under one scale
                            float acc[4] = {0.f, 0.f, 0.f, 0.f};
                            uint32_t kb[4];
                            if constexpr (Q8) {
                                const uint2 w = *reinterpret_cast<const uint2*>(keys + (b / 2 * kKvGroup + 8 * n + g) * 64 + t * 16 + b % 2 * 8);
                                codes_to_halves(w.x, kb[0], kb[1]);
                                codes_to_halves(w.y, kb[2], kb[3]);
                            } else {
                                const uint4 w = *reinterpret_cast<const uint4*>(keys + (b * kKvGroup + 8 * n + g) * 64 + t * 16);
                                kb[0] = w.x; kb[1] = w.y; kb[2] = w.z; kb[3] = w.w;
                            }
#pragma unroll
                            for (uint32_t h = 0; h < 2; ++h) {
                                const uint4 a = *reinterpret_cast<const uint4*>(sm.q[0][2 * b + h][lane]);
                                mma_f16_16816(acc, a.x, a.y, a.z, a.w, kb[2 * h], kb[2 * h + 1]);
                                if constexpr (!F16) {
                                    const uint4 low = *reinterpret_cast<const uint4*>(sm.q[1][2 * b + h][lane]);
                                    mma_f16_16816(acc, low.x, low.y, low.z, low.w, kb[2 * h], kb[2 * h + 1]);
                                }
                            }
                            float2 d = make_float2(1.f, 1.f);
                            if constexpr (Q8) d = __half22float2(*reinterpret_cast<const __half2*>(keys + kKvGroup * D + (b * kKvGroup + 8 * n + 2 * t) * 2));
                            s[k][n][0] = fmaf(acc[0], d.x, s[k][n][0]); s[k][n][1] = fmaf(acc[1], d.y, s[k][n][1]);
                            s[k][n][2] = fmaf(acc[2], d.x, s[k][n][2]); s[k][n][3] = fmaf(acc[3], d.y, s[k][n][3]);
                        }
                    }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (uint32_t k = 0; k < S::kGroups; ++k)
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n) {
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) s[k][n][c] *= c < 2 ? f0 : f1;
                        if (edge) {
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) {
                                const uint64_t slot = slot0 + k * kKvGroup + 8 * n + 2 * t + (c & 1);
                                const uint64_t word = c < 2 ? word0 : word1;
                                if (slot >= it.total || (slot >= it.length && !(word >> (slot - it.length) & 1))) s[k][n][c] = -INFINITY;
                            }
                        }
                        x0 = fmaxf(x0, fmaxf(s[k][n][0], s[k][n][1]));
                        x1 = fmaxf(x1, fmaxf(s[k][n][2], s[k][n][3]));
                    }
                // drafted slots whose values are not finite: rows that see them get NaN through the weight, and the values count as zero
                [[maybe_unused]] uint32_t drop[S::kGroups] = {};   // bit e: slot 2 t + (e & 1) + 8 (e >> 1)
                if (edge) {
#pragma unroll
                    for (uint32_t k = 0; k < S::kGroups; ++k) {
                        const uint8_t* values = stage + k * S::kGroupBytes + S::kHalf;
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            const uint64_t slot = slot0 + k * kKvGroup + 2 * t + (e & 1) + 8 * (e >> 1);
                            bool odd = false;
                            if (slot >= it.length && slot < it.total) {
                                if constexpr (Q8) {
                                    for (uint32_t b = 0; b < NB; ++b)
                                        odd |= (*reinterpret_cast<const uint16_t*>(values + kKvGroup * D + (b * kKvGroup + 2 * t + (e & 1) + 8 * (e >> 1)) * 2) & 0x7c00u) == 0x7c00u;
                                } else {
                                    for (uint32_t i = 0; i < D / 8; ++i)
                                        odd |= (*reinterpret_cast<const uint16_t*>(values + (i / 2 * 32 + lane) * 16 + i % 2 * 8 + e * 2) & 0x7c00u) == 0x7c00u;
                                }
                            }
                            if constexpr (!Q8) {
                                uint32_t v = odd;
                                v |= __shfl_xor_sync(0xffffffffu, v, 4); v |= __shfl_xor_sync(0xffffffffu, v, 8); v |= __shfl_xor_sync(0xffffffffu, v, 16);
                                odd = v;
                            }
                            if (odd) {
                                if (s[k][e >> 1][e & 1] != -INFINITY) s[k][e >> 1][e & 1] = NAN;
                                if (s[k][e >> 1][2 + (e & 1)] != -INFINITY) s[k][e >> 1][2 + (e & 1)] = NAN;
                            }
                            if (odd || slot >= it.total) drop[k] |= 1u << e;
                        }
                    }
                }
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
                x0 = fmaxf(x0, m0); x1 = fmaxf(x1, m1);
                // weights are held at 2^15 at most (2^0 under the value scales of FP32 rows): binary16 then reaches 2^-39 of the largest
                constexpr float kUp = F16 || !Q8 ? 15.f : 0.f;
                [[maybe_unused]] float up = vup;
                if constexpr (!F16 && Q8) {
                    __half2 top = __float2half2_rn(0.f);
#pragma unroll
                    for (uint32_t k = 0; k < S::kGroups; ++k)
#pragma unroll
                        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                            for (uint32_t n = 0; n < 2; ++n) {
                                uint32_t d = *reinterpret_cast<const uint32_t*>(stage + k * S::kGroupBytes + S::kHalf + kKvGroup * D + (b * kKvGroup + 8 * n + 2 * t) * 2);
                                if (drop[k] >> (2 * n) & 1) d &= 0xffff0000u;
                                if (drop[k] >> (2 * n) & 2) d &= 0x0000ffffu;
                                top = __hmax2(top, __habs2(bits_h2(d)));
                            }
                    float v = fmaxf(__low2float(top), __high2float(top));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                    const int e = static_cast<int>(__float_as_uint(v) >> 23) - 127;
                    if (v > 0.f && e < 128) {
                        const float u = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);   // v u in [2^14, 2^15)
                        up = vup == 0.f ? u : fminf(vup, u);
                    }
                }
                if (__any_sync(0xffffffffu, x0 != m0 || x1 != m1 || (!F16 && Q8 && up != vup))) {
                    float r0 = m0 == -INFINITY ? 0.f : exp2_approx(m0 - x0), r1 = m1 == -INFINITY ? 0.f : exp2_approx(m1 - x1);
                    l0 *= r0; l1 *= r1;
                    if constexpr (!F16 && Q8) { if (vup != 0.f) { const float r = up / vup; r0 *= r; r1 *= r; } vup = up; }
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) { o[b][i][0] *= r0; o[b][i][1] *= r0; o[b][i][2] *= r1; o[b][i][3] *= r1; }
                    m0 = x0; m1 = x1;
                }
                const float b0 = m0 == -INFINITY ? 0.f : m0 - kUp, b1 = m1 == -INFINITY ? 0.f : m1 - kUp;
#pragma unroll
                for (uint32_t k = 0; k < S::kGroups; ++k) {
                    const uint8_t* values = stage + k * S::kGroupBytes + S::kHalf;
                    float pr[2][4];
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) {
                            pr[n][c] = exp2_approx(s[k][n][c] - (c < 2 ? b0 : b1));
                            if (c < 2) l0 += pr[n][c]; else l1 += pr[n][c];
                        }
                    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};   // value pairs of slots 2t, 2t + 1 and 8 more
                    if (edge) {
#pragma unroll
                        for (uint32_t n = 0; n < 2; ++n) keep[n] = (drop[k] >> (2 * n) & 1 ? 0u : 0x0000ffffu) | (drop[k] >> (2 * n) & 2 ? 0u : 0xffff0000u);
                    }
                    uint32_t a[4], al[4];
                    auto split = [&](const float (&w)[2][4]) {
#pragma unroll
                        for (uint32_t r = 0; r < 4; ++r) {   // a0: row g, slots 2t..; a1: row g + 8; a2, a3: slots 8 further
                            const float u = w[r / 2][r % 2 * 2], v = w[r / 2][r % 2 * 2 + 1];
                            const __half2 h = __floats2half2_rn(u, v);
                            a[r] = h2_bits(h);
                            if constexpr (!F16) { const float2 f = __half22float2(h); al[r] = h2_bits(__floats2half2_rn(u - f.x, v - f.y)); }
                        }
                    };
                    if constexpr (F16 || !Q8) split(pr);
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b) {
                        uint32_t vb[8];
                        if constexpr (Q8) {
                            const uint4 w = *reinterpret_cast<const uint4*>(values + b * 512 + lane * 16);
                            codes_to_halves(w.x, vb[0], vb[1]); codes_to_halves(w.y, vb[2], vb[3]);
                            codes_to_halves(w.z, vb[4], vb[5]); codes_to_halves(w.w, vb[6], vb[7]);
                            uint32_t d[2];
#pragma unroll
                            for (uint32_t n = 0; n < 2; ++n) d[n] = *reinterpret_cast<const uint32_t*>(values + kKvGroup * D + (b * kKvGroup + 8 * n + 2 * t) * 2) & keep[n];
                            if constexpr (F16) {
#pragma unroll
                                for (uint32_t i = 0; i < 8; ++i) vb[i] = h2_bits(__hmul2(bits_h2(vb[i]), bits_h2(d[i & 1])));
                            } else {   // codes are exact, so the value scale goes to the weight
                                float w4[2][4];
#pragma unroll
                                for (uint32_t n = 0; n < 2; ++n) {
                                    const float2 f = __half22float2(bits_h2(d[n]));
#pragma unroll
                                    for (uint32_t c = 0; c < 4; ++c) w4[n][c] = pr[n][c] * ((c & 1 ? f.y : f.x) * vup);
                                }
                                split(w4);
                            }
                        } else {
                            const uint4 w = *reinterpret_cast<const uint4*>(values + b * 1024 + lane * 16), x = *reinterpret_cast<const uint4*>(values + b * 1024 + 512 + lane * 16);
                            vb[0] = w.x & keep[0]; vb[1] = w.y & keep[1]; vb[2] = w.z & keep[0]; vb[3] = w.w & keep[1];
                            vb[4] = x.x & keep[0]; vb[5] = x.y & keep[1]; vb[6] = x.z & keep[0]; vb[7] = x.w & keep[1];
                        }
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            if constexpr (F16) mma_f16_16816(o[b][i], a[0], a[1], a[2], a[3], vb[2 * i], vb[2 * i + 1]);
                            else {   // the tensor core cuts its sums off: a chain of two products, added up rounded
                                float acc[4];
                                mma_f16_16816_zero(acc, a[0], a[1], a[2], a[3], vb[2 * i], vb[2 * i + 1]);
                                mma_f16_16816(acc, al[0], al[1], al[2], al[3], vb[2 * i], vb[2 * i + 1]);
#pragma unroll
                                for (uint32_t c = 0; c < 4; ++c) o[b][i][c] += acc[c];
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
        }

        // ---- the warps' results meet
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if constexpr (!F16 && Q8) {
            const float down = vup == 0.f ? 0.f : 1.f / vup;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) o[b][i][c] *= down;
        }
        if (t == 0) { sm.m[warp][g] = m0; sm.m[warp][g + 8] = m1; sm.l[warp][g] = l0; sm.l[warp][g + 8] = l1; }
        if (dead && lane == 0) sm.dead = 1;
        auto put = [&](uint32_t slot) {
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (g < it.rows) *reinterpret_cast<float2*>(&sm.o[slot][g][b * 32 + i * 8 + 2 * t]) = make_float2(o[b][i][0], o[b][i][1]);
                    if (g + 8 < it.rows) *reinterpret_cast<float2*>(&sm.o[slot][g + 8][b * 32 + i * 8 + 2 * t]) = make_float2(o[b][i][2], o[b][i][3]);
                }
        };
        if constexpr (S::kSlots < kWarps) {   // wide heads: the upper half of the warps hand theirs to the lower half
            if (warp >= S::kSlots) put(warp - S::kSlots);
            named_bar_sync(1, kWarps * 32);
            if (warp < S::kSlots) {
                const uint32_t other = warp + S::kSlots;
                const float n0 = sm.m[other][g], n1 = sm.m[other][g + 8], x0 = fmaxf(m0, n0), x1 = fmaxf(m1, n1);
                const float fa0 = m0 == -INFINITY ? 0.f : exp2_approx(m0 - x0), fa1 = m1 == -INFINITY ? 0.f : exp2_approx(m1 - x1);
                const float fb0 = n0 == -INFINITY ? 0.f : exp2_approx(n0 - x0), fb1 = n1 == -INFINITY ? 0.f : exp2_approx(n1 - x1);
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        if (g < it.rows) {
                            const float2 y = *reinterpret_cast<const float2*>(&sm.o[warp][g][b * 32 + i * 8 + 2 * t]);
                            o[b][i][0] = o[b][i][0] * fa0 + (n0 == -INFINITY ? 0.f : y.x * fb0); o[b][i][1] = o[b][i][1] * fa0 + (n0 == -INFINITY ? 0.f : y.y * fb0);
                        }
                        if (g + 8 < it.rows) {
                            const float2 y = *reinterpret_cast<const float2*>(&sm.o[warp][g + 8][b * 32 + i * 8 + 2 * t]);
                            o[b][i][2] = o[b][i][2] * fa1 + (n1 == -INFINITY ? 0.f : y.x * fb1); o[b][i][3] = o[b][i][3] * fa1 + (n1 == -INFINITY ? 0.f : y.y * fb1);
                        }
                    }
                const float k0 = sm.l[other][g], k1 = sm.l[other][g + 8];
                l0 = l0 * fa0 + k0 * fb0; l1 = l1 * fa1 + k1 * fb1;
                __syncwarp();
                if (t == 0) { sm.m[warp][g] = x0; sm.m[warp][g + 8] = x1; sm.l[warp][g] = l0; sm.l[warp][g + 8] = l1; }
                put(warp);
            }
        } else put(warp);
        named_bar_sync(1, kWarps * 32);
        const bool whole = at == it.start && stop == it.end;
        const uint32_t me = blockIdx.x, place = 2 * me + (at == u0 ? 0 : 1);
        constexpr uint32_t PER = kRows * D / (kWarps * 32);
        float y[PER];
        const uint32_t c0 = static_cast<uint32_t>(it.start / quota), c1 = static_cast<uint32_t>((it.end - 1) / quota);
        bool all_dead = sm.dead != 0;
        float* part = p.parts + place * part_floats();
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const uint32_t e = tid + k * kWarps * 32, r = e / D, x = e % D;
            y[k] = 0.f;
            if (r < it.rows) {
                float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < S::kSlots; ++w) top = fmaxf(top, sm.m[w][r]);
#pragma unroll
                for (uint32_t w = 0; w < S::kSlots; ++w) {
                    const float mw = sm.m[w][r], fw = mw == -INFINITY ? 0.f : exp2_approx(mw - top);
                    if (mw != -INFINITY) acc = fmaf(sm.o[w][r][x], fw, acc);
                    sum += mw == -INFINITY ? sm.l[w][r] : sm.l[w][r] * fw;   // a row of NaN alone has a sum of NaN and no maximum
                }
                y[k] = acc;
                if (whole) y[k] = sum == 0.f ? 0.f : acc / sum;
                else {
                    __stcg(part + kPartHead + e, acc);
                    if (x == 0) { __stcg(part + r, top); __stcg(part + 16 + r, sum); }
                }
            }
        }
        if (!whole) {
            if (tid == 0) __stcg(part + 32, all_dead ? 1.f : 0.f);
            __threadfence();
            named_bar_sync(1, kWarps * 32);
            if (tid == 0) {
                const uint32_t n = atomicAdd(p.counters + c0, 1u);
                sm.last = n == c1 - c0;
                if (sm.last) { p.counters[c0] = 0; sm.dead = 0; }
            }
            named_bar_sync(1, kWarps * 32);
            if (sm.last) {
                __threadfence();
                const uint32_t n = c1 - c0 + 1;
                float (&weight)[kAttnMaxBlocks][kRows] = *reinterpret_cast<float (*)[kAttnMaxBlocks][kRows]>(&sm.o[2]);
                auto place_of = [&](uint32_t i) { return p.parts + (2 * (c0 + i) + (i == 0 && c0 * quota != it.start ? 1 : 0)) * part_floats(); };
                // weights of the partial results: a thread per row and sixteenth of them
                if (tid < 256) {
                    const uint32_t r = tid % kRows;
                    float top = -INFINITY;
                    for (uint32_t i = tid / kRows; i < n; i += 16) {
                        const float v = r < it.rows ? __ldcg(place_of(i) + r) : -INFINITY;
                        weight[i][r] = v;
                        top = fmaxf(top, v);
                        if (r == 0 && __ldcg(place_of(i) + 32) != 0.f) sm.dead = 1;
                    }
                    sm.o[0][tid / kRows][r] = top;
                }
                named_bar_sync(1, kWarps * 32);
                all_dead = sm.dead != 0;
                {
                    const uint32_t r = tid % kRows;
                    float top = -INFINITY, sum = 0.f;
                    for (uint32_t i = 0; i < 16; ++i) top = fmaxf(top, sm.o[0][i][r]);
                    for (uint32_t i = tid / kRows; i < n; i += 16) {
                        const float mw = weight[i][r], fw = mw == -INFINITY ? 0.f : exp2_approx(mw - top), l = r < it.rows ? __ldcg(place_of(i) + 16 + r) : 0.f;
                        sum += mw == -INFINITY ? l : l * fw;
                        weight[i][r] = fw;
                    }
                    sm.o[1][tid / kRows][r] = sum;
                }
                named_bar_sync(1, kWarps * 32);
#pragma unroll
                for (uint32_t k = 0; k < PER; ++k) {
                    const uint32_t e = tid + k * kWarps * 32, r = e / D;
                    float acc = 0.f, sum = 0.f;
                    if (r < it.rows) {
                        for (uint32_t i = 0; i < n; ++i) { const float fw = weight[i][r]; const float v = __ldcg(place_of(i) + kPartHead + e); if (fw != 0.f) acc = fmaf(v, fw, acc); }
                        for (uint32_t i = 0; i < 16; ++i) sum += sm.o[1][i][r];
                    }
                    y[k] = sum == 0.f ? 0.f : acc / sum;
                }
            }
        }
        if (whole || sm.last) {
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k) {
                const uint32_t r = (tid + k * kWarps * 32) / D;
                if (r < it.rows && !(F16 ? fabsf(y[k]) < 65520.f : finite_f32(y[k]))) sm.row_bad[r] = 1;
            }
            named_bar_sync(1, kWarps * 32);
            bool raise = false;
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k) {
                const uint32_t e = tid + k * kWarps * 32, r = e / D, x = e % D;
                if (r < it.rows) {
                    const uint32_t flat = it.tile * kRows + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
                    const bool bad = sm.row_bad[r] != 0;
                    raise |= bad && !all_dead;
                    const float v = bad || all_dead ? 0.f : y[k];
                    uint8_t* dst = p.out + static_cast<uint64_t>(it.row0 + node) * p.out_stride + (head * D + x) * (F16 ? 2 : 4);
                    if constexpr (F16) *reinterpret_cast<__half*>(dst) = __float2half_rn(v); else *reinterpret_cast<float*>(dst) = v;
                }
            }
            if (raise) raise_error(p.error, TSP_ERR_NONFINITE);
        }
        named_bar_sync(1, kWarps * 32);
        if (tid == 0) sm.dead = 0;
        at = stop;
    }
}

uint64_t tree_attention_scratch_bytes() { return sizeof(AttnScratch) + 2ull * kAttnMaxBlocks * part_floats() * sizeof(float); }

template <uint32_t D, bool Q8, bool F16>
static int launch_tree_attention_t(const AttnParams& p, cudaStream_t st) {
    static thread_local SmemAttrCache attr;
    const size_t smem = sizeof(AttnSmem<D, Q8, F16>);
    static_assert(sizeof(AttnSmem<D, Q8, F16>) <= 232448, "shared memory of a block");
    TSP_CUDA(ensure_dynamic_smem(tree_attention_kernel<D, Q8, F16>, attr, smem));
    static thread_local int regs_ok = -1;
    if (regs_ok < 0) {
        cudaFuncAttributes fa;
        TSP_CUDA(cudaFuncGetAttributes(&fa, tree_attention_kernel<D, Q8, F16>));
        regs_ok = fa.numRegs >= kProducerRegs && static_cast<int>(kWarps) * (kConsumerRegs - fa.numRegs) <= static_cast<int>(kProducers) * (fa.numRegs - kProducerRegs);
    }
    if (!regs_ok) return fail(TSP_E_CUDA, "attention: the kernel's register count does not allow its hand-over");
    const uint32_t blocks = static_cast<uint32_t>(sm_count()) < kAttnMaxBlocks ? static_cast<uint32_t>(sm_count()) : kAttnMaxBlocks;
    TSP_CUDA(launch_pdl(tree_attention_kernel<D, Q8, F16>, dim3(blocks ? blocks : 1), dim3(kAttnThreads), smem, st, p));
    return TSP_OK;
}

int launch_tree_attention(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const void* q, uint64_t q_stride, const uint64_t* mask, uint32_t q_heads,
                          uint32_t max_rows, float scale, void* out, uint64_t out_stride, uint32_t dtype, void* scratch, uint32_t* error, cudaStream_t st) {
    AttnScratch* head = static_cast<AttnScratch*>(scratch);
    const AttnParams p{cache, batch, static_cast<const uint8_t*>(q), q_stride, mask, static_cast<uint8_t*>(out), out_stride, q_heads / cache.kv_heads, max_rows, scale,
                       head->counters, reinterpret_cast<float*>(head + 1), error};
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    switch (cache.head_dim) {
        case 64: return q8 ? (dtype ? launch_tree_attention_t<64, true, true>(p, st) : launch_tree_attention_t<64, true, false>(p, st))
                           : (dtype ? launch_tree_attention_t<64, false, true>(p, st) : launch_tree_attention_t<64, false, false>(p, st));
        case 128: return q8 ? (dtype ? launch_tree_attention_t<128, true, true>(p, st) : launch_tree_attention_t<128, true, false>(p, st))
                            : (dtype ? launch_tree_attention_t<128, false, true>(p, st) : launch_tree_attention_t<128, false, false>(p, st));
        default: return q8 ? (dtype ? launch_tree_attention_t<256, true, true>(p, st) : launch_tree_attention_t<256, true, false>(p, st))
                           : (dtype ? launch_tree_attention_t<256, false, true>(p, st) : launch_tree_attention_t<256, false, false>(p, st));
    }
}

}  // namespace tsp
