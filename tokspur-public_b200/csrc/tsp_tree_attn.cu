// Attention of the drafted tokens of every sequence over its paged cache (tsp_tree_attention).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(f q.k_j - m), f = scale log2(e), in one pass over the cache with a running reference m and sum of every row.
//
// The query rows of one kv head (drafted tokens x heads of the group) share the head's keys and values: they are worked on in tiles of R = 8 or 16
// rows by warp MMAs (m16n8k16). With eight rows the slots of the cache (scores) and the dims (values) are the M of the MMAs and the rows their
// N; with sixteen the rows are the M. Work is cut into units of `kUnit` slots of one (sequence, head, row tile) item; the units of the whole
// batch, item after item, are dealt to the blocks in equal runs, so that one long context fills the GPU as a ragged batch does. A block is a
// warpgroup of producers (bulk copies of whole groups of 16 slots into a ring) and the consumer warps, which take the units in turn, each with its
// own reference, sum and accumulators; they join in shared memory when the item or the run ends. An item that spans blocks is joined by
// the last of them to arrive, from the partial results in the scratch, in block order: the same bits every time.
//
// Codes enter the MMAs exactly (binary16 integers). The scale of a key block multiplies the FP32 partial score of its 32 dims, that of a value block the
// FP32 weight before that is rounded to binary16 (relative to a power of two that follows the largest value scale seen): one rounding
// of 2^-11 on the whole path of binary16 rows. FP32 rows split the query (times a power of two) and the weight into two binary16 parts, 22 bits.
#include <type_traits>

#include "tsp_kv.cuh"

namespace tsp {

constexpr uint32_t kProducers = 4;
constexpr uint32_t kAttnMaxBlocks = 192;     // blocks (one per SM) that the scratch has room for
constexpr uint32_t kLeastUnits = 4;          // units of a block's run at least
// The reference of a row moves when a score passes it by more than 2^kSlack: weights stay below 2^(kSlack + 7) = 2^15 in binary16, which then
// reaches down to 2^-31 of the reference.
constexpr float kSlack = 8.f, kUp = 7.f;

// partial result of a run's first or last item: 16 references, 16 sums, a flag, then the rows
constexpr uint32_t kPartHead = 48;
__host__ __device__ constexpr uint64_t part_floats() { return kPartHead + 16 * 256; }

struct AttnParams {
    tsp_kv_cache cache;
    tsp_kv_batch batch;
    const uint8_t* q; uint64_t q_stride;
    const uint64_t* mask;
    uint8_t* out; uint64_t out_stride;
    uint32_t group, max_rows;
    float scale;
    uint32_t* counters;   // [kAttnMaxBlocks], zero between calls
    float* parts;
    uint32_t* error;
};

template <uint32_t D, bool Q8, bool F16, uint32_t R>
struct AttnShape {
    static constexpr uint32_t kWarps = R == 8 && D <= 128 ? 16 : 8, kThreads = 32 * (kWarps + kProducers), kConsumers = 32 * kWarps;
    // Registers after the hand-over between the warpgroups (setmaxnreg): the consumers' request waits for what the producers give back, so
    // kWarps * (kConsumerRegs - launch) <= kProducers * (launch - kProducerRegs) must hold for the count at launch (96 / 168); the launcher checks it.
    static constexpr int kConsumerRegs = kWarps == 16 ? 112 : 224, kProducerRegs = kWarps == 16 ? 32 : 56;
    static constexpr uint32_t kGroupBytes = kv_group_bytes(D, Q8), kHalf = kv_half_bytes(D, Q8);
    static constexpr uint32_t kRing = 139264;
    static constexpr uint32_t kGroups = kGroupBytes * 4 * kWarps <= kRing ? 2 : 1, kUnit = kGroups * kKvGroup, kStage = kGroups * kGroupBytes;
    // A multiple of the warps: a stage then always has the same consumer (and producer), so that nobody waits for a phase while the one before
    // it is open, which a wait by parity would take for done.
    static constexpr uint32_t kStages = kRing / kStage / kWarps * kWarps < 4 * kWarps ? kRing / kStage / kWarps * kWarps : 4 * kWarps;
    static_assert(kStages % kWarps == 0 && kStages % kProducers == 0, "a stage has one consumer and one producer");
    static constexpr uint32_t kSlots = D == 256 ? 4 : kWarps;              // accumulators that meet in shared memory at once
    static constexpr uint32_t kRow = D + (R == 8 ? 4 : D == 256 ? 0 : 8);  // floats between rows there: a warp's stores on 32 banks
};
template <uint32_t D, bool Q8, bool F16, uint32_t R>
struct AttnSmem {
    using S = AttnShape<D, Q8, F16, R>;
    alignas(128) uint8_t ring[S::kStages][S::kStage];
    alignas(16) uint32_t q[F16 ? 1 : 2][D / 16][32][R / 4];   // MMA fragments of the item's rows; binary16 high and low parts of FP32 rows
    alignas(16) float o[S::kSlots * R * S::kRow];
    float m[S::kWarps][R], l[S::kWarps][R], f[S::kWarps][R], sum[R];
    float qscale[R];
    uint64_t words[R];
    uint64_t full[S::kStages], empty[S::kStages];
    uint64_t cum[TSP_KV_MAX_SEQUENCES + 1];
    uint64_t warp_sums[S::kWarps + kProducers];
    uint32_t bad_stage[S::kStages];
    uint32_t row_bad[R];
    uint32_t failed, dead, last;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : exp2_approx(m - top); }
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
// four codes + 128 -> two pairs of binary16 integers: 0x64 in front of a byte is 1024 + byte
__device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    const __half2 bias = bits_h2(0x64806480u);   // 1152
    a = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4140)), bias));
    b = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4342)), bias));
}
// 8 x 8 matrix of binary16 over a warp, transposed: lane (g, t) gives entries (g, 2t), (g, 2t + 1) and gets (2t, g), (2t + 1, g)
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_low(float u, float v, uint32_t high) {   // what rounding to `high` left out
    const float2 f = __half22float2(bits_h2(high));
    return h2_bits(__floats2half2_rn(u - f.x, v - f.y));
}
__device__ __forceinline__ bool odd_half(uint32_t bits) { return (bits & 0x7c00u) == 0x7c00u; }

struct AttnItem {
    uint64_t start, end;     // units of the item
    uint64_t length, total;  // slots of the context, and with the step's own
    uint32_t seq, head, tile, row0, drafted, rows;   // rows: of this tile
    bool dead;               // out of range: zeros
};

// Geometry of a sequence: units of an item, row tiles
template <uint32_t UNIT, uint32_t R>
__device__ __forceinline__ void sequence_shape(const AttnParams& p, uint32_t s, uint32_t& row0, uint32_t& drafted, uint64_t& length, uint64_t& units, uint32_t& tiles, bool& dead) {
    row0 = p.batch.d_row_offsets[s];
    const uint32_t end = p.batch.d_row_offsets[s + 1];
    length = p.batch.d_lengths[s];
    drafted = end >= row0 && end <= p.batch.rows ? end - row0 : 0;
    const uint64_t total = length + drafted;
    dead = drafted > p.max_rows || total > static_cast<uint64_t>(p.cache.table_stride) * p.cache.page_tokens;
    units = dead ? 1 : (total + UNIT - 1) / UNIT;
    tiles = static_cast<uint32_t>((static_cast<uint64_t>(drafted) * p.group + R - 1) / R);
}

template <uint32_t UNIT, uint32_t R>
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
    sequence_shape<UNIT, R>(p, lo, i.row0, i.drafted, i.length, units, tiles, i.dead);
    i.total = i.length + i.drafted;
    const uint64_t rest = u - cum[lo];
    const uint32_t n = rest >> 32 ? static_cast<uint32_t>(rest / units) : static_cast<uint32_t>(rest) / static_cast<uint32_t>(units);
    i.start = cum[lo] + n * units;
    i.end = i.start + units;
    i.head = n / tiles;
    i.tile = n - i.head * tiles;
    i.rows = min(R, i.drafted * p.group - i.tile * R);
    return i;
}

template <uint32_t D, bool Q8, bool F16, uint32_t R>
__global__ void __launch_bounds__(AttnShape<D, Q8, F16, R>::kThreads, 1)
tree_attention_kernel(const AttnParams p) {
    using S = AttnShape<D, Q8, F16, R>;
    constexpr uint32_t UNIT = S::kUnit, NB = D / 32, W = S::kWarps, CT = S::kConsumers, G = S::kGroups;
    extern __shared__ uint8_t raw[];
    AttnSmem<D, Q8, F16, R>& sm = *reinterpret_cast<AttnSmem<D, Q8, F16, R>*>(raw);
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
        const uint32_t per = (p.batch.sequences + S::kThreads - 1) / S::kThreads;   // <= 3
        bool bad = false;
        for (uint32_t k = 0; k < per; ++k) {
            const uint32_t s = tid * per + k;
            mine[k] = sum;
            if (s < p.batch.sequences) {
                uint32_t row0, drafted, tiles;
                uint64_t length, units;
                bool dead;
                sequence_shape<UNIT, R>(p, s, row0, drafted, length, units, tiles, dead);
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
        if (tid == S::kThreads - 1) sm.cum[p.batch.sequences] = base + sum;
        if (blockIdx.x == 0) kv_check_offsets(p.batch, p.error);
        __syncthreads();
    }
    const uint64_t units = sm.cum[p.batch.sequences];
    const uint64_t quota = max(static_cast<uint64_t>(kLeastUnits), (units + gridDim.x - 1) / gridDim.x);
    const uint64_t u0 = min(units, blockIdx.x * quota), u1 = min(units, u0 + quota);
    if (u0 >= u1) return;

    if (warp >= W) {   // producers, every fourth unit each: the lanes look up the sources of 32 units, then the copies go out one after another
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kProducerRegs));
        const uint32_t mine = static_cast<uint32_t>(u1 - u0);
        for (uint32_t base = warp - W; base < mine; base += 32 * kProducers) {
            const uint32_t ahead = base + lane * kProducers;
            const uint8_t* src[G] = {};
            uint32_t groups = 0, bad = 0;
            if (ahead < mine) {
                const AttnItem it = item_of<UNIT, R>(p, sm.cum, u0 + ahead);
                if (it.dead) bad = 1;
                else {
                    const uint64_t slot = (u0 + ahead - it.start) * UNIT;
#pragma unroll
                    for (uint32_t k = 0; k < G; ++k)
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
                const uint8_t* from[G];
#pragma unroll
                for (uint32_t j = 0; j < G; ++j)
                    from[j] = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src[j]), k));
                if (round && !mbar_wait(&sm.empty[st], (round - 1) & 1)) {
                    raise_error(p.error, TSP_ERR_TIMEOUT);
                    return;   // the consumers' own waits run out
                }
                if (elect_one()) {
                    sm.bad_stage[st] = b;
                    mbar_arrive_expect_tx(&sm.full[st], gs * S::kGroupBytes);
                    if (gs == 2 && from[1 % G] == from[0] + S::kGroupBytes) bulk_g2s(sm.ring[st], from[0], 2 * S::kGroupBytes, &sm.full[st]);
                    else {
#pragma unroll
                        for (uint32_t j = 0; j < G; ++j)
                            if (j < gs) bulk_g2s(sm.ring[st] + j * S::kGroupBytes, from[j], S::kGroupBytes, &sm.full[st]);
                    }
                }
                __syncwarp();
            }
        }
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kConsumerRegs));

    for (uint64_t at = u0; at < u1;) {
        const AttnItem it = item_of<UNIT, R>(p, sm.cum, at);
        const uint64_t stop = min(it.end, u1);
        // ---- the item's rows as fragments: step x / 32 * 2 + x % 8 / 4, lane (row % 8, x % 32 / 8), the order in which a lane holds the keys
        named_bar_sync(1, CT);
        for (uint32_t r = warp; r < R; r += W) {
            const uint32_t flat = it.tile * R + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
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
            const uint32_t tt = lane / 8, s = lane % 8 / 4, e = lane % 4;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t step = 2 * b + s, reg = R == 8 ? e / 2 : (r >= 8) + e / 2 * 2, dst = (r % 8) * 4 + tt;
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
        named_bar_sync(1, CT);
        // A lane has two rows (ra, rb) and, of a group of 16 slots, four scores of each with R = 16, two with R = 8. s[group][4 * n + c], with
        // R = 16: row c / 2, slot 8 n + 2 t + c % 2 (MMA n); with R = 8: row c % 2, slot g + 8 (c / 2).
        constexpr uint32_t NS = R == 8 ? 4 : 8;
        const uint32_t ra = R == 8 ? 2 * t : g, rb = R == 8 ? 2 * t + 1 : g + 8;
        auto second = [](uint32_t i) { return R == 8 ? i % 2 != 0 : i % 4 >= 2; };
        auto slot_in = [&](uint32_t i) { return R == 8 ? g + 8 * (i / 2) : 8 * (i / 4) + 2 * t + i % 2; };
        const float fa = sm.qscale[ra], fb = sm.qscale[rb];
        uint32_t qf[F16 && D <= 128 ? D / 16 : 1][R / 4];
        if constexpr (F16 && D <= 128) {
#pragma unroll
            for (uint32_t i = 0; i < D / 16; ++i)
#pragma unroll
                for (uint32_t j = 0; j < R / 4; ++j) qf[i][j] = sm.q[0][i][lane][j];
        }

        // R = 16: [32 dims][n tile][c]: rows g, g + 8; dims 32 b + 8 i + 2 t, + 1. R = 8: [32 dims][m tile][c]: dims 32 b + 16 i + g, + 8; rows 2 t, + 1
        constexpr uint32_t NI = R == 8 ? 2 : 4;
        float o[NB][NI][4];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i)
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) o[b][i][c] = 0.f;
        float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
        [[maybe_unused]] float vup = 0.f;   // Q8_0: power of two that the weights times the value scales are held at
        bool dead = false;

        const uint32_t first = static_cast<uint32_t>(at - u0);
        for (uint32_t li = first + (warp + W - first % W) % W; li < static_cast<uint32_t>(stop - u0); li += W) {
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
                float s[G][NS];
#pragma unroll
                for (uint32_t k = 0; k < G; ++k) {
                    const uint8_t* keys = stage + k * S::kGroupBytes;
#pragma unroll
                    for (uint32_t i = 0; i < NS; ++i) s[k][i] = 0.f;
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b) {   // 32 dims: two steps under one scale
                        uint32_t kb[2][4];                // slots g and g + 8
#pragma unroll
                        for (uint32_t n = 0; n < 2; ++n) {
                            if constexpr (Q8) {
                                const uint2 w = *reinterpret_cast<const uint2*>(keys + (b / 2 * kKvGroup + 8 * n + g) * 64 + t * 16 + b % 2 * 8);
                                codes_to_halves(w.x, kb[n][0], kb[n][1]);
                                codes_to_halves(w.y, kb[n][2], kb[n][3]);
                            } else {
                                const uint4 w = *reinterpret_cast<const uint4*>(keys + (b * kKvGroup + 8 * n + g) * 64 + t * 16);
                                kb[n][0] = w.x; kb[n][1] = w.y; kb[n][2] = w.z; kb[n][3] = w.w;
                            }
                        }
                        float acc[NS / 4][4];
#pragma unroll
                        for (uint32_t n = 0; n < NS / 4; ++n)
#pragma unroll
                            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                                for (uint32_t part = 0; part < (F16 ? 1 : 2); ++part) {
                                    uint32_t q[R / 4];
#pragma unroll
                                    for (uint32_t j = 0; j < R / 4; ++j) {
                                        if constexpr (F16 && D <= 128) q[j] = qf[2 * b + h][j];
                                        else q[j] = sm.q[part][2 * b + h][lane][j];
                                    }
                                    if constexpr (R == 8) {
                                        if (h == 0 && part == 0) mma_f16_16816_zero(acc[n], kb[0][0], kb[1][0], kb[0][1], kb[1][1], q[0], q[1]);
                                        else mma_f16_16816(acc[n], kb[0][2 * h], kb[1][2 * h], kb[0][2 * h + 1], kb[1][2 * h + 1], q[0], q[1]);
                                    } else {
                                        if (h == 0 && part == 0) mma_f16_16816_zero(acc[n], q[0], q[1], q[2 % (R / 4)], q[3 % (R / 4)], kb[n][0], kb[n][1]);
                                        else mma_f16_16816(acc[n], q[0], q[1], q[2 % (R / 4)], q[3 % (R / 4)], kb[n][2 * h], kb[n][2 * h + 1]);
                                    }
                                }
                        if constexpr (Q8) {
                            const uint8_t* scales = keys + kKvGroup * D + b * kKvGroup * 2;
                            if constexpr (R == 8) {
                                const float d0 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2)), d1 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2 + 16));
                                s[k][0] = fmaf(acc[0][0], d0, s[k][0]); s[k][1] = fmaf(acc[0][1], d0, s[k][1]);
                                s[k][2] = fmaf(acc[0][2], d1, s[k][2]); s[k][3] = fmaf(acc[0][3], d1, s[k][3]);
                            } else {
#pragma unroll
                                for (uint32_t n = 0; n < NS / 4; ++n) {
                                    const float2 d = __half22float2(*reinterpret_cast<const __half2*>(scales + (8 * n + 2 * t) * 2));
#pragma unroll
                                    for (uint32_t c = 0; c < 4; ++c) s[k][4 * n + c] = fmaf(acc[n][c], c & 1 ? d.y : d.x, s[k][4 * n + c]);
                                }
                            }
                        } else {
#pragma unroll
                            for (uint32_t i = 0; i < NS; ++i) s[k][i] += acc[i / 4][i % 4];
                        }
                    }
                }
                float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
                for (uint32_t k = 0; k < G; ++k)
#pragma unroll
                    for (uint32_t i = 0; i < NS; ++i) s[k][i] *= second(i) ? fb : fa;
                // At the end of the context: what a row does not see gets no weight. Drafted slots whose values are not finite give the rows that see
                // them NaN through the weight, and count as zero themselves; slots behind the last count as zero, whatever they hold.
                [[maybe_unused]] uint32_t drop[G] = {};   // bit i: slot i of the group
                if (edge) {
                    const uint64_t wa = sm.words[ra], wb = sm.words[rb];
#pragma unroll
                    for (uint32_t k = 0; k < G; ++k) {
                        const uint8_t* values = stage + k * S::kGroupBytes + S::kHalf;
                        const uint64_t base = slot0 + k * kKvGroup;
                        uint32_t odd = 0;
                        const uint32_t there = base >= it.total ? 0u : it.total - base >= 16 ? 0xffffu : (1u << static_cast<uint32_t>(it.total - base)) - 1;
                        const uint32_t drafted = base >= it.length ? 0xffffu : it.length - base >= 16 ? 0u : 0xffffu << static_cast<uint32_t>(it.length - base);
                        if constexpr (Q8) {
                            for (uint32_t i = lane; i < NB * kKvGroup; i += 32)
                                odd |= static_cast<uint32_t>(odd_half(*reinterpret_cast<const uint16_t*>(values + kKvGroup * D + i * 2))) << i % kKvGroup;
                        } else {
                            for (uint32_t i = 0; i < D / 8; ++i)   // 32-dim block, half: eight bytes of four slots a lane
#pragma unroll
                                for (uint32_t e = 0; e < 4; ++e)
                                    odd |= static_cast<uint32_t>(odd_half(*reinterpret_cast<const uint16_t*>(values + (i / 2 * 32 + lane) * 16 + i % 2 * 8 + e * 2))) << (2 * t + (e & 1) + 8 * (e >> 1));
                        }
                        odd = __reduce_or_sync(0xffffffffu, odd) & drafted & there;
                        drop[k] = odd | (~there & 0xffffu);
#pragma unroll
                        for (uint32_t i = 0; i < NS; ++i) {
                            const uint32_t at_slot = slot_in(i);
                            const uint64_t word = second(i) ? wb : wa;
                            const bool seen = there >> at_slot & 1 && (!(drafted >> at_slot & 1) || (word >> (base + at_slot - it.length) & 1));
                            if (!seen) s[k][i] = -INFINITY;
                            else if (odd >> at_slot & 1) s[k][i] = NAN;
                        }
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < G; ++k)
#pragma unroll
                    for (uint32_t i = 0; i < NS; ++i) { if (second(i)) xb = fmaxf(xb, s[k][i]); else xa = fmaxf(xa, s[k][i]); }
                bool move = xa > ma + kSlack || xb > mb + kSlack;
                [[maybe_unused]] float up = vup;
                if constexpr (Q8) {   // largest value scale of the unit: the lanes have a part each
                    uint32_t top = 0;
#pragma unroll
                    for (uint32_t k = 0; k < G; ++k)
                        for (uint32_t i = lane; i < NB * kKvGroup / 2; i += 32) {
                            uint32_t d = *reinterpret_cast<const uint32_t*>(stage + k * S::kGroupBytes + S::kHalf + kKvGroup * D + i * 4) & 0x7fff7fffu;
                            const uint32_t out = drop[k] >> (i * 2 % kKvGroup);
                            if (out & 1) d &= 0xffff0000u;
                            if (out & 2) d &= 0x0000ffffu;
                            top = max(top, max(d & 0xffffu, d >> 16));
                        }
                    // the scale is below 2^(e - 14) (binary16 exponent field e, subnormals 2^-14): weights up to 2^kSlack times it times up stay below 2^15
                    const float limit = __uint_as_float((127u + 21u - min(max(top >> 10, 1u), 31u)) << 23);   // 2^(21 - e)
                    move |= vup == 0.f || limit < vup;
                    up = limit;
                }
                if (__any_sync(0xffffffffu, move)) {
                    if constexpr (R == 8) {
#pragma unroll
                        for (uint32_t x = 4; x < 32; x *= 2) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, x)); }
                    } else {
#pragma unroll
                        for (uint32_t x = 1; x < 4; x *= 2) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, x)); }
                    }
                    xa = fmaxf(xa, ma); xb = fmaxf(xb, mb);
                    float r0 = weight_of(ma, xa), r1 = weight_of(mb, xb);
                    la *= r0; lb *= r1;
                    ma = xa; mb = xb;
                    if constexpr (Q8) {
                        up = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(up)));
                        if (vup != 0.f) { up = fminf(up, vup); const float r = up / vup; r0 *= r; r1 *= r; }
                        vup = up;
                    }
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                        for (uint32_t i = 0; i < NI; ++i)
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) o[b][i][c] *= second(c) ? r1 : r0;
                }
                // without value scales the weights themselves are held up to 2^15
                constexpr float lift = Q8 ? 0.f : kUp;
                const float ba = ma == -INFINITY ? 0.f : ma - lift, bb = mb == -INFINITY ? 0.f : mb - lift;
#pragma unroll
                for (uint32_t k = 0; k < G; ++k) {
                    const uint8_t* values = stage + k * S::kGroupBytes + S::kHalf;
                    float pr[NS];
#pragma unroll
                    for (uint32_t i = 0; i < NS; ++i) {
                        pr[i] = exp2_approx(s[k][i] - (second(i) ? bb : ba));
                        if (second(i)) lb += pr[i]; else la += pr[i];
                    }
                    uint32_t keep[2];   // binary16 values of slots 2t, 2t + 1 and 8 more
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n)
                        keep[n] = (drop[k] >> (8 * n + 2 * t) & 1 ? 0u : 0x0000ffffu) | (drop[k] >> (8 * n + 2 * t) & 2 ? 0u : 0xffff0000u);
                    uint32_t a[R / 4], al[R / 4];
                    auto split = [&](const float (&w)[NS]) {   // R = 16: A fragment (rows g, g + 8; slots 2t.., 8 more); R = 8: B fragment, slots 2t.., 8 more, row g
#pragma unroll
                        for (uint32_t r = 0; r < R / 4; ++r) {
                            a[r] = h2_bits(__floats2half2_rn(w[2 * r], w[2 * r + 1]));
                            if constexpr (!F16) al[r] = pack_low(w[2 * r], w[2 * r + 1], a[r]);
                            if constexpr (R == 8) {
                                a[r] = transposed(a[r]);
                                if constexpr (!F16) al[r] = transposed(al[r]);
                            }
                        }
                    };
                    if constexpr (!Q8) split(pr);
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b) {
                        uint32_t vb[8];   // dims 8 i + g: slots 2t, 2t + 1 in vb[2 i], 8 further in vb[2 i + 1]
                        if constexpr (Q8) {
                            const uint4 w = *reinterpret_cast<const uint4*>(values + b * 512 + lane * 16);
                            codes_to_halves(w.x, vb[0], vb[1]); codes_to_halves(w.y, vb[2], vb[3]);
                            codes_to_halves(w.z, vb[4], vb[5]); codes_to_halves(w.w, vb[6], vb[7]);
                            const uint8_t* scales = values + kKvGroup * D + b * kKvGroup * 2;
                            float w4[NS];
                            if constexpr (R == 8) {
                                float d0 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2)) * vup, d1 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2 + 16)) * vup;
                                if (edge) { if (drop[k] >> g & 1) d0 = 0.f; if (drop[k] >> (g + 8) & 1) d1 = 0.f; }
                                w4[0] = pr[0] * d0; w4[1] = pr[1] * d0; w4[2] = pr[2] * d1; w4[3] = pr[3] * d1;
                            } else {
#pragma unroll
                                for (uint32_t n = 0; n < NS / 4; ++n) {
                                    const float2 f = __half22float2(bits_h2(*reinterpret_cast<const uint32_t*>(scales + (8 * n + 2 * t) * 2) & (edge ? keep[n] : 0xffffffffu)));
                                    const float dx = f.x * vup, dy = f.y * vup;
#pragma unroll
                                    for (uint32_t c = 0; c < 4; ++c) w4[4 * n + c] = pr[4 * n + c] * (c & 1 ? dy : dx);
                                }
                            }
                            split(w4);
                        } else {
                            const uint4 w = *reinterpret_cast<const uint4*>(values + b * 1024 + lane * 16), x = *reinterpret_cast<const uint4*>(values + b * 1024 + 512 + lane * 16);
                            vb[0] = w.x; vb[1] = w.y; vb[2] = w.z; vb[3] = w.w; vb[4] = x.x; vb[5] = x.y; vb[6] = x.z; vb[7] = x.w;
                            if (edge) {
#pragma unroll
                                for (uint32_t i = 0; i < 8; ++i) vb[i] &= keep[i & 1];
                            }
                        }
#pragma unroll
                        for (uint32_t i = 0; i < NI; ++i) {
                            auto product = [&](float (&acc)[4], const uint32_t (&w)[R / 4], bool fresh) {
                                if constexpr (R == 8) {
                                    if (fresh) mma_f16_16816_zero(acc, vb[4 * i % 8], vb[(4 * i + 2) % 8], vb[(4 * i + 1) % 8], vb[(4 * i + 3) % 8], w[0], w[1]);
                                    else mma_f16_16816(acc, vb[4 * i % 8], vb[(4 * i + 2) % 8], vb[(4 * i + 1) % 8], vb[(4 * i + 3) % 8], w[0], w[1]);
                                } else {
                                    if (fresh) mma_f16_16816_zero(acc, w[0], w[1], w[2 % (R / 4)], w[3 % (R / 4)], vb[2 * i], vb[2 * i + 1]);
                                    else mma_f16_16816(acc, w[0], w[1], w[2 % (R / 4)], w[3 % (R / 4)], vb[2 * i], vb[2 * i + 1]);
                                }
                            };
                            if constexpr (F16) product(o[b][i], a, false);
                            else {   // the tensor core cuts its sums off: a chain of two products, added up rounded
                                float acc[4];
                                product(acc, a, true);
                                product(acc, al, false);
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
#pragma unroll
        for (uint32_t x = R == 8 ? 4 : 1; x < (R == 8 ? 32 : 4); x *= 2) { la += __shfl_xor_sync(0xffffffffu, la, x); lb += __shfl_xor_sync(0xffffffffu, lb, x); }
        if constexpr (Q8) {
            const float down = vup == 0.f ? 0.f : 1.f / vup;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < NI; ++i)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) o[b][i][c] *= down;
        }
        const bool speaker = R == 8 ? g == 0 : t == 0;
        if (speaker) { sm.m[warp][ra] = ma; sm.m[warp][rb] = mb; sm.l[warp][ra] = la; sm.l[warp][rb] = lb; }
        if (dead && lane == 0) sm.dead = 1;
        auto each = [&](uint32_t slot, auto&& f) {   // a lane's accumulators beside their places in `slot`
            float* base = sm.o + slot * R * S::kRow;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < NI; ++i)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) {
                        const uint32_t r = second(c) ? rb : ra, x = R == 8 ? b * 32 + i * 16 + g + 8 * (c / 2) : b * 32 + i * 8 + 2 * t + c % 2;
                        if (r < it.rows) f(base[r * S::kRow + x], o[b][i][c], c);
                    }
        };
#pragma unroll
        for (uint32_t half = W / 2; half >= S::kSlots; half /= 2) {   // wide heads: the upper warps hand theirs to the lower ones until they fit
            if (warp >= half && warp < 2 * half) each(warp - half, [](float& place, float v, uint32_t) { place = v; });
            named_bar_sync(1, CT);
            if (warp < half) {
                const uint32_t other = warp + half;
                const float na = sm.m[other][ra], nb = sm.m[other][rb], xa = fmaxf(ma, na), xb = fmaxf(mb, nb);
                const float a0 = weight_of(ma, xa), a1 = weight_of(mb, xb), b0 = weight_of(na, xa), b1 = weight_of(nb, xb);
                each(warp, [&](float& place, float& v, uint32_t c) {
                    const float w = second(c) ? b1 : b0;
                    v = v * (second(c) ? a1 : a0) + (w == 0.f ? 0.f : place * w);
                });
                // a row of NaN alone has a sum of NaN and no reference
                la = (ma == -INFINITY ? la : la * a0) + (na == -INFINITY ? sm.l[other][ra] : sm.l[other][ra] * b0);
                lb = (mb == -INFINITY ? lb : lb * a1) + (nb == -INFINITY ? sm.l[other][rb] : sm.l[other][rb] * b1);
                ma = xa; mb = xb;
                __syncwarp();
                if (speaker) { sm.m[warp][ra] = ma; sm.m[warp][rb] = mb; sm.l[warp][ra] = la; sm.l[warp][rb] = lb; }
            }
            named_bar_sync(1, CT);
        }
        if (warp < S::kSlots) each(warp, [](float& place, float v, uint32_t) { place = v; });
        named_bar_sync(1, CT);
        const bool whole = at == it.start && stop == it.end;
        const uint32_t c0 = static_cast<uint32_t>(it.start / quota), c1 = static_cast<uint32_t>((it.end - 1) / quota);
        bool all_dead = sm.dead != 0;
        float* part = p.parts + (2 * blockIdx.x + (at == u0 ? 0 : 1)) * part_floats();
        if (tid < R * S::kSlots) {   // a thread per (slot, row)
            const uint32_t r = tid % R, w = tid / R;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < S::kSlots; ++i) top = fmaxf(top, sm.m[i][r]);
            sm.f[w][r] = weight_of(sm.m[w][r], top);
            if (w == 0) {
#pragma unroll
                for (uint32_t i = 0; i < S::kSlots; ++i) sum += sm.m[i][r] == -INFINITY ? sm.l[i][r] : sm.l[i][r] * weight_of(sm.m[i][r], top);
                sm.sum[r] = sum;
                if (!whole) { __stcg(part + r, top); __stcg(part + 16 + r, sum); }
            }
        }
        if (!whole && tid == 0) __stcg(part + 32, all_dead ? 1.f : 0.f);
        named_bar_sync(1, CT);
        constexpr uint32_t PER = (R * D / 4 + CT - 1) / CT;   // units of four dims a thread
        const uint32_t units4 = it.rows * (D / 4);
        float4 y[PER];
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const uint32_t e = tid + k * CT, r = e / (D / 4), x = e % (D / 4) * 4;
            y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (e < units4) {
#pragma unroll
                for (uint32_t w = 0; w < S::kSlots; ++w) {
                    const float fw = sm.f[w][r];
                    const float4 v = *reinterpret_cast<const float4*>(sm.o + (w * R + r) * S::kRow + x);
                    if (fw != 0.f) { y[k].x = fmaf(v.x, fw, y[k].x); y[k].y = fmaf(v.y, fw, y[k].y); y[k].z = fmaf(v.z, fw, y[k].z); y[k].w = fmaf(v.w, fw, y[k].w); }
                }
                if (!whole) __stcg(reinterpret_cast<float4*>(part + kPartHead) + e, y[k]);
            }
        }
        bool finish = whole;
        if (!whole) {
            __threadfence();
            named_bar_sync(1, CT);
            if (tid == 0) {
                const uint32_t n = atomicAdd(p.counters + c0, 1u);
                sm.last = n == c1 - c0;
                if (sm.last) { p.counters[c0] = 0; sm.dead = 0; }
            }
            named_bar_sync(1, CT);
            finish = sm.last != 0;
            if (finish) {
                __threadfence();
                const uint32_t n = c1 - c0 + 1;
                const float* part0 = p.parts + (2 * c0 + (c0 * quota != it.start ? 1 : 0)) * part_floats();
                const float* part1 = p.parts + 2 * (c0 + 1) * part_floats();
                auto part_of = [&](uint32_t i) { return i == 0 ? part0 : part1 + 2 * (i - 1) * part_floats(); };
                // weights of the partial results, [n][R] from the start of the accumulators on, behind them a reference and a sum per (run of CT / R, row)
                float* weight = sm.o;
                float* share = sm.o + kAttnMaxBlocks * R;
                const uint32_t r = tid % R, lot = tid / R;
                constexpr uint32_t LOTS = CT / R;
                float top = -INFINITY;
                for (uint32_t i = lot; i < n; i += LOTS) {
                    const float v = r < it.rows ? __ldcg(part_of(i) + r) : -INFINITY;
                    weight[i * R + r] = v;
                    top = fmaxf(top, v);
                    if (r == 0 && __ldcg(part_of(i) + 32) != 0.f) sm.dead = 1;
                }
                share[tid] = top;
                named_bar_sync(1, CT);
                all_dead = sm.dead != 0;
                for (uint32_t i = 0; i < LOTS; ++i) top = fmaxf(top, share[i * R + r]);
                float sum = 0.f;
                for (uint32_t i = lot; i < n; i += LOTS) {
                    const float v = weight[i * R + r], f = weight_of(v, top), l = r < it.rows ? __ldcg(part_of(i) + 16 + r) : 0.f;
                    sum += v == -INFINITY ? l : l * f;
                    weight[i * R + r] = f;
                }
                share[CT + tid] = sum;
                named_bar_sync(1, CT);
                if (lot == 0) {
                    for (uint32_t i = 1; i < LOTS; ++i) sum += share[CT + i * R + r];
                    sm.sum[r] = sum;
                }
                // the rows: `lanes` threads a unit, each every lanes-th partial result, several loads in flight
                const uint32_t lanes = units4 * 8 <= CT ? 8 : units4 * 4 <= CT ? 4 : units4 * 2 <= CT ? 2 : 1, mine = tid % lanes;
                for (uint32_t k = 0; k < PER; ++k) {
                    const uint32_t e = tid / lanes + k * CT;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (e < units4) {
                        const uint32_t er = e / (D / 4);
                        for (uint32_t i0 = mine; i0 < n; i0 += 8 * lanes) {
                            float4 v[8];
#pragma unroll
                            for (uint32_t j = 0; j < 8; ++j)
                                if (i0 + j * lanes < n) v[j] = __ldcg(reinterpret_cast<const float4*>(part_of(i0 + j * lanes) + kPartHead) + e);
#pragma unroll
                            for (uint32_t j = 0; j < 8; ++j)
                                if (i0 + j * lanes < n) {
                                    const float f = weight[(i0 + j * lanes) * R + er];
                                    if (f != 0.f) { acc.x = fmaf(v[j].x, f, acc.x); acc.y = fmaf(v[j].y, f, acc.y); acc.z = fmaf(v[j].z, f, acc.z); acc.w = fmaf(v[j].w, f, acc.w); }
                                }
                        }
                    }
                    for (uint32_t x = 1; x < lanes; x *= 2) {
                        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, x); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, x);
                        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, x); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, x);
                    }
                    y[k] = acc;
                    if (lanes > 1) break;   // one unit a thread
                }
                named_bar_sync(1, CT);
                if (lanes > 1) {   // back to a unit a thread, through the free end of the accumulators
                    float4* swap = reinterpret_cast<float4*>(share + 2 * CT);
                    if (mine == 0 && tid / lanes < units4) swap[tid / lanes] = y[0];
                    named_bar_sync(1, CT);
                    if (tid < units4) y[0] = swap[tid];
                }
            }
        }
        if (finish) {
            bool raise = false;
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k) {
                const uint32_t e = tid + k * CT, r = e / (D / 4);
                if (e < units4) {
                    const float sum = sm.sum[r], inv = sum == 0.f ? 0.f : 1.f / sum;
                    y[k].x *= inv; y[k].y *= inv; y[k].z *= inv; y[k].w *= inv;
                    const float top = fmaxf(fmaxf(fabsf(y[k].x), fabsf(y[k].y)), fmaxf(fabsf(y[k].z), fabsf(y[k].w)));
                    if (!(F16 ? top < 65520.f : finite_f32(top)) || y[k].x != y[k].x || y[k].y != y[k].y || y[k].z != y[k].z || y[k].w != y[k].w) sm.row_bad[r] = 1;
                }
            }
            named_bar_sync(1, CT);
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k) {
                const uint32_t e = tid + k * CT, r = e / (D / 4), x = e % (D / 4) * 4;
                if (e < units4) {
                    const uint32_t flat = it.tile * R + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
                    const bool bad = sm.row_bad[r] != 0;
                    raise |= bad && !all_dead;
                    if (bad || all_dead) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    uint8_t* dst = p.out + static_cast<uint64_t>(it.row0 + node) * p.out_stride + (head * D + x) * (F16 ? 2 : 4);
                    if constexpr (F16) *reinterpret_cast<uint2*>(dst) = make_uint2(h2_bits(__floats2half2_rn(y[k].x, y[k].y)), h2_bits(__floats2half2_rn(y[k].z, y[k].w)));
                    else *reinterpret_cast<float4*>(dst) = y[k];
                }
            }
            if (raise) raise_error(p.error, TSP_ERR_NONFINITE);
        }
        named_bar_sync(1, CT);
        if (tid == 0) sm.dead = 0;
        at = stop;
    }
}

uint64_t tree_attention_scratch_bytes() { return kAttnMaxBlocks * sizeof(uint32_t) + 2ull * kAttnMaxBlocks * part_floats() * sizeof(float); }

template <uint32_t D, bool Q8, bool F16, uint32_t R>
static int launch_tree_attention_t(const AttnParams& p, cudaStream_t st) {
    using S = AttnShape<D, Q8, F16, R>;
    using Smem = AttnSmem<D, Q8, F16, R>;
    static_assert(sizeof(Smem) <= 232448, "shared memory of a block");
    static_assert(S::kSlots * R * S::kRow >= kAttnMaxBlocks * R + 2 * S::kConsumers + 2 * S::kConsumers && (kAttnMaxBlocks * R) % 4 == 0, "the join fits the accumulators' place");
    auto kernel = tree_attention_kernel<D, Q8, F16, R>;
    static thread_local int regs_ok = -1;
    if (regs_ok < 0) {
        cudaFuncAttributes fa;
        TSP_CUDA(cudaFuncGetAttributes(&fa, kernel));
        regs_ok = fa.numRegs >= S::kProducerRegs &&
                  static_cast<int>(S::kWarps) * (S::kConsumerRegs - fa.numRegs) <= static_cast<int>(kProducers) * (fa.numRegs - S::kProducerRegs);
    }
    if (!regs_ok) return fail(TSP_E_CUDA, "attention: the kernel's register count does not allow its hand-over");
    static thread_local SmemAttrCache attr;
    TSP_CUDA(ensure_dynamic_smem(kernel, attr, sizeof(Smem)));
    const int sms = sm_count();
    const uint32_t blocks = sms < 1 ? 1 : sms < static_cast<int>(kAttnMaxBlocks) ? sms : kAttnMaxBlocks;
    TSP_CUDA(launch_pdl(kernel, dim3(blocks), dim3(S::kThreads), sizeof(Smem), st, p));
    return TSP_OK;
}

template <uint32_t D, bool Q8>
static int launch_tree_attention_d(const AttnParams& p, bool f16, cudaStream_t st) {
    // The narrow tile takes half the instructions of the wide one where the rows fit it
    const bool narrow = static_cast<uint64_t>(p.max_rows) * p.group <= 8;
    if (f16) return narrow ? launch_tree_attention_t<D, Q8, true, 8>(p, st) : launch_tree_attention_t<D, Q8, true, 16>(p, st);
    return narrow ? launch_tree_attention_t<D, Q8, false, 8>(p, st) : launch_tree_attention_t<D, Q8, false, 16>(p, st);
}

int launch_tree_attention(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const void* q, uint64_t q_stride, const uint64_t* mask, uint32_t q_heads,
                          uint32_t max_rows, float scale, void* out, uint64_t out_stride, uint32_t dtype, void* scratch, uint32_t* error, cudaStream_t st) {
    uint32_t* counters = static_cast<uint32_t*>(scratch);
    const AttnParams p{cache, batch, static_cast<const uint8_t*>(q), q_stride, mask, static_cast<uint8_t*>(out), out_stride, q_heads / cache.kv_heads, max_rows, scale,
                       counters, reinterpret_cast<float*>(counters + kAttnMaxBlocks), error};
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    switch (cache.head_dim) {
        case 64: return q8 ? launch_tree_attention_d<64, true>(p, dtype, st) : launch_tree_attention_d<64, false>(p, dtype, st);
        case 128: return q8 ? launch_tree_attention_d<128, true>(p, dtype, st) : launch_tree_attention_d<128, false>(p, dtype, st);
        default: return q8 ? launch_tree_attention_d<256, true>(p, dtype, st) : launch_tree_attention_d<256, false>(p, dtype, st);
    }
}

}  // namespace tsp
