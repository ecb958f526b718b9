// Attention of the drafted tokens of every sequence over its paged cache (tsp_tree_attention).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(f q.k_j - ref), f = scale log2(e), in one pass over the cache with a running reference and sum of every row.
//
// The query rows of one kv head (drafted tokens x heads of the group) share the head's keys and values: they are worked on in tiles of eight
// rows by warp MMAs (m16n8k16): the slots of the cache (scores) and the dims (values) are the M of the MMAs and the rows their N. (Tiles of sixteen
// rows, as the M of the MMAs, halve the reads of the cache, which come from the L2 anyway, and leave registers for eight warps instead of sixteen:
// 32 sequences of 4 rows x 4 heads over 4000 slots 72 us against 62, FP32 rows 89 against 77.) Work is cut into units of 16 slots of one
// (sequence, head, row tile) item; the units of the whole batch, item after item, are dealt to the blocks in equal runs and a block's run to its
// warps, so that one long context fills the GPU as a ragged batch does.
// A warp is on its own until the end of its run: it copies its units into its own ring of stages (bulk copies, a group of 16 slots is one contiguous
// piece), keeps reference, sum and accumulators in registers, and writes the rows of an item that lies within its run. Pieces of items
// that do not (two a warp at most) meet at the end of the block, and what still is a piece there goes to the scratch, where the last block of the
// item to arrive joins them, in order: the same bits every time. (Warps that took the units of one item in turn and met at its end: a ragged
// batch of 64 contexts 187 us, and 128 so.) Every lane fences the asynchronous proxy between its reads of a stage and the copy that fills it again: no time in
// these figures but 1 % of the chains of 256 dims, whose units are two stages.
//
// Measured, Q8_0 and binary16 rows of 32 heads over 8 kv heads of 128 dims: 64 sequences of up to 8192 slots, a token each, 128 us, 644 MB of cache at
// 5.0 TB/s, bound by instructions (unpacking, 53 % of the issue slots) and by the ragged runs' ends; FP32 rows 139. One token over 4096 slots 15.8 us, bound by a
// chain of latencies (table, copy, cold instructions, the join of a head's blocks). FP32 rows, 6 chains of up to 8 tokens x 8 heads over 6000 slots
// of binary16, 256 dims: 41.8 us, bound by the instructions of the split products (640 for the 64 MMAs of a unit and tile) at eight warps an SM.
//
// Codes enter the MMAs exactly (binary16 integers). The scale of a key block multiplies the FP32 partial score of its 32 dims, that of a value block the
// FP32 weight before that is rounded to binary16: one rounding of 2^-11 on the whole path of binary16 rows. FP32 rows split the query (times a
// power of two) and the weight into two binary16 parts, 22 bits.
#include <type_traits>

#include "tsp_tree_attn.cuh"

namespace tsp {

constexpr uint32_t kTile = 8;          // rows
constexpr uint32_t kLeastUnits = 8;    // of a block's run: one token over 1000 slots 13.2 us, 14.8 with sixteen
constexpr uint32_t kPartHead = 32;   // floats in front of a piece's rows: references, sums, a flag
__host__ __device__ constexpr uint64_t part_floats() { return kPartHead + kTile * 256; }
constexpr uint32_t kMaxWarps = 16;   // AttnParams::parts: [2 kAttnMaxBlocks] pieces of blocks, then [kAttnMaxBlocks][kMaxWarps] of warps

template <uint32_t D, bool Q8>
struct AttnShape {
    static constexpr uint32_t kGroupBytes = kv_group_bytes(D, Q8), kHalf = kv_half_bytes(D, Q8);
    // A stage holds a group, or its keys or values alone where three groups for each of eight warps do not fit shared memory (256 dims of binary16: 51 us for six
    // chains with four warps and whole groups, 41.5 so)
    static constexpr uint32_t kPieces = 8 * 3 * kGroupBytes <= 212992 ? 1 : 2, kPiece = kGroupBytes / kPieces;
    // Warps: as many as the registers allow (128 a thread with sixteen) and as three stages each fit shared memory
    static constexpr uint32_t kWarps = 16 * 3 * kPiece <= 212992 && kPieces == 1 ? 16 : 8, kThreads = 32 * kWarps;
    static constexpr uint32_t kStages = 212992 / (kWarps * kPiece) < 6 ? 212992 / (kWarps * kPiece) : 6;
    static constexpr uint32_t kRing = kStages * kPiece;   // a warp's
    static_assert(kStages >= 3 && kRing >= (kTile * D + kPartHead) * 4, "a warp's last piece lies in its ring");
};
template <uint32_t D, bool Q8>
struct AttnSmem {
    using S = AttnShape<D, Q8>;
    alignas(128) uint8_t ring[S::kWarps][S::kRing];
    uint64_t full[S::kWarps][S::kStages];
    uint64_t cum[TSP_KV_MAX_SEQUENCES + 1];
    uint64_t warp_sums[S::kWarps];
    uint64_t key[S::kWarps][2];              // first unit of the item that a piece belongs to, ~0: none
    alignas(16) float meet[S::kWarps * D];
    AttnItem item[S::kWarps][2];             // and the item itself
    AttnItem edge[2];                        // items of the run's first and last unit
    uint32_t last[2], span[2][2];            // whether the block joins its first / last item; the item's blocks
};

template <uint32_t D, bool Q8, bool F16>
__global__ void __launch_bounds__(AttnShape<D, Q8>::kThreads, 1)
tree_attention_kernel(const AttnParams p) {
    using S = AttnShape<D, Q8>;
    constexpr uint32_t NB = D / 32, W = S::kWarps, P = S::kStages, NONE = 0xffffffffu;
    extern __shared__ uint8_t raw[];
    AttnSmem<D, Q8>& sm = *reinterpret_cast<AttnSmem<D, Q8>*>(raw);
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;
    pdl_launch_dependents();
    if (lane < P) mbar_init(&sm.full[warp][lane], 1);
    mbar_fence_init();
    pdl_wait();
    if (lane < 2) sm.key[warp][lane] = ~0ull;
    unit_prefix<kTile, kKvGroup, S::kThreads>(p, sm.cum, sm.warp_sums);
    const uint64_t units = sm.cum[p.batch.sequences];
    if (!units) return;
    const AttnRuns runs(p, units, item_of<kTile>(p, sm.cum, 0), kLeastUnits);
    uint64_t u0, u1;
    runs.run(blockIdx.x, units, u0, u1);
    if (u0 >= u1) return;

    // ---- a warp's run. A lane has two rows (ra, rb) and, of a unit's 16 slots, two scores of each: s[c] of row c % 2, slot g + 8 (c / 2)
    constexpr uint32_t NS = 4;
    const uint32_t ra = 2 * t, rb = 2 * t + 1;
    auto second = [](uint32_t i) { return i % 2 != 0; };
    auto slot_in = [&](uint32_t i) { return g + 8 * (i / 2); };
    float* const warp_part = p.parts + (2ull * kAttnMaxBlocks + blockIdx.x * kMaxWarps + warp) * part_floats();
    {
        // warps without a unit are the last ones: the pieces of an item lie in neighbouring rings
        const uint32_t n = static_cast<uint32_t>(u1 - u0), mine = n / W + (warp < n % W);
        const uint64_t a = u0 + warp * (n / W) + min(warp, n % W), b = a + mine;
        constexpr uint32_t PIECES = S::kPieces;
        uint64_t src = 0;              // lane i: source of unit i of the 32 that `issued` is in
        uint32_t issued = 0, gone = 0; // issued: pieces; gone, bit st: the unit in stage st has no page
        auto issue = [&](uint32_t st) {
            if (issued >= mine * PIECES) return;
            if (issued % (32 * PIECES) == 0) {
                src = 0;
                const uint64_t u = a + issued / PIECES + lane;
                if (u < b) {
                    const AttnItem x = item_of<kTile>(p, sm.cum, u);
                    if (!x.dead) src = reinterpret_cast<uint64_t>(kv_group(p.cache, x.seq, (u - x.start) * kKvGroup, x.head, p.error));
                }
            }
            uint64_t from = __shfl_sync(NONE, src, issued / PIECES % 32);
            if (from) from += issued % PIECES * S::kPiece;
            gone = (gone & ~(1u << st)) | (from ? 0u : 1u << st);
            if (elect_one()) {
                mbar_arrive_expect_tx(&sm.full[warp][st], from ? S::kPiece : 0);
                if (from) bulk_g2s(sm.ring[warp] + st * S::kPiece, reinterpret_cast<const void*>(from), S::kPiece, &sm.full[warp][st]);
            }
            __syncwarp();
            ++issued;
        };
        for (uint32_t i = 0; i < P; ++i) issue(i);
        uint32_t stage = 0, phase = 0;

        bool lost = false;   // a wait has run out
        for (uint32_t done = 0; done < mine;) {
            const AttnItem it = item_of<kTile>(p, sm.cum, a + done);
            const uint32_t stop = static_cast<uint32_t>(min(it.end, b) - a);
            if (lane == 0) { if (a + done == u0) sm.edge[0] = it; if (a + stop == u1) sm.edge[1] = it; }
            // ---- the item's rows as fragments: step 2 b + h holds, in lane (row % 8, t), dims 32 b + 8 t + 4 h + 0..3, the order of a lane's keys
            uint32_t qf[F16 ? 1 : 2][D / 16][2];
            float fa, fb;
            [[maybe_unused]] float start[NB][2];   // Q8_0, binary16 rows: -1152 times the sum of the row's 32 dims
            auto row_of = [&](uint32_t r, uint32_t& node, uint32_t& head) {
                const uint32_t flat = it.tile * kTile + r;
                node = flat / p.group;
                head = it.head * p.group + flat % p.group;
            };
            {
                // Not 0: it multiplies minus infinity. Sums of products of binary16 rows are below 2^47, those of FP32 rows with their power of two below 2^46: no weight
                // shows what these floors add.
                if constexpr (F16) fa = fb = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 0x1p-83f);
                uint32_t node, head;
                row_of(g, node, head);   // the fragments' row
                const uint8_t* row = p.q + static_cast<uint64_t>(it.row0 + node) * p.q_stride + head * D * (F16 ? 2u : 4u);
                const bool there = g < it.rows;
                if constexpr (F16) {
                    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k) {
                        const uint4 v = there ? *reinterpret_cast<const uint4*>(row + (k * 32 + 8 * t) * 2) : make_uint4(0, 0, 0, 0);
                        qf[0][2 * k][0] = v.x ^ flip; qf[0][2 * k][1] = v.y ^ flip;
                        qf[0][2 * k + 1][0] = v.z ^ flip; qf[0][2 * k + 1][1] = v.w ^ flip;
                    }
                } else {   // the row times a power of two that puts its largest value at 2^14: both parts keep their 11 bits
                    float top = 0.f;
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k) {
                        const float4* v = reinterpret_cast<const float4*>(row + (k * 32 + 8 * t) * 4);
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const float4 x = there ? v[h] : make_float4(0.f, 0.f, 0.f, 0.f);
                            top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(NONE, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(NONE, top, 2));
                    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
                    const int shift = top > 0.f && e < 128 ? max(-115, min(126, 14 - e)) : 0;
                    const float up = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23) * (p.scale < 0.f ? -1.f : 1.f);
                    const float down = fmaxf(fabsf(p.scale) * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * 1.4426950408889634f, 0x1p-120f);   // of row g
                    fa = __shfl_sync(NONE, down, 8 * t); fb = __shfl_sync(NONE, down, 8 * t + 4);
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k) {
                        const float4* v = reinterpret_cast<const float4*>(row + (k * 32 + 8 * t) * 4);
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const float4 x = there ? v[h] : make_float4(0.f, 0.f, 0.f, 0.f);
                            const float y0 = x.x * up, y1 = x.y * up, y2 = x.z * up, y3 = x.w * up;
                            const uint32_t h0 = h2_bits(__floats2half2_rn(y0, y1)), h1 = h2_bits(__floats2half2_rn(y2, y3));
                            qf[0][2 * k + h][0] = h0; qf[0][2 * k + h][1] = h1;
                            qf[F16 ? 0 : 1][2 * k + h][0] = pack_low(y0, y1, h0); qf[F16 ? 0 : 1][2 * k + h][1] = pack_low(y2, y3, h1);
                        }
                    }
                }
                if constexpr (Q8 && F16) {
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k) {
                        float sum = 0.f;
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                            for (uint32_t j = 0; j < 2; ++j) {
                                const float2 v = __half22float2(bits_h2(qf[0][2 * k + h][j]));
                                sum += v.x + v.y;
                            }
                        sum += __shfl_xor_sync(NONE, sum, 1);
                        sum += __shfl_xor_sync(NONE, sum, 2);
                        sum *= -1152.f;
                        start[k][0] = __shfl_sync(NONE, sum, 8 * t); start[k][1] = __shfl_sync(NONE, sum, 8 * t + 4);
                    }
                }
            }

            // [32 dims][m tile][c]: dims 32 b + 16 i + g, + 8; rows 2 t, + 1
            float o[NB][2][4];
#pragma unroll
            for (uint32_t k = 0; k < NB; ++k)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) o[k][i][c] = 0.f;
            // A row's weight is 2^(score + ref), ref = lift - m: m, the score that was largest when the reference last moved; lift, Q8_0: the power of two
            // that keeps weights times the value scales of the slots that the row has seen below 2^15 (it only falls), else kUp. limit_v: the value scale that the
            // higher of the two lifts allows
            float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f, lift_a = Q8 ? 20.f : kUp, lift_b = lift_a;
            float ref_a = 0.f, ref_b = 0.f, limit_a = -INFINITY, limit_b = -INFINITY, limit_v = Q8 ? 0x1p-13f : INFINITY;
            bool dead = false;

            // false: the wait has run out, and no wait is tried again
            auto arrived = [&]() {
                const bool yes = __all_sync(NONE, !lost && (mbar_try_wait(&sm.full[warp][stage], phase) || mbar_wait(&sm.full[warp][stage], phase)));
                if (!yes) {
                    if (!lost && lane == 0) raise_error(p.error, TSP_ERR_TIMEOUT);
                    lost = dead = true;
                }
                return yes;
            };
            auto pass = [&]() {   // the stage has been read: filled again
                fence_async_smem();
                __syncwarp();
                if (!lost) issue(stage);
                if (++stage == P) { stage = 0; phase ^= 1; }
            };
            // One unit; EDGE: it reaches past the context
            auto unit = [&](auto edge_tag) {
                constexpr bool EDGE = decltype(edge_tag)::value;
                const uint8_t* keys = sm.ring[warp] + stage * S::kPiece;
                float s[NS];
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) s[i] = 0.f;
#pragma unroll
                for (uint32_t b0 = 0; b0 < NB; b0 += Q8 ? 2 : 1) {
                    uint4 w[2];   // 16 bytes of slots g and g + 8
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n) w[n] = *reinterpret_cast<const uint4*>(keys + ((Q8 ? b0 / 2 : b0) * kKvGroup + 8 * n + g) * 64 + t * 16);
#pragma unroll
                    for (uint32_t k = b0; k < b0 + (Q8 ? 2 : 1); ++k) {   // 32 dims: two steps under one scale
                        uint32_t kb[2][4];
#pragma unroll
                        for (uint32_t n = 0; n < 2; ++n) {
                            if constexpr (Q8) {
                                const uint32_t x = k & 1 ? w[n].z : w[n].x, y = k & 1 ? w[n].w : w[n].y;
                                if constexpr (F16) { biased_halves(x, kb[n][0], kb[n][1]); biased_halves(y, kb[n][2], kb[n][3]); }
                                else { codes_to_halves(x, kb[n][0], kb[n][1]); codes_to_halves(y, kb[n][2], kb[n][3]); }
                            } else { kb[n][0] = w[n].x; kb[n][1] = w[n].y; kb[n][2] = w[n].z; kb[n][3] = w[n].w; }
                        }
                        float acc[4];
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                            for (uint32_t part = 0; part < (F16 ? 1 : 2); ++part) {
                                const uint32_t (&q)[2] = qf[part][2 * k + h];
                                if (h || part) mma_f16_16816(acc, kb[0][2 * h], kb[1][2 * h], kb[0][2 * h + 1], kb[1][2 * h + 1], q[0], q[1]);
                                else if constexpr (Q8 && F16) mma_f16_16816_from(acc, kb[0][0], kb[1][0], kb[0][1], kb[1][1], q[0], q[1], start[k][0], start[k][1], start[k][0], start[k][1]);
                                else mma_f16_16816_zero(acc, kb[0][0], kb[1][0], kb[0][1], kb[1][1], q[0], q[1]);
                            }
                        if constexpr (Q8) {
                            const uint8_t* scales = keys + kKvGroup * D + k * kKvGroup * 2;
                            const float d0 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2)), d1 = __half2float(*reinterpret_cast<const __half*>(scales + g * 2 + 16));
                            s[0] = fmaf(acc[0], d0, s[0]); s[1] = fmaf(acc[1], d0, s[1]);
                            s[2] = fmaf(acc[2], d1, s[2]); s[3] = fmaf(acc[3], d1, s[3]);
                        } else {
#pragma unroll
                            for (uint32_t i = 0; i < NS; ++i) s[i] += acc[i];
                        }
                    }
                }
                if constexpr (PIECES == 2) { pass(); (void)arrived(); }
                const uint8_t* values = PIECES == 2 ? sm.ring[warp] + stage * S::kPiece : keys + S::kHalf;
                // At the end of the context: what a row does not see gets no weight. Drafted slots whose values are not finite give the rows that see
                // them NaN through the weight, and count as zero themselves; slots behind the last count as zero, whatever they hold.
                uint32_t keep[2] = {NONE, NONE};   // values of slots 2t, 2t + 1 and 8 more
                uint32_t drop = 0;                 // bit i: slot i of the unit
                if constexpr (EDGE) {
                    const uint64_t slot0 = (a + done - it.start) * kKvGroup;
                    uint32_t odd = 0;
                    const uint32_t there = it.total - slot0 >= kKvGroup ? 0xffffu : (1u << static_cast<uint32_t>(it.total - slot0)) - 1;
                    const uint32_t drafted = slot0 >= it.length ? 0xffffu : 0xffffu << static_cast<uint32_t>(it.length - slot0);
                    if constexpr (Q8) {
                        for (uint32_t i = lane; i < NB * kKvGroup; i += 32)
                            odd |= static_cast<uint32_t>(odd_half(*reinterpret_cast<const uint16_t*>(values + kKvGroup * D + i * 2))) << i % kKvGroup;
                    } else {
                        for (uint32_t i = 0; i < D / 8; ++i)   // 16 dims, half of them: eight bytes of four slots a lane
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e)
                                odd |= static_cast<uint32_t>(odd_half(*reinterpret_cast<const uint16_t*>(values + (i / 2 * 32 + lane) * 16 + i % 2 * 8 + e * 2))) << (2 * t + (e & 1) + 8 * (e >> 1));
                    }
                    odd = __reduce_or_sync(NONE, odd) & drafted & there;
                    drop = odd | (~there & 0xffffu);
                    uint64_t wa, wb;
                    {
                        uint32_t node, head;
                        row_of(ra, node, head);
                        wa = ra >= it.rows ? 0 : p.mask ? p.mask[it.row0 + node] : ~0ull >> (63 - min(node, 63u));
                        row_of(rb, node, head);
                        wb = rb >= it.rows ? 0 : p.mask ? p.mask[it.row0 + node] : ~0ull >> (63 - min(node, 63u));
                    }
#pragma unroll
                    for (uint32_t i = 0; i < NS; ++i) {
                        const uint32_t x = slot_in(i);
                        const bool seen = there >> x & 1 && (!(drafted >> x & 1) || ((second(i) ? wb : wa) >> (slot0 + x - it.length) & 1));
                        if (!seen) s[i] = -INFINITY;
                        else if (odd >> x & 1) s[i] = NAN;
                    }
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n)
                        keep[n] = (drop >> (8 * n + 2 * t) & 1 ? 0u : 0x0000ffffu) | (drop >> (8 * n + 2 * t) & 2 ? 0u : 0xffff0000u);
                }
                [[maybe_unused]] float dv[Q8 ? NB : 1][2];   // value scales of slots g, g + 8
                // largest value scale that a row sees: not that of a slot hidden from it, which would push the weights of the others under binary16's
                // smallest numbers. Inside the context both rows see every slot.
                float widest_a = 0.f, widest_b = 0.f;
                if constexpr (Q8) {
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k) {
                        const uint8_t* scales = values + kKvGroup * D + k * kKvGroup * 2;
                        dv[k][0] = __half2float(*reinterpret_cast<const __half*>(scales + g * 2));
                        dv[k][1] = __half2float(*reinterpret_cast<const __half*>(scales + g * 2 + 16));
                        if constexpr (EDGE) { if (drop >> g & 1) dv[k][0] = 0.f; if (drop >> (g + 8) & 1) dv[k][1] = 0.f; }
                        if constexpr (EDGE) {
#pragma unroll
                            for (uint32_t n = 0; n < 2; ++n) {
                                if (s[2 * n] != -INFINITY) widest_a = fmaxf(widest_a, fabsf(dv[k][n]));
                                if (s[2 * n + 1] != -INFINITY) widest_b = fmaxf(widest_b, fabsf(dv[k][n]));
                            }
                        } else widest_a = fmaxf(widest_a, fmaxf(fabsf(dv[k][0]), fabsf(dv[k][1])));
                    }
                    if constexpr (!EDGE) widest_b = widest_a;
                }
                float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) { if (second(i)) xb = fmaxf(xb, s[i]); else xa = fmaxf(xa, s[i]); }
                xa *= fa; xb *= fb;
                if (__any_sync(NONE, xa > limit_a || xb > limit_b || fmaxf(widest_a, widest_b) > limit_v)) {
#pragma unroll
                    for (uint32_t x = 4; x < 32; x *= 2) { xa = fmaxf(xa, __shfl_xor_sync(NONE, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(NONE, xb, x)); }
                    xa = fmaxf(xa, ma); xb = fmaxf(xb, mb);
                    float fall_a = 0.f, fall_b = 0.f;
                    if constexpr (Q8) {   // widest < 2^(e + 1): weights up to 2^kSlack times it times 2^lift stay below 2^15
                        uint32_t wa, wb;
                        if constexpr (EDGE) {
#pragma unroll
                            for (uint32_t x = 4; x < 32; x *= 2) {
                                widest_a = fmaxf(widest_a, __shfl_xor_sync(NONE, widest_a, x)); widest_b = fmaxf(widest_b, __shfl_xor_sync(NONE, widest_b, x));
                            }
                            wa = __float_as_uint(widest_a); wb = __float_as_uint(widest_b);
                        } else wa = wb = __reduce_max_sync(NONE, __float_as_uint(widest_a));
                        auto lowered = [](float lift, uint32_t bits) { return fminf(lift, 6.f - static_cast<float>(static_cast<int>(min(bits >> 23, 143u)) - 127)); };
                        const float now_a = lowered(lift_a, wa), now_b = lowered(lift_b, wb);
                        fall_a = now_a - lift_a; fall_b = now_b - lift_b;
                        lift_a = now_a; lift_b = now_b;
                        limit_v = exp2f(7.f - fmaxf(lift_a, lift_b));
                    }
                    const float r0 = ma == -INFINITY ? 0.f : exp2_approx(ma - xa + fall_a), r1 = mb == -INFINITY ? 0.f : exp2_approx(mb - xb + fall_b);
                    la *= ma == -INFINITY ? 1.f : r0; lb *= mb == -INFINITY ? 1.f : r1;   // a NaN stays
                    ma = xa; mb = xb;
                    limit_a = ma + kSlack; limit_b = mb + kSlack;
                    ref_a = ma == -INFINITY ? 0.f : lift_a - ma; ref_b = mb == -INFINITY ? 0.f : lift_b - mb;
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k)
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) o[k][i][c] *= second(c) ? r1 : r0;
                }
                float pr[NS];
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) {
                    pr[i] = exp2_approx(fmaf(s[i], second(i) ? fb : fa, second(i) ? ref_b : ref_a));
                    if (second(i)) lb += pr[i]; else la += pr[i];
                }
                uint32_t wf[2];
                [[maybe_unused]] uint32_t wl[2];
                auto split = [&](const float (&w)[NS]) {   // B fragment: slots 2t.., 8 more, of row g
#pragma unroll
                    for (uint32_t r = 0; r < 2; ++r) {
                        const uint32_t high = h2_bits(__floats2half2_rn(w[2 * r], w[2 * r + 1]));
                        if constexpr (!F16) wl[r] = transposed(pack_low(w[2 * r], w[2 * r + 1], high));
                        wf[r] = transposed(high);
                    }
                };
                if constexpr (!Q8) split(pr);
#pragma unroll
                for (uint32_t k = 0; k < NB; ++k) {
                    uint32_t vb[8];   // dims 8 i + g: slots 2t, 2t + 1 in vb[2 i], 8 further in vb[2 i + 1]
                    if constexpr (Q8) {
                        const uint4 w = *reinterpret_cast<const uint4*>(values + k * 512 + lane * 16);
                        codes_to_halves(w.x, vb[0], vb[1]); codes_to_halves(w.y, vb[2], vb[3]);
                        codes_to_halves(w.z, vb[4], vb[5]); codes_to_halves(w.w, vb[6], vb[7]);
                        float w4[NS];
#pragma unroll
                        for (uint32_t i = 0; i < NS; ++i) w4[i] = pr[i] * dv[k][i / 2];
                        split(w4);
                    } else {
                        const uint4 w = *reinterpret_cast<const uint4*>(values + k * 1024 + lane * 16), x = *reinterpret_cast<const uint4*>(values + k * 1024 + 512 + lane * 16);
                        vb[0] = w.x; vb[1] = w.y; vb[2] = w.z; vb[3] = w.w; vb[4] = x.x; vb[5] = x.y; vb[6] = x.z; vb[7] = x.w;
                        if constexpr (EDGE) {
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) vb[i] &= keep[i & 1];
                        }
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const uint32_t a0 = vb[4 * i], a1 = vb[4 * i + 2], a2 = vb[4 * i + 1], a3 = vb[4 * i + 3];
                        if constexpr (F16) mma_f16_16816(o[k][i], a0, a1, a2, a3, wf[0], wf[1]);
                        else {   // the tensor core cuts its sums off: a chain of two products, added up rounded
                            float acc[4];
                            mma_f16_16816_zero(acc, a0, a1, a2, a3, wf[0], wf[1]);
                            mma_f16_16816(acc, a0, a1, a2, a3, wl[0], wl[1]);
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) o[k][i][c] += acc[c];
                        }
                    }
                }
            };
            const uint64_t plain = it.start + it.length / kKvGroup;   // units before this one lie in the context
            const uint32_t inner = plain <= a ? 0u : static_cast<uint32_t>(min(plain - a, static_cast<uint64_t>(stop)));
            auto step = [&](auto edge_tag) {
                if (arrived() && !(gone >> stage & 1)) unit(edge_tag);
                else {
                    dead = true;
                    if constexpr (PIECES == 2) { pass(); (void)arrived(); }
                }
                pass();
            };
            for (; done < inner; ++done) step(std::false_type{});
            for (; done < stop; ++done) step(std::true_type{});

            // ---- end of the item or of the run
#pragma unroll
            for (uint32_t x = 4; x < 32; x *= 2) { la += __shfl_xor_sync(NONE, la, x); lb += __shfl_xor_sync(NONE, lb, x); }
            auto dim_of = [&](uint32_t k, uint32_t i, uint32_t c) { return k * 32 + i * 16 + g + 8 * (c / 2); };
            if (it.start >= a && it.end <= b) {   // the whole item: its rows go out
                const float ia = la == 0.f ? 0.f : 1.f / la, ib = lb == 0.f ? 0.f : 1.f / lb;
                uint32_t bad = 0;   // bit 0, 1: row ra, rb
#pragma unroll
                for (uint32_t k = 0; k < NB; ++k)
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) {
                            o[k][i][c] *= second(c) ? ib : ia;
                            if (!(F16 ? fabsf(o[k][i][c]) < 65520.f : finite_f32(o[k][i][c]))) bad |= second(c) ? 2u : 1u;
                        }
#pragma unroll
                for (uint32_t x = 4; x < 32; x *= 2) bad |= __shfl_xor_sync(NONE, bad, x);
#pragma unroll
                for (uint32_t side = 0; side < 2; ++side) {
                    const uint32_t r = side ? rb : ra;
                    if (r >= it.rows) continue;
                    const bool zero = dead || bad >> side & 1;
                    if (zero && !dead) raise_error(p.error, TSP_ERR_NONFINITE);
                    const uint32_t flat = it.tile * kTile + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
                    uint8_t* dst = p.out + static_cast<uint64_t>(it.row0 + node) * p.out_stride + head * D * (F16 ? 2u : 4u);
#pragma unroll
                    for (uint32_t k = 0; k < NB; ++k)
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c)
                                if (second(c) == (side != 0)) {
                                    const float v = zero ? 0.f : o[k][i][c];
                                    if constexpr (F16) reinterpret_cast<__half*>(dst)[dim_of(k, i, c)] = __float2half_rn(v);
                                    else reinterpret_cast<float*>(dst)[dim_of(k, i, c)] = v;
                                }
                }
            } else {
                const uint32_t which = stop == mine ? 1 : 0;   // 1: the run's last item, into the ring, where no copy is under way any more
                float* part = which ? reinterpret_cast<float*>(sm.ring[warp]) : warp_part;
                if (g == 0) {
                    part[ra] = ma == -INFINITY ? ma : -ref_a; part[rb] = mb == -INFINITY ? mb : -ref_b;
                    part[kTile + ra] = la; part[kTile + rb] = lb;
                }
                if (lane == 0) { sm.key[warp][which] = it.start; sm.item[warp][which] = it; part[2 * kTile] = dead ? 1.f : 0.f; }
#pragma unroll
                for (uint32_t k = 0; k < NB; ++k)
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) {
                            const uint32_t r = second(c) ? rb : ra;
                            if (r < it.rows) part[kPartHead + r * D + dim_of(k, i, c)] = o[k][i][c];
                        }
            }
        }
    }
    __syncthreads();

    // ---- pieces of an item meet: first those of the block's warps, one item after another, then, where this block is the last of an item's to arrive,
    // those of its blocks. All of it is one loop: what runs once per launch waits for its instructions more than for anything else (unrolled
    // code of their own took the two joins 10 us of a call of 22).
    constexpr uint32_t LANES = D / 4 < 32 ? D / 4 : 32, V = D / 4 / LANES;   // lanes of a row, float4s a lane
    const bool has_row = lane < LANES;
    auto block_part = [&](uint64_t block, bool at_start) { return p.parts + (2 * block + (at_start ? 0 : 1)) * part_floats(); };
    // Piece j (lane j) is warp j / 2's first or last item; consecutive pieces of one item are a group
    const uint64_t key = lane < 2 * W ? sm.key[lane / 2][lane % 2] : ~0ull;
    const uint32_t there = __ballot_sync(NONE, key != ~0ull), below = there & ((1u << lane) - 1);
    const uint64_t before = __shfl_sync(NONE, key, below ? 31 - __clz(below) : 0);
    uint32_t heads = __ballot_sync(NONE, key != ~0ull && (!below || before != key));
    const AttnItem &first = sm.edge[0], &last = sm.edge[1];
    const bool open0 = first.start < u0 || first.end > u1, open1 = last.start != first.start && last.end > u1;
    float4* const meet = reinterpret_cast<float4*>(sm.meet);
    uint32_t task = warp;   // inside the block every warp takes every W-th row of all items' together
#pragma unroll 1
    for (uint32_t side = 0; side < 2;) {
        // n pieces: at p0, then p1 + stride (i - 1), the last of them at pl
        const AttnItem* item;
        const float *p0, *p1, *pl;
        uint32_t n, stride;
        const bool inside = heads != 0;
        if (inside) {
            const uint32_t head = __ffs(heads) - 1, next = heads & (heads - 1);
            const uint32_t members = there & ~((1u << head) - 1) & (next ? (1u << (__ffs(next) - 1)) - 1 : NONE), tail = 31 - __clz(members);
            auto piece = [&](uint32_t j) { return j % 2 ? reinterpret_cast<const float*>(sm.ring[j / 2]) : p.parts + (2ull * kAttnMaxBlocks + blockIdx.x * kMaxWarps + j / 2) * part_floats(); };
            item = &sm.item[head / 2][head % 2];
            n = __popc(members);
            p0 = piece(head); pl = piece(tail);
            p1 = reinterpret_cast<const float*>(sm.ring[head / 2 + (n > 1)]);
            stride = S::kRing / 4;
            heads = next;
        } else {
            if (side == 0) {   // the block's own pieces are written: count it in
                if (!open0 && !open1) return;
                __syncthreads();
                if (tid < 2) {
                    __threadfence();   // they go before the count
                    const AttnItem& it = tid ? last : first;
                    uint32_t joins = 0;
                    if (tid ? open1 : open0) {
                        const uint32_t c0 = runs.first(it.start), count = runs.count(it.start, it.end);
                        joins = atomicAdd(p.counters + c0, 1u) == count - 1;
                        if (joins) p.counters[c0] = 0;
                        sm.span[tid][0] = c0; sm.span[tid][1] = count;
                    }
                    sm.last[tid] = joins;
                    __threadfence();
                }
                __syncthreads();
            }
            const uint32_t mine = side++;
            if (!sm.last[mine]) continue;
            item = mine ? &last : &first;
            const uint32_t c0 = sm.span[mine][0];
            n = sm.span[mine][1];
            p0 = block_part(c0, runs.at_run_start(item->start));
            p1 = block_part(c0 + 1, true);
            stride = 2 * static_cast<uint32_t>(part_floats());
            pl = n > 1 ? p1 + static_cast<uint64_t>(n - 2) * stride : p0;
        }
        auto part_of = [&](uint32_t i) { return i == 0 ? p0 : i == n - 1 ? pl : p1 + static_cast<uint64_t>(i - 1) * stride; };
        // a row by `ways` warps, each every ways-th piece of every 32; the references of all of them go by all the warps, so that theirs is the same
        const uint32_t rows = item->rows, wide = min(W, rows), ways = inside ? 1 : W / wide, way = inside ? 0 : warp / wide;
        uint32_t r = inside ? task : warp % wide;
#pragma unroll 1
        for (; inside ? r < rows : r < (rows + wide - 1) / wide * wide; r += inside ? W : wide) {
            const bool on = way < ways && r < rows;
            float4 y[V];
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, sum = 0.f;
            bool dead = false;
            if (on) {
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < n; i0 += 32) {
                    const uint32_t i = i0 + lane, count = min(32u, n - i0);
                    const float* head = part_of(min(i, n - 1));
                    float m = load_piece(head + r), l = load_piece(head + kTile + r);
                    dead |= load_piece(head + 2 * kTile) != 0.f;
                    if (i >= n) { m = -INFINITY; l = 0.f; }
                    float now = m;
#pragma unroll
                    for (uint32_t x = 16; x; x /= 2) now = fmaxf(now, __shfl_xor_sync(NONE, now, x));
                    now = fmaxf(now, top);
                    const float f = weight_of(m, now), old = weight_of(top, now);
                    sum = (top == -INFINITY ? sum : sum * old) + (m == -INFINITY ? l : l * f);   // a row of NaN alone has a sum of NaN and no reference
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k) { y[k].x *= old; y[k].y *= old; y[k].z *= old; y[k].w *= old; }
                    top = now;
#pragma unroll 1
                    for (uint32_t j0 = way; j0 < count; j0 += 4 * ways) {
                        float4 v[4][V];
                        float fj[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            const uint32_t at = min(j0 + j * ways, count - 1);
                            fj[j] = __shfl_sync(NONE, f, at);
                            if (j0 + j * ways >= count) fj[j] = 0.f;
#pragma unroll
                            for (uint32_t x = 0; x < V; ++x) v[j][x] = load_piece4(part_of(i0 + at) + kPartHead + r * D + (x * LANES + lane % LANES) * 4);
                        }
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j)
                            if (fj[j] != 0.f)
#pragma unroll
                                for (uint32_t x = 0; x < V; ++x) {
                                    y[x].x = fmaf(v[j][x].x, fj[j], y[x].x); y[x].y = fmaf(v[j][x].y, fj[j], y[x].y);
                                    y[x].z = fmaf(v[j][x].z, fj[j], y[x].z); y[x].w = fmaf(v[j][x].w, fj[j], y[x].w);
                                }
                    }
                }
#pragma unroll
                for (uint32_t x = 16; x; x /= 2) sum += __shfl_xor_sync(NONE, sum, x);
                dead = __any_sync(NONE, dead);
                if (way && has_row)
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k) meet[(warp * V + k) * LANES + lane] = y[k];
            }
            if (ways > 1) __syncthreads();
            if (on && !way) {
#pragma unroll 1
                for (uint32_t x = 1; x < ways; ++x)
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k) {
                        const float4 v = meet[((warp + x * wide) * V + k) * LANES + lane % LANES];
                        y[k].x += v.x; y[k].y += v.y; y[k].z += v.z; y[k].w += v.w;
                    }
                if (inside && (item->start < u0 || item->end > u1)) {   // still a piece
                    float* part = block_part(blockIdx.x, item->start <= u0);
                    if (has_row)
#pragma unroll
                        for (uint32_t k = 0; k < V; ++k) __stcg(reinterpret_cast<float4*>(part + kPartHead + r * D) + k * LANES + lane, y[k]);
                    if (lane == 0) { __stcg(part + r, top); __stcg(part + kTile + r, sum); __stcg(part + 2 * kTile, dead ? 1.f : 0.f); }
                } else {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    bool ok = sum == sum;
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k) {
                        y[k].x *= inv; y[k].y *= inv; y[k].z *= inv; y[k].w *= inv;
                        ok &= in_range<F16>(y[k].x) && in_range<F16>(y[k].y) && in_range<F16>(y[k].z) && in_range<F16>(y[k].w);
                    }
                    ok = __all_sync(NONE, ok);
                    if (!ok && !dead && lane == 0) raise_error(p.error, TSP_ERR_NONFINITE);
                    const uint32_t flat = item->tile * kTile + r, node = flat / p.group, head = item->head * p.group + flat % p.group;
                    uint8_t* dst = p.out + static_cast<uint64_t>(item->row0 + node) * p.out_stride + head * D * (F16 ? 2u : 4u);
                    if (has_row)
#pragma unroll
                        for (uint32_t k = 0; k < V; ++k) {
                            if (!ok || dead) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            const uint32_t x = k * LANES + lane;
                            if constexpr (F16) reinterpret_cast<uint2*>(dst)[x] = make_uint2(h2_bits(__floats2half2_rn(y[k].x, y[k].y)), h2_bits(__floats2half2_rn(y[k].z, y[k].w)));
                            else reinterpret_cast<float4*>(dst)[x] = y[k];
                        }
                }
            }
            if (ways > 1) __syncthreads();
        }
        if (inside) task = r - rows;
    }
}

uint64_t tree_mma_parts_bytes();
uint64_t tree_attention_scratch_bytes() {
    const uint64_t here = (2ull + kMaxWarps) * kAttnMaxBlocks * part_floats() * sizeof(float), there = tree_mma_parts_bytes();
    return kAttnMaxBlocks * sizeof(uint32_t) + (here > there ? here : there);
}

template <uint32_t D, bool Q8, bool F16>
static int launch_tree_attention_t(const AttnParams& p, cudaStream_t st) {
    using S = AttnShape<D, Q8>;
    using Smem = AttnSmem<D, Q8>;
    static_assert(sizeof(Smem) <= 232448, "shared memory of a block");
    auto kernel = tree_attention_kernel<D, Q8, F16>;
    static thread_local SmemAttrCache attr;
    TSP_CUDA(ensure_dynamic_smem(kernel, attr, sizeof(Smem)));
    const int sms = sm_count();
    const uint32_t blocks = sms < 1 ? 1 : sms < static_cast<int>(kAttnMaxBlocks) ? sms : kAttnMaxBlocks;
    TSP_CUDA(launch_pdl(kernel, dim3(blocks), dim3(S::kThreads), sizeof(Smem), st, p));
    return TSP_OK;
}

int launch_tree_mma(const AttnParams&, cudaStream_t);
int tree_mma_registers(const AttnParams&, int&);

template <uint32_t D, bool Q8>
static int launch_tree_attention_d(const AttnParams& p, bool f16, cudaStream_t st) {
    const uint64_t rows = static_cast<uint64_t>(p.max_rows) * p.group;
    if (wide_tiles(D, f16, rows, kTmLaunchRegs)) {   // if the registers of that kernel are right, that is
        int registers;
        if (int rc = tree_mma_registers(p, registers)) return rc;
        if (wide_tiles(D, f16, rows, registers)) return launch_tree_mma(p, st);
    }
    return f16 ? launch_tree_attention_t<D, Q8, true>(p, st) : launch_tree_attention_t<D, Q8, false>(p, st);
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
