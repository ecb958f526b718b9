// Attention of drafted tokens, many binary16 rows per key / value head (tsp_tree_attention): the tiles on the 5th-generation tensor cores.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(f q.k_j + ref), as in tsp_tree_attn.cu, with 128 query rows of a kv head (drafted tokens x heads of the group) as
// the M of tcgen05 MMAs: S = Q K^T (N = 64 slots, K = dims) and O += P V (N = dims, K = 64 slots), both with the left operand in tensor memory and the cache's
// tile in shared memory. Units are 64 slots; they are dealt to the blocks as there, and pieces of items that span blocks are joined the same way.
//
// Roles of a block's 16 warps (one block per SM): 0 copies groups of 16 slots into a ring; 3 looks at what came; 1 issues the MMAs; 4..7 are the softmax, a thread per query row:
// a score row from tensor memory to registers, weights back to tensor memory as binary16, reference, sum and the rare rescaling of the accumulator, and at an
// item's end the accumulator's row; 8..11 turn codes into the MMAs' tiles of K, 12..15 into those of V. Scores, weights, query rows and tiles are double-buffered, so
// the QK of one unit runs under the softmax of the one before and the PV of the one before that.
//
// Measured: a tree of 64 tokens x 32 heads over 131072 slots of 8 kv heads, Q8_0, 128 dims: 281 us back to back, 315 to 320 among other calls (867 with tiles of
// eight rows on the warps' MMAs; 293 with K and V tiles by the same warps), the bytes alone 44 us, the products alone 84; four trees of 32 tokens over up to 20000
// slots: 69 and 73 us (115). A unit takes about
// 2050 cycles at 1.75 GHz, 1024 of them MMAs; without the tiles' arithmetic it takes 1850, without half of the MMAs 1880, without these, the softmax's and the
// copies 1450: no stage alone but the hand-overs between them (barrier, fence, commit) bound it.
//
// Rounding: a Q8_0 value is code times scale, 18 bits. Tiles hold it as two binary16 numbers, high and low (exact, times a power of two that puts the unit's
// largest scale at 2^7), and the MMAs run over both: what is left between the cache and a binary16 row is the weights' rounding, as on the warp MMAs. (High
// parts alone: errors against 64 bits 4.1e-4 instead of 2.9e-4, half the MMAs.) A binary16 cache needs no low parts.
// That power of two goes by all slots of the unit, also by drafted ones that some rows do not see. Up to 2^kTmSpread between their scales this costs such a
// row nothing: values are exact up to 2^20, and weights reach down to 2^-24 of the row's largest. Beyond ("wild", at the end of the context only), warp 3
// raises every slot's scales to the largest one's octave; its scores go back down by as much, its weights as far as the row's accumulator asks, both in
// tensor memory and in rolled loops that no other unit enters (on the registers of the ordinary path they took 18 % of every call).
#include <type_traits>

#include "tsp_tree_attn.cuh"

namespace tsp {

constexpr uint32_t kTmLeastUnits = 4;   // of a block's run: 13 tokens over 1000 slots 18.8 us, 22.5 with eight
// Octaves between the largest scales of two slots of a unit above which, at the end of the context, every slot gets a power of two of its own
constexpr uint32_t kTmSpread = 8;
constexpr uint32_t kTmRows = 128, kTmUnit = 64, kTmGroups = kTmUnit / kKvGroup;
constexpr uint32_t kTmSoftmax = 4, kTmTiles = 8, kTmTileWarps = 8, kTmThreads = 32 * (kTmTiles + kTmTileWarps);   // first softmax warp, first tile warp
// Registers after the hand-over between the warpgroups (setmaxnreg): together no more than the count at launch times the four warpgroups, or the softmax
// would wait for ever; a kernel of another count is not launched (tsp_tree_rule.h). At the end all go back to that count.
constexpr int kTmIssueRegs = 104, kTmSoftmaxRegs = 192, kTmTileRegs = 104;
static_assert(kTmIssueRegs + kTmSoftmaxRegs + kTmTileWarps / 4 * kTmTileRegs <= (2 + kTmTileWarps / 4) * kTmLaunchRegs, "hand-over of registers");
// piece of an item: references and sums of 128 rows, a flag, then the rows' dims four by four, rows side by side: [dim / 4][row][4]
constexpr uint32_t kTmPartHead = 288;
__host__ __device__ constexpr uint64_t tm_part_floats() { return kTmPartHead + kTmRows * 128; }

template <uint32_t D, bool Q8>
struct TmShape {
    static constexpr uint32_t kGroupBytes = kv_group_bytes(D, Q8), kHalf = kv_half_bytes(D, Q8), kStage = kTmGroups * kGroupBytes;
    static constexpr uint32_t kStages = 3, kParts = Q8 ? 2 : 1;   // parts: high, low. Four stages: no faster over long contexts, 2 % slower over short ones
    static constexpr uint32_t kKPart = kTmUnit * D * 2, kVPart = kTmUnit * D * 2;      // bytes of a part of a K tile ([64 dims][64 slots][64]) and a V tile ([dims][64 slots])
    // tensor memory: query rows (two buffers), scores (two), weights (two), accumulator
    static constexpr uint32_t kQ = 0, kS = kQ + 2 * (D / 2), kP = kS + 2 * kTmUnit, kO = kP + 2 * (kTmUnit / 2), kCols = 512;
    static_assert(kO + D <= kCols, "tensor memory");
};
template <uint32_t D, bool Q8>
struct TmSmem {
    using S = TmShape<D, Q8>;
    alignas(1024) uint8_t k[2][S::kParts][S::kKPart];
    alignas(1024) uint8_t v[2][S::kParts][S::kVPart];
    alignas(128) uint8_t ring[S::kStages][S::kStage];
    uint64_t cum[TSP_KV_MAX_SEQUENCES + 1];
    uint64_t warp_sums[kTmThreads / 32];
    uint64_t code_full[S::kStages], code_known[S::kStages], code_empty[S::kStages];
    uint64_t k_ready[2], v_ready[2], s_full[2], s_free[2], p_ready[2], pv_done[2], q_ready[2];
    AttnItem edge[2];
    // per unit (mod 8: the copies are four units ahead of the softmax at most): no page; the tiles' powers of two; drafted slots whose
    // values are not finite; slots that count as zero
    uint32_t gone[8], k_lift[8], v_lift[8], odd[8][2], drop[8][2];
    uint32_t wild[8];                                     // units at the end of the context; bit 0: of keys, 1: of values
    uint8_t k_raised[8][kTmUnit], v_raised[8][kTmUnit];   // octaves, by slot
    uint32_t tmem, last[2], span[2][2], bad_rows[kTmRows / 32];
    float tops[4][kTmRows];   // of the join
};

__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_ld32(uint32_t at, float (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
                   "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]),
                   "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
                 : "r"(at));
}
__device__ __forceinline__ uint32_t tm_ld1(uint32_t at) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void tm_st1(uint32_t at, uint32_t v) { asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void tm_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 64 of K: four D (+)= A[tensor memory] * B[shared memory], binary16, FP32 sums; B: rows of 128 bytes under the 128-byte swizzle, eight rows every 1024 bytes
template <uint32_t N>
__device__ __forceinline__ void tm_mma64(uint32_t d, uint32_t a, uint32_t b_smem, uint32_t accumulate) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29), idesc = (1u << 4) | ((N >> 3) << 17) | ((kTmRows >> 4) << 24);
    const uint32_t b_lo = ((b_smem & 0x3FFFFu) >> 4) | (1u << 16);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
        asm volatile("{\n\t.reg .pred q;\n\t.reg .b64 b;\n\tsetp.ne.b32 q, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, q;\n\t}"
                     ::"r"(d), "r"(a + k * 8), "r"(b_lo + k * 2), "r"(idesc), "r"(accumulate | k), "n"(hi) : "memory");
}
__device__ __forceinline__ void tm_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded wait by a whole warp. Every try may sleep for up to a millisecond: warps that asked again at once took issue slots and shared memory's time from the
// others (the case above 323 us). Two seconds in all, then the caller gives up.
__device__ __forceinline__ bool tm_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t at = smem_u32(bar);
    uint32_t done = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < 2000 && !done; ++i)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(at), "r"(parity), "r"(1000000u) : "memory");
    return __all_sync(0xffffffffu, done != 0);
}
// Three at once: where all are complete, for the time of one. The third may be NULL.
__device__ __forceinline__ bool tm_wait3(uint64_t* a, uint32_t a_parity, uint64_t* b, uint32_t b_parity, uint64_t* c, uint32_t c_parity) {
    uint32_t x, y, z = 1;
    auto test = [](uint64_t* bar, uint32_t parity, uint32_t& done) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    };
    test(a, a_parity, x); test(b, b_parity, y);
    if (c) test(c, c_parity, z);
    return __all_sync(0xffffffffu, x & y & z) || (tm_wait(a, a_parity) && tm_wait(b, b_parity) && (!c || tm_wait(c, c_parity)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {   // two FP32 operations in one
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <uint32_t D, bool Q8>
__global__ void __launch_bounds__(kTmThreads, 1)
tree_mma_kernel(const AttnParams p) {
    using S = TmShape<D, Q8>;
    constexpr uint32_t NONE = 0xffffffffu, NB = D / 32, K_LINES = kKvGroup * D * (Q8 ? 1 : 2) / 512;   // rows of 512 bytes that a group's keys (and values) are
    extern __shared__ uint8_t raw[];
    TmSmem<D, Q8>& sm = *reinterpret_cast<TmSmem<D, Q8>*>(raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u));
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = __shfl_sync(NONE, tid / 32, 0);
    pdl_launch_dependents();
    if (tid == 0) {
        for (uint32_t i = 0; i < S::kStages; ++i) { mbar_init(&sm.code_full[i], 1); mbar_init(&sm.code_known[i], 1); mbar_init(&sm.code_empty[i], kTmTileWarps); }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&sm.k_ready[i], kTmTileWarps / 2); mbar_init(&sm.v_ready[i], kTmTileWarps / 2); mbar_init(&sm.s_full[i], 2); mbar_init(&sm.s_free[i], 4);
            mbar_init(&sm.p_ready[i], 4); mbar_init(&sm.pv_done[i], 1); mbar_init(&sm.q_ready[i], 4);
        }
        mbar_fence_init();
    }
    pdl_wait();
    unit_prefix<kTmRows, kTmUnit, kTmThreads>(p, sm.cum, sm.warp_sums);
    const uint64_t units = sm.cum[p.batch.sequences];
    if (!units) return;
    const AttnRuns runs(p, units, item_of<kTmRows, kTmUnit>(p, sm.cum, 0), kTmLeastUnits);
    uint64_t u0, u1;
    runs.run(blockIdx.x, units, u0, u1);
    if (u0 >= u1) return;
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(S::kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    const uint32_t tmem = __shfl_sync(NONE, sm.tmem, 0), n = static_cast<uint32_t>(u1 - u0);
    auto part_at = [&](uint64_t block, bool at_start) { return p.parts + (2 * block + (at_start ? 0 : 1)) * tm_part_floats(); };
    bool ok = true;
    // A role's warpgroup asks for its registers in its own branch, and goes back to the count at launch at its end: not before the softmax has been given
    // what it asks for (a short role that took its own back first would leave it waiting), so all meet once that is done
    if (warp < kTmSoftmax) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTmIssueRegs));
        __syncthreads();
        if (warp == 0) {
            // ---- copies: the lanes look up the groups of eight units, then the units go out one after another
            for (uint32_t base = 0; base < n && ok; base += 8) {
                const uint32_t j = base + lane / 4, part = lane % 4;
                const uint8_t* src = nullptr;
                bool wanted = false, bad = false;
                if (j < n) {
                    const AttnItem it = item_of<kTmRows, kTmUnit>(p, sm.cum, u0 + j);
                    const uint64_t slot = (u0 + j - it.start) * kTmUnit + part * kKvGroup;
                    if (it.dead) bad = true;
                    else if (slot < it.total) {
                        wanted = true;
                        src = kv_group(p.cache, it.seq, slot, it.head, p.error);
                        bad = !src;
                    }
                }
                const uint32_t bads = __ballot_sync(NONE, bad), wants = __ballot_sync(NONE, wanted);
                const uint64_t first = __shfl_sync(NONE, reinterpret_cast<uint64_t>(src), lane & ~3u);
                const uint32_t rows = __ballot_sync(NONE, reinterpret_cast<uint64_t>(src) == first + part * S::kGroupBytes);
                for (uint32_t k = 0; k < 8 && base + k < n; ++k) {
                    const uint32_t u = base + k, st = u % S::kStages, round = u / S::kStages;
                    ok = !round || tm_wait(&sm.code_empty[st], (round - 1) & 1);
                    if (!ok) break;
                    const uint32_t gone = bads >> (4 * k) & 15u, want = gone ? 0u : wants >> (4 * k) & 15u;
                    if (elect_one()) {
                        sm.gone[u % 8] = gone;
                        mbar_arrive_expect_tx(&sm.code_full[st], __popc(want) * S::kGroupBytes);
                    }
                    __syncwarp();
                    const bool whole = want == 15u && (rows >> (4 * k) & 15u) == 15u;
                    if (lane / 4 == k && (whole ? part == 0 : (want >> part & 1) != 0))
                        bulk_g2s(sm.ring[st] + part * S::kGroupBytes, src, whole ? S::kStage : S::kGroupBytes, &sm.code_full[st]);
                    __syncwarp();
                }
            }
        } else if (warp == 1) {
            // ---- MMAs: QK of a unit, then PV of the unit before
            uint64_t end = u0;
            uint32_t item = 0;
            bool fresh_next = true;
            for (uint32_t j = 0; j <= n; ++j) {
                const bool fresh = fresh_next;   // of unit j - 1: its PV starts an accumulator
                if (j < n) {
                    if (u0 + j >= end) {
                        end = item_of<kTmRows, kTmUnit>(p, sm.cum, u0 + j).end;
                        ok = tm_wait(&sm.q_ready[item & 1], (item >> 1) & 1);
                        if (!ok) break;
                        ++item;
                        fresh_next = true;
                    } else fresh_next = false;
                    const uint32_t buf = j & 1, turn = (j >> 1) & 1;
                    ok = tm_wait(&sm.k_ready[buf], turn) && (j < 2 || tm_wait(&sm.s_free[buf], turn ^ 1));
                    if (!ok) break;
                    tm_fence_after();
                    if (elect_one()) {
                        const uint32_t q = tmem + S::kQ + ((item - 1) & 1) * (D / 2), s = tmem + S::kS + buf * kTmUnit;
#pragma unroll
                        for (uint32_t part = 0; part < S::kParts; ++part)
#pragma unroll
                            for (uint32_t c = 0; c < D / 64; ++c) tm_mma64<kTmUnit>(s, q + c * 32, smem_u32(sm.k[buf][part]) + c * (kTmUnit * 128), part | c);
                        mbar_arrive(&sm.s_full[buf]);   // what the tile warps say of the unit
                        tm_commit(&sm.s_full[buf]);
                    }
                    __syncwarp();
                }
                if (j) {
                    const uint32_t buf = (j - 1) & 1, turn = ((j - 1) >> 1) & 1;
                    ok = tm_wait(&sm.v_ready[buf], turn) && tm_wait(&sm.p_ready[buf], turn);
                    if (!ok) break;
                    tm_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t part = 0; part < S::kParts; ++part)
                            tm_mma64<D>(tmem + S::kO, tmem + S::kP + buf * (kTmUnit / 2), smem_u32(sm.v[buf][part]), part | (fresh ? 0u : 1u));
                        tm_commit(&sm.pv_done[buf]);
                    }
                    __syncwarp();
                }
            }
        } else if (warp == 2) {
            if (lane < 2) sm.edge[lane] = item_of<kTmRows, kTmUnit>(p, sm.cum, lane ? u1 - 1 : u0);
        } else if (warp == 3) {
            // ---- what there is to know of a unit before its tiles are made: slots that count as zero, largest scales
            uint64_t end = u0, start = 0, length = 0, total = 0;
            for (uint32_t j = 0; j < n; ++j) {
                if (u0 + j >= end) {
                    const AttnItem it = item_of<kTmRows, kTmUnit>(p, sm.cum, u0 + j);
                    end = it.end; start = it.start; length = it.length; total = it.total;
                }
                const uint32_t st = j % S::kStages;
                ok = tm_wait(&sm.code_full[st], (j / S::kStages) & 1);
                if (!ok) break;
                uint8_t* stage = sm.ring[st];
                const uint64_t slot0 = (u0 + j - start) * kTmUnit;
                // Two copies of the code, as the softmax has: what the end of the context needs delays no unit inside it (one copy: 8 % more)
                auto look = [&](auto edge_tag) {
                    constexpr bool EDGE = decltype(edge_tag)::value;
                    uint64_t drop = 0, odd_slots = 0;
                    const bool gone = EDGE && sm.gone[j % 8] != 0;
                    if (EDGE && !gone) {
                        const uint64_t there = total - slot0 >= 64 ? ~0ull : (1ull << (total - slot0)) - 1;
                        const uint64_t drafted = slot0 >= length ? ~0ull : ~0ull << (length - slot0);
                        uint32_t odd[2] = {0, 0};
                        if constexpr (Q8) {
                            for (uint32_t i = lane; i < kTmGroups * NB * kKvGroup; i += 32) {
                                const uint32_t gi = i / (NB * kKvGroup), x = i % (NB * kKvGroup), slot = gi * kKvGroup + x % kKvGroup;
                                const uint32_t is = (*reinterpret_cast<const uint16_t*>(stage + gi * S::kGroupBytes + S::kHalf + kKvGroup * D + x * 2) & 0x7c00u) == 0x7c00u;
                                if (slot < 32) odd[0] |= is << slot; else odd[1] |= is << (slot - 32);
                            }
                        } else {
                            for (uint32_t i = lane; i < kTmUnit * D; i += 32) {   // halves of V: [group][32 dims][m][g][t][i][e]
                                const uint32_t gi = i / (kKvGroup * D), x = i % (kKvGroup * D), e = x % 4, tt = x / 8 % 4, slot = gi * kKvGroup + 2 * tt + (e & 1) + 8 * (e >> 1);
                                const uint32_t is = (*reinterpret_cast<const uint16_t*>(stage + gi * S::kGroupBytes + S::kHalf + x * 2) & 0x7c00u) == 0x7c00u;
                                if (slot < 32) odd[0] |= is << slot; else odd[1] |= is << (slot - 32);
                            }
                        }
                        odd_slots = (static_cast<uint64_t>(__reduce_or_sync(NONE, odd[1])) << 32 | __reduce_or_sync(NONE, odd[0])) & drafted & there;
                        drop = odd_slots | ~there;
                    }
                    int ek = 21, ev = 21;
                    [[maybe_unused]] uint32_t wild = 0;
                    if constexpr (Q8) {   // largest scales: below 2^(e - 14), e the binary16 exponent; the tiles are times 2^(21 - e), codes times scales below 2^14
                        uint32_t top[2];
                        [[maybe_unused]] uint32_t low[2];   // smallest scales that are not zero, less one
#pragma unroll
                        for (uint32_t side = 0; side < 2; ++side) {
                            constexpr uint32_t EACH = NB * 2;   // 16-byte pieces of a group's scales: eight slots of a block of 32 dims
                            const uint32_t gi = lane / EACH % kTmGroups, x = lane % EACH;   // head_dim 64: the upper lanes look at the same again
                            const uint4 d = *reinterpret_cast<const uint4*>(stage + gi * S::kGroupBytes + side * S::kHalf + kKvGroup * D + x * 16);
                            uint32_t words[4] = {d.x & 0x7fff7fffu, d.y & 0x7fff7fffu, d.z & 0x7fff7fffu, d.w & 0x7fff7fffu};
                            if constexpr (EDGE) {
                                const uint32_t out = static_cast<uint32_t>(drop >> (gi * kKvGroup + x % 2 * 8));
                                uint32_t least = 0xffffffffu;
#pragma unroll
                                for (uint32_t c = 0; c < 4; ++c) {
                                    words[c] &= (out >> (2 * c) & 1 ? 0u : 0x0000ffffu) | (out >> (2 * c) & 2 ? 0u : 0xffff0000u);
                                    least = __vminu2(least, __vsub2(words[c], 0x00010001u));   // zero wraps
                                }
                                low[side] = min(least & 0xffffu, least >> 16);
                            }
                            const uint32_t most = __vmaxu2(__vmaxu2(words[0], words[1]), __vmaxu2(words[2], words[3]));
                            top[side] = max(most & 0xffffu, most >> 16);
                        }
                        ek = static_cast<int>(min(max(__reduce_max_sync(NONE, top[0]) >> 10, 1u), 30u));
                        ev = static_cast<int>(min(max(__reduce_max_sync(NONE, top[1]) >> 10, 1u), 30u));
                        if constexpr (EDGE) {
                            // no two blocks so far apart: no two slots
                            auto far = [&](uint32_t side) { return static_cast<uint32_t>(side ? ev : ek) > max((side ? low[1] : low[0]) >> 10, 1u) + kTmSpread; };
                            if (__any_sync(NONE, far(0) || far(1)) && !gone) {
#pragma unroll 1
                                for (uint32_t side = 0; side < 2; ++side) {
                                    if (!__any_sync(NONE, far(side))) continue;
                                    wild |= 1u << side;
                                    auto scale_of = [&](uint32_t slot, uint32_t b) {
                                        return reinterpret_cast<__half*>(stage + slot / kKvGroup * S::kGroupBytes + side * S::kHalf + kKvGroup * D) + b * kKvGroup + slot % kKvGroup;
                                    };
#pragma unroll 1
                                    for (uint32_t slot = lane; slot < kTmUnit; slot += 32) {
                                        uint32_t own = 0;
#pragma unroll 1
                                        for (uint32_t b = 0; b < NB; ++b) own = max(own, __half_as_ushort(*scale_of(slot, b)) & 0x7fffu);
                                        const uint32_t up = drop >> slot & 1 || !own ? 0u : static_cast<uint32_t>(side ? ev : ek) - min(max(own >> 10, 1u), 30u);
                                        (side ? sm.v_raised : sm.k_raised)[j % 8][slot] = static_cast<uint8_t>(up);
#pragma unroll 1
                                        for (uint32_t b = 0; up && b < NB; ++b) *scale_of(slot, b) = __float2half_rn(__half2float(*scale_of(slot, b)) * pow2(static_cast<int>(up)));
                                    }
                                }
                                fence_async_smem();   // the lanes' writes, before the copy that fills the stage next
                                __syncwarp();
                            }
                        }
                    }
                    if (lane == 0) {
                        sm.k_lift[j % 8] = 21 - ek; sm.v_lift[j % 8] = 21 - ev;
                        if constexpr (EDGE) sm.wild[j % 8] = wild;
                        sm.odd[j % 8][0] = static_cast<uint32_t>(odd_slots); sm.odd[j % 8][1] = static_cast<uint32_t>(odd_slots >> 32);
                        sm.drop[j % 8][0] = static_cast<uint32_t>(drop); sm.drop[j % 8][1] = static_cast<uint32_t>(drop >> 32);
                        mbar_arrive(&sm.code_known[st]);
                    }
                    __syncwarp();
                };
                if (slot0 + kTmUnit > length) look(std::true_type{}); else look(std::false_type{});
            }
        }
        __syncwarp();
        __syncthreads();   // a warp that asked for registers now would keep asking until the others are done
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTmLaunchRegs));
    } else if (warp >= kTmTiles) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTmTileRegs));
        __syncthreads();
        // ---- tiles: four warps make those of K, four those of V, each its group of 16 slots, so that one side's waits and fences lie under the other's work
        const uint32_t gi = warp % 4, g = lane / 4, t = lane % 4;
        if (warp < kTmTiles + 4) {
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t st = j % S::kStages, round = j / S::kStages, buf = j & 1, turn = (j >> 1) & 1;
                ok = tm_wait3(&sm.code_known[st], round & 1, &sm.code_full[st], round & 1, j < 2 ? nullptr : &sm.s_full[buf], turn ^ 1);   // QK of unit j - 2 has read this tile
                if (!ok) break;
                const uint8_t* group = sm.ring[st] + gi * S::kGroupBytes;
                const float k_up = pow2(static_cast<int>(sm.k_lift[j % 8]));
                if (!sm.gone[j % 8]) {
                    // [64 dims][64 slots] rows of 128 bytes; a lane's 16 bytes are dims 8 t.. of both 32s (Q8_0) or 8 t.. of one (binary16) of slot 8 n + g
#pragma unroll
                    for (uint32_t x = 0; x < K_LINES; ++x) {
                        const uint32_t in = x % 2 * 8 + g, slot = gi * kKvGroup + in;
                        const uint4 c = *reinterpret_cast<const uint4*>(group + x * 512 + lane * 16);
                        if constexpr (Q8) {
                            // odd slots put their second half first: eight lanes on eight different 16 bytes
                            const uint32_t panel = x / 2, turned = g & 1;
                            const uint32_t words[4] = {turned ? c.z : c.x, turned ? c.w : c.y, turned ? c.x : c.z, turned ? c.y : c.w};
                            const uint8_t* scales = group + kKvGroup * D + (2 * panel * kKvGroup + in) * 2;
                            uint8_t* to = sm.k[buf][0] + panel * (kTmUnit * 128) + slot * 128;
#pragma unroll
                            for (uint32_t side = 0; side < 2; ++side) {
                                const uint32_t h = side ^ turned;
                                const __half2 d = __float2half2_rn(__half2float(*reinterpret_cast<const __half*>(scales + h * (kKvGroup * 2))) * k_up);
                                uint32_t high[4], low[4];
#pragma unroll
                                for (uint32_t x2 = 0; x2 < 2; ++x2) {
                                    uint32_t y[2];
                                    codes_to_halves(words[2 * side + x2], y[0], y[1]);
#pragma unroll
                                    for (uint32_t z = 0; z < 2; ++z) {
                                        const __half2 v = __hmul2(bits_h2(y[z]), d);
                                        high[2 * x2 + z] = h2_bits(v);
                                        low[2 * x2 + z] = h2_bits(__hfma2(bits_h2(y[z]), d, __hneg2(v)));
                                    }
                                }
                                const uint32_t at = ((4 * h + t) ^ (slot & 7)) << 4;
                                *reinterpret_cast<uint4*>(to + at) = make_uint4(high[0], high[1], high[2], high[3]);
                                *reinterpret_cast<uint4*>(to + (S::kParts - 1) * S::kKPart + at) = make_uint4(low[0], low[1], low[2], low[3]);
                            }
                        } else {
                            const uint32_t b = x / 2;   // 32 dims
                            *reinterpret_cast<uint4*>(sm.k[buf][0] + b / 2 * (kTmUnit * 128) + slot * 128 + (((b % 2 * 4 + t) ^ (slot & 7)) << 4)) = c;
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&sm.k_ready[buf]); mbar_arrive(&sm.code_empty[st]); }
            }
        } else {
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t st = j % S::kStages, round = j / S::kStages, buf = j & 1, turn = (j >> 1) & 1;
                ok = tm_wait3(&sm.code_known[st], round & 1, &sm.code_full[st], round & 1, j < 2 ? nullptr : &sm.pv_done[buf], turn ^ 1);   // PV of unit j - 2 has read this tile
                if (!ok) break;
                const uint8_t* values = sm.ring[st] + gi * S::kGroupBytes + S::kHalf;
                const float v_up = pow2(static_cast<int>(sm.v_lift[j % 8]));
                if (!sm.gone[j % 8]) {
                    uint32_t keep[2] = {NONE, NONE};
                    const uint32_t out = sm.drop[j % 8][gi / 2] >> (gi % 2 * kKvGroup) & 0xffffu;
                    if (out) {
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) keep[h] = (out >> (8 * h + 2 * t) & 1 ? 0u : 0x0000ffffu) | (out >> (8 * h + 2 * t) & 2 ? 0u : 0xffff0000u);
                    }
                    auto put = [&](uint32_t part, uint32_t dim, uint32_t h, uint32_t pair) {   // slots gi * 16 + 8 h + 2 t, + 1 of a dim
                        *reinterpret_cast<uint32_t*>(sm.v[buf][part] + dim * 128 + (((2 * gi + h) ^ (dim & 7)) << 4) + 4 * t) = pair;
                    };
                    // [dims][64 slots], rows of 128 bytes; a lane's 16 bytes are dims 8 i + g, slots 2 t, 2 t + 1, 8 more
#pragma unroll
                    for (uint32_t x = 0; x < K_LINES; ++x) {
                        const uint4 c = *reinterpret_cast<const uint4*>(values + x * 512 + lane * 16);
                        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
                        if constexpr (Q8) {
                            __half2 d[2];
#pragma unroll
                            for (uint32_t h = 0; h < 2; ++h) {
                                const float2 f = __half22float2(bits_h2(*reinterpret_cast<const uint32_t*>(values + kKvGroup * D + (x * kKvGroup + 8 * h + 2 * t) * 2) & keep[h]));
                                d[h] = __floats2half2_rn(f.x * v_up, f.y * v_up);
                            }
#pragma unroll
                            for (uint32_t q = 0; q < 4; ++q) {
                                uint32_t y[2];
                                codes_to_halves(words[q], y[0], y[1]);
#pragma unroll
                                for (uint32_t h = 0; h < 2; ++h) {
                                    const __half2 v = __hmul2(bits_h2(y[h]), d[h]);
                                    put(0, 32 * x + 8 * q + g, h, h2_bits(v));
                                    put(S::kParts - 1, 32 * x + 8 * q + g, h, h2_bits(__hfma2(bits_h2(y[h]), d[h], __hneg2(v))));
                                }
                            }
                        } else {
#pragma unroll
                            for (uint32_t q = 0; q < 2; ++q)
#pragma unroll
                                for (uint32_t h = 0; h < 2; ++h) put(0, 16 * x + 8 * q + g, h, words[2 * q + h] & keep[h]);
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&sm.v_ready[buf]); mbar_arrive(&sm.code_empty[st]); }
            }
        }
        __syncwarp();
        __syncthreads();   // a warp that asked for registers now would keep asking until the others are done
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTmLaunchRegs));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTmSoftmaxRegs));
        __syncthreads();
        // ---- softmax: a thread per query row
        const uint32_t quarter = warp - kTmSoftmax, r = quarter * 32 + lane, base = tmem + (quarter << 21);   // the warp's lanes of tensor memory
        const float f = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 0x1p-83f);   // as on the warps' MMAs
        auto place = [&](const AttnItem& it, uint32_t& node, uint32_t& head) {
            const uint32_t flat = it.tile * kTmRows + r;
            node = flat / p.group;
            head = it.head * p.group + flat % p.group;
        };
        auto load_q = [&](const AttnItem& it, uint32_t item) {
            uint32_t node, head;
            place(it, node, head);
            const uint8_t* row = p.q + static_cast<uint64_t>(it.row0 + node) * p.q_stride + head * D * 2;
            const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
            for (uint32_t h = 0; h < D / 64; ++h) {
                uint32_t x[32];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint4 v = r < it.rows ? reinterpret_cast<const uint4*>(row)[h * 8 + i] : make_uint4(0, 0, 0, 0);
                    x[4 * i] = v.x ^ flip; x[4 * i + 1] = v.y ^ flip; x[4 * i + 2] = v.z ^ flip; x[4 * i + 3] = v.w ^ flip;
                }
                tm_st32(base + S::kQ + (item & 1) * (D / 2) + h * 32, x);
            }
            tm_st_wait();
            tm_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_ready[item & 1]);
        };
        // An item is looked up where something of it is wanted, not kept: a score row of 64 leaves no registers for it
        auto item_at = [&](uint32_t unit) { return item_of<kTmRows, kTmUnit>(p, sm.cum, u0 + unit); };
        load_q(item_at(0), 0);
        uint32_t j = 0;
        for (uint32_t item = 0; j < n && ok; ++item) {
            const uint32_t first = j;
            uint32_t stop, inner;   // units of the run's part of the item, of those inside the context
            {
                const AttnItem it = item_at(j);
                stop = static_cast<uint32_t>(min(it.end, u1) - u0);
                const uint64_t plain = it.start + it.length / kTmUnit;
                inner = plain <= u0 ? 0u : static_cast<uint32_t>(min(plain - u0, static_cast<uint64_t>(stop)));
                if (stop < n) load_q(item_at(stop), item + 1);   // that buffer's last readers, the scores of the item before this one, are done
            }
            float m = -INFINITY, l = 0.f, ref = 0.f, limit = -INFINITY;
            int lift = 64;   // of the V tiles: the row's accumulator is at the smallest so far of what it sees
            bool dead = false;
            // One unit; EDGE: it reaches past the context. Two copies of the code, so that the units inside run past none of what only the others need
            // (one copy: 5 % more). False: a wait has run out.
            auto unit = [&](auto edge_tag) {
                constexpr bool EDGE = decltype(edge_tag)::value;
                const uint32_t buf = j & 1, turn = (j >> 1) & 1;
                ok = tm_wait(&sm.s_full[buf], turn);
                if (!ok) return false;
                tm_fence_after();
                if (Q8 && EDGE && (sm.wild[j % 8] & 1)) {   // scores of raised keys
#pragma unroll 1
                    for (uint32_t c = 0; c < kTmUnit; ++c) {
                        const uint32_t at = base + S::kS + buf * kTmUnit + c;
                        tm_st1(at, __float_as_uint(__uint_as_float(tm_ld1(at)) * pow2(-static_cast<int>(sm.k_raised[j % 8][c]))));
                    }
                    tm_st_wait();
                }
                float s[2][32];
                tm_ld32(base + S::kS + buf * kTmUnit, s[0]);
                tm_ld32(base + S::kS + buf * kTmUnit + 32, s[1]);
                tm_ld_wait();
                tm_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.s_free[buf]);
                dead |= sm.gone[j % 8] != 0;
                const int k_lift = Q8 ? static_cast<int>(sm.k_lift[j % 8]) : 0, v_lift = Q8 ? static_cast<int>(sm.v_lift[j % 8]) : 0;
                const float fj = Q8 ? f * pow2(-k_lift) : f;
                int v_row = v_lift;   // the power of two that the row's accumulator has to be at: of the slots that it sees, if it sees any
                if constexpr (EDGE) {
                    const AttnItem it = item_at(j);
                    const uint64_t slot0 = (u0 + j - it.start) * kTmUnit;
                    uint64_t word = 0;
                    if (r < it.rows) {
                        uint32_t node, head;
                        place(it, node, head);
                        word = p.mask ? p.mask[it.row0 + node] : ~0ull >> (63 - min(node, 63u));
                    }
                    // the slots of this unit that the row sees
                    const uint64_t there = it.total - slot0 >= 64 ? ~0ull : (1ull << (it.total - slot0)) - 1;
                    uint64_t seen = slot0 >= it.length ? word >> (slot0 - it.length) : (word << (it.length - slot0)) | ((1ull << (it.length - slot0)) - 1);
                    seen &= there;
                    if (Q8 && (sm.wild[j % 8] & 2)) {
                        uint32_t least = 64;
#pragma unroll 1
                        for (uint32_t c = 0; c < kTmUnit; ++c)
                            if (seen >> c & 1) least = min(least, static_cast<uint32_t>(sm.v_raised[j % 8][c]));
                        v_row += static_cast<int>(least);
                    }
                    if (Q8 && !seen) v_row = 64;
#pragma unroll
                    for (uint32_t c = 0; c < 64; ++c) {
                        if (!(seen >> c & 1)) s[c / 32][c % 32] = -INFINITY;
                        else if (sm.odd[j % 8][c / 32] >> (c % 32) & 1) s[c / 32][c % 32] = NAN;
                    }
                }
                float x4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (uint32_t c = 0; c < 64; ++c) x4[c % 4] = fmaxf(x4[c % 4], s[c / 32][c % 32]);
                const float x = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])) * fj;
                const bool fresh = j == first;
                if (__any_sync(NONE, x > limit || v_row < lift)) {
                    float old = 1.f;
                    if (x > limit) {
                        old = m == -INFINITY ? 0.f : exp2_approx(m - x);
                        l *= m == -INFINITY ? 1.f : old;   // a NaN stays
                        m = x; limit = m + kSlack; ref = kUp - m;
                    }
                    if (!fresh) {   // the accumulator, once the products so far are in it
                        const uint32_t last = j - 1;
                        ok = tm_wait(&sm.pv_done[last & 1], (last >> 1) & 1);
                        if (!ok) return false;
                        tm_fence_after();
                        if (v_row < lift) old *= pow2(max(v_row - lift, -120));
#pragma unroll 1
                        for (uint32_t c = 0; c < D / 32; ++c) {
                            float o[32];
                            uint32_t y[32];
                            tm_ld32(base + S::kO + c * 32, o);
                            tm_ld_wait();
#pragma unroll
                            for (uint32_t i = 0; i < 32; ++i) y[i] = __float_as_uint(o[i] * old);
                            tm_st32(base + S::kO + c * 32, y);
                        }
                        tm_st_wait();
                    }
                    lift = min(lift, v_row);
                }
                // V tiles at a higher power of two than the accumulator: the weights take what is between, and the sum gives it back
                const float shift = Q8 ? static_cast<float>(min(max(lift - v_lift, -100), 0)) : 0.f;   // above 0: raised slots, or none that the row sees
                uint32_t w[32];
                float2 sum[4] = {};
                const float2 fj2 = make_float2(fj, fj), ref2 = make_float2(ref + shift, ref + shift);
#pragma unroll
                for (uint32_t c = 0; c < 32; ++c) {
                    float2 x2 = fma2(make_float2(s[c / 16][2 * c % 32], s[c / 16][2 * c % 32 + 1]), fj2, ref2);
                    x2.x = exp2_approx(x2.x); x2.y = exp2_approx(x2.y);
                    sum[c % 4] = add2(sum[c % 4], x2);
                    w[c] = h2_bits(__floats2half2_rn(x2.x, x2.y));
                }
                sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
                l = fmaf(sum[0].x + sum[0].y, Q8 ? exp2_approx(-shift) : 1.f, l);
                ok = j < 2 || tm_wait(&sm.pv_done[buf], turn ^ 1);   // PV of unit j - 2 has read this buffer
                if (!ok) return false;
                tm_fence_after();
                tm_st32(base + S::kP + buf * (kTmUnit / 2), w);
                tm_st_wait();
                if (Q8 && EDGE && (sm.wild[j % 8] & 2)) {   // weights of raised values
                    const int above = max(lift - v_lift, 0);
#pragma unroll 1
                    for (uint32_t c = 0; c < kTmUnit / 2; ++c) {
                        const uint32_t at = base + S::kP + buf * (kTmUnit / 2) + c;
                        const float2 y = __half22float2(bits_h2(tm_ld1(at)));
                        tm_st1(at, h2_bits(__floats2half2_rn(y.x * pow2(min(above - sm.v_raised[j % 8][2 * c], 0)), y.y * pow2(min(above - sm.v_raised[j % 8][2 * c + 1], 0)))));
                    }
                    tm_st_wait();
                }
                tm_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[buf]);
                return true;
            };
            for (; j < inner && unit(std::false_type{});) ++j;
            for (; ok && j < stop && unit(std::true_type{});) ++j;
            if (!ok) break;
            const uint32_t last = j - 1;
            ok = tm_wait(&sm.pv_done[last & 1], (last >> 1) & 1);
            if (!ok) break;
            tm_fence_after();
            const AttnItem it = item_at(first);
            const bool whole = it.start >= u0 && it.end <= u1;
            const float scale = Q8 ? pow2(max(min(-lift, 120), -120)) : 1.f;
            if (whole) {
                const float inv = (l == 0.f ? 0.f : 1.f / l) * scale;
                uint32_t node, head;
                place(it, node, head);
                uint8_t* dst = p.out + static_cast<uint64_t>(it.row0 + node) * p.out_stride + head * D * 2;
                bool bad = l != l;
#pragma unroll 1
                for (uint32_t pass = 0; pass < 2; ++pass) {   // whether all of it is finite, then the row
#pragma unroll 1
                    for (uint32_t c = 0; c < D / 32; ++c) {
                        float o[32];
                        tm_ld32(base + S::kO + c * 32, o);
                        tm_ld_wait();
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) { o[i] *= inv; bad |= !(fabsf(o[i]) < 65520.f); }
                        if (pass && r < it.rows) {
                            const bool zero = bad || dead;
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) {
                                uint4 v;
                                v.x = zero ? 0u : h2_bits(__floats2half2_rn(o[8 * i], o[8 * i + 1])); v.y = zero ? 0u : h2_bits(__floats2half2_rn(o[8 * i + 2], o[8 * i + 3]));
                                v.z = zero ? 0u : h2_bits(__floats2half2_rn(o[8 * i + 4], o[8 * i + 5])); v.w = zero ? 0u : h2_bits(__floats2half2_rn(o[8 * i + 6], o[8 * i + 7]));
                                reinterpret_cast<uint4*>(dst)[c * 4 + i] = v;
                            }
                        }
                    }
                }
                if (bad && !dead && r < it.rows) raise_error(p.error, TSP_ERR_NONFINITE);
            } else {
                float* part = part_at(blockIdx.x, it.start <= u0);
                __stcg(part + r, m == -INFINITY ? m : -ref);
                __stcg(part + kTmRows + r, l);
                if (r == 0) __stcg(part + 2 * kTmRows, dead ? 1.f : 0.f);
                float4* rows = reinterpret_cast<float4*>(part + kTmPartHead);
#pragma unroll 1
                for (uint32_t c = 0; c < D / 32; ++c) {
                    float o[32];
                    tm_ld32(base + S::kO + c * 32, o);
                    tm_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (r < it.rows) __stcg(rows + (c * 8 + i) * kTmRows + r, make_float4(o[4 * i] * scale, o[4 * i + 1] * scale, o[4 * i + 2] * scale, o[4 * i + 3] * scale));
                }
            }
            tm_fence_before();   // the accumulator is read before the next item's first weights are said to be ready
        }
        __syncwarp();
        __syncthreads();   // a warp that asked for registers now would keep asking until the others are done
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTmLaunchRegs));
    }
    if (!ok && lane == 0) raise_error(p.error, TSP_ERR_TIMEOUT);
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kCols) : "memory");

    // ---- pieces of the block: of the item at its start, and of another at its end
    const AttnItem &first = sm.edge[0], &last = sm.edge[1];
    const bool open0 = first.start < u0 || first.end > u1, open1 = last.start != first.start && last.end > u1;
    if (!open0 && !open1) return;
    if (tid < 2) {
        __threadfence();   // the pieces, which the barrier has ordered before this, go before the count
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
    if (tid < kTmRows / 32) sm.bad_rows[tid] = 0;
    __syncthreads();
    const uint32_t r = tid % kTmRows, lot = tid / kTmRows;   // a row by four threads, each every fourth float4; the other warps only meet them
    constexpr uint32_t LOTS = 4, V = D / 4 / LOTS;
#pragma unroll 1
    for (uint32_t side = 0; side < 2; ++side) {
        if (!sm.last[side]) continue;
        const AttnItem& it = side ? last : first;
        const uint32_t c0 = sm.span[side][0], pieces = sm.span[side][1];
        const float* part0 = part_at(c0, runs.at_run_start(it.start));
        const float* part1 = part_at(c0 + 1, true);
        auto part_of = [&](uint32_t i) { return i == 0 ? part0 : part1 + 2ull * (i - 1) * tm_part_floats(); };
        // the reference of all pieces: each lot looks at every fourth
        const bool on = lot < LOTS && r < it.rows;
        float top = -INFINITY, sum = 0.f;
        bool dead = false;
#pragma unroll 4
        for (uint32_t i = lot; i < (on ? pieces : 0); i += LOTS) top = fmaxf(top, load_piece(part_of(i) + r));
        if (on) sm.tops[lot][r] = top;
        __syncthreads();
        if (on)
#pragma unroll
            for (uint32_t x = 0; x < LOTS; ++x) top = fmaxf(top, sm.tops[x][r]);
        float4 y[V];
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (uint32_t i = 0; i < (on ? pieces : 0); ++i) {
            const float* part = part_of(i);
            const float m = load_piece(part + r), l = load_piece(part + kTmRows + r), fi = weight_of(m, top);
            dead |= load_piece(part + 2 * kTmRows) != 0.f;
            sum += m == -INFINITY ? l : l * fi;   // a row of NaN alone has a sum of NaN and no reference
            float4 v[V];
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) v[k] = load_piece4(part + kTmPartHead + ((k * LOTS + lot) * kTmRows + r) * 4);
            if (fi != 0.f)
#pragma unroll
                for (uint32_t k = 0; k < V; ++k) {
                    y[k].x = fmaf(v[k].x, fi, y[k].x); y[k].y = fmaf(v[k].y, fi, y[k].y); y[k].z = fmaf(v[k].z, fi, y[k].z); y[k].w = fmaf(v[k].w, fi, y[k].w);
                }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        bool good = sum == sum;
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            y[k].x *= inv; y[k].y *= inv; y[k].z *= inv; y[k].w *= inv;
            good &= in_range<true>(y[k].x) && in_range<true>(y[k].y) && in_range<true>(y[k].z) && in_range<true>(y[k].w);
        }
        if (!good && on) atomicOr(&sm.bad_rows[r / 32], 1u << r % 32);
        __syncthreads();
        if (on) {
            const bool bad = sm.bad_rows[r / 32] >> r % 32 & 1;
            if (bad && !dead && lot == 0) raise_error(p.error, TSP_ERR_NONFINITE);
            const uint32_t flat = it.tile * kTmRows + r, node = flat / p.group, head = it.head * p.group + flat % p.group;
            uint2* dst = reinterpret_cast<uint2*>(p.out + static_cast<uint64_t>(it.row0 + node) * p.out_stride + head * D * 2);
#pragma unroll
            for (uint32_t k = 0; k < V; ++k)
                dst[k * LOTS + lot] = bad || dead ? make_uint2(0u, 0u) : make_uint2(h2_bits(__floats2half2_rn(y[k].x, y[k].y)), h2_bits(__floats2half2_rn(y[k].z, y[k].w)));
        }
        __syncthreads();
        if (tid < kTmRows / 32) sm.bad_rows[tid] = 0;
        __syncthreads();
    }
}

uint64_t tree_mma_parts_bytes() { return 2ull * kAttnMaxBlocks * tm_part_floats() * sizeof(float); }

template <uint32_t D, bool Q8>
static int launch_tree_mma_t(const AttnParams& p, cudaStream_t st) {
    constexpr size_t smem = sizeof(TmSmem<D, Q8>) + 1024;
    static_assert(smem <= 232448, "shared memory of a block");
    static thread_local SmemAttrCache attr;
    TSP_CUDA(ensure_dynamic_smem(tree_mma_kernel<D, Q8>, attr, smem));
    const int sms = sm_count();
    const uint32_t blocks = sms < 1 ? 1 : sms < static_cast<int>(kAttnMaxBlocks) ? sms : kAttnMaxBlocks;
    TSP_CUDA(launch_pdl(tree_mma_kernel<D, Q8>, dim3(blocks), dim3(kTmThreads), smem, st, p));
    return TSP_OK;
}

template <uint32_t D, bool Q8>
static int tree_mma_registers_t(int& registers) {
    static thread_local int known = 0;
    if (!known) {
        cudaFuncAttributes fa;
        TSP_CUDA(cudaFuncGetAttributes(&fa, tree_mma_kernel<D, Q8>));
        known = fa.numRegs;
    }
    registers = known;
    return TSP_OK;
}
int tree_mma_registers(const AttnParams& p, int& registers) {
    const bool q8 = p.cache.type == TSP_TYPE_Q8_0;
    if (p.cache.head_dim == 64) return q8 ? tree_mma_registers_t<64, true>(registers) : tree_mma_registers_t<64, false>(registers);
    return q8 ? tree_mma_registers_t<128, true>(registers) : tree_mma_registers_t<128, false>(registers);
}

int launch_tree_mma(const AttnParams& p, cudaStream_t st) {   // binary16 rows, head_dim 64 or 128
    const bool q8 = p.cache.type == TSP_TYPE_Q8_0;
    if (p.cache.head_dim == 64) return q8 ? launch_tree_mma_t<64, true>(p, st) : launch_tree_mma_t<64, false>(p, st);
    return q8 ? launch_tree_mma_t<128, true>(p, st) : launch_tree_mma_t<128, false>(p, st);
}

}  // namespace tsp
