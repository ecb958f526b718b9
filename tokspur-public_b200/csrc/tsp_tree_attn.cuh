// What the two kernels of tsp_tree_attention share: parameters, the items that a batch is cut into, small arithmetic.
#pragma once

#include "tsp_kv.cuh"
#include "tsp_tree_rule.h"

namespace tsp {

constexpr uint32_t kAttnMaxBlocks = 192;     // blocks (one per SM) that the scratch has room for
// The reference of a row moves when a score passes it by more than 2^kSlack: weights (times value scales, times a power of two 2^lift) stay below 2^15 in
// binary16, which then reaches down to 2^-31 of the reference.
constexpr float kSlack = 8.f, kUp = 7.f;

struct AttnParams {
    tsp_kv_cache cache;
    tsp_kv_batch batch;
    const uint8_t* q; uint64_t q_stride;
    const uint64_t* mask;
    uint8_t* out; uint64_t out_stride;
    uint32_t group, max_rows;
    float scale;
    uint32_t* counters;   // [kAttnMaxBlocks], zero between calls
    float* parts;         // pieces of items, the kernel's own layout
    uint32_t* error;
};

struct AttnItem {
    uint64_t start, end;     // units of the item
    uint64_t length, total;  // slots of the context, and with the step's own
    uint32_t seq, head, tile, row0, drafted, rows;   // rows: of this tile
    bool dead;               // out of range: zeros
};

// Between a thread's reads (or writes) of shared memory and what asynchronous copies (or MMAs) do to it next: the copies write through another proxy, so that
// neither a warp barrier nor an arrival alone keeps them behind reads whose values nobody has used yet. Every thread that has read fences, then the warp meets.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Pieces lie in shared memory or were written by other blocks: generic addresses, past the L1
__device__ __forceinline__ float load_piece(const float* p) {
    float v;
    asm volatile("ld.relaxed.gpu.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_piece4(const float* p) {
    float4 v;
    asm volatile("ld.relaxed.gpu.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
template <bool F16> __device__ __forceinline__ bool in_range(float v) { return F16 ? fabsf(v) < 65520.f : finite_f32(v); }
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : exp2_approx(m - top); }
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
// four codes + 128 -> two pairs of binary16 integers: 0x64 in front of a byte is 1024 + byte
__device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    const __half2 bias = bits_h2(0x64806480u);   // 1152
    a = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4140)), bias));
    b = h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, 0x4342)), bias));
}
// the same bytes as 1024 + code + 128, for products whose sum starts at -1152 times the sum of the other side
__device__ __forceinline__ void biased_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    a = __byte_perm(w, 0x64646464u, 0x4140);
    b = __byte_perm(w, 0x64646464u, 0x4342);
}
__device__ __forceinline__ void mma_f16_16816_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t pack_low(float u, float v, uint32_t high) {   // what rounding to `high` left out
    const float2 f = __half22float2(bits_h2(high));
    return h2_bits(__floats2half2_rn(u - f.x, v - f.y));
}
__device__ __forceinline__ bool odd_half(uint32_t bits) { return (bits & 0x7c00u) == 0x7c00u; }

// Geometry of a sequence: units of an item, row tiles
template <uint32_t R, uint32_t UNIT = kKvGroup>
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

template <uint32_t R, uint32_t UNIT = kKvGroup>
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
    sequence_shape<R, UNIT>(p, lo, i.row0, i.drafted, i.length, units, tiles, i.dead);
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

// Units before every sequence, cum[sequences]: all of them; by a block of THREADS, which meets at the end
template <uint32_t R, uint32_t UNIT, uint32_t THREADS>
__device__ __forceinline__ void unit_prefix(const AttnParams& p, uint64_t* cum, uint64_t* warp_sums) {
    constexpr uint32_t EACH = (TSP_KV_MAX_SEQUENCES + THREADS - 1) / THREADS;
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32, per = (p.batch.sequences + THREADS - 1) / THREADS;
    uint64_t mine[EACH], sum = 0;
    bool bad = false;
#pragma unroll
    for (uint32_t k = 0; k < EACH; ++k) {
        const uint32_t s = tid * per + k;
        mine[k] = sum;
        if (k < per && s < p.batch.sequences) {
            uint32_t row0, drafted, tiles;
            uint64_t length, units;
            bool dead;
            sequence_shape<R, UNIT>(p, s, row0, drafted, length, units, tiles, dead);
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
    if (lane == 31) warp_sums[warp] = run;
    __syncthreads();
    uint64_t base = run - sum;
    for (uint32_t w = 0; w < warp; ++w) base += warp_sums[w];
#pragma unroll
    for (uint32_t k = 0; k < EACH; ++k) {
        const uint32_t s = tid * per + k;
        if (k < per && s < p.batch.sequences) cum[s] = base + mine[k];
    }
    if (tid == THREADS - 1) cum[p.batch.sequences] = base + sum;
    if (blockIdx.x == 0) kv_check_offsets(p.batch, p.error);
    __syncthreads();
}

// Which units a block runs over, and which blocks an item has. The units of a ragged batch are dealt in equal runs, whatever item they are of. A single
// sequence's items (heads, row tiles) are all alike: where there are no more of them than blocks, every item gets the same number of blocks of its
// own, so that no block has pieces of two to join (one token over 4096 slots 15.8 us, in equal runs 19).
struct AttnRuns {
    uint64_t quota, item;   // units of a block's run; of an item where items have blocks of their own, else 0
    uint32_t blocks;        // of an item then

    __device__ __forceinline__ AttnRuns(const AttnParams& p, uint64_t units, const AttnItem& any, uint32_t least) : item(0), blocks(0) {
        const uint64_t each = any.end - any.start, items = units / each;
        if (p.batch.sequences == 1 && items <= gridDim.x) {
            item = each;
            blocks = gridDim.x / static_cast<uint32_t>(items);
            quota = max(static_cast<uint64_t>(least), (each + blocks - 1) / blocks);
        } else quota = max(static_cast<uint64_t>(least), (units + gridDim.x - 1) / gridDim.x);
    }
    __device__ __forceinline__ void run(uint32_t block, uint64_t units, uint64_t& u0, uint64_t& u1) const {
        if (item) {
            const uint64_t start = block / blocks * item;
            u0 = min(start + block % blocks * quota, start + item);
            u1 = min(u0 + quota, start + item);
            if (start >= units) u0 = u1 = units;
        } else {
            u0 = min(units, block * quota);
            u1 = min(units, u0 + quota);
        }
    }
    // first block of the item that starts at unit `start`, and how many it has
    __device__ __forceinline__ uint32_t first(uint64_t start) const { return static_cast<uint32_t>(item ? start / item * blocks : start / quota); }
    __device__ __forceinline__ uint32_t count(uint64_t start, uint64_t end) const {
        return static_cast<uint32_t>(item ? (item + quota - 1) / quota : (end - 1) / quota - start / quota + 1);
    }
    __device__ __forceinline__ bool at_run_start(uint64_t start) const { return item != 0 || start % quota == 0; }   // of that first block
};

}  // namespace tsp
