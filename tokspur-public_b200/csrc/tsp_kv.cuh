// Paged key / value cache: where a slot's values lie. The layout (include/tsp_moe.h) is
// the order in which the attention kernels' MMA operands want the bytes: a lane's 16 bytes of K are 16 dims of one slot (8 + 8 of two blocks
// of 32, so that the products of one MMA share a scale), its 16 bytes of V are 4 dims x 4 slots; both are whole 512-byte rows per warp.
#pragma once

#include "tsp_common.cuh"

namespace tsp {

constexpr uint32_t kKvGroup = 16;   // slots whose bytes lie together

// Bytes of one group's K part (values and scales); V has as many. dim * 16 codes + dim / 32 * 16 scales of two bytes, or dim * 16 halves.
__host__ __device__ constexpr uint32_t kv_half_bytes(uint32_t dim, bool q8) { return q8 ? 17u * dim : 32u * dim; }
__host__ __device__ constexpr uint32_t kv_group_bytes(uint32_t dim, bool q8) { return 2u * kv_half_bytes(dim, q8); }

// Byte of dim x of slot t (0..15) within the K part of its group, of its scale within the K or V part
__device__ __forceinline__ uint32_t kv_k_byte(uint32_t x, uint32_t t, bool q8) {
    return q8 ? (x / 64 * kKvGroup + t) * 64 + x % 32 / 8 * 16 + x % 64 / 32 * 8 + x % 8 : (x / 32 * kKvGroup + t) * 64 + x % 32 * 2;
}
__device__ __forceinline__ uint32_t kv_scale_byte(uint32_t x, uint32_t t, uint32_t dim) { return kKvGroup * dim + (x / 32 * kKvGroup + t) * 2; }

// Start of the group of `slot` of head h, NULL (and TSP_ERR_INDEX) where the table does not hold the slot or its entry names no page
__device__ __forceinline__ uint8_t* kv_group(const tsp_kv_cache& c, uint32_t seq, uint64_t slot, uint32_t h, uint32_t* error) {
    const uint64_t entry = slot / c.page_tokens;
    if (entry < c.table_stride) {
        const uint32_t page = c.d_page_table[static_cast<uint64_t>(seq) * c.table_stride + entry];
        if (page < c.pages) {
            const uint32_t group = h * (c.page_tokens / kKvGroup) + static_cast<uint32_t>(slot % c.page_tokens) / kKvGroup;
            return static_cast<uint8_t*>(c.d_pages) + page * c.page_stride_bytes + static_cast<uint64_t>(group) * kv_group_bytes(c.head_dim, c.type == TSP_TYPE_Q8_0);
        }
    }
    raise_error(error, TSP_ERR_INDEX);
    return nullptr;
}

// Sequence of a row, by a whole warp in two steps of 32 offsets each (sequences <= 1024); false for a row of the padding
__device__ __forceinline__ bool kv_row(const tsp_kv_batch& b, uint32_t row, uint32_t lane, uint32_t& seq, uint32_t& node) {
    const uint32_t step = (b.sequences + 31) / 32;
    const uint32_t a = __popc(__ballot_sync(0xffffffffu, (lane + 1) * step <= b.sequences && b.d_row_offsets[min((lane + 1) * step, b.sequences)] <= row)) * step;
    seq = a + __popc(__ballot_sync(0xffffffffu, lane < step && a + lane + 1 <= b.sequences && b.d_row_offsets[min(a + lane + 1, b.sequences)] <= row));
    if (seq >= b.sequences) return false;
    const uint32_t first = b.d_row_offsets[seq], end = b.d_row_offsets[seq + 1];
    node = row - first;
    return first <= row && row < end && end <= b.rows;
}

// 8 x 8 matrix of binary16 over a warp, transposed: lane (g, t) gives entries (g, 2t), (g, 2t + 1) and gets (2t, g), (2t + 1, g)
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Offsets that do not start at 0, descend or pass the rows: raised by the threads of one block
__device__ __forceinline__ void kv_check_offsets(const tsp_kv_batch& b, uint32_t* error) {
    bool bad = false;
    for (uint32_t i = threadIdx.x; i <= b.sequences; i += blockDim.x) {
        const uint32_t at = b.d_row_offsets[i];
        bad |= at > b.rows || (i == 0 ? at != 0 : b.d_row_offsets[i - 1] > at);
    }
    if (bad) raise_error(error, TSP_ERR_INDEX);
}

}  // namespace tsp
