// Attention of the drafted tokens of every sequence over its paged cache (tsp_tree_attention).
#include "tsp_kv.cuh"

namespace tsp {

// One block per (row, kv head): the slots go round the warps, each with a running maximum and sum, joined at the end.
template <uint32_t D, bool F16>
__global__ void __launch_bounds__(256)
tree_attention_kernel(const tsp_kv_cache cache, const tsp_kv_batch batch, const uint8_t* q, uint64_t q_stride, const uint64_t* mask, uint32_t q_heads,
                      uint32_t max_rows, float scale, uint8_t* out, uint64_t out_stride, uint32_t* error) {
    constexpr uint32_t NV = D / 32;
    __shared__ float sm[8], sl[8], so[8][D];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t row = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    if (row == 0 && blockIdx.y == 0) kv_check_offsets(batch, error);
    uint32_t seq, node;
    if (!kv_row(batch, row, lane, seq, node)) return;
    const uint32_t drafted = batch.d_row_offsets[seq + 1] - batch.d_row_offsets[seq];
    const uint64_t length = batch.d_lengths[seq], total = length + drafted;
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    const uint32_t hb = kv_half_bytes(D, q8), group = q_heads / cache.kv_heads, es = F16 ? 2 : 4;
    bool dead = false;
    if (drafted > max_rows || total > static_cast<uint64_t>(cache.table_stride) * cache.page_tokens) { raise_error(error, TSP_ERR_INDEX); dead = true; }
    const uint64_t word = mask ? mask[row] : ~0ull >> (63 - min(node, 63u));
    for (uint32_t g = 0; g < group; ++g) {
        const uint32_t head = blockIdx.y * group + g;
        float qv[NV], o[NV], m = -INFINITY, l = 0.f;
        for (uint32_t i = 0; i < NV; ++i) {
            const uint8_t* p = q + row * q_stride + (head * D + lane * NV + i) * es;
            qv[i] = (F16 ? __half2float(*reinterpret_cast<const __half*>(p)) : *reinterpret_cast<const float*>(p)) * scale;
            o[i] = 0.f;
        }
        for (uint64_t slot = warp; slot < total && !dead; slot += 8) {
            if (slot >= length && !(word >> (slot - length) & 1)) continue;
            const uint8_t* part = kv_group(cache, seq, slot, blockIdx.y, error);
            if (!part) { l = NAN; break; }
            const uint32_t t = slot % kKvGroup, x0 = lane * NV;
            const float dk = q8 ? __half2float(*reinterpret_cast<const __half*>(part + kv_scale_byte(x0, t, D))) : 1.f;
            const float dv = q8 ? __half2float(*reinterpret_cast<const __half*>(part + hb + kv_scale_byte(x0, t, D))) : 1.f;
            float s = 0.f, v[NV];
            for (uint32_t i = 0; i < NV; ++i) {
                const uint8_t *pk = part + kv_k_byte(x0 + i, t, q8), *pv = part + hb + kv_v_byte(x0 + i, t, q8);
                const float k = q8 ? (static_cast<int>(*pk) - 128) * dk : __half2float(*reinterpret_cast<const __half*>(pk));
                v[i] = q8 ? (static_cast<int>(*pv) - 128) * dv : __half2float(*reinterpret_cast<const __half*>(pv));
                s = fmaf(qv[i], k, s);
            }
            for (int x = 16; x; x /= 2) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float top = fmaxf(m, s), f = expf(m - top), p = expf(s - top);
            l = l * f + p;
            for (uint32_t i = 0; i < NV; ++i) o[i] = o[i] * f + p * v[i];
            m = top;
        }
        __syncthreads();
        if (lane == 0) { sm[warp] = m; sl[warp] = l; }
        for (uint32_t i = 0; i < NV; ++i) so[warp][lane * NV + i] = o[i];
        __syncthreads();
        float top = -INFINITY, sum = 0.f;
        bool ok = true;
        for (int w = 0; w < 8; ++w) top = fmaxf(top, sm[w]);
        for (int w = 0; w < 8; ++w) sum += sm[w] == -INFINITY && !(sl[w] != sl[w]) ? 0.f : sl[w] * (sm[w] == -INFINITY ? 1.f : expf(sm[w] - top));
        float y = 0.f;
        if (threadIdx.x < D) {
            for (int w = 0; w < 8; ++w) if (sm[w] != -INFINITY) y += so[w][threadIdx.x] * expf(sm[w] - top);
            y = sum == 0.f ? 0.f : y / sum;
            ok = F16 ? fabsf(y) < 65520.f : finite_f32(y);
        }
        ok = __syncthreads_and(ok);
        if (!ok && threadIdx.x == 0) raise_error(error, TSP_ERR_NONFINITE);
        if (threadIdx.x < D) {
            uint8_t* p = out + row * out_stride + (head * D + threadIdx.x) * es;
            if (F16) *reinterpret_cast<__half*>(p) = __float2half_rn(ok ? y : 0.f); else *reinterpret_cast<float*>(p) = ok ? y : 0.f;
        }
    }
}

int launch_tree_attention(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const void* q, uint64_t q_stride, const uint64_t* mask, uint32_t q_heads,
                          uint32_t max_rows, float scale, void* out, uint64_t out_stride, uint32_t dtype, void* scratch, uint32_t* error, cudaStream_t st) {
    (void)scratch;
    auto kernel = cache.head_dim == 64    ? (dtype ? tree_attention_kernel<64, true> : tree_attention_kernel<64, false>)
                  : cache.head_dim == 128 ? (dtype ? tree_attention_kernel<128, true> : tree_attention_kernel<128, false>)
                                          : (dtype ? tree_attention_kernel<256, true> : tree_attention_kernel<256, false>);
    TSP_CUDA(launch_pdl(kernel, dim3(batch.rows, cache.kv_heads), dim3(256), 0, st, cache, batch, static_cast<const uint8_t*>(q), q_stride, mask, q_heads, max_rows,
                        scale, static_cast<uint8_t*>(out), out_stride, error));
    return TSP_OK;
}

uint64_t tree_attention_scratch_bytes() { return 16; }

}  // namespace tsp
