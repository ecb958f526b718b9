// Query / key head norm and rotation, and the paged key / value cache that the rows go into: written (quantised), read back, compacted.
#include <type_traits>

#include "tsp_kv.cuh"

namespace tsp {

constexpr uint32_t kHeadThreads = 256;

template <bool F16> __device__ __forceinline__ float load1(const uint8_t* p, uint32_t i) {
    if constexpr (F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    else return reinterpret_cast<const float*>(p)[i];
}
template <bool F16> __device__ __forceinline__ void load4(const uint8_t* p, uint32_t i, float (&v)[4]) {
    if constexpr (F16) {
        const uint2 u = *reinterpret_cast<const uint2*>(p + i * 2);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    } else {
        const float4 u = *reinterpret_cast<const float4*>(p + i * 4);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
}
template <bool F16> __device__ __forceinline__ void store4(uint8_t* p, uint32_t i, const float (&v)[4]) {
    if constexpr (F16) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(p + i * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else *reinterpret_cast<float4*>(p + i * 4) = make_float4(v[0], v[1], v[2], v[3]);
}
template <bool F16> __device__ __forceinline__ bool fits(float v) { return F16 ? fabsf(v) < 65520.f : finite_f32(v); }   // 65520 rounds to infinity in binary16

// y / d rounded half to even, of the exact quotient: the rounded product may be one off, or sit on the wrong side of a tie; the remainder
// y - r d is exact (r and d have 18 bits between them, and |y - r d| <= d over a grid of 2^-24 d at least)
template <typename T> __device__ __forceinline__ int code_of(T y, T d, T inv) {
    const T r0 = rint(y * inv), e2 = 2 * fma(-r0, d, y);
    int r = static_cast<int>(fmax(fmin(r0, static_cast<T>(128)), static_cast<T>(-128)));
    if (e2 > d || (e2 == d && (r & 1))) ++r;
    else if (e2 < -d || (e2 == -d && (r & 1))) --r;
    return max(-127, min(127, r));
}

// One head of K or V (a warp, lane l holds dims l NV .. l NV + NV - 1) into its slot. Returns false where it wrote zeros for it.
template <uint32_t D, typename T>
__device__ __forceinline__ bool put_head(uint8_t* half, uint32_t t, bool is_v, bool q8, uint32_t lane, T (&y)[D / 32]) {
    constexpr uint32_t NV = D / 32;
    const uint32_t x0 = lane * NV;
    bool ok = true;
    if (q8) {
        T top = 0;
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) { ok &= finite_f32(static_cast<float>(y[i])); top = fmax(top, fabs(y[i])); }
#pragma unroll
        for (uint32_t o = 1; o < 32 / NV; o *= 2) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        const __half d16 = __float2half_rn(static_cast<float>(static_cast<double>(top) / 127.0));
        ok &= !__hisinf(d16);
        ok = __all_sync(0xffffffffu, ok);
        const T d = ok ? static_cast<T>(__half2float(d16)) : static_cast<T>(0), inv = d > 0 ? 1 / d : 0;
        uint8_t code[NV];
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) code[i] = static_cast<uint8_t>(d > 0 ? code_of<T>(y[i], d, inv) + 128 : 128);
        if (is_v) {
#pragma unroll
            for (uint32_t i = 0; i < NV; ++i) half[kv_v_byte(x0 + i, t, true)] = code[i];
        } else {
            uint8_t* p = half + kv_k_byte(x0, t, true);
            if constexpr (NV == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(code[0] | code[1] << 8);
            else {
#pragma unroll
                for (uint32_t i = 0; i < NV; i += 4)
                    *reinterpret_cast<uint32_t*>(p + i) = code[i] | code[i + 1] << 8 | code[i + 2] << 16 | static_cast<uint32_t>(code[i + 3]) << 24;
            }
        }
        if (x0 % 32 == 0) *reinterpret_cast<__half*>(half + kv_scale_byte(x0, t, D)) = ok ? d16 : __ushort_as_half(0);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) ok &= fits<true>(static_cast<float>(y[i]));
        ok = __all_sync(0xffffffffu, ok);
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) {
            const __half v = ok ? __float2half_rn(static_cast<float>(y[i])) : __ushort_as_half(0);
            *reinterpret_cast<__half*>(half + (is_v ? kv_v_byte(x0 + i, t, false) : kv_k_byte(x0 + i, t, false))) = v;
        }
    }
    return ok;
}

struct HeadRows {
    const uint8_t *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    uint8_t *q_out, *k_out;
    uint64_t q_out_stride, k_out_stride;
    const uint32_t* positions;
    uint32_t q_heads, kv_heads;   // kv_heads: of k_out (no cache)
};

// A block per row. Angles once per row; then eight lanes' worth of pairs per group of D / 8 lanes for the rows that go out as rows, a warp per
// head for those that go into the cache.
template <uint32_t D, bool IN16, bool OUT16, bool CACHE>
__global__ void __launch_bounds__(kHeadThreads)
head_rows_kernel(const tsp_qk_norm_rope_args a, const HeadRows r, const tsp_kv_cache cache, const tsp_kv_batch batch, uint32_t* error) {
    __shared__ float cs[D / 2], sn[D / 2];
    __shared__ double cs64[CACHE ? D / 2 : 1], sn64[CACHE ? D / 2 : 1];
    __shared__ double exchange[CACHE ? kHeadThreads / 32 : 1][CACHE ? D : 1];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    uint32_t seq = 0, node = 0;
    if constexpr (CACHE) {
        if (row == 0) kv_check_offsets(batch, error);
        if (!kv_row(batch, row, lane, seq, node)) return;
    }
    const uint32_t half = a.rotary_dim / 2;
    if (half) {
        const double pos = r.positions[row];
        for (uint32_t p = tid; p < half; p += kHeadThreads) {
            const double angle = pos * static_cast<double>(a.d_inv_freq[p]);
            double s, c;
            sincos(angle, &s, &c);
            c *= a.magnitude; s *= a.magnitude;
            cs[p] = static_cast<float>(c); sn[p] = static_cast<float>(s);
            if constexpr (CACHE) { cs64[p] = c; sn64[p] = s; }
        }
        __syncthreads();
    }
    bool bad = false;
    constexpr uint32_t LANES = D / 8, PER = kHeadThreads / LANES;   // lanes of a head, heads in flight
    const uint32_t out_heads = r.q_heads + (CACHE ? 0 : r.kv_heads);
    for (uint32_t h0 = tid / LANES; h0 < (out_heads + PER - 1) / PER * PER; h0 += PER) {   // whole warps stay together for the shuffles
        const uint32_t h = min(h0, out_heads - 1), l = tid % LANES;
        const bool is_k = h >= r.q_heads;
        const uint8_t* in = is_k ? r.k + row * r.k_stride + (h - r.q_heads) * D * (IN16 ? 2 : 4) : r.q + row * r.q_stride + h * D * (IN16 ? 2 : 4);
        uint8_t* out = is_k ? r.k_out + row * r.k_out_stride + (h - r.q_heads) * D * (OUT16 ? 2 : 4) : r.q_out + row * r.q_out_stride + h * D * (OUT16 ? 2 : 4);
        const float* w = is_k ? a.d_k_norm : a.d_q_norm;
        // four pairs a lane: (u, v) at dims xu.., xv.., or interleaved in eight dims from xu on; the dims behind the rotated ones pair up as halves
        const uint32_t p0 = 4 * l, rest = p0 - half;
        const bool turned = p0 < half, pairs = turned && a.style == TSP_ROPE_PAIRS;
        const uint32_t xu = turned ? (pairs ? 2 * p0 : p0) : a.rotary_dim + rest, xv = turned ? (pairs ? xu + 4 : p0 + half) : xu + (D - a.rotary_dim) / 2;
        float u[4], v[4];
        load4<IN16>(in, xu, u);
        load4<IN16>(in, xv, v);
        float wu[4] = {1.f, 1.f, 1.f, 1.f}, wv[4] = {1.f, 1.f, 1.f, 1.f};
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
#pragma unroll
            for (uint32_t o = LANES / 2; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = 1.f / sqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) { wu[i] = w[xu + i]; wv[i] = w[xv + i]; u[i] = u[i] * inv * wu[i]; v[i] = v[i] * inv * wv[i]; }
        }
        if (turned) {
            if (pairs) {
                float t[4] = {u[0], u[2], v[0], v[2]}, s[4] = {u[1], u[3], v[1], v[3]};
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) { const float c = cs[p0 + i], n = sn[p0 + i], x = t[i]; t[i] = x * c - s[i] * n; s[i] = s[i] * c + x * n; }
                u[0] = t[0]; u[1] = s[0]; u[2] = t[1]; u[3] = s[1]; v[0] = t[2]; v[1] = s[2]; v[2] = t[3]; v[3] = s[3];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) { const float c = cs[p0 + i], n = sn[p0 + i], x = u[i]; u[i] = x * c - v[i] * n; v[i] = v[i] * c + x * n; }
            }
        }
        bool ok = true;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) ok &= fits<OUT16>(u[i]) && fits<OUT16>(v[i]);
        const uint32_t group = LANES == 32 ? 0xffffffffu : ((1u << (LANES % 32)) - 1) << (lane / LANES * LANES);
        ok = (__ballot_sync(0xffffffffu, ok) & group) == group;
        if (!ok) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) u[i] = v[i] = 0.f;
        }
        if (h0 < out_heads) {
            bad |= !ok;
            store4<OUT16>(out, xu, u);
            store4<OUT16>(out, xv, v);
        }
    }
    if constexpr (CACHE) {
        constexpr uint32_t NV = D / 32;
        const bool q8 = cache.type == TSP_TYPE_Q8_0;
        const uint64_t slot = static_cast<uint64_t>(batch.d_lengths[seq]) + node;
        const uint32_t t = slot % kKvGroup, hb = kv_half_bytes(D, q8);
        for (uint32_t h = warp; h < 2 * cache.kv_heads; h += kHeadThreads / 32) {
            const bool is_v = h >= cache.kv_heads;
            const uint32_t head = is_v ? h - cache.kv_heads : h;
            uint8_t* group = kv_group(cache, seq, slot, head, error);
            if (!group) continue;
            const uint8_t* in = is_v ? r.v + row * r.v_stride + head * D * (IN16 ? 2 : 4) : r.k + row * r.k_stride + head * D * (IN16 ? 2 : 4);
            if (is_v) {
                float y[NV];
#pragma unroll
                for (uint32_t i = 0; i < NV; ++i) y[i] = load1<IN16>(in, lane * NV + i);
                bad |= !put_head<D, float>(group + hb, t, true, q8, lane, y);
            } else {
                double y[NV];
#pragma unroll
                for (uint32_t i = 0; i < NV; ++i) y[i] = load1<IN16>(in, lane * NV + i);
                if (a.d_k_norm) {
                    double ss = 0;
#pragma unroll
                    for (uint32_t i = 0; i < NV; ++i) ss = fma(y[i], y[i], ss);
#pragma unroll
                    for (uint32_t o = 16; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const double inv = 1.0 / sqrt(ss / D + static_cast<double>(a.eps));
#pragma unroll
                    for (uint32_t i = 0; i < NV; ++i) y[i] = y[i] * inv * static_cast<double>(a.d_k_norm[lane * NV + i]);
                }
                if (half) {
                    double* mine = exchange[warp];
                    __syncwarp();
#pragma unroll
                    for (uint32_t i = 0; i < NV; ++i) mine[lane * NV + i] = y[i];
                    __syncwarp();
#pragma unroll
                    for (uint32_t i = 0; i < NV; ++i) {
                        const uint32_t x = lane * NV + i;
                        if (x < a.rotary_dim) {
                            const bool pairs = a.style == TSP_ROPE_PAIRS, second = pairs ? x & 1 : x >= half;
                            const uint32_t p = pairs ? x / 2 : (second ? x - half : x), other = pairs ? x ^ 1 : (second ? x - half : x + half);
                            y[i] = second ? y[i] * cs64[p] + mine[other] * sn64[p] : y[i] * cs64[p] - mine[other] * sn64[p];
                        }
                    }
                }
                bad |= !put_head<D, double>(group, t, false, q8, lane, y);
            }
        }
    }
    if (bad) raise_error(error, TSP_ERR_NONFINITE);
}

template <uint32_t D, bool OUT16>
__global__ void __launch_bounds__(256)
cache_read_kernel(const tsp_kv_cache cache, const tsp_kv_batch batch, uint8_t* k, uint64_t k_stride, uint8_t* v, uint64_t v_stride, uint32_t* error) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr uint32_t NV = D / 32;
    const uint32_t row = blockIdx.x, lane = threadIdx.x % 32;
    if (row == 0) kv_check_offsets(batch, error);
    uint32_t seq, node;
    if (!kv_row(batch, row, lane, seq, node)) return;
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    const uint64_t slot = static_cast<uint64_t>(batch.d_lengths[seq]) + node;
    const uint32_t t = slot % kKvGroup, hb = kv_half_bytes(D, q8), x0 = lane * NV;
    for (uint32_t h = threadIdx.x / 32; h < 2 * cache.kv_heads; h += 8) {
        const bool is_v = h >= cache.kv_heads;
        const uint32_t head = is_v ? h - cache.kv_heads : h;
        uint8_t* out = is_v ? v : k;
        if (!out) continue;
        out += row * (is_v ? v_stride : k_stride) + head * D * (OUT16 ? 2 : 4);
        const uint8_t* part = kv_group(cache, seq, slot, head, error);
        if (!part) continue;
        part += is_v ? hb : 0;
        const float d = q8 ? __half2float(*reinterpret_cast<const __half*>(part + kv_scale_byte(x0, t, D))) : 1.f;
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) {
            const uint8_t* p = part + (is_v ? kv_v_byte(x0 + i, t, q8) : kv_k_byte(x0 + i, t, q8));
            const float y = q8 ? static_cast<float>(static_cast<int>(*p) - 128) * d : __half2float(*reinterpret_cast<const __half*>(p));
            if constexpr (OUT16) reinterpret_cast<__half*>(out)[x0 + i] = __float2half_rn(y);
            else reinterpret_cast<float*>(out)[x0 + i] = y;
        }
    }
}

// A block per (sequence, head): every source row is in shared memory before the first destination is written (a destination may be a
// later row's source only through an index below it, which ascending indices rule out, but rows move in parallel here).
__global__ void __launch_bounds__(256)
cache_keep_kernel(const tsp_kv_cache cache, const tsp_kv_batch batch, const uint32_t* accepted, const uint32_t* counts, uint32_t* error) {
    extern __shared__ uint8_t staged[];
    __shared__ uint32_t from[TSP_KV_MAX_DRAFT];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t s = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    if (s == 0 && h == 0) kv_check_offsets(batch, error);
    const uint32_t first = batch.d_row_offsets[s], end = batch.d_row_offsets[s + 1], n = counts[s];
    if (n == 0) return;
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    const uint64_t length = batch.d_lengths[s];
    bool bad = end < first || end > batch.rows || n > TSP_KV_MAX_DRAFT || n > end - first;
    if (!bad && tid < n) {
        const uint32_t x = accepted[first + tid];
        bad = x >= end - first || (tid && accepted[first + tid - 1] >= x);
        from[tid] = x;
    }
    if (__syncthreads_or(bad)) { if (tid == 0) raise_error(error, TSP_ERR_INDEX); return; }
    const uint32_t dim = cache.head_dim, row_bytes = q8 ? 2 * (dim + dim / 16) : 4 * dim, hb = kv_half_bytes(dim, q8);
    // every page that is read or written exists
    if (tid < n) bad = !kv_group(cache, s, length + from[tid], h, error) || !kv_group(cache, s, length + tid, h, error);
    if (__syncthreads_or(bad)) return;
    const uint32_t unit = q8 ? 1 : 2, values = dim * 2, per = values + (q8 ? dim / 16 : 0);   // values of K and V, then scales
    for (int pass = 0; pass < 2; ++pass) {
        for (uint32_t i = tid; i < n * per; i += 256) {
            const uint32_t j = i / per, c = i % per;
            const uint64_t slot = length + (pass ? j : from[j]);
            uint8_t* part = kv_group(cache, s, slot, h, error);
            const uint32_t t = slot % kKvGroup;
            uint8_t* mine = staged + j * row_bytes;
            if (c < values) {
                const bool is_v = c >= dim;
                const uint32_t x = is_v ? c - dim : c;
                uint8_t* p = part + (is_v ? hb + kv_v_byte(x, t, q8) : kv_k_byte(x, t, q8));
                if (q8) { if (pass) *p = mine[c]; else mine[c] = *p; }
                else if (pass) *reinterpret_cast<uint16_t*>(p) = reinterpret_cast<uint16_t*>(mine)[c];
                else reinterpret_cast<uint16_t*>(mine)[c] = *reinterpret_cast<uint16_t*>(p);
            } else {
                const uint32_t b = c - values, is_v = b >= dim / 32;
                uint16_t* p = reinterpret_cast<uint16_t*>(part + (is_v ? hb : 0) + kv_scale_byte((is_v ? b - dim / 32 : b) * 32, t, dim));
                uint16_t* m = reinterpret_cast<uint16_t*>(mine + values * unit) + b;
                if (pass) *p = *m; else *m = *p;
            }
        }
        __syncthreads();
    }
}

template <uint32_t D, bool IN16, bool OUT16>
static int launch_head_rows_d(const tsp_qk_norm_rope_args& a, const HeadRows& r, const tsp_kv_cache* cache, const tsp_kv_batch* batch, uint32_t rows, uint32_t* error,
                              cudaStream_t st) {
    if (cache) TSP_CUDA(launch_pdl(head_rows_kernel<D, IN16, OUT16, true>, dim3(rows), dim3(kHeadThreads), 0, st, a, r, *cache, *batch, error));
    else TSP_CUDA(launch_pdl(head_rows_kernel<D, IN16, OUT16, false>, dim3(rows), dim3(kHeadThreads), 0, st, a, r, tsp_kv_cache{}, tsp_kv_batch{}, error));
    return TSP_OK;
}

template <uint32_t D>
static int launch_head_rows_t(const tsp_qk_norm_rope_args& a, const HeadRows& r, uint32_t in_dtype, uint32_t out_dtype, const tsp_kv_cache* cache,
                              const tsp_kv_batch* batch, uint32_t rows, uint32_t* error, cudaStream_t st) {
    return in_dtype ? (out_dtype ? launch_head_rows_d<D, true, true>(a, r, cache, batch, rows, error, st) : launch_head_rows_d<D, true, false>(a, r, cache, batch, rows, error, st))
                    : (out_dtype ? launch_head_rows_d<D, false, true>(a, r, cache, batch, rows, error, st) : launch_head_rows_d<D, false, false>(a, r, cache, batch, rows, error, st));
}

int launch_head_rows(const tsp_qk_norm_rope_args& a, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride,
                     uint32_t in_dtype, const uint32_t* positions, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, void* q_out, uint64_t q_out_stride,
                     void* k_out, uint64_t k_out_stride, uint32_t out_dtype, const tsp_kv_cache* cache, const tsp_kv_batch* batch, uint32_t* error, cudaStream_t st) {
    const HeadRows r{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), q_stride, k_stride, v_stride,
                     static_cast<uint8_t*>(q_out), static_cast<uint8_t*>(k_out), q_out_stride, k_out_stride, positions, q_heads, kv_heads};
    return a.head_dim == 64    ? launch_head_rows_t<64>(a, r, in_dtype, out_dtype, cache, batch, rows, error, st)
           : a.head_dim == 128 ? launch_head_rows_t<128>(a, r, in_dtype, out_dtype, cache, batch, rows, error, st)
                               : launch_head_rows_t<256>(a, r, in_dtype, out_dtype, cache, batch, rows, error, st);
}

int launch_cache_read(const tsp_kv_cache& cache, const tsp_kv_batch& batch, void* k, uint64_t k_stride, void* v, uint64_t v_stride, uint32_t dtype, uint32_t* error,
                      cudaStream_t st) {
    auto kernel = cache.head_dim == 64    ? (dtype ? cache_read_kernel<64, true> : cache_read_kernel<64, false>)
                  : cache.head_dim == 128 ? (dtype ? cache_read_kernel<128, true> : cache_read_kernel<128, false>)
                                          : (dtype ? cache_read_kernel<256, true> : cache_read_kernel<256, false>);
    TSP_CUDA(launch_pdl(kernel, dim3(batch.rows), dim3(256), 0, st, cache, batch, static_cast<uint8_t*>(k), k_stride, static_cast<uint8_t*>(v), v_stride, error));
    return TSP_OK;
}

int launch_cache_keep(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const uint32_t* accepted, const uint32_t* counts, uint32_t* error, cudaStream_t st) {
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    const size_t smem = TSP_KV_MAX_DRAFT * (q8 ? 2 * (cache.head_dim + cache.head_dim / 16) : 4 * cache.head_dim);
    static thread_local SmemAttrCache attr;
    TSP_CUDA(ensure_dynamic_smem(cache_keep_kernel, attr, smem));
    TSP_CUDA(launch_pdl(cache_keep_kernel, dim3(batch.sequences, cache.kv_heads), dim3(256), smem, st, cache, batch, accepted, counts, error));
    return TSP_OK;
}

}  // namespace tsp
