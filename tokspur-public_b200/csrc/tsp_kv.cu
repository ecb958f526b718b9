// Query / key head norm and rotation, and the paged key / value cache that the rows go into: written (quantised), read back, compacted.
#include "tsp_kv.cuh"

namespace tsp {

constexpr uint32_t kHeadThreads = 256;

template <bool F16> __device__ __forceinline__ float2 load2(const uint8_t* p, uint32_t i) {
    if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(p + i * 2));
    else return *reinterpret_cast<const float2*>(p + i * 4);
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
template <bool F16, uint32_t N> __device__ __forceinline__ void load_run(const uint8_t* p, uint32_t i, float (&v)[N]) {   // N = 2, 4, 8 values
#pragma unroll
    for (uint32_t k = 0; k < N; k += N < 4 ? 2 : 4) {
        if constexpr (N < 4) { const float2 x = load2<F16>(p, i); v[0] = x.x; v[1] = x.y; }
        else { float x[4]; load4<F16>(p, i + k, x); for (uint32_t c = 0; c < 4; ++c) v[k + c] = x[c]; }
    }
}
template <bool F16> __device__ __forceinline__ void store4(uint8_t* p, uint32_t i, const float (&v)[4]) {
    if constexpr (F16) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(p + i * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else *reinterpret_cast<float4*>(p + i * 4) = make_float4(v[0], v[1], v[2], v[3]);
}
template <bool F16> __device__ __forceinline__ bool fits(float v) { return F16 ? fabsf(v) < 65520.f : finite_f32(v); }   // 65520 rounds to infinity in binary16

// N values y over d rounded half to even, of the exact quotients, within +-127. The product with an approximate reciprocal rounds to a neighbour of the
// quotient at worst; the remainder y - r d is exact (r and d have 18 bits between them, and |y - r d| <= d over a grid of 2^-24 d at least), and
// tells where that matters: near the middle between two codes (and where d is subnormal, so that codes pass 127), all are put right.
template <typename T, uint32_t N> __device__ __forceinline__ void codes_of(const T (&y)[N], float d, float inv, float (&code)[N]) {
    float far = 0.f;
    T e[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        code[i] = __fadd_rn(__fadd_rn(static_cast<float>(y[i]) * inv, 12582912.f), -12582912.f);   // to the nearest whole number
        e[i] = fma(static_cast<T>(-code[i]), static_cast<T>(d), y[i]);
        far = fmaxf(far, fabsf(static_cast<float>(e[i])));
    }
    if (far > 0.49999f * d || d < 0x1p-14f) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const float r0 = fmaxf(fminf(code[i], 128.f), -128.f);
            const T e2 = 2 * fma(static_cast<T>(-r0), static_cast<T>(d), y[i]), w = d;
            const int r = static_cast<int>(r0), odd = r & 1;
            code[i] = static_cast<float>(max(-127, min(127, r + (e2 > w || (odd && e2 == w)) - (e2 < -w || (odd && e2 == -w)))));
        }
    }
}
__device__ __forceinline__ float reciprocal(float d) {   // for codes_of(); d is a binary16 number above 0
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}

// One head of K (a warp, lane l holds dims l NV .. l NV + NV - 1) into its slot. Returns false where it wrote zeros for it.
template <uint32_t D>
__device__ __forceinline__ bool put_keys(uint8_t* half, uint32_t t, bool q8, uint32_t lane, double (&y)[D / 32]) {
    constexpr uint32_t NV = D / 32;
    const uint32_t x0 = lane * NV;
    bool ok = true;
    if (q8) {
        double top = 0;
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) { ok &= finite_f32(static_cast<float>(y[i])); top = fmax(top, fabs(y[i])); }
#pragma unroll
        for (uint32_t o = 1; o < 32 / NV; o *= 2) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        const __half d16 = __float2half_rn(static_cast<float>(top * (1.0 / 127.0)));
        ok &= !__hisinf(d16);
        ok = __all_sync(0xffffffffu, ok);
        const float d32 = ok ? __half2float(d16) : 0.f;
        float whole[NV];
        uint8_t code[NV];
        if (d32 > 0.f) codes_of<double, NV>(y, d32, reciprocal(d32), whole);
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) code[i] = static_cast<uint8_t>(d32 > 0.f ? static_cast<int>(whole[i]) + 128 : 128);
        uint8_t* p = half + kv_k_byte(x0, t, true);
        if constexpr (NV == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(code[0] | code[1] << 8);
        else {
#pragma unroll
            for (uint32_t i = 0; i < NV; i += 4)
                *reinterpret_cast<uint32_t*>(p + i) = code[i] | code[i + 1] << 8 | code[i + 2] << 16 | static_cast<uint32_t>(code[i + 3]) << 24;
        }
        if (x0 % 32 == 0) *reinterpret_cast<__half*>(half + kv_scale_byte(x0, t, D)) = ok ? d16 : __ushort_as_half(0);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) ok &= fits<true>(static_cast<float>(y[i]));
        ok = __all_sync(0xffffffffu, ok);
#pragma unroll
        for (uint32_t i = 0; i < NV; i += 2)
            *reinterpret_cast<__half2*>(half + kv_k_byte(x0 + i, t, false)) = ok ? __floats2half2_rn(static_cast<float>(y[i]), static_cast<float>(y[i + 1])) : __half2half2(__ushort_as_half(0));
    }
    return ok;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 slots of a head's values, a warp: lane (g, t) takes dims 8 i + 2 t, + 1 of slots g and g + 8, in the order of an MMA fragment, and a transposing
// move of 8 x 8 matrices puts four slots beside each other as the cache holds them: whole 512-byte rows go out. `rows`: slots of the group that are
// written (bit i: slot i), b0 .. b1: blocks of 32 dims that are, `at(slot)`: a slot's values. (A warp per row and head, byte by byte: 4024 rows of three prompts with 32 + 8 + 8 heads of 128
// dims, normed, rotated, written and read back, 100 us, and 76 so; 49 with all later changes.)
template <uint32_t D, bool IN16, typename At>
__device__ __forceinline__ bool put_values(uint8_t* half, uint32_t rows, bool q8, uint32_t lane, uint32_t b0, uint32_t b1, At&& at) {
    const uint32_t g = lane / 4, t = lane % 4;
    bool fine = true;
    const bool on[2] = {(rows >> g & 1) != 0, (rows >> (g + 8) & 1) != 0};
    const uint8_t* src[2] = {on[0] ? at(g) : nullptr, on[1] ? at(g + 8) : nullptr};
    // a head whose values are not finite is zeros as a whole: look at all of it first (the second read comes from the L1)
    bool ok[2] = {true, true};
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n) {
        if (on[n]) {
#pragma unroll
            for (uint32_t b = 0; b < D / 32; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float2 v = load2<IN16>(src[n], 32 * b + 8 * i + 2 * t);
                    // a block's scale is finite in binary16 when its largest value over 127 rounds below infinity
                    ok[n] &= q8 ? fabsf(v.x) < 127.f * 65520.f && fabsf(v.y) < 127.f * 65520.f : fits<true>(v.x) && fits<true>(v.y);
                }
        }
        uint32_t v = ok[n];
        v &= __shfl_xor_sync(0xffffffffu, v, 1);
        v &= __shfl_xor_sync(0xffffffffu, v, 2);
        ok[n] = v != 0;
        fine &= ok[n];
    }
    // rolled: a step of a few rows waits for its instructions (unrolled, 24 rows took 13 us, half of it for those)
#pragma unroll 1
    for (uint32_t b = b0; b < b1; ++b) {
        float v[2][8];
        uint32_t out[4][2];   // [i][slots 2t, 2t + 1 | 8 more]: binary16 values, or codes
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) {
            float top = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float2 x = on[n] && ok[n] ? load2<IN16>(src[n], 32 * b + 8 * i + 2 * t) : make_float2(0.f, 0.f);
                v[n][2 * i] = x.x; v[n][2 * i + 1] = x.y;
                top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            if (q8) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const __half d16 = __float2half_rn(top / 127.f);
                const float d = __half2float(d16);
                float whole[8];
                if (d > 0.f) codes_of<float, 8>(v[n], d, reciprocal(d), whole);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) v[n][i] = d > 0.f ? whole[i] : 0.f;
                if (on[n] && t == 0) *reinterpret_cast<__half*>(half + kv_scale_byte(32 * b, g + 8 * n, D)) = d16;
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) out[i][n] = transposed(half2_bits(v[n][2 * i], v[n][2 * i + 1]));
        }
        const bool whole = rows == 0xffffu;
        if (q8) {
            uint32_t word[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {   // code + 128 as the low byte of 1152 + code
                const __half2 bias = __half2half2(__ushort_as_half(0x6480));
                const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&out[i][0]), bias), y = __hadd2(*reinterpret_cast<const __half2*>(&out[i][1]), bias);
                word[i] = __byte_perm(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y), 0x6420);
            }
            uint8_t* dst = half + b * 512 + lane * 16;
            if (whole) *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
            else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (rows >> (2 * t + (e & 1) + 8 * (e >> 1)) & 1)
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) dst[i * 4 + e] = static_cast<uint8_t>(word[i] >> (8 * e));
            }
        } else {
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m) {
                uint8_t* dst = half + (b * 2 + m) * 512 + lane * 16;
                if (whole) *reinterpret_cast<uint4*>(dst) = make_uint4(out[2 * m][0], out[2 * m][1], out[2 * m + 1][0], out[2 * m + 1][1]);
                else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e)
                        if (rows >> (2 * t + (e & 1) + 8 * (e >> 1)) & 1)
#pragma unroll
                            for (uint32_t i = 0; i < 2; ++i) reinterpret_cast<uint16_t*>(dst)[i * 4 + e] = static_cast<uint16_t>(out[2 * m + i][e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
    return fine;
}

// Groups of 16 slots that a step touches, without a scan: sequence s gets the places from d_row_offsets[s] / 16 + 2 s on. T rows touch (T + 30) / 16 groups at
// most, and the next sequence's places start T / 16 + 2 later at least. False: a place without slots.
__host__ __device__ constexpr uint32_t kv_group_places(uint32_t rows, uint32_t sequences) { return rows / 16 + 2 * sequences; }
__device__ __forceinline__ bool kv_group_of_place(const tsp_kv_batch& b, uint32_t place, uint32_t lane, uint32_t& seq, uint64_t& slot0, uint32_t& row0, uint32_t& mask) {
    auto before = [&](uint32_t s) { return b.d_row_offsets[s] / 16 + 2 * s <= place; };
    const uint32_t step = (b.sequences + 31) / 32;
    const uint32_t a = __popc(__ballot_sync(0xffffffffu, (lane + 1) * step < b.sequences && before(min((lane + 1) * step, b.sequences)))) * step;
    seq = a + __popc(__ballot_sync(0xffffffffu, lane + 1 < step && a + lane + 1 < b.sequences && before(min(a + lane + 1, b.sequences))));
    const uint32_t first = b.d_row_offsets[seq], end = b.d_row_offsets[seq + 1];
    if (end < first || end > b.rows) return false;
    const uint64_t length = b.d_lengths[seq], total = length + (end - first), start = length / 16 * 16 + 16ull * (place - (first / 16 + 2 * seq));
    if (start >= total) return false;
    slot0 = start;
    mask = total - start >= 16 ? 0xffffu : (1u << static_cast<uint32_t>(total - start)) - 1;
    if (start < length) mask &= 0xffffu << static_cast<uint32_t>(length - start);
    row0 = static_cast<uint32_t>(first + start - length);   // row of the group's slot 0, modulo 2^32: that slot may lie in front of the step's first
    return mask != 0;
}

struct HeadRows {
    const uint8_t *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    uint8_t *q_out, *k_out;
    uint64_t q_out_stride, k_out_stride;
    const uint32_t* positions;
    uint32_t q_heads, kv_heads;   // kv_heads: of k_out (no cache)
};

template <bool F16> struct Raw4;   // four values as they lie in memory
template <> struct Raw4<true> {
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void to(float (&v)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
};
template <> struct Raw4<false> {
    float4 w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void to(float (&v)[4]) const { v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w; }
};
// Blocks of three kinds. Rows that go out as rows: a block takes RB rows and as many heads as its threads hold at eight dims each; the rows' values are under
// way while the threads compute the rows' angles, one each. Keys that go into the cache: a block per four slots, a warp per head. Values that do: a
// warp per group of 16 slots and head. Measured, 32 + 8 heads of 128 dims: 8 FP32 rows 2.1 us, the pitch of launches; 4096 binary16 rows 18 us (FP32 rows 29 among other calls), 84 MB at 4.6 TB/s, from
// the L2 in part, bound by instructions (71 % of the issue slots). Into a Q8_0 cache: 38 rows of six drafts 6.6 us, a chain of latencies; 4024 rows of
// prompts 39.5 us, bound by the 64-bit arithmetic of the keys and by instructions (67 % of the issue slots), and without norm and rotation 17.8.
// Squares of FP32 heads may leave FP32: whether the mean of a head's, with eps, says what it should
__device__ __forceinline__ bool mean_in_range(float mean) { return __float_as_uint(mean) - 0x12800000u < 0x7f800000u - 0x12800000u; }   // [2^-90, infinity)
// The norm of a head where it does not: the head and sqrt(eps) times a power of two that puts the larger of them near one. By whole warps.
template <uint32_t LANES>
__device__ __forceinline__ void scaled_norm(float eps, float (&u)[4], float (&v)[4]) {
    float top = sqrtf(eps), ss = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(u[i]), fabsf(v[i])));
#pragma unroll
    for (uint32_t o = LANES / 2; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) { u[i] *= down; v[i] *= down; ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss)); }
#pragma unroll
    for (uint32_t o = LANES / 2; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / (8 * LANES)) + eps * down * down);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) { u[i] *= inv; v[i] *= inv; }
}
template <uint32_t D, bool IN16, bool OUT16, uint32_t RB>
__device__ __forceinline__ void turn_rows(const tsp_qk_norm_rope_args& a, const HeadRows& r, uint32_t pass, uint32_t row0, uint32_t end, uint32_t* error) {
    __shared__ __align__(16) float cs[RB][D / 2], sn[RB][D / 2];
    constexpr uint32_t LANES = D / 8, IE = IN16 ? 2 : 4, OE = OUT16 ? 2 : 4;   // lanes of a head
    const uint32_t tid = threadIdx.x, lane = tid % 32, half = a.rotary_dim / 2, heads = r.q_heads + r.kv_heads, l = tid % LANES;
    const uint32_t h0 = pass * (blockDim.x / LANES) + tid / LANES, h = min(h0, heads - 1);   // a lane behind the last head takes that one again: whole warps shuffle
    // four pairs a lane: (u, v) at dims xu.., xv.., or interleaved in eight dims from xu on; the dims behind the rotated ones pair up as halves
    const uint32_t p0 = 4 * l;
    const bool turned = p0 < half, pairs = turned && a.style == TSP_ROPE_PAIRS, is_k = h >= r.q_heads;
    const uint32_t xu = turned ? (pairs ? 2 * p0 : p0) : half + p0, xv = turned ? (pairs ? xu + 4 : p0 + half) : xu + (D - a.rotary_dim) / 2;
    const uint32_t hh = is_k ? h - r.q_heads : h;
    const uint64_t in_stride = is_k ? r.k_stride : r.q_stride, out_stride = is_k ? r.k_out_stride : r.q_out_stride;
    const uint8_t* in = (is_k ? r.k : r.q) + row0 * in_stride + (hh * D + xu) * IE;
    uint8_t* out = (is_k ? r.k_out : r.q_out) + row0 * out_stride + (hh * D + xu) * OE;
    const uint32_t iv = (xv - xu) * IE, ov = (xv - xu) * OE;
    Raw4<IN16> ru[RB], rv[RB];
#pragma unroll
    for (uint32_t j = 0; j < RB; ++j)
        if (row0 + j < end) { ru[j].load(in + j * in_stride); rv[j].load(in + j * in_stride + iv); }
    const float* w = is_k ? a.d_k_norm : a.d_q_norm;
    Raw4<false> wu, wv;
    wu.w = wv.w = make_float4(1.f, 1.f, 1.f, 1.f);
    if (w) { wu.load(reinterpret_cast<const uint8_t*>(w + xu)); wv.load(reinterpret_cast<const uint8_t*>(w + xv)); }
    if (half) {
        for (uint32_t i = tid; i < RB * half; i += blockDim.x) {
            const uint32_t j = RB == 1 ? 0 : i / half, p = RB == 1 ? i : i - j * half;
            if (row0 + j >= end) break;
            const double turns = static_cast<double>(r.positions[row0 + j]) * static_cast<double>(a.d_inv_freq[p]) * 0.15915494309189535;
            float s, c;
            sincospif(static_cast<float>(2 * (turns - rint(turns))), &s, &c);   // half turns, reduced in 64 bits
            cs[j][p] = c * a.magnitude; sn[j][p] = s * a.magnitude;
        }
        __syncthreads();
    }
    bool bad = false;
    const bool normed = __any_sync(0xffffffffu, w != nullptr);   // a warp may hold heads of both sides, one without a norm, and all of it shuffles
    const uint32_t group = LANES == 32 ? 0xffffffffu : ((1u << (LANES % 32)) - 1) << (lane / LANES * LANES);
    float fu[4], fv[4];
    wu.to(fu); wv.to(fv);
    auto turn = [&](uint32_t j, float (&u)[4], float (&v)[4]) {
        if (!turned) return;
        const float4 c4 = *reinterpret_cast<const float4*>(cs[j] + p0), n4 = *reinterpret_cast<const float4*>(sn[j] + p0);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, n[4] = {n4.x, n4.y, n4.z, n4.w};
        if (pairs) {
            float t[4] = {u[0], u[2], v[0], v[2]}, s[4] = {u[1], u[3], v[1], v[3]};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) { const float x = t[i]; t[i] = x * c[i] - s[i] * n[i]; s[i] = s[i] * c[i] + x * n[i]; }
            u[0] = t[0]; u[1] = s[0]; u[2] = t[1]; u[3] = s[1]; v[0] = t[2]; v[1] = s[2]; v[2] = t[3]; v[3] = s[3];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) { const float x = u[i]; u[i] = x * c[i] - v[i] * n[i]; v[i] = v[i] * c[i] + x * n[i]; }
        }
    };
    auto put = [&](uint32_t j, float (&u)[4], float (&v)[4], bool mine) {
        // magnitudes as integers: NaN lies above infinity
        uint32_t top = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) top = max(top, max(__float_as_uint(u[i]) & 0x7fffffffu, __float_as_uint(v[i]) & 0x7fffffffu));
        const bool ok = (__ballot_sync(0xffffffffu, top < (OUT16 ? 0x477ff000u : 0x7f800000u)) & group) == group;   // 65520 rounds to infinity in binary16
        mine &= h0 < heads;
        if (!ok) {
            bad |= mine;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) u[i] = v[i] = 0.f;
        }
        if (mine) {
            store4<OUT16>(out + j * out_stride, 0, u);
            store4<OUT16>(out + j * out_stride + ov, 0, v);
        }
    };
    uint32_t again = 0;
#pragma unroll
    for (uint32_t j = 0; j < RB; ++j) {
        if (row0 + j >= end) break;
        float u[4], v[4];
        ru[j].to(u); rv[j].to(v);
        bool odd = false;
        if (normed) {
            float ss = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
#pragma unroll
            for (uint32_t o = LANES / 2; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float mean = ss * (1.f / D) + a.eps;
            const float inv = w ? rsqrtf(mean) : 1.f;   // a side without a norm: times one
            if constexpr (!IN16) odd = w && !mean_in_range(mean);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) { u[i] = u[i] * inv * fu[i]; v[i] = v[i] * inv * fv[i]; }
        }
        turn(j, u, v);
        put(j, u, v, !odd);
        again |= static_cast<uint32_t>(odd) << j;
    }
    // Heads whose squares leave FP32, which those of binary16 rows cannot: nothing of them has been written. (A branch beside the sums, or in front of the stores,
    // keeps the rows from overlapping: 4096 FP32 rows of 40 heads 29 us, and 33 so.)
    if constexpr (!IN16)
        if (__any_sync(0xffffffffu, again != 0))
#pragma unroll 1
            for (uint32_t j = 0; j < RB && row0 + j < end; ++j) {
                float u[4], v[4];
                uint32_t row = row0 + j;
                asm volatile("" : "+r"(row));   // the address anew: kept from the loads above it would cost the loop two registers
                const uint8_t* from = (is_k ? r.k : r.q) + row * (is_k ? r.k_stride : r.q_stride) + (hh * D + xu) * IE;
                load4<IN16>(from, 0, u); load4<IN16>(from + (xv - xu) * IE, 0, v);
                scaled_norm<LANES>(a.eps, u, v);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) { u[i] *= fu[i]; v[i] *= fv[i]; }
                turn(j, u, v);
                put(j, u, v, again >> j & 1);
            }
    if (bad) raise_error(error, TSP_ERR_NONFINITE);
}

template <uint32_t D, bool IN16, bool OUT16, uint32_t RB>
__global__ void __launch_bounds__(512)
turn_rows_kernel(const tsp_qk_norm_rope_args a, const HeadRows r, uint32_t passes, uint32_t rows, uint32_t* error) {
    pdl_launch_dependents();
    pdl_wait();
    turn_rows<D, IN16, OUT16, RB>(a, r, blockIdx.x % passes, blockIdx.x / passes * RB, rows, error);
}

// Grid: value blocks (a warp per group, head and `parts`-th of its dims), key blocks, then `passes` blocks for every RB query rows. A key block: RB slots of a group (a row), a warp per head.
template <uint32_t D, bool IN16, bool OUT16, uint32_t RB>
__global__ void __launch_bounds__(kHeadThreads, D < 256 ? 4 : 1)   // 64 registers (left alone, 76 for FP32 rows of 128 dims: 4024 rows into the cache and back 70 us, and 65)
append_rows_kernel(const tsp_qk_norm_rope_args a, const HeadRows r, const tsp_kv_cache cache, const tsp_kv_batch batch, uint32_t values, uint32_t parts, uint32_t keys,
                   uint32_t passes, uint32_t* error) {
    __shared__ double cs[RB][D / 2], sn[RB][D / 2], exchange[kHeadThreads / 32][D];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32, places = kv_group_places(batch.rows, batch.sequences);
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    if (blockIdx.x == 0) kv_check_offsets(batch, error);
    if (blockIdx.x >= values + keys) {
        const uint32_t block = blockIdx.x - values - keys;
        turn_rows<D, IN16, OUT16, RB>(a, r, block % passes, block / passes * RB, min(batch.rows, batch.d_row_offsets[batch.sequences]), error);
        return;
    }
    uint32_t seq, row0, mask;
    uint64_t slot0;
    if (blockIdx.x < values) {
        const uint32_t task = blockIdx.x * (kHeadThreads / 32) + warp, part = task % parts, place = task / parts / cache.kv_heads, head = task / parts % cache.kv_heads;
        if (place >= places || !kv_group_of_place(batch, place, lane, seq, slot0, row0, mask)) return;
        uint8_t* group = kv_group(cache, seq, slot0, head, error);
        if (!group) return;
        const bool fine = put_values<D, IN16>(group + kv_half_bytes(D, q8), mask, q8, lane, part * (D / 32 / parts), (part + 1) * (D / 32 / parts),
                                              [&](uint32_t t) { return r.v + static_cast<uint64_t>(row0 + t) * r.v_stride + head * D * (IN16 ? 2u : 4u); });
        if (!fine) raise_error(error, TSP_ERR_NONFINITE);
        return;
    }
    constexpr uint32_t NV = D / 32, LOTS = kKvGroup / RB;
    const uint32_t half = a.rotary_dim / 2;
    if constexpr (RB == 1) {   // a block is a row
        uint32_t node;
        if (!kv_row(batch, blockIdx.x - values, lane, seq, node)) return;
        const uint64_t slot = static_cast<uint64_t>(batch.d_lengths[seq]) + node;
        const uint32_t t = static_cast<uint32_t>(slot % kKvGroup);
        slot0 = slot - t;
        row0 = blockIdx.x - values - t;   // modulo 2^32
        mask = 1u << t;
    } else {
        const uint32_t lot = (blockIdx.x - values) % LOTS;
        if (!kv_group_of_place(batch, (blockIdx.x - values) / LOTS, lane, seq, slot0, row0, mask)) return;
        mask &= ((1u << RB) - 1) << (lot * RB);
        if (!mask) return;
    }
    const uint32_t t0 = __ffs(mask) - 1, t1 = 32 - __clz(mask);   // the lot's slots of this step
    auto key_row = [&](uint32_t t, uint32_t h) { return r.k + static_cast<uint64_t>(row0 + t) * r.k_stride + h * D * (IN16 ? 2u : 4u); };
    float next[NV];
    if (warp < cache.kv_heads) load_run<IN16>(key_row(t0, warp), lane * NV, next);
    if (half) {
        for (uint32_t i = tid; i < (t1 - t0) * half; i += kHeadThreads) {
            const uint32_t j = i / half, p = i - j * half;
            const double turns = static_cast<double>(r.positions[row0 + t0 + j]) * static_cast<double>(a.d_inv_freq[p]) * 0.15915494309189535;
            double s, c;
            sincospi(2 * (turns - rint(turns)), &s, &c);
            cs[j][p] = c * a.magnitude; sn[j][p] = s * a.magnitude;
        }
        __syncthreads();
    }
    bool bad = false;
#pragma unroll 1
    for (uint32_t h = warp; h < cache.kv_heads; h += kHeadThreads / 32) {
        uint8_t* group = kv_group(cache, seq, slot0, h, error);
        if (!group) continue;
        if (h >= kHeadThreads / 32) load_run<IN16>(key_row(t0, h), lane * NV, next);
#pragma unroll 1
        for (uint32_t t = t0; t < t1; ++t) {
            double y[NV];
#pragma unroll
            for (uint32_t i = 0; i < NV; ++i) y[i] = next[i];
            if (t + 1 < t1) load_run<IN16>(key_row(t + 1, h), lane * NV, next);
            if (a.d_k_norm) {
                double ss = 0;
#pragma unroll
                for (uint32_t i = 0; i < NV; ++i) ss = fma(y[i], y[i], ss);
#pragma unroll
                for (uint32_t o = 16; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const double inv = rsqrt(ss * (1.0 / D) + static_cast<double>(a.eps));
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
                        const double s = sn[t - t0][p];
                        y[i] = y[i] * cs[t - t0][p] + mine[other] * (second ? s : -s);
                    }
                }
            }
            bad |= !put_keys<D>(group, t, q8, lane, y);
        }
    }
    if (bad) raise_error(error, TSP_ERR_NONFINITE);
}

template <uint32_t D, bool OUT16>
__device__ __forceinline__ void store8(uint8_t* row, uint32_t x, const float (&v)[8]) {   // eight dims from x on
    if constexpr (OUT16) *reinterpret_cast<uint4*>(row + x * 2) = make_uint4(half2_bits(v[0], v[1]), half2_bits(v[2], v[3]), half2_bits(v[4], v[5]), half2_bits(v[6], v[7]));
    else {
        reinterpret_cast<float4*>(row + x * 4)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(row + x * 4)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}
// two words of codes + 128 -> eight values
__device__ __forceinline__ void values_of(uint32_t a, uint32_t b, float d, float (&v)[8]) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = static_cast<float>(static_cast<int>((i < 4 ? a : b) >> (8 * (i % 4)) & 0xffu) - 128) * d;
}
// A warp per group of 16 slots and head: every load is a whole 512-byte row of the group, all of them under way at once; K leaves in the order it lies in,
// V through transposing moves as it came. (A warp per row and head, byte by byte: 57000 rows of 8 heads of 128 dims 238 us, and 64 now: 361 MB at 5.6 TB/s, the
// writes to memory bound it.)
template <uint32_t D, bool OUT16, bool Q8>
__global__ void __launch_bounds__(256)
cache_read_kernel(const tsp_kv_cache cache, const tsp_kv_batch batch, uint8_t* k, uint64_t k_stride, uint8_t* v, uint64_t v_stride, uint32_t* error) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr uint32_t ES = OUT16 ? 2 : 4, HALF = kv_half_bytes(D, Q8), ROWS = Q8 ? D / 32 : D / 16;   // 512-byte rows of K's (and V's) values
    const uint32_t lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    if (blockIdx.x == 0) kv_check_offsets(batch, error);
    const uint32_t task = blockIdx.x * 8 + threadIdx.x / 32, place = task / cache.kv_heads, head = task % cache.kv_heads;
    uint32_t seq, row0, mask;
    uint64_t slot0;
    if (place >= kv_group_places(batch.rows, batch.sequences) || !kv_group_of_place(batch, place, lane, seq, slot0, row0, mask)) return;
    const uint8_t* group = kv_group(cache, seq, slot0, head, error);
    if (!group) return;
    uint4 wk[ROWS], wv[ROWS];
    if (k)
#pragma unroll
        for (uint32_t i = 0; i < ROWS; ++i) wk[i] = reinterpret_cast<const uint4*>(group)[i * 32 + lane];
    if (v)
#pragma unroll
        for (uint32_t i = 0; i < ROWS; ++i) wv[i] = reinterpret_cast<const uint4*>(group + HALF)[i * 32 + lane];
    const bool on[2] = {(mask >> g & 1) != 0, (mask >> (g + 8) & 1) != 0};
    if (k) {
        uint8_t* base = k + head * D * ES;
        const __half* scales = reinterpret_cast<const __half*>(group + kKvGroup * D);
#pragma unroll
        for (uint32_t i = 0; i < ROWS; ++i) {   // Q8: 64 dims (i / 2), slots 8 (i % 2) + g, dims 8 t of both halves; F16: 32 dims, 8 dims
            const uint32_t slot = i % 2 * 8 + g;
            if (!on[i % 2]) continue;
            uint8_t* row = base + static_cast<uint64_t>(row0 + slot) * k_stride;
            if constexpr (Q8) {
                float x[8];
                values_of(wk[i].x, wk[i].y, __half2float(scales[(i / 2 * 2) * kKvGroup + slot]), x);
                store8<D, OUT16>(row, i / 2 * 64 + 8 * t, x);
                values_of(wk[i].z, wk[i].w, __half2float(scales[(i / 2 * 2 + 1) * kKvGroup + slot]), x);
                store8<D, OUT16>(row, i / 2 * 64 + 32 + 8 * t, x);
            } else {
                const uint32_t x = i / 2 * 32 + 8 * t;
                if constexpr (OUT16) *reinterpret_cast<uint4*>(row + x * 2) = wk[i];
                else {
                    float y[8];
                    const uint32_t w[4] = {wk[i].x, wk[i].y, wk[i].z, wk[i].w};
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j])); y[2 * j] = f.x; y[2 * j + 1] = f.y; }
                    store8<D, OUT16>(row, x, y);
                }
            }
        }
    }
    if (v) {
        uint8_t* base = v + head * D * ES;
        const __half* scales = reinterpret_cast<const __half*>(group + HALF + kKvGroup * D);
#pragma unroll
        for (uint32_t b = 0; b < D / 32; ++b) {
            uint32_t h[4][2];   // [i][slots 2t, 2t + 1 | 8 more] of dim 8 i + g; transposed: [i][slot g | g + 8] of dims 8 i + 2 t, + 1
            if constexpr (Q8) {
                const uint32_t w[4] = {wv[b].x, wv[b].y, wv[b].z, wv[b].w};
                const __half2 bias = __half2half2(__ushort_as_half(0x6480));   // 1152
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t x = __byte_perm(w[i], 0x64646464u, 0x4140), y = __byte_perm(w[i], 0x64646464u, 0x4342);
                    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), bias), q = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
                    h[i][0] = *reinterpret_cast<const uint32_t*>(&p); h[i][1] = *reinterpret_cast<const uint32_t*>(&q);
                }
            } else {
                const uint4 x = wv[2 * b % ROWS], y = wv[(2 * b + 1) % ROWS];
                h[0][0] = x.x; h[0][1] = x.y; h[1][0] = x.z; h[1][1] = x.w; h[2][0] = y.x; h[2][1] = y.y; h[3][0] = y.z; h[3][1] = y.w;
            }
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) {
                const uint32_t slot = g + 8 * n;
                const float d = Q8 ? __half2float(scales[b * kKvGroup + slot]) : 1.f;
                uint32_t o[4];
                float2 f[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    o[i] = transposed(h[i][n]);
                    f[i] = __half22float2(*reinterpret_cast<const __half2*>(&o[i]));
                    if constexpr (Q8) { f[i].x *= d; f[i].y *= d; o[i] = half2_bits(f[i].x, f[i].y); }
                }
                uint8_t* row = base + static_cast<uint64_t>(row0 + slot) * v_stride;
                if constexpr (OUT16) {   // neighbouring lanes swap, so that a lane has four dims in a row and four lanes a 32-byte sector
#pragma unroll
                    for (uint32_t i = 0; i < 4; i += 2) {
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, t & 1 ? o[i] : o[i + 1], 1);
                        if (on[n]) *reinterpret_cast<uint2*>(row + (32 * b + 8 * (i + (t & 1)) + t / 2 * 4) * 2) = t & 1 ? make_uint2(got, o[i + 1]) : make_uint2(o[i], got);
                    }
                } else if (on[n]) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) *reinterpret_cast<float2*>(row + (32 * b + 8 * i + 2 * t) * 4) = f[i];
                }
            }
        }
    }
}

// A block per (sequence, head): every source slot is in shared memory before the first destination is written. Pieces of a slot: 16 bytes of K, the four
// bytes (two halves) of V that a group of its 512-byte rows has of the slot, scales. Latencies one behind the other bound it (offsets, indices, table, source,
// destination): one tree of 24 tokens 5.0 us, 64 sequences of up to 16 7.6 (with a thread's pieces one after another
// 10.3).
template <uint32_t D, bool Q8>
__global__ void __launch_bounds__(256)
cache_keep_kernel(const tsp_kv_cache cache, const tsp_kv_batch batch, const uint32_t* accepted, const uint32_t* counts, uint32_t* error) {
    constexpr uint32_t KP = D * (Q8 ? 1 : 2) / 16, VP = Q8 ? D / 4 : D / 2, SP = Q8 ? D / 16 : 0, PER = KP + VP + SP, HALF = kv_half_bytes(D, Q8);
    extern __shared__ uint4 staged[];   // [slots][KP] K, then words [slots][VP] V, then halves [slots][SP]
    __shared__ uint8_t* place[2][TSP_KV_MAX_DRAFT];   // groups of sources and destinations
    __shared__ uint32_t from[TSP_KV_MAX_DRAFT];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t s = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    if (s == 0 && h == 0) kv_check_offsets(batch, error);
    const uint32_t first = batch.d_row_offsets[s], end = batch.d_row_offsets[s + 1], n = counts[s];
    const uint64_t length = batch.d_lengths[s];
    if (n == 0) return;
    bool bad = end < first || end > batch.rows || n > TSP_KV_MAX_DRAFT || n > end - first;
    uint32_t x = ~0u;
    if (!bad && tid < n) {
        x = accepted[first + tid];
        bad = x >= end - first || (tid && accepted[first + tid - 1] >= x);
        from[tid] = x;
        if (!bad) {
            place[0][tid] = kv_group(cache, s, length + x, h, error);
            place[1][tid] = kv_group(cache, s, length + tid, h, error);
            bad = !place[0][tid] || !place[1][tid];
        }
    }
    if (__syncthreads_or(bad)) { if (tid == 0) raise_error(error, TSP_ERR_INDEX); return; }
    // ascending indices are at their places up to the first that is not: those slots stay where they are (all of a chain's)
    const uint32_t stay = __syncthreads_count(x == tid);
    uint32_t* words = reinterpret_cast<uint32_t*>(staged + n * KP);
    uint16_t* halves = reinterpret_cast<uint16_t*>(words + n * VP);
#pragma unroll 1
    for (uint32_t pass = 0; pass < 2; ++pass) {
#pragma unroll 4
        for (uint32_t i = stay * PER + tid; i < n * PER; i += 256) {
            const uint32_t j = i / PER, c = i % PER, t = static_cast<uint32_t>((length + (pass ? j : from[j])) % kKvGroup), lane = t % 8 / 2, e = t % 2 + t / 8 * 2;
            uint8_t* group = place[pass][j];
            if (c < KP) {
                uint4 *p = reinterpret_cast<uint4*>(group + (c / 4 * kKvGroup + t) * 64 + c % 4 * 16), *m = staged + j * KP + c;
                if (pass) *p = *m; else *m = *p;
            } else if (c < KP + VP) {
                const uint32_t u = c - KP;
                uint8_t* p = group + HALF + (u * 4 + lane) * 16;
                uint32_t* m = words + j * VP + u;
                if constexpr (Q8) {
                    if (pass) { const uint32_t w = *m; p[e] = w; p[4 + e] = w >> 8; p[8 + e] = w >> 16; p[12 + e] = w >> 24; }
                    else *m = p[e] | p[4 + e] << 8 | p[8 + e] << 16 | static_cast<uint32_t>(p[12 + e]) << 24;
                } else {
                    uint16_t* q = reinterpret_cast<uint16_t*>(p);
                    if (pass) { const uint32_t w = *m; q[e] = w; q[4 + e] = w >> 16; }
                    else *m = q[e] | static_cast<uint32_t>(q[4 + e]) << 16;
                }
            } else {
                const uint32_t u = c - KP - VP, is_v = u >= D / 32;
                uint16_t *p = reinterpret_cast<uint16_t*>(group + (is_v ? HALF : 0) + kKvGroup * D) + (u - is_v * (D / 32)) * kKvGroup + t, *m = halves + j * SP + u;
                if (pass) *p = *m; else *m = *p;
            }
        }
        __syncthreads();
    }
}

static uint32_t value_blocks(const tsp_kv_cache& c, const tsp_kv_batch& b, uint32_t parts) {
    return (kv_group_places(b.rows, b.sequences) * c.kv_heads * parts + kHeadThreads / 32 - 1) / (kHeadThreads / 32);
}

template <uint32_t D, bool IN16, bool OUT16>
static int launch_head_rows_d(const tsp_qk_norm_rope_args& a, const HeadRows& r, const tsp_kv_cache* cache, const tsp_kv_batch* batch, uint32_t rows, uint32_t* error,
                              cudaStream_t st) {
    // Four rows a block, so that a thread computes an angle or two and has 64 bytes under way (4096 rows of 40 heads of 128 binary16 values: a row a block 24 us);
    // one while that is no more than two blocks per SM
    const uint32_t lanes = (r.q_heads + r.kv_heads) * (D / 8), threads = cache ? kHeadThreads : 0, sms = static_cast<uint32_t>(sm_count() > 0 ? sm_count() : 1);
    if (!cache) {   // as few idle threads as passes of at most 512 allow: 40 heads of 128 dims in two passes of 320 threads
        const uint32_t passes = (lanes + 511) / 512, width = ((lanes + passes - 1) / passes + 31) / 32 * 32;
        if (rows * passes <= 2 * sms) TSP_CUDA(launch_pdl(turn_rows_kernel<D, IN16, OUT16, 1>, dim3(passes * rows), dim3(width), 0, st, a, r, passes, rows, error));
        else TSP_CUDA(launch_pdl(turn_rows_kernel<D, IN16, OUT16, 4>, dim3(passes * ((rows + 3) / 4)), dim3(width), 0, st, a, r, passes, rows, error));
        return TSP_OK;
    }
    // Few groups: a warp for each 32 dims of a group and head, which looks at the whole head but writes a quarter (of 128 dims): a warp's chain of latencies is the
    // call's time. With the keys a row a block, 16 sequences of one token 6.7 us and 4.8 so, 772 rows of 64 (176 blocks without) 13.5 and 11.8; more blocks have
    // enough warps without: 256 sequences of one token (528) 12.5 and 16.9 so.
    const uint32_t parts = 4 * value_blocks(*cache, *batch, 1) <= 5 * sms ? D / 32 : 1, values = value_blocks(*cache, *batch, parts);
    const uint32_t passes = (lanes + threads - 1) / threads, at_least_one = passes ? passes : 1;
    if (rows * at_least_one <= 2 * sms) {
        TSP_CUDA(launch_pdl(append_rows_kernel<D, IN16, OUT16, 1>, dim3(values + rows + passes * rows), dim3(threads), 0, st, a, r, *cache, *batch, values, parts, rows, at_least_one, error));
    } else {
        const uint32_t keys = kv_group_places(batch->rows, batch->sequences) * (kKvGroup / 4);
        TSP_CUDA(launch_pdl(append_rows_kernel<D, IN16, OUT16, 4>, dim3(values + keys + passes * ((rows + 3) / 4)), dim3(threads), 0, st, a, r, *cache, *batch, values, parts, keys, at_least_one, error));
    }
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

template <uint32_t D>
static int launch_cache_read_d(const tsp_kv_cache& cache, const tsp_kv_batch& batch, uint8_t* k, uint64_t k_stride, uint8_t* v, uint64_t v_stride, bool out16, uint32_t* error,
                               cudaStream_t st) {
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    auto kernel = q8 ? (out16 ? cache_read_kernel<D, true, true> : cache_read_kernel<D, false, true>) : (out16 ? cache_read_kernel<D, true, false> : cache_read_kernel<D, false, false>);
    const uint32_t tasks = kv_group_places(batch.rows, batch.sequences) * cache.kv_heads;
    TSP_CUDA(launch_pdl(kernel, dim3((tasks + 7) / 8), dim3(256), 0, st, cache, batch, k, k_stride, v, v_stride, error));
    return TSP_OK;
}

int launch_cache_read(const tsp_kv_cache& cache, const tsp_kv_batch& batch, void* k, uint64_t k_stride, void* v, uint64_t v_stride, uint32_t dtype, uint32_t* error,
                      cudaStream_t st) {
    uint8_t *kb = static_cast<uint8_t*>(k), *vb = static_cast<uint8_t*>(v);
    return cache.head_dim == 64    ? launch_cache_read_d<64>(cache, batch, kb, k_stride, vb, v_stride, dtype, error, st)
           : cache.head_dim == 128 ? launch_cache_read_d<128>(cache, batch, kb, k_stride, vb, v_stride, dtype, error, st)
                                   : launch_cache_read_d<256>(cache, batch, kb, k_stride, vb, v_stride, dtype, error, st);
}

template <uint32_t D, bool Q8>
static int launch_cache_keep_d(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const uint32_t* accepted, const uint32_t* counts, uint32_t* error, cudaStream_t st) {
    constexpr size_t smem = TSP_KV_MAX_DRAFT * (Q8 ? 2 * (D + D / 16) : 4 * D);
    static thread_local SmemAttrCache attr;
    TSP_CUDA(ensure_dynamic_smem(cache_keep_kernel<D, Q8>, attr, smem));
    TSP_CUDA(launch_pdl(cache_keep_kernel<D, Q8>, dim3(batch.sequences, cache.kv_heads), dim3(256), smem, st, cache, batch, accepted, counts, error));
    return TSP_OK;
}

int launch_cache_keep(const tsp_kv_cache& cache, const tsp_kv_batch& batch, const uint32_t* accepted, const uint32_t* counts, uint32_t* error, cudaStream_t st) {
    const bool q8 = cache.type == TSP_TYPE_Q8_0;
    switch (cache.head_dim) {
        case 64: return q8 ? launch_cache_keep_d<64, true>(cache, batch, accepted, counts, error, st) : launch_cache_keep_d<64, false>(cache, batch, accepted, counts, error, st);
        case 128: return q8 ? launch_cache_keep_d<128, true>(cache, batch, accepted, counts, error, st) : launch_cache_keep_d<128, false>(cache, batch, accepted, counts, error, st);
        default: return q8 ? launch_cache_keep_d<256, true>(cache, batch, accepted, counts, error, st) : launch_cache_keep_d<256, false>(cache, batch, accepted, counts, error, st);
    }
}

}  // namespace tsp
