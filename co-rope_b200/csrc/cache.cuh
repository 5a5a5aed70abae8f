// The 8-bit paged key / value cache: what its kernels share.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace corope {

struct CacheView {
    uint8_t *k, *v;
    float *k_scale, *v_scale, *weight;
    Strides sk, sv;              // block (b), head (h), row (n); bytes, as codes have one
    int num_blocks, Hkv, bs_log2;
};
struct SeqView {
    const int* table;
    int64_t table_stride;
    int B, max_blocks;
    const int *lens, *new_lens, *positions;
    const float *cos, *sin;
    int64_t rope_stride;
    int table_rows;
};
struct CacheAppendParams {
    CacheView c;
    SeqView s;
    const void *k, *v;
    Strides sk, sv;
    int T, D, code, dtype;
    int *status, *mirror;
};
struct CacheAttnParams {
    CacheView c;
    SeqView s;
    const void* q;
    void* o;
    Strides sq, so;
    int Hq, G, T, D, code, dtype, causal, accumulate;
    int parts;                   // blocks (a cluster) per item, 0 = ranges of the batch's units
    int row_tiles;               // tiles of query rows per K / V head (row = t * G + head of the group)
    float scale;                 // sm_scale * log2(e)
    bool vec_o;                  // rows of o take stores of four elements
    bool rows_packed;            // rows of codes follow one another without gaps
    float* part;                 // partial results: two slots per block of the main kernel
    float* part_ml;              // their maxima and sums
    float* lse;                  // [B, Hkv, T * G] log2 of each row's sum (accumulate only)
    float* scores;               // [B, Hkv, capacity, score_rows] scores in units of log2, or null (accumulate only)
    int capacity, score_rows;    // slots of a block table; rows a K / V head, rounded up to even
    int *status, *mirror;
};
struct CacheEvictParams {
    CacheView c;
    SeqView s;
    const int* out_table;
    int64_t out_stride;
    int out_blocks, budget, recent, D, code;
    bool vec_weight;             // weights take loads of four
    int *new_lens, *kept;
    int *status, *mirror;
};

int launch_cache_append(const CacheAppendParams& p, cudaStream_t s);
size_t cache_attn_workspace_bytes(int B, int Hkv, int G, int T, int D, int max_blocks, int block_size, int dtype, int accumulate);
int launch_cache_attn(CacheAttnParams p, void* ws, cudaStream_t s);
int launch_cache_evict(const CacheEvictParams& p, cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ void report_bad_index(int* status, int* mirror) {
    if (status == nullptr) return;
    atomicOr(status, COROPE_DEV_BAD_INDEX);
    report_to_mirror(status, mirror);
}
// A sequence's length and its new tokens, brought into range.  A new token count above the length is one whose first tokens have no
// slot: not an error (an empty place in a padded batch).
__device__ __forceinline__ int cache_len(const SeqView& s, int bs_log2, int b, bool& bad) {
    const int len = s.lens[b], most = s.max_blocks << bs_log2;
    bad |= len < 0 || len > most;
    return min(max(len, 0), most);
}
__device__ __forceinline__ int cache_new(const SeqView& s, int T, int b, bool& bad) {
    if (s.new_lens == nullptr) return T;
    const int n = s.new_lens[b];
    bad |= n < 0 || n > T;
    return min(max(n, 0), T);
}
// the block that holds slot `slot` of sequence b, or -1
__device__ __forceinline__ int cache_page(const SeqView& s, int bs_log2, int num_blocks, int b, int slot, bool& bad) {
    const int page = s.table[(int64_t)b * s.table_stride + (slot >> bs_log2)];
    const bool ok = (unsigned)page < (unsigned)num_blocks;
    bad |= !ok;
    return ok ? page : -1;
}
// row of the cos / sin tables for token t of this call, whose slot is `slot`
__device__ __forceinline__ int cache_position(const SeqView& s, int b, int t, int slot, bool& bad) {
    const int64_t pos = s.positions == nullptr ? (int64_t)slot : (int64_t)s.positions[b] + t;
    bad |= pos < 0 || pos >= s.table_rows;
    return (int)min(max(pos, (int64_t)0), (int64_t)s.table_rows - 1);
}

// ---- codes.  Every step is an fp32 operation of its own (no contraction), so that codes do not depend on how a compiler joins them.
template <int CODE> constexpr float kPerCode = 1.f / (CODE == COROPE_CODE_E4M3 ? 448.f : 127.f);   // scale of a block per unit of its largest element

template <int CODE>
__device__ __forceinline__ uint32_t to_code(float x, float scale) {
    const float y = scale == 0.f ? 0.f : __fdiv_rn(x, scale);
    if constexpr (CODE == COROPE_CODE_E4M3) return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
    else return (uint32_t)(int)fminf(fmaxf(rintf(y != y ? 0.f : y), -127.f), 127.f) & 0xffu;
}
// Four codes of x / scale without a division.  x times a reciprocal is within 4 units of 2^-24 of the fp32 quotient, so it has the quotient's code
// unless a tie lies that near (one number in 10^4 for e4m3; for int8, whose band is 2^-12 of a step on either side, one in 2000, so one call in 500 and
// one warp in 16): then, and where the scale has no usable reciprocal, all four are divided.
// `near` = reciprocal(scale); |x| <= (1 + 2^-22) * scale * largest code, or `plain` is false.
__device__ __forceinline__ float reciprocal(float scale) { return scale > 1e-30f && scale < 1e30f ? __frcp_rn(scale) : __int_as_float(0x7fffffff); }
template <int CODE>
__device__ __noinline__ uint32_t divided4(float a, float b, float c, float d, float scale) {
    return to_code<CODE>(a, scale) | to_code<CODE>(b, scale) << 8 | to_code<CODE>(c, scale) << 16 | to_code<CODE>(d, scale) << 24;
}
template <int CODE>
__device__ __forceinline__ bool codes4_near(const float (&y)[4], uint32_t& w) {
    if constexpr (CODE == COROPE_CODE_E4M3) {   // the numbers 2^-20 below and above have the same code
        constexpr float kBelow = 1.f - 0x1p-20f, kAbove = 1.f + 0x1p-20f;
        uint16_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = i % 2 ? kAbove : kBelow;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r[i]) : "f"(y[i / 2 * 2 + 1] * f), "f"(y[i / 2 * 2] * f));
        }
        const uint32_t lo = (uint32_t)r[0] | (uint32_t)r[2] << 16, hi = (uint32_t)r[1] | (uint32_t)r[3] << 16;
        w = lo;
        return lo == hi;
    } else {   // rounded by the addition of 1.5 * 2^23, and not within 2^-12 of a tie (the error is 2^-24 * 4 * 127 = 2^-15 at most)
        float r[4], off = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[i] = y[i] + 12582912.f;
            off = fmaxf(off, fabsf(y[i] - (r[i] - 12582912.f)));
        }
        w = __byte_perm(__byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040), __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040), 0x5410);
        return off < 0.5f - 0x1p-12f;
    }
}
template <int CODE>
__device__ __forceinline__ uint32_t codes4(const float4& x, float scale, float near, bool plain) {
    uint32_t w;
    const float y[4] = {x.x * near, x.y * near, x.z * near, x.w * near};
    if (codes4_near<CODE>(y, w) && plain) return w;
    return divided4<CODE>(x.x, x.y, x.z, x.w, scale);
}
template <int CODE>
__device__ __forceinline__ void from_codes4(uint32_t w, float (&x)[4]) {
    if constexpr (CODE == COROPE_CODE_E4M3) {
        uint32_t a, b;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
        const float2 u = unpack_half2(a), v = unpack_half2(b);
        x[0] = u.x; x[1] = u.y; x[2] = v.x; x[3] = v.y;
    } else {   // the byte c + 128 as the last digits of 2^23 + 128 + c
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7540 + i)) - 8388736.f;
    }
}
// four codes of scale `old` written for a larger `scale`
template <int CODE>
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float old, float scale, float near) {
    const bool plain = near == near && old < scale;   // not NaN, either
    const float ratio = old * near;
    uint32_t w;
    float x[4];
    if constexpr (CODE == COROPE_CODE_INT8) {
        // c * ratio in units of 2^-24: u * r + (2^23 - 128 r) with u = c + 128 has the rounded product in its top byte.  r is off by 3 at most, the product
        // by 400, the fp32 quotient by as much: not within 1024 of a tie, it has the quotient's code.
        const uint32_t r = __float2uint_rn(ratio * 16777216.f), shift = 8388608u - 128u * r, u = codes ^ 0x80808080u;
        uint32_t t[4], least = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t[i] = __byte_perm(u, 0u, 0x4440 + i) * r + shift;
            least = min(least, t[i] * 256u + 1024u * 256u);
        }
        if (least >= 2048u * 256u && plain) return __byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x0073), 0x5410);
        from_codes4<CODE>(codes, x);
    } else {
        from_codes4<CODE>(codes, x);
        const float y[4] = {x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio};
        if (codes4_near<CODE>(y, w) && plain) return w;
    }
    return divided4<CODE>(__fmul_rn(x[0], old), __fmul_rn(x[1], old), __fmul_rn(x[2], old), __fmul_rn(x[3], old), scale);
}
// max(a, b), NaN if one of them is
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// elements i .. i + 3 of a row, of any of the three types; `vec`: aligned to four elements
__device__ __forceinline__ float load1(const void* base, int64_t i, int dtype) {
    if (dtype == COROPE_DTYPE_F32) return static_cast<const float*>(base)[i];
    if (dtype == COROPE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
    return __half2float(static_cast<const __half*>(base)[i]);
}
__device__ __forceinline__ float4 load4(const void* base, int64_t i, int dtype, bool vec) {
    if (!vec) return make_float4(load1(base, i, dtype), load1(base, i + 1, dtype), load1(base, i + 2, dtype), load1(base, i + 3, dtype));
    if (dtype == COROPE_DTYPE_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
    const float2 a = dtype == COROPE_DTYPE_BF16 ? unpack_bf162(u.x) : unpack_half2(u.x), b = dtype == COROPE_DTYPE_BF16 ? unpack_bf162(u.y) : unpack_half2(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store1(void* base, int64_t i, int dtype, float x) {
    if (dtype == COROPE_DTYPE_F32) static_cast<float*>(base)[i] = x;
    else if (dtype == COROPE_DTYPE_BF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
    else static_cast<__half*>(base)[i] = __float2half_rn(x);
}
__device__ __forceinline__ void store4(void* base, int64_t i, int dtype, bool vec, float4 x) {
    if (!vec) {
        store1(base, i, dtype, x.x); store1(base, i + 1, dtype, x.y); store1(base, i + 2, dtype, x.z); store1(base, i + 3, dtype, x.w);
    } else if (dtype == COROPE_DTYPE_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = x;
    } else if (dtype == COROPE_DTYPE_BF16) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(pack_bf162(x.x, x.y), pack_bf162(x.z, x.w));
    } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(pack_half2(x.x, x.y), pack_half2(x.z, x.w));
    }
}
#endif  // __CUDACC__

// rows whose groups of four elements start at multiples of their size
inline bool rows_in_fours(const void* ptr, const Strides& st, int dtype) {
    return (uintptr_t)ptr % (4 * dtype_bytes(dtype)) == 0 && st.b % 4 == 0 && st.h % 4 == 0 && st.n % 4 == 0;
}

}  // namespace corope
