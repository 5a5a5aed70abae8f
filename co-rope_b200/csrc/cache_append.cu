// corope_cache_append: keys rotated, keys and values quantised into the blocks of the 8-bit cache.
//
// One thread block per (cache block with new tokens, K / V head): a block's scale is known once all its new rows have been seen, so they wait in
// registers (up to four rows a thread, as fp32) for the block-wide maximum.  Keys first, then values.  Bound by the reads of k and v.
#include "cache.cuh"

namespace corope {
namespace {

constexpr int kSteps = 4;        // rows a thread holds

// x1' = x1 c - x2 s, x2' = x2 c + x1 s, each operation rounded by itself: the codes are those of that formula in fp32
__device__ __forceinline__ void rotate4(float4& a, float4& b, const float4& c, const float4& s) {
    const float4 x = a, y = b;
    a = make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                    __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
    b = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                    __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }
__device__ __forceinline__ float finite_amax4(const float4& a) { return fmaxf(fmaxf(finite_abs(a.x), finite_abs(a.y)), fmaxf(finite_abs(a.z), finite_abs(a.w))); }
// max(top, |a|), infinite or NaN if an element is
__device__ __forceinline__ float amax4(float top, const float4& a) { return fmax3_nan(fmax3_nan(top, fabsf(a.x), fabsf(a.y)), fabsf(a.z), fabsf(a.w)); }

// four elements as they are stored
template <bool WIDE> struct Raw;
template <> struct Raw<true> {
    float4 x;
    __device__ __forceinline__ void load(const void* base, int64_t i, int dtype, bool vec) { x = load4(base, i, dtype, vec); }
    __device__ __forceinline__ float4 get(int) const { return x; }
};
template <> struct Raw<false> {
    uint2 x;
    __device__ __forceinline__ void load(const void* base, int64_t i, int, bool vec) {
        const uint16_t* from = static_cast<const uint16_t*>(base) + i;
        if (vec) x = *reinterpret_cast<const uint2*>(from);
        else x = make_uint2((uint32_t)from[0] | (uint32_t)from[1] << 16, (uint32_t)from[2] | (uint32_t)from[3] << 16);
    }
    __device__ __forceinline__ float4 get(int dtype) const {
        const float2 a = dtype == COROPE_DTYPE_BF16 ? unpack_bf162(x.x) : unpack_half2(x.x), b = dtype == COROPE_DTYPE_BF16 ? unpack_bf162(x.y) : unpack_half2(x.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
};

// largest value of the thread block, in every thread; `words`: 32 floats, a different array for each use
__device__ __forceinline__ float block_max(float x, float* words) {
#pragma unroll
    for (int m = 16; m; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
    if (threadIdx.x % 32 == 0) words[threadIdx.x / 32] = x;
    __syncthreads();
    x = threadIdx.x % 32 < blockDim.x / 32 ? words[threadIdx.x % 32] : 0.f;
#pragma unroll
    for (int m = 16; m; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
    return x;
}

// WIDE: fp32 rows.  MOST: threads of the largest block launched.
template <int CODE, bool WIDE, int MOST>
__global__ void __launch_bounds__(MOST) cache_append_kernel(const CacheAppendParams p, int touched, int per_row_log2, bool vec_k, bool vec_v, bool vec_t) {
    __shared__ float words[2][32];
    const unsigned item = blockIdx.x / (unsigned)touched;
    const int j = (int)(blockIdx.x - item * (unsigned)touched), b = (int)(item / (unsigned)p.c.Hkv), h = (int)(item - (unsigned)b * (unsigned)p.c.Hkv);
    const int bs = 1 << p.c.bs_log2, half = p.D / 2;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), n = cache_new(p.s, p.T, b, bad);
    const int first = len - n;                                        // slot of token 0; negative: the tokens before slot 0 are left out
    const int block = (max(first, 0) >> p.c.bs_log2) + j, base = block << p.c.bs_log2;
    const int lo = max(first, base), hi = min(len, base + bs);        // the block's new slots
    const int page = n > 0 && lo < hi ? cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, base, bad) : -1;
    // 2^per_row_log2 threads share a row, each has four elements of its first half and their partners in the second
    const int d = ((int)threadIdx.x & ((1 << per_row_log2) - 1)) * 4, g = (int)threadIdx.x >> per_row_log2, groups = (int)blockDim.x >> per_row_log2;
    if (bad && threadIdx.x == 0) report_bad_index(p.status, p.mirror);
    if (page < 0) return;
    bad = false;

    // all of the thread's rows are on their way before the first is looked at
    Raw<WIDE> raw[2][kSteps][2];
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int slot = lo + g + i * groups;
            if (slot >= hi) continue;
            const Strides st = part ? p.sv : p.sk;
            const int64_t from = (int64_t)b * st.b + (int64_t)h * st.h + (int64_t)(slot - first) * st.n + d;
            raw[part][i][0].load(part ? p.v : p.k, from, p.dtype, part ? vec_v : vec_k);
            raw[part][i][1].load(part ? p.v : p.k, from + half, p.dtype, part ? vec_v : vec_k);
        }
    const int64_t at = (int64_t)page * p.c.Hkv + h;
    const int held = lo - base;                                       // older tokens of the block
#pragma unroll
    for (int part = 0; part < 2; ++part) {                            // keys, values
        const Strides sc = part ? p.c.sv : p.c.sk;
        uint8_t* to = (part ? p.c.v : p.c.k) + (int64_t)page * sc.b + (int64_t)h * sc.h + d;
        float* scale_at = (part ? p.c.v_scale : p.c.k_scale) + at;
        const float old = held ? *scale_at : 0.f;
        float4 x1[kSteps], x2[kSteps];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int slot = lo + g + i * groups;
            if (slot >= hi) continue;
            x1[i] = raw[part][i][0].get(p.dtype);
            x2[i] = raw[part][i][1].get(p.dtype);
            if (part == 0 && p.s.cos != nullptr) {
                const int64_t row = (int64_t)cache_position(p.s, b, slot - first, slot, bad) * p.s.rope_stride + d;
                rotate4(x1[i], x2[i], load4(p.s.cos, row, COROPE_DTYPE_F32, vec_t), load4(p.s.sin, row, COROPE_DTYPE_F32, vec_t));
            }
            top = amax4(amax4(top, x1[i]), x2[i]);
        }
        const bool finite = top <= 3.402823466e38f;
        if (!finite) {
            top = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (lo + g + i * groups < hi) top = fmaxf(top, fmaxf(finite_amax4(x1[i]), finite_amax4(x2[i])));
        }
        top = block_max(top, words[part]);                            // (every thread has read the old scale)
        const float scale = max_nan(old, __fmul_rn(top, kPerCode<CODE>)), near = reciprocal(scale);
        const bool plain = finite && near == near;
        if (threadIdx.x == 0) *scale_at = scale;
        if (held && scale != old)
            for (int r = g; r < held; r += groups) {
                uint32_t *w1 = reinterpret_cast<uint32_t*>(to + (int64_t)r * sc.n), *w2 = reinterpret_cast<uint32_t*>(to + (int64_t)r * sc.n + half);
                *w1 = rescale4<CODE>(*w1, old, scale, near);
                *w2 = rescale4<CODE>(*w2, old, scale, near);
            }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int slot = lo + g + i * groups;
            if (slot >= hi) continue;
            *reinterpret_cast<uint32_t*>(to + (int64_t)(slot - base) * sc.n) = codes4<CODE>(x1[i], scale, near, plain);
            *reinterpret_cast<uint32_t*>(to + (int64_t)(slot - base) * sc.n + half) = codes4<CODE>(x2[i], scale, near, plain);
            if (part && p.c.weight != nullptr && d == 0) p.c.weight[(at << p.c.bs_log2) + slot - base] = 0.f;
        }
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

template <int CODE, bool WIDE>
int launch_t(const CacheAppendParams& p, unsigned blocks, int threads, int touched, int per_row_log2, cudaStream_t s) {
    const bool vec_k = rows_in_fours(p.k, p.sk, p.dtype), vec_v = rows_in_fours(p.v, p.sv, p.dtype);
    const bool vec_t = (uintptr_t)p.s.cos % 16 == 0 && (uintptr_t)p.s.sin % 16 == 0 && p.s.rope_stride % 4 == 0;
    count_launch();
    if (threads <= 512) cache_append_kernel<CODE, WIDE, 512><<<blocks, threads, 0, s>>>(p, touched, per_row_log2, vec_k, vec_v, vec_t);
    else cache_append_kernel<CODE, WIDE, 1024><<<blocks, threads, 0, s>>>(p, touched, per_row_log2, vec_k, vec_v, vec_t);
    return (int)cudaGetLastError();
}

}  // namespace

int launch_cache_append(const CacheAppendParams& p, cudaStream_t s) {
    const int bs = 1 << p.c.bs_log2, touched = (p.T + bs - 2) / bs + 1;
    const uint64_t blocks = (uint64_t)p.s.B * p.c.Hkv * touched;
    if (blocks >= (1ull << 31)) return COROPE_ERR_TOO_LARGE;
    // a thread for every four elements of kSteps rows: 1024 for 256 rows of 16 threads, the most there are
    const int per_row_log2 = p.D == 128 ? 4 : p.D == 64 ? 3 : 2, rows = p.T < bs ? p.T : bs;
    int threads = 64;
    while (threads * kSteps < rows << per_row_log2) threads *= 2;
    const bool wide = p.dtype == COROPE_DTYPE_F32;
    if (p.code == COROPE_CODE_E4M3)
        return wide ? launch_t<COROPE_CODE_E4M3, true>(p, (unsigned)blocks, threads, touched, per_row_log2, s)
                    : launch_t<COROPE_CODE_E4M3, false>(p, (unsigned)blocks, threads, touched, per_row_log2, s);
    return wide ? launch_t<COROPE_CODE_INT8, true>(p, (unsigned)blocks, threads, touched, per_row_log2, s)
                : launch_t<COROPE_CODE_INT8, false>(p, (unsigned)blocks, threads, touched, per_row_log2, s);
}

}  // namespace corope
