// corope_cache_append: keys rotated, keys and values quantised into the blocks of the 8-bit cache.
//
// One thread block per (cache block with new tokens, K / V head): a block's scale is known once all its new rows have been seen, so they wait in
// registers (two rows a thread where that takes no more than 1024 threads, else four) for the block-wide maxima.  Bound by instruction issue (62 % of the slots at
// 4 prompts of up to 4096 tokens, 33 instructions a code), not by the reads of k and v (a third of the time).
#include "cache.cuh"

namespace corope {
namespace {


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

// Largest values (none negative: their bits are in the same order) of the thread block, in every thread; `words`: 64 words.
__device__ __forceinline__ void block_max(float& k, float& v, uint32_t* words) {
    const uint32_t a = __reduce_max_sync(0xffffffffu, __float_as_uint(k)), b = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    const int lane = threadIdx.x % 32;
    if (lane == 0) words[threadIdx.x / 32] = a, words[32 + threadIdx.x / 32] = b;
    __syncthreads();
    const bool there = lane < (int)blockDim.x / 32;
    k = __uint_as_float(__reduce_max_sync(0xffffffffu, there ? words[lane] : 0u));
    v = __uint_as_float(__reduce_max_sync(0xffffffffu, there ? words[32 + lane] : 0u));
}

// WIDE: fp32 rows.  kSteps: rows a thread holds.  MOST: threads of the largest block launched.
template <int CODE, bool WIDE, int kSteps, int MOST>
__global__ void __launch_bounds__(MOST, 1024 / MOST) cache_append_kernel(const CacheAppendParams p, int touched, int per_row_log2, bool vec_k, bool vec_v, bool vec_t) {
    __shared__ uint32_t words[64];
    const unsigned item = blockIdx.x / (unsigned)touched;
    const int j = (int)(blockIdx.x - item * (unsigned)touched), b = (int)(item / (unsigned)p.c.Hkv), h = (int)(item - (unsigned)b * (unsigned)p.c.Hkv);
    const int bs = 1 << p.c.bs_log2, half = p.D / 2;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), n = cache_new(p.s, p.T, b, bad);
    const int first = len - n;                                        // slot of token 0; negative: the tokens before slot 0 are left out
    const int block = (max(first, 0) >> p.c.bs_log2) + j, base = block << p.c.bs_log2;
    const int lo = max(first, base), hi = min(len, base + bs);        // the block's new slots
    // a length or a number of new tokens out of range does not tell where the tokens belong: none is stored
    const int page = !bad && n > 0 && lo < hi ? cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, base, bad) : -1;
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
    const float old_k = held ? p.c.k_scale[at] : 0.f, old_v = held ? p.c.v_scale[at] : 0.f;
    float4 x[2][kSteps][2];
    float top[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int slot = lo + g + i * groups;
        if (slot >= hi) continue;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            x[part][i][0] = raw[part][i][0].get(p.dtype);
            x[part][i][1] = raw[part][i][1].get(p.dtype);
        }
        if (p.s.cos != nullptr) {
            const int64_t row = (int64_t)cache_position(p.s, b, slot - first, slot, bad) * p.s.rope_stride + d;
            rotate4(x[0][i][0], x[0][i][1], load4(p.s.cos, row, COROPE_DTYPE_F32, vec_t), load4(p.s.sin, row, COROPE_DTYPE_F32, vec_t));
        }
#pragma unroll
        for (int part = 0; part < 2; ++part) top[part] = amax4(amax4(top[part], x[part][i][0]), x[part][i][1]);
    }
    bool finite[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        finite[part] = top[part] <= 3.402823466e38f;
        if (finite[part]) continue;
        top[part] = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (lo + g + i * groups < hi) top[part] = fmaxf(top[part], fmaxf(finite_amax4(x[part][i][0]), finite_amax4(x[part][i][1])));
    }
    block_max(top[0], top[1], words);                                 // (every thread has read the old scales)
#pragma unroll
    for (int part = 0; part < 2; ++part) {                            // keys, values
        const Strides sc = part ? p.c.sv : p.c.sk;
        uint8_t* to = (part ? p.c.v : p.c.k) + (int64_t)page * sc.b + (int64_t)h * sc.h + d;
        const float old = part ? old_v : old_k, scale = max_nan(old, __fmul_rn(top[part], kPerCode<CODE>)), near = reciprocal(scale);
        const bool plain = finite[part] && near == near;
        if (threadIdx.x == 0) (part ? p.c.v_scale : p.c.k_scale)[at] = scale;
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
            *reinterpret_cast<uint32_t*>(to + (int64_t)(slot - base) * sc.n) = codes4<CODE>(x[part][i][0], scale, near, plain);
            *reinterpret_cast<uint32_t*>(to + (int64_t)(slot - base) * sc.n + half) = codes4<CODE>(x[part][i][1], scale, near, plain);
            if (part && p.c.weight != nullptr && d == 0) p.c.weight[(at << p.c.bs_log2) + slot - base] = 0.f;
        }
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

template <int CODE, bool WIDE>
int launch_t(const CacheAppendParams& p, unsigned blocks, int rows, int touched, int per_row_log2, cudaStream_t s) {
    const bool vec_k = rows_in_fours(p.k, p.sk, p.dtype), vec_v = rows_in_fours(p.v, p.sv, p.dtype);
    const bool vec_t = (uintptr_t)p.s.cos % 16 == 0 && (uintptr_t)p.s.sin % 16 == 0 && p.s.rope_stride % 4 == 0;
    count_launch();
    const int wanted = rows << per_row_log2;   // threads, with a row each
    auto threads = [&](int steps) {
        int t = 64;
        while (t * steps < wanted) t *= 2;
        return t;
    };
    if (threads(2) <= 512) cache_append_kernel<CODE, WIDE, 2, 512><<<blocks, threads(2), 0, s>>>(p, touched, per_row_log2, vec_k, vec_v, vec_t);
    else if (threads(2) <= 1024) cache_append_kernel<CODE, WIDE, 2, 1024><<<blocks, threads(2), 0, s>>>(p, touched, per_row_log2, vec_k, vec_v, vec_t);
    else cache_append_kernel<CODE, WIDE, 4, 1024><<<blocks, threads(4), 0, s>>>(p, touched, per_row_log2, vec_k, vec_v, vec_t);   // 256 rows of 16 threads, the most there are
    return (int)cudaGetLastError();
}

}  // namespace

int launch_cache_append(const CacheAppendParams& p, cudaStream_t s) {
    const int bs = 1 << p.c.bs_log2, touched = (p.T + bs - 2) / bs + 1;
    const uint64_t blocks = (uint64_t)p.s.B * p.c.Hkv * touched;
    if (blocks >= (1ull << 31)) return COROPE_ERR_TOO_LARGE;
    const int per_row_log2 = p.D == 128 ? 4 : p.D == 64 ? 3 : 2, rows = p.T < bs ? p.T : bs;
    const bool wide = p.dtype == COROPE_DTYPE_F32;
    if (p.code == COROPE_CODE_E4M3)
        return wide ? launch_t<COROPE_CODE_E4M3, true>(p, (unsigned)blocks, rows, touched, per_row_log2, s)
                    : launch_t<COROPE_CODE_E4M3, false>(p, (unsigned)blocks, rows, touched, per_row_log2, s);
    return wide ? launch_t<COROPE_CODE_INT8, true>(p, (unsigned)blocks, rows, touched, per_row_log2, s)
                : launch_t<COROPE_CODE_INT8, false>(p, (unsigned)blocks, rows, touched, per_row_log2, s);
}

}  // namespace corope
