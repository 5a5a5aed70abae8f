// corope_cache_append: keys rotated, keys and values quantised into the blocks of the 8-bit cache.
//
// One thread block per (cache block with new tokens, K / V head).  A block's scale is known only once all its new rows have been seen, so
// they are read twice, the second time from L1 / L2: first for the largest element, then for the codes.
#include "cache.cuh"

namespace corope {
namespace {

constexpr int kThreads = 128;

// x1' = x1 c - x2 s, x2' = x2 c + x1 s, each operation rounded by itself: the codes are those of that formula in fp32
__device__ __forceinline__ void rotate4(float4& a, float4& b, const float4& c, const float4& s) {
    const float4 x = a, y = b;
    a = make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                    __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
    b = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                    __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }
__device__ __forceinline__ float amax4(const float4& a) { return fmaxf(fmaxf(finite_abs(a.x), finite_abs(a.y)), fmaxf(finite_abs(a.z), finite_abs(a.w))); }
template <int CODE>
__device__ __forceinline__ uint32_t codes4(const float4& a, float scale) {
    return to_code<CODE>(a.x, scale) | to_code<CODE>(a.y, scale) << 8 | to_code<CODE>(a.z, scale) << 16 | to_code<CODE>(a.w, scale) << 24;
}

// largest value of the thread block, in every thread
__device__ __forceinline__ float block_max(float x, float* words) {
#pragma unroll
    for (int m = 16; m; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
    if (threadIdx.x % 32 == 0) words[threadIdx.x / 32] = x;
    __syncthreads();
    x = words[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) x = fmaxf(x, words[i]);
    return x;
}

template <int CODE>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const CacheAppendParams p, int touched, bool vec_k, bool vec_v, bool vec_t) {
    __shared__ float words_k[kThreads / 32], words_v[kThreads / 32];
    const unsigned item = blockIdx.x / (unsigned)touched;
    const int j = (int)(blockIdx.x - item * (unsigned)touched), b = (int)(item / (unsigned)p.c.Hkv), h = (int)(item - (unsigned)b * (unsigned)p.c.Hkv);
    const int bs = 1 << p.c.bs_log2, D = p.D, half = D / 2;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), n = cache_new(p.s, p.T, b, bad);
    const int first = len - n;                                        // slot of token 0; negative: the tokens before slot 0 are left out
    const int block = (max(first, 0) >> p.c.bs_log2) + j, base = block << p.c.bs_log2;
    const int lo = max(first, base), hi = min(len, base + bs);        // the block's new slots
    const bool work = n > 0 && lo < hi;
    const int page = work ? cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, base, bad) : -1;
    const int per_row = half / 4, groups = kThreads / per_row;        // threads per row, rows per step
    const int d = (threadIdx.x % per_row) * 4, g = threadIdx.x / per_row;
    if (bad && threadIdx.x == 0) report_bad_index(p.status, p.mirror);
    if (page < 0) return;

    auto load_k = [&](int slot, float4& x1, float4& x2) {
        const int t = slot - first;
        const int64_t at = (int64_t)b * p.sk.b + (int64_t)h * p.sk.h + (int64_t)t * p.sk.n + d;
        x1 = load4(p.k, at, p.dtype, vec_k);
        x2 = load4(p.k, at + half, p.dtype, vec_k);
        if (p.s.cos == nullptr) return;
        const int64_t row = (int64_t)cache_position(p.s, b, t, slot, bad) * p.s.rope_stride + d;
        rotate4(x1, x2, load4(p.s.cos, row, COROPE_DTYPE_F32, vec_t), load4(p.s.sin, row, COROPE_DTYPE_F32, vec_t));
    };
    auto load_v = [&](int slot, float4& x1, float4& x2) {
        const int64_t at = (int64_t)b * p.sv.b + (int64_t)h * p.sv.h + (int64_t)(slot - first) * p.sv.n + d;
        x1 = load4(p.v, at, p.dtype, vec_v);
        x2 = load4(p.v, at + half, p.dtype, vec_v);
    };

    float mk = 0.f, mv = 0.f;
    for (int slot = lo + g; slot < hi; slot += groups) {
        float4 x1, x2;
        load_k(slot, x1, x2);
        mk = fmaxf(mk, fmaxf(amax4(x1), amax4(x2)));
        load_v(slot, x1, x2);
        mv = fmaxf(mv, fmaxf(amax4(x1), amax4(x2)));
    }
    if (bad) report_bad_index(p.status, p.mirror);
    mk = block_max(mk, words_k);
    mv = block_max(mv, words_v);

    const int64_t at = (int64_t)page * p.c.Hkv + h;
    const int held = lo - base;                                       // older tokens of the block
    const float old_k = held ? p.c.k_scale[at] : 0.f, old_v = held ? p.c.v_scale[at] : 0.f;
    const float new_k = max_nan(old_k, __fmul_rn(mk, kPerCode<CODE>)), new_v = max_nan(old_v, __fmul_rn(mv, kPerCode<CODE>));
    uint8_t* kb = p.c.k + (int64_t)page * p.c.sk.b + (int64_t)h * p.c.sk.h;
    uint8_t* vb = p.c.v + (int64_t)page * p.c.sv.b + (int64_t)h * p.c.sv.h;
    for (int r = g; r < held; r += groups) {
        if (new_k != old_k) {
            uint32_t *w1 = reinterpret_cast<uint32_t*>(kb + (int64_t)r * p.c.sk.n + d), *w2 = reinterpret_cast<uint32_t*>(kb + (int64_t)r * p.c.sk.n + d + half);
            *w1 = rescale4<CODE>(*w1, old_k, new_k);
            *w2 = rescale4<CODE>(*w2, old_k, new_k);
        }
        if (new_v != old_v) {
            uint32_t *w1 = reinterpret_cast<uint32_t*>(vb + (int64_t)r * p.c.sv.n + d), *w2 = reinterpret_cast<uint32_t*>(vb + (int64_t)r * p.c.sv.n + d + half);
            *w1 = rescale4<CODE>(*w1, old_v, new_v);
            *w2 = rescale4<CODE>(*w2, old_v, new_v);
        }
    }
    for (int slot = lo + g; slot < hi; slot += groups) {
        const int r = slot - base;
        float4 x1, x2;
        load_k(slot, x1, x2);
        *reinterpret_cast<uint32_t*>(kb + (int64_t)r * p.c.sk.n + d) = codes4<CODE>(x1, new_k);
        *reinterpret_cast<uint32_t*>(kb + (int64_t)r * p.c.sk.n + d + half) = codes4<CODE>(x2, new_k);
        load_v(slot, x1, x2);
        *reinterpret_cast<uint32_t*>(vb + (int64_t)r * p.c.sv.n + d) = codes4<CODE>(x1, new_v);
        *reinterpret_cast<uint32_t*>(vb + (int64_t)r * p.c.sv.n + d + half) = codes4<CODE>(x2, new_v);
        if (p.c.weight != nullptr && d == 0) p.c.weight[(at << p.c.bs_log2) + r] = 0.f;
    }
    __syncthreads();   // every thread has read the old scales
    if (threadIdx.x == 0) p.c.k_scale[at] = new_k, p.c.v_scale[at] = new_v;
}

}  // namespace

int launch_cache_append(const CacheAppendParams& p, cudaStream_t s) {
    const int bs = 1 << p.c.bs_log2, touched = (p.T + bs - 2) / bs + 1;
    const uint64_t blocks = (uint64_t)p.s.B * p.c.Hkv * touched;
    if (blocks >= (1ull << 31)) return COROPE_ERR_TOO_LARGE;
    const bool vec_k = rows_in_fours(p.k, p.sk, p.dtype), vec_v = rows_in_fours(p.v, p.sv, p.dtype);
    const bool vec_t = (uintptr_t)p.s.cos % 16 == 0 && (uintptr_t)p.s.sin % 16 == 0 && p.s.rope_stride % 4 == 0;
    count_launch();
    if (p.code == COROPE_CODE_E4M3) cache_append_kernel<COROPE_CODE_E4M3><<<(unsigned)blocks, kThreads, 0, s>>>(p, touched, vec_k, vec_v, vec_t);
    else cache_append_kernel<COROPE_CODE_INT8><<<(unsigned)blocks, kThreads, 0, s>>>(p, touched, vec_k, vec_v, vec_t);
    return (int)cudaGetLastError();
}

}  // namespace corope
