// corope_cache_evict: the slots of largest accumulated weight, and their move to new blocks.
//
// Two kernels.  The first finds, per (sequence, K / V head), the weight of the last slot kept by counting digits of the weights' ordered bit
// patterns from the top, and writes the kept slots in ascending order.  The second fills one new block per thread block: its scale is the
// largest of its sources' scales.
#include "cache.cuh"

namespace corope {
namespace {

constexpr int kSelectThreads = 1024, kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kMoveThreads = 256;

// unsigned numbers in the order of the weights: -0 as 0, NaN above everything
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    if (w != w) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) cache_select_kernel(const CacheEvictParams p) {
    __shared__ unsigned counts[kDigits];
    __shared__ unsigned chosen, above;
    __shared__ unsigned warp_sums[2][32];
    const int b = blockIdx.x / p.c.Hkv, h = blockIdx.x - b * p.c.Hkv, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), keep = min(len, p.budget);
    if (h == 0 && threadIdx.x == 0) p.new_lens[b] = keep;
    int* kept = p.kept + (int64_t)blockIdx.x * p.budget;
    for (int i = keep + threadIdx.x; i < p.budget; i += kSelectThreads) kept[i] = -1;
    if (len <= p.budget) {
        for (int i = threadIdx.x; i < len; i += kSelectThreads) kept[i] = i;
        if (bad && threadIdx.x == 0) report_bad_index(p.status, p.mirror);
        return;
    }
    const int open = len - min(p.recent, len);             // slots that compete
    const unsigned need = (unsigned)(keep - (len - open));  // that many of them stay
    auto key = [&](int slot) -> uint32_t {
        const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad);
        return page < 0 ? 0u : ordered(p.c.weight[(((int64_t)page * p.c.Hkv + h) << p.c.bs_log2) + (slot & ((1 << p.c.bs_log2) - 1))]);
    };
    uint32_t prefix = 0, mask = 0;   // the digits of the last kept key that are known
    unsigned rest = need;            // slots to keep among those that share them
    for (int shift = 32 - kDigitBits; shift >= 0 && need > 0; shift -= kDigitBits) {
        for (int i = threadIdx.x; i < kDigits; i += kSelectThreads) counts[i] = 0;
        __syncthreads();
        for (int slot = threadIdx.x; slot < open; slot += kSelectThreads) {
            const uint32_t k = key(slot);
            if ((k & mask) == prefix) atomicAdd(&counts[(k >> shift) & (kDigits - 1)], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned sum = 0;
            int digit = kDigits - 1;
            while (digit > 0 && sum + counts[digit] < rest) sum += counts[digit--];
            chosen = (unsigned)digit;
            above = sum;
        }
        __syncthreads();
        prefix |= chosen << shift;
        mask |= (uint32_t)(kDigits - 1) << shift;
        rest -= above;
    }
    // keys above `prefix` stay, and of the equal ones the first `rest`
    unsigned written = 0, equal_seen = 0;
    for (int base = 0; base < len; base += kSelectThreads) {
        const int slot = base + threadIdx.x;
        const uint32_t k = slot < open && need > 0 ? key(slot) : 0u;
        const bool late = slot >= open && slot < len, equal = slot < open && need > 0 && k == prefix, over = slot < open && need > 0 && k > prefix;
        const unsigned eq = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) warp_sums[0][warp] = __popc(eq);
        __syncthreads();
        unsigned before = equal_seen, all = 0;
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? warp_sums[0][w] : 0u;
            all += warp_sums[0][w];
        }
        equal_seen += all;
        const bool stays = late || over || (equal && before + __popc(eq & ((1u << lane) - 1u)) < rest);
        const unsigned st = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) warp_sums[1][warp] = __popc(st);
        __syncthreads();
        before = written;
        all = 0;
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? warp_sums[1][w] : 0u;
            all += warp_sums[1][w];
        }
        written += all;
        if (stays) kept[before + __popc(st & ((1u << lane) - 1u))] = slot;
        // warp_sums[0] is written again only after the second barrier, [1] after the next first one
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

template <int CODE>
__global__ void __launch_bounds__(kMoveThreads) cache_move_kernel(const CacheEvictParams p, int out_used) {
    __shared__ int64_t from[256];       // (page * Hkv + h) of each slot's source block, or -1
    __shared__ int rows[256];
    __shared__ float old_k[256], old_v[256];
    __shared__ float tops[2][kMoveThreads / 32];
    const unsigned bh = blockIdx.x / (unsigned)out_used;
    const int j = (int)(blockIdx.x - bh * (unsigned)out_used), b = (int)(bh / (unsigned)p.c.Hkv), h = (int)(bh - (unsigned)b * (unsigned)p.c.Hkv);
    const int bs = 1 << p.c.bs_log2, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    bool bad = false;
    const int count = min(min(cache_len(p.s, p.c.bs_log2, b, bad), p.budget) - (j << p.c.bs_log2), bs);
    pdl_wait();
    if (count <= 0) return;
    const int out = p.out_table[(int64_t)b * p.out_stride + j];
    if ((unsigned)out >= (unsigned)p.c.num_blocks) {
        if (threadIdx.x == 0) report_bad_index(p.status, p.mirror);
        return;
    }
    const int64_t to = (int64_t)out * p.c.Hkv + h;
    float top_k = 0.f, top_v = 0.f;
    for (int i = threadIdx.x; i < count; i += kMoveThreads) {
        const int slot = p.kept[(int64_t)bh * p.budget + (j << p.c.bs_log2) + i];
        const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad), r = slot & (bs - 1);
        const int64_t at = (int64_t)page * p.c.Hkv + h;
        from[i] = page < 0 ? -1 : page;
        rows[i] = r;
        old_k[i] = page < 0 ? 0.f : p.c.k_scale[at];
        old_v[i] = page < 0 ? 0.f : p.c.v_scale[at];
        top_k = max_nan(top_k, old_k[i]);
        top_v = max_nan(top_v, old_v[i]);
        p.c.weight[(to << p.c.bs_log2) + i] = page < 0 ? 0.f : p.c.weight[(at << p.c.bs_log2) + r];
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        top_k = max_nan(top_k, __shfl_xor_sync(0xffffffffu, top_k, m));
        top_v = max_nan(top_v, __shfl_xor_sync(0xffffffffu, top_v, m));
    }
    if (lane == 0) tops[0][warp] = top_k, tops[1][warp] = top_v;
    __syncthreads();
    for (int w = 0; w < kMoveThreads / 32; ++w) top_k = max_nan(top_k, tops[0][w]), top_v = max_nan(top_v, tops[1][w]);
    if (threadIdx.x == 0) p.c.k_scale[to] = top_k, p.c.v_scale[to] = top_v;

    const int per_row = p.D / 16;   // 16-byte runs
    for (int x = threadIdx.x; x < count * per_row; x += kMoveThreads) {
        const int i = x / per_row, col = (x - i * per_row) * 16;
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (from[i] >= 0) {
            k = *reinterpret_cast<const uint4*>(p.c.k + from[i] * p.c.sk.b + (int64_t)h * p.c.sk.h + (int64_t)rows[i] * p.c.sk.n + col);
            v = *reinterpret_cast<const uint4*>(p.c.v + from[i] * p.c.sv.b + (int64_t)h * p.c.sv.h + (int64_t)rows[i] * p.c.sv.n + col);
            if (old_k[i] != top_k)
                k = make_uint4(rescale4<CODE>(k.x, old_k[i], top_k), rescale4<CODE>(k.y, old_k[i], top_k), rescale4<CODE>(k.z, old_k[i], top_k),
                               rescale4<CODE>(k.w, old_k[i], top_k));
            if (old_v[i] != top_v)
                v = make_uint4(rescale4<CODE>(v.x, old_v[i], top_v), rescale4<CODE>(v.y, old_v[i], top_v), rescale4<CODE>(v.z, old_v[i], top_v),
                               rescale4<CODE>(v.w, old_v[i], top_v));
        }
        *reinterpret_cast<uint4*>(p.c.k + (int64_t)out * p.c.sk.b + (int64_t)h * p.c.sk.h + (int64_t)i * p.c.sk.n + col) = k;
        *reinterpret_cast<uint4*>(p.c.v + (int64_t)out * p.c.sv.b + (int64_t)h * p.c.sv.h + (int64_t)i * p.c.sv.n + col) = v;
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

}  // namespace

int launch_cache_evict(const CacheEvictParams& p, cudaStream_t s) {
    const int bs = 1 << p.c.bs_log2, out_used = (p.budget + bs - 1) / bs;
    const uint64_t items = (uint64_t)p.s.B * p.c.Hkv;
    if (items * out_used >= (1ull << 31)) return COROPE_ERR_TOO_LARGE;
    count_launch(2);
    cache_select_kernel<<<(unsigned)items, kSelectThreads, 0, s>>>(p);
    if (int e = (int)cudaGetLastError()) return e;
    const unsigned blocks = (unsigned)(items * out_used);
    if (p.code == COROPE_CODE_E4M3) return launch_dependent(cache_move_kernel<COROPE_CODE_E4M3>, blocks, kMoveThreads, 0, s, p, out_used);
    return launch_dependent(cache_move_kernel<COROPE_CODE_INT8>, blocks, kMoveThreads, 0, s, p, out_used);
}

}  // namespace corope
