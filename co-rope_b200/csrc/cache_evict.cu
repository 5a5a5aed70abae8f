// corope_cache_evict: the slots of largest accumulated weight, and their move to new blocks.
//
// Two kernels.  The first finds, per (sequence, K / V head), the weight of the last slot kept by counting digits of the weights' ordered bit
// patterns from the top (11, 11 and 10 bits), and writes the kept slots in ascending order.  A cluster of blocks shares an item where there are fewer
// items than SMs: each block holds its slots' patterns in shared memory, so weights are read once, and adds up the counts of all.  Bound by latency:
// three rounds of counting, each a few microseconds, behind one pass over the weights.
// The second fills one new block per thread block: its scale is the largest of its sources' scales.  Bound by the reads and writes of the codes.
#include <cooperative_groups.h>

#include "cache.cuh"

namespace corope {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelectThreads = 1024, kBins = 2048;
constexpr int kHeldSlots = 48 * 1024;      // patterns a block holds; a longer share is read again from the cache in every round
constexpr int kMoveThreads = 256;

// unsigned numbers in the order of the weights: -0 as 0, NaN above everything
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    if (w != w) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the threads before this one, and over all; `words`: 32 words, not in use by an earlier call that a thread may still be in.
__device__ __forceinline__ unsigned sum_before(unsigned x, unsigned* words, unsigned& all) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    unsigned up = x;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const unsigned y = __shfl_up_sync(0xffffffffu, up, m);
        if (lane >= m) up += y;
    }
    if (lane == 31) words[warp] = up;
    __syncthreads();
    unsigned w = words[lane];
    all = w;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const unsigned y = __shfl_up_sync(0xffffffffu, w, m);
        if (lane >= m) w += y;
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    return up - x + (warp ? __shfl_sync(0xffffffffu, w, max(warp - 1, 0)) : 0u);
}

// `parts` blocks (a cluster) per item; `held`: slots a block has shared memory for
__global__ void __launch_bounds__(kSelectThreads, 1) cache_select_kernel(const CacheEvictParams p, int parts, int held) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ unsigned counts[3][kBins];
    __shared__ unsigned words[5][32];   // of the three rounds, and of the two sums behind them
    __shared__ unsigned chosen[3], above[3], found[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = (int)(blockIdx.x % (unsigned)parts), item = (int)(blockIdx.x / (unsigned)parts), b = item / p.c.Hkv, h = item - b * p.c.Hkv;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), keep = min(len, p.budget), bs_mask = (1 << p.c.bs_log2) - 1;
    const bool all_stay = len <= p.budget;
    const int open = all_stay ? 0 : len - p.recent;                     // slots that compete for `need` places
    const unsigned need = (unsigned)(keep - (len - open));
    int* kept = p.kept + (int64_t)item * p.budget;
    if (part == 0) {
        if (h == 0 && threadIdx.x == 0) p.new_lens[b] = keep;
        for (int i = keep + threadIdx.x; i < p.budget; i += kSelectThreads) kept[i] = -1;
        for (int i = open + threadIdx.x; i < len; i += kSelectThreads) kept[keep - len + i] = i;   // the last ones
    }
    if (open == 0 || need == 0) {                                       // the same in all blocks of a cluster
        if (bad && threadIdx.x == 0) report_bad_index(p.status, p.mirror);
        return;
    }
    // this block's slots, and the consecutive ones of each thread among them (an odd number: neighbours' words lie in different banks)
    const int share = ((open + parts - 1) / parts + 3) & ~3, lo = min(part * share, open), n = min(share, open - lo);
    const int each = ((share + kSelectThreads - 1) / kSelectThreads) | 1;
    const bool in_smem = n <= held;
    auto weight_key = [&](int slot) -> uint32_t {
        const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad);
        return page < 0 ? 0u : ordered(p.c.weight[(((int64_t)page * p.c.Hkv + h) << p.c.bs_log2) + (slot & bs_mask)]);
    };
    auto key = [&](int i) -> uint32_t { return in_smem ? keys[i] : weight_key(lo + i); };
    for (int i = threadIdx.x; i < 3 * kBins; i += kSelectThreads) (&counts[0][0])[i] = 0;
    __syncthreads();
    if (in_smem) {   // patterns to shared memory, the first digit counted on the way; four slots at a time: they lie in one block
#pragma unroll 2
        for (int i = 4 * threadIdx.x; i < n; i += 4 * kSelectThreads) {
            const int slot = lo + i, page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad);
            const float* from = p.c.weight + (((int64_t)max(page, 0) * p.c.Hkv + h) << p.c.bs_log2) + (slot & bs_mask);
            float w[4];
            if (p.vec_weight) {
                const float4 x = *reinterpret_cast<const float4*>(from);   // (what lies behind the share is not used)
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
#pragma unroll
                for (int y = 0; y < 4; ++y) w[y] = from[y];
            }
            uint32_t k[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                k[y] = page < 0 ? 0u : ordered(w[y]);
                if (i + y < n) atomicAdd(&counts[0][k[y] >> 21], 1u);
            }
            *reinterpret_cast<uint4*>(keys + i) = make_uint4(k[0], k[1], k[2], k[3]);
        }
    }

    uint32_t prefix = 0, mask = 0;   // the digits of the last kept key that are known
    unsigned rest = need;            // slots to keep among those that share them
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
        const uint32_t digit_mask = round == 2 ? 1023u : 2047u;
        if (!in_smem) {
            for (int i = threadIdx.x; i < n; i += kSelectThreads) {
                const uint32_t k = key(i);
                if ((k & mask) == prefix) atomicAdd(&counts[round][(k >> shift) & digit_mask], 1u);
            }
        } else if (round > 0) {
            for (int i = 4 * threadIdx.x; i < n; i += 4 * kSelectThreads) {
                const uint4 x = *reinterpret_cast<const uint4*>(keys + i);
                const uint32_t k[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    if ((k[y] & mask) == prefix && i + y < n) atomicAdd(&counts[round][(k[y] >> shift) & digit_mask], 1u);
            }
        }
        if (parts > 1) cluster.sync();
        else __syncthreads();
        // bins from the top: thread t has bins 2047 - 2 t and one below
        unsigned c0 = 0, c1 = 0;
        const int top = kBins - 1 - 2 * (int)threadIdx.x;
        for (int q = 0; q < parts; ++q) {
            const unsigned* far = parts > 1 ? cluster.map_shared_rank(&counts[round][0], q) : &counts[round][0];
            c0 += far[top];
            c1 += far[top - 1];
        }
        unsigned all;
        const unsigned before = sum_before(c0 + c1, words[round], all);
        if (before < rest && rest <= before + c0) chosen[round] = (unsigned)top, above[round] = before;
        else if (before + c0 < rest && rest <= before + c0 + c1) chosen[round] = (unsigned)top - 1u, above[round] = before + c0;
        __syncthreads();
        prefix |= chosen[round] << shift;
        mask |= digit_mask << shift;
        rest -= above[round];
    }
    // keys above `prefix` stay, and of the equal ones the first `rest`
    const int from = min((int)threadIdx.x * each, n), to = min(from + each, n);
    unsigned equal = 0, over = 0;
    for (int i = from; i < to; ++i) {
        const uint32_t k = key(i);
        equal += k == prefix;
        over += k > prefix;
    }
    unsigned all_equal, all_over;
    unsigned equal_before = sum_before(equal, words[3], all_equal);
    unsigned over_before = sum_before(over, words[4], all_over);
    if (parts > 1) {
        if (threadIdx.x == 0) found[0] = all_equal, found[1] = all_over;
        cluster.sync();
        for (int q = 0; q < part; ++q) {
            const unsigned* far = cluster.map_shared_rank(&found[0], q);
            equal_before += far[0];
            over_before += far[1];
        }
    }
    unsigned at = over_before + min(equal_before, rest);
    for (int i = from; i < to; ++i) {
        const uint32_t k = key(i);
        if (k > prefix || (k == prefix && equal_before++ < rest)) kept[at++] = lo + i;
    }
    if (bad) report_bad_index(p.status, p.mirror);
    if (parts > 1) cluster.sync();   // no block ends while another reads its counts
}

template <int CODE>
__global__ void __launch_bounds__(kMoveThreads, 8) cache_move_kernel(const CacheEvictParams p, int out_used) {
    __shared__ int64_t from[256];       // each slot's source block, or -1
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
    const float near_k = reciprocal(top_k), near_v = reciprocal(top_v);
    uint8_t* k_to = p.c.k + (int64_t)out * p.c.sk.b + (int64_t)h * p.c.sk.h;
    uint8_t* v_to = p.c.v + (int64_t)out * p.c.sv.b + (int64_t)h * p.c.sv.h;
    auto rescale = [](uint4& w, float old, float scale, float near) {
        if (old != scale)
            w = make_uint4(rescale4<CODE>(w.x, old, scale, near), rescale4<CODE>(w.y, old, scale, near), rescale4<CODE>(w.z, old, scale, near),
                           rescale4<CODE>(w.w, old, scale, near));
    };
    constexpr int kRuns = 1;        // a thread's runs in flight: the blocks beside hide more (8 an SM; 2 runs and 4 blocks took 80 us in place of 66)
    for (int base = threadIdx.x; base < count * per_row; base += kRuns * kMoveThreads) {
        uint4 k[kRuns], v[kRuns];
#pragma unroll
        for (int u = 0; u < kRuns; ++u) {
            const int x = base + u * kMoveThreads, i = x / per_row, col = (x - i * per_row) * 16;
            k[u] = v[u] = make_uint4(0u, 0u, 0u, 0u);
            if (x < count * per_row && from[i] >= 0) {
                k[u] = *reinterpret_cast<const uint4*>(p.c.k + from[i] * p.c.sk.b + (int64_t)h * p.c.sk.h + (int64_t)rows[i] * p.c.sk.n + col);
                v[u] = *reinterpret_cast<const uint4*>(p.c.v + from[i] * p.c.sv.b + (int64_t)h * p.c.sv.h + (int64_t)rows[i] * p.c.sv.n + col);
            }
        }
#pragma unroll
        for (int u = 0; u < kRuns; ++u) {
            const int x = base + u * kMoveThreads, i = x / per_row, col = (x - i * per_row) * 16;
            if (x >= count * per_row) break;
            rescale(k[u], old_k[i], top_k, near_k);
            rescale(v[u], old_v[i], top_v, near_v);
            *reinterpret_cast<uint4*>(k_to + (int64_t)i * p.c.sk.n + col) = k[u];
            *reinterpret_cast<uint4*>(v_to + (int64_t)i * p.c.sv.n + col) = v[u];
        }
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

}  // namespace

int launch_cache_evict(const CacheEvictParams& p, cudaStream_t s) {
    const int bs = 1 << p.c.bs_log2, out_used = (p.budget + bs - 1) / bs;
    const uint64_t items = (uint64_t)p.s.B * p.c.Hkv;
    if (items * out_used >= (1ull << 31)) return COROPE_ERR_TOO_LARGE;
    // Blocks per item: as many as fill the SMs, up to a portable cluster, each with 4096 slots or more of the longest sequence there can be.
    const int64_t most = (int64_t)p.s.max_blocks << p.c.bs_log2;
    int parts = 1;
    while (parts < 8 && items * parts * 2 <= (uint64_t)sm_count() && most / (parts * 2) >= 4096) parts *= 2;
    const int64_t share = ((most + parts - 1) / parts + 3) / 4 * 4;
    const int held = (int)(share < kHeldSlots ? share : kHeldSlots);
    static std::atomic<uint64_t> done{0};
    if (int e = allow_smem(cache_select_kernel, kHeldSlots * 4, done)) return e;
    count_launch(2);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(items * parts));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = (size_t)held * 4;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CacheEvictParams q = p;
    q.vec_weight = (uintptr_t)p.c.weight % 16 == 0;
    if (int e = (int)cudaLaunchKernelEx(&cfg, cache_select_kernel, q, parts, held)) return e;
    const unsigned blocks = (unsigned)(items * out_used);
    if (p.code == COROPE_CODE_E4M3) return launch_dependent(cache_move_kernel<COROPE_CODE_E4M3>, blocks, kMoveThreads, 0, s, p, out_used);
    return launch_dependent(cache_move_kernel<COROPE_CODE_INT8>, blocks, kMoveThreads, 0, s, p, out_used);
}

}  // namespace corope
