// What the kernels of corope_cache_attn share: codes as fp16, and the division of a batch's work among blocks.
#pragma once
#include "cache.cuh"

namespace corope {

#ifdef __CUDACC__
__host__ __device__ constexpr int log2_of(int x) { return x > 1 ? 1 + log2_of(x / 2) : 0; }

constexpr float kLowest = -1e30f;             // running maximum before any score: finite, so that differences from it are no NaN

// Values of a block whose scale of V is below this count as 0 (as those of a scale of 0 do): the scale enters the exponents, and its reciprocal the sums
// of fp32 probabilities, which 2^27 slots of the largest exponent then still fit.
constexpr float kLeastScale = 1e-30f;
__device__ __forceinline__ bool no_values(float v_scale) { return v_scale < kLeastScale; }

// The power of two 2^-e that brings a row whose largest element is m to [2^10, 2^11), so that the second of two fp16 parts is a normal number too; as `up` =
// 2^-e and `down` = 2^e.  Rows below 2^-100 stay below 2^10; rows with infinities or NaN are left as they are.
__device__ __forceinline__ void row_scaling(float m, float& up, float& down) {
    const bool finite = m > 0.f && m <= 3.402823466e38f;
    const int e = finite ? max((int)(__float_as_uint(m) >> 23) - 127 - 10, -110) : 0;
    up = __uint_as_float((uint32_t)(127 - e) << 23);
    down = __uint_as_float((uint32_t)(127 + e) << 23);
}

// four codes as fp16: (0, 1), (2, 3)
template <int CODE>
__device__ __forceinline__ void codes_to_half(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if constexpr (CODE == COROPE_CODE_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(word));
    } else {   // the byte c + 128 behind the fp16 exponent of 1024 reads as 1024 + 128 + c
        const uint32_t u = word ^ 0x80808080u, bias = 0x64806480u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// A query that sees no slot (an empty place of a padded batch) is not read: its position need not be in the tables.
__device__ __forceinline__ bool sees_something(const CacheAttnParams& p, int len, int n, int t) { return (p.causal ? len - n + t + 1 : len) > 0; }

// ------------------------------------------------------------------------------------------------ division of the work
// Work is counted in units of `unit` slots of one item, a (K / V head, tile of query rows) of a sequence: sequence b has items(b) = Hkv * (row tiles in
// use) items of units(b) units each, one after the other.  Tiles whose rows all come before slot 0 (causal, more queries than tokens) are no
// items: the joining kernel writes their zeros.
// What an item costs beside its units (queries made ready, parts joined and written) is counted as `extra` units in front of them, so that a block
// with the ends of several items has as long to do as one with the middle of one.
struct Load {
    int len, n, units, items, cost;   // cost: of an item, extra units included
};
// Rows of a tile and slots of a unit are powers of two, given by their logarithms: the joining kernel has them as arguments and would divide.
// The first tile with a row that sees a slot (of a sequence that has slots):
__device__ __forceinline__ int first_tile(const CacheAttnParams& p, int rows_log2, int len, int n) { return p.causal ? max(n - len, 0) * p.G >> rows_log2 : 0; }
__device__ __forceinline__ int tiles_in_use(const CacheAttnParams& p, int rows_log2, int len, int n) {
    return ((n * p.G + (1 << rows_log2) - 1) >> rows_log2) - first_tile(p, rows_log2, len, n);
}
__device__ __forceinline__ Load load_of(const CacheAttnParams& p, int rows_log2, int unit_log2, int extra, int b, bool& bad) {
    Load l;
    l.len = cache_len(p.s, p.c.bs_log2, b, bad);
    l.n = cache_new(p.s, p.T, b, bad);
    l.units = (l.len + (1 << unit_log2) - 1) >> unit_log2;
    l.items = p.c.Hkv * tiles_in_use(p, rows_log2, l.len, l.n);
    l.cost = l.units > 0 ? l.units + extra : 0;
    return l;
}
// The range of units that a block has (its first THREADS threads look at the sequences), as a place to start (sequence b, `off` into its own) and a number of units; 0 of
// them: the block is not needed.  `load(b)` tells a sequence's load.
struct Range {
    int b;
    int64_t off, left;
};
template <int THREADS, typename LoadFn>
__device__ __forceinline__ Range take_range(int B, const LoadFn& load) {
    constexpr int kWarps = THREADS / 32;
    __shared__ int64_t words[kWarps], start_off;
    __shared__ int start_b;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int per = (B + THREADS - 1) / THREADS, b0 = min((int)threadIdx.x * per, B), b1 = min(b0 + per, B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        const Load l = load(b);
        mine += (int64_t)l.cost * l.items;
    }
    int64_t sum = mine;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, m);
        if (lane >= m) sum += up;
    }
    if (lane == 31 && warp < kWarps) words[warp] = sum;
    __syncthreads();
    int64_t at = sum - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += words[w];
        total += words[w];
    }
    const int64_t ranges = min((int64_t)gridDim.x, total);
    if (blockIdx.x >= ranges) return Range{0, 0, 0};
    const int64_t lo = total * blockIdx.x / ranges, hi = total * (blockIdx.x + 1) / ranges;
    if (lo >= at && lo < at + mine)
        for (int b = b0; b < b1; ++b) {
            const Load l = load(b);
            const int64_t u = (int64_t)l.cost * l.items;
            if (lo >= at && lo < at + u) start_b = b, start_off = lo - at;
            at += u;
        }
    __syncthreads();
    return Range{start_b, start_off, hi - lo};
}

#endif  // __CUDACC__

// Attention of many query rows a K / V head on tcgen05 (16-bit types): the steps of launch_cache_attn that are its own.
constexpr int kTileRows = 128;                // query rows of a tile, and slots of a unit
// Units that an item counts beside its own in sharing out the work (queries loaded, parts written).  0 / 2 / 4 / 8, us, 32 / 8 heads of 128: 32
// sequences of up to 4096 tokens with 16 queries each 137 / 116 / 109 / 109, one of 4096 with 256 59.4 / 53.8 / 51.5 / 53.3, one of 9001 with 1024
// 216 / 216 / 217 / 226.
constexpr int kTileItemCost = 4;
bool cache_tile_pairs(int rows, int D, bool two_parts);   // items of two tiles of rows
size_t cache_tile_workspace_bytes(int B, int Hkv, int image_tiles, int D, bool two_parts);
int launch_cache_attn_tiles(const CacheAttnParams& p, void* ws, bool two_parts, bool pair, unsigned blocks, cudaStream_t s);
int launch_cache_weight_tiles(const CacheAttnParams& p, void* ws, bool pair, cudaStream_t s);

}  // namespace corope
