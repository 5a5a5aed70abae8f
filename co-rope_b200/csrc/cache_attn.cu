// corope_cache_attn: attention of a few query rows per K / V head over the 8-bit cache.
//
// With R = G * T query rows a head, 2 D bytes of cache are read per slot for 4 R D operations: memory bound up to R of about 100.  So the kernel is built
// around the reads:
//   * Work is counted in units of 64 slots of one (sequence, K / V head, tile of query rows) and cut into equal contiguous ranges, one per resident
//     block, from the lengths on the device: a batch of unequal lengths loads every SM alike.  A range that starts or ends inside an item leaves
//     its part (fp32 sums, maximum, total) in the workspace, and a second kernel joins the parts in a fixed order.  Short sequences are cut
//     evenly among the blocks of a cluster instead, which join their parts through each other's shared memory: one kernel, no workspace.
//   * Each warp streams its own 16-slot pieces (a piece lies in one block, so one scale) through its own ring in shared memory with
//     cp.async, without block-wide barriers.
//   * Products on mma.sync with slots as the M extent and query rows as N = 8: S^T = K Q^T, O^T = V^T P^T.  Codes become fp16 in registers,
//     exactly.  Which elements a lane takes is chosen so that it reads whole 16-byte runs: the order of the sum over d is free, and so is the
//     order of the rows of O^T.
//   * Rotated queries are scaled by a power of two per row and split into two fp16 numbers (22 bits), so scores have fp32 accuracy.
//     exp2(s + log2(v scale) - M) is rounded to fp16 (11 bits) for 16-bit outputs, whose own rounding is coarser or equal, and split in two for
//     fp32 ones; the sum of the probabilities stays fp32.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "cache_attn.cuh"

namespace corope {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kPiece = 16;                    // slots per step of a warp; a block of the cache holds a whole number of them
constexpr int kUnit = kWarps * kPiece, kUnitLog2 = log2_of(kUnit);        // slots per unit of work
// Tensor cores truncate where they add to their sums, by up to 2^-23 of the sum in each step, and always towards 0.  So the sums of a block's units of an
// item are added in fp32 after this many of them (a step each; 2^-13 of the result at most).  With one sum for all of 2^20 slots fp16 results came out
// 1.8e-3 too small.
constexpr int kMostUnits = 1024;
// Units that an item counts beside its own in sharing out the work.  With 8 rows 0 / 4 / 6 / 12, us, 32 / 8 heads of 128: 64 x up to 4096 tokens 68.1 / 62.6 /
// 60.5 / 63.1, 256 x up to 1000 97.6 / 80.3 / 80.6 / 81.8, 8 x 16384 58.0 / 56.4 / 56.5 / 57.6.
// Two more for each further eight rows: 6 / 8 with 16 rows, 16 x up to 4000 tokens and their weights, 45.4 / 43.7; 6 / 12 / 20 with 32 rows, 64 x up to
// 4000, 157.6 / 152.7 / 161.2.
__host__ __device__ constexpr int item_cost(int groups) { return 4 + 2 * groups; }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool real) {   // zeros where not real
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int WORDS> __device__ __forceinline__ void load_words(uint32_t (&w)[WORDS], int at, uint32_t addr) {   // 1, 2 or 4 words to w[at ..]
    static_assert(WORDS == 1 || WORDS == 2 || WORDS % 4 == 0, "");
    if constexpr (WORDS == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[at]) : "r"(addr));
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[at]), "=r"(w[at + 1]) : "r"(addr));
    else asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[at]), "=r"(w[at + 1]), "=r"(w[at + 2]), "=r"(w[at + 3]) : "r"(addr));
}

// ------------------------------------------------------------------------------------------------ queries
// Shared-memory form of a tile of query rows: for k-step w, row group nt and lane, {hi b0, b1, lo b0, b1} of the B operand.
// Lane (g, c) of the MMA holds row g and the columns c * D / 4 + 4 w .. + 3.
template <int D, int NT>
__device__ __forceinline__ void pack_queries(const CacheAttnParams& p, int b, int h, int row0, int len, int n, uint32_t* packed, float* factor,
                                             bool& bad) {
    constexpr int kHalf = D / 2, kPairLanes = kHalf / 2;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int r = warp; r < 8 * NT; r += kWarps) {
        const int row = row0 + r, t = row / p.G;
        float x[4] = {0.f, 0.f, 0.f, 0.f};   // columns 2 lane, + 1, and their partners D / 2 further on
        if (t < n && sees_something(p, len, n, t) && lane < kPairLanes) {
            const int64_t at = (int64_t)b * p.sq.b + (int64_t)(h * p.G + row - t * p.G) * p.sq.h + (int64_t)t * p.sq.n + 2 * lane;
            x[0] = load1(p.q, at, p.dtype); x[1] = load1(p.q, at + 1, p.dtype);
            x[2] = load1(p.q, at + kHalf, p.dtype); x[3] = load1(p.q, at + kHalf + 1, p.dtype);
            if (p.s.cos != nullptr) {
                const int64_t tr = (int64_t)cache_position(p.s, b, t, len - n + t, bad) * p.s.rope_stride + 2 * lane;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float c = p.s.cos[tr + i], s = p.s.sin[tr + i], u = x[i], v = x[i + 2];
                    x[i] = u * c - v * s;
                    x[i + 2] = v * c + u * s;
                }
            }
        }
        float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
        for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
        float up, down;
        row_scaling(m, up, down);
        if (lane == 0) factor[r] = down * p.scale;
        if (lane < kPairLanes) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 2 * lane + i * kHalf, c = d / (D / 4), w = d % (D / 4) / 4, j = d % 4 / 2;
                const float u = x[2 * i] * up, v = x[2 * i + 1] * up;
                const uint32_t hi = pack_half2(u, v);
                const float2 back = unpack_half2(hi);
                uint32_t* to = packed + ((w * NT + r / 8) * 32 + r % 8 * 4 + c) * 4 + j;
                to[0] = hi;
                to[2] = pack_half2(u - back.x, v - back.y);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ main kernel
template <int D, int NT>
struct Shape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kStages = D == 128 ? 3 : D == 64 ? 6 : 8;
    static constexpr int kStageBytes = 2 * kPiece * D;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kJoin = kWarps * kRows * D * 4;                    // the warps' sums, in the place of the rings
    static constexpr int kBig = kRing > kJoin ? kRing : kJoin;
    static constexpr int kPacked = D / 16 * NT * 32 * 16;
    static constexpr int kMeta = kWarps * kStages * 16;                     // {k scale, v scale, block found} of each stage
    static constexpr int kSmem = kBig + kPacked + kMeta + kRows * 4 + 2 * kWarps * kRows * 4 + 2 * kRows * 4;
    static constexpr int kBlocks = NT == 1 ? 4 : NT == 2 ? 3 : 2;                         // resident per SM
};

template <int D, int CODE, int NT, bool EXACT_P>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kBlocks) cache_attn_kernel(const CacheAttnParams p) {
    using S = Shape<D, NT>;
    constexpr int kItemCost = item_cost(NT);
    constexpr int kRows = S::kRows, kRowsLog2 = log2_of(kRows), kKSteps = D / 16, kVWords = D / 32, kStages = S::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    uint32_t* packed = reinterpret_cast<uint32_t*>(smem + S::kBig);
    float* meta = reinterpret_cast<float*>(smem + S::kBig + S::kPacked);
    float* factor = meta + S::kMeta / 4;
    float* warp_max = factor + kRows;
    float* warp_sum = warp_max + kWarps * kRows;
    float* part_max = warp_sum + kWarps * kRows;
    float* part_sum = part_max + kRows;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
    bool bad = false;

    auto load = [&](int b) { return load_of(p, kRowsLog2, kUnitLog2, kItemCost, b, bad); };
    __shared__ int nan_v;   // NaN in V where some rows must not see it
    // The block's share of the item at work: its first unit, whether sums of earlier units wait in the block's part, and whether units are still to come.
    // (Not in registers, of which there are none left.)
    __shared__ int share0, carried, more;
    if (p.parts == 0 && threadIdx.x == 0) more = 0;
    // Either a range of the batch's units, or (p.parts) this block's share of one item, whose other shares are with the blocks of its cluster.
    int b, part_of = 0, cluster_item = 0;
    int64_t off = 0, left = 0;   // position in sequence b's units, units left
    if (p.parts == 0) {
        const Range range = take_range<kThreads>(p.s.B, load);
        pdl_trigger();
        if (range.left == 0) {
            if (bad) report_bad_index(p.status, p.mirror);
            return;
        }
        b = range.b;
        off = range.off;
        left = range.left;
    } else {
        cluster_item = (int)(blockIdx.x / (unsigned)p.parts);
        part_of = (int)(blockIdx.x - (unsigned)cluster_item * p.parts);
        b = cluster_item / (p.c.Hkv * p.row_tiles);
    }
    Load l = load(b);

    uint8_t* ring = smem + warp * (kStages * S::kStageBytes);
    float* my_meta = meta + warp * kStages * 4;
    const uint32_t ring_at = smem_u32(ring), meta_at = smem_u32(my_meta), packed_at = smem_u32(packed) + lane * 16;
    // A stage holds 16 rows of K, then of V; the 16-byte run x of a tile sits at run x ^ (x / 8 % 8), which keeps the reads below off one
    // another's banks.  Lane's share of a copy: runs lane + 32 i, rows copy_row + kCopyRows i.
    constexpr int kCopyRows = 512 / D;
    const int copy_row = lane / (D / 16), copy_col = lane % (D / 16) * 16;
    const uint32_t copy_to = (uint32_t)(lane ^ (lane >> 3)) * 16;
    // K: row g, its c-th quarter.  V: row 2 c, its g-th eighth; the row after it and the rows 8 further on are one XOR and one addition away.
    constexpr uint32_t kNext8Xor = D == 128 ? 0 : D == 64 ? 64 : 32, kNextXor = D == 128 ? 16 : D == 64 ? 64 : 32, kNextAdd = D == 128 ? 128 : 0;
    const uint32_t k_run = (g * D + c * (D / 4)) / 16, v_run = (2 * c * D + g * (D / 8)) / 16;
    const uint32_t k_from = (k_run ^ (k_run >> 3 & 7)) * 16 + c * (D / 4) % 16, v_from = (v_run ^ (v_run >> 3 & 7)) * 16 + g * (D / 8) % 16;

    do {
        int h, tile, u0, u1;
        bool goes_on = false;
        if (p.parts == 0) {
            while (off >= (int64_t)l.cost * l.items) {
                off -= (int64_t)l.cost * l.items;
                l = load(++b);
            }
            const int item = (int)(off / l.cost), tiles = l.items / p.c.Hkv;
            h = item / tiles;
            tile = item % tiles + first_tile(p, kRowsLog2, l.len, l.n);
            u0 = (int)(off - (int64_t)item * l.cost);
            const int end = (int)min((int64_t)l.cost, u0 + left);
            u1 = min(end, max(u0, kItemCost) + kMostUnits);
            off += u1 - u0;
            left -= u1 - u0;
            goes_on = u1 < end;
            u0 = max(u0 - kItemCost, 0);
            u1 -= kItemCost;
            if (u1 <= 0) continue;   // the range ends before the item's first unit
        } else {
            const int item = cluster_item - b * p.c.Hkv * p.row_tiles;
            h = item / p.row_tiles;
            tile = item - h * p.row_tiles;
            const int units = tile * kRows < l.n * p.G ? l.units : 0;
            u0 = units * part_of / p.parts;
            u1 = units * (part_of + 1) / p.parts;
        }
        const int row0 = tile * kRows, len = l.len, n = l.n;
        // slots below least_seen are seen by every row of the tile (rows without a query see what they like)
        const int least_seen = p.causal ? len - n + row0 / p.G + 1 : len;
        __syncthreads();   // the tile before is written out
        if (threadIdx.x == 0) {
            nan_v = 0;
            if (p.parts == 0) {
                carried = more;
                more = goes_on;
                if (!carried) share0 = u0;
            }
        }
        // pieces first, first + 4, .. of this warp
        const int first = u0 * kWarps + warp, end = min(u1 * kWarps, (len + kPiece - 1) / kPiece);
        const int count = end > first ? (end - first + kWarps - 1) / kWarps : 0;
        const int* table = p.s.table + (int64_t)b * p.s.table_stride;
        const int shift = p.c.bs_log2 - 4, in_block_mask = (1 << p.c.bs_log2) - 1;
        const uint8_t* k_lane = p.c.k + (int64_t)h * p.c.sk.h + (int64_t)copy_row * p.c.sk.n + copy_col;
        const uint8_t* v_lane = p.c.v + (int64_t)h * p.c.sv.h + (int64_t)copy_row * p.c.sv.n + copy_col;
        const float* scale_lane = (lane ? p.c.v_scale : p.c.k_scale) + h;
        const uint32_t k_block = (uint32_t)p.c.sk.b, v_block = (uint32_t)p.c.sv.b, k_row = (uint32_t)p.c.sk.n, v_row = (uint32_t)p.c.sv.n;   // below 2^32
        const int* entry = table + (first >> shift);   // of the next piece to be copied
        int next_page = count > 0 ? *entry : 0;
        uint32_t fill = ring_at + copy_to, fill_meta = meta_at + lane * 4;   // where its copy goes
        int next_piece = first;
        auto issue = [&](int j) {
            if (j < count) {
                const bool found = (unsigned)next_page < (unsigned)p.c.num_blocks;
                const uint32_t page = found ? (uint32_t)next_page : 0u, in_block = (uint32_t)(next_piece << 4) & (uint32_t)in_block_mask;
                const int rows = len - (next_piece << 4);
                next_piece += kWarps;
                if (j + 1 < count) next_page = table[next_piece >> shift];
                const uint8_t* kb = k_lane + (uint64_t)page * k_block + (uint64_t)in_block * k_row;
                const uint8_t* vb = v_lane + (uint64_t)page * v_block + (uint64_t)in_block * v_row;
                const uint32_t other = fill ^ 64;
                if (found && rows >= kPiece && p.rows_packed && !bad) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        copy16_async((i % 2 ? other : fill) + 512 * i, kb + i * 512);
                        copy16_async((i % 2 ? other : fill) + 512 * i + kPiece * D, vb + i * 512);
                    }
                } else {   // slots behind the last one, and those of a block that is not there, become zeros
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const bool real = found && copy_row + i * kCopyRows < rows;
                        copy16_async((i % 2 ? other : fill) + 512 * i, real ? kb + (uint64_t)(i * kCopyRows) * k_row : p.c.k, real);
                        copy16_async((i % 2 ? other : fill) + 512 * i + kPiece * D, real ? vb + (uint64_t)(i * kCopyRows) * v_row : p.c.v, real);
                    }
                    bad |= !found;
                    if (lane == 2) my_meta[j % kStages * 4 + 2] = found ? 1.f : 0.f;   // (1 before the first bad one)
                }
                if (lane < 2) copy4_async(fill_meta, scale_lane + (uint64_t)page * (uint32_t)p.c.Hkv);
            }
            commit_copies();
            fill += S::kStageBytes;
            fill_meta += 16;
            if (fill == ring_at + copy_to + kStages * S::kStageBytes) fill = ring_at + copy_to, fill_meta = meta_at + lane * 4;
        };
        if (lane < kStages) my_meta[lane * 4 + 2] = 1.f;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kStages - 1; ++j) issue(j);   // on their way while the queries are made ready

        pack_queries<D, NT>(p, b, h, row0, len, n, packed, factor, bad);
        __syncthreads();

        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) fac[nt][i] = factor[8 * nt + 2 * c + i];
        // slots below this are seen by the row
        auto sees = [&](int nt, int i) { return p.causal ? len - n + (row0 + 8 * nt + 2 * c + i) / p.G + 1 : len; };
        // m: reference of the exponents, which are at most 8 (exp2 of that fits fp16): it moves when one is beyond `most`, -infinity before the first
        float o[NT][D / 16][4], m[NT][2], most[NT][2], sum[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][x][i] = 0.f;
            m[nt][0] = m[nt][1] = 0.f;
            most[nt][0] = most[nt][1] = -INFINITY;
            sum[nt][0] = sum[nt][1] = 0.f;
        }

        uint32_t stage_at = ring_at;
        int stage = 0;
        for (int j = 0; j < count; ++j) {
            issue(j + kStages - 1);   // into the stage that step j - 1 has read
            wait_copies<kStages - 1>();
            __syncwarp();
            const int slot0 = (first + j * kWarps) * kPiece;
            const uint32_t k_at = stage_at + k_from, v_at = stage_at + kPiece * D + v_from;
            const float4 said = *reinterpret_cast<const float4*>(my_meta + stage * 4);
            const float k_scale = said.x, v_scale = said.y;
            const bool found = said.z != 0.f;

            // S^T: slots g and g + 8 by rows 2 c and 2 c + 1
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
            float rest[NT][4];   // the second parts' products apart: their sum's truncations are 2^-11 of those of the first
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) rest[nt][0] = rest[nt][1] = rest[nt][2] = rest[nt][3] = 0.f;
            uint32_t k0[D / 16], k1[D / 16];
#pragma unroll
            for (int i = 0; i < (D + 63) / 64; ++i) {
                load_words(k0, 4 * i, k_at ^ (16 * i));
                load_words(k1, 4 * i, (k_at ^ (16 * i) ^ kNext8Xor) + kPiece * D / 2);
            }
#pragma unroll
            for (int w = 0; w < kKSteps; ++w) {
                uint32_t a[4];
                codes_to_half<CODE>(k0[w], a[0], a[2]);
                codes_to_half<CODE>(k1[w], a[1], a[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t q[4];   // read each time: held in registers they would cost more than they save
                    load_words(q, 0, packed_at + (w * NT + nt) * 512);
                    mma16816(s[nt], a, q[0], q[1]);
                    mma16816(rest[nt], a, q[2], q[3]);
                }
            }

            // scores in units of log2, the scale of V folded into the exponent: O = sum of exp2(s + log2 v_scale - M) * code
            // (a scale without values is left out of the exponent, and its slots out of O)
            const bool no_v = no_values(v_scale);
            const float v_size = no_v ? 1.f : v_scale, lift = fast_log2(v_size), drop = fast_reciprocal(v_size);
            bool higher = false;
            const bool masked = !found || slot0 + kPiece > least_seen;
            auto hide = [&]() {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = found && slot0 + g + 8 * (i / 2) < sees(nt, i % 2) ? s[nt][i] : -INFINITY;
            };
            // s becomes the exponent, relative to m
            if (p.scores == nullptr) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = fac[nt][0] * k_scale, f1 = fac[nt][1] * k_scale, a0 = lift - m[nt][0], a1 = lift - m[nt][1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = fmaf(s[nt][i] + rest[nt][i], i % 2 ? f1 : f0, i % 2 ? a1 : a0);
                }
                if (masked) hide();
            } else {   // the scores are kept for the weights: whole rows of `score_rows` numbers a slot
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = fac[nt][0] * k_scale, f1 = fac[nt][1] * k_scale;
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = (s[nt][i] + rest[nt][i]) * (i % 2 ? f1 : f0);
                }
                if (masked) hide();
                float* to = p.scores + (((int64_t)b * p.c.Hkv + h) * p.capacity + slot0 + g) * p.score_rows + 2 * c;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (8 * nt + 2 * c < p.score_rows) {
                        if (slot0 + g < len) *reinterpret_cast<float2*>(to + 8 * nt) = make_float2(s[nt][0], s[nt][1]);
                        if (slot0 + g + 8 < len) *reinterpret_cast<float2*>(to + 8 * p.score_rows + 8 * nt) = make_float2(s[nt][2], s[nt][3]);
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = s[nt][i] == -INFINITY ? s[nt][i] : s[nt][i] + (lift - m[nt][i % 2]);   // (hidden whatever the lift)
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) higher |= fmaxf(s[nt][i], s[nt][i + 2]) > most[nt][i];
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float up = fmaxf(s[nt][i], s[nt][i + 2]);
#pragma unroll
                        for (int k = 4; k < 32; k *= 2) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, k));
                        const bool begins = most[nt][i] < 0.f;
                        if (begins && up == -INFINITY) continue;   // no score yet
                        if (!begins) up = fmaxf(up, 0.f);
                        const float shrink = begins ? 0.f : fast_exp2(-up);
                        m[nt][i] += up;
                        most[nt][i] = 8.f;
                        s[nt][i] -= up;
                        s[nt][i + 2] -= up;
                        sum[nt][i] *= shrink;
#pragma unroll
                        for (int x = 0; x < D / 16; ++x) o[nt][x][i] *= shrink, o[nt][x][i + 2] *= shrink;
                    }
            }
            uint32_t pb[NT][2], pl[EXACT_P ? NT : 1][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = fast_exp2(s[nt][i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float both = w[i] + w[i + 2];
                    sum[nt][i] = both == 0.f ? sum[nt][i] : fmaf(both, drop, sum[nt][i]);   // hidden slots of a block whose scale is NaN count nothing
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t hi = no_v ? 0u : pack_half2(w[2 * i], w[2 * i + 1]);
                    pb[nt][i] = transpose8x8(hi);
                    if constexpr (EXACT_P) {
                        const float2 back = unpack_half2(hi);
                        pl[nt][i] = transpose8x8(no_v ? 0u : pack_half2(w[2 * i] - back.x, w[2 * i + 1] - back.y));
                    }
                }
            }

            // O^T: columns g * D / 8 + 2 x and + 1 of V by rows 2 c and 2 c + 1
            uint32_t v[4][kVWords];
#pragma unroll
            for (int i = 0; i < 4; ++i)   // slots 2 c, 2 c + 1, and 8 further on
                load_words(v[i], 0, (v_at ^ (i % 2 * kNextXor) ^ (i / 2 * kNext8Xor)) + i % 2 * kNextAdd + i / 2 * (kPiece * D / 2));
            // NaN in V reaches the rows that see its slot, and 0 * NaN would bring it to the others: it is left out here and put in when the rows are written
            if (CODE == COROPE_CODE_E4M3 && slot0 + kPiece > least_seen) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) {
                        const uint32_t where = __vcmpeq4(v[i][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        if (where) nan_v = 1;
                        v[i][w] &= ~where;
                    }
            }
#pragma unroll
            for (int w = 0; w < kVWords; ++w) {
                uint32_t a[2][4];
                codes_to_half<CODE>(__byte_perm(v[0][w], v[1][w], 0x5140), a[0][0], a[0][1]);
                codes_to_half<CODE>(__byte_perm(v[2][w], v[3][w], 0x5140), a[0][2], a[0][3]);
                codes_to_half<CODE>(__byte_perm(v[0][w], v[1][w], 0x7362), a[1][0], a[1][1]);
                codes_to_half<CODE>(__byte_perm(v[2][w], v[3][w], 0x7362), a[1][2], a[1][3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        if constexpr (EXACT_P) {   // the long sum in fp32 additions, as MMA accumulation truncates
                            float t[4] = {0.f, 0.f, 0.f, 0.f};
                            mma16816(t, a[y], pb[nt][0], pb[nt][1]);
                            mma16816(t, a[y], pl[nt][0], pl[nt][1]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[nt][2 * w + y][i] += t[i];
                        } else {
                            mma16816(o[nt][2 * w + y], a[y], pb[nt][0], pb[nt][1]);
                        }
                    }
            }
            stage_at += S::kStageBytes;
            if (++stage == kStages) stage = 0, stage_at = ring_at;
            __syncwarp();   // the stage has been read
        }
        wait_copies<0>();

        // join the four warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (most[nt][i] < 0.f) m[nt][i] = kLowest;
#pragma unroll
                for (int k = 4; k < 32; k *= 2) sum[nt][i] += __shfl_xor_sync(0xffffffffu, sum[nt][i], k);
                if (g == 0) {
                    warp_max[warp * kRows + 8 * nt + 2 * c + i] = m[nt][i];
                    warp_sum[warp * kRows + 8 * nt + 2 * c + i] = sum[nt][i];
                }
            }
        __syncthreads();
        float* join = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * nt + 2 * c + i;
                float top = warp_max[r];
#pragma unroll
                for (int k = 1; k < kWarps; ++k) top = fmaxf(top, warp_max[k * kRows + r]);
                const float shrink = fast_exp2(m[nt][i] - top);
                float2* to = reinterpret_cast<float2*>(join + (warp * kRows + r) * D + g * (D / 8));
#pragma unroll
                for (int x = 0; x < D / 16; ++x) to[x] = make_float2(o[nt][x][i] * shrink, o[nt][x][i + 2] * shrink);
            }
        __syncthreads();
        auto write_row = [&](int r, int d, const float4& y, float all) {
            const int row = row0 + r, t = row / p.G;
            const float f = 1.f / all;
            store4(p.o, (int64_t)b * p.so.b + (int64_t)(h * p.G + row - t * p.G) * p.so.h + (int64_t)t * p.so.n + d, p.dtype, p.vec_o,
                   t >= n || all == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
        };
        bool whole = false, add = false;   // the block has all of the item; its part holds sums to be added
        int64_t part = 0;
        if (p.parts == 0) {
            whole = share0 == 0 && u1 == l.units;
            add = carried != 0;
            part = 2 * (int64_t)blockIdx.x + (share0 == 0 ? 1 : 0);
            if (add) {
                if (threadIdx.x < kRows) {
                    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (part * kRows + threadIdx.x) * 2);
                    part_max[threadIdx.x] = ml.x;
                    part_sum[threadIdx.x] = ml.y;
                }
                __syncthreads();
            }
        }
        for (int x = threadIdx.x; x < kRows * (D / 4); x += kThreads) {
            const int r = x / (D / 4), d = x % (D / 4) * 4, row = row0 + r, t = row / p.G;
            float top = warp_max[r], all = 0.f;
#pragma unroll
            for (int k = 1; k < kWarps; ++k) top = fmaxf(top, warp_max[k * kRows + r]);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) all = fmaf(warp_sum[k * kRows + r], fast_exp2(warp_max[k * kRows + r] - top), all);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float4 z = *reinterpret_cast<const float4*>(join + (k * kRows + r) * D + d);
                y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            }
            if (CODE == COROPE_CODE_E4M3 && nan_v != 0) {
                const int sees_row = t >= n ? 0 : p.causal ? len - n + t + 1 : len;   // (never behind the last slot, whose block the table still has)
#pragma unroll 1
                for (int slot = max(u0 * kUnit, least_seen / kPiece * kPiece); slot < min(sees_row, u1 * kUnit); ++slot) {   // from where it was left out
                    const int page = table[slot >> p.c.bs_log2];
                    if ((unsigned)page >= (unsigned)p.c.num_blocks || no_values(p.c.v_scale[(int64_t)page * p.c.Hkv + h])) continue;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(p.c.v + (int64_t)page * p.c.sv.b + (int64_t)h * p.c.sv.h + (int64_t)(slot & in_block_mask) * p.c.sv.n + d);
                    if ((word & 0x7fu) == 0x7fu) y.x = __int_as_float(0x7fffffff);
                    if ((word >> 8 & 0x7fu) == 0x7fu) y.y = __int_as_float(0x7fffffff);
                    if ((word >> 16 & 0x7fu) == 0x7fu) y.z = __int_as_float(0x7fffffff);
                    if ((word >> 24 & 0x7fu) == 0x7fu) y.w = __int_as_float(0x7fffffff);
                }
            }
            if (p.parts != 0) {   // for the cluster: in the place of warp 0's sums
                *reinterpret_cast<float4*>(join + r * D + d) = y;
                if (d == 0) part_max[r] = top, part_sum[r] = all;
                continue;
            }
            if (add) {   // (this thread has written them)
                const float best = fmaxf(top, part_max[r]), now = fast_exp2(top - best), then = fast_exp2(part_max[r] - best);
                const float4 was = *reinterpret_cast<const float4*>(p.part + (part * kRows + r) * D + d);
                y = make_float4(fmaf(was.x, then, y.x * now), fmaf(was.y, then, y.y * now), fmaf(was.z, then, y.z * now), fmaf(was.w, then, y.w * now));
                all = fmaf(part_sum[r], then, all * now);
                top = best;
            }
            if (!whole) {
                *reinterpret_cast<float4*>(p.part + (part * kRows + r) * D + d) = y;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (part * kRows + r) * 2) = make_float2(top, all);
            } else if (t < p.T) {
                write_row(r, d, y, all);
                if (p.lse != nullptr && d == 0) p.lse[((int64_t)b * p.c.Hkv + h) * p.T * p.G + row] = t >= n || all == 0.f ? INFINITY : top + log2f(all);
            }
        }
        if (p.parts != 0) {
            // The blocks of the cluster have the item's parts in their shared memories: each writes its share of the output's runs of four, and adds the
            // weights of its own slots.
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            auto whole_row = [&](int r, float& top, float& all) {
                top = kLowest;
                all = 0.f;
                for (int q = 0; q < p.parts; ++q) top = fmaxf(top, *cluster.map_shared_rank(part_max + r, q));
                for (int q = 0; q < p.parts; ++q) all = fmaf(*cluster.map_shared_rank(part_sum + r, q), fast_exp2(*cluster.map_shared_rank(part_max + r, q) - top), all);
            };
            for (int x = part_of * kThreads + threadIdx.x; x < kRows * (D / 4); x += p.parts * kThreads) {
                const int r = x / (D / 4), d = x % (D / 4) * 4;
                if ((row0 + r) / p.G >= p.T) break;
                float top, all;
                whole_row(r, top, all);
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int q = 0; q < p.parts; ++q) {
                    const float4 z = *reinterpret_cast<const float4*>(cluster.map_shared_rank(join + r * D + d, q));
                    const float f = fast_exp2(*cluster.map_shared_rank(part_max + r, q) - top);
                    y.x = fmaf(z.x, f, y.x); y.y = fmaf(z.y, f, y.y); y.z = fmaf(z.z, f, y.z); y.w = fmaf(z.w, f, y.w);
                }
                write_row(r, d, y, all);
            }
            if (p.scores != nullptr) {
                const int rows = min(kRows, n * p.G - row0);   // one tile
                if (threadIdx.x < rows) {
                    float top, all;
                    whole_row(threadIdx.x, top, all);
                    warp_max[threadIdx.x] = all == 0.f ? INFINITY : top + log2f(all);
                }
                __syncthreads();
                for (int slot = u0 * kUnit + threadIdx.x; slot < min(u1 * kUnit, len); slot += kThreads) {
                    const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad);
                    const float* from = p.scores + (((int64_t)b * p.c.Hkv + h) * p.capacity + slot) * p.score_rows;
                    float w = 0.f;
                    for (int r = 0; r < rows; ++r) w += fast_exp2(from[r] - warp_max[r]);
                    if (page >= 0) atomicAdd(p.c.weight + (((int64_t)page * p.c.Hkv + h) << p.c.bs_log2) + (slot & in_block_mask), w);
                }
            }
            cluster.sync();   // no block ends while another reads its part
        }
    } while (left > 0);
    if (bad) report_bad_index(p.status, p.mirror);
}

// ------------------------------------------------------------------------------------------------ joining parts
// A warp per query row, a block per eight rows of an item.  An item that one block of the main kernel did alone is finished; the parts of the others are
// added in the order of their ranges.  Rows that no unit stands for are written here: 0.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads, 6) cache_attn_join_kernel(const CacheAttnParams p, int rows_log2, int unit_log2, int extra, int main_blocks) {
    __shared__ int64_t words[2][kJoinThreads / 32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int rows_per_tile = 1 << rows_log2;
    const unsigned blocks_log2 = rows_log2 - log2_of(kJoinThreads / 32), item = blockIdx.x >> blocks_log2;
    const int tile = (int)(item % (unsigned)p.row_tiles), bh = (int)(item / (unsigned)p.row_tiles), b = bh / p.c.Hkv, h = bh - b * p.c.Hkv;
    bool bad = false;
    int64_t before = 0, total = 0;
    for (int i = threadIdx.x; i < p.s.B; i += kJoinThreads) {
        const Load l = load_of(p, rows_log2, unit_log2, extra, i, bad);
        const int64_t u = (int64_t)l.cost * l.items;
        total += u;
        if (i < b) before += u;
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, m);
        total += __shfl_xor_sync(0xffffffffu, total, m);
    }
    if (lane == 0) words[0][warp] = before, words[1][warp] = total;
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) before += words[0][w], total += words[1][w];

    const Load l = load_of(p, rows_log2, unit_log2, extra, b, bad);
    const int tiles = tiles_in_use(p, rows_log2, l.len, l.n), tile0 = first_tile(p, rows_log2, l.len, l.n);
    const bool empty = l.units == 0 || tile < tile0 || tile >= tile0 + tiles;
    const int64_t ranges = min((int64_t)main_blocks, total);
    int r0 = 0, r1 = 0;
    if (!empty) {
        const int64_t u0 = before + (int64_t)(h * tiles + tile - tile0) * l.cost + extra, u1 = u0 + l.units - 1;
        r0 = (int)(((u0 + 1) * ranges - 1) / total);   // the range that holds a unit
        r1 = (int)(((u1 + 1) * ranges - 1) / total);
    }
    pdl_wait();   // by every block: the end of this kernel has to stand for the end of the one before
    if (!empty && r0 == r1) return;
    {
        const int r = (int)(blockIdx.x - (item << blocks_log2)) * (kJoinThreads / 32) + warp, row = tile * rows_per_tile + r, t = row / p.G;
        if (t >= p.T) return;
        float top = kLowest, all = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!empty && t < l.n) {
            // a part that starts its item is in the second slot of its block, the others are in the first; 32 parts at a time, a lane each
            for (int base = r0; base <= r1; base += 32) {
                const int here = min(r1 - base + 1, 32);
                auto row_of = [&](int k) { return (int64_t)((2 * (base + k) + (base + k == r0 ? 1 : 0)) * rows_per_tile + r); };
                const float2 ml = lane < here ? *reinterpret_cast<const float2*>(p.part_ml + row_of(lane) * 2) : make_float2(kLowest, 0.f);
                float best = ml.x;
#pragma unroll
                for (int m = 16; m; m >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
                best = fmaxf(best, top);
                const float shrink = fast_exp2(top - best), f = lane < here ? fast_exp2(ml.x - best) : 0.f;
                top = best;
                float add = ml.y * f;
#pragma unroll
                for (int m = 16; m; m >>= 1) add += __shfl_xor_sync(0xffffffffu, add, m);
                all = fmaf(all, shrink, add);
                y = make_float4(y.x * shrink, y.y * shrink, y.z * shrink, y.w * shrink);
#pragma unroll 4
                for (int k = 0; k < here; ++k) {
                    const float fk = __shfl_sync(0xffffffffu, f, k);
                    if (lane < D / 4) {
                        const float4 z = *reinterpret_cast<const float4*>(p.part + row_of(k) * D + 4 * lane);
                        y.x = fmaf(z.x, fk, y.x); y.y = fmaf(z.y, fk, y.y); y.z = fmaf(z.z, fk, y.z); y.w = fmaf(z.w, fk, y.w);
                    }
                }
            }
        }
        const float f = 1.f / all;
        if (lane < D / 4)
            store4(p.o, (int64_t)b * p.so.b + (int64_t)(h * p.G + row - t * p.G) * p.so.h + (int64_t)t * p.so.n + 4 * lane, p.dtype, p.vec_o,
                   all == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
        if (p.lse != nullptr && lane == 0) p.lse[((int64_t)b * p.c.Hkv + h) * p.T * p.G + row] = all == 0.f ? INFINITY : top + log2f(all);
    }
}

// ------------------------------------------------------------------------------------------------ accumulated weights
// Few query rows (one tile): the main kernel has left the scores, 4 bytes a row and slot, and a thread sums a slot's exp2(s - lse).  K is not read
// again, which would be D bytes a slot and all of its products.
constexpr int kSumUnit = kThreads, kSumBlocks = 16;   // blocks an SM: a unit is a chain of two loads, what is beside it hides them
template <bool FOURS>
__global__ void __launch_bounds__(kThreads, kSumBlocks) cache_attn_sum_kernel(const CacheAttnParams p) {
    bool bad = false;
    auto load = [&](int b) {
        Load l = load_of(p, 0, log2_of(kSumUnit), 0, b, bad);
        l.items = l.n > 0 ? p.c.Hkv : 0;
        return l;
    };
    const Range range = take_range<kThreads>(p.s.B, load);
    pdl_wait();
    if (range.left == 0) return;
    int b = range.b;
    int64_t off = range.off;
    Load l = load(b);
    for (int64_t left = range.left; left > 0; --left, ++off) {
        while (off >= (int64_t)l.units * l.items) {
            off -= (int64_t)l.units * l.items;
            l = load(++b);
        }
        const int h = (int)(off / l.units), slot = (int)(off - (int64_t)h * l.units) * kSumUnit + threadIdx.x;
        if (slot >= l.len) continue;
        const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot, bad), rows = l.n * p.G;
        const int64_t bh = (int64_t)b * p.c.Hkv + h;
        const float* s = p.scores + (bh * p.capacity + slot) * p.score_rows;
        const float* lse = p.lse + bh * p.T * p.G;
        float w = 0.f;
        if constexpr (FOURS) {
#pragma unroll 2
            for (int r = 0; r < rows; r += 4) {
                const float4 x = *reinterpret_cast<const float4*>(s + r);
                w += fast_exp2(x.x - lse[r]);
                if (r + 1 < rows) w += fast_exp2(x.y - lse[r + 1]);
                if (r + 2 < rows) w += fast_exp2(x.z - lse[r + 2]);
                if (r + 3 < rows) w += fast_exp2(x.w - lse[r + 3]);
            }
        } else {
            for (int r = 0; r < rows; r += 2) {
                const float2 x = *reinterpret_cast<const float2*>(s + r);
                w += fast_exp2(x.x - lse[r]);
                if (r + 1 < rows) w += fast_exp2(x.y - lse[r + 1]);
            }
        }
        // one addition per slot and call; atomic because sequences may share blocks
        if (page >= 0) atomicAdd(p.c.weight + (((int64_t)page * p.c.Hkv + h) << p.c.bs_log2) + (slot & ((1 << p.c.bs_log2) - 1)), w);
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

// Many rows, or no room for the scores: weight[slot] += sum over rows of exp2(s - lse).  The scores are formed again, K being read once more: the same division into units, but a
// unit's block goes through all tiles of query rows, so that each slot's sum is one addition in a fixed order.
template <int D, int CODE, int NT>
__global__ void __launch_bounds__(kThreads) cache_attn_weight_kernel(const CacheAttnParams p) {
    constexpr int kRows = 8 * NT, kKSteps = D / 16;
    __shared__ __align__(16) uint32_t packed[Shape<D, NT>::kPacked / 4];
    __shared__ float factor[kRows], lse[kRows];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
    bool bad = false;
    auto load = [&](int b) {
        Load l = load_of(p, log2_of(kRows), kUnitLog2, 0, b, bad);
        l.items = l.n > 0 ? p.c.Hkv : 0;
        return l;
    };   // items of this kernel: K / V heads
    const Range range = take_range<kThreads>(p.s.B, load);
    if (range.left == 0) return;
    int b = range.b, had = -1;
    int64_t off = range.off;
    Load l = load(b);
    for (int64_t left = range.left; left > 0; --left, ++off) {
        while (off >= (int64_t)l.units * l.items) {
            off -= (int64_t)l.units * l.items;
            l = load(++b);
            had = -1;
        }
        const int h = (int)(off / l.units), slot0 = (int)(off - (int64_t)h * l.units) * kUnit + warp * kPiece;
        const int page = slot0 < l.len ? cache_page(p.s, p.c.bs_log2, p.c.num_blocks, b, slot0, bad) : -1;
        const int in_block = slot0 & ((1 << p.c.bs_log2) - 1);
        uint32_t k[2][D / 16];
        float k_scale = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 0; w < D / 16; ++w) k[i][w] = 0u;
        if (page >= 0) {
            k_scale = p.c.k_scale[(int64_t)page * p.c.Hkv + h];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (slot0 + g + 8 * i >= l.len) continue;
                const uint8_t* from = p.c.k + (int64_t)page * p.c.sk.b + (int64_t)h * p.c.sk.h + (int64_t)(in_block + g + 8 * i) * p.c.sk.n + c * (D / 4);
                if constexpr (D == 32) {
                    const uint2 u = *reinterpret_cast<const uint2*>(from);
                    k[i][0] = u.x; k[i][1] = u.y;
                } else {
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        const uint4 u = reinterpret_cast<const uint4*>(from)[x];
                        k[i][4 * x] = u.x; k[i][4 * x + 1] = u.y; k[i][4 * x + 2] = u.z; k[i][4 * x + 3] = u.w;
                    }
                }
            }
        }
        float w0 = 0.f, w1 = 0.f;
        const int tiles = (l.n * p.G + kRows - 1) / kRows;
        for (int tile = 0; tile < tiles; ++tile) {
            if (tiles > 1 || had != h) {
                __syncthreads();
                pack_queries<D, NT>(p, b, h, tile * kRows, l.len, l.n, packed, factor, bad);
                for (int r = threadIdx.x; r < kRows; r += kThreads) {
                    const int row = tile * kRows + r;
                    lse[r] = row < l.n * p.G ? p.lse[((int64_t)b * p.c.Hkv + h) * p.T * p.G + row] : INFINITY;
                }
                __syncthreads();
                had = h;
            }
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int w = 0; w < kKSteps; ++w) {
                uint32_t a[4];
                codes_to_half<CODE>(k[0][w], a[0], a[2]);
                codes_to_half<CODE>(k[1][w], a[1], a[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint4 qf = reinterpret_cast<const uint4*>(packed)[(w * NT + nt) * 32 + lane];
                    mma16816(s[nt], a, qf.x, qf.y);
                    mma16816(s[nt], a, qf.z, qf.w);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 8 * nt + 2 * c + i, t = (tile * kRows + r) / p.G;
                    const int sees = t >= l.n ? 0 : p.causal ? l.len - l.n + t + 1 : l.len;
                    const float f = factor[r] * k_scale, z = lse[r];
                    if (slot0 + g < sees) w0 += fast_exp2(fmaf(s[nt][i], f, -z));
                    if (slot0 + g + 8 < sees) w1 += fast_exp2(fmaf(s[nt][i + 2], f, -z));
                }
        }
#pragma unroll
        for (int m = 1; m < 4; m *= 2) {
            w0 += __shfl_xor_sync(0xffffffffu, w0, m);
            w1 += __shfl_xor_sync(0xffffffffu, w1, m);
        }
        // one addition per slot and call; atomic because sequences may share blocks
        if (page >= 0 && c == 0) {
            float* to = p.c.weight + (((int64_t)page * p.c.Hkv + h) << p.c.bs_log2) + in_block;
            if (slot0 + g < l.len) atomicAdd(to + g, w0);
            if (slot0 + g + 8 < l.len) atomicAdd(to + g + 8, w1);
        }
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

// rows of a tile by the number of query rows: 8 (one N extent of the MMA), 16 or 32
constexpr int kClusterUnits = 16;
int row_groups(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }
int resident_blocks(int groups) { return groups == 1 ? 4 : groups == 2 ? 3 : 2; }
// How a call is done and where its workspace's parts lie (the parts of joined sums come first).
struct Layout {
    bool tiles, two_parts, pair;  // tcgen05 kernels; queries in two fp16 parts; two tiles of 128 rows an item
    int groups, row_tiles, rows_per_tile;
    unsigned blocks;
    int parts;                    // blocks of a cluster per item, 0 = ranges of units
    int score_rows;               // numbers a slot in `scores`, 0 = the scores are formed again
    size_t part_ml, lse, scores, images, total;
};
Layout layout_of(int B, int Hkv, int G, int T, int D, int max_blocks, int block_size, int dtype, int accumulate) {
    Layout l{};
    const int rows = G * T;
    const uint64_t slots = (uint64_t)max_blocks * block_size;
    // 16-bit tensors of more than 32 rows a head: products on tcgen05.  This kernel with tiles of 32 rows / tcgen05, us on the GPU, bf16, 32 / 8 heads of
    // 128, sequences x tokens: 36 rows 1 x 300 18.9 / 22.6, 8 x 1024 33.2 / 33.8, 8 x 4096 68 / 52, 64 x 4096 416 / 275; 64 rows 1 x 1024 20.0 / 23.7,
    // 8 x 300 25.5 / 28.7, 64 x 300 103 / 95.5; 256 rows 1 x 300 22.4 / 25.9, 1 x 4096 44 / 34.5, 8 x 1024 89 / 50; 1024 rows 1 x 300 35.7 / 34.4,
    // 8 x 4096 866 / 236.  With weights 64 rows 8 x 1024 80 / 56.5.  So calls of little work lose up to 5 us by the rule: what they would take depends on
    // lengths that the host does not know.  fp32 tensors stay with the kernel that splits P as well.
    l.tiles = dtype != COROPE_DTYPE_F32 && rows > 32;
    // one part of q is off by 2^-12 of it: next to a bf16 result's 2^-9 that is nothing, an fp16 result or a weight would feel it
    l.two_parts = l.tiles && (dtype == COROPE_DTYPE_F16 || accumulate);
    l.pair = l.tiles && cache_tile_pairs(rows, D, l.two_parts);
    l.groups = row_groups(rows);
    l.rows_per_tile = l.tiles ? kTileRows * (l.pair ? 2 : 1) : 8 * l.groups;
    l.row_tiles = (rows + l.rows_per_tile - 1) / l.rows_per_tile;
    const uint64_t items = (uint64_t)B * Hkv * l.row_tiles, unit = l.tiles ? kTileRows : kUnit;
    const uint64_t item_units = (slots + unit - 1) / unit, units = items * (item_units + (l.tiles ? kTileItemCost : item_cost(l.groups))), most = (uint64_t)sm_count() * (l.tiles ? 1 : resident_blocks(l.groups));
    l.blocks = (unsigned)(units < most ? units : most);
    // Room for the scores of every slot that the block tables could hold.  Beyond half a gigabyte (long tables that the sequences may not fill) K is
    // read again instead: 32 sequences of up to 8192 tokens, 4 rows a head, take 80 us with the scores, 137 without.
    const size_t score_bytes = (size_t)B * Hkv * slots * ((rows + 1) / 2 * 2) * 4;
    l.score_rows = accumulate && !l.tiles && l.row_tiles == 1 && score_bytes <= (512u << 20) ? (rows + 1) / 2 * 2 : 0;
    // A cluster per item where all of them are resident at once and no block has more than kClusterUnits units of the longest sequence there can be:
    // the sequences' own lengths are not known here, so the longest sets the pace.  Ranges and a joining kernel / clusters, us, 32 / 8 heads of 128: 1 x
    // 777 tokens 11.5 / 8.5, 1 x 4096 27.2 / 11.5, 16 x 1024 17.3 / 13.6, 16 x up to 4096 24.2 / 25.9, 64 x up to 1024 26.5 / 24.7.
    if (!l.tiles && items <= most && (!accumulate || l.score_rows)) {
        l.parts = 1;
        while (l.parts < 8 && items * l.parts * 2 <= most && item_units >= (uint64_t)l.parts * 2) l.parts *= 2;
        if (item_units > (uint64_t)l.parts * kClusterUnits) l.parts = 0;
        else l.blocks = (unsigned)(items * l.parts);
    }
    const size_t part_rows = l.parts ? 0 : (size_t)2 * l.blocks * l.rows_per_tile;
    l.part_ml = align_up(part_rows * D * 4, 256);
    l.lse = l.part_ml + align_up(part_rows * 8, 256);
    l.scores = l.lse + (accumulate ? align_up((size_t)B * Hkv * rows * 4, 256) : 0);
    l.images = l.scores + (l.score_rows ? align_up(score_bytes, 256) : 0);
    l.total = l.images + (l.tiles ? cache_tile_workspace_bytes(B, Hkv, l.row_tiles * (l.pair ? 2 : 1), D, l.two_parts) : 0);
    if (l.total < 256) l.total = 256;
    return l;
}

template <int D>
int launch_join(const CacheAttnParams& p, const Layout& l, int unit_log2, int extra, cudaStream_t s) {
    count_launch();
    return launch_dependent(cache_attn_join_kernel<D>, (unsigned)(p.s.B * p.c.Hkv * p.row_tiles * (l.rows_per_tile / 8)), kJoinThreads, 0, s, p, log2_of(l.rows_per_tile), unit_log2, extra, (int)l.blocks);
}
template <int D, int CODE, int NT, bool EXACT_P>
int launch_main(const CacheAttnParams& p, unsigned blocks, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (int e = allow_smem(cache_attn_kernel<D, CODE, NT, EXACT_P>, Shape<D, NT>::kSmem, done)) return e;
    count_launch();
    if (p.parts == 0) {
        cache_attn_kernel<D, CODE, NT, EXACT_P><<<blocks, kThreads, Shape<D, NT>::kSmem, s>>>(p);
        return (int)cudaGetLastError();
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<D, NT>::kSmem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, cache_attn_kernel<D, CODE, NT, EXACT_P>, p);
}
template <int D, int CODE, int NT>
int launch_rows(const CacheAttnParams& p, const Layout& l, cudaStream_t s) {
    if (int e = p.dtype == COROPE_DTYPE_F32 ? launch_main<D, CODE, NT, true>(p, l.blocks, s) : launch_main<D, CODE, NT, false>(p, l.blocks, s)) return e;
    if (l.parts) return COROPE_OK;
    if (int e = launch_join<D>(p, l, kUnitLog2, item_cost(NT), s)) return e;
    if (!p.accumulate) return COROPE_OK;
    count_launch();
    const int unit = p.scores != nullptr ? kSumUnit : kUnit;
    const uint64_t units = (uint64_t)p.s.B * p.c.Hkv * ((uint64_t)(p.capacity + unit - 1) / unit), most = (uint64_t)sm_count() * (p.scores != nullptr ? kSumBlocks : 8);
    const unsigned grid = (unsigned)(units < most ? units : most);
    if (p.scores != nullptr) return launch_dependent(p.score_rows % 4 == 0 ? cache_attn_sum_kernel<true> : cache_attn_sum_kernel<false>, grid, kThreads, 0, s, p);
    cache_attn_weight_kernel<D, CODE, NT><<<grid, kThreads, 0, s>>>(p);
    return (int)cudaGetLastError();
}
template <int D, int CODE>
int by_rows(const CacheAttnParams& p, const Layout& l, cudaStream_t s) {
    return l.groups == 1 ? launch_rows<D, CODE, 1>(p, l, s) : l.groups == 2 ? launch_rows<D, CODE, 2>(p, l, s) : launch_rows<D, CODE, 4>(p, l, s);
}
template <int D>
int by_kernel(const CacheAttnParams& p, const Layout& l, void* images, cudaStream_t s) {
    if (!l.tiles) return p.code == COROPE_CODE_E4M3 ? by_rows<D, COROPE_CODE_E4M3>(p, l, s) : by_rows<D, COROPE_CODE_INT8>(p, l, s);
    if (int e = launch_cache_attn_tiles(p, images, l.two_parts, l.pair, l.blocks, s)) return e;
    if (int e = launch_join<D>(p, l, log2_of(kTileRows), kTileItemCost, s)) return e;
    return p.accumulate ? launch_cache_weight_tiles(p, images, l.pair, s) : COROPE_OK;
}

}  // namespace

size_t cache_attn_workspace_bytes(int B, int Hkv, int G, int T, int D, int max_blocks, int block_size, int dtype, int accumulate) {
    return layout_of(B, Hkv, G, T, D, max_blocks, block_size, dtype, accumulate).total;
}

int launch_cache_attn(CacheAttnParams p, void* ws, cudaStream_t s) {
    const Layout l = layout_of(p.s.B, p.c.Hkv, p.G, p.T, p.D, p.s.max_blocks, 1 << p.c.bs_log2, p.dtype, p.accumulate);
    auto part = [&](size_t at) { return reinterpret_cast<float*>(static_cast<char*>(ws) + at); };
    p.row_tiles = l.row_tiles;
    p.parts = l.parts;
    p.part = part(0);
    p.part_ml = part(l.part_ml);
    p.lse = p.accumulate ? part(l.lse) : nullptr;
    p.capacity = p.s.max_blocks << p.c.bs_log2;
    p.score_rows = l.score_rows;
    p.scores = l.score_rows ? part(l.scores) : nullptr;
    p.vec_o = rows_in_fours(p.o, p.so, p.dtype);
    p.rows_packed = p.c.sk.n == p.D && p.c.sv.n == p.D;
    void* images = part(l.images);
    return p.D == 128 ? by_kernel<128>(p, l, images, s) : p.D == 64 ? by_kernel<64>(p, l, images, s) : by_kernel<32>(p, l, images, s);
}

}  // namespace corope
