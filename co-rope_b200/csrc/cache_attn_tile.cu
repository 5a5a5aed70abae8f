// corope_cache_attn for many query rows a K / V head (R = G * T > 32, 16-bit types): tcgen05 MMAs on codes turned into fp16 in shared memory.
//
// A unit of work is 128 query rows by 128 slots; a block per SM takes a contiguous range of a batch's units (see cache_attn.cuh) and walks it
// piece by piece, a piece being units of one tile of rows (a long share of an item is several pieces, see most_units).  Warp roles (896 threads, registers divided again with setmaxnreg):
//   warp 0        brings the query tile of an item's first piece (an image of its place in shared memory that a pre-pass has written) with bulk copies
//   warp 2        MMA issuer and TMEM owner
//   warp 3        scout: walks the range ahead of the others and tells them the pieces, and of each unit the addresses of its codes and their scales
//   warps 4-7     K: 16 codes a lane and step turned into fp16 (exact) and stored as the MMA wants them;  warps 8-11: V likewise
//   warps 12-19   softmax of the even units of a piece, two threads a row (64 slots each);  warps 20-27: of the odd ones
// TMEM: S0 [0,128) S1 [128,256) O0 [256,384) O1 [384,512); P (fp16) goes over S.  Even and odd units have sums of their own, so one group's
// exponentials run beside the other's MMAs, and are joined when the piece is written.
// With more than 128 rows a head (PAIR) an item is two tiles of rows, a group to each: K and V are turned into operands once for both, which halves
// that work and the reads from L2.  Not for D = 128 with two parts, whose four query tiles leave no room for two stages of K and V.
// Scales: a block of 16 slots or more has one scale of K, which multiplies the scores of its columns in fp32, and one of V, which enters the
// exponent: P = exp2(s + log2 v_scale - M), and its sum is taken back to probabilities by the same number.
// Queries are scaled by a power of two per row and rounded to fp16 (11 bits); with two parts (fp16 tensors, and where weights are gathered) the
// remainder of the rounding is a second operand and scores have 22 bits.
// Bound by the chain scores ready -> exponentials -> P ready -> P V and the next Q K^T of a tile, as P stands over S: a unit of 256 x 128 takes 5300 cycles,
// of which the exponentials (16 a clock and SM) and the MMAs have 2048 each (XU and tensor pipe at 37 %, 1024 queries over 9001 tokens).
#include <cstddef>

#include "cache_attn.cuh"

namespace corope {
namespace {

constexpr int kN = kTileRows;
constexpr int kThreads = 896;
constexpr int kMmaWarp = 2, kConvWarp0 = 4, kSmxWarp0 = 12;
constexpr int kLaunchRegs = 72, kRegsCtl = 40, kRegsConv = 56, kRegsSmx = 88;
static_assert(128 * (kRegsCtl + 2 * kRegsConv + 4 * kRegsSmx) <= kThreads * kLaunchRegs, "register budget");
constexpr int kStages = 2;                    // of K and of V
constexpr int kUnitSlots = 8, kPieceSlots = 4;   // what the scout has told and is kept
constexpr int kFlagSlots = 8;                 // pieces whose flag is kept

enum Bar { Q_FULL = 0, Q_EMPTY, K_FULL, K_EMPTY = K_FULL + kStages, V_FULL = K_EMPTY + kStages, V_EMPTY = V_FULL + kStages, S_FULL = V_EMPTY + kStages,
           P_FULL = S_FULL + 2, O_FULL = P_FULL + 2, O_FREE = O_FULL + 2, UNIT_FULL = O_FREE + 1, UNIT_EMPTY = UNIT_FULL + kUnitSlots,
           PIECE_FULL = UNIT_EMPTY + kUnitSlots, PIECE_EMPTY = PIECE_FULL + kPieceSlots, NUM_BARS = PIECE_EMPTY + kPieceSlots };

// shared memory of head dimension D (32 is widened to 64 with zeros)
__host__ __device__ constexpr int wide(int D) { return D == 128 ? 128 : 64; }
__host__ __device__ constexpr size_t tile_bytes(int D) { return (size_t)kN * wide(D) * 2; }
// A unit's 16-slot groups: where their rows begin, how many there are (0: the block is not there, or has no values), their scales.
struct alignas(16) UnitNote {   // its floats are read four at a time
    uint64_t k[8], v[8];
    float k_scale[8], lift[8], drop[8];
    int k_rows[8], v_rows[8];
    int piece;       // number of its piece among those with units, -1: there is no unit any more
    int hidden;      // some row of the tile does not see some slot
    int full;        // every group has 16 rows, of K and of V
    int pad;
};
static_assert(sizeof(UnitNote) % 16 == 0 && offsetof(UnitNote, k_scale) % 16 == 0 && offsetof(UnitNote, lift) % 16 == 0 && offsetof(UnitNote, drop) % 16 == 0, "");
// A piece: units [u0, u0 + count) of the item.  b < 0: there is none any more.
struct PieceNote {
    int b, h, tile, u0, count, len, n, whole;
    int seen;           // slots below this are seen by every row
    int share0;         // the block's first unit of the item
    int carried, more;  // the sums of the block's earlier units of the item wait in its part; units are still to come
};
// Units of a piece at most: tensor cores truncate where they add to their sums (see the kernel for few rows), 8 steps a unit, so longer shares of an item are
// added piece by piece in fp32.  With one sum for 2^17 / 2^20 slots fp16 results came out 8e-4 / 8e-3 too small.  (Without PAIR a piece has two sums.)
__host__ __device__ constexpr int most_units(bool pair) { return pair ? 128 : 256; }
struct alignas(16) Small {
    UnitNote units[kUnitSlots];
    PieceNote pieces[kPieceSlots];
    float half_max[2][2][kN];                 // exchanged between the two threads of a row
    float end_max[2][kN], end_sum[2][2][kN];  // [group][half]
    uint64_t bars[NUM_BARS];
    int left;                                 // the softmax warps leave
    int nan_v[kFlagSlots];                    // a piece has NaN in V where some rows must not see it
    uint32_t tmem;
    int abort;
};
constexpr size_t queue_bytes(int D, bool two, bool pair) { return (size_t)(D == 128 && (two || pair) ? 4 : D / 16) * 16 * 128; }   // of codes on their way, per group
constexpr size_t smem_bytes(int D, bool two, bool pair) {
    return ((two ? 2 : 1) * (pair ? 2 : 1) + 2 * kStages) * tile_bytes(D) + 2 * queue_bytes(D, two, pair) + sizeof(Small) + 1024;
}
static_assert(smem_bytes(128, true, false) <= 232448 - 128 && smem_bytes(128, false, false) <= 232448 - 128 && smem_bytes(128, false, true) <= 232448 - 128, "shared memory budget");   // (and take_range's)

// byte offset of 16-byte run `run` (8 elements) of row r in the image of a tile: boxes of 64 columns, 128-byte swizzle
__device__ __forceinline__ uint32_t image_at(int r, int run) { return (uint32_t)((run >> 3) * (kN * 128) + r * 128 + (((run & 7) ^ (r & 7)) << 4)); }

__device__ __forceinline__ void store16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ------------------------------------------------------------------------------------------------ queries
// Rotates, scales and rounds the rows, and writes them as images of their tiles: a warp per row, 16 blocks per tile.
constexpr int kPackWarps = 8, kPackBlocks = kN / kPackWarps;
template <int D, bool TWO>
__global__ void __launch_bounds__(kPackWarps * 32) cache_pack_kernel(const CacheAttnParams p, int image_tiles, uint8_t* images, float* factors) {
    constexpr int kHalf = D / 2, kPairs = kHalf / 2;
    const unsigned item = blockIdx.x / (unsigned)kPackBlocks;
    const int tile = (int)(item % (unsigned)image_tiles), bh = (int)(item / (unsigned)image_tiles), b = bh / p.c.Hkv, h = bh - b * p.c.Hkv;
    const int lane = threadIdx.x % 32, r = (int)(blockIdx.x - item * kPackBlocks) * kPackWarps + (int)threadIdx.x / 32;
    bool bad = false;
    const int len = cache_len(p.s, p.c.bs_log2, b, bad), n = cache_new(p.s, p.T, b, bad);
    uint8_t* image = images + (size_t)item * (TWO ? 2 : 1) * tile_bytes(D);
    {
        const int row = tile * kN + r, t = row / p.G;
        float x[4] = {0.f, 0.f, 0.f, 0.f};   // columns 2 lane, + 1, and their partners D / 2 further on
        if (t < n && sees_something(p, len, n, t) && lane < kPairs) {
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
        if (lane == 0) factors[(size_t)item * kN + r] = down * p.scale;
        if (lane < kPairs) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 2 * lane + i * kHalf;
                const uint32_t at = image_at(r, d / 8) + d % 8 * 2;
                const float u = x[2 * i] * up, v = x[2 * i + 1] * up;
                const uint32_t hi = pack_half2(u, v);
                *reinterpret_cast<uint32_t*>(image + at) = hi;
                if (TWO) {
                    const float2 back = unpack_half2(hi);
                    *reinterpret_cast<uint32_t*>(image + tile_bytes(D) + at) = pack_half2(u - back.x, v - back.y);
                }
            }
        }
        if (D == 32 && lane < 16) {   // columns 32 .. 63
            const uint32_t at = image_at(r, 4 + lane / 4) + lane % 4 * 4;
            *reinterpret_cast<uint32_t*>(image + at) = 0u;
            if (TWO) *reinterpret_cast<uint32_t*>(image + tile_bytes(D) + at) = 0u;
        }
    }
    if (bad) report_bad_index(p.status, p.mirror);
}

// ------------------------------------------------------------------------------------------------ codes to operands
// A group of 128 threads turns a unit's 128 slots into an operand in kSteps steps, 16 codes a thread and step.  The codes wait in a queue in
// shared memory of the thread's own (cp.async brings them, nobody else reads them), kDepth steps ahead.
template <int D, bool TWO, bool PAIR>
struct Steps {
    static constexpr int kLanes = D / 16, kRowsPerStep = 128 / kLanes, kSteps = kN / kRowsPerStep;
    static constexpr int kDepth = D == 128 && (TWO || PAIR) ? 4 : kSteps;
    static constexpr int kAtOnce = kDepth >= 8 ? 4 : 2;     // steps whose loads are under way together
    static constexpr int kQueueBytes = kDepth * 16 * 128;   // of one group
};
// the block of slots 16 lane .. of unit u, lane < 8, or -1
template <typename X>
__device__ __forceinline__ int unit_page(const CacheAttnParams& p, const X& x, int u, int lane, bool& bad) {
    const int slot = u * kN + 16 * lane;
    return lane < 8 && slot < x.len ? cache_page(p.s, p.c.bs_log2, p.c.num_blocks, x.b, slot, bad) : -1;
}
__device__ __forceinline__ void copy_codes(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy_codes(uint32_t to, const void* from, bool real) {   // zeros where not real
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint2 load8(uint32_t at) {
    uint2 w;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(at));
    return w;
}
__device__ __forceinline__ bool has_nan(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w & ~__vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// Eight codes to a run of the image of a tile.  A thread's 16 codes make two runs of a row; eight lanes that store at one time have to reach eight
// different runs of a 128-byte line, so at D = 128 the lanes of the second box begin with their second run (`swap`).
template <int CODE>
__device__ __forceinline__ void store_codes(const uint2& w, uint32_t at) {
    uint32_t h[4];
    codes_to_half<CODE>(w.x, h[0], h[1]);
    codes_to_half<CODE>(w.y, h[2], h[3]);
    store16(at, h[0], h[1], h[2], h[3]);
}

// ------------------------------------------------------------------------------------------------ main kernel
template <int D, int CODE, bool TWO, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) cache_attn_tile_kernel(const CacheAttnParams p, const uint8_t* images, const float* factors) {
    using S = Steps<D, TWO, PAIR>;
    constexpr int kD = wide(D), kBox = kN * 128, kParts = TWO ? 2 : 1, kQTiles = PAIR ? 2 : 1, kItemRows = kQTiles * kN;
    constexpr uint32_t kTile = (uint32_t)tile_bytes(D);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = sm;
    uint8_t* sK = sQ + kQTiles * kParts * kTile;   // (queries: [tile][part])
    uint8_t* sV = sK + kStages * kTile;
    uint8_t* queues = sV + kStages * kTile;
    Small& z = *reinterpret_cast<Small*>(queues + 2 * S::kQueueBytes);
    uint64_t* bars = z.bars;
    volatile int* abort_flag = &z.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    bool bad = false;
    const Range range = take_range<128>(p.s.B, [&](int b) { return load_of(p, log2_of(kItemRows), log2_of(kN), kTileItemCost, b, bad); });
    pdl_trigger();
    if (bad) report_bad_index(p.status, p.mirror);
    // after a wait that ran out, in this launch's block or in an earlier launch, none starts anew until the host has seen it
    const bool gave_up = p.status != nullptr && (*reinterpret_cast<volatile int*>(p.status) & COROPE_DEV_WAIT_EXPIRED);
    if (__syncthreads_or(gave_up) || range.left == 0) {
        if (threadIdx.x == 0 && gave_up) report_to_mirror(p.status, p.mirror);
        pdl_wait();   // no launch ends before the one in front of it
        return;
    }
    if (threadIdx.x == 0) {
        z.abort = z.left = 0;
        for (int i = 0; i < kFlagSlots; ++i) z.nan_v[i] = 0;
        mbar_init(&bars[Q_FULL], 1);
        mbar_init(&bars[Q_EMPTY], 1);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bars[K_FULL + i], 4);
            mbar_init(&bars[K_EMPTY + i], 1);
            mbar_init(&bars[V_FULL + i], 4);
            mbar_init(&bars[V_EMPTY + i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[S_FULL + i], 1);
            mbar_init(&bars[P_FULL + i], 8);
            mbar_init(&bars[O_FULL + i], 1);
        }
        mbar_init(&bars[O_FREE], 16);
        for (int i = 0; i < kUnitSlots; ++i) {
            mbar_init(&bars[UNIT_FULL + i], 1);
            mbar_init(&bars[UNIT_EMPTY + i], 8);         // K and V warps
        }
        for (int i = 0; i < kPieceSlots; ++i) {
            mbar_init(&bars[PIECE_FULL + i], 1);
            mbar_init(&bars[PIECE_EMPTY + i], 1 + 1 + 16);   // query loader, MMA issuer, softmax warps
        }
        fence_mbar_init();
    }
    if (D == 32)   // columns 32 .. 63 of K and V are never written
        for (int i = threadIdx.x; i < (int)(2 * kStages * kTile / 16); i += kThreads) reinterpret_cast<uint4*>(sK)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
    __syncthreads();
    if (warp == kMmaWarp) {
        tmem_alloc(&z.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = z.tmem;

    if (warp < kConvWarp0) {
        reg_dealloc<kRegsCtl>();
        if (warp == 0) {
            // -------------------------------------------------------------- query tiles
            if (lane == 0) {
                pdl_wait();
                int n = 0;
                for (int k = 0;; ++k) {
                    const int slot = k % kPieceSlots;
                    if (!mbar_wait(&bars[PIECE_FULL + slot], (k / kPieceSlots) & 1, p.status, PIECE_FULL, abort_flag)) break;
                    const PieceNote& x = z.pieces[slot];
                    if (x.b < 0) break;
                    const int64_t item = (int64_t)(x.b * p.c.Hkv + x.h) * p.row_tiles + x.tile;
                    const bool some = x.count > 0 && !x.carried;   // (the tile of a piece that goes on is there)
                    mbar_arrive(&bars[PIECE_EMPTY + slot]);
                    if (!some) continue;
                    if (n > 0 && !mbar_wait(&bars[Q_EMPTY], (n - 1) & 1, p.status, Q_EMPTY, abort_flag)) break;
                    mbar_arrive_expect_tx(&bars[Q_FULL], kQTiles * kParts * kTile);
                    for (int i = 0; i < kQTiles * kParts; ++i)
                        bulk_load_1d(sQ + i * kTile, images + ((size_t)item * (kQTiles * kParts) + i) * kTile, kTile, &bars[Q_FULL]);
                    ++n;
                }
            }
            __syncwarp();
        } else if (warp == kMmaWarp) {
            // -------------------------------------------------------------- MMA issuer
            const bool leader = elect_one();
            const uint32_t idesc_qk = make_idesc(0, 0, 0, 0, kN, kN), idesc_pv = make_idesc(0, 0, 0, 1, kN, kD);
            constexpr uint32_t kHi = sdesc_hi(1024);
            const uint32_t q_lo = sdesc_lo(smem_u32(sQ), 0), k_lo = sdesc_lo(smem_u32(sK), 0), v_lo = sdesc_lo(smem_u32(sV), kBox);
            auto issue_qk = [&](int i, int stage) {
                const uint32_t b0 = k_lo + stage * (kTile >> 4), d = tmem + i * 128;
#pragma unroll
                for (int part = 0; part < kParts; ++part)
#pragma unroll
                    for (int kk = 0; kk < kD / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
                        // the second part first: its sum is small, and so are its truncations
                        if (leader) umma_ss2(d, q_lo + ((PAIR ? i * kParts : 0) + kParts - 1 - part) * (kTile >> 4) + off, kHi, b0 + off, kHi, idesc_qk, part + kk > 0);
                    }
            };
            auto issue_pv = [&](int i, int stage, bool add) {
                const uint32_t b0 = v_lo + stage * (kTile >> 4), d = tmem + 256 + i * 128, a = tmem + i * 128;
#pragma unroll
                for (int kk = 0; kk < kN / 16; ++kk)
                    if (leader) umma_ts2(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b0 + kk * (2048 >> 4), kHi, idesc_pv, (add || kk > 0) ? 1u : 0u);
            };
            int gk = 0, gv = 0, pieces = 0, query_tiles = 0, done0 = 0, done1 = 0;
            bool ok = true;
            for (int k = 0; ok; ++k) {
                const int slot = k % kPieceSlots;
                if (!(ok = mbar_wait_warp(&bars[PIECE_FULL + slot], (k / kPieceSlots) & 1, p.status, PIECE_FULL, abort_flag))) break;
                const int count = z.pieces[slot].b < 0 ? -1 : z.pieces[slot].count;
                const bool new_tile = !z.pieces[slot].carried, last_use = !z.pieces[slot].more;
                mbar_arrive_warp(&bars[PIECE_EMPTY + slot], lane);
                if (count < 0) break;
                if (count == 0) continue;
                if (new_tile && !(ok = mbar_wait_warp(&bars[Q_FULL], query_tiles++ & 1, p.status, Q_FULL, abort_flag))) break;
                if constexpr (PAIR) {
                    // PV0(j) QK0(j + 1) | PV1(j) QK1(j + 1); j = -1 forms the scores of unit 0
                    for (int j = -1; ok && j < count; ++j) {
                        const bool have_next = j + 1 < count;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (j >= 0) {
                                const int stage = gv % kStages;
                                if (i == 0 && !(ok = mbar_wait_warp(&bars[V_FULL + stage], (gv / kStages) & 1, p.status, V_FULL, abort_flag))) break;
                                if (!(ok = mbar_wait_warp(&bars[P_FULL + i], (i ? done1 : done0) & 1, p.status, P_FULL, abort_flag))) break;
                                if (i == 0 && j == 0 && pieces > 0 && !(ok = mbar_wait_warp(&bars[O_FREE], (pieces - 1) & 1, p.status, O_FREE, abort_flag))) break;
                                tc_fence_after();
                                issue_pv(i, stage, j > 0);
                                if (leader) umma_commit(&bars[O_FULL + i]);
                                if (i == 0) {
                                    ++done0;
                                } else {
                                    if (leader) umma_commit(&bars[V_EMPTY + stage]);
                                    ++done1;
                                    ++gv;
                                }
                            }
                            if (have_next) {
                                const int stage = gk % kStages;
                                if (i == 0 && !(ok = mbar_wait_warp(&bars[K_FULL + stage], (gk / kStages) & 1, p.status, K_FULL, abort_flag))) break;
                                tc_fence_after();
                                issue_qk(i, stage);
                                if (leader) umma_commit(&bars[S_FULL + i]);
                                if (i == 1) {
                                    if (leader) umma_commit(&bars[K_EMPTY + stage]);
                                    if (j + 2 == count && last_use && leader) umma_commit(&bars[Q_EMPTY]);
                                    ++gk;
                                }
                            }
                        }
                    }
                } else {
                    auto next_scores = [&](int j) {   // Q K^T of the piece's unit j
                        if (!(ok = mbar_wait_warp(&bars[K_FULL + gk % kStages], (gk / kStages) & 1, p.status, K_FULL, abort_flag))) return;
                        tc_fence_after();
                        issue_qk(j & 1, gk % kStages);
                        if (leader) {
                            umma_commit(&bars[S_FULL + (j & 1)]);
                            umma_commit(&bars[K_EMPTY + gk % kStages]);
                            if (j + 1 == count && last_use) umma_commit(&bars[Q_EMPTY]);
                        }
                        ++gk;
                    };
                    next_scores(0);
                    if (ok && count > 1) next_scores(1);
                    for (int j = 0; ok && j < count; ++j) {
                        const int i = j & 1, stage = gv % kStages;
                        if (!(ok = mbar_wait_warp(&bars[V_FULL + stage], (gv / kStages) & 1, p.status, V_FULL, abort_flag))) break;
                        if (!(ok = mbar_wait_warp(&bars[P_FULL + i], (i ? done1 : done0) & 1, p.status, P_FULL, abort_flag))) break;
                        if (j == 0 && pieces > 0 && !(ok = mbar_wait_warp(&bars[O_FREE], (pieces - 1) & 1, p.status, O_FREE, abort_flag))) break;
                        tc_fence_after();
                        issue_pv(i, stage, j > 1);
                        if (leader) {
                            umma_commit(&bars[O_FULL + i]);
                            umma_commit(&bars[V_EMPTY + stage]);
                        }
                        if (i) ++done1;
                        else ++done0;
                        ++gv;
                        if (j + 2 < count) next_scores(j + 2);
                    }
                }
                ++pieces;
            }
            __syncwarp();
        } else if (warp == 3) {
            // -------------------------------------------------------------- scout
            // A unit is finished by its converters when the next one has been told, and a piece by the softmax warps when its last unit has.  So the note of
            // a piece's first unit must not wait for the end of the piece before: no more pieces without units may follow one another than notes
            // are kept.  There is one at most, the first of the range (the end of an item whose rows see none of the last slots): a tile of rows that
            // sees nothing is no item, and every item's first unit is seen by some row.
            Range r = range;
            Load l = load_of(p, log2_of(kItemRows), log2_of(kN), kTileItemCost, r.b, bad);
            int q = 0, told = 0, pieces = 0;   // units, pieces, pieces with units so far
            int share0 = 0, carried = 0;
            bool ok = true;
            const int bs_mask = (1 << p.c.bs_log2) - 1;
            // A note may be written over when the converters are through with a unit three later than its own: then its product is issued, and the
            // exponentials of the note's unit are done.
            auto unit_slot_free = [&]() {
                return q < kUnitSlots || mbar_wait_warp(&bars[UNIT_EMPTY + (q + 3) % kUnitSlots], ((q - kUnitSlots + 3) / kUnitSlots) & 1, p.status, UNIT_EMPTY, abort_flag);
            };
            while (ok) {
                const int slot = told % kPieceSlots;
                if (told >= kPieceSlots && !(ok = mbar_wait_warp(&bars[PIECE_EMPTY + slot], ((told / kPieceSlots) - 1) & 1, p.status, PIECE_EMPTY, abort_flag))) break;
                PieceNote x{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                while (r.left > 0 && x.b < 0) {
                    while (r.off >= (int64_t)l.cost * l.items) {
                        r.off -= (int64_t)l.cost * l.items;
                        l = load_of(p, log2_of(kItemRows), log2_of(kN), kTileItemCost, ++r.b, bad);
                    }
                    const int item = (int)(r.off / l.cost), tiles = l.items / p.c.Hkv;
                    x.h = item / tiles; x.tile = item - x.h * tiles + first_tile(p, log2_of(kItemRows), l.len, l.n); x.len = l.len; x.n = l.n;
                    const int last = min(l.n - 1, (x.tile * kItemRows + kItemRows - 1) / p.G);   // the item's last query
                    const int most = p.causal ? max(l.len - l.n + last + 1, 0) : l.len;   // slots that some row sees
                    const int seen_units = (most + kN - 1) / kN;
                    const int at = (int)(r.off - (int64_t)item * l.cost), end = (int)min((int64_t)l.cost, at + r.left);
                    int stop = min(end, max(at, kTileItemCost) + most_units(PAIR));
                    if (stop - kTileItemCost >= seen_units) stop = end;   // the rest is hidden from all rows: no piece of its own
                    r.off += stop - at;
                    r.left -= stop - at;
                    const int u1 = stop - kTileItemCost;
                    if (u1 <= 0) continue;   // the range ends before the item's first unit
                    x.b = r.b;
                    x.u0 = max(at - kTileItemCost, 0);
                    x.count = max(min(seen_units, u1) - x.u0, 0);
                    x.carried = carried;
                    x.more = carried = stop < end;
                    if (!x.carried) share0 = x.u0;
                    x.share0 = share0;
                    x.whole = share0 == 0 && u1 == l.units;
                    x.seen = p.causal ? max(l.len - l.n + x.tile * kItemRows / p.G + 1, 0) : l.len;
                }
                if (lane == 0) z.pieces[slot] = x;
                mbar_arrive_warp(&bars[PIECE_FULL + slot], lane);
                ++told;
                if (x.b < 0) break;
                for (int u = x.u0; u < x.u0 + x.count; ++u, ++q) {
                    if (!(ok = unit_slot_free())) break;
                    UnitNote& note = z.units[q % kUnitSlots];
                    const int page = unit_page(p, x, u, lane, bad);
                    if (lane < 8) {
                        const int slot0 = u * kN + 16 * lane, rows = page >= 0 ? min(x.len - slot0, 16) : 0;
                        const int64_t at = (int64_t)max(page, 0) * p.c.Hkv + x.h, row = slot0 & bs_mask;
                        const float ks = p.c.k_scale[at], vs = p.c.v_scale[at], size = no_values(vs) ? 1.f : vs;
                        note.k[lane] = (uint64_t)(p.c.k + (int64_t)max(page, 0) * p.c.sk.b + (int64_t)x.h * p.c.sk.h + row * p.c.sk.n);
                        note.v[lane] = (uint64_t)(p.c.v + (int64_t)max(page, 0) * p.c.sv.b + (int64_t)x.h * p.c.sv.h + row * p.c.sv.n);
                        note.k_rows[lane] = rows;
                        note.v_rows[lane] = no_values(vs) ? 0 : rows;                // zeros, whatever the codes are
                        note.k_scale[lane] = page >= 0 ? ks : 0.f;
                        note.lift[lane] = page >= 0 ? __log2f(size) : -INFINITY;     // slots of a block that is not there count nothing
                        note.drop[lane] = 1.f / size;
                        const bool full = __all_sync(0xffu, rows == 16 && !no_values(vs));
                        if (lane == 0) note.piece = pieces, note.hidden = (u + 1) * kN > x.seen, note.full = full;
                    }
                    mbar_arrive_warp(&bars[UNIT_FULL + q % kUnitSlots], lane);
                }
                pieces += x.count > 0;
            }
            if (ok && unit_slot_free()) {
                if (lane == 0) z.units[q % kUnitSlots].piece = -1;
                mbar_arrive_warp(&bars[UNIT_FULL + q % kUnitSlots], lane);
            }
            if (bad) report_bad_index(p.status, p.mirror);
        }
    } else if (warp < kSmxWarp0) {
        // ------------------------------------------------------------------ K and V: codes to fp16 operands
        if constexpr (kRegsConv < kLaunchRegs) reg_dealloc<kRegsConv>();
        const bool is_v = warp >= kConvWarp0 + 4;
        const int tid = (threadIdx.x - kConvWarp0 * 32) & 127;
        const uint32_t tiles = smem_u32(is_v ? sV : sK);
        const int full = is_v ? V_FULL : K_FULL, empty = is_v ? V_EMPTY : K_EMPTY;
        const int col = tid % S::kLanes * 16, row0 = tid / S::kLanes, row_in_group = row0 & 15;
        const int64_t row_offset = (int64_t)row_in_group * (is_v ? p.c.sv.n : p.c.sk.n) + col;
        const uint32_t queue = smem_u32(queues) + (is_v ? S::kQueueBytes : 0) + tid * 16;   // step k at queue + k * 2048
        // rows row0 + kRowsPerStep k: the same row of a swizzle atom in every step, where steps are multiples of 8 rows
        static_assert(S::kRowsPerStep % 16 == 0, "");
        const int run = col / 8, swap = D == 128 ? run >> 3 : 0;
        const uint32_t first_at = (run >> 3) * kBox + row0 * 128 + ((((run & 7) ^ (row0 & 7)) ^ swap) << 4), second_at = first_at ^ 16;
        const uint32_t first_from = queue + swap * 8, second_from = queue + (1 - swap) * 8;
        auto copy = [&](const UnitNote& note, int step, int place) {
            const int group = (step * S::kRowsPerStep + row0) >> 4;
            const uint8_t* from = reinterpret_cast<const uint8_t*>(is_v ? note.v[group] : note.k[group]);
            if (note.full) {
                copy_codes(queue + place * 2048, from + row_offset);
            } else {
                const bool real = row_in_group < (is_v ? note.v_rows[group] : note.k_rows[group]);
                copy_codes(queue + place * 2048, real ? from + row_offset : from, real);
            }
        };
        auto wait_note = [&](int q) { return mbar_wait_warp(&bars[UNIT_FULL + q % kUnitSlots], (q / kUnitSlots) & 1, p.status, UNIT_FULL, abort_flag); };
        bool more = wait_note(0) && z.units[0].piece >= 0;
        if (more)
#pragma unroll
            for (int k = 0; k < S::kDepth; ++k) {
                copy(z.units[0], k, k);
                commit_copies();
            }
        for (int q = 0; more; ++q) {
            const int stage = q % kStages;
            const UnitNote &note = z.units[q % kUnitSlots], &next = z.units[(q + 1) % kUnitSlots];
            if (!wait_note(q + 1)) break;
            more = next.piece >= 0;
            if (q >= kStages && !mbar_wait_warp(&bars[empty + stage], ((q / kStages) - 1) & 1, p.status, empty, abort_flag)) break;
            // NaN in V that some rows must not see is left out here and put in at the end of the piece
            const bool hidden = is_v && CODE == COROPE_CODE_E4M3 && note.hidden != 0;
            const uint32_t first = tiles + stage * kTile + first_at, second = tiles + stage * kTile + second_at;
#pragma unroll
            for (int k0 = 0; k0 < S::kSteps; k0 += S::kAtOnce) {
                wait_copies<S::kDepth - S::kAtOnce>();
                uint2 w[S::kAtOnce][2];
#pragma unroll
                for (int i = 0; i < S::kAtOnce; ++i) {
                    const int place = (k0 + i) % S::kDepth * 2048;
                    w[i][0] = load8(first_from + place);
                    w[i][1] = load8(second_from + place);
                }
#pragma unroll
                for (int i = 0; i < S::kAtOnce; ++i) {
                    const int k = k0 + i + S::kDepth;
                    if (k < S::kSteps) copy(note, k, k % S::kDepth);
                    else if (more) copy(next, k - S::kSteps, k % S::kDepth);
                    commit_copies();
                }
                if (hidden) {
#pragma unroll
                    for (int i = 0; i < S::kAtOnce; ++i)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            if (has_nan(w[i][y].x) || has_nan(w[i][y].y)) z.nan_v[note.piece % kFlagSlots] = 1;
                            w[i][y] = make_uint2(without_nan(w[i][y].x), without_nan(w[i][y].y));
                        }
                }
#pragma unroll
                for (int i = 0; i < S::kAtOnce; ++i) {
                    store_codes<CODE>(w[i][0], first + (k0 + i) * (S::kRowsPerStep * 128));
                    store_codes<CODE>(w[i][1], second + (k0 + i) * (S::kRowsPerStep * 128));
                }
            }
            fence_proxy_async();
            mbar_arrive_warp(&bars[full + stage], lane);
            if (lane == 0) mbar_arrive(&bars[UNIT_EMPTY + q % kUnitSlots]);
        }
        wait_copies<0>();
    } else {
        // ------------------------------------------------------------------ softmax groups
        reg_alloc<kRegsSmx>();
        const int wsm = warp - kSmxWarp0, grp = wsm >> 3, half = (wsm >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
        const int pair_bar = 1 + grp * 4 + quad;   // the two warps that hold the same 32 rows
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + lane_base + grp * 128 + half * 64, tO = tmem + lane_base + 256;
        pdl_wait();        // the rows' factors
        int q = 0, pieces = 0, gs = 0;             // units, pieces with units, units of this group so far
        int ends0 = 0, ends1 = 0;                  // units of both groups at the end of the piece
        bool ok = true;
        // A wait that ran out is not left by: the warps of both groups meet at barriers, so each goes through all that the scout has told, if on what
        // happens to be there (the host learns of it), and waits for nothing more.  What is told comes from the scout's own
        // waits; if that gave up, all 16 warps look at the same note, the one behind the last, and find the flag or the end.
        auto wait = [&](int bar, int parity) {
            if (ok) ok = mbar_wait_warp(&bars[bar], parity, p.status, bar, abort_flag);
            tc_fence_after();
        };
        for (int k = 0;; ++k) {
            const int place = k % kPieceSlots;
            // all leave together: the first to find no piece in time tells the others at the barrier
            if (!mbar_wait_warp(&bars[PIECE_FULL + place], (k / kPieceSlots) & 1, p.status, PIECE_FULL, abort_flag)) z.left = 1;
            named_bar_sync(9, 512);
            const PieceNote& x = z.pieces[place];
            if (z.left != 0 || x.b < 0) break;
            const int count = x.count, item_row = PAIR ? grp * kN + row : row, grow = x.tile * kItemRows + item_row, t = grow / p.G, u0 = x.u0;
            const float factor = factors[((int64_t)(x.b * p.c.Hkv + x.h) * p.row_tiles + x.tile) * kItemRows + item_row];
            const int sees = p.causal ? x.len - x.n + t + 1 : x.len;
            float m = kLowest, l = 0.f;
            for (int j = PAIR ? 0 : grp; j < count; j += PAIR ? 1 : 2, ++gs) {
                const UnitNote& note = z.units[(q + j) % kUnitSlots];
                wait(S_FULL + grp, gs & 1);
                uint32_t s0[32], s1[32];
                COROPE_TMEM_LD32(tS, s0);
                COROPE_TMEM_LD32(tS + 32, s1);
                const float4 ks = *reinterpret_cast<const float4*>(&note.k_scale[half * 4]), up = *reinterpret_cast<const float4*>(&note.lift[half * 4]);
                tmem_wait_ld();
                // to units of log2, the scale of V in the exponent
                auto scale_group = [&](uint32_t* s, float k_scale, float lift) {
                    const float f = factor * k_scale;
                    const uint64_t f2 = f2_pack(f, f), a2 = f2_pack(lift, lift);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float a, b;
                        f2_unpack(f2_fma(f2_pack_bits(s[i], s[i + 1]), f2, a2), a, b);
                        s[i] = __float_as_uint(a);
                        s[i + 1] = __float_as_uint(b);
                    }
                };
                scale_group(s0, ks.x, up.x);
                scale_group(s0 + 16, ks.y, up.y);
                scale_group(s1, ks.z, up.z);
                scale_group(s1 + 16, ks.w, up.w);
                if (note.hidden) {
                    const int last = sees - (u0 + j) * kN - half * 64;   // columns from here on are hidden
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (i >= last) s0[i] = 0xff800000u;
                        if (32 + i >= last) s1[i] = 0xff800000u;
                    }
                }
                float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    mx0 = fmax3(mx0, __uint_as_float(s0[i]), __uint_as_float(s0[i + 1]));
                    mx1 = fmax3(mx1, __uint_as_float(s1[i]), __uint_as_float(s1[i + 1]));
                }
                const float top_half = fmaxf(mx0, mx1);
                z.half_max[grp][half][row] = top_half;
                named_bar_sync(pair_bar, 64);
                const float top = fmaxf(m, fmaxf(top_half, z.half_max[grp][half ^ 1][row]));
                named_bar_sync(pair_bar, 64);   // both have read before either writes again
                const bool need = top > m + 8.f;   // exp2 of up to 8 above M fits fp16
                const float m_old = m;
                m = need ? top : m;
                const uint64_t neg_m = f2_pack(-m, -m);
                const float4 drop = *reinterpret_cast<const float4*>(&note.drop[half * 4]);
                float add = 0.f;
                auto exp_group = [&](const uint32_t* s, float drop_g, uint32_t* pk) {
                    uint64_t sum = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float d0, d1;
                        f2_unpack(f2_add(f2_pack_bits(s[2 * i], s[2 * i + 1]), neg_m), d0, d1);
                        const float p0 = fast_exp2(d0), p1 = fast_exp2(d1);
                        pk[i] = pack_half2(p0, p1);
                        sum = f2_add(sum, f2_pack(p0, p1));
                    }
                    float a, b;
                    f2_unpack(sum, a, b);
                    add = a + b == 0.f ? add : fmaf(a + b, drop_g, add);   // hidden slots of a block whose scale is NaN count nothing
                };
                {
                    uint32_t pk[16];
                    exp_group(s0, drop.x, pk);
                    exp_group(s0 + 16, drop.y, pk + 8);
                    COROPE_TMEM_ST16(tS, pk);
                }
                {
                    uint32_t pk[16];
                    exp_group(s1, drop.z, pk);
                    exp_group(s1 + 16, drop.w, pk + 8);
                    COROPE_TMEM_ST16(tS + 16, pk);
                }
                if (j > (PAIR ? 0 : 1) && __any_sync(0xffffffffu, need)) {
                    wait(O_FULL + grp, (gs - 1) & 1);
                    const float shrink = fast_exp2(m_old - m);
#pragma unroll
                    for (int k = 0; k < kD / 64; ++k) {
                        const uint32_t at = tO + grp * 128 + half * (kD / 2) + k * 32;
                        uint32_t r[32];
                        COROPE_TMEM_LD32(at, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * shrink);
                        COROPE_TMEM_ST32(at, r);
                    }
                    l *= shrink;
                }
                l += add;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive_warp(&bars[P_FULL + grp], lane);
            }
            q += count;
            ends0 += (count + 1) / 2;
            ends1 += count / 2;

            // The piece's sums.  PAIR: the group's O, half of the columns to each warpgroup.  Else both groups' O, a quarter of them to each.
            const int64_t part = (2 * (int64_t)blockIdx.x + (x.share0 == 0 ? 1 : 0)) * kItemRows + item_row;
            // what waits in the block's part: read before the barrier, as one thread of the row writes it again behind it
            const bool carried = x.carried != 0;
            const float2 had = carried ? *reinterpret_cast<const float2*>(p.part_ml + part * 2) : make_float2(kLowest, 0.f);
            if (half == 0) z.end_max[grp][row] = m;
            z.end_sum[grp][half][row] = l;
            named_bar_sync(9, 512);   // (the exchange is written again behind the next piece's first barrier at the earliest)
            if (PAIR) {
                if (count > 0) wait(O_FULL + grp, (gs - 1) & 1);
            } else {
                if (count > 0) wait(O_FULL, (ends0 - 1) & 1);
                if (count > 1) wait(O_FULL + 1, (ends1 - 1) & 1);
            }
            const int other = PAIR ? grp : 0;
            const bool whole = x.whole != 0;
            const float m0 = PAIR ? m : z.end_max[0][row], m1 = PAIR ? kLowest : z.end_max[1][row], top = fmaxf(fmaxf(m0, m1), had.x);
            const float w0 = fast_exp2(m0 - top), w1 = fast_exp2(m1 - top), w_old = fast_exp2(had.x - top);
            const float own = z.end_sum[other][0][row] + z.end_sum[other][1][row];
            const float all = fmaf(had.y, w_old, PAIR ? own * w0 : own * w0 + (z.end_sum[1][0][row] + z.end_sum[1][1][row]) * w1);
            const bool some = t < x.n && all != 0.f;
            const float inv = whole ? 1.f / all : 1.f;
            constexpr int kCols = PAIR ? kD / 2 : kD / 4;
            const int col0 = (PAIR ? half : grp * 2 + half) * kCols;
            const uint32_t tO0 = tO + other * 128;
            const int64_t to = (int64_t)x.b * p.so.b + (int64_t)(x.h * p.G + grow - t * p.G) * p.so.h + (int64_t)t * p.so.n;
            const bool fix = CODE == COROPE_CODE_E4M3 && count > 0 && z.nan_v[pieces % kFlagSlots] != 0;
#pragma unroll
            for (int k = 0; k < kCols; k += 16) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = 0.f;
                if (count > 0) {
                    uint32_t r[16];
                    COROPE_TMEM_LD16(tO0 + col0 + k, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(r[i]) * w0;
                    if (!PAIR && count > 1) {
                        COROPE_TMEM_LD16(tO + 128 + col0 + k, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = fmaf(__uint_as_float(r[i]), w1, y[i]);
                    }
                }
                if (col0 + k >= D) continue;
                if (carried) {   // (this thread has written them)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 was = *reinterpret_cast<const float4*>(p.part + part * D + col0 + k + i);
                        y[i] = fmaf(was.x, w_old, y[i]); y[i + 1] = fmaf(was.y, w_old, y[i + 1]); y[i + 2] = fmaf(was.z, w_old, y[i + 2]); y[i + 3] = fmaf(was.w, w_old, y[i + 3]);
                    }
                }
                if (fix) {   // NaN in V, slot by slot: to the rows that see it
#pragma unroll 1
                    for (int s = max(u0, x.seen / kN) * kN; s < (t < x.n ? min(sees, (u0 + count) * kN) : 0); ++s) {   // (never behind the last slot, whose block the table still has)
                        bool far = false;
                        const int page = cache_page(p.s, p.c.bs_log2, p.c.num_blocks, x.b, s, far);
                        if (page < 0 || no_values(p.c.v_scale[(int64_t)page * p.c.Hkv + x.h])) continue;
                        const uint8_t* v = p.c.v + (int64_t)page * p.c.sv.b + (int64_t)x.h * p.c.sv.h + (int64_t)(s & ((1 << p.c.bs_log2) - 1)) * p.c.sv.n + col0 + k;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((v[i] & 0x7f) == 0x7f) y[i] = __int_as_float(0x7fffffff);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(p.part + part * D + col0 + k + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                } else if (t < p.T) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        store4(p.o, to + col0 + k + i, p.dtype, p.vec_o,
                               some ? make_float4(y[i] * inv, y[i + 1] * inv, y[i + 2] * inv, y[i + 3] * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
                }
            }
            if ((PAIR || grp == 0) && half == 0) {
                if (!whole) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(top, all);
                else if (p.lse != nullptr && t < p.T) p.lse[((int64_t)x.b * p.c.Hkv + x.h) * p.T * p.G + grow] = some ? top + log2f(all) : INFINITY;
            }
            if (count > 0) {
                tc_fence_before();
                mbar_arrive_warp(&bars[O_FREE], lane);
                // the flag of the piece before: every thread has read it, and its place is not taken again before this thread has come by
                if (wsm == 0 && lane == 0 && pieces > 0) z.nan_v[(pieces - 1) % kFlagSlots] = 0;
                ++pieces;
            }
            mbar_arrive_warp(&bars[PIECE_EMPTY + place], lane);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) report_expired_wait(p.status, *abort_flag, p.mirror);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------------ accumulated weights
// S^T = K Q^T with slots as rows: a thread has a slot and sums exp2(s - lse) over the columns, the query rows, so nothing crosses threads.  A unit
// is 128 slots of a K / V head: its K stays, and the tiles of query rows (both parts) stream by.  Bound by the exponentials.
//   warp 0  query tiles, with their rows' factors and lse;  warp 1  MMA issuer;  warps 4-7  K;  warps 8-11, 12-15  the even and odd tiles
constexpr int kSumThreads = 512;
constexpr int kRowSlots = 4;
__host__ __device__ constexpr int sum_stages(int D) { return D == 128 ? 2 : 4; }   // of query tiles
enum SumBar { W_K_FULL = 0, W_K_EMPTY = 2, W_S_FULL = 4, W_S_FREE = 6, W_ROWS = 8, W_Q_FULL = W_ROWS + kRowSlots, W_Q_EMPTY = W_Q_FULL + 4, W_ROWS_FREE = W_Q_EMPTY + 4, W_NUM_BARS = W_ROWS_FREE + kRowSlots };
struct alignas(16) SumSmall {   // factor and lse are read four at a time
    float factor[kRowSlots][kN], lse[kRowSlots][kN], sum[2][kN];
    float k_scale[2][8];
    int page[2][8];
    uint64_t bars[W_NUM_BARS];
    uint32_t tmem;
    int abort;
};
constexpr size_t sum_smem_bytes(int D) { return (2 * sum_stages(D) + 2) * tile_bytes(D) + sizeof(SumSmall) + 1024; }
static_assert(sum_smem_bytes(128) <= 232448 - 1024, "shared memory budget");

struct Unit {
    int b, h, u, len, n, tile0, tiles;   // tiles [tile0, tiles) have rows that see a slot of the unit
};
struct UnitWalk {
    Range r;
    Load l;
    bool bad = false;
    __device__ __forceinline__ Load load(const CacheAttnParams& p, int b) {
        Load l = load_of(p, log2_of(kN), log2_of(kN), 0, b, bad);
        l.items = l.n > 0 ? p.c.Hkv : 0;
        return l;
    }
    __device__ __forceinline__ UnitWalk(const CacheAttnParams& p, const Range& range) : r(range) { l = load(p, r.b); }
    __device__ __forceinline__ bool next(const CacheAttnParams& p, Unit& x) {
        for (; r.left > 0; --r.left, ++r.off) {
            while (r.off >= (int64_t)l.units * l.items) {
                r.off -= (int64_t)l.units * l.items;
                l = load(p, ++r.b);
            }
            x.b = r.b; x.len = l.len; x.n = l.n;
            x.h = (int)(r.off / l.units);
            x.u = (int)(r.off - (int64_t)x.h * l.units);
            const int64_t first = p.causal ? max((int64_t)x.u * kN - (l.len - l.n), (int64_t)0) * p.G : 0;   // the first row that sees a slot
            x.tiles = (l.n * p.G + kN - 1) / kN;
            x.tile0 = (int)min(first / kN, (int64_t)x.tiles);
            if (x.tile0 < x.tiles) {
                --r.left;
                ++r.off;
                return true;
            }
        }
        return false;
    }
};

template <int D, int CODE>
__global__ void __launch_bounds__(kSumThreads, 1) cache_weight_tile_kernel(const CacheAttnParams p, int image_tiles, const uint8_t* images, const float* factors) {
    constexpr int kD = wide(D), kBox = kN * 128;
    constexpr uint32_t kTile = (uint32_t)tile_bytes(D);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kQStages = sum_stages(D);
    uint8_t* sQ = sm;                            // [stage][part]
    uint8_t* sK = sQ + 2 * kQStages * kTile;     // [stage]
    SumSmall& z = *reinterpret_cast<SumSmall*>(sK + 2 * kTile);
    uint64_t* bars = z.bars;
    volatile int* abort_flag = &z.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool bad = false;
    const Range range = take_range<128>(p.s.B, [&](int b) {
        Load l = load_of(p, log2_of(kN), log2_of(kN), 0, b, bad);
        l.items = l.n > 0 ? p.c.Hkv : 0;
        return l;
    });
    const bool gave_up = p.status != nullptr && (*reinterpret_cast<volatile int*>(p.status) & COROPE_DEV_WAIT_EXPIRED);
    if (__syncthreads_or(gave_up) || range.left == 0) {
        if (threadIdx.x == 0 && gave_up) report_to_mirror(p.status, p.mirror);
        return;
    }
    if (threadIdx.x == 0) {
        z.abort = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[W_K_FULL + i], 4);
            mbar_init(&bars[W_K_EMPTY + i], 4);      // the group that ends a unit
            mbar_init(&bars[W_S_FULL + i], 1);
            mbar_init(&bars[W_S_FREE + i], 4);
        }
        for (int i = 0; i < kQStages; ++i) {
            mbar_init(&bars[W_Q_FULL + i], 1);
            mbar_init(&bars[W_Q_EMPTY + i], 1);
        }
        for (int i = 0; i < kRowSlots; ++i) {
            mbar_init(&bars[W_ROWS + i], 1);
            mbar_init(&bars[W_ROWS_FREE + i], 4);    // the group whose tile it is
        }
        fence_mbar_init();
    }
    if (D == 32)
        for (int i = threadIdx.x; i < (int)(2 * kTile / 16); i += kSumThreads) reinterpret_cast<uint4*>(sK)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
    __syncthreads();
    if (warp == 1) {
        tmem_alloc(&z.tmem, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = z.tmem;
    UnitWalk walk(p, range);
    Unit x;
    bool ok = true;

    if (warp == 0) {
        // ------------------------------------------------------------------ query tiles
        int q = 0;
        while (ok && walk.next(p, x))
            for (int t = x.tile0; ok && t < x.tiles; ++t, ++q) {
                const int i = q % kQStages, slot = q % kRowSlots;
                const int64_t item = (int64_t)(x.b * p.c.Hkv + x.h) * image_tiles + t;
                if (q >= kQStages && !(ok = mbar_wait_warp(&bars[W_Q_EMPTY + i], ((q / kQStages) - 1) & 1, p.status, W_Q_EMPTY, abort_flag))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&bars[W_Q_FULL + i], 2 * kTile);
                    for (int part = 0; part < 2; ++part) bulk_load_1d(sQ + (2 * i + part) * kTile, images + ((size_t)item * 2 + part) * kTile, kTile, &bars[W_Q_FULL + i]);
                }
                float f[kN / 32], e[kN / 32];
#pragma unroll
                for (int k = 0; k < kN / 32; ++k) {
                    const int row = t * kN + 32 * k + lane;
                    f[k] = factors[item * kN + 32 * k + lane];
                    e[k] = row < x.n * p.G ? p.lse[((int64_t)x.b * p.c.Hkv + x.h) * p.T * p.G + row] : INFINITY;
                }
                // The slot's last tile has been summed.  A barrier of the slot's own: its next phase needs the rows that are posted here, so the parity is never
                // that of two phases back (the group's W_S_FREE can be one tile further on).
                if (q >= kRowSlots && !(ok = mbar_wait_warp(&bars[W_ROWS_FREE + slot], ((q / kRowSlots) - 1) & 1, p.status, W_ROWS_FREE, abort_flag))) break;
#pragma unroll
                for (int k = 0; k < kN / 32; ++k) z.factor[slot][32 * k + lane] = f[k], z.lse[slot][32 * k + lane] = e[k];
                mbar_arrive_warp(&bars[W_ROWS + slot], lane);
            }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        const bool leader = elect_one();
        const uint32_t idesc = make_idesc(0, 0, 0, 0, kN, kN);
        constexpr uint32_t kHi = sdesc_hi(1024);
        const uint32_t q_lo = sdesc_lo(smem_u32(sQ), 0), k_lo = sdesc_lo(smem_u32(sK), 0);
        int q = 0, units = 0;
        while (ok && walk.next(p, x)) {
            const int stage = units & 1;
            if (!(ok = mbar_wait_warp(&bars[W_K_FULL + stage], (units >> 1) & 1, p.status, W_K_FULL, abort_flag))) break;
            for (int t = x.tile0; t < x.tiles; ++t, ++q) {
                const int i = q & 1;
                const int from = q % kQStages;
                if (!(ok = mbar_wait_warp(&bars[W_Q_FULL + from], (q / kQStages) & 1, p.status, W_Q_FULL, abort_flag))) break;
                if (q >= 2 && !(ok = mbar_wait_warp(&bars[W_S_FREE + i], ((q >> 1) - 1) & 1, p.status, W_S_FREE, abort_flag))) break;
                tc_fence_after();
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                    for (int kk = 0; kk < kD / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
                        if (leader) umma_ss2(tmem + i * 128, k_lo + stage * (kTile >> 4) + off, kHi, q_lo + (2 * from + part) * (kTile >> 4) + off, kHi, idesc, part == 0 || kk > 0);
                    }
                if (leader) {
                    umma_commit(&bars[W_S_FULL + i]);
                    umma_commit(&bars[W_Q_EMPTY + from]);
                }
            }
            ++units;
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 8) {
        // ------------------------------------------------------------------ K
        using S = Steps<D, true, false>;
        const int tid = threadIdx.x & 127, col = tid % S::kLanes * 16, row0 = tid / S::kLanes, in_block_mask = (1 << p.c.bs_log2) - 1;
        const int run = col / 8, swap = D == 128 ? run >> 3 : 0;
        const uint32_t first_at = (run >> 3) * kBox + row0 * 128 + ((((run & 7) ^ (row0 & 7)) ^ swap) << 4);
        int units = 0;
        while (walk.next(p, x)) {
            const int stage = units & 1;
            const int page = unit_page(p, x, x.u, lane, bad);
            if (units >= 2 && !mbar_wait_warp(&bars[W_K_EMPTY + stage], ((units >> 1) - 1) & 1, p.status, W_K_EMPTY, abort_flag)) break;
            if (tid < 8) {
                z.k_scale[stage][tid] = page >= 0 ? p.c.k_scale[(int64_t)page * p.c.Hkv + x.h] : 0.f;
                z.page[stage][tid] = page;
            }
            uint4 w[S::kSteps];
#pragma unroll
            for (int k = 0; k < S::kSteps; ++k) {
                const int row = k * S::kRowsPerStep + row0, slot = x.u * kN + row, pg = __shfl_sync(0xffffffffu, page, row >> 4);
                w[k] = make_uint4(0u, 0u, 0u, 0u);
                if (pg >= 0 && slot < x.len)
                    w[k] = *reinterpret_cast<const uint4*>(p.c.k + (int64_t)pg * p.c.sk.b + (int64_t)x.h * p.c.sk.h + (int64_t)(slot & in_block_mask) * p.c.sk.n + col);
            }
#pragma unroll
            for (int k = 0; k < S::kSteps; ++k) {
                const uint32_t at = smem_u32(sK) + stage * kTile + first_at + k * (S::kRowsPerStep * 128);
                store_codes<CODE>(swap ? make_uint2(w[k].z, w[k].w) : make_uint2(w[k].x, w[k].y), at);
                store_codes<CODE>(swap ? make_uint2(w[k].x, w[k].y) : make_uint2(w[k].z, w[k].w), at ^ 16);
            }
            fence_proxy_async();
            mbar_arrive_warp(&bars[W_K_FULL + stage], lane);
            ++units;
        }
    } else if (warp >= 8) {
        // ------------------------------------------------------------------ sums
        const int grp = (warp - 8) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + grp * 128;
        int q = 0, units = 0;
        auto wait = [&](int bar, int parity) {   // as in the main kernel: nobody leaves a barrier that others come to
            if (ok) ok = mbar_wait_warp(&bars[bar], parity, p.status, bar, abort_flag);
        };
        while (walk.next(p, x)) {
            const int stage = units & 1, slot = x.u * kN + row, count = x.tiles - x.tile0;
            wait(W_K_FULL + stage, (units >> 1) & 1);
            const float ks = z.k_scale[stage][row >> 4];
            const int page = z.page[stage][row >> 4];
            const uint64_t ks2 = f2_pack(ks, ks);
            float w = 0.f;
            for (int j = 0; j < count; ++j, ++q) {
                if ((q & 1) != grp) continue;
                const int rows = q % kRowSlots;
                wait(W_ROWS + rows, (q / kRowSlots) & 1);
                wait(W_S_FULL + grp, (q >> 1) & 1);
                tc_fence_after();
                // columns that see the slot: from the first row whose query does to the last row with a query
                const int tile = x.tile0 + j;
                const int64_t first = p.causal ? (int64_t)max(slot - (x.len - x.n), 0) * p.G - (int64_t)tile * kN : 0;
                const int from = (int)min(max(first, (int64_t)0), (int64_t)kN), to = min(x.n * p.G - tile * kN, kN);
                const bool every = __all_sync(0xffffffffu, from == 0 && to == kN);
#pragma unroll
                for (int k = 0; k < kN; k += 32) {
                    uint32_t s[32];
                    COROPE_TMEM_LD32(tS + k, s);
                    tmem_wait_ld();
                    uint64_t sum = 0;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&z.factor[rows][k + i]), e = *reinterpret_cast<const float4*>(&z.lse[rows][k + i]);
                        float d[4];
                        f2_unpack(f2_fma(f2_pack_bits(s[i], s[i + 1]), f2_mul(f2_pack(f.x, f.y), ks2), f2_pack(-e.x, -e.y)), d[0], d[1]);
                        f2_unpack(f2_fma(f2_pack_bits(s[i + 2], s[i + 3]), f2_mul(f2_pack(f.z, f.w), ks2), f2_pack(-e.z, -e.w)), d[2], d[3]);
                        if (!every) {
#pragma unroll
                            for (int y = 0; y < 4; ++y) d[y] = k + i + y >= from && k + i + y < to ? d[y] : -INFINITY;
                        }
                        sum = f2_add(sum, f2_pack(fast_exp2(d[0]), fast_exp2(d[1])));
                        sum = f2_add(sum, f2_pack(fast_exp2(d[2]), fast_exp2(d[3])));
                    }
                    float a, b;
                    f2_unpack(sum, a, b);
                    w += a + b;
                }
                tc_fence_before();
                mbar_arrive_warp(&bars[W_S_FREE + grp], lane);
                if (lane == 0) mbar_arrive(&bars[W_ROWS_FREE + rows]);
            }
            z.sum[grp][row] = w;
            named_bar_sync(1, 256);
            if (grp == 0 && page >= 0 && slot < x.len) {   // one addition per slot and call; atomic because sequences may share blocks
                const int bs_mask = (1 << p.c.bs_log2) - 1;
                atomicAdd(p.c.weight + (((int64_t)page * p.c.Hkv + x.h) << p.c.bs_log2) + (slot & bs_mask), w + z.sum[1][row]);
            }
            named_bar_sync(1, 256);
            // every tile of the unit has been read, so its products are complete
            if (grp == 0) mbar_arrive_warp(&bars[W_K_EMPTY + stage], lane);
            ++units;
        }
        tc_fence_before();
    }
    if (bad || walk.bad) report_bad_index(p.status, p.mirror);
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) report_expired_wait(p.status, *abort_flag, p.mirror);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 256);
    }
}

struct TileLayout {
    size_t factors, total;   // the images come first
};
TileLayout tile_layout(int B, int Hkv, int image_tiles, int D, bool two) {
    const size_t items = (size_t)B * Hkv * image_tiles;
    TileLayout l;
    l.factors = items * (two ? 2 : 1) * tile_bytes(D);
    l.total = align_up(l.factors + items * kN * 4, 256);
    return l;
}

template <int D, int CODE, bool TWO, bool PAIR>
int launch_t(const CacheAttnParams& p, uint8_t* images, float* factors, unsigned blocks, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (int e = allow_smem(cache_attn_tile_kernel<D, CODE, TWO, PAIR>, smem_bytes(D, TWO, PAIR), done)) return e;
    const int image_tiles = p.row_tiles * (PAIR ? 2 : 1);
    count_launch(2);
    cache_pack_kernel<D, TWO><<<(unsigned)(p.s.B * p.c.Hkv * image_tiles * kPackBlocks), kPackWarps * 32, 0, s>>>(p, image_tiles, images, factors);
    if (int e = (int)cudaGetLastError()) return e;
    return launch_dependent(cache_attn_tile_kernel<D, CODE, TWO, PAIR>, blocks, kThreads, smem_bytes(D, TWO, PAIR), s, p, (const uint8_t*)images, (const float*)factors);
}
template <int D, int CODE>
int by_shape(const CacheAttnParams& p, uint8_t* images, float* factors, bool two, bool pair, unsigned blocks, cudaStream_t s) {
    if constexpr (D != 128)
        if (two && pair) return launch_t<D, CODE, true, true>(p, images, factors, blocks, s);
    if (pair) return launch_t<D, CODE, false, true>(p, images, factors, blocks, s);
    return two ? launch_t<D, CODE, true, false>(p, images, factors, blocks, s) : launch_t<D, CODE, false, false>(p, images, factors, blocks, s);
}
template <int D>
int by_code(const CacheAttnParams& p, uint8_t* images, float* factors, bool two, bool pair, unsigned blocks, cudaStream_t s) {
    return p.code == COROPE_CODE_E4M3 ? by_shape<D, COROPE_CODE_E4M3>(p, images, factors, two, pair, blocks, s)
                                      : by_shape<D, COROPE_CODE_INT8>(p, images, factors, two, pair, blocks, s);
}
template <int D, int CODE>
int launch_weight_t(const CacheAttnParams& p, int image_tiles, const uint8_t* images, const float* factors, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (int e = allow_smem(cache_weight_tile_kernel<D, CODE>, sum_smem_bytes(D), done)) return e;
    const uint64_t units = (uint64_t)p.s.B * p.c.Hkv * ((p.capacity + kN - 1) / kN);
    count_launch();
    cache_weight_tile_kernel<D, CODE><<<(unsigned)(units < (uint64_t)sm_count() ? units : sm_count()), kSumThreads, sum_smem_bytes(D), s>>>(p, image_tiles, images, factors);
    return (int)cudaGetLastError();
}
template <int D>
int weight_by_code(const CacheAttnParams& p, int image_tiles, const uint8_t* images, const float* factors, cudaStream_t s) {
    return p.code == COROPE_CODE_E4M3 ? launch_weight_t<D, COROPE_CODE_E4M3>(p, image_tiles, images, factors, s)
                                      : launch_weight_t<D, COROPE_CODE_INT8>(p, image_tiles, images, factors, s);
}

}  // namespace

bool cache_tile_pairs(int rows, int D, bool two_parts) { return rows > kN && !(D == 128 && two_parts); }

size_t cache_tile_workspace_bytes(int B, int Hkv, int image_tiles, int D, bool two_parts) { return tile_layout(B, Hkv, image_tiles, D, two_parts).total; }

int launch_cache_attn_tiles(const CacheAttnParams& p, void* ws, bool two_parts, bool pair, unsigned blocks, cudaStream_t s) {
    uint8_t* images = static_cast<uint8_t*>(ws);
    float* factors = reinterpret_cast<float*>(images + tile_layout(p.s.B, p.c.Hkv, p.row_tiles * (pair ? 2 : 1), p.D, two_parts).factors);
    return p.D == 128 ? by_code<128>(p, images, factors, two_parts, pair, blocks, s) : p.D == 64 ? by_code<64>(p, images, factors, two_parts, pair, blocks, s)
                                                                                               : by_code<32>(p, images, factors, two_parts, pair, blocks, s);
}

int launch_cache_weight_tiles(const CacheAttnParams& p, void* ws, bool pair, cudaStream_t s) {
    const int image_tiles = p.row_tiles * (pair ? 2 : 1);
    const uint8_t* images = static_cast<const uint8_t*>(ws);
    const float* factors = reinterpret_cast<const float*>(images + tile_layout(p.s.B, p.c.Hkv, image_tiles, p.D, true).factors);
    return p.D == 128 ? weight_by_code<128>(p, image_tiles, images, factors, s) : p.D == 64 ? weight_by_code<64>(p, image_tiles, images, factors, s)
                                                                                          : weight_by_code<32>(p, image_tiles, images, factors, s);
}

}  // namespace corope
