/*
 * corope_b200 -- C ABI of the B200 (sm_100a) fused-RoPE attention and Co-RoPE GQA attention kernels.
 *
 * Plain pointers and sizes only; no C++ or torch types cross this boundary.  All tensor
 * pointers are DEVICE pointers.  q/k/v/o/dO/dq/dk/dv are row-major contiguous [B, H, N, D]
 * in the element type named by `dtype` (the *_strided entry points take other layouts).  Every call enqueues work on `stream` (a
 * cudaStream_t passed as void*) and returns without synchronising.
 *
 * Return value: 0 = OK, < 0 = argument error found on the host (nothing was launched),
 * > 0 = a cudaError_t from a launch.  Kernels never trap: a device-side bounded wait that
 * expires writes a non-zero code into `*status_word` (device memory, may be NULL) and the
 * kernel exits cleanly.  While the word is non-zero, later tensor-core launches that are given the
 * same word return without computing (their outputs are then undefined): read and clear it on the
 * host after synchronising.  The Python modules of this package do that for the caller: every call
 * first looks at a pinned host mirror of the word, which a failing kernel writes too, and
 * raises (and clears the word) if it was set.
 *
 * Supported value range of 16-bit inputs: the tensor-core kernels feed fp16 operands to the MMAs
 * (rotated Q / K, dS) with saturating conversions, so results are exact in kind for |q|, |k| up to
 * a few hundred and for gradient magnitudes |dO| up to about 2^10; beyond that single products may
 * clamp to +-65504 and results lose accuracy without becoming inf / NaN.  fp32 inputs have no such
 * limit (fp32 arithmetic throughout).
 *
 * Each entry point names the interface of the reference (Superposition09m/Co-RoPE) it stands in for.
 */
#ifndef COROPE_B200_H_
#define COROPE_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of q/k/v/o and gradients */
#define COROPE_DTYPE_F32 0
#define COROPE_DTYPE_BF16 1
#define COROPE_DTYPE_F16 2

/* `op` values for corope_workspace_bytes */
#define COROPE_OP_ROPE_FWD 0
#define COROPE_OP_ROPE_BWD 1
#define COROPE_OP_GQA_FWD 2
#define COROPE_OP_GQA_BWD 3
#define COROPE_OP_ROPE_FWD_FREQS 4   /* corope_rope_attn_fwd_freqs: as ROPE_FWD plus room for the synthesized tables */
#define COROPE_OP_ROPE_BWD_FREQS 5
#define COROPE_OP_FLASH_FWD 6        /* corope_flash_attn_fwd (Hq query heads, Hkv K / V heads) */
#define COROPE_OP_FLASH_BWD 7

/* host-side argument errors */
#define COROPE_OK 0
#define COROPE_ERR_NULL_POINTER (-1)
#define COROPE_ERR_BAD_SHAPE (-2)      /* non-positive extent */
#define COROPE_ERR_BAD_HEAD_DIM (-3)   /* D outside the supported set (fused_rope_attn.py:661 asserts the same way) */
#define COROPE_ERR_BAD_DTYPE (-4)
#define COROPE_ERR_WORKSPACE (-5)      /* workspace missing, too small or misaligned (needs 256-byte alignment) */
#define COROPE_ERR_BAD_GROUP (-6)      /* Hq % Hkv != 0 or group size > 8 (flash_attn_co_rope_gqa_triton.py:421-425) */
#define COROPE_ERR_SEQ_NOT_128 (-7)    /* backward needs N % 128 == 0 (fused_rope_attn.py:750) -- only when strict_n is set */
#define COROPE_ERR_TENSOR_MAP (-8)     /* TMA descriptor could not be encoded */
#define COROPE_ERR_NO_DEVICE (-9)      /* no sm_100 device / driver entry point */
#define COROPE_ERR_TOO_LARGE (-10)     /* size beyond what the entry point supports */
#define COROPE_ERR_BAD_STRIDE (-11)    /* row stride below D, or a negative stride */
#define COROPE_ERR_BAD_CACHE (-12)     /* code type, block size or strides that the cache operators do not take */

/* device-side status codes: bits of *status_word, which stay until the host clears them (of several expired waits the first one's id) */
#define COROPE_DEV_OK 0
#define COROPE_DEV_WAIT_EXPIRED 0x1000 /* | barrier id: a bounded mbarrier wait ran out */
#define COROPE_DEV_RANGE 0x2000        /* a gradient term left the range of the 16-bit Co-RoPE backward and was clamped */
#define COROPE_DEV_BAD_INDEX 0x4000    /* a block table entry, length or position of a cache operator pointed outside its tensor */

int corope_abi_version(void);

/*
 * Host mirror of a status word, for callers that want to learn of a device-side error without ever synchronising:
 * `_refresh` makes a side stream of the library copy *status_word to *host_mirror (pinned host memory) once `stream` has
 * executed everything enqueued so far -- `stream` itself only records an event -- so that reading *host_mirror on the host
 * before a later call shows whether an earlier call failed.  `_register` lets the kernels themselves write a failure to the
 * mirror of the word they are handed (nothing has to be enqueued behind a call then).  `_clear` resets both (it waits for
 * the side stream first).
 * No counterpart in the reference, whose kernels report nothing.
 */
int corope_status_mirror_register(const int* status_word, int* host_mirror);
int corope_status_mirror_refresh(const int* status_word, int* host_mirror, void* stream);
int corope_status_mirror_clear(int* status_word, int* host_mirror, void* stream);
const char* corope_status_string(int status);

/* Bytes of caller-provided scratch (device memory, 256-byte aligned) an op needs.  Contents
 * need not be initialised by the caller.  For MHA pass Hkv == Hq.  For 16-bit inputs at D = 64 or 128 with
 * N % 128 == 0 the fused-RoPE and plain ops keep a rotated fp16 copy of K (forward) or Q (backward) there, so the
 * size grows with B*H*N*D (forward: 2 bytes per element of k; backward: 6 bytes per element of q; for D = 64 this
 * function answers 16 and 32 per element of q).  Always ask this function. */
size_t corope_workspace_bytes(int op, int B, int Hq, int Hkv, int N, int D, int dtype);

/* The size with which an op runs on tensor cores at every N, not only at whole tiles: 16-bit D = 64 or 128 inputs of a ragged N, and
 * fp32 D = 64 inputs of 256 rows or more, then go to kernels that split every fp32 operand into three 16-bit numbers, which hold its
 * 24 bits, and keep fp32 accuracy (6 bytes per element of k, in the backward also of q; for fp32 also of v and, backward, of d_o); so does the Co-RoPE forward
 * at D = 64, a ragged N or rows that are not aligned to 16 bytes.  A call that is handed at least this much uses them; with
 * corope_workspace_bytes() bytes it runs on the CUDA-core kernels.  Never more than corope_workspace_bytes() for the fused-RoPE and plain
 * ops on 16-bit inputs where N is a whole number of tiles. */
size_t corope_workspace_bytes_any_n(int op, int B, int Hq, int Hkv, int N, int D, int dtype);

/*
 * Fused RoPE attention forward.  Replaces the launch in _attention.forward
 * (fused-rope/fused_rope_attn.py:655-722, kernels _attn_fwd / _attn_fwd_inner :47-320).
 *   cos, sin : fp32 tables, row n at cos + n*table_row_stride, only columns [0, D/2) are read
 *              (fused_rope_attn.py:88-93, 279-284) -- both [N, D] "cat" and [N, D/2] tables work.
 *   o        : [B,H,N,D] output in `dtype`.
 *   lse2     : [B,H,N] fp32, log2-domain log-sum-exp of the scaled scores (the reference's M, :316).
 */
int corope_rope_attn_fwd(const void* q, const void* k, const void* v,
                         const float* cos, const float* sin, int64_t table_row_stride,
                         void* o, float* lse2,
                         int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                         void* workspace, size_t workspace_bytes,
                         int* status_word, void* stream);

/*
 * Fused RoPE attention forward that allocates nothing and takes no workspace.  It has no counterpart in the
 * reference.  It exists for callers that may not allocate device memory at the point of the call and have no
 * spare buffer to lend: code running under a framework that hands out a fixed, fully planned memory arena,
 * inference servers with a hard memory budget, or a call site where an allocation would synchronise the device.
 * Same arguments and results as corope_rope_attn_fwd minus the workspace.  The one piece of scratch the forward
 * uses (the packed cos/sin table) lives in a 2 MiB array inside the library image, per GPU, until the process
 * exits.  Limit: N * (D/2) <= 524288 (N <= 8192 at D = 128); larger sizes return COROPE_ERR_TOO_LARGE.
 * The first call on each device looks up the array's device address (cudaGetSymbolAddress, with that device
 * current); make that first call outside any stream capture.  All calls on a device share the array: two calls
 * whose kernels can overlap on the GPU (different streams, no ordering between them) race on it; calls ordered
 * on one stream are safe, and nothing left by an earlier call is ever read.  Calls no cudaMalloc/cudaFree.
 */
int corope_rope_attn_fwd_noalloc(const void* q, const void* k, const void* v,
                                 const float* cos, const float* sin, int64_t table_row_stride,
                                 void* o, float* lse2,
                                 int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                                 int* status_word, void* stream);

/*
 * Fused RoPE attention backward.  Replaces _attention.backward
 * (fused-rope/fused_rope_attn.py:725-777: the K pre-scale :746-748, _attn_bwd_preprocess :324-337,
 * _attn_bwd :474-649).  o and lse2 are the forward's outputs; dq/dk/dv are written in `dtype`.
 */
int corope_rope_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                         const float* lse2,
                         const float* cos, const float* sin, int64_t table_row_stride,
                         void* dq, void* dk, void* dv,
                         int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                         void* workspace, size_t workspace_bytes,
                         int* status_word, void* stream);

/*
 * Strides, in elements, of the eight [B, H, N, D] tensors an op can touch: {batch, head, row} each; the head-dim stride is
 * always 1.  The reference hands all four strides of q / k / v / o to its kernels (fused-rope/fused_rope_attn.py:709-710,
 * flash_attn_v2_triton.py:601-603), so views such as a [B, N, H, D] buffer transposed to [B, H, N, D] need no copy there;
 * the *_strided entry points below take them here.  Fields an op does not use (d_o, dq, dk, dv in a forward) are ignored.
 * The tensor-core kernels need every used stride and base pointer to be a multiple of 16 bytes (8 elements for 16-bit
 * types); other strides run on the CUDA-core kernels.  lse2 (and the tables) stay contiguous.  A NULL `strides` means
 * contiguous tensors, i.e. the plain entry point.
 */
typedef struct corope_strides_t {
    int64_t q[3], k[3], v[3], o[3], d_o[3], dq[3], dk[3], dv[3];
} corope_strides_t;

int corope_rope_attn_fwd_strided(const void* q, const void* k, const void* v,
                                 const float* cos, const float* sin, int64_t table_row_stride,
                                 void* o, float* lse2,
                                 int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                                 void* workspace, size_t workspace_bytes,
                                 int* status_word, void* stream, const corope_strides_t* strides);
int corope_rope_attn_bwd_strided(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                                 const float* lse2,
                                 const float* cos, const float* sin, int64_t table_row_stride,
                                 void* dq, void* dk, void* dv,
                                 int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                                 void* workspace, size_t workspace_bytes,
                                 int* status_word, void* stream, const corope_strides_t* strides);

/*
 * Fused RoPE attention with the cos / sin tables synthesized on the device instead of read from the caller: the angle
 * of position n and pair d is float(n) * inv_freq[d] in fp32, exactly how precompute_freqs_cis forms it
 * (fused-rope/rope_attn_pytorch.py:29-47: inv_freq[d] = 1 / theta^(2d/D), positions 0 .. N-1), followed by cosf / sinf.
 * For callers whose tables are that function's output, this removes the tables from the interface and from HBM
 * traffic; corope_rope_attn_fwd / _bwd with explicit tables remain the general case (arbitrary positions, scaled
 * or interpolated frequencies).   inv_freq : D/2 floats in device memory.  Workspace: COROPE_OP_ROPE_FWD_FREQS /
 * COROPE_OP_ROPE_BWD_FREQS.  Everything else as corope_rope_attn_fwd / corope_rope_attn_bwd.
 */
int corope_rope_attn_fwd_freqs(const void* q, const void* k, const void* v, const float* inv_freq,
                               void* o, float* lse2,
                               int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                               void* workspace, size_t workspace_bytes,
                               int* status_word, void* stream);
int corope_rope_attn_bwd_freqs(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                               const float* lse2, const float* inv_freq,
                               void* dq, void* dk, void* dv,
                               int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                               void* workspace, size_t workspace_bytes,
                               int* status_word, void* stream);

/* The same from the base theta: inv_freq[d] = 1 / theta^(2d/D) is formed on the device too, in fp32 as precompute_freqs_cis forms
 * it.  Workspace: COROPE_OP_ROPE_FWD_FREQS / COROPE_OP_ROPE_BWD_FREQS.  `strides` as in the *_strided entry points (NULL =
 * contiguous). */
int corope_rope_attn_fwd_theta(const void* q, const void* k, const void* v, float theta,
                               void* o, float* lse2,
                               int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                               void* workspace, size_t workspace_bytes,
                               int* status_word, void* stream, const corope_strides_t* strides);
int corope_rope_attn_bwd_theta(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                               const float* lse2, float theta,
                               void* dq, void* dk, void* dv,
                               int B, int H, int N, int D, int dtype, int causal, float sm_scale,
                               void* workspace, size_t workspace_bytes,
                               int* status_word, void* stream, const corope_strides_t* strides);

/*
 * Plain flash attention (no RoPE) with grouped K / V heads.  Replaces _attention.forward / .backward of the reference's
 * un-fused kernel (fused-rope/flash_attn_v2_triton.py:513-631; head mapping off_h_kv = off_h_q // GROUP_SIZE :194-196);
 * the math is that of assets/flashattn-gqa/attn_gqa_pytorch.py:17-190.
 *   q, o, d_o, dq : [B,Hq,N,D];  k, v, dk, dv : [B,Hkv,N,D];  Hq % Hkv == 0 (any group size);  lse2 : [B,Hq,N].
 * dk / dv are summed over each group (the reference's backward takes Hq == Hkv only, :560; this one takes both).
 * Same kernels as the fused-RoPE ops with the rotation switched off.  Workspace: COROPE_OP_FLASH_FWD / COROPE_OP_FLASH_BWD.
 */
int corope_flash_attn_fwd(const void* q, const void* k, const void* v,
                          void* o, float* lse2,
                          int B, int Hq, int Hkv, int N, int D, int dtype, int causal, float sm_scale,
                          void* workspace, size_t workspace_bytes,
                          int* status_word, void* stream);
int corope_flash_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                          const float* lse2,
                          void* dq, void* dk, void* dv,
                          int B, int Hq, int Hkv, int N, int D, int dtype, int causal, float sm_scale,
                          void* workspace, size_t workspace_bytes,
                          int* status_word, void* stream);

int corope_flash_attn_fwd_strided(const void* q, const void* k, const void* v,
                                  void* o, float* lse2,
                                  int B, int Hq, int Hkv, int N, int D, int dtype, int causal, float sm_scale,
                                  void* workspace, size_t workspace_bytes,
                                  int* status_word, void* stream, const corope_strides_t* strides);
int corope_flash_attn_bwd_strided(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                                  const float* lse2,
                                  void* dq, void* dk, void* dv,
                                  int B, int Hq, int Hkv, int N, int D, int dtype, int causal, float sm_scale,
                                  void* workspace, size_t workspace_bytes,
                                  int* status_word, void* stream, const corope_strides_t* strides);

/*
 * Co-RoPE GQA attention forward (causal only).  Replaces the launch in _attention.forward
 * (corope-exp/flash_attn_co_rope_gqa_triton.py:406-456, kernel _corope_fwd_backbone :47-400);
 * the math is that of corope-exp/corope_attn_gqa_pytorch.py:56-124.
 *   q, o   : [B,Hq,N,D];  k, v : [B,Hkv,N,D];  Hq % Hkv == 0, Hq/Hkv <= 8.
 *   lse2   : [B,Hq,N] fp32 (log2 domain);  a_diag : [B,Hkv,N] fp32, the leader mileage a_ii.
 * For 16-bit inputs at D = 128 and N % 64 == 0 the workspace holds fp16 operand copies of K and V
 * (4 bytes per element of k); otherwise the forward needs none (corope_workspace_bytes returns the 256-byte minimum).
 */
int corope_gqa_fwd(const void* q, const void* k, const void* v,
                   void* o, float* lse2, float* a_diag,
                   int B, int Hq, int Hkv, int N, int D, int dtype, float sm_scale, float theta,
                   void* workspace, size_t workspace_bytes,
                   int* status_word, void* stream);

/* corope_gqa_fwd with every tensor's own {batch, head, row} strides (the q, k, v, o fields of `strides`, in elements; NULL =
 * contiguous).  Replaces the stride arguments of the reference's kernel launch (flash_attn_co_rope_gqa_triton.py:439-442).
 * The tensor-core kernels run when all pointers and strides are multiples of 16 bytes, the CUDA-core kernels otherwise. */
int corope_gqa_fwd_strided(const void* q, const void* k, const void* v,
                           void* o, float* lse2, float* a_diag,
                           int B, int Hq, int Hkv, int N, int D, int dtype, float sm_scale, float theta,
                           void* workspace, size_t workspace_bytes,
                           int* status_word, void* stream, const corope_strides_t* strides);

/*
 * Co-RoPE GQA attention backward.  Replaces _attention.backward
 * (corope-exp/flash_attn_co_rope_gqa_triton.py:459-577, dense PyTorch there); the math is that of
 * corope-exp/corope_attn_gqa_pytorch.py:138-300.  dk/dv are [B,Hkv,N,D] (summed over the group).
 */
int corope_gqa_bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                   const float* lse2, const float* a_diag,
                   void* dq, void* dk, void* dv,
                   int B, int Hq, int Hkv, int N, int D, int dtype, float sm_scale, float theta,
                   void* workspace, size_t workspace_bytes,
                   int* status_word, void* stream);

/* corope_gqa_bwd with every tensor's own strides (all eight fields of `strides`; NULL = contiguous). */
int corope_gqa_bwd_strided(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                           const float* lse2, const float* a_diag,
                           void* dq, void* dk, void* dv,
                           int B, int Hq, int Hkv, int N, int D, int dtype, float sm_scale, float theta,
                           void* workspace, size_t workspace_bytes,
                           int* status_word, void* stream, const corope_strides_t* strides);

/*
 * ---- Paged key / value cache with 8-bit codes -----------------------------------------------------------------------------
 *
 * What generation needs next to the attention above: keys and values of the tokens so far, one byte per element, in blocks of
 * `block_size` tokens that sequences own through a block table; a code c of block p and head h stands for c * scale[p][h].
 * No counterpart in the reference, which has no cache; the rotation is that of the fused-RoPE attention (half layout, tables with
 * columns [0, D/2) read), applied to keys before they are stored and to queries when they are read.
 *
 * All index arrays are device memory and are never read on the host.  An entry that points outside its tensor (a block id outside
 * [0, num_blocks), a length beyond the block table or below 0, a position beyond the tables) is not followed: the tokens concerned are
 * left out (a position is clamped; a sequence whose length or number of new tokens is out of range stores nothing, while attention and
 * eviction clamp the number) and COROPE_DEV_BAD_INDEX is added to the status word.  These kernels run whatever an earlier kernel left in
 * the word, but for those of corope_cache_attn with waits of their own (16-bit tensors, more than 32 query rows a K / V head), which do not after
 * COROPE_DEV_WAIT_EXPIRED.  They take fp32 / bf16 / fp16 tensors, hold scores, sums and scales in fp32 and have no backward pass.  Scales are
 * not negative.
 */
#define COROPE_CODE_E4M3 0   /* 8-bit floats, largest finite value 448 */
#define COROPE_CODE_INT8 1   /* whole numbers -127 .. 127 */

typedef struct corope_kv_cache_t {
    void *k, *v;                   /* codes [num_blocks, Hkv, block_size, D], 16-byte aligned */
    float *k_scale, *v_scale;      /* [num_blocks, Hkv] contiguous */
    float* weight;                 /* [num_blocks, Hkv, block_size] contiguous, accumulated attention weight of each slot, or NULL */
    int64_t k_stride[3], v_stride[3];   /* {block, head, row} in elements, multiples of 16; 0 for blocks or heads only where nothing is written */
    int num_blocks, Hkv, block_size, D; /* block_size 16, 32, 64, 128 or 256; D 32, 64 or 128 */
    int code;                      /* COROPE_CODE_* */
} corope_kv_cache_t;

typedef struct corope_cache_seqs_t {
    const int* block_table;        /* [B, max_blocks]: block_table[b * table_stride + i] holds slots i * block_size .. of sequence b */
    int64_t table_stride;
    int B, max_blocks;
    const int* seq_lens;           /* [B] tokens in the cache, those of this call included */
    const int* new_lens;           /* [B] tokens of this call, at most T, or NULL = T each */
    const int* positions;          /* [B] position of the first token of this call, or NULL = its slot */
    const float *cos, *sin;        /* [table_rows, D/2 or more], or NULL = no rotation */
    int64_t rope_stride;
    int table_rows;
} corope_cache_seqs_t;

/*
 * Stores n = new_lens[b] tokens of k, v [B, Hkv, T, D] (strides {batch, head, row} in elements) in slots seq_lens[b] - n .. of each
 * sequence, keys rotated; a token whose slot would be negative is left out, slots behind and blocks without a new token stay as they were.
 *   scale of a block: max(its scale so far, if it holds older tokens; largest |finite new element| * r), r = the fp32 number next to 1/448 or 1/127
 *   code = x / scale rounded to nearest even, saturated; NaN stays NaN (e4m3) or becomes 0 (int8); a scale of 0 has codes 0
 * Older codes of a block whose scale grows are written again for the new one.  weight (if any) of the new slots becomes 0.
 * A block that a token is written to must stand in one place of the block table only.
 */
int corope_cache_append(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const void* k, const void* v, const int64_t k_strides[3],
                        const int64_t v_strides[3], int T, int dtype, int* status_word, void* stream);

/*
 * Attention of q [B, Hq, T, D] over the cache: query t < n of sequence b (its last n tokens) sees slots below
 * seq_lens[b] - n + t + 1 (causal) or all seq_lens[b].  Query head h reads K / V head h / (Hq / Hkv), any group size.  o [B, Hq, T, D] in
 * `dtype`; rows without a visible slot and rows t >= n are 0, whatever their query and position.  accumulate: weight[slot] += the slot's probabilities summed over
 * the queries and the heads of its group.  Scores have fp32 accuracy; for bf16 tensors of more than 32 query rows a K / V head without `accumulate`
 * the rotated queries are rounded to 11 bits first.  Probabilities are rounded to 11 bits for 16-bit tensors, to 22 for fp32 ones, and where they are
 * far below a row's largest to 2^-25 of it.  Sums over long contexts are added in fp32, in pieces of 1024 steps of the tensor cores (which truncate).
 * Values of a block whose scale of V is below 1e-30 (the largest is then below 4.5e-28) count as 0.
 * The workspace (ask with the call's own arguments and the same current device): parts of results, with `accumulate` also 4 bytes per slot of the
 * block tables and query row (where that is at most 512 MiB), for more than 32 rows fp16 copies of q.
 */
size_t corope_cache_attn_workspace_bytes(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, int Hq, int T, int dtype, int accumulate);
int corope_cache_attn(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const void* q, void* o, const int64_t q_strides[3],
                      const int64_t o_strides[3], int Hq, int T, int dtype, int causal, float sm_scale, int accumulate, void* workspace,
                      size_t workspace_bytes, int* status_word, void* stream);

/*
 * Thins each head's cache to `budget` slots: the last `recent` ones and, of the others, those of largest weight (equal weights: the
 * lowest slot; NaN counts as the largest).  The slots kept move in order to slots 0 .. of the blocks in out_table [B, out_blocks], weights
 * too; sequences of at most `budget` tokens move whole.  A new block's scale is the largest scale of the blocks its slots come from: codes of
 * that scale move bit for bit, the others become code * scale / new scale, rounded.  Reads seq_lens and block_table of `seqs` only;
 * out_table's blocks belong to one sequence each and to no block_table row of the call; source blocks are not written, they may be shared.
 *   new_lens [B] = min(seq_lens, budget);  kept [B, Hkv, budget] = the slots kept, ascending, -1 behind them.
 */
int corope_cache_evict(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const int* out_table, int64_t out_table_stride, int out_blocks,
                       int budget, int recent, int* new_lens, int* kept, int* status_word, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* COROPE_B200_H_ */
