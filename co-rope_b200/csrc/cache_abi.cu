// extern "C" entry points of the 8-bit paged cache: argument checks and the kernels' parameters.
#include "cache.cuh"

using namespace corope;

namespace {

Strides bytes_of(const int64_t (&a)[3]) { return Strides{a[0], a[1], a[2]}; }
Strides strides_of(const int64_t* a) { return Strides{a[0], a[1], a[2]}; }

// rows of codes move in 16-byte runs
bool cache_rows_ok(const void* ptr, const Strides& st, int D) {
    return (uintptr_t)ptr % 16 == 0 && st.b % 16 == 0 && st.h % 16 == 0 && st.n % 16 == 0 && st.n >= D && st.b >= 0 && st.h >= 0 &&
           st.b < (1ll << 32) && st.n < (1ll << 32);   // (strides are 32-bit numbers in the kernels)
}

// blocks and heads have codes of their own, as who writes them needs
bool cache_rows_apart(const corope_kv_cache_t* c, const int64_t* st) { return (c->num_blocks == 1 || st[0] > 0) && (c->Hkv == 1 || st[1] > 0); }

int view_of(CacheView& v, const corope_kv_cache_t* c, bool written) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return COROPE_ERR_NULL_POINTER;
    if (c->num_blocks <= 0 || c->Hkv <= 0) return COROPE_ERR_BAD_SHAPE;
    if (c->D != 32 && c->D != 64 && c->D != 128) return COROPE_ERR_BAD_HEAD_DIM;
    int log2 = 4;
    while (log2 < 8 && (1 << log2) != c->block_size) ++log2;
    if ((1 << log2) != c->block_size) return COROPE_ERR_BAD_CACHE;
    if (c->code != COROPE_CODE_E4M3 && c->code != COROPE_CODE_INT8) return COROPE_ERR_BAD_CACHE;
    v.k = static_cast<uint8_t*>(c->k); v.v = static_cast<uint8_t*>(c->v);
    v.k_scale = c->k_scale; v.v_scale = c->v_scale; v.weight = c->weight;
    v.sk = bytes_of(c->k_stride); v.sv = bytes_of(c->v_stride);
    v.num_blocks = c->num_blocks; v.Hkv = c->Hkv; v.bs_log2 = log2;
    if (!cache_rows_ok(c->k, v.sk, c->D) || !cache_rows_ok(c->v, v.sv, c->D)) return COROPE_ERR_BAD_CACHE;
    if (written && !(cache_rows_apart(c, c->k_stride) && cache_rows_apart(c, c->v_stride))) return COROPE_ERR_BAD_CACHE;
    return COROPE_OK;
}

int view_of(SeqView& v, const corope_cache_seqs_t* q, const CacheView& c, int D) {
    if (!q || !q->block_table || !q->seq_lens) return COROPE_ERR_NULL_POINTER;
    if ((q->cos == nullptr) != (q->sin == nullptr)) return COROPE_ERR_NULL_POINTER;
    if (q->B <= 0 || q->max_blocks <= 0) return COROPE_ERR_BAD_SHAPE;
    if (q->table_stride < (q->B > 1 ? q->max_blocks : 0)) return COROPE_ERR_BAD_STRIDE;
    if (q->cos && (q->table_rows <= 0)) return COROPE_ERR_BAD_SHAPE;
    if (q->cos && q->table_rows > 1 && q->rope_stride < D / 2) return COROPE_ERR_BAD_STRIDE;
    // slots and rows are 32-bit numbers in the kernels
    if (((uint64_t)q->max_blocks << c.bs_log2) >= (1ull << 30) || (uint64_t)q->B * c.Hkv >= (1ull << 24)) return COROPE_ERR_TOO_LARGE;
    v.table = q->block_table; v.table_stride = q->table_stride; v.B = q->B; v.max_blocks = q->max_blocks;
    v.lens = q->seq_lens; v.new_lens = q->new_lens; v.positions = q->positions;
    v.cos = q->cos; v.sin = q->sin; v.rope_stride = q->rope_stride; v.table_rows = q->table_rows;
    return COROPE_OK;
}

bool dtype_ok(int dtype) { return dtype == COROPE_DTYPE_F32 || dtype == COROPE_DTYPE_BF16 || dtype == COROPE_DTYPE_F16; }
int rows_ok(const int64_t* st) { return st[0] >= 0 && st[1] >= 0 && st[2] >= 0; }

int tokens_ok(int T) { return T <= 0 ? COROPE_ERR_BAD_SHAPE : T > (1 << 20) ? COROPE_ERR_TOO_LARGE : COROPE_OK; }

int attn_sizes(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, int Hq, int T) {
    if (int e = tokens_ok(T)) return e;
    if (Hq <= 0) return COROPE_ERR_BAD_SHAPE;
    if (Hq % cache->Hkv != 0) return COROPE_ERR_BAD_GROUP;
    if ((uint64_t)seqs->B * Hq * T >= (1ull << 30)) return COROPE_ERR_TOO_LARGE;
    return COROPE_OK;
}

}  // namespace

extern "C" {

int corope_cache_append(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const void* k, const void* v, const int64_t k_strides[3],
                        const int64_t v_strides[3], int T, int dtype, int* status_word, void* stream) {
    if (!k || !v || !k_strides || !v_strides) return COROPE_ERR_NULL_POINTER;
    CacheAppendParams p{};
    if (int e = view_of(p.c, cache, true)) return e;
    if (int e = view_of(p.s, seqs, p.c, cache->D)) return e;
    if (int e = tokens_ok(T)) return e;
    if (!dtype_ok(dtype)) return COROPE_ERR_BAD_DTYPE;
    if (!rows_ok(k_strides) || !rows_ok(v_strides)) return COROPE_ERR_BAD_STRIDE;
    p.k = k; p.v = v; p.sk = strides_of(k_strides); p.sv = strides_of(v_strides);
    p.T = T; p.D = cache->D; p.code = cache->code; p.dtype = dtype;
    p.status = status_word; p.mirror = status_mirror_of(status_word);
    return launch_cache_append(p, (cudaStream_t)stream);
}

size_t corope_cache_attn_workspace_bytes(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, int Hq, int T, int dtype, int accumulate) {
    CacheAttnParams p{};
    if (view_of(p.c, cache, false) || view_of(p.s, seqs, p.c, cache->D) || attn_sizes(cache, seqs, Hq, T)) return 0;
    return cache_attn_workspace_bytes(seqs->B, cache->Hkv, Hq / cache->Hkv, T, cache->D, seqs->max_blocks, cache->block_size, dtype, accumulate);
}

int corope_cache_attn(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const void* q, void* o, const int64_t q_strides[3],
                      const int64_t o_strides[3], int Hq, int T, int dtype, int causal, float sm_scale, int accumulate, void* workspace,
                      size_t workspace_bytes, int* status_word, void* stream) {
    if (!q || !o || !q_strides || !o_strides) return COROPE_ERR_NULL_POINTER;
    CacheAttnParams p{};
    if (int e = view_of(p.c, cache, false)) return e;
    if (int e = view_of(p.s, seqs, p.c, cache->D)) return e;
    if (int e = attn_sizes(cache, seqs, Hq, T)) return e;
    if (!dtype_ok(dtype)) return COROPE_ERR_BAD_DTYPE;
    if (accumulate && !cache->weight) return COROPE_ERR_NULL_POINTER;
    if (!rows_ok(q_strides) || !rows_ok(o_strides)) return COROPE_ERR_BAD_STRIDE;
    p.q = q; p.o = o; p.sq = strides_of(q_strides); p.so = strides_of(o_strides);
    p.Hq = Hq; p.G = Hq / cache->Hkv; p.T = T; p.D = cache->D; p.code = cache->code; p.dtype = dtype;
    p.causal = causal ? 1 : 0; p.accumulate = accumulate ? 1 : 0;
    p.scale = (float)((double)sm_scale * 1.4426950408889634);
    const size_t need = cache_attn_workspace_bytes(seqs->B, cache->Hkv, p.G, T, cache->D, seqs->max_blocks, cache->block_size, dtype, accumulate);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256 != 0) return COROPE_ERR_WORKSPACE;
    p.status = status_word; p.mirror = status_mirror_of(status_word);
    return launch_cache_attn(p, workspace, (cudaStream_t)stream);
}

int corope_cache_evict(const corope_kv_cache_t* cache, const corope_cache_seqs_t* seqs, const int* out_table, int64_t out_table_stride, int out_blocks,
                       int budget, int recent, int* new_lens, int* kept, int* status_word, void* stream) {
    if (!out_table || !new_lens || !kept) return COROPE_ERR_NULL_POINTER;
    CacheEvictParams p{};
    if (int e = view_of(p.c, cache, true)) return e;
    if (int e = view_of(p.s, seqs, p.c, cache->D)) return e;
    if (!cache->weight) return COROPE_ERR_NULL_POINTER;
    if (budget <= 0 || recent < 0 || recent > budget) return COROPE_ERR_BAD_SHAPE;
    if (budget >= (1 << 30)) return COROPE_ERR_TOO_LARGE;
    if (out_blocks <= 0 || ((int64_t)out_blocks << p.c.bs_log2) < budget) return COROPE_ERR_BAD_SHAPE;
    if (out_table_stride < (seqs->B > 1 ? out_blocks : 0)) return COROPE_ERR_BAD_STRIDE;
    p.out_table = out_table; p.out_stride = out_table_stride; p.out_blocks = out_blocks;
    p.budget = budget; p.recent = recent; p.D = cache->D; p.code = cache->code; p.new_lens = new_lens; p.kept = kept;
    p.status = status_word; p.mirror = status_mirror_of(status_word);
    return launch_cache_evict(p, (cudaStream_t)stream);
}

}  // extern "C"
