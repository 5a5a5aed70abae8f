"""Generation: a paged key / value cache with 8-bit codes, the append that fills it, the attention that reads it and its eviction.

    cache = KVCache(num_blocks, num_heads, block_size, head_dim, dtype=torch.float8_e4m3fn, weights=True)
    seq_lens += 1                                        # tokens in the cache, this step's included
    cache_append(k, v, cache, block_table, seq_lens, freqs_cos, freqs_sin, positions)
    o = cache_attention(q, cache, block_table, seq_lens, True, sm_scale, freqs_cos, freqs_sin, positions, accumulate=True)
    seq_lens, kept = cache_evict(cache, block_table, seq_lens, new_table, budget, recent)

The reference has no counterpart: its entry points are a training step's.  Rotation, head grouping (query head h reads K / V head
h // (Hq // Hkv)), layouts ([B, H, T, D], own strides) and dtypes (bf16, fp16, fp32) are those of fused_rope_attn.py and
flash_attn_v2_triton.py: what was trained through them is served through these.  Head dims 32, 64, 128.

A code c of block p and head h stands for c * scale[p, h].  Sequence b's slot s is in block block_table[b, s // block_size].
block_table [B, blocks], seq_lens, new_lens and positions [B] are int32 CUDA tensors; they are read on the device only, so a step
captured into a CUDA graph follows what they hold at replay.  An entry that points outside its tensor is not followed: the tokens
concerned are left out and the next call on the device raises RuntimeError.  (A length or a number of new tokens out of range: nothing
of the sequence is stored; attention and eviction take the nearest number in range, and so does a position.)  Block table
entries behind a sequence's last block are not read.  A place of a padded batch that holds no sequence has a length of 0.  No
operator has a backward pass: tensors that require a gradient are refused outside torch.no_grad(), duals of forward mode everywhere.
What an operator writes to in place counts as modified for autograd.
"""

import torch

try:
    from . import _ext
except ImportError:  # imported as a top-level module (directory on sys.path, the way the reference's scripts import it)
    import _ext


class KVCache:
    """Holds k, v [num_blocks, num_heads, block_size, head_dim] codes (float8_e4m3fn or int8), k_scale, v_scale [num_blocks,
    num_heads] fp32 and, with weights=True, weight [num_blocks, num_heads, block_size] fp32, the attention weight that each
    slot has gathered.  The operators take any object with these attributes (weight may be None), so that a program can
    keep them as views of its own buffers: rows need 16-byte alignment (and memory of their own where they are written to), the
    scales and weights have to be contiguous."""

    def __init__(self, num_blocks, num_heads, block_size, head_dim, dtype=torch.float8_e4m3fn, device="cuda", weights=False):
        shape = (num_blocks, num_heads, block_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        self.weight = torch.zeros(shape[:3], dtype=torch.float32, device=device) if weights else None


def cache_append(k, v, cache, block_table, seq_lens, freqs_cos=None, freqs_sin=None, positions=None, new_lens=None):
    """Stores k, v [B, Hkv, T, D]: the first n = new_lens[b] (default T) tokens of sequence b go to slots seq_lens[b] - n and on.

    freqs_cos / freqs_sin [N, D] or [N, D/2]: keys are rotated by row positions[b] + t of the tables (default: by the slot).
    A block's scale is the largest finite element it holds times 1 / 448 (e4m3) or 1 / 127 (int8), one for k and one for v; when a
    new token raises it, the block's older codes are written again.  Codes are x / scale rounded to nearest even; infinities
    saturate, NaN stays NaN in e4m3 and becomes 0 in int8; a scale of 0 has codes 0.  cache.weight of the new slots becomes 0.
    Blocks that are written to must stand in one place of block_table; full blocks may be shared."""
    _ext.native().cache_append(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight, block_table, seq_lens, freqs_cos, freqs_sin, positions, new_lens)


def cache_attention(q, cache, block_table, seq_lens, causal, sm_scale, freqs_cos=None, freqs_sin=None, positions=None, new_lens=None, accumulate=False):
    """Attention of q [B, Hq, T, D] over the cache -> o, laid out like q.

    Queries t < n = new_lens[b] (default T) belong to the last n tokens of sequence b: with `causal` query t sees slots below
    seq_lens[b] - n + t + 1, without it all of them.  Queries are rotated like the keys of cache_append.  Rows t >= n and rows that
    see nothing are 0.  V of a block whose scale is below 1e-30 counts as 0.  accumulate: cache.weight[slot] += the slot's probabilities, summed over the queries and the query heads of
    its K / V head (sequences that share a block all add to it, in any order)."""
    return _ext.native().cache_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight, block_table, seq_lens, causal, sm_scale, freqs_cos, freqs_sin,
                                         positions, new_lens, accumulate)


def cache_evict(cache, block_table, seq_lens, out_table, budget, recent=0):
    """Thins every sequence to `budget` slots a head -> (new_lens [B], kept [B, Hkv, budget] int32).

    Each K / V head keeps the last `recent` slots and the slots of largest cache.weight among the others (of equal weights the
    lowest slots; NaN counts as the largest).  They move in order, with their weights, to slots 0 .. of the blocks in out_table [B, blocks],
    which the caller takes from its pool: blocks of no other sequence and of no row of block_table.  Codes are kept bit for bit
    where a new block's scale, the largest among its slots' old ones, is their own, and rounded to it otherwise.  Sequences of at most
    `budget` tokens move whole.  Source blocks stay as they are, so they may be shared; afterwards the caller frees them.  kept lists the
    slots, ascending, -1 behind the last.  Tokens keep the rotation of their position: pass `positions` from then on, slots no longer tell."""
    return _ext.native().cache_evict(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight, block_table, seq_lens, out_table, budget, recent)
