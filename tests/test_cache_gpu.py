"""The 8-bit paged cache on the GPU against the CPU oracle (oracle/kv_cache_oracle.py): codes bit for bit, attention in 64 bits."""

import pytest
import torch

from helpers import draw, ext, pkg
from oracle import kv_cache_oracle as ref
from oracle import precompute_freqs_cis

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def make_cache(blocks, Hkv, bs, D, code, seed=0, weights=True, layout="hnd"):
    """(cache object on the GPU, its dict on the CPU): random codes and scales everywhere, as a pool in use has them."""
    cache = pkg.KVCache(blocks, Hkv, bs, D, dtype=code, weights=weights)
    if layout == "nhd":            # [blocks, block_size, Hkv, D] buffers
        cache.k, cache.v = (torch.zeros((blocks, bs, Hkv, D), dtype=torch.uint8, device="cuda").view(code).transpose(1, 2) for _ in range(2))
    elif layout == "pairs":        # keys and values of a block side by side in one buffer
        both = torch.zeros((blocks, 2, Hkv, bs, D), dtype=torch.uint8, device="cuda").view(code)
        cache.k, cache.v = both[:, 0], both[:, 1]
    host = {}
    for i, name in enumerate(("k", "v")):
        x = draw((blocks, Hkv, bs, D), seed + i, F32)
        scale = x.abs().amax(dim=(2, 3)) / ref.LARGEST[code] * (1.0 + torch.arange(blocks)[:, None] % 3)
        host[name] = ref.to_codes(x, scale[:, :, None, None], code)
        host[name + "_scale"] = scale
        getattr(cache, name).view(torch.uint8).copy_(host[name].view(torch.uint8).cuda())
        getattr(cache, name + "_scale").copy_(scale.cuda())
    host["weight"] = draw((blocks, Hkv, bs), seed + 2, F32).exp() if weights else None
    if weights:
        cache.weight.copy_(host["weight"].cuda())
    return cache, host


def make_table(B, wide, blocks, lens, bs, seed=0, behind=-1):
    """Blocks in any order; `behind` stands where a sequence has none."""
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[:B * wide].view(B, wide).to(torch.int32)
    used = torch.arange(wide)[None] * bs < torch.as_tensor(lens)[:, None]
    return torch.where(used, order, torch.full((), behind, dtype=torch.int32)).contiguous()


def gpu(*ts):
    return [None if t is None else t.cuda() for t in ts]


def same_cache(cache, host):
    for name in ("k", "v"):
        got, want = getattr(cache, name).cpu(), host[name]
        if got.dtype == E4M3:
            got, want = got.float(), want.float()
            assert torch.equal(got.isnan(), want.isnan()), name
            got, want = got.nan_to_num(), want.nan_to_num()
        assert torch.equal(got, want), (name, (got != want).nonzero()[:5])
        got, want = getattr(cache, name + "_scale").cpu(), host[name + "_scale"]
        assert torch.equal(got, want), (name + "_scale", got - want)
    if host["weight"] is not None:
        assert torch.equal(cache.weight.cpu(), host["weight"])


# ------------------------------------------------------------------------------------------------------------------ append
APPENDS = [
    # lens (this call's tokens included), new tokens, T, Hkv, D, bs, dtype, code, rope
    ([1, 17, 64, 0], None, 1, 2, 128, 16, BF16, E4M3, True),
    ([5, 16, 33], [5, 0, 3], 5, 3, 64, 16, F16, INT8, True),
    ([100, 70], [100, 7], 100, 2, 32, 64, F32, E4M3, True),
    ([130, 257, 64], [129, 33, 64], 129, 1, 128, 32, BF16, INT8, False),
    ([300, 255], None, 255, 2, 64, 256, F16, E4M3, True),
    ([40, 3], None, 40, 2, 32, 16, F32, INT8, False),      # 3 tokens of 40: the first 37 have no slot
]


@pytest.mark.parametrize("lens,new,T,Hkv,D,bs,dtype,code,rope", APPENDS)
def test_append(lens, new, T, Hkv, D, bs, dtype, code, rope):
    B, wide = len(lens), 300 // bs + 2
    blocks = B * wide + 1
    cache, host = make_cache(blocks, Hkv, bs, D, code, weights=dtype != F32)
    table = make_table(B, wide, blocks, lens, bs)
    k, v = draw((B, Hkv, T, D), 5, dtype), 3 * draw((B, Hkv, T, D), 6, dtype)
    cos, sin = precompute_freqs_cis(D, 400, 10000.0) if rope else (None, None)
    positions = ints([max(n - T, 0) + 7 * i for i, n in enumerate(lens)]) if rope and new is None else None
    if new is None and positions is not None and lens[-1] == 3:
        positions = None
    new_lens = None if new is None else ints(new)
    ref.append(host, k, v, table, lens, cos, sin, positions, new)
    pkg.cache_append(*gpu(k, v), cache, *gpu(table, ints(lens), cos, sin, positions, new_lens))
    pkg.check_status()
    same_cache(cache, host)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_token_by_token(code):
    """Blocks fill up, scales grow and older codes are written again; a second call with the same tokens changes nothing."""
    B, Hkv, D, bs = 2, 2, 64, 16
    cache, host = make_cache(9, Hkv, bs, D, code)
    table = make_table(B, 4, 9, [50, 50], bs)
    for step in range(20):
        lens = [step + 1, step + 30]
        k, v = (draw((B, Hkv, 1, D), 10 * step + i, BF16) * (1 + step % 7) for i in range(2))
        for _ in range(2):
            pkg.cache_append(*gpu(k, v), cache, *gpu(table, ints(lens)))
        ref.append(host, k, v, table, lens)
    pkg.check_status()
    same_cache(cache, host)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_odd_numbers(code):
    """Infinities saturate, NaN stays NaN or becomes 0, neither touches the scale; rows of zeros; numbers next to the smallest normal one."""
    D, bs = 32, 16
    cache, host = make_cache(4, 1, bs, D, code)
    k = draw((3, 1, 4, D), 1, F32)
    k[0, 0, 1, 3], k[0, 0, 2, 5], k[0, 0, 3, 7] = float("inf"), float("-inf"), float("nan")
    k[1] = 0.0
    k[2] *= 2.0 ** -120
    v = k.flip(0).contiguous()
    table, lens = make_table(3, 1, 4, [4, 4, 4], bs), [4, 4, 4]
    ref.append(host, k, v, table, lens)
    pkg.cache_append(*gpu(k, v), cache, *gpu(table, ints(lens)))
    pkg.check_status()
    same_cache(cache, host)


@pytest.mark.parametrize("kind", ["bnhd", "slice", "odd", "shared", "reversed"])
def test_append_layouts(kind):
    """Projections' own layout, rows inside wider ones, rows off any alignment, one head shared by all, a head dimension without unit stride."""
    B, Hkv, T, D, bs = 2, 3, 21, 64, 16
    wide = draw((B, T, Hkv, 2 * D + 8), 3, F16)
    k = {"bnhd": wide[..., :D].contiguous().transpose(1, 2), "slice": wide[..., 8:8 + D].transpose(1, 2), "odd": wide[..., 1:1 + D].transpose(1, 2),
         "shared": wide[:, :, :1, :D].transpose(1, 2).expand(B, Hkv, T, D), "reversed": wide[..., :2 * D:2].transpose(1, 2)}[kind]
    v = wide[..., D:2 * D].transpose(1, 2)
    cos, sin = precompute_freqs_cis(D, 60, 10000.0)
    if kind == "odd":
        cos, sin = torch.cat((cos, cos[:, :1]), dim=1)[:, :D], torch.cat((sin, sin[:, :1]), dim=1)[:, :D]
    for layout in ("nhd", "pairs"):
        cache, host = make_cache(7, Hkv, bs, D, E4M3, layout=layout)
        table, lens = make_table(B, 3, 7, [33, 40], bs), [33, 40]
        ref.append(host, k.contiguous(), v.contiguous(), table, lens, cos, sin)
        wide_g = wide.cuda()
        kg = k.cuda() if kind in ("bnhd", "shared") else torch.as_strided(wide_g, k.shape, k.stride(), k.storage_offset())
        pkg.cache_append(kg, torch.as_strided(wide_g, v.shape, v.stride(), v.storage_offset()), cache, *gpu(table, ints(lens), cos, sin))
        pkg.check_status()
        same_cache(cache, host)


# --------------------------------------------------------------------------------------------------------------- attention
def tolerance(dtype, o, bulk, slack, one_part=False):
    """What o may be off, element by element.

    s: its terms' sum, `slack` (natural units), is rounded by the split of q (2 parts of 11 bits: 2^-21), by the fp32 sums of 2 D <= 256 products
    in MMA steps of 16 (some 2^-24 each, truncated: 32 steps of 2^-23) and by the arithmetic of exp2 (argument up to 2 slack, 2^-22): below
    2^-17 slack.  (one_part: bf16 calls of more than 32 query rows a head without weights round the rotated q to 11 bits, another 2^-11 slack.)  A
    probability is off by at most twice that (its own score and the normalisation), and by fp16's half step 2^-11 where p is rounded
    to fp16 (2^-21 for fp32's two parts); sums of p |v| are `bulk`; the MMA's long fp32 sums truncate: 2^-23 for each of up to 64 steps.
    The result is rounded to its type: eps / 2 of it, and below the smallest normal number `tiny` half the subnormals' step tiny * eps (f16:
    2^-14 * 2^-10 / 2 = 2^-25)."""
    p = 2 * (2.0 ** -17 + (2.0 ** -11 if one_part else 0.0)) * slack + (2.0 ** -21 if dtype == F32 else 2.0 ** -11) + 64 * 2.0 ** -23
    return torch.finfo(dtype).eps / 2 * o.abs().clamp(min=torch.finfo(dtype).tiny) + 1.01 * p * bulk


def check_attention(cache, host, q, table, lens, causal, sm_scale, cos=None, sin=None, positions=None, new_lens=None, accumulate=False, q_gpu=None):
    o, bulk, slack, weight = ref.attention(host, q, table, lens, causal, sm_scale, cos, sin, positions, new_lens)
    got = pkg.cache_attention(q.cuda() if q_gpu is None else q_gpu, cache, *gpu(table, ints(lens)), causal, sm_scale, *gpu(cos, sin, positions), new_lens=None if new_lens is None else
                              ints(new_lens).cuda(), accumulate=accumulate)
    pkg.check_status()
    assert got.dtype == q.dtype and got.shape == q.shape
    one_part = q.dtype == BF16 and not accumulate and q.shape[1] // host["k"].shape[1] * q.shape[2] > 32
    excess = (got.double().cpu() - o).abs() - tolerance(q.dtype, o, bulk, slack, one_part)
    assert not (excess > 0).any() and not got.isnan().any(), excess.max()
    assert torch.equal(got.cpu()[bulk == 0].float(), torch.zeros_like(got.cpu()[bulk == 0].float()))
    if accumulate:
        rows = q.shape[1] // host["k"].shape[1] * q.shape[2] * len(lens)
        off = (cache.weight.double().cpu() - host["weight"].double() - weight).abs()
        # each probability is off by 2 * 2^-17 slack, the sums of up to `rows` of them and the addition by an fp32 step each
        allowed = 2 * 2.0 ** -17 * slack.max() * weight + (rows + 2) * 2.0 ** -23 * (host["weight"].double() + weight)
        assert not (off > allowed).any(), (off - allowed).max()
    return got


ATTENDS = [
    # lens, new tokens, T, Hkv, G, D, bs, dtype, code, rope, causal, accumulate
    ([1, 2, 15, 16, 17, 0], None, 1, 2, 4, 128, 16, BF16, E4M3, True, True, True),
    ([63, 64, 65, 500], None, 1, 1, 8, 128, 64, F16, INT8, True, True, True),
    ([300], None, 1, 3, 1, 64, 32, F32, INT8, True, True, True),
    ([129, 255, 7], None, 1, 2, 3, 32, 256, F32, E4M3, False, True, False),
    ([40, 90, 3], [4, 1, 3], 4, 2, 4, 128, 16, BF16, E4M3, True, True, True),      # 16 rows a head
    ([40, 90, 3], [5, 0, 3], 5, 1, 5, 64, 16, F32, INT8, True, True, True),        # 25 rows: tiles of 32
    ([200, 33], [33, 20], 33, 2, 3, 64, 32, F16, E4M3, True, True, True),          # several tiles
    ([200, 33], None, 12, 1, 12, 128, 128, F32, E4M3, True, False, True),
    ([70, 5], None, 9, 2, 1, 32, 16, BF16, INT8, False, True, True),               # 5 tokens, 9 queries: 4 rows see nothing
    ([90, 61], None, 61, 1, 2, 128, 64, F16, INT8, True, False, False),
    ([2300, 1], None, 1, 2, 12, 64, 16, BF16, E4M3, True, True, True),
    ([140, 160], [130, 160], 160, 1, 4, 128, 64, BF16, E4M3, True, True, True),    # a chunk: 640 rows a head
    ([1031], None, 200, 2, 3, 64, 32, F16, INT8, True, True, False),
    ([300, 77], [65, 64], 65, 1, 2, 32, 16, F32, E4M3, True, True, True),
    ([2500, 1900, 0], [200, 131, 0], 200, 2, 4, 64, 32, F16, E4M3, True, True, True),    # hundreds of 128 x 128 units: several a block, pieces of items
    ([5000, 4000], [70, 300], 300, 2, 1, 128, 16, BF16, INT8, True, True, True),
    ([1500], None, 300, 5, 2, 32, 128, F16, INT8, False, False, True),
    ([700, 260], [100, 130], 130, 2, 3, 128, 64, BF16, E4M3, True, True, False),     # one part of q, two tiles of rows an item
    ([700, 64], [30, 20], 30, 2, 4, 64, 32, BF16, INT8, True, True, False),          # one part, one tile
]


@pytest.mark.parametrize("lens,new,T,Hkv,G,D,bs,dtype,code,rope,causal,accumulate", ATTENDS)
def test_attention(lens, new, T, Hkv, G, D, bs, dtype, code, rope, causal, accumulate):
    B, wide = len(lens), max(lens) // bs + 2
    blocks = B * wide + 1
    cache, host = make_cache(blocks, Hkv, bs, D, code)
    table = make_table(B, wide, blocks, lens, bs)
    q = 2 * draw((B, Hkv * G, T, D), 9, dtype)
    cos, sin = precompute_freqs_cis(D, max(lens) + T + 100, 10000.0) if rope else (None, None)
    positions = ints([n + 3 * i for i, n in enumerate(lens)]) if rope and dtype != F16 else None
    if rope and positions is None and any(n < (T if new is None else new[i]) for i, n in enumerate(lens)):
        positions = ints([0] * B)
    check_attention(cache, host, q, table, lens, causal, D ** -0.5, cos, sin, positions, new, accumulate)


@pytest.mark.parametrize("layout", ["nhd", "pairs"])
@pytest.mark.parametrize("kind", ["bnhd", "odd", "shared"])
def test_attention_layouts(layout, kind):
    B, Hkv, G, T, D, bs, lens = 2, 2, 2, 3, 64, 16, [50, 20]
    cache, host = make_cache(9, Hkv, bs, D, INT8, layout=layout)
    table = make_table(B, 4, 9, lens, bs)
    wide = draw((B, T, Hkv * G, D + 8), 4, BF16)
    q = {"bnhd": wide[..., :D].contiguous().transpose(1, 2), "odd": wide[..., 1:1 + D].transpose(1, 2), "shared": wide[:, :, :1, :D].transpose(1, 2).expand(B, Hkv * G, T, D)}[kind]
    q_gpu = torch.as_strided(wide.cuda(), q.shape, q.stride(), q.storage_offset()) if kind == "odd" else None
    check_attention(cache, host, q, table, lens, True, 0.2, accumulate=True, q_gpu=q_gpu)


@pytest.mark.parametrize("strides", [(1000, 300, 1, 1), (1, 1, 1, 1), (64, 1, 2, 1), (0, 0, 1, 1), (0, 1, 0, 1), (7, 1, 3, 1)])
@pytest.mark.parametrize("T,dtype", [(1, F32), (3, BF16), (20, F16)])
def test_queries_that_overlap(T, dtype, strides):
    """Windows that slide over one row: what lies next to what in q says nothing about o."""
    B, Hq, D, bs, lens = 2, 4, 64, 16, [50, 30]
    cache, host = make_cache(9, 2, bs, D, INT8)
    table = make_table(B, 4, 9, lens, bs)
    row = draw((4000,), 4, dtype)
    q = row.as_strided((B, Hq, T, D), strides)
    check_attention(cache, host, q.contiguous(), table, lens, True, 0.2, q_gpu=row.cuda().as_strided((B, Hq, T, D), strides))


def shared_context(B, S, D, code, bs=256):
    """A cache of one sequence of S tokens that B sequences read, with their table."""
    cache, host = make_cache(S // bs, 1, bs, D, code)
    return cache, host, torch.arange(S // bs, dtype=torch.int32)[None].expand(B, -1).contiguous()


def long_attention(host, q, rows, length, causal, sm_scale):
    """(o, bulk, slack) as the oracle's, of rows `rows` of one sequence's q [Hq, T, D] over the first `length` tokens of the one K / V head, in 64 bits on the GPU."""
    k, v = ((host[x].view(torch.uint8).cuda().view(host[x].dtype).double() * host[x + "_scale"].cuda().double()[:, :, None, None])[:, 0].flatten(0, 1)[:length] for x in ("k", "v"))
    T, q = q.shape[1], q[:, rows].double()
    sees = torch.tensor([length - T + t + 1 if causal else length for t in rows], device="cuda")[:, None]
    hidden = torch.arange(length, device="cuda") >= sees
    p = torch.softmax((q @ k.T * sm_scale).masked_fill(hidden, float("-inf")), dim=-1).nan_to_num(0.0)
    return p @ v, p @ v.abs(), (q.abs() @ k.abs().T * sm_scale).masked_fill(hidden, 0.0).amax(dim=-1, keepdim=True)


@pytest.mark.parametrize("B,G,T,dtype,S,causal", [
    (600, 1, 1, F16, 2 ** 20, False), (600, 1, 1, BF16, 2 ** 20, False), (150, 2, 64, F16, 2 ** 19, False), (150, 1, 33, F16, 2 ** 19, True), (150, 2, 65, BF16, 2 ** 19, True),
])
def test_long_sums_are_not_truncated(B, G, T, dtype, S, causal):
    """Values of one sign and equal weights over a context that one block of threads goes through: rounding errors of single results go up and down,
    so the mean of many shows what is lost in adding.  Allowed are 2^-13 (1024 additions that truncate by up to 2^-23 each, at all lengths) and for the mean
    of over 64 roundings by up to eps / 2 each five of its standard deviations, 5 * eps / 2 / sqrt(3 * 64) < 0.37 * eps / 2."""
    D = 64
    cache, host, table = shared_context(B, S, D, INT8)
    gen = torch.Generator().manual_seed(7)
    host["v"] = torch.randint(64, 128, host["v"].shape, generator=gen, dtype=torch.int8)
    host["v_scale"] = torch.full_like(host["v_scale"], 1 / 127)
    cache.v.copy_(host["v"].cuda())
    cache.v_scale.copy_(host["v_scale"].cuda())
    q = (draw((B, G, T, D), 1, F32) / 100).to(dtype).cuda()
    got = pkg.cache_attention(q, cache, table.cuda(), torch.full((B,), S, dtype=torch.int32, device="cuda"), causal, 0.1)
    pkg.check_status()
    for b in (0, B // 2, B - 1):
        o, _, _ = long_attention(host, q[b], [T - 1], S, causal, 0.1)
        off = ((got[b, :, -1:].double() - o) / o).mean().abs()
        assert off < 2.0 ** -13 + 0.37 * torch.finfo(dtype).eps / 2, off


@pytest.mark.parametrize("B,G,T,D,dtype,code,most,causal", [
    (700, 2, 1, 64, F16, E4M3, 150000, True), (700, 1, 3, 32, F32, INT8, 140000, True), (160, 5, 4, 32, BF16, E4M3, 700000, False), (300, 4, 8, 32, F32, INT8, 150000, True),
    (160, 1, 64, 32, F16, INT8, 60000, True), (160, 1, 140, 64, BF16, E4M3, 50000, True), (150, 2, 200, 32, F16, E4M3, 60000, True), (160, 1, 40, 128, F16, INT8, 50000, False),
    (40, 1, 3000, 32, BF16, INT8, 40000, True),
])
def test_shares_in_several_pieces(B, G, T, D, dtype, code, most, causal):
    """Blocks of threads that go through more of an item than is added in one sum: whole items, ends, beginnings and middles of them."""
    S = -(-most // 256) * 256
    cache, host, table = shared_context(B, S, D, code)
    lens = torch.randint(most // 2, most + 1, (B,), generator=torch.Generator().manual_seed(B + T), dtype=torch.int32)
    lens[0], lens[1], lens[-1] = most, 5, most - 300
    q = draw((B, G, T, D), 1, dtype).cuda()
    cache.weight.zero_()
    accumulate = T <= 4
    got = pkg.cache_attention(q, cache, *gpu(table, lens), causal, 0.2, accumulate=accumulate)
    pkg.check_status()
    one_part = dtype == BF16 and not accumulate and G * T > 32
    # beside the usual: 1024 truncating additions, or (fp32) 2^12 that round, which go up and down: 5 * 2^-24 * sqrt(2^12 / 3) < 2^-16
    adding = 2.0 ** -16 if dtype == F32 else 2.0 ** -13
    for b in [0, 1, B - 1] + list(range(2, B - 1, max(B // 9, 1))):
        rows = sorted({0, T // 2, T - 1})
        o, bulk, slack = long_attention(host, q[b], rows, int(lens[b]), causal, 0.2)
        x = got[b][:, rows].double()
        assert not ((x - o).abs() > tolerance(dtype, o, bulk, slack, one_part) + adding * bulk).any() and not x.isnan().any(), b
    if accumulate:   # every row that sees something has probabilities of 1 in all; 2^-10 of it covers 2 * 2^-17 of a score of below 60
        rows = sum(min(T, int(n)) if causal else T for n in lens) * G
        assert abs(cache.weight.double().sum().item() / rows - 1) < 2.0 ** -10


@pytest.mark.parametrize("dtype,T,G", [(BF16, 1, 4), (F32, 1, 4), (F16, 100, 4)])
def test_attention_extremes(dtype, T, G):
    """Scores of some hundred (one slot has all the weight), equal scores, blocks whose scales differ by 2^20, scales of 0."""
    D, bs, lens = 64, 16, [90 + T, 40 + T]
    cache, host = make_cache(40, 1, bs, D, E4M3)
    table = make_table(2, 13, 40, lens, bs)
    for x, name in ((cache.k_scale, "k_scale"), (cache.v_scale, "v_scale")):
        host[name] *= torch.exp2((torch.arange(40) % 5 * 5 - 10.0))[:, None] if name == "v_scale" else 1.0
        host[name][int(table[0, 1])] = 0.0
        x.copy_(host[name].cuda())
    q = draw((2, G, T, D), 4, dtype)
    q[0] *= 60
    q[1] = 0.0
    check_attention(cache, host, q, table, lens, True, 1.0, accumulate=True)


@pytest.mark.parametrize("T,G,dtype", [(4, 2, BF16), (4, 4, F32), (90, 2, BF16)])
def test_hidden_numbers_stay_hidden(T, G, dtype):
    """NaN codes and scales behind a sequence's end, in blocks of nobody, and in tokens that a query must not see yet."""
    D, bs, lens = 64, 16, [40 + T, 6 + T]
    cache, host = make_cache(20, 1, bs, D, E4M3)
    table = make_table(2, 9, 20, lens, bs)
    clean = {k: v.clone() for k, v in host.items()}
    nan = 0x7F
    for x in ("k", "v"):
        host[x].view(torch.uint8)[int(table[0, (lens[0] - 1) // bs]), 0, (lens[0] - 1) % bs + 1:] = nan      # behind the end
        host[x].view(torch.uint8)[int(table[1, (lens[1] - 1) // bs]), 0, (lens[1] - 1) % bs] = nan           # the last token of sequence 1
        getattr(cache, x).view(torch.uint8).copy_(host[x].view(torch.uint8).cuda())
    q = draw((2, G, T, D), 4, dtype)
    o, bulk, slack, _ = ref.attention(clean, q, table, lens, True, 0.125)
    got = pkg.cache_attention(q.cuda(), cache, *gpu(table, ints(lens)), True, 0.125)
    pkg.check_status()
    seen = torch.ones_like(o, dtype=torch.bool)
    seen[1, :, T - 1] = False                                                                                # its own query sees it
    assert got[1, :, T - 1].isnan().all()
    excess = (got.double().cpu() - o).abs() - tolerance(dtype, o, bulk, slack)
    assert not (excess[seen] > 0).any() and not got.cpu()[seen].isnan().any()


@pytest.mark.parametrize("T,G,dtype", [(1, 4, BF16), (3, 4, F32), (50, 3, BF16), (30, 2, F32)])
def test_queries_of_any_size(T, G, dtype):
    """Queries of 2^110 and 2^-115 beside an sm_scale that makes their scores ordinary ones."""
    D, bs, lens = 64, 16, [90 + T, 33 + T]
    cache, host = make_cache(30, 2, bs, D, E4M3)
    table, q = make_table(2, 12, 30, lens, bs), draw((2, 2 * G, T, D), 4, dtype)
    usual = pkg.cache_attention(q.cuda(), cache, *gpu(table, ints(lens)), True, 0.125)
    assert torch.equal(usual, pkg.cache_attention(q.cuda() * 2.0 ** 110, cache, *gpu(table, ints(lens)), True, 0.125 * 2.0 ** -110))
    check_attention(cache, host, q * 2.0 ** -115, table, lens, True, 0.125 * 2.0 ** 115)
    check_attention(cache, host, q * 2.0 ** 110, table, lens, True, 0.125 * 2.0 ** -110, accumulate=True)


@pytest.mark.parametrize("T,G,dtype", [(1, 4, BF16), (3, 4, F32), (50, 3, BF16), (30, 2, F32)])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_values_below_the_least_scale_are_zeros(T, G, dtype, code):
    """Blocks of scale 2^-120 are not read as ones of a larger scale: alone they give zeros, beside others nothing."""
    D, bs, lens = 64, 16, [90 + T, 33 + T]
    cache, host = make_cache(30, 1, bs, D, code)
    table, q = make_table(2, 12, 30, lens, bs), draw((2, G, T, D), 4, dtype)
    cache.v_scale.fill_(2.0 ** -120)
    got = pkg.cache_attention(q.cuda(), cache, *gpu(table, ints(lens)), True, 0.125)
    assert (got == 0).all()
    host["v_scale"][table[:, 1].long()] = 2.0 ** -120
    cache.v_scale.copy_(host["v_scale"].cuda())
    check_attention(cache, host, q, table, lens, True, 0.125, accumulate=True)


@pytest.mark.parametrize("T,G,dtype,new", [(4, 1, BF16, [1, 3]), (7, 3, F32, [2, 7]), (90, 2, BF16, [3, 70]), (300, 1, F16, [10, 299])])
def test_hidden_nan_with_a_table_that_ends_with_the_sequence(T, G, dtype, new):
    """Rows without a query stand behind the last one: they must not make anyone look behind the last block of the table."""
    D, bs, lens = 64, 16, [16 * (T // 16) + 32, 16 * (T // 16) + 32]
    wide = lens[0] // bs
    cache, host = make_cache(2 * wide, 1, bs, D, E4M3)
    table = make_table(2, wide, 2 * wide, lens, bs)
    for b in range(2):      # the last token
        host["v"].view(torch.uint8)[int(table[b, -1]), 0, bs - 1] = 0x7F
    cache.v.view(torch.uint8).copy_(host["v"].view(torch.uint8).cuda())
    q = draw((2, G, T, D), 4, dtype)
    o, bulk, slack, _ = ref.attention(host, q, table, lens, True, 0.125, new_lens=new)
    got = pkg.cache_attention(q.cuda(), cache, *gpu(table, ints(lens)), True, 0.125, new_lens=ints(new).cuda()).double().cpu()
    pkg.check_status()
    assert torch.equal(got.isnan(), o.isnan())
    assert all(o[b, :, new[b] - 1].isnan().all() and not o[b, :, :new[b] - 1].isnan().any() and (got[b, :, new[b]:] == 0).all() for b in range(2))
    excess = (got - o).abs() - tolerance(dtype, o, bulk, slack, dtype == BF16 and T * G > 32)
    assert not (excess > 0).any()


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("scale", [float("nan"), float("inf")])
@pytest.mark.parametrize("T,G,dtype,wide", [(4, 2, BF16, 9), (4, 2, F16, 400), (6, 3, F32, 9), (70, 2, F16, 9)])
def test_hidden_scales_stay_hidden(T, G, dtype, wide, scale, accumulate):
    """A block whose scales are no finite numbers, of which the first queries see nothing, in every way that scores are kept."""
    D, bs = 64, 16
    length = -(-(T + 20) // bs) * bs + 2        # the last two tokens begin a block
    cache, host = make_cache(20, 2, bs, D, INT8)
    table = make_table(1, 9, 20, [length], bs)
    table = torch.cat((table, torch.full((1, wide - 9), -1, dtype=torch.int32)), dim=1)
    q = draw((1, 2 * G, T, D), 4, dtype)
    o, bulk, slack, _ = ref.attention(host, q, table, [length], True, 0.125)
    for x in ("k_scale", "v_scale"):
        getattr(cache, x)[int(table[0, length // bs])] = scale
    got = pkg.cache_attention(q.cuda(), cache, *gpu(table, ints([length])), True, 0.125, accumulate=accumulate)[:, :, :T - 2].double().cpu()
    pkg.check_status()
    assert not got.isnan().any() and not ((got - o[:, :, :T - 2]).abs() > tolerance(dtype, o, bulk, slack)[:, :, :T - 2]).any()


@pytest.mark.parametrize("T,G,dtype", [(2, 2, BF16), (2, 2, F32), (64, 2, BF16)])
def test_hidden_nan_costs_little_behind_a_long_context(T, G, dtype):
    """A NaN that some queries must not see is looked for where it can be, not through all of the context."""
    D, bs, length = 128, 256, 400000
    wide = -(-length // bs)
    cache = pkg.KVCache(wide, 4, bs, D)
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(1.0)
    table, lens = torch.arange(wide, dtype=torch.int32, device="cuda")[None], ints([length]).cuda()
    q = draw((1, 4 * G, T, D), 4, dtype).cuda()

    def fastest():
        times = []
        for _ in range(6):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            got = pkg.cache_attention(q, cache, table, lens, True, 0.1)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times), got

    clean, zeros = fastest()
    assert (zeros == 0).all()
    cache.v.view(torch.uint8)[-1, :, (length - 1) % bs, 5] = 0x7F       # the last token
    once, got = fastest()
    pkg.check_status()
    assert got[:, :, -1, 5].isnan().all() and (got[:, :, :-1] == 0).all() and got.isnan().sum() == 4 * G
    assert once < 3 * clean, (once, clean)


def test_rows_behind_the_last_query_are_zero_and_others_untouched():
    D, bs, lens, new = 32, 16, [20, 9], [2, 0]
    cache, host = make_cache(6, 2, bs, D, INT8, weights=False)
    table = make_table(2, 2, 6, lens, bs)
    before = [getattr(cache, x).view(torch.uint8).clone() for x in ("k", "v")]
    got = check_attention(cache, host, draw((2, 4, 6, D), 1, F16), table, lens, True, 0.3, new_lens=new)
    assert (got[0, :, 2:] == 0).all() and (got[1] == 0).all()
    assert all(torch.equal(getattr(cache, x).view(torch.uint8), y) for x, y in zip(("k", "v"), before))


@pytest.mark.parametrize("T", [1, 3, 20])
@pytest.mark.parametrize("causal", [True, False])
def test_empty_places_have_no_position(T, causal):
    """Sequences of no tokens, and queries without a slot, beside a table of positions: their slots are below its first row."""
    D, bs, lens = 64, 16, [0, 37, 2 if causal else 0, 0]
    cache, host = make_cache(12, 2, bs, D, E4M3)
    table = make_table(4, 3, 12, lens, bs)
    cos, sin = precompute_freqs_cis(D, 50, 10000.0)
    check_attention(cache, host, draw((4, 4, T, D), 1, F16), table, lens, causal, 0.3, cos, sin, accumulate=True)
    check_attention(cache, host | {"weight": cache.weight.cpu()}, draw((4, 4, T, D), 1, F32), table, lens, causal, 0.3, cos, sin, new_lens=[T, 1, T, T])


@pytest.mark.parametrize("B,Hkv,G,T,D,dtype,accumulate", [
    (8, 8, 4, 600, 128, BF16, False),     # two tiles of 128 rows an item: most items in front of slot 0, several of them a block
    (8, 8, 4, 600, 64, F16, False),
    (6, 8, 4, 600, 128, F16, False),      # one tile an item
    (40, 4, 1, 300, 32, BF16, False),
    (3, 3, 2, 200, 32, F32, True),        # tiles of 32 rows
    (8, 8, 4, 600, 64, F16, True),
    (6, 8, 4, 600, 128, F16, True),
])
def test_tiles_of_rows_before_the_first_slot(B, Hkv, G, T, D, dtype, accumulate):
    """Far more queries than tokens: whole tiles of rows see nothing, many in a row, between ones that see some slots."""
    bs, lens = 16, [(29 * i) % 41 for i in range(B)]
    lens[0], lens[-1] = 150, 3
    cache, host = make_cache(10 + 3 * B, Hkv, bs, D, E4M3)
    table = torch.full((B, 10), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, :-(-n // bs)] = torch.arange(at, at + -(-n // bs), dtype=torch.int32)
        at += -(-n // bs)
    got = check_attention(cache, host, draw((B, Hkv * G, T, D), 1, dtype), table, lens, True, 0.2, accumulate=accumulate)
    assert (got[-1, :, :T - 3] == 0).all()


@pytest.mark.parametrize("D,Hkv,T,long,empty", [(128, 2, 320, 12900, 150), (32, 1, 700, 26000, 300), (64, 3, 256, 10000, 40)])
def test_weights_of_sequences_far_apart(D, Hkv, T, long, empty):
    """Five and more tiles of rows a head, weights, and empty places between two long sequences: a block looks for its next unit while its sums go on."""
    bs, lens = 64, [long] + [0] * empty + [long - 77, 5]
    wide = -(-long // bs)
    cache, host = make_cache(2 * wide + 1, Hkv, bs, D, E4M3)
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    for i, b in enumerate((0, empty + 1, empty + 2)):
        table[b, :-(-lens[b] // bs)] = torch.arange(i * wide, i * wide + -(-lens[b] // bs), dtype=torch.int32)
    check_attention(cache, host, draw((len(lens), 2 * Hkv, T, D), 1, F16), table, lens, True, 0.1, accumulate=True)


def test_many_sequences():
    """More sequences than a block has threads, most of them short or empty."""
    B, D, bs = 300, 32, 16
    lens = [(7 * i) % 23 * (i % 3) for i in range(B)]
    cache, host = make_cache(3 * B, 1, bs, D, INT8)
    table = make_table(B, 3, 3 * B, lens, bs)
    check_attention(cache, host, draw((B, 2, 1, D), 1, F16), table, lens, True, 0.3, accumulate=True)
    check_attention(cache, host | {"weight": cache.weight.cpu()}, draw((B, 2, 20, D), 2, BF16), table, lens, True, 0.3, new_lens=[i % 21 for i in range(B)], accumulate=True)


@pytest.mark.parametrize("B,Hkv,T,dtype,wide,most", [
    (60, 12, 1, BF16, 32, 500),      # more heads than resident blocks: several items a block
    (3, 2, 1, F16, 600, 9600),       # tables too long for clusters
    (3, 2, 1, BF16, 600, 200),       # .. and hardly filled: most blocks have no slot to read
    (5, 2, 7, F32, 600, 1500),
    (5, 3, 20, F32, 300, 900),       # two tiles of rows
    (7, 3, 20, BF16, 300, 900),
    (6, 2, 70, BF16, 100, 1500),
    (2, 3, 70, F16, 12, 190),
])
def test_work_shared_out(B, Hkv, T, dtype, wide, most):
    """Ranges that begin and end everywhere in an item: in its slots, between two items, in what an item costs beside its slots."""
    D, bs = 32, 16
    lens = torch.randint(0, most + 1, (B,), generator=torch.Generator().manual_seed(B * T)).tolist()
    lens[B // 2], lens[-1] = 1, most
    needed = sum(-(-n // bs) for n in lens)
    cache, host = make_cache(needed + 1, Hkv, bs, D, INT8)
    table, at = torch.full((B, wide), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        table[b, :-(-n // bs)] = torch.arange(at, at + -(-n // bs), dtype=torch.int32)
        at += -(-n // bs)
    check_attention(cache, host, draw((B, 2 * Hkv, T, D), 1, dtype), table, lens, True, 0.3, accumulate=True)


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_scales_of_any_sign(T, dtype):
    """A score times a negative number is that of the negated query, bit for bit; times 0 all slots count the same."""
    D, bs, lens = 64, 16, [70, 45]
    cache, host = make_cache(12, 2, bs, D, E4M3, weights=False)
    table, q = make_table(2, 5, 12, lens, bs), draw((2, 4, T, D), 1, dtype)
    got = [pkg.cache_attention(x.cuda(), cache, *gpu(table, ints(lens)), True, s) for x, s in ((q, -0.4), (-q, 0.4))]
    assert torch.equal(*got)
    check_attention(cache, host, q, table, lens, True, 0.0)


def test_weights_without_room_for_scores():
    """Block tables so wide that the scores of all their slots are not kept."""
    B, Hkv, D, bs, lens = 4, 2, 64, 256, [300, 700, 1, 0]
    cache, host = make_cache(20, Hkv, bs, D, E4M3)
    table = torch.cat((make_table(B, 4, 20, lens, bs), torch.full((B, 33000), -1, dtype=torch.int32)), dim=1)
    assert B * Hkv * table.shape[1] * bs * 2 * 4 > 512 << 20
    check_attention(cache, host, draw((B, 2 * Hkv, 1, D), 1, BF16), table, lens, True, 0.2, accumulate=True)


def test_caches_beyond_32_bits():
    """A pool of more than 2^32 codes: what is done in its last blocks is what is done in a pool of those blocks alone."""
    Hkv, bs, D, big, few = 64, 256, 128, 2100, 6
    assert big * Hkv * bs * D > 2 ** 32
    small, _ = make_cache(few, Hkv, bs, D, INT8)
    large = pkg.KVCache(big, Hkv, bs, D, dtype=INT8, weights=True)
    for x in ("k", "v", "k_scale", "v_scale", "weight"):
        getattr(large, x)[-few:] = getattr(small, x)
    table, out, lens = ints([[0, 1, 2], [3, 4, -1]]).cuda(), ints([[5, 4]]).cuda(), ints([700, 300]).cuda()
    for shift, cache in ((0, small), (big - few, large)):
        at = torch.where(table >= 0, table + shift, table)
        res = []
        for T, dtype in ((1, F32), (40, BF16)):
            k, q = draw((2, Hkv, T, D), T, dtype).cuda(), draw((2, Hkv, T, D), 50 + T, dtype).cuda()
            pkg.cache_append(k, q, cache, at, lens)
            res.append(pkg.cache_attention(q, cache, at, lens, True, 0.05, accumulate=True))
        res += pkg.cache_evict(cache, at[:1], lens[:1], out + shift, 300, 20)
        res += [getattr(cache, x)[-few:].clone() for x in ("k", "v", "k_scale", "v_scale", "weight")]
        pkg.check_status()
        if shift == 0:
            want = res
    assert [torch.equal(x, y) for x, y in zip(res, want)] == [True] * len(want)


# ---------------------------------------------------------------------------------------------------------------- eviction
EVICTS = [
    # lens, budget, recent, Hkv, D, bs, code
    ([40, 17, 16, 0, 100], 17, 4, 2, 64, 16, E4M3),
    ([300, 301], 64, 0, 3, 32, 32, INT8),
    ([300, 2500], 256, 256, 1, 128, 64, E4M3),
    ([70, 33], 1, 0, 2, 32, 16, INT8),
    ([700, 90], 600, 17, 2, 128, 256, E4M3),
]


@pytest.mark.parametrize("weights", ["random", "ties", "odd"])
@pytest.mark.parametrize("lens,budget,recent,Hkv,D,bs,code", EVICTS)
def test_evict(lens, budget, recent, Hkv, D, bs, code, weights):
    B, wide, outs = len(lens), max(lens) // bs + 2, (budget + bs - 1) // bs + 1
    blocks = B * (wide + outs)
    cache, host = make_cache(blocks, Hkv, bs, D, code)
    if weights != "random":   # few different weights: the lowest slots win;  NaN, infinities, zeros of both signs, negative numbers
        pick = torch.randint(0, 3 if weights == "ties" else 8, host["weight"].shape, generator=torch.Generator().manual_seed(3))
        host["weight"] = torch.tensor([0.0, 1.0, 1.5, float("nan"), float("inf"), -0.0, -2.0, float("-inf")])[pick]
        if weights == "odd":
            cache.weight.copy_(host["weight"].cuda())
            host["weight"] = host["weight"].clone()
    cache.weight.copy_(host["weight"].cuda())
    both = make_table(B, wide + outs, blocks, [10 ** 6] * B, bs)
    table, out = both[:, :wide].contiguous(), both[:, wide:].contiguous()
    new_lens, kept = ref.evict(host, table, lens, out, budget, recent)
    got_lens, got_kept = pkg.cache_evict(cache, *gpu(table, ints(lens), out), budget, recent)
    pkg.check_status()
    assert torch.equal(got_lens.cpu(), new_lens) and torch.equal(got_kept.cpu(), kept)
    nan = host["weight"].isnan()
    assert torch.equal(cache.weight.cpu().isnan(), nan)
    cache.weight.nan_to_num_(nan=7.0)
    host["weight"] = torch.where(nan, 7.0, host["weight"]).nan_to_num(nan=7.0)
    cache.weight.nan_to_num_()
    same_cache(cache, host)


@pytest.mark.parametrize("length,budget", [(20000, 9000), (430000, 3000)])
def test_evict_long(length, budget):
    """One head of one sequence: a cluster shares it; beyond 8 x 48 K slots the weights are read in every round."""
    bs, D = 256, 32
    wide, outs = length // bs + 1, (budget + bs - 1) // bs
    cache, host = make_cache(wide + outs, 1, bs, D, INT8)
    order = torch.randperm(wide + outs, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None]
    table, out = order[:, :wide].contiguous(), order[:, wide:].contiguous()
    new_lens, kept = ref.evict(host, table, [length], out, budget, 100)
    got_lens, got_kept = pkg.cache_evict(cache, *gpu(table, ints([length]), out), budget, 100)
    pkg.check_status()
    assert torch.equal(got_lens.cpu(), new_lens) and torch.equal(got_kept.cpu(), kept)
    same_cache(cache, host)


def test_evict_reads_shared_blocks():
    """Two sequences begin with the same block: eviction leaves it as it was."""
    bs, D = 16, 32
    cache, host = make_cache(8, 1, bs, D, E4M3)
    table, out, lens = ints([[0, 1], [0, 2]]), ints([[3], [4]]), [30, 25]
    new_lens, kept = ref.evict(host, table, lens, out, 10, 3)
    got_lens, got_kept = pkg.cache_evict(cache, *gpu(table, ints(lens), out), 10, 3)
    assert torch.equal(got_kept.cpu(), kept) and torch.equal(got_lens.cpu(), new_lens)
    same_cache(cache, host)


# ------------------------------------------------------------------------------------------------------- all of them together
def test_generation_with_eviction():
    """A prompt, decode steps, an eviction and more steps: every output against the oracle on the cache's own codes, and the first ones against
    fused_rope_attention, off by no more than the codes are."""
    B, Hkv, G, D, bs, prompt = 2, 2, 2, 64, 16, 40
    cos, sin = precompute_freqs_cis(D, 200, 10000.0)
    cache, host = make_cache(24, Hkv, bs, D, INT8)
    ks, vs = (draw((B, Hkv, 80, D), i, BF16) for i in range(2))
    qs = draw((B, Hkv * G, 80, D), 2, BF16)
    table = make_table(B, 5, 20, [80] * B, bs)
    lens, at = ints([0] * B), 0
    out = torch.arange(20, 24, dtype=torch.int32).view(B, 2)
    whole = pkg.fused_rope_attention(*gpu(qs, ks.repeat_interleave(G, dim=1), vs.repeat_interleave(G, dim=1)), True, D ** -0.5, *gpu(cos, sin)).cpu()
    positions = ints([0] * B)
    for step in range(12):
        T = prompt if step == 0 else 1
        if step == 8:
            ref_lens, ref_kept = ref.evict(host, table, lens, out, 24, 6)
            lens_g, kept = pkg.cache_evict(cache, *gpu(table, lens, out), 24, 6)
            assert torch.equal(kept.cpu(), ref_kept) and torch.equal(lens_g.cpu(), ref_lens)
            lens, table = lens_g.cpu(), out
        lens = lens + T
        k, v, q = (x[:, :, at:at + T] for x in (ks, vs, qs))
        pkg.cache_append(*gpu(k, v), cache, *gpu(table, lens, cos, sin, positions))
        ref.append(host, k, v, table, lens, cos, sin, positions)
        host["weight"] = cache.weight.cpu()          # sums differ in their last bits, and eviction compares them
        got = check_attention(cache, host, q, table, lens.tolist(), True, D ** -0.5, cos, sin, positions, accumulate=True)
        host["weight"] = cache.weight.cpu()
        same_cache(cache, host)
        if step < 8:
            # |v| <= 5, codes are off by half a step of at most 5 / 127 / 2 = 0.02 in v and 0.02 per element of k: scores by 0.02 sum |q| / 8 <= 0.02 * 64 *
            # 0.8 / 8 = 0.13 on average signs cancel; p changes by up to 2 * 0.13 of sum p |v| ~ 0.8; 0.25 covers v's own 0.02 as well
            assert (got.float().cpu() - whole[:, :, at:at + T].float()).abs().max() < 0.25
        at += T
        positions = positions + T


def test_steps_replay_from_a_graph():
    """A decode step captured once and replayed: lengths, positions and tables are what they are at replay."""
    B, Hkv, G, D, bs = 3, 2, 4, 128, 16
    cos, sin = (t.cuda() for t in precompute_freqs_cis(D, 100, 10000.0))
    cache, host = make_cache(20, Hkv, bs, D, E4M3)
    table = make_table(B, 6, 20, [96] * B, bs)
    table_g, lens, positions = table.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(B, Hkv, 1, D, dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros(B, Hkv * G, 1, D, dtype=BF16, device="cuda")

    def step():
        pkg.cache_append(k, v, cache, table_g, lens, cos, sin, positions)
        return pkg.cache_attention(q, cache, table_g, lens, True, D ** -0.5, cos, sin, positions, accumulate=True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()            # lengths of 0: nothing is stored, nothing is seen
    side.synchronize()
    graphs = []
    for _ in range(2):    # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="relaxed"):
            o = step()
        graphs.append((graph, o))
    for i in range(20):
        x = [draw(t.shape, 50 + 3 * i + j, BF16) for j, t in enumerate((k, v, q))]
        for t, y in zip((k, v, q), x):
            t.copy_(y)
        now = [min(i + 1, 96) + 20 * b for b in range(B)]
        if i == 0:
            now = [1, 21, 41]
        lens.copy_(ints(now))
        positions.copy_(ints([n + 1 for n in now]))
        host["weight"] = cache.weight.cpu()
        graph, o = graphs[i % 2]
        graph.replay()
        pkg.check_status()
        ref.append(host, x[0], x[1], table, now, cos.cpu(), sin.cpu(), ints([n + 1 for n in now]))
        ref_o, bulk, slack, weight = ref.attention(host, x[2], table, now, True, D ** -0.5, cos.cpu(), sin.cpu(), ints([n + 1 for n in now]))
        assert not ((o.double().cpu() - ref_o).abs() > tolerance(BF16, ref_o, bulk, slack)).any()
        assert ((cache.weight.double().cpu() - host["weight"].double() - weight).abs() <= 2.0 ** -15 * (weight * slack.max() + host["weight"].double() + weight)).all()


@pytest.mark.parametrize("T,dtype", [(2, F16), (60, BF16), (20, F32)])
def test_calls_on_two_streams_and_twice_are_the_same(T, dtype):
    D, bs, lens = 128, 32, [700, 64, 333]
    cache, host = make_cache(80, 4, bs, D, E4M3, weights=False)
    table, n = gpu(make_table(3, 24, 80, lens, bs), ints(lens))
    q = draw((3, 16, T, D), 1, dtype).cuda()
    want = pkg.cache_attention(q, cache, table, n, True, 0.1)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(pkg.cache_attention(q, cache, table, n, True, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got)


def test_writes_in_place_are_known_to_autograd():
    """A tensor of the cache that a backward pass has saved cannot be written to unnoticed; inference tensors are taken as they are."""
    cache = pkg.KVCache(6, 1, 16, 32, weights=True)
    names = ("k", "v", "k_scale", "v_scale", "weight")
    table, out, lens = gpu(ints([[0, 1]]), ints([[2]]), ints([20]))
    x = draw((1, 1, 20, 32), 1, BF16).cuda()

    def bumped(call):
        before = [getattr(cache, n)._version for n in names]
        call()
        return [n for n, was in zip(names, before) if getattr(cache, n)._version > was]

    assert bumped(lambda: pkg.cache_append(x, x, cache, table, lens)) == list(names)
    assert bumped(lambda: pkg.cache_attention(x, cache, table, lens, True, 0.1)) == []
    assert bumped(lambda: pkg.cache_attention(x, cache, table, lens, True, 0.1, accumulate=True)) == ["weight"]
    assert bumped(lambda: pkg.cache_evict(cache, table, lens, out, 16)) == list(names)
    y = torch.ones(6, 1, 16, device="cuda", requires_grad=True)
    loss = (cache.weight * y).sum()
    pkg.cache_attention(x, cache, table, lens, True, 0.1, accumulate=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        cache = pkg.KVCache(6, 1, 16, 32, weights=True)
        pkg.cache_append(x, x, cache, table, lens)
    pkg.cache_append(x, x, cache, table, lens)
    pkg.cache_attention(x, cache, table, lens, True, 0.1, accumulate=True)
    pkg.check_status()


def test_sequences_may_share_blocks():
    """A common prefix: reads are shared, and each sequence's weights are added."""
    D, bs, lens = 64, 16, [40, 36]
    cache, host = make_cache(6, 1, bs, D, INT8)
    check_attention(cache, host, draw((2, 2, 1, D), 1, BF16), ints([[0, 1, 2], [0, 1, 3]]), lens, True, 0.2, accumulate=True)


# ---------------------------------------------------------------------------------------------------- indices out of range
def test_bad_indices_are_not_followed():
    """A block id beyond the pool, a length beyond the table, new tokens and positions out of range: the call does what it can, and the next
    one on the device raises."""
    D, bs = 64, 16
    cache, host = make_cache(6, 1, bs, D, E4M3)
    q = draw((1, 2, 1, D), 1, F32)
    k = draw((1, 1, 1, D), 2, F32).cuda()
    cos, sin = (t.cuda() for t in precompute_freqs_cis(D, 50, 10000.0))
    full = ints([[0, 1, 2]])

    def raises():
        with pytest.raises(RuntimeError, match="0x4000"):
            torch.cuda.synchronize()
            pkg.check_status()
        pkg.check_status()

    for bad in (-1, 6, 2 ** 31 - 1):      # the block's tokens are left out
        got = pkg.cache_attention(q.cuda(), cache, *gpu(ints([[0, bad, 2]]), ints([40])), True, 0.2, accumulate=True)
        raises()
        short, _, _, _ = ref.attention(host, q, ints([[0, 2]]), [24], True, 0.2)
        assert (got.double().cpu() - short).abs().max() < 1e-4
        pkg.cache_append(k, k, cache, *gpu(ints([[0, bad, 2]]), ints([20])))
        raises()
        pkg.cache_evict(cache, *gpu(ints([[0, bad, 2]]), ints([40]), ints([[4]])), 16)
        raises()
        pkg.cache_evict(cache, *gpu(full, ints([40]), ints([[bad]])), 16)
        raises()
    for length in (49, -1, 2 ** 31 - 1, -2 ** 31):
        pkg.cache_attention(q.cuda(), cache, *gpu(full, ints([length])), True, 0.2, accumulate=True)
        raises()
        pkg.cache_append(k, k, cache, *gpu(full, ints([length])))
        raises()
        pkg.cache_evict(cache, *gpu(full, ints([length]), ints([[4]])), 16)
        raises()
    for new in (2, -1, 2 ** 31 - 1):
        pkg.cache_attention(q.cuda(), cache, *gpu(full, ints([20])), True, 0.2, new_lens=ints([new]).cuda())
        raises()
        pkg.cache_append(k, k, cache, *gpu(full, ints([20])), new_lens=ints([new]).cuda())
        raises()
    for position in (50, -1, 2 ** 31 - 1):
        pkg.cache_attention(q.cuda(), cache, *gpu(full, ints([20])), True, 0.2, cos, sin, ints([position]).cuda())
        raises()
        pkg.cache_append(k, k, cache, *gpu(full, ints([20])), cos, sin, ints([position]).cuda())
        raises()
    # the attention entry points beside the cache raise too, once, for what a cache operator met
    pkg.cache_attention(q.cuda(), cache, *gpu(full, ints([49])), True, 0.2)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="0x4000"):
        pkg.flash_attention(k, k, k, True, 0.2)
    pkg.check_status()
    pkg.flash_attention(k, k, k, True, 0.2)


@pytest.mark.parametrize("what,value", [("length", 49), ("length", 60), ("length", 2 ** 31 - 1), ("length", -1), ("new", 3), ("new", 2 ** 31 - 1), ("new", -1)])
def test_tokens_of_a_sequence_out_of_range_are_not_stored_elsewhere(what, value):
    """A length beyond the table, or more new tokens than there are: older slots stay as they were, and the other sequences get theirs."""
    D, bs, T = 32, 16, 2
    cache, host = make_cache(10, 2, bs, D, E4M3)
    table, lens, new = make_table(3, 3, 10, [48, 48, 48], bs), [20, 48, 33], [2, 2, 1]
    k, v = (draw((3, 2, T, D), i, BF16) for i in range(2))
    for b in (0, 2):
        ref.append(host, k[b:b + 1], v[b:b + 1], table[b:b + 1], lens[b:b + 1], new_lens=new[b:b + 1])
    if what == "length":
        lens[1] = value
    else:
        new[1] = value
    pkg.cache_append(*gpu(k, v), cache, *gpu(table, ints(lens)), new_lens=ints(new).cuda())
    with pytest.raises(RuntimeError, match="0x4000"):
        pkg.check_status()
    same_cache(cache, host)


@pytest.mark.parametrize("wide,bs,accumulate", [(63, 16, True), (63, 16, False), (16, 64, True), (1000, 16, True), (300, 64, False)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_bad_block_hides_no_other(D, wide, bs, accumulate):
    """Bad entries near the start, hundreds of good slots behind them in the same block of threads: only the tokens of the bad blocks are left out."""
    length, Hkv = 1000, 300
    blocks = -(-length // bs) + 2
    cache, host = make_cache(blocks, Hkv, bs, D, INT8)
    whole = torch.arange(wide, dtype=torch.int32) % blocks
    good = [i for i in range(-(-length // bs)) if i not in (1, 6)]
    for T, dtype, bad in ((1, F16, -1), (4, F32, 2 ** 30)):
        q = draw((1, Hkv, T, D), T, dtype)
        table = whole.clone()
        table[[1, 6]] = bad
        some = torch.tensor([0, 1, 137, 200, 299])                        # heads that are compared
        few = {x: t.view(torch.uint8)[:, some].view(t.dtype) if x in ("k", "v") else t[:, some] for x, t in host.items()}
        o, bulk, slack, weight = ref.attention(few, q[:, some], whole[good][None], [length - 2 * bs], True, 0.2)
        cache.weight.copy_(host["weight"].cuda())
        got = pkg.cache_attention(q.cuda(), cache, *gpu(table[None], ints([length])), True, 0.2, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="0x4000"):
            pkg.check_status()
        assert not ((got[:, some.cuda()].double().cpu() - o).abs() > tolerance(dtype, o, bulk, slack)).any()
        if accumulate:
            off = (cache.weight.cpu()[:, some].double() - few["weight"].double() - weight).abs()
            assert not (off > 2 * 2.0 ** -17 * slack.max() * weight + (T + 2) * 2.0 ** -23 * (few["weight"].double() + weight)).any()


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    D, bs = 64, 16
    cache = pkg.KVCache(6, 2, bs, D)
    table, lens = gpu(ints([[0, 1]]), ints([20]))
    q, k = draw((1, 4, 1, D), 1, BF16).cuda(), draw((1, 2, 1, D), 2, BF16).cuda()

    def attend(**kw):
        a = dict(q=q, cache=cache, block_table=table, seq_lens=lens, causal=True, sm_scale=0.1)
        a.update(kw)
        return pkg.cache_attention(**a)

    class Other:
        def __init__(self, **kw):
            for x in ("k", "v", "k_scale", "v_scale", "weight"):
                setattr(self, x, kw.get(x, getattr(cache, x)))

    attend()
    for kw in (dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.double()), dict(q=q.expand(2, 4, 1, D)), dict(seq_lens=lens.long()), dict(seq_lens=lens[None]),
               dict(block_table=table.long()), dict(block_table=table[0]), dict(block_table=table[:, :0]), dict(new_lens=lens.long()), dict(positions=lens.expand(2)),
               dict(accumulate=True), dict(freqs_cos=torch.zeros(30, 32, device="cuda")), dict(freqs_cos=torch.zeros(30, 16, device="cuda"), freqs_sin=torch.zeros(30, 16, device="cuda")),
               dict(cache=Other(k=cache.k.view(torch.uint8), v=cache.v.view(torch.uint8))), dict(cache=Other(v=cache.v[:5])), dict(cache=Other(k_scale=cache.k_scale[:5])),
               dict(cache=Other(k_scale=cache.k_scale.half())), dict(cache=Other(weight=torch.zeros(6, 2, 8, device="cuda"))),
               dict(cache=Other(k=cache.k[:, :, :8], v=cache.v[:, :, :8])),
               dict(cache=Other(k=torch.zeros(6, 2, bs, D + 8, dtype=torch.uint8, device="cuda").view(E4M3)[..., :D]))):
        with pytest.raises(ValueError):
            attend(**kw)
    for kw in (dict(q=q.cpu()), dict(seq_lens=lens.cpu()), dict(block_table=table.cpu())):
        with pytest.raises(RuntimeError):
            attend(**kw)
    with pytest.raises(RuntimeError, match="no backward"):
        attend(q=q.clone().requires_grad_(True))
    with torch.no_grad():
        attend(q=q.clone().requires_grad_(True))
    for bad in ((k[:, :1], k[:, :1]), (k, k[:, :1]), (k, k.float()), (k[..., :32], k[..., :32])):
        with pytest.raises(ValueError):
            pkg.cache_append(*bad, cache, table, lens)
    for args in ((table, 8, 0), (table, 0, 0), (table, 8, 9), (table, 33, 0), (table.long(), 8, 0)):
        with pytest.raises(ValueError):
            pkg.cache_evict(cache, table, lens, *args)
    pkg.check_status()


def test_one_block_read_as_many_heads():
    """Heads that share their codes are read; append and eviction refuse them."""
    D, bs, lens = 64, 16, [30]
    cache, host = make_cache(3, 1, bs, D, INT8)
    wide = pkg.KVCache(3, 4, bs, D, dtype=INT8, weights=True)
    for x in ("k", "v", "k_scale", "v_scale"):
        t = getattr(cache, x).expand((3, 4) + getattr(cache, x).shape[2:])
        setattr(wide, x, t if x in ("k", "v") else t.contiguous())
    table, q = ints([[0, 1]]), draw((1, 4, 1, D), 1, F32)
    got = pkg.cache_attention(q.cuda(), wide, *gpu(table, ints(lens)), True, 0.2)
    assert torch.equal(got, pkg.cache_attention(q.cuda(), cache, *gpu(table, ints(lens)), True, 0.2))
    with pytest.raises(ValueError, match="share memory"):
        pkg.cache_append(q.cuda(), q.cuda(), wide, *gpu(table, ints(lens)))
    with pytest.raises(ValueError, match="share memory"):
        pkg.cache_evict(wide, *gpu(table, ints(lens), ints([[2]])), 8)
    pkg.check_status()


def test_budgets_of_32_bits():
    """A table of 2^28 + 1 blocks of 16 has room for a budget beyond 32 bits; 2^32 + 8 is not taken for 8."""
    cache = pkg.KVCache(6, 2, 16, 64, weights=True)
    table, lens, wide = *gpu(ints([[0, 1]]), ints([20])), torch.zeros(1, 2 ** 28 + 1, dtype=torch.int32, device="cuda")
    for budget in (2 ** 30, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="budget"):
            pkg.cache_evict(cache, table, lens, wide, budget)
