"""The cache operators without a GPU: refusals of the C ABI and of the entry points, and the oracle against itself."""

import ctypes

import pytest
import torch

from helpers import draw, ext, pkg
from oracle import kv_cache_oracle as ref


def _structs(**kw):
    c = ext.KVCacheView(k=256, v=256, k_scale=256, v_scale=256, weight=256, num_blocks=4, Hkv=2, block_size=16, D=64, code=0)
    c.k_stride[:] = c.v_stride[:] = [2 * 16 * 64, 16 * 64, 64]
    s = ext.CacheSeqs(block_table=256, table_stride=3, B=2, max_blocks=3, seq_lens=256)
    for name, value in kw.items():
        to = c if hasattr(c, name) else s
        if name in ("k_stride", "v_stride"):
            getattr(to, name)[:] = value
        else:
            setattr(to, name, value)
    return ctypes.byref(c), ctypes.byref(s)


_ROWS = (ctypes.c_int64 * 3)(4 * 64, 64, 64)


def _append(T=1, dtype=1, k=256, rows=_ROWS, **kw):
    return ext.lib().corope_cache_append(*_structs(**kw), k, 256, rows, rows, T, dtype, None, None)


def _attend(Hq=4, T=1, dtype=1, accumulate=0, q=256, ws=256, ws_bytes=8, **kw):
    return ext.lib().corope_cache_attn(*_structs(**kw), q, 256, _ROWS, _ROWS, Hq, T, dtype, 1, 0.1, accumulate, ws, ws_bytes, None, None)


def _evict(out=256, stride=1, out_blocks=1, budget=16, recent=0, **kw):
    return ext.lib().corope_cache_evict(*_structs(**kw), out, stride, out_blocks, budget, recent, 256, 256, None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(k_scale=None), -1), (dict(seq_lens=None), -1), (dict(block_table=None), -1), (dict(cos=256), -1), (dict(num_blocks=0), -2), (dict(B=0), -2),
    (dict(max_blocks=0), -2), (dict(cos=256, sin=256, table_rows=0), -2), (dict(D=48), -3), (dict(block_size=8), -12), (dict(block_size=48), -12),
    (dict(block_size=512), -12), (dict(code=2), -12), (dict(k=264), -12), (dict(k_stride=[2048, 1024, 56]), -12), (dict(v_stride=[2048, 1024, 72]), -12),
    (dict(v_stride=[-2048, 1024, 64]), -12), (dict(table_stride=2), -11), (dict(cos=256, sin=256, table_rows=9, rope_stride=16), -11),
    (dict(max_blocks=1 << 27, table_stride=1 << 27), -10), (dict(B=1 << 24), -10),
])
def test_every_operator_checks_the_cache_and_the_sequences(kw, rc):
    kw = dict(kw)
    k = kw.pop("k", None)
    if k is not None:      # the cache's own pointer, not the rows'
        c, s = _structs()
        c._obj.k = k
        assert ext.lib().corope_cache_append(c, s, 256, 256, _ROWS, _ROWS, 1, 1, None, None) == rc
        return
    assert _append(**kw) == rc
    assert _attend(**kw) == rc
    if "cos" not in kw:
        assert _evict(out_blocks=9, stride=9, **kw) == rc


def test_operators_check_their_own_arguments():
    assert _append(k=None) == -1 and _append(T=0) == -2 and _append(T=1 << 21) == -10 and _append(dtype=5) == -4
    assert _append(rows=(ctypes.c_int64 * 3)(-64, 64, 64)) == -11
    assert _attend(q=None) == -1 and _attend(Hq=0) == -2 and _attend(Hq=3) == -6 and _attend(T=0) == -2 and _attend(dtype=7) == -4
    assert _attend(accumulate=1, weight=None) == -1 and _attend(Hq=1 << 20, T=1 << 10) == -10
    assert _attend() == -5 and _attend(ws=None, ws_bytes=1 << 40) == -5 and _attend(ws=264, ws_bytes=1 << 40) == -5
    assert _evict(out=None) == -1 and _evict(weight=None) == -1 and _evict(budget=0) == -2 and _evict(recent=17) == -2 and _evict(recent=-1) == -2
    assert _evict(budget=17) == -2 and _evict(out_blocks=0) == -2 and _evict(stride=0) == -11
    assert b"16 bytes" in ext.lib().corope_status_string(-12)


def test_workspace_grows_with_the_call():
    def size(**kw):
        Hq, T, acc = kw.pop("Hq", 4), kw.pop("T", 1), kw.pop("accumulate", 0)
        return ext.lib().corope_cache_attn_workspace_bytes(*_structs(**kw), Hq, T, 1, acc)

    assert 0 < size() <= size(Hq=64) and size() < size(accumulate=1) and size(max_blocks=2, table_stride=2) <= size()
    assert size(D=48) == 0 and size(Hq=3) == 0 and size(T=0) == 0


def test_entry_points_refuse_cpu_tensors():
    cache = pkg.KVCache(4, 2, 16, 64, device="cpu", weights=True)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = draw((1, 2, 1, 64), 0, torch.bfloat16)
    for call in (lambda: pkg.cache_append(x, x, cache, table, lens), lambda: pkg.cache_attention(x, cache, table, lens, True, 0.1),
                 lambda: pkg.cache_evict(cache, table, lens, table, 16)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_entry_points_refuse_what_expects_a_derivative():
    """Tensors of the cache count as well; forward-mode duals are refused whatever the grad mode."""
    import torch.autograd.forward_ad as fwd

    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = draw((1, 2, 1, 64), 0, torch.float32)

    def calls(cache, k):
        return (lambda: pkg.cache_append(k, x, cache, table, lens), lambda: pkg.cache_append(x, k, cache, table, lens),
                lambda: pkg.cache_attention(k, cache, table, lens, True, 0.1), lambda: pkg.cache_evict(cache, table, lens, table, 16))

    cache = pkg.KVCache(4, 2, 16, 64, device="cpu", weights=True)
    for call in calls(cache, x.clone().requires_grad_(True))[:3]:
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    for name in ("k_scale", "v_scale", "weight"):
        cache = pkg.KVCache(4, 2, 16, 64, device="cpu", weights=True)
        getattr(cache, name).requires_grad_(True)
        for call in calls(cache, x):
            with pytest.raises(RuntimeError, match="no backward"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):
                call()
    cache = pkg.KVCache(4, 2, 16, 64, device="cpu", weights=True)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in calls(cache, dual)[:3]:
            with pytest.raises(RuntimeError, match="dual"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="dual"):
                call()
        cache.weight = fwd.make_dual(cache.weight, torch.ones_like(cache.weight))
        for call in calls(cache, x):
            with pytest.raises(RuntimeError, match="dual"):
                call()


@pytest.mark.parametrize("code,worst", [(torch.float8_e4m3fn, 2.0 ** -4), (torch.int8, 0.5 / 127)])
def test_codes_stand_for_what_was_stored(code, worst):
    """The oracle's codes: within half a step of the element (e4m3: 2^-4 of it, or of the smallest normal code; int8: of the block's largest)."""
    B, H, T, D, bs = 2, 2, 37, 32, 16
    cache = {x: torch.zeros(8, H, bs, D, dtype=torch.uint8).view(code) for x in ("k", "v")}
    cache.update(k_scale=torch.zeros(8, H), v_scale=torch.zeros(8, H), weight=None)
    k, v = (draw((B, H, T, D), i, torch.float32) for i in range(2))
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    ref.append(cache, k, v, table, [T, T])
    for b in range(B):
        for h in range(H):
            got, at, _ = ref._tokens(cache, "v", table, b, h, T)
            scale = cache["v_scale"][at, h].double()[:, None]
            step = worst * (v[b, h].double().abs().clamp(min=0) + scale * 2.0 ** -6) if code != torch.int8 else worst * 127 * scale
            assert ((got - v[b, h].double()).abs() <= 1.0001 * step).all()


def test_sizes_beyond_32_bits_are_refused():
    assert _evict(budget=1 << 30, out_blocks=1 << 26, stride=1 << 26) == -10
    for wide in ([1 << 32, 1024, 64], [1 << 40, 1024, 1 << 32]):
        assert _append(k_stride=wide) == -12 and _attend(v_stride=wide) == -12 and _evict(k_stride=wide) == -12


def test_codes_that_share_memory_are_not_written():
    for shared in ([0, 1024, 64], [2048, 0, 64]):
        for name in ("k_stride", "v_stride"):
            assert _append(**{name: shared}) == -12 and _evict(**{name: shared}) == -12
            assert _attend(**{name: shared}) == -5      # (reads them; the workspace is missing)
    assert _append(num_blocks=1, Hkv=1, k_stride=[0, 0, 64], T=0) == -2


def test_eviction_order():
    """Largest weights first, lowest slots among equal ones, NaN before everything, the last slots always."""
    bs = 16
    cache = {x: torch.zeros(4, 1, bs, 32, dtype=torch.int8) for x in ("k", "v")}
    cache.update(k_scale=torch.ones(4, 1), v_scale=torch.ones(4, 1), weight=torch.zeros(4, 1, bs))
    cache["weight"][0, 0, :8] = torch.tensor([1.0, 3.0, 1.0, float("nan"), 0.0, 3.0, 0.0, 0.0])
    lens, kept = ref.evict(cache, torch.tensor([[0, 1]]), [8], torch.tensor([[2, 3]]), 5, 1)
    assert lens.tolist() == [5] and kept[0, 0].tolist() == [0, 1, 3, 5, 7]
