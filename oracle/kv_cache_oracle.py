"""CPU oracle of the 8-bit paged cache: append, attention, eviction.

TEST INFRASTRUCTURE ONLY -- never imported by the shipped package.

The reference (Superposition09m/Co-RoPE) has no cache; the rotation is its half layout (fused-rope/rope_attn_pytorch.py:52-84).  Token by
token and head by head, with plain lists of (block, row) pairs in place of any tiling:

  codes      fp32, one rounding per operation, as the operator defines them
  attention  fp64
  eviction   the order of (weight, -slot) pairs

A cache is a dict of CPU tensors: k, v (codes), k_scale, v_scale, weight (or None).
"""

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
PER_CODE = {dtype: 1.0 / torch.tensor(largest) for dtype, largest in LARGEST.items()}   # fp32


def codes_of(x, scale):
    """Codes (as numbers, fp32) of x for `scale`: no type yet."""
    return torch.where(scale == 0, torch.zeros_like(x), x / scale)


def to_codes(x, scale, dtype):
    y = codes_of(x, scale)
    if dtype == torch.int8:
        return torch.where(y.isnan(), torch.zeros_like(y), y).round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(dtype)


def rotate(x, cos, sin, position):
    """One row [D] (or rows [H, D]) turned by row `position` of the tables (columns [0, D/2))."""
    if cos is None:
        return x
    half = x.shape[-1] // 2
    c, s = cos[position, :half].to(x.dtype), sin[position, :half].to(x.dtype)
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def append(cache, k, v, table, lens, cos=None, sin=None, positions=None, new_lens=None):
    """In place on the dict's tensors."""
    B, H, T, D = k.shape
    dtype, bs = cache["k"].dtype, cache["k"].shape[2]
    for b in range(B):
        n = T if new_lens is None else int(new_lens[b])
        first = int(lens[b]) - n
        for block in range(max(first, 0) // bs, (int(lens[b]) + bs - 1) // bs if n else 0):
            slots = [s for s in range(block * bs, min(int(lens[b]), (block + 1) * bs)) if s >= first]
            if not slots:
                continue
            page, held = int(table[b, block]), slots[0] - block * bs
            for name, src in (("k", k), ("v", v)):
                codes, scales = cache[name], cache[name + "_scale"]
                rows = []
                for s in slots:
                    row = src[b, :, s - first].float()
                    if name == "k":
                        row = rotate(row, cos, sin, s if positions is None else int(positions[b]) + s - first)
                    rows.append(row)
                rows = torch.stack(rows, dim=1)                                       # [H, slots, D]
                largest = torch.where(rows.isfinite(), rows.abs(), torch.zeros(())).amax(dim=(1, 2))
                scale = largest * PER_CODE[dtype]
                if held:
                    old = scales[page].clone()
                    scale = torch.maximum(old, scale)
                    for h in range(H):
                        if scale[h] != old[h]:
                            codes[page, h, :held] = to_codes(codes[page, h, :held].float() * old[h], scale[h], dtype)
                codes[page, :, held:held + len(slots)] = to_codes(rows, scale[:, None, None], dtype)
                scales[page] = scale
            if cache["weight"] is not None:
                cache["weight"][page, :, held:held + len(slots)] = 0.0


def _tokens(cache, name, table, b, h, length):
    """[length, D] fp64 values of head h of sequence b."""
    bs = cache["k"].shape[2]
    pages = [int(table[b, s // bs]) for s in range(length)]
    rows = torch.arange(length) % bs
    at = torch.tensor(pages, dtype=torch.long)
    return cache[name][:, h].view(torch.uint8)[at, rows].view(cache[name].dtype).double() * cache[name + "_scale"][at, h].double()[:, None], at, rows


def attention(cache, q, table, lens, causal, sm_scale, cos=None, sin=None, positions=None, new_lens=None):
    """(o, bulk, slack, weight): o [B, Hq, T, D] fp64; bulk = sum of p |v|, the size against which errors of p and of sums count; slack
    [B, Hq, T, 1] = the largest sum over d of |q k| sm_scale over the visible slots, the size of a score's terms; weight = what accumulate adds, as
    a tensor like cache["weight"]."""
    B, Hq, T, D = q.shape
    Hkv = cache["k"].shape[1]
    G = Hq // Hkv
    o, bulk, slack = torch.zeros(B, Hq, T, D, dtype=torch.float64), torch.zeros(B, Hq, T, D, dtype=torch.float64), torch.zeros(B, Hq, T, 1, dtype=torch.float64)
    weight = torch.zeros(cache["k"].shape[:3], dtype=torch.float64)
    for b in range(B):
        n, length = T if new_lens is None else int(new_lens[b]), int(lens[b])
        for h in range(Hkv):
            k, at, rows = _tokens(cache, "k", table, b, h, length)
            v, _, _ = _tokens(cache, "v", table, b, h, length)
            for t in range(min(n, T)):
                sees = length - n + t + 1 if causal else length
                if sees <= 0:
                    continue
                for g in range(G):
                    row = rotate(q[b, h * G + g, t].double(), cos, sin, length - n + t if positions is None else int(positions[b]) + t)
                    s = (k[:sees] @ row) * sm_scale
                    p = torch.softmax(s, dim=0)
                    o[b, h * G + g, t] = p @ v[:sees]
                    bulk[b, h * G + g, t] = p @ v[:sees].abs()
                    slack[b, h * G + g, t] = (k[:sees].abs() @ row.abs()).max() * sm_scale
                    weight[:, h].index_put_((at[:sees], rows[:sees]), p, accumulate=True)
    return o, bulk, slack, weight


def evict(cache, table, lens, out_table, budget, recent):
    """In place; returns (new_lens, kept)."""
    B, (_, Hkv, bs, _) = len(lens), cache["k"].shape
    dtype = cache["k"].dtype
    new_lens, kept = torch.zeros(B, dtype=torch.int32), torch.full((B, Hkv, budget), -1, dtype=torch.int32)
    before = {x: cache[x].clone() for x in ("k", "v", "k_scale", "v_scale", "weight")}
    for b in range(B):
        length = int(lens[b])
        new_lens[b] = min(length, budget)
        for h in range(Hkv):
            w = [before["weight"][int(table[b, s // bs]), h, s % bs].item() for s in range(length)]
            slots = list(range(length))
            if length > budget:
                early = slots[:length - recent]
                early.sort(key=lambda s: (0, 0.0, s) if w[s] != w[s] else (1, -w[s], s))   # NaN first
                slots = sorted(early[:budget - recent]) + slots[length - recent:]
            for j in range(0, len(slots), bs):
                part, out = slots[j:j + bs], int(out_table[b, j // bs])
                for x in ("k", "v"):
                    src = [before[x + "_scale"][int(table[b, s // bs]), h] for s in part]
                    scale = torch.stack(src).amax()
                    cache[x + "_scale"][out, h] = scale
                    for i, s in enumerate(part):
                        row = before[x][int(table[b, s // bs]), h, s % bs]
                        cache[x][out, h, i] = row if src[i] == scale else to_codes(row.float() * src[i], scale, dtype)
                for i, s in enumerate(part):
                    cache["weight"][out, h, i] = w[s]
            kept[b, h, :len(slots)] = torch.tensor(slots, dtype=torch.int32)
    return new_lens, kept
