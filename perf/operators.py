"""The 8-bit paged KV cache as a serving program uses it: tokens appended, attention over the cache, eviction by attention weight.

A case is a dict of plain values:
    op      "append"  new keys and values rotated, quantised and stored (corope_b200.cache_append)
            "attend"  attention of T queries a sequence over the cache (corope_b200.cache_attention)
            "evict"   the slots of largest accumulated weight move to new blocks (corope_b200.cache_evict)
    B, Hkv, G (query heads a K / V head), D, bs (tokens a block), S (the longest sequence, in tokens), T (new tokens a sequence)
    dtype   of q, k, v and o;  cache: "e4m3" or "int8"
    ragged  False: every sequence has S tokens.  True: lengths spread over [S / 8, S], new tokens over [1, T], and from 8 sequences on
            the last one is an empty place of a padded batch
    rope    keys and queries are rotated by position (tables as a model keeps them)
    weights attention adds its weights to the cache's;  budget, recent: what eviction keeps
One pass is one call of the public entry point.

Codes of the cache come back as they are stored, with their scales: float8 numbers, or int8 numbers that have to be equal, since every
step of their arithmetic is an fp32 operation of its own.
"""

import math
import types

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
THETA = 10000.0


# ---------------------------------------------------------------------------------------------------------------- cases
def _append(name, B, Hkv, D, bs, S, T, dtype, cache, ragged=True, rope=True):
    return {"name": name, "op": "append", "B": B, "Hkv": Hkv, "D": D, "bs": bs, "S": S, "T": T, "dtype": dtype, "cache": cache, "ragged": ragged, "rope": rope}


def _attend(name, B, Hkv, G, D, bs, S, T, dtype, cache, ragged=True, rope=True, weights=False, causal=True):
    return {"name": name, "op": "attend", "B": B, "Hkv": Hkv, "G": G, "D": D, "bs": bs, "S": S, "T": T, "dtype": dtype, "cache": cache, "ragged": ragged,
            "rope": rope, "weights": weights, "causal": causal}


def _evict(name, B, Hkv, D, bs, S, budget, recent, cache, ragged=True):
    return {"name": name, "op": "evict", "B": B, "Hkv": Hkv, "D": D, "bs": bs, "S": S, "budget": budget, "recent": recent, "cache": cache, "ragged": ragged}


def listed():
    return [
        # a decode step's append: one token of each sequence of a batch
        _append("append-token", 16, 8, 128, 64, 1000, 1, "bf16", "e4m3"),
        # prompts written to the cache after their prefill, lengths as they come
        _append("append-prompts", 4, 8, 128, 32, 4096, 4096, "f16", "int8"),
        # one user, a short conversation, grouped heads of 32 / 8 as in the benchmark: what a step costs when there is little to read
        _attend("token-short", 1, 8, 4, 128, 64, 777, 1, "bf16", "e4m3", ragged=False),
        # a server's decode step: many sequences of all lengths, small blocks
        _attend("token-batch", 64, 8, 4, 128, 16, 4096, 1, "bf16", "e4m3"),
        # two very long documents, 8 query heads a K / V head: the largest read
        _attend("token-long", 2, 8, 8, 128, 128, 131072, 1, "f16", "int8", ragged=False),
        # equal heads of a small model in fp32, the setting in which a served model is checked
        _attend("token-heads-f32", 8, 16, 1, 64, 32, 1999, 1, "f32", "int8"),
        # four draft tokens a sequence, weights gathered for eviction
        _attend("draft-weights", 16, 8, 4, 128, 64, 4000, 4, "bf16", "e4m3", weights=True),
        # a decode step of a server that evicts
        _attend("token-weights", 32, 8, 4, 128, 64, 8192, 1, "f16", "int8", weights=True),
        # a chunk of a long prompt over what the cache holds already
        _attend("chunk-prompt", 1, 8, 4, 128, 64, 9001, 1024, "bf16", "e4m3", ragged=False),
        # chunks of short prompts of a small model, weights gathered
        _attend("chunk-weights", 2, 4, 4, 64, 32, 2048, 512, "f16", "e4m3", weights=True),
        # a short cache thinned by a third
        _evict("evict-short", 4, 8, 128, 64, 1536, 1024, 64, "e4m3"),
        # long caches cut down to an eighth
        _evict("evict-long", 16, 8, 128, 64, 32768, 4096, 512, "int8"),
    ]


def _spread(lo, hi, i):
    """Whole numbers spread over [lo, hi]; the first is hi."""
    return hi - int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0))


def _lens(case):
    """(tokens in the cache, new ones among them) of each sequence."""
    B, S, T = case["B"], case["S"], case.get("T", 0)
    if not case["ragged"]:
        return [S] * B, [T] * B
    lens = [_spread(max(T, S // 8, 1), S, i) for i in range(B)]
    new = [_spread(min(T, 1), T, i) for i in range(B)]
    if B >= 8:
        lens[-1] = new[-1] = 0
    return lens, new


def work(case):
    """Every input read once, every output written once; two products over the visible (query, slot) pairs."""
    lens, new = _lens(case)
    Hkv, D = case["Hkv"], case["D"]
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": Hkv * (4.0 * sum(lens) + kept * (4 * D + 4 + 8)), "flops": 0.0}
    e = 4 if case["dtype"] == "f32" else 2
    table = 4.0 * D * max(new) if case["rope"] else 0.0
    if case["op"] == "append":
        return {"bytes": Hkv * sum(new) * 2.0 * D * (e + 1) + table, "flops": 0.0}
    G = case["G"]
    pairs = sum(t * n - (t * (t - 1) / 2 if case["causal"] else 0) for n, t in zip(lens, new))
    nbytes = Hkv * sum(lens) * (2.0 * D + (8 if case["weights"] else 0)) + 2.0 * e * Hkv * G * D * sum(new) + table
    return {"bytes": nbytes, "flops": 4.0 * D * Hkv * G * pairs}


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same kinds: sizes spread over their logarithms, cut down until it costs no more than the listed ones of its kind."""
    kind = rng.choice(("append", "token", "token", "token", "draft", "chunk", "evict"))
    D, bs = rng.choice((32, 64, 128, 128)), rng.choice((16, 32, 64, 128, 256))
    dtype, cache = rng.choice(("bf16", "bf16", "f16", "f16", "f32")), rng.choice(("e4m3", "int8"))
    ragged, rope = rng.random() < 0.7, rng.random() < 0.7
    B, Hkv, G = _log_uniform(rng, 1, 64), rng.choice((1, 2, 4, 5, 8, 16)), rng.choice((1, 2, 3, 4, 4, 8, 12))
    bytes_most, flops_most = {"append": (9e7, 1), "token": (5e8, 1e11), "draft": (2e8, 1e11), "chunk": (2e8, 1.2e11), "evict": (3e8, 1)}[kind]
    while True:
        if kind == "append":
            T = rng.choice((1, 1, _log_uniform(rng, 2, 4096)))
            case = _append("", B, Hkv, D, bs, T + _log_uniform(rng, 1, 4000), T, dtype, cache, ragged, rope)
        elif kind == "evict":
            S = _log_uniform(rng, 100, 32768)
            budget = max(2, int(S * rng.uniform(0.1, 0.9)))
            case = _evict("", B, Hkv, D, bs, S, budget, int(budget * rng.uniform(0, 0.5)), cache, ragged)
        else:
            T = 1 if kind == "token" else rng.randint(2, 8) if kind == "draft" else _log_uniform(rng, 16, 1024)
            S = T + _log_uniform(rng, 1, 65536 if kind == "token" else 8192)
            case = _attend("", B, Hkv, G, D, bs, S, T, dtype, cache, ragged, rope, weights=kind != "token" and rng.random() < 0.5 or rng.random() < 0.2,
                           causal=rng.random() < 0.9)
        w = work(case)
        # the plain form also holds the scores of every query row
        scores = case.get("T", 0) * case.get("G", 0) * Hkv * B * case["S"] * 4.0 if case["op"] == "attend" else 0.0
        if w["bytes"] <= bytes_most and w["flops"] <= flops_most and scores <= 1.5e9:
            del case["name"]
            return case
        B, Hkv = max(1, B // 2), Hkv if B > 1 else max(1, Hkv // 2)


# --------------------------------------------------------------------------------------------------------------- inputs
def _quantised(gen, blocks, Hkv, bs, D, cache):
    """Codes and scales of normal numbers whose channels differ in size, as keys and values of a trained model do."""
    dtype, qmax = CODES[cache]
    x = torch.randn((blocks, Hkv, bs, D), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((Hkv, 1, D), generator=gen, device="cuda"))
    scale = x.abs().amax(dim=(2, 3)) / qmax
    x /= scale[:, :, None, None]
    return (x.round_().to(dtype) if dtype == torch.int8 else x.to(dtype)), scale


def prepare(case, seed):
    """The cache with its block tables (blocks in any order; the pool's last block stands in the table where a sequence has none), lengths
    and the call's tensors."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, D, bs, S = (case[x] for x in ("B", "Hkv", "D", "bs", "S"))
    lens, new = _lens(case)
    wide = -(-S // bs)
    outs = -(-case["budget"] // bs) if case["op"] == "evict" else 0
    blocks = B * (wide + outs) + 1
    cache = types.SimpleNamespace(weight=None)
    cache.k, cache.k_scale = _quantised(gen, blocks, Hkv, bs, D, case["cache"])
    cache.v, cache.v_scale = _quantised(gen, blocks, Hkv, bs, D, case["cache"])
    order = torch.randperm(blocks - 1, generator=gen, device="cuda").to(torch.int32).view(B, wide + outs)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    used = torch.arange(wide, device="cuda")[None] * bs < seq_lens[:, None]
    state = {"case": case, "cache": cache, "seq_lens": seq_lens, "new_lens": torch.tensor(new, dtype=torch.int32, device="cuda"), "scale": D ** -0.5,
             "block_table": torch.where(used, order[:, :wide], blocks - 1).to(torch.int32).contiguous()}
    if case["op"] == "evict" or case.get("weights"):
        # sums of probabilities: most slots little, a few much, some nothing at all
        w = torch.exp(2.0 * torch.randn((blocks, Hkv, bs), generator=gen, device="cuda") - 4.0)
        cache.weight = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.05)
    if case["op"] == "evict":
        state["out_table"] = order[:, wide:].contiguous()
        return state
    dtype = DTYPES[case["dtype"]]
    T = case["T"]
    if case["op"] == "append":
        state["k"], state["v"] = (torch.randn((B, T, Hkv, D), generator=gen, device="cuda").to(dtype).transpose(1, 2) for _ in range(2))
    else:
        state["q"] = (1.5 * torch.randn((B, T, Hkv * case["G"], D), generator=gen, device="cuda")).to(dtype).transpose(1, 2)
    state["cos"] = state["sin"] = state["positions"] = None
    if case["rope"]:
        # the sequences went through more tokens than the cache still holds
        ahead = torch.randint(0, 100, (B,), generator=gen, device="cuda", dtype=torch.int32)
        state["positions"] = (seq_lens - state["new_lens"] + ahead).to(torch.int32)
        freq = THETA ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        angle = torch.outer(torch.arange(S + T + 100, device="cuda", dtype=torch.float64), freq)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# -------------------------------------------------------------------------------------------------------- the plain form
def _bytes(t):
    return t.view(torch.uint8)


def _rotate(x, state):
    """Half layout: pairs (d, d + D / 2) of the rows of x [B, H, T, D] turned by their position's angle, fp32."""
    x = x.float()
    if state["cos"] is None:
        return x
    at = state["positions"].long()[:, None] + torch.arange(x.shape[2], device=x.device)
    c, s = (t[at.clamp(0, t.shape[0] - 1)][:, None] for t in (state["cos"], state["sin"]))
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def _codes(x, scale, dtype, qmax):
    y = torch.where(scale == 0, 0.0, x / scale)
    if dtype == torch.int8:
        return torch.where(y.isnan(), 0.0, y).round().clamp(-qmax, qmax).to(dtype)
    return y.clamp(-qmax, qmax).to(dtype)


def _rescaled(codes, old, scale, qmax):
    """Codes of scale `old` written with `scale`: the same bits where the two are equal."""
    y = _codes(codes.float() * old, scale, codes.dtype, qmax)
    return torch.where((old == scale).expand(y.shape), _bytes(codes), _bytes(y)).view(codes.dtype)


def _append_plain(state):
    case, cache, bs = state["case"], state["cache"], state["case"]["bs"]
    dtype, qmax = CODES[case["cache"]]
    T, table = case["T"], state["block_table"].long()
    n = state["new_lens"].long()
    first = state["seq_lens"].long() - n                                  # the first new slot
    touched = first[:, None] // bs + torch.arange((T + bs - 2) // bs + 1, device=n.device)                  # [B, J] blocks of a sequence
    slot = touched[:, :, None] * bs + torch.arange(bs, device=n.device)                                     # [B, J, bs]
    t = slot - first[:, None, None]
    is_new = (t >= 0) & (t < n[:, None, None])
    is_old = t < 0
    live = is_new.any(dim=2)                                              # [B, J]: the others go to the pool's spare block, as it was
    page = torch.where(live, table.gather(1, touched.clamp(max=table.shape[1] - 1)), cache.k.shape[0] - 1)
    new_row, old_row = (m[:, :, None, :, None] for m in (is_new, is_old & live[:, :, None]))                # [B, J, 1, bs, 1]
    b = torch.arange(t.shape[0], device=n.device)[:, None, None]
    for x, codes, scales in ((_rotate(state["k"], state), cache.k, cache.k_scale), (state["v"].float(), cache.v, cache.v_scale)):
        x = x[b, :, t.clamp(0, T - 1)].transpose(2, 3)                    # [B, J, Hkv, bs, D]
        was, old = _bytes(codes)[page].view(dtype), scales[page]          # [B, J, Hkv, bs, D], [B, J, Hkv]
        amax = torch.where(new_row & x.isfinite(), x.abs(), 0.0).amax(dim=(3, 4))
        before = torch.where(old_row.any(dim=3).squeeze(-1), old, 0.0)
        scale = torch.where(live[:, :, None], torch.maximum(before, amax / qmax), old)
        s = scale[:, :, :, None, None]
        row = torch.where(new_row, _bytes(_codes(x, s, dtype, qmax)), torch.where(old_row, _bytes(_rescaled(was, before[:, :, :, None, None], s, qmax)), _bytes(was)))
        _bytes(codes)[page] = row
        scales[page] = scale
    return {"k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}


def _dense(codes, scales, table):
    """[B, Hkv, S, D] in fp32."""
    x = _bytes(codes)[table].view(codes.dtype).float() * scales[table][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend_plain(state):
    case, cache = state["case"], state["cache"]
    table, q = state["block_table"].long(), state["q"]
    B, Hq, T, D = q.shape
    Hkv, G = case["Hkv"], case["G"]
    lens, n = state["seq_lens"].long(), state["new_lens"].long()
    k, v = _dense(cache.k, cache.k_scale, table), _dense(cache.v, cache.v_scale, table)
    slot, t = torch.arange(k.shape[2], device=q.device), torch.arange(T, device=q.device)
    sees = (lens - n)[:, None] + t + 1 if case["causal"] else lens[:, None].expand(B, T)
    sees = torch.where(t < n[:, None], sees.clamp(min=0), 0)              # [B, T]
    seen = (slot < sees[:, :, None])[:, None, None]                       # [B, 1, 1, T, S]
    v = torch.where((slot < lens[:, None])[:, None, :, None], v, 0.0)
    s = (_rotate(q, state).reshape(B, Hkv, G * T, D) @ k.transpose(2, 3)).view(B, Hkv, G, T, -1) * state["scale"]
    s = torch.where(seen, s, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
    total = p.sum(dim=-1, keepdim=True)
    p = torch.where(total == 0, 0.0, p / total)
    o = (p.view(B, Hkv, G * T, -1) @ v).view(B, Hq, T, D).to(q.dtype)
    if not case["weights"]:
        return {"o": o}
    w = p.sum(dim=(2, 3)).view(B, Hkv, -1, case["bs"]).transpose(1, 2)    # [B, blocks, Hkv, bs]
    cache.weight.index_put_((table,), w, accumulate=True)
    return {"o": o, "weight": cache.weight}


def _evict_plain(state):
    case, cache, bs = state["case"], state["cache"], state["case"]["bs"]
    dtype, qmax = CODES[case["cache"]]
    table, out, lens = state["block_table"].long(), state["out_table"].long(), state["seq_lens"].long()
    B, budget = lens.shape[0], case["budget"]
    w = cache.weight[table].transpose(1, 2).flatten(2)                    # [B, Hkv, S]
    S = w.shape[2]
    slot = torch.arange(S, device=w.device)
    live = slot < lens[:, None]
    rank = torch.where(live, torch.where(slot >= (lens - case["recent"])[:, None], 2, 1), 0)[:, None].expand(w.shape)
    by_weight = w.sort(dim=2, descending=True, stable=True).indices
    order = by_weight.gather(2, rank.gather(2, by_weight).sort(dim=2, descending=True, stable=True).indices)[:, :, :budget]
    count = lens.clamp(max=budget)
    wide = out.shape[1] * bs
    order = torch.cat((order, order.new_full(order.shape[:2] + (wide - order.shape[2],), S)), dim=2)
    taken = (torch.arange(wide, device=w.device) < count[:, None])[:, None].expand(order.shape)
    at = torch.where(taken, order, S).sort(dim=2).values
    kept = torch.where(taken, at, -1)[:, :, :budget].to(torch.int32)
    at = at.clamp(max=S - 1)
    page, row, head = table[torch.arange(B, device=w.device)[:, None, None], at // bs], at % bs, torch.arange(w.shape[1], device=w.device)[:, None]
    some = taken[:, 0].view(B, -1, bs)                                    # [B, blocks, bs]
    to = torch.where(some.any(dim=2), out, cache.k.shape[0] - 1)          # blocks that get nothing: the spare one, as it was

    def blocks(x):
        return x.unflatten(2, (-1, bs)).transpose(1, 2)                   # [B, blocks, Hkv, bs, ...]

    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        moved, old = blocks(_bytes(codes)[page, head, row]).view(dtype), blocks(scales[page, head])
        scale = torch.where(some[:, :, None], old, 0.0).amax(dim=3)
        was = _bytes(codes)[to]
        new = _bytes(_rescaled(moved, old[..., None], scale[:, :, :, None, None], qmax))
        _bytes(codes)[to] = torch.where(some[:, :, None, :, None], new, was)
        scales[to] = torch.where(some.any(dim=2)[:, :, None], scale, scales[to])
    cache.weight[to] = torch.where(some[:, :, None], blocks(w.gather(2, at)), cache.weight[to])
    return {"new_lens": count.to(torch.int32), "kept": kept, "k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "weight": cache.weight}


# -------------------------------------------------------------------------------------------------------------- one pass
def _own_run(state):
    import corope_b200

    case, cache = state["case"], state["cache"]
    if case["op"] == "append":
        corope_b200.cache_append(state["k"], state["v"], cache, state["block_table"], state["seq_lens"], state["cos"], state["sin"], state["positions"],
                                 state["new_lens"])
        return {"k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    if case["op"] == "attend":
        o = corope_b200.cache_attention(state["q"], cache, state["block_table"], state["seq_lens"], case["causal"], state["scale"], state["cos"], state["sin"],
                                        state["positions"], state["new_lens"], accumulate=case["weights"])
        return {"o": o, "weight": cache.weight} if case["weights"] else {"o": o}
    new_lens, kept = corope_b200.cache_evict(cache, state["block_table"], state["seq_lens"], state["out_table"], case["budget"], case["recent"])
    return {"new_lens": new_lens, "kept": kept, "k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "weight": cache.weight}


def run(state):
    if own:
        return _own_run(state)
    return {"append": _append_plain, "attend": _attend_plain, "evict": _evict_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """Sequence by sequence (and head by head for attention), token lists in place of blocks, everything in 64 bits."""
    state = prepare(case, seed)
    cache, bs = state["cache"], case["bs"]
    lens, new = _lens(case)
    dtype, qmax = CODES[case["cache"]]
    table = state["block_table"].long()
    if case["op"] == "attend":
        return _exact_attention(case, state, lens, new)
    codes = {"k": _bytes(cache.k).view(dtype).double(), "v": _bytes(cache.v).view(dtype).double()}
    scales = {"k": cache.k_scale.double(), "v": cache.v_scale.double()}
    if case["op"] == "append":
        for b in range(case["B"]):
            n, first = new[b], lens[b] - new[b]
            if n == 0:
                continue
            rows = {"k": _turned(state["k"][b, :, :n].double(), state, b), "v": state["v"][b, :, :n].double()}
            for j in range(first // bs, (lens[b] - 1) // bs + 1):
                page, lo, hi = table[b, j], max(first, j * bs), min(lens[b], (j + 1) * bs)
                for x in ("k", "v"):
                    part = rows[x][:, lo - first:hi - first]
                    scale, held = part.abs().amax(dim=(1, 2)) / qmax, lo - j * bs
                    if held:
                        scale = torch.maximum(scale, scales[x][page])
                        codes[x][page, :, :held] = _nearest(codes[x][page, :, :held] * (scales[x][page] / scale)[:, None, None], dtype)
                    codes[x][page, :, held:held + hi - lo] = _nearest(part / scale[:, None, None], dtype)
                    scales[x][page] = scale
        whole = dtype == torch.int8   # int8 codes are compared for equality
        return {"k": None if whole else codes["k"], "v": None if whole else codes["v"], "k_scale": scales["k"], "v_scale": scales["v"]}
    weight = cache.weight.clone()
    for b in range(case["B"]):
        if lens[b] == 0:
            continue
        slot = torch.arange(lens[b], device="cuda")
        pages, row = table[b, slot // bs], slot % bs
        for h in range(case["Hkv"]):
            w = cache.weight[pages, h, row].double()
            if lens[b] > case["budget"]:
                late = slot >= lens[b] - case["recent"]
                rest = case["budget"] - case["recent"]
                early = slot[~late]
                best = torch.sort(-w[~late], stable=True).indices[:rest]
                keep = torch.cat((early[best].sort().values, slot[late]))
            else:
                keep = slot
            weight[state["out_table"][b, slot[:len(keep)] // bs].long(), h, slot[:len(keep)] % bs] = cache.weight[pages[keep], h, row[keep]]
            for x in ("k", "v"):
                size = scales[x][pages[keep], h]
                full = torch.zeros(-(-len(keep) // bs) * bs, dtype=torch.float64, device="cuda")
                full[:len(keep)] = size
                best = full.view(-1, bs).amax(dim=1)
                moved = _nearest(codes[x][pages[keep], h, row[keep]] * (size / best.repeat_interleave(bs)[:len(keep)])[:, None], dtype)
                to = state["out_table"][b].long()
                codes[x][to[slot[:len(keep)] // bs], h, slot[:len(keep)] % bs] = moved
                scales[x][to[:len(best)], h] = best
    whole = dtype == torch.int8
    return {"new_lens": None, "kept": None, "k": None if whole else codes["k"], "v": None if whole else codes["v"], "k_scale": scales["k"],
            "v_scale": scales["v"], "weight": weight.double()}


def _nearest(x, dtype):
    return x.round() if dtype == torch.int8 else x.to(dtype).double()


def _turned(x, state, b):
    """Rows of x [H, n, D], fp64, as complex numbers times exp(i angle)."""
    if state["cos"] is None:
        return x
    start, half = int(state["positions"][b]), x.shape[-1] // 2
    turn = torch.complex(state["cos"].double(), state["sin"].double())[start:start + x.shape[1]]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
    return torch.cat((z.real, z.imag), dim=-1)


def _exact_attention(case, state, lens, new):
    cache, bs, G = state["cache"], case["bs"], case["G"]
    o = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    weight = cache.weight.double() if case["weights"] else None
    for b in range(case["B"]):
        if new[b] == 0 or lens[b] == 0:
            continue
        slot = torch.arange(lens[b], device="cuda")
        page, row = state["block_table"][b].long()[slot // bs], slot % bs
        q = _turned(state["q"][b, :, :new[b]].double(), state, b)
        for h in range(case["Hkv"]):
            k = cache.k[:, h].view(torch.uint8)[page, row].view(cache.k.dtype).double() * cache.k_scale[page, h].double()[:, None]
            v = cache.v[:, h].view(torch.uint8)[page, row].view(cache.v.dtype).double() * cache.v_scale[page, h].double()[:, None]
            s = torch.einsum("gtd,sd->gts", q[h * G:(h + 1) * G], k) * case["D"] ** -0.5
            if case["causal"]:
                s += torch.triu(torch.full((new[b], lens[b]), -math.inf, dtype=torch.float64, device="cuda"), lens[b] - new[b] + 1)
            p = torch.softmax(s, dim=-1)
            o[b, h * G:(h + 1) * G, :new[b]] = torch.einsum("gts,sd->gtd", p, v)
            if case["weights"]:
                weight[page, h, row] += p.sum(dim=(0, 1))
    return {"o": o, "weight": weight} if case["weights"] else {"o": o}
