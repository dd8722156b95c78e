"""Attention over the paged cache, eviction by its weights, and the cases they are measured on.

What an engine does between two compressions and instead of scoring keys: one decoding step of attention
over the cache that adds up the weight every cached token received (``ops.attend_paged``), the same for a
tree of drafted tokens, eviction of the tokens with the least accumulated weight (``ops.evict_step``,
``ops.select_by_weight``), and attention over the blocks that bounds of their keys select for each query
(``ops.update_block_bounds``, ``ops.attend_blocks``).

A case is one call on one layer (evictions: on every layer of a request).  The plain form is the same
operator in elementary torch operations in 32 bits (block scores in 64: they decide which blocks are read);
``exact`` is the definition once more in 64 bits, one sequence at a time.  Calls that update the cache or
the weights in place first write the values that the engine left there, so every pass sees the same data.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
# (query heads, KV heads, head dim) of the models the repository's configurations name
HEADS = {"qwen3_8b": (32, 8, 128), "qwen3_32b": (64, 8, 128), "qwen_7b": (28, 4, 128), "gpt_oss": (64, 8, 64),
         "dim256": (32, 8, 256)}


def _case(kind: str, model: str, seqs: int, tokens: int, **more) -> dict:
    q, kv, d = HEADS[model]
    case = {"kind": kind, "q_heads": q, "kv_heads": kv, "head_dim": d, "seqs": seqs, "tokens": tokens,
            "shortest": tokens, "lens_seed": 0, "layers": 1, "block": 16, "dtype": "bf16", "query": "bf16",
            "row_scales": False}
    if kind == "attend":
        case["mode"] = "add"
    elif kind == "tree":
        case.update(drafts=16, fewest=16)
    elif kind in ("evict", "pick"):
        case.update(budget=tokens // 2, window=128, reduce="mean", prefill=0)
    elif kind == "blocks":
        case.update(top=64, sinks=1, recent=2, group="max", new=1)
    case.update(more)
    return case


def listed() -> list:
    return [
        # The smallest decoding step: one request that has just begun.
        _case("attend", "qwen3_8b", 1, 160, name="attend_one_160"),
        # The steady state of compressed requests: sixteen of them, budget + 128 tokens each.
        _case("attend", "qwen3_8b", 16, 2176, name="attend_16x2176"),
        # Long contexts in an fp8 cache with a scale per row, sixteen requests.
        _case("attend", "qwen3_8b", 16, 16384, dtype="fp8", row_scales=True, name="attend_fp8_16x16k"),
        # Requests of every length, head dimension 64, the weights of this step alone.
        _case("attend", "gpt_oss", 24, 12001, shortest=1500, lens_seed=5, mode="set", name="attend_ragged_d64"),
        # One request, sixteen drafted tokens.
        _case("tree", "qwen3_8b", 1, 1217, name="tree_one_16"),
        # Eight requests with up to thirty-two drafted tokens each, eight query heads per KV head.
        _case("tree", "qwen3_32b", 8, 4096, drafts=32, fewest=5, shortest=2500, lens_seed=3, name="tree_8x32_g8"),
        # Two long contexts, sixty drafted tokens each, fp16.
        _case("tree", "qwen3_8b", 2, 32768, drafts=60, fewest=60, dtype="fp16", query="fp16", name="tree_2x60_32k"),
        # A whole eviction of one decoding request over every layer of a model: the layers agree on a keep set per head.
        _case("evict", "qwen3_8b", 1, 2176, layers=36, budget=2048, name="evict_one_request"),
        # The keep sets alone, one per layer, for eight prompts.
        _case("pick", "qwen3_8b", 8, 8192, layers=36, budget=2048, reduce="none", name="pick_8x8k_per_layer"),
        # A decoding step over the blocks worth reading: one short request, sixteen long ones, one very long one.
        _case("blocks", "qwen3_8b", 1, 3001, top=32, name="blocks_one_3k"),
        _case("blocks", "qwen3_8b", 16, 16384, top=128, name="blocks_16x16k"),
        # The first step after a prompt: the bounds of every block are new.
        _case("blocks", "qwen_7b", 2, 131072, top=256, new=0, name="blocks_after_prompt_128k"),
    ]


def _spread(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "tree", "tree", "tree", "evict", "pick", "blocks", "blocks", "blocks"])
    model = rng.choice(sorted(HEADS))
    q, kv, d = HEADS[model]
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp8"])
    more = {"dtype": dtype, "query": dtype if dtype != "fp8" else rng.choice(["bf16", "fp16"]),
            "row_scales": dtype == "fp8" and rng.random() < 0.5, "block": rng.choice([16, 16, 16, 32, 64, 8, 1, 24]),
            "lens_seed": rng.randrange(1 << 20)}
    size = 1 if dtype == "fp8" else 2
    tokens = _spread(rng, 40, 40000)
    seqs = _spread(rng, 1, 32)
    if kind == "attend":
        seqs = max(1, min(seqs, int(2.6e8 / (tokens * kv * d * size))))
        more["mode"] = rng.choice(["add", "add", "set"])
    elif kind == "tree":
        seqs = max(1, min(seqs, int(6e7 / (tokens * kv * d))))
        drafts = max(2, min(_spread(rng, 2, 64), tokens, int(6e10 / (4 * tokens * seqs * q * d))))
        more.update(drafts=drafts, fewest=rng.choice([drafts, 1]))
    elif kind in ("evict", "pick"):
        layers = _spread(rng, 1, 36)
        tokens = _spread(rng, 300, 16000)
        most = 1.4e8 if kind == "evict" else 8e8
        seqs = max(1, min(seqs, int(most / (tokens * layers * kv * d * size))))
        layers = max(1, min(layers, int(most / (tokens * seqs * kv * d * size))))
        more.update(layers=layers, budget=max(140, int(tokens * rng.uniform(0.1, 0.95))), window=rng.choice([0, 32, 128]),
                    reduce=rng.choice(["mean", "max", "none"]), prefill=rng.choice([0, 0, 33]))
    else:
        more["block"] = rng.choice([16, 16, 32, 64])
        tokens = _spread(rng, 300, 130000)
        seqs = max(1, min(seqs, int(2.5e8 / (tokens * kv * d * size))))
        top = min(_spread(rng, 8, 300), -(-tokens // more["block"]) + 3)
        more.update(top=top, sinks=rng.choice([0, 1, 2]), recent=rng.choice([1, 2, 4]), group=rng.choice(["max", "mean"]),
                    new=rng.choice([1, 1, 1, 0]))
    more["shortest"] = tokens if rng.random() < 0.5 else rng.randint(max(1, tokens // 8), tokens)
    if kind in ("evict", "pick"):
        more["shortest"] = max(more["shortest"], min(tokens, 150))
    elif kind == "tree":
        more["shortest"] = max(more["shortest"], more["drafts"])
    return _case(kind, model, seqs, tokens, **more)


# ------------------------------------------------------------------------------- inputs
def _lens(case: dict) -> list:
    """Cached tokens of every sequence: the longest first, the others drawn down to the shortest."""
    rng = random.Random(case["lens_seed"])
    return [case["tokens"]] + [rng.randint(case["shortest"], case["tokens"]) for _ in range(case["seqs"] - 1)]


def _draft_counts(case: dict) -> list:
    rng = random.Random(case["lens_seed"] + 1)
    return [case["drafts"]] + [rng.randint(case["fewest"], case["drafts"]) for _ in range(case["seqs"] - 1)]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    lens, bs, hkv, d, layers = _lens(case), case["block"], case["kv_heads"], case["head_dim"], case["layers"]
    counts = [-(-t // bs) for t in lens]
    pool = sum(counts) + sum(counts) // 10 + 1
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    ends = [sum(counts[:i + 1]) for i in range(len(counts))]
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=DEV)
    for b, n in enumerate(counts):
        table[b, :n] = order[ends[b] - n:ends[b]]
    s = {"case": case, "lens": lens, "table": table, "lens_dev": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "pool": pool}

    # (a keep set goes by the weights alone: one layer's rows stand for those of every layer)
    held = layers if case["kind"] != "pick" else 1
    for side in ("k", "v"):
        s[side] = torch.empty(held, pool, bs, hkv, d, dtype=DTYPES[case["dtype"]], device=DEV)
        s[side + "_scales"] = torch.empty(held, pool * bs * hkv, device=DEV) if case["row_scales"] else None
        for layer in range(held):
            x = torch.randn(pool, bs, hkv, d, generator=g, device=DEV)
            if side == "k":
                x = x + 0.5 * torch.randn(1, 1, hkv, d, generator=g, device=DEV)
            if case["dtype"] == "fp8":
                if case["row_scales"]:
                    sc = x.abs().amax(-1, keepdim=True) / 448
                    s[side + "_scales"][layer] = sc.flatten()
                    x = x / sc
                x = x.clamp(-448, 448)
            s[side][layer] = x.to(DTYPES[case["dtype"]])
    if case["kind"] in ("attend", "tree", "blocks"):
        drafts = _draft_counts(case) if case["kind"] == "tree" else [1] * len(lens)
        s["drafts"] = drafts
        starts = [sum(drafts[:i]) for i in range(len(drafts) + 1)]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        # every drafted token hangs on an earlier one, or on the last cached token
        parents = [host.randint(max(-1, i - 5), i - 1) if i else -1 for n in drafts for i in range(n)]
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
        s["q"] = (2 * torch.randn(starts[-1], case["q_heads"], d, generator=g, device=DEV)).to(DTYPES[case["query"]])
        s["q"] = s["q"].contiguous()
        s["scale"] = d ** -0.5
    if case["kind"] in ("attend", "evict", "pick"):
        u = torch.rand(layers, pool, bs, hkv, generator=g, device=DEV)
        s["weights_before"] = u.pow(4) * 20
        s["weights"] = s["weights_before"].clone()
    if case["kind"] == "evict":
        for name in ("k", "v") + (("k_scales", "v_scales") if case["row_scales"] else ()):
            s[name + "_before"] = s[name].clone()
    if case["kind"] in ("evict", "pick"):
        s["budgets"] = [min(case["budget"], t) for t in lens]
        s["budgets_dev"] = torch.tensor(s["budgets"], dtype=torch.int32, device=DEV)
    if case["kind"] == "blocks":
        kind = DTYPES[case["dtype"]] if case["dtype"] != "fp8" else torch.bfloat16
        s["bounds"] = torch.zeros(1, pool, hkv, 2, d, dtype=kind, device=DEV)
        if case["new"]:
            _plain_bounds(s, 0)        # the steps before this one have left the bounds of their blocks
    return s


# --------------------------------------------------------------------------- plain forms
def _take(cache, page, off, head=None):
    """Rows of a cache layer in 32 bits (an fp8 cache is indexed by its bytes)."""
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    x = raw[page, off] if head is None else raw[page, off, head]
    return x.view(cache.dtype).float()


def _take_scaled(s, side, page, off, head=None):
    x = _take(s[side][0], page, off, head)
    sc = s[side + "_scales"]
    if sc is not None:
        hkv = s["case"]["kv_heads"]
        sc = sc[0].view(s["pool"], s["case"]["block"], hkv)
        x = x * (sc[page, off] if head is None else sc[page, off, head]).unsqueeze(-1)
    return x


def _softmax_rows(scores):
    """Weights and logarithm of the sum along the last axis; a row of -inf alone gives zeros and -inf."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total), (torch.log(total) + top).squeeze(-1)


def _plain_attend(s):
    """Every row of a sequence sees the cached tokens before the sequence's own new ones, its ancestors among
    those, and itself.  Returns (out, lse, weight of every (sequence, token, KV head))."""
    case = s["case"]
    hkv, g, bs = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["block"]
    n, nb, dev = max(s["drafts"]), len(s["lens"]), s["q"].device
    t = torch.arange(max(s["lens"]), device=dev)
    page = s["table"].long()[:, t // bs]
    live = t[None] < s["lens_dev"][:, None]
    keys = _take_scaled(s, "k", page, (t % bs)[None].expand_as(page))
    values = _take_scaled(s, "v", page, (t % bs)[None].expand_as(page)) * live[..., None, None]
    starts = s["starts"].long()
    i = torch.arange(n, device=dev)
    have = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + i).clamp(max=starts.numel() and s["q"].shape[0] - 1)
    q = s["q"][at].float().view(nb, n, hkv, g, -1).permute(0, 2, 1, 3, 4).reshape(nb, hkv, n * g, -1)
    scores = torch.matmul(q, keys.permute(0, 2, 3, 1).contiguous()) * s["scale"]
    # ancestors: the reach of the parent relation
    par = s["parents"].long()[at]
    step = ((par[:, :, None] == i) & (i[None, :, None] < have[:, None, None])).float()
    reach = torch.linalg.matrix_power(step + torch.eye(n, device=dev), n) > 0
    base = (s["lens_dev"].long() - have)[:, None]
    draft = t[None] - base
    sees = (draft < 0)[:, None] | torch.gather(reach, 2, draft.clamp(0, n - 1)[:, None].expand(nb, n, t.numel())) & (draft >= 0)[:, None]
    sees = sees & live[:, None]
    scores = scores.view(nb, hkv, n, g, -1).masked_fill(~sees[:, None, :, None], -math.inf)
    p, lse = _softmax_rows(scores)
    out = torch.matmul(p.view(nb, hkv, n * g, -1), values.permute(0, 2, 1, 3).contiguous()).view(nb, hkv, n, g, -1)
    row = torch.arange(s["q"].shape[0], device=dev)
    seq = torch.searchsorted(starts, row, right=True) - 1
    k = row - starts[seq]
    out = out[seq, :, k].reshape(row.numel(), hkv * g, -1).to(s["q"].dtype)
    lse = lse[seq, :, k].reshape(row.numel(), hkv * g)
    weight = (p * (i < have[:, None])[:, None, :, None, None]).sum((2, 3)).permute(0, 2, 1)
    return out, lse, weight, live, page, t


def _plain_add_weights(s, weight, live, page, t):
    """Adds (or, for the newest token and in mode "set", writes) the weights of the live tokens in their slots."""
    case = s["case"]
    w = s["weights"][0].view(-1, case["kv_heads"])
    slot = page * case["block"] + t % case["block"]
    fresh = t[None] >= (s["lens_dev"] - 1)[:, None] if case["mode"] == "add" else torch.ones_like(live)
    new = torch.where(fresh[..., None], weight, w[slot] + weight)
    w.index_put_((torch.where(live, slot, slot[:, :1]),), torch.where(live[..., None], new, new[:, :1]))


def _plain_bounds(s, new):
    """Least and largest key per block, KV head and dimension, of the blocks that hold the `new` last tokens
    of every sequence (0: of all its blocks)."""
    case = s["case"]
    bs, nb = case["block"], s["table"].shape[1]
    j = torch.arange(nb, device=DEV)
    first = (s["lens_dev"].long() - new).clamp(min=0) // bs if new else torch.zeros_like(s["lens_dev"]).long()
    if new:
        j = first[:, None] + torch.arange((new + bs - 2) // bs + 1, device=DEV)
    else:
        j = j[None].expand(len(s["lens"]), nb)
    inside = j * bs < s["lens_dev"][:, None]
    jc = torch.minimum(j, (s["lens_dev"].long()[:, None] - 1) // bs)     # behind the end: the last block once more
    page = s["table"].long().gather(1, jc)
    off = torch.arange(bs, device=DEV)
    keys = _take_scaled(s, "k", page[..., None].expand(*page.shape, bs), off.expand(*page.shape, bs))
    live = (jc[..., None] * bs + off < s["lens_dev"][:, None, None])[..., None, None]
    b = s["bounds"][0]
    low = keys.masked_fill(~live, math.inf).amin(2).to(b.dtype)
    high = keys.masked_fill(~live, -math.inf).amax(2).to(b.dtype)
    b[page] = torch.stack([low, high], 3)


def _plain_blocks(s):
    case = s["case"]
    hkv, g, bs, d = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["block"], case["head_dim"]
    nseq, nb, dev = len(s["lens"]), s["table"].shape[1], s["q"].device
    count = (s["lens_dev"].long() + bs - 1) // bs
    j = torch.arange(nb, device=dev)
    bounds = s["bounds"][0][s["table"].long()]                       # [B, nb, H, 2, D]
    q = s["q"].view(nseq, hkv, g, d)
    # max(q * low, q * high) summed: the positive part of q meets the largest key, the negative part the least
    low, high = (bounds[:, :, :, k].permute(0, 2, 3, 1).double().contiguous() for k in (0, 1))
    bound = torch.matmul(q.double().clamp(min=0), high) + torch.matmul(q.double().clamp(max=0), low)
    score = (bound.amax(2) if case["group"] == "max" else bound.mean(2)).float()
    forced = (j < case["sinks"]) | (j >= (count - case["recent"])[:, None])
    score = score.masked_fill(forced[:, None], math.inf).masked_fill((j >= count[:, None])[:, None], -math.inf)
    k = min(case["top"], nb)
    # the lowest index first among equals
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k]
    used = torch.arange(k, device=dev) < count[:, None, None]
    best = torch.sort(torch.where(used, best, torch.full_like(best, nb)), -1).values
    used = best < nb
    chosen = torch.where(used, best, torch.zeros_like(best))
    page = s["table"].long().gather(1, chosen.view(nseq, -1)).view(nseq, hkv, k)
    off = torch.arange(bs, device=dev)
    live = used[..., None] & (chosen[..., None] * bs + off < s["lens_dev"][:, None, None, None])
    shape = (nseq, hkv, k, bs)
    at = (page[..., None].expand(shape), off.expand(shape), torch.arange(hkv, device=dev).view(1, -1, 1, 1).expand(shape))
    keys = _take_scaled(s, "k", *at).view(nseq, hkv, k * bs, d)
    values = (_take_scaled(s, "v", *at) * live[..., None]).view(nseq, hkv, k * bs, d)
    scores = torch.matmul(q.float(), keys.transpose(2, 3).contiguous()) * s["scale"]
    scores = scores.masked_fill(~live.view(nseq, hkv, 1, k * bs), -math.inf)
    p, lse = _softmax_rows(scores)
    out = torch.matmul(p, values).view(nseq, hkv * g, d).to(s["q"].dtype)
    ids = torch.full((nseq, hkv, case["top"]), -1, dtype=torch.int32, device=dev)
    ids[..., :k] = torch.where(used, best, torch.full_like(best, -1)).int()
    return out, lse.view(nseq, hkv * g), ids


def _plain_pick(s):
    """Keep rows [B (x layers), Hkv, budget] (-1 behind a sequence's own budget) and the selection scores."""
    case = s["case"]
    bs, nseq = case["block"], len(s["lens"])
    t = torch.arange(max(s["lens"]), device=DEV)
    slot = s["table"].long()[:, t // bs] * bs + t % bs
    w = s["weights"].view(case["layers"], -1, case["kv_heads"])[:, slot].permute(1, 0, 3, 2)       # [B, L, H, T]
    if case["reduce"] == "mean":
        w = (w.double().sum(1, keepdim=True) / case["layers"]).float()
    elif case["reduce"] == "max":
        w = w.amax(1, keepdim=True)
    count = s["lens_dev"].view(-1, 1, 1, 1)
    forced = (t >= count - case["window"]) | (t < case["prefill"])
    w = w.masked_fill(forced, math.inf).masked_fill(t >= count, -math.inf)
    k = max(s["budgets"])
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :k]
    used = torch.arange(k, device=DEV) < s["budgets_dev"].view(-1, 1, 1, 1)
    keep = torch.sort(torch.where(used, best, torch.full_like(best, 1 << 30)), -1).values
    keep = torch.where(used, keep, torch.full_like(keep, -1)).int()
    return keep.view(-1, k), w


def _plain_evict(s):
    case = s["case"]
    bs, nseq, hkv = case["block"], len(s["lens"]), case["kv_heads"]
    keep, _ = _plain_pick(s)
    k = keep.shape[1]
    per = keep.view(nseq, -1, hkv, k).expand(nseq, case["layers"], hkv, k).long()
    j = torch.arange(k, device=DEV)
    used = per >= 0
    src = torch.where(used, per, j.clamp(max=k - 1).expand_as(per))
    # behind a budget: row j onto itself (the table's last block once more where it has none there)
    last = (s["table"].shape[1] * bs) - 1
    src = src.clamp(max=last)
    seq = torch.arange(nseq, device=DEV).view(-1, 1, 1, 1)
    slot_of = s["table"].long()[:, torch.arange(s["table"].shape[1] * bs, device=DEV) // bs] * bs \
        + torch.arange(s["table"].shape[1] * bs, device=DEV) % bs
    source = slot_of[seq, src]                                        # [B, L, H, k]
    target = slot_of[seq, j.expand_as(src)]
    # targets behind a budget write what their first slot gets, so that no slot has two values
    source = torch.where(used, source, source[..., :1])
    target = torch.where(used, target, target[..., :1])
    layer = torch.arange(case["layers"], device=DEV).view(1, -1, 1, 1).expand_as(src)
    head = torch.arange(hkv, device=DEV).view(1, 1, -1, 1).expand_as(src)
    w = s["weights"].view(case["layers"], -1, hkv)
    w.index_put_((layer, target, head), w[layer, source, head])
    for side in ("k", "v"):
        for layer, cache in enumerate(s[side]):
            raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
            flat = raw.view(-1, hkv, case["head_dim"])
            flat.index_put_((target[:, layer], head[:, layer]), flat[source[:, layer], head[:, layer]])
            if s[side + "_scales"] is not None:
                sc = s[side + "_scales"][layer].view(-1, hkv)
                sc.index_put_((target[:, layer], head[:, layer]), sc[source[:, layer], head[:, layer]])
    return keep


def _restore(s):
    """What the engine writes between two calls on one cache: here everything that a call changes."""
    case = s["case"]
    if case["kind"] == "attend" and case["mode"] == "add" or case["kind"] == "evict":
        s["weights"].copy_(s["weights_before"])
    if case["kind"] == "evict":
        for name in ("k", "v", "k_scales", "v_scales"):
            if s[name] is not None:
                s[name].copy_(s[name + "_before"])


def _evict_outputs(s, keep):
    """The keep rows and the whole cache: rows, scales where it has them, weights."""
    got = {"keep": keep, "k": s["k"], "v": s["v"], "weights": s["weights"]}
    if s["k_scales"] is not None:
        got["k_scales"], got["v_scales"] = s["k_scales"], s["v_scales"]
    return got


# --------------------------------------------------------------------------------- calls
def _handles(s):
    """The description of the cache and of the batch that a program keeps over its calls."""
    if "kv" not in s:
        from triattention_amd import ops
        case = s["case"]
        held = [layer % s["k"].shape[0] for layer in range(case["layers"])]
        per_layer = [None if s[name] is None else [s[name][layer] for layer in held]
                     for name in ("k", "v", "k_scales", "v_scales")]
        s["kv"] = ops.PagedKV(per_layer[0], per_layer[1], "half", per_layer[2], per_layer[3])
        evicts = case["kind"] in ("evict", "pick")
        s["batch"] = ops.StepBatch(torch.device(DEV), s["lens"], block_tables=s["table"],
                                   budgets=s["budgets"] if evicts else None,
                                   prefill_lens=[case["prefill"]] * len(s["lens"]) if evicts else None)
        if evicts:
            s["evict"] = ops.EvictConfig(window_size=case["window"], protect_prefill=case["prefill"] > 0,
                                         layer_reduce=None if case["reduce"] == "none" else case["reduce"])
    return s["kv"], s["batch"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    _restore(s)
    if own:
        from triattention_amd import ops
        kv, batch = _handles(s)
        if kind == "attend":
            out, lse = ops.attend_paged(kv, batch, s["q"], scale=s["scale"], weights=s["weights"],
                                        weight_mode=case["mode"], want_lse=True)
            return out, lse, s["weights"]
        if kind == "tree":
            return ops.attend_paged(kv, batch, s["q"], scale=s["scale"], row_starts=s["starts"], parents=s["parents"],
                                    max_rows=case["drafts"], want_lse=True)
        if kind == "blocks":
            ops.update_block_bounds(kv, batch, s["bounds"], new_tokens=case["new"] or None)
            out, lse, ids = ops.attend_blocks(kv, batch, s["q"], s["bounds"], top_blocks=case["top"], sink_blocks=case["sinks"],
                                              recent_blocks=case["recent"], group_reduce=case["group"], scale=s["scale"],
                                              want_lse=True)
            return out, lse, ids, s["bounds"]
        if kind == "pick":
            keep, scores = ops.select_by_weight(kv, batch, s["weights"], s["evict"], want_scores=True)
            return keep, scores
        keep = ops.evict_step(kv, batch, s["weights"], s["evict"])
        return _evict_outputs(s, keep)
    if kind in ("attend", "tree"):
        out, lse, *weighted = _plain_attend(s)
        if kind == "tree":
            return out, lse
        _plain_add_weights(s, *weighted)
        return out, lse, s["weights"]
    if kind == "blocks":
        _plain_bounds(s, case["new"])
        return (*_plain_blocks(s), s["bounds"])
    if kind == "pick":
        keep, w = _plain_pick(s)
        return keep, w.reshape(-1, w.shape[-1])
    return _evict_outputs(s, _plain_evict(s))


# ---------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    lens, hkv, hq, d, layers = _lens(case), case["kv_heads"], case["q_heads"], case["head_dim"], case["layers"]
    size = 1 if case["dtype"] == "fp8" else 2
    row = d * size + (4 if case["row_scales"] else 0)
    total = sum(lens)
    slots = (sum(-(-t // case["block"]) for t in lens) * 11 // 10 + 1) * case["block"]
    if case["kind"] == "attend":
        weights = total * hkv * 4 * (2 if case["mode"] == "add" else 1) + (2 * slots * hkv * 4 if case["mode"] == "add" else 0)
        return {"bytes": total * hkv * row * 2 + len(lens) * hq * (d * 4 + 4) + weights, "flops": 4 * total * hq * d}
    if case["kind"] == "tree":
        drafts = _draft_counts(case)
        return {"bytes": total * hkv * row * 2 + sum(drafts) * hq * (d * 4 + 4),
                "flops": sum(4 * t * n * hq * d for t, n in zip(lens, drafts))}
    if case["kind"] == "blocks":
        bs = case["block"]
        counts = [-(-t // bs) for t in lens]
        fresh = total if not case["new"] else len(lens) * bs
        read = sum(min(t, case["top"] * bs) for t in lens)
        bsize = 2 if case["dtype"] == "fp8" else size
        written = sum(counts) if not case["new"] else len(lens)
        return {"bytes": fresh * hkv * row + (sum(counts) + written) * hkv * 2 * d * bsize + read * hkv * row * 2
                + len(lens) * hq * (d * 4 + 4), "flops": 4 * read * hq * d + 4 * sum(counts) * hq * d}
    keeps = sum(min(case["budget"], t) for t in lens) * hkv * (layers if case["reduce"] == "none" else 1) * 4
    weights = total * layers * hkv * 4
    if case["kind"] == "pick":
        rows = len(lens) * hkv * (layers if case["reduce"] == "none" else 1)
        return {"bytes": weights + keeps + rows * max(lens) * 4, "flops": weights / 4}
    kept = sum(min(case["budget"], t) for t in lens) * layers * hkv
    restored = slots * layers * hkv * (2 * row + 4)
    # moved rows are read and written, restored ones too
    return {"bytes": weights + keeps + 2 * kept * (2 * row + 4) + 2 * restored, "flops": weights / 4}


# --------------------------------------------------------------------------------- exact
def _exact_rows(s, side, b, layer=0):
    """Rows [T, H, D] of sequence b in 64 bits."""
    case, t = s["case"], s["lens"][b]
    bs = case["block"]
    pages = s["table"][b].tolist()[:-(-t // bs)]
    cache = s[side][layer]
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    x = raw[torch.tensor(pages, device=DEV)].view(cache.dtype).double().flatten(0, 1)[:t]
    if s[side + "_scales"] is not None:
        sc = s[side + "_scales"][layer].view(s["pool"], bs, -1)[torch.tensor(pages, device=DEV)].flatten(0, 1)[:t]
        x = x * sc.double().unsqueeze(-1)
    return x


def _exact_slots(s, b):
    t, bs = s["lens"][b], s["case"]["block"]
    pages = s["table"][b].tolist()
    return torch.tensor([pages[i // bs] * bs + i % bs for i in range(t)], device=DEV)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    hkv, g, kind = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["kind"]
    if kind in ("attend", "tree"):
        starts, parents = s["starts"].tolist(), s["parents"].tolist()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
        weights = s["weights_before"].double().view(-1, hkv) if kind == "attend" else None
        for b, t in enumerate(s["lens"]):
            keys, values = _exact_rows(s, "k", b), _exact_rows(s, "v", b)
            n = starts[b + 1] - starts[b]
            line = []
            for i in range(n):
                p = parents[starts[b] + i]
                line.append({i} | (line[p] if p >= 0 else set()))
            hidden = torch.zeros(n, t, dtype=torch.bool, device=DEV)
            hidden[:, t - n:] = torch.tensor([[j not in line[i] for j in range(n)] for i in range(n)], device=DEV)
            for h in range(hkv):
                q = s["q"][starts[b]:starts[b + 1], h * g:(h + 1) * g].double()
                sc = torch.einsum("ngd,td->ngt", q, keys[:, h]) * s["scale"]
                sc = sc.masked_fill(hidden[:, None], -math.inf)
                z = torch.logsumexp(sc, -1)
                p = torch.exp(sc - z[..., None])
                out[starts[b]:starts[b + 1], h * g:(h + 1) * g] = torch.einsum("ngt,td->ngd", p, values[:, h])
                lse[starts[b]:starts[b + 1], h * g:(h + 1) * g] = z
                if weights is not None:
                    slots = _exact_slots(s, b) if h == 0 else slots
                    had = weights[slots, h]
                    if case["mode"] == "set":
                        had = torch.zeros_like(had)
                    had[t - n:] = 0
                    weights[slots, h] = had + p.sum((0, 1))
        return (out, lse) if kind == "tree" else (out, lse, weights.view(s["weights"].shape))
    if kind == "blocks":
        bs, d = case["block"], case["head_dim"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
        ids = torch.full((len(s["lens"]), hkv, case["top"]), -1, dtype=torch.int32, device=DEV)
        bounds = s["bounds"].double()
        for b, t in enumerate(s["lens"]):
            keys, values = _exact_rows(s, "k", b), _exact_rows(s, "v", b)
            nb = -(-t // bs)
            pages = s["table"][b, :nb].long()
            full = torch.nn.functional.pad(keys, (0, 0, 0, 0, 0, nb * bs - t), value=math.nan).view(nb, bs, hkv, d)
            # (the keys of a scaled fp8 cache are products in 32 bits before the bound is rounded)
            low = full.nan_to_num(nan=math.inf).amin(1).float().to(s["bounds"].dtype)
            high = full.nan_to_num(nan=-math.inf).amax(1).float().to(s["bounds"].dtype)
            bounds[0, pages] = torch.stack([low, high], 2).double()
            q = s["q"][b].double().view(hkv, g, d)
            for h in range(hkv):
                sc = torch.maximum(q[h][:, None] * low[:, h].double(), q[h][:, None] * high[:, h].double()).sum(-1) if nb < 4096 else \
                    torch.stack([torch.maximum(x * low[:, h].double(), x * high[:, h].double()).sum(-1) for x in q[h]])
                sc = (sc.amax(0) if case["group"] == "max" else sc.mean(0)).float()
                sc[:case["sinks"]] = math.inf
                sc[max(0, nb - case["recent"]):] = math.inf
                best = torch.sort(sc, descending=True, stable=True).indices[:case["top"]].sort().values
                ids[b, h, :best.numel()] = best.int()
                at = (best[:, None] * bs + torch.arange(bs, device=DEV)).flatten()
                at = at[at < t]
                w = (q[h] @ keys[at, h].t()) * s["scale"]
                z = torch.logsumexp(w, -1)
                out[b, h * g:(h + 1) * g] = torch.exp(w - z[:, None]) @ values[at, h]
                lse[b, h * g:(h + 1) * g] = z
        return out, lse, ids, bounds
    # keep sets: one row at a time
    k, longest = max(s["budgets"]), max(s["lens"])
    keep, scores = [], []
    flat = s["weights_before"].double().view(case["layers"], -1, hkv)
    for b, t in enumerate(s["lens"]):
        w = flat[:, _exact_slots(s, b)].permute(0, 2, 1)
        w = w.mean(0, keepdim=True) if case["reduce"] == "mean" else w.amax(0, keepdim=True) if case["reduce"] == "max" else w
        w = w.float().reshape(-1, t)
        w[:, max(0, t - case["window"]):] = math.inf
        w[:, :case["prefill"]] = math.inf
        best = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :s["budgets"][b]].sort(-1).values
        keep.append(torch.nn.functional.pad(best.int(), (0, k - best.shape[1]), value=-1))
        scores.append(torch.nn.functional.pad(w, (0, longest - t), value=-math.inf))
    keep, scores = torch.cat(keep), torch.cat(scores)
    if kind == "pick":
        return keep, scores
    per = keep.view(len(s["lens"]), -1, hkv, k)
    got = {"keep": keep}
    for name in ("k", "v", "k_scales", "v_scales", "weights"):
        if s[name] is not None:
            x = s[name + "_before"].float() if s[name].dtype == torch.float8_e4m3fn else s[name + "_before"].clone()
            got[name] = x.view(case["layers"], -1, hkv, case["head_dim"]) if name in ("k", "v") else x.view(case["layers"], -1, hkv)
    for b in range(len(s["lens"])):
        slots, n = _exact_slots(s, b), s["budgets"][b]
        for layer in range(case["layers"]):
            rows = per[b, layer if per.shape[1] > 1 else 0, :, :n].long()
            for h in range(hkv):
                for name in [x for x in got if x != "keep"]:
                    got[name][layer, slots[:n], h] = got[name][layer, slots[rows[h]], h]
    return {name: x if name == "keep" else x.view(s[name].shape) for name, x in got.items()}
