"""What a decoding step does on the paged cache around attention, and the cases it is measured on.

Before attention the new tokens' queries and keys are normalised per head, rotated by their positions, and keys and values
written (quantised, in an fp8 cache) into their slots (``ops.write_paged``); cached rows come back as dense
tensors (``ops.read_paged``).  After it drafted tokens are verified against the target's logits (``ops.verify_drafts``)
and the accepted ones' rows moved one behind the other in every layer (``ops.accept_drafts``).

A case is one call: on one layer, or for ``accept_drafts`` on all layers of a model.  The plain form is the same in elementary torch
operations, in 32 bits, but for angles, weights of tokens and their sums, which are 64 bits: a token must not depend on
the order of a sum.  ``exact`` is the definition once more in 64 bits, verification one sequence at a time.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
# (query heads, KV heads, head dim) of the models the repository's configurations name
HEADS = {"qwen3_8b": (32, 8, 128), "qwen3_32b": (64, 8, 128), "qwen_7b": (28, 4, 128), "gpt_oss": (64, 8, 64),
         "dim256": (32, 8, 256)}
FP8_MOST = 448.0                 # the largest number of e4m3
LEAST_SCALE = 2.0 ** -126        # of a row, also of a row of zeros
EPS = 1e-6
THETA = 1e6


def _case(kind: str, model: str, seqs: int, **more) -> dict:
    case = {"kind": kind, "seqs": seqs, "lens_seed": 0}
    if kind != "verify":
        q, kv, d = HEADS[model]
        case.update(q_heads=q, kv_heads=kv, head_dim=d, block=16, dtype="bf16", row_scales=False, layers=1)
    if kind == "write":
        case.update(new=1, fewest=1, past=0, query="bf16", norm=True, axes=1, style="half", far=0)
    elif kind == "read":
        case.update(tokens=1024, shortest=1024, out="bf16")
    elif kind == "verify":
        case.update(vocab=32768, new=6, fewest=6, logits="bf16", draft_probs=False, tree=False, greedy=0)
    elif kind == "accept":
        case.update(past=200, new=16, fewest=16, most=5, layers=36, weights=False)
    case.update(more)
    if kind == "read" and "shortest" not in more:
        case["shortest"] = case["tokens"]
    if "new" in case and "fewest" not in more:
        case["fewest"] = case["new"]
    return case


def listed() -> list:
    return [
        # The smallest step: one new token of one request.
        _case("write", "qwen3_8b", 1, past=700, name="write_one_token"),
        # A decoding step of many requests far into long contexts, an fp8 cache with a scale per row.
        _case("write", "qwen3_32b", 64, past=500, dtype="fp8", row_scales=True, far=900000, name="write_64_fp8_far"),
        # A long prompt.
        _case("write", "qwen3_8b", 1, new=16384, name="write_prompt_16k"),
        # Prompts with images and video: positions on three axes, no norm, a scale per tensor, lengths of every size.
        _case("write", "qwen_7b", 6, new=4001, fewest=37, dtype="fp8", norm=False, axes=3, lens_seed=4, name="write_axes_6x4k"),
        # What a short request has cached, as dense rows.
        _case("read", "qwen3_8b", 1, tokens=2176, name="read_one_2176"),
        # Prompts out of an fp8 cache with a scale per row.
        _case("read", "qwen3_8b", 16, tokens=8192, shortest=3000, lens_seed=2, dtype="fp8", row_scales=True, name="read_16x8k_fp8"),
        # Five drafted tokens of one request, a small vocabulary.
        _case("verify", "", 1, draft_probs=True, name="verify_one_chain"),
        # Many requests with up to seven drafted tokens, some of them greedy, a large vocabulary.
        _case("verify", "", 48, vocab=131072, new=8, fewest=2, draft_probs=True, greedy=4, lens_seed=6, name="verify_48_chains"),
        # A tree of sixty drafted tokens, greedy.
        _case("verify", "", 1, vocab=131072, new=60, tree=True, greedy=1, name="verify_tree_60_greedy"),
        # Trees of requests that sample, an odd vocabulary, logits in 32 bits.
        _case("verify", "", 8, vocab=100003, new=32, fewest=9, tree=True, logits="fp32", lens_seed=7, name="verify_8_trees"),
        # The accepted path of one request's tree, every layer of a model.
        _case("accept", "qwen3_8b", 1, name="accept_one"),
        # Those of many requests, an fp8 cache with a scale per row and accumulated weights.
        _case("accept", "qwen3_8b", 32, new=32, fewest=6, most=7, dtype="fp8", row_scales=True, weights=True, lens_seed=8,
              name="accept_32_fp8"),
    ]


def _spread(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["write", "write", "write", "read", "verify", "verify", "verify", "accept"])
    more = {"lens_seed": rng.randrange(1 << 20)}
    if kind == "verify":
        vocab = _spread(rng, 1000, 140000)
        tree = rng.random() < 0.5
        new = _spread(rng, 1, 64) if tree else _spread(rng, 1, 12)
        seqs = max(1, min(_spread(rng, 1, 64), int(3.2e7 / (vocab * new))))
        new = max(1, min(new, int(3.2e7 / (vocab * seqs))))
        more.update(vocab=vocab, new=new, fewest=rng.choice([new, 1]), tree=tree, draft_probs=not tree and rng.random() < 0.7,
                    logits=rng.choice(["bf16", "bf16", "fp16", "fp32"]), greedy=rng.choice([0, 0, 1, 3]))
        return _case(kind, "", seqs, **more)
    model = rng.choice(sorted(HEADS))
    q, kv, d = HEADS[model]
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp8"])
    more.update(dtype=dtype, row_scales=dtype == "fp8" and rng.random() < 0.6, block=rng.choice([16, 16, 16, 32, 64, 8, 1, 24]))
    if kind == "write":
        prompt = rng.random() < 0.5
        seqs = _spread(rng, 1, 128)
        new = _spread(rng, 2, 16000) if prompt else _spread(rng, 1, 16)
        new = max(1, min(new, int(1e8 / (seqs * (q + 2 * kv) * d))))
        more.update(new=new, fewest=rng.choice([new, 1]), past=rng.choice([0, 0, rng.randrange(1, 600)]),
                    query=dtype if dtype != "fp8" else rng.choice(["bf16", "fp16"]), norm=rng.random() < 0.7,
                    axes=rng.choice([1, 1, 3]), style=rng.choice(["half", "half", "interleaved"]),
                    far=rng.choice([0, 0, rng.randrange(1, 1 << 20)]))
    elif kind == "read":
        tokens = _spread(rng, 30, 60000)
        seqs = max(1, min(_spread(rng, 1, 64), int(1.2e8 / (tokens * kv * d))))
        more.update(tokens=tokens, shortest=tokens if rng.random() < 0.5 else rng.randint(1, tokens),
                    out=rng.choice(["bf16", "fp16", "fp32"]) if dtype == "fp8" else rng.choice([dtype, dtype, "fp32"]))
    else:
        layers, new = _spread(rng, 1, 64), _spread(rng, 2, 64)
        past = rng.randrange(1, 300)
        seqs = max(1, min(_spread(rng, 1, 64), int(2.5e8 / (layers * kv * d * (past + new)))))
        more.update(layers=layers, new=new, fewest=rng.choice([new, 1]), past=past, most=min(_spread(rng, 2, 16), new),
                    weights=rng.random() < 0.5)
    return _case(kind, model, seqs, **more)


# ------------------------------------------------------------------------------- inputs
def _rows(case: dict) -> list:
    """New tokens (read: tokens) of every sequence, the most first."""
    rng = random.Random(case["lens_seed"])
    most, least = (case["tokens"], case["shortest"]) if case["kind"] == "read" else (case["new"], case["fewest"])
    return [most] + [rng.randint(least, most) for _ in range(case["seqs"] - 1)]


def _inv_freq(d: int):
    return (1.0 / (THETA ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)


def _prepare_cache(s, g) -> None:
    case, lens, bs = s["case"], s["lens"], s["case"]["block"]
    counts = [-(-t // bs) for t in lens]
    pool = sum(counts) + sum(counts) // 10 + 1
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    ends = [sum(counts[:i + 1]) for i in range(len(counts))]
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=DEV)
    for b, n in enumerate(counts):
        table[b, :n] = order[ends[b] - n:ends[b]]
    s.update(table=table, pool=pool, lens_dev=torch.tensor(lens, dtype=torch.int32, device=DEV))
    hkv, d, layers = case["kv_heads"], case["head_dim"], case["layers"]
    for side in ("k", "v"):
        s[side] = torch.empty(layers, pool, bs, hkv, d, dtype=DTYPES[case["dtype"]], device=DEV)
        s[side + "_scales"] = torch.empty(layers, pool * bs, hkv, device=DEV) if case["row_scales"] else None
        for layer in range(layers):
            x = torch.randn(pool, bs, hkv, d, generator=g, device=DEV)
            if case["row_scales"]:
                sc = x.abs().amax(-1, keepdim=True) / FP8_MOST
                s[side + "_scales"][layer] = sc.view(-1, hkv)
                x = x / sc
            s[side][layer] = (x.clamp(-FP8_MOST, FP8_MOST) if case["dtype"] == "fp8" else x).to(DTYPES[case["dtype"]])
    # a cache with one scale per tensor has those of its calibration
    s["k_scale"], s["v_scale"] = (0.05, 0.02) if case["dtype"] == "fp8" and not case["row_scales"] else (1.0, 1.0)


def _prepare_write(s, g, host) -> None:
    case, rows = s["case"], s["rows"]
    n, hq, hkv, d = sum(rows), case["q_heads"], case["kv_heads"], case["head_dim"]
    kind = DTYPES[case["query"]]
    # one product gives the three: q, k and v are views of its rows
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device=DEV)
    qkv[:, hq:hq + hkv] += 0.5 * torch.randn(1, hkv, d, generator=g, device=DEV)
    qkv = (1.5 * qkv).to(kind)
    s["q"], s["k_new"], s["v_new"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    s["q_norm"], s["k_norm"] = ((1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(kind) if case["norm"] else None for _ in range(2))
    s["inv_freq"] = _inv_freq(d)
    first = [case["past"] + (host.randrange(case["far"]) if case["far"] else 0) for _ in rows]
    line = torch.cat([torch.arange(a, a + m) for a, m in zip(first, rows)])
    s["freq_axes"] = None
    if case["axes"] == 1:
        s["positions"] = line.to(device=DEV, dtype=torch.int64)
    else:
        # frames of 12 x 20 patches between pieces of text: time advances with the frame, height and width inside it
        inside = torch.arange(n) % 240
        s["positions"] = torch.stack([line // 240, line // 240 + inside // 20, line // 240 + inside % 20]).to(device=DEV, dtype=torch.int64)
        f = d // 2
        t, h = f // 4, f // 4 + (f - f // 4 + 1) // 2
        axes = torch.zeros(f, dtype=torch.int32)
        axes[t:h], axes[h:] = 1, 2
        s["freq_axes"] = axes.to(DEV)


def _tree(rows: list, tree: bool, host) -> list:
    """Parent of every row, counted from its sequence's first; that one, the last token decided, hangs on the cache."""
    return [(host.randint(max(0, i - 6), i - 1) if tree else i - 1) if i else -1 for n in rows for i in range(n)]


def _prepare_verify(s, g, host) -> None:
    case, rows, parents = s["case"], s["rows"], s["parents_host"]
    n, v = sum(rows), case["vocab"]
    greedy = [case["greedy"] and b % case["greedy"] == 0 for b in range(len(rows))]
    s["temperatures"] = torch.tensor([0.0 if x else host.choice([0.6, 0.8, 1.0]) for x in greedy], device=DEV)
    # a peaked distribution: a few tokens hold most of it
    logits = torch.randn(n, v, generator=g, device=DEV) * 1.5
    top = torch.randint(0, v, (n, 24), generator=g, device=DEV)
    logits.scatter_add_(1, top, 6 + 4 * torch.rand(n, 24, generator=g, device=DEV))
    s["logits"] = logits.to(DTYPES[case["logits"]])
    temp = torch.repeat_interleave(s["temperatures"], torch.tensor(rows, device=DEV))
    # the row whose logits say what may stand in a row
    first = [i for i, r in zip(_starts(rows), rows) for _ in range(r)]
    at = torch.tensor([i + max(p, 0) for i, p in zip(first, parents)], device=DEV)
    s["draft_probs"] = None
    noisy = s["logits"].float()[at] + 0.4 * torch.randn(n, v, generator=g, device=DEV)
    if case["draft_probs"]:
        noisy /= temp.clamp(min=0.3)[:, None]
        s["draft_probs"] = torch.softmax(noisy, -1)
        u = torch.rand(n, 1, generator=g, device=DEV, dtype=torch.float64)
        s["tokens"] = torch.searchsorted(s["draft_probs"].double().cumsum(-1), u).clamp(max=v - 1).view(-1).to(torch.int32)
    else:
        # the r-th child of a row holds the draft's r-th best token
        rank, seen = [], {}
        for i, p in zip(at.tolist(), parents):
            rank.append(seen.get(i, 0))
            seen[i] = rank[-1] + (p >= 0)
        best = torch.topk(noisy, min(v, 1 + max(rank)), -1).indices
        s["tokens"] = best.gather(1, torch.tensor(rank, device=DEV)[:, None]).view(-1).to(torch.int32)
    s["uniforms"] = torch.rand(n, 2, generator=g, device=DEV)
    del logits, noisy


def _prepare_accept(s, g, host) -> None:
    case, rows = s["case"], s["rows"]
    hkv = case["kv_heads"]
    counts = [1 + host.randrange(min(case["most"], n)) for n in rows]
    paths = [[0] + sorted(host.sample(range(1, n), c - 1)) for n, c in zip(rows, counts)]
    width = max(rows)
    s["path"] = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32, device=DEV)
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    s["weights"] = (torch.rand(case["layers"], s["pool"], case["block"], hkv, generator=g, device=DEV) * 8 if case["weights"] else None)
    # what a call overwrites, so that every pass finds the rows that a step left
    table, bs = s["table"].tolist(), case["block"]
    slots = [table[b][t // bs] * bs + t % bs for b, (total, n, c) in enumerate(zip(s["lens"], rows, counts))
             for t in range(total - n + 1, total - n + c)]
    s["dirty"] = torch.tensor(slots, dtype=torch.int64, device=DEV)
    s["before"] = {name: _slots_of(s, name).index_select(1, s["dirty"]) for name in _moved(s)}


def _moved(s) -> list:
    return [name for name in ("k", "v", "k_scales", "v_scales", "weights") if s.get(name) is not None]


def _slots_of(s, name):
    """[layers, slots, ...] of a tensor of the cache or beside it (an fp8 cache by its bytes)."""
    x = s[name].view(torch.uint8) if s[name].dtype == torch.float8_e4m3fn else s[name]
    return x.view(s["case"]["layers"], s["pool"] * s["case"]["block"], s["case"]["kv_heads"], -1)


def _starts(rows: list) -> list:
    return [sum(rows[:i]) for i in range(len(rows))]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    rows = _rows(case)
    s = {"case": case, "rows": rows, "starts": torch.tensor(_starts(rows) + [sum(rows)], dtype=torch.int32, device=DEV)}
    if case["kind"] != "verify":
        s["lens"] = [n + case.get("past", 0) for n in rows]
        _prepare_cache(s, g)
    if case["kind"] == "write":
        _prepare_write(s, g, host)
    elif case["kind"] == "verify":
        s["parents_host"] = _tree(rows, case["tree"], host)
        s["parents"] = torch.tensor(s["parents_host"], dtype=torch.int32, device=DEV)
        _prepare_verify(s, g, host)
    elif case["kind"] == "accept":
        _prepare_accept(s, g, host)
    return s


# --------------------------------------------------------------------------- plain forms
def _row_places(s):
    """Sequence and slot of every row: the rows of a sequence are its last tokens."""
    starts, bs = s["starts"].long(), s["case"]["block"]
    row = torch.arange(sum(s["rows"]), device=DEV)
    seq = torch.searchsorted(starts, row, right=True) - 1
    t = s["lens_dev"].long()[seq] - starts[seq + 1] + row
    return seq, s["table"].long()[seq, t // bs] * bs + t % bs


def _plain_norm(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain_rotate(x, cos, sin, style):
    if style == "half":
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _plain_write(s):
    case, d = s["case"], s["case"]["head_dim"]
    pos = s["positions"][None] if case["axes"] == 1 else s["positions"]
    axes = torch.zeros(d // 2, dtype=torch.long, device=DEV) if case["axes"] == 1 else s["freq_axes"].long()
    angle = pos[axes].t().double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _plain_rotate(_plain_norm(s["q"], s["q_norm"]), cos, sin, case["style"]).to(s["q"].dtype)
    k = _plain_rotate(_plain_norm(s["k_new"], s["k_norm"]), cos, sin, case["style"])
    _, slot = _row_places(s)
    _plain_store(s, "k", slot, k)
    _plain_store(s, "v", slot, s["v_new"].float())
    return q


def _plain_store(s, side, slot, x):
    case = s["case"]
    cache = _slots_of(s, side)[0]
    if case["dtype"] != "fp8":
        cache.index_copy_(0, slot, x.to(cache.dtype))
        return
    scale = s[side + "_scale"]
    if case["row_scales"]:
        scale = (x.abs().amax(-1, keepdim=True) / FP8_MOST).clamp(min=LEAST_SCALE)
        s[side + "_scales"][0].index_copy_(0, slot, scale.squeeze(-1))
    cache.index_copy_(0, slot, (x / scale).clamp(-FP8_MOST, FP8_MOST).to(torch.float8_e4m3fn).view(torch.uint8))


def _plain_read(s):
    _, slot = _row_places(s)
    got = []
    for side in ("k", "v"):
        x = _slots_of(s, side)[0][slot]
        x = (x.view(torch.float8_e4m3fn) if s["case"]["dtype"] == "fp8" else x).float()
        if s[side + "_scales"] is not None:
            x = x * s[side + "_scales"][0][slot].unsqueeze(-1)
        got.append((x * s[side + "_scale"]).to(DTYPES[s["case"]["out"]]))
    return tuple(got)


def _plain_draws(w, u):
    """The least token with a running sum above u of the whole, per row."""
    running = w.cumsum(-1)
    return (running <= (u * running[:, -1])[:, None]).sum(-1).clamp(max=w.shape[1] - 1)


def _plain_verify(s):
    """Accepted rows [B, most rows] (-1 behind the last), how many, and the token that follows them."""
    case, dev = s["case"], s["logits"].device
    starts, n, v = s["starts"].long(), max(s["rows"]), case["vocab"]
    row = torch.arange(s["logits"].shape[0], device=dev)
    seq = torch.searchsorted(starts, row, right=True) - 1
    temp = s["temperatures"].double()[seq]
    x = s["logits"].double()
    best = x.amax(-1, keepdim=True)
    top = torch.where(x == best, torch.arange(v, device=dev), v).amin(-1)
    w = torch.exp((x - best) / torch.where(temp > 0, temp, torch.ones_like(temp))[:, None])
    total = w.sum(-1)
    u = s["uniforms"].double()
    i = torch.arange(n, device=dev)
    have = (starts[1:] - starts[:-1])[:, None]
    at = (starts[:-1, None] + i).clamp(max=row.numel() - 1)                    # [B, n]
    parent = s["parents"].long()[at]
    up = (starts[:-1, None] + parent.clamp(min=0))                             # the parent's row
    token = s["tokens"].long()[at]
    if case["draft_probs"]:
        q = s["draft_probs"].double()
        fits = u[at, 0] * q[at, token] * total[up] < w[up, token]
        matches = torch.where(temp[at] > 0, fits, token == top[up])
    else:
        picked = torch.where(temp > 0, _plain_draws(w, u[:, 1]), top)
        matches = token == picked[up]
        # of siblings that hold the same token the first
        same = (parent[:, :, None] == parent[:, None]) & (token[:, :, None] == token[:, None]) & (i[:, None] > i)
        matches &= ~same.any(-1)
    matches = matches & (i < have) & (parent >= 0) | (i == 0)
    # a row is accepted if every row on its way to the first matches: the reach of "is my matching parent's child"
    step = ((parent[:, :, None] == i) & (i < have)[..., None] & matches[..., None] & (i[:, None] > 0)).float()
    accepted = torch.linalg.matrix_power(step + torch.eye(n, device=dev), n)[:, :, 0] > 0
    accepted = accepted & (i < have)
    count = accepted.sum(-1)
    path = torch.sort(torch.where(accepted, i, n), -1).values
    last = path.gather(1, (count[:, None] - 1).clamp(min=0)).view(-1).clamp(max=n - 1)
    at_last = starts[:-1] + last
    if case["draft_probs"]:
        rejected = last + 1 < have[:, 0]
        nxt = (at_last + 1).clamp(max=row.numel() - 1)
        p = w[at_last]
        rest = (p / total[at_last, None] - q[nxt]).clamp(min=0)
        p = torch.where((rejected & (rest.sum(-1) > 0))[:, None], rest, p)
        token = torch.where(temp[at_last] > 0, _plain_draws(p, u[at_last, 1]), top[at_last])
    else:
        token = picked[at_last]
    return torch.where(path < n, path, torch.full_like(path, -1)).int(), count.int(), token.int()


def _plain_accept(s):
    starts, bs = s["starts"].long(), s["case"]["block"]
    n = s["path"].shape[1]
    j = torch.arange(n, device=DEV)
    used = j < s["counts"][:, None]
    first = s["lens_dev"].long() - (starts[1:] - starts[:-1])
    # behind a path its first row onto itself
    to = first[:, None] + torch.where(used, j, torch.zeros_like(j))
    of = first[:, None] + torch.where(used, s["path"].long(), 0)
    seq = torch.arange(first.numel(), device=DEV)[:, None]
    table = s["table"].long()
    to, of = (table[seq, t // bs] * bs + t % bs for t in (to, of))
    to, of = to.flatten(), of.flatten()
    moved = [_slots_of(s, name) for name in _moved(s)]
    [x.index_copy_(1, to, x.index_select(1, of)) for x in moved]
    return (first + s["counts"]).int()


# --------------------------------------------------------------------------------- calls
def _handles(s):
    """The description of the cache and of the batch that a program keeps over its calls."""
    if "kv" not in s:
        from triattention_amd import ops
        layers = range(s["case"]["layers"])
        per_layer = [None if s[name] is None else [s[name][layer] for layer in layers] for name in ("k", "v", "k_scales", "v_scales")]
        s["kv"] = ops.PagedKV(per_layer[0], per_layer[1], s["case"].get("style", "half"), per_layer[2], per_layer[3])
        s["batch"] = ops.StepBatch(torch.device(DEV), s["lens"], block_tables=s["table"])
    return s["kv"], s["batch"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "accept":
        [_slots_of(s, name).index_copy_(1, s["dirty"], x) for name, x in s["before"].items()]
    if kind == "write":
        if own:
            from triattention_amd import ops
            kv, batch = _handles(s)
            out = ops.write_paged(kv, batch, s["q"], s["k_new"], s["v_new"], s["positions"], s["inv_freq"], row_starts=s["starts"],
                                  freq_axes=s["freq_axes"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, k_scale=s["k_scale"],
                                  v_scale=s["v_scale"])
        else:
            out = _plain_write(s)
        got = {"out": out, "k": s["k"], "v": s["v"]}
        if case["row_scales"]:
            got.update(k_scales=s["k_scales"], v_scales=s["v_scales"])
        return got
    if kind == "read":
        if own:
            from triattention_amd import ops
            kv, batch = _handles(s)
            return ops.read_paged(kv, batch, s["starts"], sum(s["rows"]), dtype=DTYPES[case["out"]], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return _plain_read(s)
    if kind == "verify":
        if own:
            from triattention_amd import ops
            return ops.verify_drafts(s["logits"], s["tokens"], s["starts"], s["uniforms"], max_rows=max(s["rows"]),
                                     parents=s["parents"] if case["tree"] else None, draft_probs=s["draft_probs"],
                                     temperatures=s["temperatures"])
        return _plain_verify(s)
    if own:
        from triattention_amd import ops
        kv, batch = _handles(s)
        lens = ops.accept_drafts(kv, batch, s["starts"], s["path"], s["counts"], weights=s["weights"])
    else:
        lens = _plain_accept(s)
    return {"lens": lens, **{name: s[name] for name in _moved(s)}}


# ---------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    rows = _rows(case)
    n = sum(rows)
    if case["kind"] == "verify":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["logits"]]
        sampled = sum(1 for b in range(len(rows)) if not (case["greedy"] and b % case["greedy"] == 0))
        drafted = 4 * case["vocab"] * sampled if case["draft_probs"] and case["new"] > 1 else 0
        # a subtraction, a product, an exponential (eight more) and a sum for every logit
        return {"bytes": n * case["vocab"] * size + drafted + n * 24, "flops": 11 * n * case["vocab"]}
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    row = hkv * (d * (1 if case["dtype"] == "fp8" else 2) + (4 if case["row_scales"] else 0))
    if case["kind"] == "write":
        return {"bytes": n * ((2 * hq + 2 * hkv) * d * 2 + 2 * row + 8 * case["axes"]), "flops": n * (15 * (hq + hkv) + 4 * hkv) * d}
    if case["kind"] == "read":
        out = {"bf16": 2, "fp16": 2, "fp32": 4}[case["out"]]
        return {"bytes": n * (2 * row + 2 * hkv * d * out), "flops": 2 * n * hkv * d}
    moved = sum((1 + min(case["most"], r)) / 2 - 1 for r in rows) * case["layers"] * (2 * row + (4 * hkv if case["weights"] else 0))
    # the rows a pass restores are read and written too
    return {"bytes": 4 * moved + 16 * sum(rows), "flops": sum(rows)}


# --------------------------------------------------------------------------------- exact
def _exact_store(s, side, x, got):
    """The cache's layer in 64 bits with x [rows, H, D] in the slots of the rows: codes before they are rounded."""
    case, bs = s["case"], s["case"]["block"]
    held = s[side].double().view(-1, case["kv_heads"], case["head_dim"])
    scales = None if s[side + "_scales"] is None else s[side + "_scales"].double().view(-1, case["kv_heads"])
    at = 0
    for b, n in enumerate(s["rows"]):
        t = torch.arange(s["lens"][b] - n, s["lens"][b], device=DEV)
        slot = s["table"][b].long()[t // bs] * bs + t % bs
        part = x[at:at + n]
        if case["dtype"] == "fp8":
            sc = part.abs().amax(-1).div(FP8_MOST).clamp(min=LEAST_SCALE) if case["row_scales"] else torch.full(part.shape[:2], s[side + "_scale"],
                                                                                                    dtype=torch.float64, device=DEV)
            part = (part / sc[..., None]).clamp(-FP8_MOST, FP8_MOST)
            if scales is not None:
                scales[slot] = sc
        held[slot] = part
        at += n
    got[side] = held.view(s[side].shape)
    if scales is not None:
        got[side + "_scales"] = scales.view(s[side + "_scales"].shape)


def _exact_turn(x, w, s):
    """Norm and rotation of x [rows, heads, D] as complex numbers in 64 bits."""
    case, f = s["case"], s["case"]["head_dim"] // 2
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    pos = s["positions"].double().view(-1, x.shape[0])
    axis = [0] * f if case["axes"] == 1 else s["freq_axes"].tolist()
    angle = torch.stack([pos[axis[k]] * float(s["inv_freq"][k]) for k in range(f)], -1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if case["style"] == "half":
        z = torch.complex(x[..., :f], x[..., f:]) * turn
        return torch.cat([z.real, z.imag], -1)
    return torch.view_as_real(torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) * turn).flatten(-2)


def _exact_draw(p, u):
    total = float(p.sum())
    above = (torch.cumsum(p, 0) > u * total).nonzero()
    return int(above[0]) if above.numel() else int((p > 0).nonzero()[-1])


def _exact_sequence(s, b):
    """The walk of one sequence, row by row."""
    case, at, n = s["case"], int(s["starts"][b]), s["rows"][b]
    temp, line, here = float(s["temperatures"][b]), [0], 0
    parents = s["parents_host"][at:at + n]
    while True:
        x = s["logits"][at + here].double()
        u = [float(y) for y in s["uniforms"][at + here]]
        p = torch.softmax(x / temp, -1) if temp > 0 else None
        children = [j for j in range(here + 1, n) if parents[j] == here]
        nxt, picked = None, int((x == x.max()).nonzero()[0]) if p is None else None
        if p is not None and case["draft_probs"]:
            if children:
                j = children[0]
                tok, q = int(s["tokens"][at + j]), s["draft_probs"][at + j].double()
                if float(s["uniforms"][at + j, 0]) * float(q[tok]) < float(p[tok]):
                    nxt = j
                else:
                    rest = (p - q).clamp(min=0)
                    picked = _exact_draw(rest if float(rest.sum()) > 0 else p, u[1])
            else:
                picked = _exact_draw(p, u[1])
        else:
            picked = picked if p is None else _exact_draw(p, u[1])
            nxt = next((j for j in children if int(s["tokens"][at + j]) == picked), None)
        if nxt is None:
            return line, picked
        line.append(nxt)
        here = nxt


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "write":
        got = {"out": _exact_turn(s["q"], s["q_norm"], s)}
        _exact_store(s, "k", _exact_turn(s["k_new"], s["k_norm"], s), got)
        _exact_store(s, "v", s["v_new"].double(), got)
        return got
    if kind == "read":
        got = []
        for side in ("k", "v"):
            parts = []
            for b, t in enumerate(s["lens"]):
                pages = s["table"][b, :-(-t // case["block"])].long()
                x = (s[side][0].view(torch.uint8) if case["dtype"] == "fp8" else s[side][0])[pages]
                x = (x.view(torch.float8_e4m3fn) if case["dtype"] == "fp8" else x).double().flatten(0, 1)[:t] * s[side + "_scale"]
                if s[side + "_scales"] is not None:
                    x = x * s[side + "_scales"][0].view(s["pool"], case["block"], -1)[pages].flatten(0, 1)[:t].double()[..., None]
                parts.append(x)
            got.append(torch.cat(parts))
        return tuple(got)
    if kind == "verify":
        walks = [_exact_sequence(s, b) for b in range(len(s["rows"]))]
        width = max(s["rows"])
        return (torch.tensor([line + [-1] * (width - len(line)) for line, _ in walks], dtype=torch.int32),
                torch.tensor([len(line) for line, _ in walks], dtype=torch.int32), torch.tensor([t for _, t in walks], dtype=torch.int32))
    got = {name: (s[name].float() if s[name].dtype == torch.float8_e4m3fn else s[name]).double() for name in _moved(s)}
    table, bs = s["table"].tolist(), case["block"]
    lens = []
    for b, (total, n) in enumerate(zip(s["lens"], s["rows"])):
        rows = s["path"][b, :int(s["counts"][b])].tolist()
        lens.append(total - n + len(rows))
        slot = [table[b][t // bs] * bs + t % bs for t in range(total - n, total)]
        for x in got.values():
            flat = x.view(case["layers"], s["pool"] * bs, -1)
            flat[:, slot[:len(rows)]] = flat[:, [slot[r] for r in rows]]
    return {"lens": torch.tensor(lens, dtype=torch.int32), **got}
