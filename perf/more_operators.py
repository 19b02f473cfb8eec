"""The paged key-value cache beyond one token of one sequence, as cases that can be timed and
compared: prompts whose new tokens attend over it, scores that are capped, leaned on by distance or
masked by document and prefix, batches that share a long prefix, and eviction by accumulated weight.

A case is one pass through an operator, called as a serving program calls it: the cache, its tables
and the lengths are kept between passes, nothing synchronises.  Queries, keys and values are normal,
in BF16 or, keys and values, 8-bit codes with a scale per row.  Lengths of a batch are spread between
a quarter of the longest and the longest.

Kinds:
  prompt  prompt_attention of up to ``new`` tokens a sequence that follow up to ``past`` ones
  token   paged_attention of one token a sequence with capped scores or a bias by distance
  shared  shared_prefix_attention of ``sequences`` tokens in ``groups`` that share a prefix each
  weigh   attention_weights: what each token of the cache got of the new token's attention
  evict   cache_evict down to ``keep`` tokens a head, into other pages; of codes, with the sequences
          read back as values

``own`` says which form runs: the plain one, in elementary operations in 32 bits, or the library's.
"""

import math

import torch

own = False


def listed():
    heads = dict(heads=64, kv_heads=8, dim=128)
    prompt = dict(kind="prompt", window=0, cap=0.0, slopes=False, prefix=False, documents=False)
    token = dict(kind="token", window=0, cap=0.0, slopes=False)
    return [
        # A short question of which a first part is seen both ways, with a bias by distance: latency.
        dict(prompt, name="prompt_short", batch=1, new=37, past=0, heads=12, kv_heads=4, dim=64, page=16, bits=16,
             slopes=True, prefix=True),
        # A ragged batch of prompts in which documents are packed one behind another.
        dict(prompt, name="prompt_documents", batch=9, new=2048, past=0, page=64, bits=16, documents=True, **heads),
        # One long prompt (the largest).
        dict(prompt, name="prompt_long", batch=1, new=16384, past=0, page=64, bits=16, **heads),
        # Chunks of prompts behind a long past in 8 bits, wide heads, capped scores.
        dict(prompt, name="prompt_chunk", batch=4, new=1024, past=30000, heads=16, kv_heads=8, dim=256, page=32, bits=8,
             cap=50.0),
        # A batch's new tokens with capped scores and wide heads.
        dict(token, name="token_capped", batch=16, length=4096, heads=16, kv_heads=8, dim=256, page=64, bits=16, cap=50.0,
             empty=False),
        # The same with a bias by distance: narrow heads of their own, odd pages, an empty sequence, codes.
        dict(token, name="token_distance", batch=37, length=3001, heads=12, kv_heads=12, dim=64, page=24, bits=8,
             slopes=True, empty=True),
        # Many answers to one long document.
        dict(token, name="shared_one", **dict(heads, kind="shared"), groups=1, sequences=64, prefix=32768, length=512,
             page=64, bits=16),
        # Several system prompts with a few users each, in 8 bits.
        dict(token, name="shared_groups", **dict(kind="shared", heads=28, kv_heads=4, dim=128), groups=5, sequences=37,
             prefix=6000, length=700, page=16, bits=8),
        # Weights of a ragged batch.
        dict(token, name="weigh_batch", **dict(heads, kind="weigh"), batch=64, length=8192, page=64, bits=16, empty=False),
        # Weights of one very long sequence in 8 bits.
        dict(token, name="weigh_long", **dict(heads, kind="weigh"), batch=1, length=131072, page=64, bits=8, empty=False),
        # A few short conversations cut to a small budget, in 8 bits.
        dict(name="evict_small", kind="evict", batch=3, length=700, keep=256, first=4, recent=32, kv_heads=4, dim=128,
             page=16, bits=8),
        # Long sequences cut to a quarter.
        dict(name="evict_long", kind="evict", batch=16, length=16384, keep=4096, first=4, recent=256, kv_heads=8, dim=128,
             page=64, bits=16),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of these ranges; no larger than the largest listed ones."""
    kind = rng.choice(["prompt", "prompt", "prompt", "token", "shared", "shared", "weigh", "evict"])
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16])
    page, bits = rng.choice([8, 16, 16, 24, 32, 64, 100, 128]), rng.choice([8, 16])
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, bits=bits,
                window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                slopes=rng.random() < 0.3)
    if kind == "prompt":
        batch, past = _log_int(rng, 1, 32), rng.choice([0, 0, _log_int(rng, 1, 30000)])
        tokens = 16384 * 64 * 128 // (heads * dim) // batch
        new = max(1, min(_log_int(rng, 1, 8192), tokens, 8192 * 8192 * 64 * 128 // ((past + 4096) * heads * dim * batch)))
        case.update(batch=batch, new=new, past=past, prefix=rng.random() < 0.3, documents=rng.random() < 0.3)
        return case
    if kind == "token" or kind == "weigh":
        batch = _log_int(rng, 1, 128)
        most = 48 * 8192 * 8 * 128 // (batch * kv_heads * dim)
        case.update(batch=batch, length=max(1, min(_log_int(rng, 1, 131072), most)), empty=batch > 1 and rng.random() < 0.3)
        return case
    if kind == "shared":
        sequences = _log_int(rng, 1, 128)
        groups = min(sequences, _log_int(rng, 1, 8))
        most = 2**31 // (groups * kv_heads * dim * 64)
        prefix = max(1, min(_log_int(rng, 1, 32768), most, 64 * 64 * 128 * 32768 // (sequences * heads * dim)))
        case.update(groups=groups, sequences=sequences, prefix=prefix, length=_log_int(rng, 1, 700))
        return case
    batch = _log_int(rng, 1, 32)
    length = max(2, min(_log_int(rng, 2, 65536), 16 * 16384 * 8 * 128 // (batch * kv_heads * dim)))
    keep = rng.randint(1, max(1, length // 2))
    first = rng.randint(0, min(4, keep))
    return dict(kind=kind, batch=batch, length=length, keep=keep, first=first, recent=rng.randint(0, min(64, keep - first)),
                kv_heads=kv_heads, dim=dim, page=page, bits=bits)


# --------------------------------------------------------------------- inputs --

def _spread(count, most):
    """`count` lengths up to `most`, the first of them that, the others from a quarter of it on."""
    low = max(1, most // 4)
    return [most] + [low + int((most - low + 1) * (i * 0.6180339887498949 % 1)) for i in range(1, count)]


def _extents(case):
    """Each sequence's tokens in the cache and, of a prompt, how many of them are new."""
    if case["kind"] == "prompt":
        new = _spread(case["batch"], case["new"])
        past = _spread(case["batch"], case["past"]) if case["past"] else [0] * case["batch"]
        return [n + p for n, p in zip(new, past)], new
    count = case["sequences"] if case["kind"] == "shared" else case["batch"]
    lengths = _spread(count, case["length"])
    if case.get("empty"):
        lengths[-1] = 0
    return lengths, [1] * count


def _groups(case):
    """Of sequences that share prefixes: where each group's sequences begin, with the end, and the prefixes' lengths."""
    weights = [1 + i % 3 for i in range(case["groups"])]
    spare, offsets = case["sequences"] - case["groups"], [0]
    for i in range(case["groups"]):
        offsets.append(offsets[-1] + 1 + spare * sum(weights[: i + 1]) // sum(weights) - spare * sum(weights[:i]) // sum(weights))
    return offsets, _spread(case["groups"], case["prefix"])


def _masks(case):
    """Of a prompt's new tokens: first position of each one's document, and of each sequence the tokens seen both ways."""
    lengths, new = _extents(case)
    starts, prefixes = [], []
    for n, length in zip(new, lengths):
        document = 1 + length // 5
        starts.append([(length - n + i) // document * document if case["documents"] else 0 for i in range(n)])
        prefixes.append(1 + length // 3 if case["prefix"] else 0)
    return starts, prefixes


def _normal(shape, g):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(torch.bfloat16)


def _cache(pages, case, g):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    made = {}
    for name in ("k", "v"):
        x = _normal(shape, g)
        if case["bits"] == 8:
            x = x.float()
            scale = x.abs().amax(dim=-1) / 127
            x = (torch.round(x / torch.where(scale > 0, scale, 1.0)[..., None]) + 128).to(torch.uint8)
            made[name + "_scale"] = scale
        made[name] = x
    return made


def _tables(counts, g):
    """Tables of pages, in no order and none of them twice, one for each list of page counts: int32
    [sequences, pages of the longest], -1 behind a sequence's last; and how many pages there are."""
    total = max(1, sum(sum(used) for used in counts))
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    made, done = [], 0
    for used in counts:
        at = torch.arange(max(max(used), 1), device="cuda")[None, :]
        count = torch.tensor(used, device="cuda")[:, None]
        first = done + torch.tensor([0] + used[:-1], device="cuda").cumsum(0)[:, None]
        made.append(torch.where(at < count, order[(first + at).clamp(max=total - 1)], -1).to(torch.int32).contiguous())
        done += sum(used)
    return made, total


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state, kind, page = dict(case), case["kind"], case["page"]
    lengths, new = _extents(case)
    counts = [[-(-n // page) for n in lengths]]
    if kind == "shared":
        offsets, prefixes = _groups(case)
        counts.append([-(-n // page) for n in prefixes])
        state["group_offsets"], state["prefix_lengths"] = _int32(offsets), _int32(prefixes)
    if kind == "evict":
        counts.append([-(-min(n, case["keep"]) // page) for n in lengths])
    (state["tables"], *other), pages = _tables(counts, g)
    if other:
        state["new_tables" if kind == "evict" else "prefix_tables"] = other[0]
    state["lengths"] = _int32(lengths)
    state.update(_cache(pages, case, g))
    if own:  # the handle of the cache
        from chord_b200 import KVCache

        state["cache"] = KVCache(state["k"], state["v"], state.get("k_scale"), state.get("v_scale"))
    if kind == "evict":
        # a few tokens have most of the weight, many none
        shape = (case["batch"], case["kv_heads"], state["tables"].shape[1] * page)
        weights = torch.rand(shape, device="cuda", generator=g).pow_(6).mul_(50)
        weights = torch.where(torch.rand(shape, device="cuda", generator=g) < 0.2, 0.0, weights)
        behind = torch.arange(shape[2], device="cuda") >= state["lengths"][:, None, None]
        state["weights"] = weights.masked_fill_(behind, 0.0)
        kept = [min(n, case["keep"]) for n in lengths]
        state["offsets"] = _int32([0] + torch.tensor(kept).cumsum(0).tolist())
        state["kept_rows"] = sum(kept)
        return state
    heads = case["heads"]
    rows = sum(new)
    state["q"] = _normal((rows, heads, case["dim"]), g).mul_(1.5)
    state["slope_values"] = None
    if case["slopes"]:
        state["slope_values"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
    state["lse"] = torch.empty((rows, heads), dtype=torch.float32, device="cuda")
    if kind == "prompt":
        state["offsets"] = _int32([0] + torch.tensor(new).cumsum(0).tolist())
        starts, prefixes = _masks(case)
        state["starts"] = _int32([s for of in starts for s in of]) if case["documents"] else None
        state["prefixes"] = _int32(prefixes) if case["prefix"] else None
    if kind == "weigh":  # the sums of the attention that went before
        for b, (length, scores) in enumerate(_token_scores(state)):
            state["lse"][b] = torch.logsumexp(scores, dim=2).reshape(heads) if length else -math.inf
    return state


# ---------------------------------------------------------------- plain forms --

def _gather(s, name, pages, count):
    """The first `count` rows of some pages, in 32 bits: [kv_heads, count, dim]."""
    pages = pages[: -(-count // s["page"])].long()
    x = s[name][pages].float()
    if s["bits"] == 8:
        x = (x - 128) * s[name + "_scale"][pages][..., None]
    return x.transpose(0, 1).reshape(s["kv_heads"], -1, s["dim"])[:, :count]


def _shape_scores(s, scores, distance, slopes):
    """Scores capped, and leaned on by distance."""
    if s["cap"]:
        scores = torch.tanh(scores / s["cap"]) * s["cap"]
    if slopes is not None:
        scores = scores - slopes * distance.abs().float()
    return scores


def _plain_attend(s, q, keys, values, position, low, high):
    """Rows q [rows, heads, dim] over keys and values [kv_heads, tokens, dim]: row r, at position[r], sees
    tokens low[r] to high[r].  In 32 bits: out [rows, heads, dim], lse [rows, heads]."""
    kv_heads, tokens, dim = keys.shape
    group = s["heads"] // kv_heads
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    at = torch.arange(tokens, device=q.device)
    step = max(1, 2**28 // (s["heads"] * max(tokens, 1)))
    slopes = s["slope_values"]
    if slopes is not None:
        slopes = slopes.view(kv_heads, 1, group, 1)
    for r in range(0, q.shape[0], step):
        rows = slice(r, min(r + step, q.shape[0]))
        n = rows.stop - rows.start
        x = q[rows].float().view(n, kv_heads, group, dim).transpose(0, 1).reshape(kv_heads, n * group, dim)
        scores = torch.matmul(x, keys.transpose(1, 2)).mul_(dim**-0.5).view(kv_heads, n, group, tokens)
        scores = _shape_scores(s, scores, (at - position[rows, None]).view(1, n, 1, tokens), slopes)
        seen = (at >= low[rows, None]) & (at < high[rows, None])
        scores = scores.masked_fill(~seen.view(1, n, 1, tokens), -math.inf)
        top = scores.amax(dim=-1, keepdim=True) if tokens else scores.new_full((kv_heads, n, group, 1), -math.inf)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp_(scores.sub_(top))
        total = p.sum(dim=-1, keepdim=True)
        y = torch.matmul(p.view(kv_heads, n * group, tokens), values).view(kv_heads, n, group, dim)
        y = y / torch.where(total > 0, total, 1.0)
        out[rows] = y.transpose(0, 1).reshape(n, s["heads"], dim)
        lse[rows] = (top + torch.log(total)).transpose(0, 1).reshape(n, s["heads"])
    return out, lse


def _plain_prompt(s):
    lengths, new = _extents(s)
    out, lse, done = [], [], 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        position = torch.arange(length - n, length, device=s["q"].device)
        low, high = torch.zeros_like(position), position + 1
        if s["window"]:
            low = (high - s["window"]).clamp(min=0)
        if s["starts"] is not None:
            low = torch.maximum(low, s["starts"][done:done + n].long())
        if s["prefixes"] is not None:
            high = torch.maximum(high, s["prefixes"][b].long().clamp(max=length))
        keys, values = (_gather(s, name, s["tables"][b], length) for name in ("k", "v"))
        one = _plain_attend(s, s["q"][done:done + n], keys, values, position, low, high)
        out.append(one[0].to(torch.bfloat16))
        lse.append(one[1])
        done += n
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _plain_tokens(s):
    """One token a sequence, with or without a prefix that its group shares."""
    lengths, _ = _extents(s)
    shared = s["kind"] == "shared"
    offsets, prefixes = _groups(s) if shared else (None, None)
    out, lse, group, before = [], [], -1, 0
    for b, length in enumerate(lengths):
        if shared and b == offsets[group + 1]:
            group += 1
            before = prefixes[group]
            prefix = [_gather(s, name, s["prefix_tables"][group], before) for name in ("k", "v")]
        keys, values = (_gather(s, name, s["tables"][b], length) for name in ("k", "v"))
        if shared:
            keys, values = (torch.cat(parts, dim=1) for parts in zip(prefix, (keys, values)))
        high = torch.tensor([before + length], device=keys.device)
        low = (high - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(high)
        one = _plain_attend(s, s["q"][b:b + 1], keys, values, high - 1, low, high)
        out.append(one[0].to(torch.bfloat16))
        lse.append(one[1])
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _token_scores(s):
    """Of each sequence its length and its new token's scores [kv_heads, group, length], masked."""
    lengths, _ = _extents(s)
    group = s["heads"] // s["kv_heads"]
    for b, length in enumerate(lengths):
        keys = _gather(s, "k", s["tables"][b], length)
        scores = torch.matmul(s["q"][b].float().view(s["kv_heads"], group, -1), keys.transpose(1, 2)) * s["dim"] ** -0.5
        at = torch.arange(length, device=keys.device)
        slopes = s["slope_values"]
        scores = _shape_scores(s, scores, at - (length - 1), None if slopes is None else slopes.view(-1, group, 1))
        if s["window"]:
            scores = scores.masked_fill(at < length - s["window"], -math.inf)
        yield length, scores


def _plain_weigh(s):
    weights = torch.zeros((s["batch"], s["kv_heads"], s["tables"].shape[1] * s["page"]), device=s["q"].device)
    for b, (length, scores) in enumerate(_token_scores(s)):
        if length:
            weights[b, :, :length] = torch.exp(scores - s["lse"][b].view(s["kv_heads"], -1, 1)).sum(dim=1)
    return weights


def _plain_evict(s):
    lengths, _ = _extents(s)
    names = ("k", "v") if s["bits"] == 16 else ("k", "v", "k_scale", "v_scale")
    new_lengths, weights = s["lengths"].clamp(max=s["keep"]), torch.zeros_like(s["weights"])
    head = torch.arange(s["kv_heads"], device=weights.device)[:, None]
    for b, length in enumerate(lengths):
        kept = min(length, s["keep"])
        ranked = s["weights"][b, :, :length].clone()
        if length > kept:
            ranked[:, : s["first"]] = math.inf
            ranked[:, length - s["recent"]:] = math.inf
        order = torch.sort(ranked, dim=1, descending=True, stable=True).indices[:, :kept].sort(dim=1).values
        weights[b, :, :kept] = s["weights"][b].gather(1, order)
        at = torch.arange(kept, device=weights.device)[None, :]
        source, target = s["tables"][b].long(), s["new_tables"][b].long()
        for name in names:
            s[name][target[at // s["page"]], head, at % s["page"]] = s[name][source[order // s["page"]], head, order % s["page"]]
    if s["bits"] == 16:
        return {"lengths": new_lengths, "weights": weights, "k": s["k"], "v": s["v"]}
    rows = {}
    for name in ("k", "v"):
        kept = [min(n, s["keep"]) for n in lengths]
        rows[name] = torch.cat([_gather(s, name, s["new_tables"][b], n).transpose(0, 1) for b, n in enumerate(kept)]).to(torch.bfloat16)
    return {"lengths": new_lengths, "weights": weights, **rows}


# ------------------------------------------------------------------- one pass --

def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"prompt": _plain_prompt, "token": _plain_tokens, "shared": _plain_tokens, "weigh": _plain_weigh,
                "evict": _plain_evict}[kind](s)
    import chord_b200

    if kind == "evict":
        lengths, weights = chord_b200.cache_evict(s["cache"], s["tables"], s["lengths"], s["weights"], s["keep"],
                                                  first=s["first"], recent=s["recent"], new_tables=s["new_tables"])
        if s["bits"] == 16:
            return {"lengths": lengths, "weights": weights, "k": s["k"], "v": s["v"]}
        k, v = chord_b200.cache_read(s["cache"], s["new_tables"], s["offsets"], s["kept_rows"])
        return {"lengths": lengths, "weights": weights, "k": k, "v": v}
    shape = dict(window=s["window"] or None, cap=s["cap"] or None, slopes=s["slope_values"])
    if kind == "weigh":
        return chord_b200.attention_weights(s["q"], s["cache"], s["tables"], s["lengths"], s["lse"], **shape)
    if kind == "prompt":
        out = chord_b200.prompt_attention(s["q"], s["cache"], s["tables"], s["lengths"], s["offsets"], starts=s["starts"],
                                          prefixes=s["prefixes"], lse=s["lse"], **shape)
    elif kind == "shared":
        out = chord_b200.shared_prefix_attention(s["q"], s["cache"], s["prefix_tables"], s["prefix_lengths"],
                                                 s["group_offsets"], s["tables"], s["lengths"], lse=s["lse"], **shape)
    else:
        out = chord_b200.paged_attention(s["q"], s["cache"], s["tables"], s["lengths"], lse=s["lse"], **shape)
    return {"out": out, "lse": s["lse"]}


def _seen(case):
    """Pairs of a query token and a token that it sees, and tokens of the cache that any of them sees."""
    lengths, new = _extents(case)
    window = case["window"] or math.inf
    if case["kind"] == "shared":
        offsets, prefixes = _groups(case)
        pairs, rows = 0, 0
        for g, prefix in enumerate(prefixes):
            of = lengths[offsets[g]:offsets[g + 1]]
            pairs += sum(min(prefix + n, window) for n in of)
            rows += sum(min(n, window) for n in of) + max(max(0, min(prefix, window - n)) for n in of)
        return pairs, rows
    if case["kind"] != "prompt":
        return (sum(min(n, window) for n in lengths),) * 2
    starts, prefixes = _masks(case)
    pairs = rows = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        lowest, highest = length, 0
        for i in range(n):
            high = max(length - n + i + 1, min(prefixes[b], length))
            low = max(starts[b][i], length - n + i + 1 - window, 0)
            if high > low:
                pairs += high - low
                lowest, highest = min(lowest, low), max(highest, high)
        rows += max(0, highest - lowest)
    return pairs, rows


def work(case):
    kv_heads, dim = case["kv_heads"], case["dim"]
    row = 2 * dim if case["bits"] == 16 else dim + 4
    lengths, new = _extents(case)
    if case["kind"] == "evict":  # rows read and written, weights read and written whole
        kept = sum(min(n, case["keep"]) for n in lengths) * kv_heads
        every = case["batch"] * kv_heads * (-(-max(lengths) // case["page"]) * case["page"])
        read_back = 2 * kept * (row + 2 * dim) if case["bits"] == 8 else 0
        return {"bytes": 4 * kept * row + 4 * (sum(lengths) * kv_heads + every) + read_back, "flops": sum(lengths) * kv_heads}
    pairs, rows = _seen(case)
    queries = sum(new) * case["heads"]
    if case["kind"] == "weigh":
        every = case["batch"] * kv_heads * (-(-max(lengths) // case["page"]) * case["page"])
        return {"bytes": rows * kv_heads * row + 4 * every + queries * (2 * dim + 4), "flops": 2 * pairs * case["heads"] * dim}
    return {"bytes": 2 * rows * kv_heads * row + queries * (4 * dim + 4), "flops": 4 * pairs * case["heads"] * dim}


# -------------------------------------------------------------- 64-bit values --

def _rows64(state, name, pages, head, count):
    """One head's first `count` rows of a table's pages, in 64 bits."""
    at = torch.arange(count, device="cuda")
    page, place = pages.long()[at // state["page"]], at % state["page"]
    x = state[name][page, head, place].double()
    if state["bits"] == 8:
        x = (x - 128) * state[name + "_scale"][page, head, place].double()[:, None]
    return x


def _logits64(state, q, keys, position, head):
    z = q.double() @ keys.t() / math.sqrt(state["dim"])
    if state["cap"]:
        z = state["cap"] * torch.tanh(z / state["cap"])
    if state["slope_values"] is not None:
        steps = position.double()[:, None] - torch.arange(keys.shape[0], device="cuda", dtype=torch.float64)[None, :]
        z = z - state["slope_values"][head].double() * steps.abs()
    return z


def _exact_attention(case, state):
    lengths, new = _extents(case)
    shared, prompt = case["kind"] == "shared", case["kind"] == "prompt"
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first_row = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        before = 0
        if shared:
            offsets, prefixes = _groups(case)
            g = max(i for i in range(case["groups"]) if offsets[i] <= b)
            before = prefixes[g]
        total = before + length
        position = torch.arange(total - n, total, device="cuda")
        at = torch.arange(total, device="cuda")[None, :]
        seen = at <= position[:, None]
        if prompt and case["prefix"]:
            seen = seen | (at < int(state["prefixes"][b]))
        if prompt and case["documents"]:
            seen = seen & (at >= state["starts"][first_row:first_row + n, None])
        if case["window"]:
            seen = seen & (at > position[:, None] - case["window"])
        for h in range(case["kv_heads"]) if total else ():
            keys, values = (_rows64(state, name, state["tables"][b], h, length) for name in ("k", "v"))
            if shared:
                keys = torch.cat([_rows64(state, "k", state["prefix_tables"][g], h, before), keys])
                values = torch.cat([_rows64(state, "v", state["prefix_tables"][g], h, before), values])
            for head in range(h * group, (h + 1) * group):
                z = _logits64(state, state["q"][first_row:first_row + n, head], keys, position, head)
                z = torch.where(seen, z, -math.inf)
                sums = torch.logsumexp(z, dim=1)
                lse[first_row:first_row + n, head] = sums
                z = torch.exp(z - torch.where(sums == -math.inf, 0.0, sums)[:, None])
                out[first_row:first_row + n, head] = z @ values
        first_row += n
    return {"out": out, "lse": lse}


def _exact_weights(case, state):
    lengths, _ = _extents(case)
    group = case["heads"] // case["kv_heads"]
    weights = torch.zeros((case["batch"], case["kv_heads"], state["tables"].shape[1] * case["page"]), dtype=torch.float64,
                          device="cuda")
    for b, length in enumerate(lengths):
        low = max(0, length - case["window"]) if case["window"] else 0
        for head in range(case["heads"]) if length else ():
            h = head // group
            keys = _rows64(state, "k", state["tables"][b], h, length)
            z = _logits64(state, state["q"][b, head][None, :], keys, torch.tensor([length - 1], device="cuda"), head)[0]
            weights[b, h, low:length] += torch.exp(z[low:] - state["lse"][b, head].double())
    return weights


def _exact_eviction(case, state):
    lengths, _ = _extents(case)
    page, keep = case["page"], case["keep"]
    weights = torch.zeros(state["weights"].shape, dtype=torch.float64, device="cuda")
    coded = case["bits"] == 8
    made = {name: [] if coded else state[name].clone() for name in ("k", "v")}
    for b, length in enumerate(lengths):
        kept = min(length, keep)
        at = torch.arange(length, device="cuda")
        held = (at < case["first"]) | (at >= length - case["recent"])
        rows = {"k": [], "v": []}
        for h in range(case["kv_heads"]):
            chosen = torch.ones(length, dtype=torch.bool, device="cuda")
            if length > keep:
                free = at[~held]
                w = state["weights"][b, h, :length][free].double()
                least = torch.sort(w, descending=True).values[keep - case["first"] - case["recent"] - 1] if keep > case["first"] + case["recent"] else math.inf
                above, level = w > least, w == least
                room = keep - case["first"] - case["recent"] - int(above.sum())
                chosen = held.clone()
                chosen[free] = above | (level & (level.long().cumsum(0) <= room))
            order = at[chosen]
            weights[b, h, :kept] = state["weights"][b, h, order].double()
            for name in ("k", "v"):
                found = _rows64(state, name, state["tables"][b], h, length)[order]
                rows[name].append(found)
                if not coded:
                    place = torch.arange(kept, device="cuda")
                    made[name][state["new_tables"][b].long()[place // page], h, place % page] = found.to(torch.bfloat16)
        if coded:
            for name in ("k", "v"):
                made[name].append(torch.stack(rows[name], dim=1))
    if coded:
        made = {name: torch.cat(x) for name, x in made.items()}
    return {"lengths": torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device="cuda"), "weights": weights, **made}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_eviction(case, state)
    if case["kind"] == "weigh":
        return _exact_weights(case, state)
    return _exact_attention(case, state)
