"""The attention half of a decoder layer that is served with 4-bit weights, as cases that can be
timed and compared: products of a few rows with packed weights, norms of queries and keys with the
position rotation, the paged key-value cache as it is written and read back, and the attention of
one new token over it.

A case is one pass through an operator, called as a serving program calls it: the weights, the cache
and its tables are kept between passes, nothing synchronises.  Weights are INT4 codes with BF16
scales per 32 input channels in the library's packed layout (uniform codes, scales uniform in [0.005,
0.02]); activations are BF16 N(0, 1).

Kinds:
  gemv     gemv of ``rows`` rows with one weight [n, k]
  experts  gemv of ``tokens`` tokens, each with ``top_k`` of ``experts_total`` experts' weights, of
           which this GPU holds the first ``experts``
  rotate   qk_norm_rope of ``tokens`` tokens
  step     qk_norm_rope_write of ``tokens`` tokens of ragged sequences into the cache, and the
           sequences read back
  cache    cache_write of ``tokens`` tokens of ragged sequences, and the sequences read back
  attend   paged_attention of ``batch`` new tokens over sequences of up to ``length`` tokens

``own`` says which form runs: the plain one, in elementary operations in 32 bits, or the library's.
"""

import math

import torch

own = False

EPS = 1e-6

# Layer widths that the library's benchmark has.
HIDDEN, INTER, TOP_K = 7168, 2048, 8


def listed():
    heads = dict(heads=64, kv_heads=8, dim=128)
    return [
        # One token in a small layer: nothing but launch and call latency.
        dict(name="gemv_small", kind="gemv", rows=1, n=1024, k=512),
        # One interactive user: gate_up of an expert that every token takes.
        dict(name="gemv_one_token", kind="gemv", rows=1, n=2 * INTER, k=HIDDEN),
        # An odd small batch through the down projection of the same.
        dict(name="gemv_rows_13", kind="gemv", rows=13, n=HIDDEN, k=INTER),
        # One token's own experts, gate_up, all on this GPU (the largest product).
        dict(name="gemv_experts", kind="experts", tokens=1, top_k=TOP_K, experts=48, experts_total=48,
             n=2 * INTER, k=HIDDEN),
        # Heads of one new token.
        dict(name="rotate_one_token", kind="rotate", tokens=1, rotary=128, interleaved=False, **heads),
        # Heads of a long prompt.
        dict(name="rotate_prompt", kind="rotate", tokens=8192, rotary=128, interleaved=False, **heads),
        # Heads of an odd number of tokens, half of each head rotated in pairs, into an 8-bit cache.
        dict(name="step_61", kind="step", tokens=61, batch=7, heads=28, kv_heads=4, dim=128, rotary=64,
             interleaved=True, page=16, bits=8),
        # A prompt's keys and values into the 8-bit cache and back.
        dict(name="cache_prompt", kind="cache", tokens=16384, batch=5, kv_heads=8, dim=128, page=32, bits=8),
        # One sequence of a few hundred tokens: latency.
        dict(name="attend_short", kind="attend", batch=1, length=333, page=16, bits=16, window=0, empty=False, **heads),
        # A batch of ragged sequences in 16 bits (the largest attention).
        dict(name="attend_batch", kind="attend", batch=64, length=8192, page=64, bits=16, window=0, empty=False,
             **heads),
        # One very long sequence in 8 bits: work split over its length.
        dict(name="attend_long", kind="attend", batch=1, length=131072, page=64, bits=8, window=0, empty=False,
             **heads),
        # Odd sizes: a head each, narrow heads, pages that end inside tiles, a window, an empty sequence.
        dict(name="attend_window_odd", kind="attend", batch=37, length=3001, page=24, bits=8, window=1000, empty=True,
             heads=12, kv_heads=12, dim=64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of these ranges; no larger than the largest listed ones."""
    kind = rng.choice(["gemv", "gemv", "experts", "rotate", "step", "cache", "attend", "attend", "attend"])
    if kind in ("gemv", "experts"):
        n, k = 128 * _log_int(rng, 2, 112), 64 * _log_int(rng, 4, 224)
        if kind == "gemv":
            k = min(k, 235_000_000 // n // 64 * 64)
            return dict(kind=kind, rows=rng.choice([1, 1, 2, 3, 4, 6, 8, 11, 16]), n=n, k=k)
        tokens, top_k = rng.choice([1, 1, 2, 3, 4]), rng.randint(1, 8)
        n = max(128, min(n, 235_000_000 // (tokens * top_k * k) // 128 * 128))
        experts = rng.randint(8, 64)
        return dict(kind=kind, tokens=tokens, top_k=top_k, experts=experts, experts_total=experts * rng.choice([1, 1, 2]),
                    n=n, k=k)
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16])
    page, bits = rng.choice([8, 16, 16, 24, 32, 64, 100, 128]), rng.choice([8, 16])
    if kind == "attend":
        batch = _log_int(rng, 1, 256)
        length = min(_log_int(rng, 1, 131072), max(1, 64 * 8192 * 8 * 128 // (batch * kv_heads * dim)))
        return dict(kind=kind, batch=batch, length=length, page=page, bits=bits,
                    window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), empty=batch > 1 and rng.random() < 0.3,
                    heads=heads, kv_heads=kv_heads, dim=dim)
    tokens = max(1, min(_log_int(rng, 1, 16384), 8192 * 72 * 128 // ((heads + kv_heads) * dim)))
    case = dict(kind=kind, tokens=tokens, kv_heads=kv_heads, dim=dim)
    if kind in ("step", "cache"):
        case.update(batch=min(tokens, _log_int(rng, 1, 32)), page=page, bits=bits)
    if kind in ("step", "rotate"):
        case.update(heads=heads, rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.4)
    return case


# --------------------------------------------------------------------- inputs --

def _normal(shape, g):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(torch.bfloat16)


def _randint(high, shape, g, low=0):
    return torch.randint(low, high, shape, device="cuda", generator=g, dtype=torch.int32)


def _weight(experts, n, k, g):
    """Packed words [experts, k / 16, 2 n] and permuted scales [experts, k / 32, n]: any words are codes."""
    words = _randint(2**31 - 1, (experts, k // 16, 2 * n), g, -2**31)
    scale = torch.rand((experts, k // 32, n), device="cuda", generator=g).mul_(0.015).add_(0.005)
    return words, scale.to(torch.bfloat16)


def _cache(pages, case, g=None):
    """Pages of keys and values [pages, heads, page, dim], in 8 bits with a scale per row; empty or,
    with a generator, filled with normal values."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    made = {}
    for name in ("k", "v"):
        x = _normal(shape, g) if g is not None else torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        if case["bits"] == 8:
            x, made[name + "_scale"] = _quantise(x.float())
        made[name] = x
    return made


def _tables(lengths, page, g):
    """int32 [batch, pages of the longest]: each sequence's pages, in no order; -1 behind its last."""
    used = [-(-n // page) for n in lengths]
    most, total = max(max(used), 1), max(sum(used), 1)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    first = torch.tensor(used, device="cuda").cumsum(0)[:, None] - torch.tensor(used, device="cuda")[:, None]
    at = torch.arange(most, device="cuda")[None, :]
    there = at < torch.tensor(used, device="cuda")[:, None]
    return torch.where(there, order[(first + at).clamp(max=total - 1)], -1).to(torch.int32).contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    kind = case["kind"]
    if kind in ("gemv", "experts"):
        experts = case.get("experts", 1)
        state["words"], state["scales"] = _weight(experts, case["n"], case["k"], g)
        state["x"] = _normal((case.get("rows") or case["tokens"], case["k"]), g)
        if kind == "experts":
            scores = torch.rand((case["tokens"], case["experts_total"]), device="cuda", generator=g)
            state["ids"] = scores.topk(case["top_k"], dim=1).indices.to(torch.int32).contiguous()
        if own:  # the handle that a program keeps of its packed weight
            from chord_b200 import PreparedWeight

            state["weight"] = PreparedWeight(packed=state["words"], scale=state["scales"], n=case["n"], k=case["k"],
                                             num_experts=experts)
        return state
    heads, kv_heads, dim = case.get("heads", 0), case["kv_heads"], case["dim"]
    cut = torch.Generator().manual_seed(seed)
    if kind == "attend":
        lengths = torch.randint(max(1, case["length"] // 4), case["length"] + 1, (case["batch"],), generator=cut)
        lengths[0] = case["length"]
        if case["empty"]:
            lengths[-1] = 0
        state["tables"], pages = _tables(lengths.tolist(), case["page"], g)
        state["lengths"] = lengths.to(torch.int32).cuda()
        state["q"] = _normal((case["batch"], heads, dim), g).mul_(1.5)
        state["lse"] = torch.empty((case["batch"], heads), dtype=torch.float32, device="cuda")
        state.update(_cache(pages, case, g))
    else:
        # queries, keys and values of each token as one projection leaves them
        qkv = _normal((case["tokens"], heads + 2 * kv_heads, dim), g)
        state["q"], state["k_new"], state["v_new"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
        if "rotary" in case:
            state["q_weight"], state["k_weight"] = (torch.rand(dim, device="cuda", generator=g).add_(0.5).to(torch.bfloat16)
                                                    for _ in range(2))
            most = 2 * case["tokens"] + 64
            rate = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
            angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * rate[None, :]
            state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
            state["positions"] = _randint(most, (case["tokens"],), g)
    if kind in ("step", "cache"):
        # the tokens are those of `batch` sequences, one after another
        ends = torch.cat([torch.randperm(case["tokens"] - 1, generator=cut)[: case["batch"] - 1].add(1).sort().values,
                          torch.tensor([case["tokens"]])])
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), ends[:-1]])
        state["tables"], pages = _tables((ends - starts).tolist(), case["page"], g)
        state["offsets"] = torch.cat([starts[:1], ends]).to(torch.int32).cuda()
        sequence = torch.repeat_interleave(torch.arange(case["batch"]), ends - starts).cuda()
        at = torch.arange(case["tokens"], device="cuda") - starts.cuda()[sequence]
        state["sequence"], state["at"] = sequence, at
        state["slots"] = (state["tables"][sequence, at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)
        state.update(_cache(pages, case))
    if own and "k" in state:  # the handle of the cache
        from chord_b200 import KVCache

        state["cache"] = KVCache(state["k"], state["v"], state.get("k_scale"), state.get("v_scale"))
    return state


# ---------------------------------------------------------------- plain forms --

def _quantise(x):
    """Codes round(x / scale) + 128 and the row's scale, largest |x| / 127."""
    scale = x.abs().amax(dim=-1) / 127
    codes = torch.round(x / torch.where(scale > 0, scale, 1.0)[..., None]) + 128
    return codes.to(torch.uint8), scale


def _values(words, scales, n, k):
    """The weights [.., n, k] that packed words stand for, in 32 bits."""
    e = words.shape[0]
    # word (kb, n / 64, t, s), bit 4 (2 rh + kh) + 16 kk: row 16 s + 8 rh + t / 4, column 8 kh + 2 (t % 4) + kk
    shifts = torch.tensor([[[0, 16], [4, 20]], [[8, 24], [12, 28]]], dtype=torch.int32, device=words.device)
    codes = (words.view(e, k // 16, n // 64, 8, 4, 4, 1, 1, 1) >> shifts) & 15
    codes = codes.permute(0, 2, 5, 6, 3, 1, 7, 4, 8).reshape(e, n, k // 32, 32)
    scale = scales.view(e, k // 32, n // 64, 8, 8).transpose(3, 4).reshape(e, k // 32, n).transpose(1, 2)
    return ((codes - 8).float() * scale.float()[..., None]).view(e, n, k)


def _plain_product(s):
    x = s["x"].float()
    if s["kind"] == "gemv":
        return (x @ _values(s["words"], s["scales"], s["n"], s["k"])[0].t()).to(torch.bfloat16)
    ids = s["ids"].reshape(-1).long()
    here = ids < s["experts"]
    ids = torch.where(here, ids, 0)
    w = _values(s["words"][ids], s["scales"][ids], s["n"], s["k"])
    y = torch.bmm(w, x.repeat_interleave(s["top_k"], dim=0)[:, :, None])[:, :, 0]
    return torch.where(here[:, None], y, 0.0).to(torch.bfloat16)


def _plain_rotate(s, x, weight):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    half = s["rotary"] // 2
    angles = s["cos_sin"][s["positions"].long()][:, None, :]
    cos, sin = angles[..., :half], angles[..., half:]
    turned, rest = x[..., : s["rotary"]], x[..., s["rotary"]:]
    if s["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_write_read(s, name, x):
    pages = s[name].permute(0, 2, 1, 3)
    page, row = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    found = s["tables"][s["sequence"], s["at"] // s["page"]].long()
    if s["bits"] == 16:
        pages[page, row] = x.to(torch.bfloat16)
        return pages[found, s["at"] % s["page"]]
    scales = s[name + "_scale"].permute(0, 2, 1)
    pages[page, row], scales[page, row] = _quantise(x.float())
    codes, scale = pages[found, s["at"] % s["page"]], scales[found, s["at"] % s["page"]]
    return ((codes.float() - 128) * scale[..., None]).to(torch.bfloat16)


def _plain_attend(s):
    batch, heads, dim = s["q"].shape
    kv_heads, page = s["kv_heads"], s["page"]
    tables = s["tables"].long().clamp(min=0)
    length = tables.shape[1] * page

    def values(name):
        x = s[name][tables].float()
        if s["bits"] == 8:
            x = (x - 128) * s[name + "_scale"][tables][..., None]
        return x.transpose(1, 2).reshape(batch, kv_heads, length, dim)

    q = s["q"].float().view(batch, kv_heads, heads // kv_heads, dim)
    scores = torch.matmul(q, values("k").transpose(2, 3)) * dim**-0.5
    at, last = torch.arange(length, device=q.device), s["lengths"][:, None, None, None]
    seen = (at < last) & (at >= (last - s["window"] if s["window"] else 0))
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, values("v")) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).view(batch, heads)
    return {"out": out.view(batch, heads, dim).to(torch.bfloat16), "lse": lse}


def _plain(s):
    kind = s["kind"]
    if kind in ("gemv", "experts"):
        return _plain_product(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "cache":
        return {"k": _plain_write_read(s, "k", s["k_new"]), "v": _plain_write_read(s, "v", s["v_new"])}
    q, k = _plain_rotate(s, s["q"], s["q_weight"]).to(torch.bfloat16), _plain_rotate(s, s["k_new"], s["k_weight"])
    if kind == "rotate":
        return {"q": q, "k": k.to(torch.bfloat16)}
    return {"q": q, "k": _plain_write_read(s, "k", k), "v": _plain_write_read(s, "v", s["v_new"])}


# ------------------------------------------------------------------- one pass --

def run(state):
    if not own:
        return _plain(state)
    import chord_b200

    s, kind = state, state["kind"]
    if kind == "gemv":
        return chord_b200.gemv(s["x"], s["weight"])
    if kind == "experts":
        return chord_b200.gemv(s["x"], s["weight"], expert_ids=s["ids"], top_k=s["top_k"])
    if kind == "attend":
        out = chord_b200.paged_attention(s["q"], s["cache"], s["tables"], s["lengths"], window=s["window"] or None,
                                         lse=s["lse"])
        return {"out": out, "lse": s["lse"]}
    if kind == "rotate":
        q, k = chord_b200.qk_norm_rope(s["q"], s["k_new"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"],
                                       eps=EPS, interleaved=s["interleaved"])
        return {"q": q, "k": k}
    if kind == "step":
        q = chord_b200.qk_norm_rope_write(s["q"], s["k_new"], s["v_new"], s["q_weight"], s["k_weight"], s["cos_sin"],
                                          s["positions"], s["cache"], s["slots"], eps=EPS, interleaved=s["interleaved"])
    else:
        chord_b200.cache_write(s["k_new"], s["v_new"], s["cache"], s["slots"])
    k, v = chord_b200.cache_read(s["cache"], s["tables"], s["offsets"], s["tokens"])
    return {"q": q, "k": k, "v": v} if kind == "step" else {"k": k, "v": v}


def work(case):
    kind = case["kind"]
    if kind in ("gemv", "experts"):
        n, k = case["n"], case["k"]
        if kind == "gemv":
            inputs = rows = case["rows"]
            reads = 1
        else:
            inputs = case["tokens"]
            rows = inputs * case["top_k"]
            # routes to experts that are held elsewhere read nothing; an expert is read once for all its rows
            share = case["experts"] / case["experts_total"]
            reads = min(rows, case["experts_total"]) * share
        weight = n * k // 2 + n * k // 16
        return {"bytes": reads * weight + 2 * (inputs * k + rows * n), "flops": 2 * reads * n * k * (rows if kind == "gemv" else 1)}
    kv_heads, dim = case["kv_heads"], case["dim"]
    row = 2 * dim if case.get("bits", 16) == 16 else dim + 4
    if kind == "attend":
        # the longest and, on average, 5 / 8 of it for the others
        others = case["batch"] - 1 - (1 if case["empty"] else 0)
        seen = min(case["length"], case["window"] or case["length"])
        tokens = seen + others * min(seen, case["length"] * 5 / 8)
        return {"bytes": 2 * tokens * kv_heads * row + 4 * case["batch"] * case["heads"] * (dim + 1),
                "flops": 4 * tokens * case["heads"] * dim}
    tokens = case["tokens"]
    kv = 2 * tokens * kv_heads
    if kind == "cache":  # read as BF16, kept, read, given out as BF16
        return {"bytes": kv * (4 * dim + 2 * row), "flops": kv * 4 * dim}
    rotated = tokens * (case["heads"] + kv_heads)
    if kind == "rotate":
        return {"bytes": rotated * 4 * dim + tokens * 4 * case["rotary"], "flops": rotated * 10 * dim}
    return {"bytes": tokens * case["heads"] * 4 * dim + kv * (4 * dim + 2 * row) + tokens * 4 * case["rotary"],
            "flops": rotated * 10 * dim + kv * 4 * dim}


# -------------------------------------------------------------- 64-bit values --

def _exact_row(state, row):
    """One row's product, in 64 bits, from the layout's definition: word c of line kb holds the codes of
    weights (64 (c / 128) + 16 s + 8 rh + t / 4, 16 kb + 8 kh + 2 (t % 4) + kk), t = c % 128 / 4, s = c % 4."""
    n, k = state["n"], state["k"]
    expert, token = 0, row
    if state["kind"] == "experts":
        expert, token = int(state["ids"].reshape(-1)[row]), row // state["top_k"]
        if expert >= state["experts"]:
            return torch.zeros(n, dtype=torch.float64, device="cuda")
    words = state["words"][expert].long() & 0xFFFFFFFF
    c = torch.arange(2 * n, device="cuda")
    t, s = c % 128 // 4, c % 4
    at = torch.arange(n, device="cuda")
    scale = state["scales"][expert].double()[:, at // 64 * 64 + 8 * (at % 8) + at % 64 // 8]  # [k / 32, n]
    x = state["x"][token].double()
    result = torch.zeros(n, dtype=torch.float64, device="cuda")
    line = torch.arange(k // 16, device="cuda")
    for rh in range(2):
        target = 64 * (c // 128) + 16 * s + 8 * rh + t // 4
        for kh in range(2):
            for kk in range(2):
                code = (words >> (4 * (2 * rh + kh) + 16 * kk)) & 15
                column = 16 * line[:, None] + (8 * kh + 2 * (t % 4) + kk)[None, :]
                terms = x[column] * (code - 8).double() * scale[(line // 2)[:, None], target[None, :]]
                result.index_add_(0, target, terms.sum(dim=0))
    return result


def _exact_heads(state, x, weight):
    x, half = x.double(), state["rotary"] // 2
    x = x / ((x ** 2).mean(dim=2, keepdim=True) + EPS).sqrt() * weight.double()
    table = state["cos_sin"].double()[state["positions"].long()]
    result = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if state["interleaved"] else (i, i + half)
        cos, sin = table[:, i, None], table[:, half + i, None]
        result[:, :, a] = x[:, :, a] * cos - x[:, :, b] * sin
        result[:, :, b] = x[:, :, b] * cos + x[:, :, a] * sin
    return result


def _exact_kept(state, x):
    """What the cache gives back of rows x (64 bits in): BF16 as it is, 8 bits as the code's value."""
    if state["bits"] == 16:
        return x
    step = x.abs().amax(dim=2, keepdim=True) / 127
    return torch.where(step > 0, (x / step).round() * step, 0.0)


def _exact_attention(state):
    q, page = state["q"].double(), state["page"]
    batch, heads, dim = q.shape
    group = heads // state["kv_heads"]
    out, lse = torch.zeros_like(q), torch.full((batch, heads), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(batch):
        last = int(state["lengths"][b])
        first = max(0, last - state["window"]) if state["window"] else 0
        if last == first:
            continue
        pages = state["tables"][b].long()[: -(-last // page)]
        for h in range(state["kv_heads"]):
            got = []
            for name in ("k", "v"):
                x = state[name][pages, h].double()
                if state["bits"] == 8:
                    x = (x - 128) * state[name + "_scale"][pages, h].double()[..., None]
                got.append(x.reshape(-1, dim)[first:last])
            scores = q[b, h * group:(h + 1) * group] @ got[0].t() / math.sqrt(dim)
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(scores, dim=1)
            out[b, h * group:(h + 1) * group] = torch.softmax(scores, dim=1) @ got[1]
    return {"out": out, "lse": lse}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind in ("gemv", "experts"):
        rows = case["rows"] if kind == "gemv" else case["tokens"] * case["top_k"]
        return torch.stack([_exact_row(state, r) for r in range(rows)])
    if kind == "attend":
        return _exact_attention(state)
    if kind == "cache":
        return {name: _exact_kept(state, state[name + "_new"].double()) for name in ("k", "v")}
    q, k = (_exact_heads(state, state[x], state[w]) for x, w in (("q", "q_weight"), ("k_new", "k_weight")))
    if kind == "rotate":
        return {"q": q, "k": k}
    return {"q": q, "k": _exact_kept(state, k), "v": _exact_kept(state, state["v_new"].double())}
