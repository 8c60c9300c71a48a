"""What the operators of a bounded paged cache are timed and compared on: norms of query and key
heads with the position rotation in the same pass, forward and backward; the append to a paged
cache with those norms, at positions that count evicted tokens; the attention weight that each
cached key has received; and the eviction of all but the heaviest tokens.

A cache is an array of pages [pages, page, kv_heads, dim] for the keys and one for the values; the
weights are [pages, page, kv_heads] in 32 bits, the slots of a head side by side.  Which pages a
sequence owns is a CSR structure, int64 ``indptr``/``indices``.

A case is {"name", "op", "dtype", "dim", "kv_heads", ...}:
  op "norm"     tokens, heads, rotary (dims that are rotated), layout (half | interleaved),
                scaling (none | linear | yarn), positions (the largest), weight (its type),
                per_head (a weight for each head instead of one for all), backward
  op "append"   sequences, max_query (new tokens per sequence, 1 to that many), offset (of the
                positions), evicted (tokens that a sequence has lost, at most), max_length, page,
                heads, rotary, layout, scaling
  op "weights"  sequences, max_query, prefix (tokens before the sequences' own, which take their
                share of the attention), max_length, page, heads, decay
  op "evict"    sequences, min_length, max_length (tokens held), keep, recent and first (tokens
                that stay whatever their weight), page, move_weights
"""

import math
import random

import numpy as np
import torch

own = False

BASE = 10000.0
TRAINED = 4096              # positions that the unscaled frequencies were made for
EPSILON = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # queries and keys of a decode step of 8 sequences: one launch, latency alone
        {"name": "norm_decode", "op": "norm", "dtype": "bf16", "tokens": 8, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "yarn",
         "positions": 131072, "weight": "bf16", "per_head": False, "backward": False},
        # a training step's queries and keys, forward
        {"name": "norm_train", "op": "norm", "dtype": "bf16", "tokens": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "none",
         "positions": 4096, "weight": "bf16", "per_head": False, "backward": False},
        # its backward pass: gradients of the heads and, summed over all tokens, of the weights
        {"name": "norm_backward", "op": "norm", "dtype": "bf16", "tokens": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "none",
         "positions": 4096, "weight": "bf16", "per_head": False, "backward": True},
        # in single precision: a part of an odd head size turned, a weight for each head, an odd
        # token count
        {"name": "norm_backward_part", "op": "norm", "dtype": "f32", "tokens": 4095, "heads": 20,
         "kv_heads": 5, "dim": 96, "rotary": 64, "layout": "interleaved", "scaling": "linear",
         "positions": 16384, "weight": "f32", "per_head": True, "backward": True},
        # a decode step of a bounded cache: one new token each, many already evicted
        {"name": "append_decode", "op": "append", "dtype": "bf16", "sequences": 32,
         "max_query": 1, "offset": 8192, "evicted": 20000, "max_length": 1024, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half",
         "scaling": "yarn"},
        # prompts of mixed lengths, small heads, interleaved pairs in half of each head
        {"name": "append_ragged", "op": "append", "dtype": "f16", "sequences": 17,
         "max_query": 700, "offset": 0, "evicted": 900, "max_length": 1500, "page": 24,
         "heads": 12, "kv_heads": 4, "dim": 64, "rotary": 32, "layout": "interleaved",
         "scaling": "none"},
        # a handful of short sequences: latency alone
        {"name": "weights_small", "op": "weights", "dtype": "f16", "sequences": 4,
         "max_query": 1, "prefix": 0, "max_length": 300, "page": 16, "heads": 8, "kv_heads": 2,
         "dim": 64, "decay": 1.0},
        # an ordinary decode step, old weights fading
        {"name": "weights_decode", "op": "weights", "dtype": "bf16", "sequences": 32,
         "max_query": 1, "prefix": 8192, "max_length": 4096, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "decay": 0.98},
        # prompts of up to 4096 tokens, every query counted: matrix products throughout
        {"name": "weights_prompt", "op": "weights", "dtype": "bf16", "sequences": 4,
         "max_query": 4096, "prefix": 0, "max_length": 4500, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "decay": 1.0},
        # three short sequences of odd sizes: latency alone
        {"name": "evict_small", "op": "evict", "dtype": "f16", "sequences": 3, "min_length": 90,
         "max_length": 210, "keep": 101, "recent": 17, "first": 3, "page": 24, "kv_heads": 3,
         "dim": 96, "move_weights": True},
        # every 64 steps of a decode loop, down to 1024 tokens again
        {"name": "evict_step", "op": "evict", "dtype": "bf16", "sequences": 32,
         "min_length": 1025, "max_length": 1088, "keep": 1024, "recent": 256, "first": 4,
         "page": 16, "kv_heads": 8, "dim": 128, "move_weights": True},
        # long prompts cut to an eighth, their weights not needed again
        {"name": "evict_prompt", "op": "evict", "dtype": "bf16", "sequences": 4,
         "min_length": 12000, "max_length": 16384, "keep": 2048, "recent": 128, "first": 16,
         "page": 64, "kv_heads": 8, "dim": 128, "move_weights": False},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _rotary(rng, dim):
    return rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 2])


def draw(rng):
    op = rng.choice(["norm", "append", "weights", "evict"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([g for g in (1, 2, 3, 4, 8, 16) if g * kv_heads <= 64])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "dim": dim, "kv_heads": kv_heads}
    if op == "norm":
        dtype = rng.choice(["bf16", "f16", "f32"])
        size = 4 if dtype == "f32" else 2
        rows = (group + 1) * kv_heads
        tokens = _between(rng, 1, min(16384, 16384 * 40 * 128 * 2 // (size * rows * dim)))
        return dict(case, dtype=dtype, tokens=tokens, heads=group * kv_heads,
                    rotary=_rotary(rng, dim), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn"]),
                    positions=_between(rng, tokens, 131072), weight=rng.choice([dtype, "f32"]),
                    per_head=rng.random() < 0.3, backward=rng.random() < 0.5)
    case["page"] = rng.choice([16, 16, 24, 32, 64, 128])
    sequences = _between(rng, 1, 128)
    if op == "append":
        most = min(16384, 16384 * 40 * 128 // ((group + 2) * kv_heads * dim))
        max_query = _between(rng, 1, max(1, most // sequences)) if rng.random() < 0.6 else 1
        return dict(case, dtype=rng.choice(["bf16", "f16", "f32"]), sequences=sequences,
                    max_query=max_query, offset=rng.choice([0, _between(rng, 1, 65536)]),
                    evicted=rng.choice([0, _between(rng, 1, 65536)]),
                    max_length=max_query + _between(rng, 1, 1024), heads=group * kv_heads,
                    rotary=_rotary(rng, dim), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn"]))
    if op == "weights":
        max_query = 1 if rng.random() < 0.6 else _between(rng, 2, max(3, 4096 // sequences))
        rows = sequences * max_query * group * kv_heads
        most = min(16384, 2e9 * 128 / (rows * dim), 1.3e8 / (sequences * kv_heads * dim))
        return dict(case, sequences=sequences, max_query=max_query,
                    prefix=rng.choice([0, _between(rng, 1, 65536)]),
                    max_length=max_query + _between(rng, 1, max(2, most)),
                    heads=group * kv_heads, decay=rng.choice([1.0, 0.98, 0.9]))
    max_length = _between(rng, 2, min(32768, 1.3e8 / (sequences * kv_heads * dim)))
    keep = _between(rng, 1, max_length)
    recent = rng.choice([0, rng.randint(0, keep), rng.randint(0, keep // 4)])
    return dict(case, dtype=rng.choice(["bf16", "f16", "f32"]), sequences=sequences,
                min_length=rng.randint(1, max_length), max_length=max_length, keep=keep,
                recent=recent, first=rng.choice([0, min(4, keep - recent)]),
                move_weights=rng.random() < 0.7)


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _frequency(case, dev):
    """(radians per position of each pair, magnitude): base^(-2i/rotary), positions divided by
    4 (linear), or low frequencies divided by 32 with a ramp between 1 and 32 turns over the
    trained length and the rotated part scaled by 0.1 ln 32 + 1 (yarn)."""
    n = case["rotary"]
    f = BASE ** (-torch.arange(0, n, 2, dtype=torch.float64, device=dev) / n)
    if case["scaling"] == "linear":
        return f / 4, 1.0
    if case["scaling"] == "yarn":
        keep = ((TRAINED * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f * keep + f / 32 * (1 - keep), 0.1 * math.log(32) + 1
    return f, 1.0


def _spread(n, lo, hi):
    """n whole numbers evenly from lo to hi (both there where n > 1)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sequences(case):
    """Of each sequence: its new tokens, and those that its pages held when they came; in an
    order that has nothing to do with the seed."""
    n = case["sequences"]
    if case["op"] == "evict":
        return [(0, x) for x in _spread(n, case["min_length"], case["max_length"])]
    before = _spread(n, 0, case["max_length"] - case["max_query"])
    random.Random(1).shuffle(before)
    return list(zip(_spread(n, 1, case["max_query"]), before))


def _indptr(counts, dev):
    return torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(dev)


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op, H, D = case["op"], case["kv_heads"], case["dim"]

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    def learned(heads):
        """A norm's weight, near one."""
        kind = DTYPES[case.get("weight", case["dtype"])]
        shape = (heads, D) if case.get("per_head") else (D,)
        return (1 + 0.2 * normal(*shape, dtype=torch.float32)).to(kind)

    s = {"case": case}
    if "rotary" in case:
        f, s["magnitude"] = _frequency(case, dev)
        s["frequency"] = f
        last = (case["positions"] if op == "norm" else
                case["offset"] + case["evicted"] + case["max_length"])
        angle = torch.arange(last, dtype=torch.float64, device=dev)[:, None] * f
        # the tables that the plain form looks its rotations up in
        s["cos"] = (angle.cos() * s["magnitude"]).float()
        s["sin"] = (angle.sin() * s["magnitude"]).float()
        s["query_weight"], s["key_weight"] = learned(case["heads"]), learned(H)
    if op == "norm":
        n, heads = case["tokens"], case["heads"]
        # a decode step's tokens stand anywhere; a longer call's follow one another
        s["positions"] = torch.randint(case["positions"], (n if n <= 64 else 1,), generator=g,
                                       device=dev)
        if n > 64:
            s["positions"] = (s["positions"] + torch.arange(n, device=dev)) % case["positions"]
        # queries and keys stand in one packed projection, of tokens of different sizes
        x = (normal(n, heads + 2 * H, D, dtype=torch.float32)
             * (0.5 * normal(n, 1, 1, dtype=torch.float32)).exp()).to(dtype)
        s["query"], s["key"] = x[:, :heads], x[:, heads:heads + H]
        if case["backward"]:
            s["grad_query"], s["grad_key"] = normal(n, heads, D), normal(n, H, D)
        return s
    rng = random.Random(seed)
    page = case["page"]
    sequences = _sequences(case)
    rng.shuffle(sequences)
    counts = [new for new, _ in sequences]
    lengths = [new + before for new, before in sequences]
    owned = [-(-n // page) + i % 2 for i, n in enumerate(lengths)]   # every other holds a spare
    pages = sum(owned) + 3
    order = torch.randperm(pages, generator=g, device=dev)
    s.update(
        indices=order[:sum(owned)], indptr=_indptr(owned, dev),
        lengths=torch.tensor(lengths, dtype=torch.int64, device=dev),
        key_cache=normal(pages, page, H, D))
    if op != "weights":
        s["value_cache"] = normal(pages, page, H, D)
    if op != "append":
        # heavy-tailed, and some keys that nothing has looked at
        w = (1.5 * normal(pages, H, page, dtype=torch.float32)).exp()
        w = w * (torch.rand(w.shape, generator=g, device=dev) > 0.05)
        s["weights"] = w.transpose(1, 2)
    if op == "evict":
        return s
    s["query"] = normal(sum(counts), case["heads"], D)
    s["query_indptr"] = _indptr(counts, dev) if case["max_query"] > 1 else None
    if op == "append":
        s["key"], s["value"] = normal(sum(counts), H, D), normal(sum(counts), H, D)
        s["shift"] = torch.randint(case["evicted"] + 1, (len(counts),), generator=g, device=dev)
        return s
    # some keys are longer than others, and draw more attention
    s["key_cache"] *= (0.4 * normal(pages, page, H, 1, dtype=torch.float32)).exp().to(dtype)
    s["lse"] = _log_sums(s, counts, lengths, g)
    return s


def _log_sums(s, counts, lengths, g):
    """The logarithm of each row's sum of exponentials, over its own keys and a prefix's, as
    attention leaves it."""
    case, lse, t = s["case"], [], 0
    H, D = case["kv_heads"], case["dim"]
    G, rows = case["heads"] // H, s["indptr"].tolist()
    for b, (n, length) in enumerate(zip(counts, lengths)):
        k = s["key_cache"][s["indices"][rows[b]:rows[b + 1]]].flatten(0, 1)[:length].float()
        q = s["query"][t:t + n].float().reshape(n, H, G, D).transpose(0, 1).reshape(H, n * G, D)
        score = (q @ k.permute(1, 2, 0).contiguous()).reshape(H, n, G, length) * D ** -0.5
        at = torch.arange(length, device=k.device)
        hidden = at > (length - n + torch.arange(n, device=k.device))[:, None]
        score.masked_fill_(hidden[:, None], -math.inf)
        lse.append(score.logsumexp(-1).transpose(0, 1).reshape(n, H * G))
        t += n
    lse = torch.cat(lse)
    if case["prefix"]:
        more = torch.randn(lse.shape, generator=g, device=lse.device) * 0.2
        lse = torch.logaddexp(lse, more + math.log(case["prefix"]) + 0.5)
    return lse


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def _pairs(y, n, layout):
    return (y[..., :n // 2], y[..., n // 2:n]) if layout == "half" else (y[..., 0:n:2],
                                                                         y[..., 1:n:2])


def _rotate(y, cos, sin, layout, back=False):
    """Pairs of y[..., :rotary] turned by their angles; the rest as it is."""
    n = 2 * cos.shape[-1]
    cos, sin = cos[:, None], -sin[:, None] if back else sin[:, None]
    a, b = _pairs(y, n, layout)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, y[..., n:]], -1)


def _normed(x, weight, cos, sin, layout):
    y = x.float()
    r = (y.square().mean(-1, keepdim=True) + EPSILON).rsqrt()
    return _rotate(y * r * weight.float(), cos, sin, layout).to(x.dtype)


def _normed_back(grad, x, weight, cos, sin, layout):
    y, u = x.float(), _rotate(grad.float(), cos, sin, layout, back=True)
    r = (y.square().mean(-1, keepdim=True) + EPSILON).rsqrt()
    y = y * r
    dw = (u * y).sum(0 if weight.dim() == 2 else (0, 1))
    v = u * weight.float()
    dx = r * (v - y * (v * y).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(weight.dtype)


def _tokens(s):
    """Each new token's sequence, its place among the sequence's new ones, and its slot."""
    n = s["query"].shape[0]
    at = torch.arange(n, device=s["query"].device)
    if s["query_indptr"] is None:
        return at, torch.zeros_like(at), s["lengths"] - 1
    seq = torch.searchsorted(s["query_indptr"], at, right=True) - 1
    nth = at - s["query_indptr"][seq]
    return seq, nth, (s["lengths"] - s["query_indptr"].diff())[seq] + nth


def _plain_append(s):
    case = s["case"]
    seq, _, slot = _tokens(s)
    position = case["offset"] + s["shift"][seq] + slot
    cos, sin = s["cos"][position], s["sin"][position]
    page = s["indices"][s["indptr"][seq] + slot // case["page"]]
    slot = slot % case["page"]
    s["key_cache"][page, slot] = _normed(s["key"], s["key_weight"], cos, sin, case["layout"])
    s["value_cache"][page, slot] = s["value"]
    return _normed(s["query"], s["query_weight"], cos, sin, case["layout"])


def _places(s, length):
    """Page and slot of positions 0 .. length - 1 of each sequence (past its end: any)."""
    page = s["case"]["page"]
    at = torch.arange(length, device=s["indptr"].device)
    listed_at = (s["indptr"][:-1, None] + at // page).clamp(max=s["indices"].numel() - 1)
    return s["indices"][listed_at], (at % page).expand(listed_at.shape)


def _plain_weights(s):
    case = s["case"]
    B, H, D = case["sequences"], case["kv_heads"], case["dim"]
    G, n, L = case["heads"] // H, case["max_query"], case["max_length"]
    T = s["query"].shape[0]
    seq, nth, position = _tokens(s)
    page, slot = _places(s, L)
    k = s["key_cache"][page, slot].float().permute(0, 2, 3, 1)          # [B, H, D, L]
    q, lse = k.new_zeros(B, n, H, G, D), k.new_full((B, n, H, G), math.inf)
    q[seq, nth] = s["query"].float().reshape(T, H, G, D)
    lse[seq, nth] = s["lse"].reshape(T, H, G)
    score = q.transpose(1, 2).reshape(B, H, n * G, D) @ k.contiguous()
    score.mul_(D ** -0.5).sub_(lse.transpose(1, 2).reshape(B, H, n * G, 1)).exp_()
    seen = torch.full((B, n), -1, dtype=torch.int64, device=k.device)
    seen[seq, nth] = position
    at = torch.arange(L, device=k.device)
    hidden = (at > seen[:, :, None]).repeat_interleave(G, 1)[:, None]
    got = score.masked_fill_(hidden, 0).sum(2)                          # [B, H, L]
    # into the slots that sequences hold, new ones from nothing
    counts = s["query_indptr"].diff() if s["query_indptr"] is not None else 1
    held = sum(new + before for new, before in _sequences(case))
    b = torch.repeat_interleave(s["lengths"], output_size=held)
    at = torch.arange(held, device=k.device) - (s["lengths"].cumsum(0) - s["lengths"])[b]
    old = s["weights"][page[b, at], slot[b, at]] * case["decay"]
    old = old * (at < (s["lengths"] - counts)[b])[:, None]
    s["weights"][page[b, at], slot[b, at]] = old + got[b, :, at]
    return s["weights"]


def _plain_evict(s):
    case = s["case"]
    B, H, L, K = case["sequences"], case["kv_heads"], case["max_length"], case["keep"]
    page, slot = _places(s, L)
    lengths = s["lengths"][:, None, None]
    at = torch.arange(L, device=page.device)
    live = at < lengths
    w = s["weights"][page, slot].transpose(1, 2)                        # [B, H, L]
    w = w.masked_fill((at < case["first"]) | (at >= lengths - case["recent"]), math.inf)
    w = w.masked_fill(~live, -math.inf)
    order = w.sort(dim=-1, descending=True, stable=True).indices[..., :K]
    chosen = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, order, True) & live
    # the kept of the front stay; the others, ascending, fill its holes; the recent move down
    gone = (s["lengths"] - K).clamp(min=0)
    front, to = K - case["recent"], torch.arange(K, device=page.device)
    inside = chosen[..., :front]
    others = (chosen & (at >= front) & (at < lengths - case["recent"]))
    others = torch.where(others, at, L).sort(dim=-1).values
    nth = ((~inside).cumsum(-1) - 1).clamp(min=0)
    kept = (to + gone[:, None, None]).expand(B, H, K).clone()
    kept[..., :front] = torch.where(inside, to[:front], others.gather(-1, nth))
    lengths = s["lengths"] - gone
    valid = to < lengths[:, None, None]
    kept = torch.where(valid, kept, -1)
    # rows past the end do as the first row does
    b = torch.arange(B, device=page.device)[:, None, None]
    h = torch.arange(H, device=page.device)[:, None]
    source, to = torch.where(valid, kept, kept[..., :1]), torch.where(valid, to, 0)
    names = ("key_cache", "value_cache") + (("weights",) if case["move_weights"] else ())
    out = {"lengths": lengths, "kept": kept.int()}
    for name in names:
        cache = s[name]
        cache[page[b, to], slot[b, to], h] = cache[page[b, source], slot[b, source], h]
        out[name] = cache
    return out


def run(state):
    s, case = state, state["case"]
    if own:
        from tilegen_amd import attention
    if case["op"] == "norm" and not case["backward"]:
        if own:
            return attention.norm_rope(
                s["query"], s["key"], s["positions"], s["frequency"], s["query_weight"],
                s["key_weight"], epsilon=EPSILON, layout=case["layout"],
                magnitude=s["magnitude"])
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return (_normed(s["query"], s["query_weight"], cos, sin, case["layout"]),
                _normed(s["key"], s["key_weight"], cos, sin, case["layout"]))
    if case["op"] == "norm":
        if own:
            return attention.norm_rope_backward(
                s["grad_query"], s["grad_key"], s["query"], s["key"], s["positions"],
                s["frequency"], s["query_weight"], s["key_weight"], epsilon=EPSILON,
                layout=case["layout"], magnitude=s["magnitude"])
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        dq, dqw = _normed_back(s["grad_query"], s["query"], s["query_weight"], cos, sin,
                               case["layout"])
        dk, dkw = _normed_back(s["grad_key"], s["key"], s["key_weight"], cos, sin,
                               case["layout"])
        return dq, dk, dqw, dkw
    if case["op"] == "append":
        if own:
            query = attention.paged_append(
                s["key"], s["value"], s["key_cache"], s["value_cache"], s["indptr"],
                s["indices"], s["lengths"], s["frequency"], query=s["query"],
                query_indptr=s["query_indptr"], offset=case["offset"], layout=case["layout"],
                magnitude=s["magnitude"], query_weight=s["query_weight"],
                key_weight=s["key_weight"], epsilon=EPSILON, shift=s["shift"])
        else:
            query = _plain_append(s)
        return {"query": query, "key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    if case["op"] == "weights":
        if own:
            return attention.attention_weights(
                s["query"], s["lse"], s["key_cache"], s["weights"], s["indptr"], s["indices"],
                s["lengths"], query_indptr=s["query_indptr"], max_query=case["max_query"],
                max_length=case["max_length"], decay=case["decay"])
        return _plain_weights(s)
    if own:
        lengths, kept = attention.paged_evict(
            s["weights"], s["key_cache"], s["value_cache"], s["indptr"], s["indices"],
            s["lengths"], keep=case["keep"], recent=case["recent"], first=case["first"],
            max_length=case["max_length"], move_weights=case["move_weights"])
        out = {"lengths": lengths, "kept": kept, "key_cache": s["key_cache"],
               "value_cache": s["value_cache"]}
        return dict(out, weights=s["weights"]) if case["move_weights"] else out
    return _plain_evict(s)


# --------------------------------------------------------------------------- #
# what a pass cannot do without, and what it should give
# --------------------------------------------------------------------------- #
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "norm":
        rows, back = case["tokens"] * (case["heads"] + H), case["backward"]
        learned = (case["heads"] + H if case["per_head"] else 2) * D * DTYPES[
            case["weight"]].itemsize
        return {"bytes": (3 if back else 2) * rows * D * size + 8 * case["tokens"]
                + 4 * case["rotary"] + (2 if back else 1) * learned,
                "flops": rows * ((12 if back else 4) * D + 3 * case["rotary"])}
    sequences = _sequences(case)
    if case["op"] == "append":
        tokens = sum(new for new, _ in sequences)
        rows = tokens * (case["heads"] + H)
        return {"bytes": 2 * (rows + tokens * H) * D * size + 8 * case["sequences"] * 4,
                "flops": rows * (4 * D + 3 * case["rotary"])}
    if case["op"] == "weights":
        tokens = sum(new for new, _ in sequences)
        keys = sum(new + before for new, before in sequences)
        old = sum(before for _, before in sequences)
        # a new token sees what its sequence had, and the new ones up to itself
        pairs = sum(new * before + new * (new + 1) // 2 for new, before in sequences)
        return {"bytes": keys * H * (D * size + 4) + 4 * old * H
                + tokens * case["heads"] * (D * size + 4) + 8 * keys // case["page"],
                "flops": pairs * case["heads"] * (2 * D + 3)}
    K, R, F = case["keep"], case["recent"], case["first"]
    n, moved, looked = 0, 0.0, 0
    for _, length in sequences:
        n += min(K, length)
        if length > K:
            looked += length - R - F
            # the recent move down; of the others that stay, as many as stand past the front
            moved += R + (K - R - F) * (length - K) / max(1, length - R - F)
    row = 2 * D * size + (4 if case["move_weights"] else 0)
    return {"bytes": H * (2 * moved * row + 4 * looked + 4 * case["sequences"] * K)
            + 16 * case["sequences"], "flops": H * looked}


def exact(case, seed):
    """From the definitions, in 64 bits: pairs as complex numbers, gradients by automatic
    differentiation; each sequence's tokens as one list."""
    s = prepare(case, seed)
    dev = s["query"].device if "query" in s else s["lengths"].device

    def normed(x, weight, positions):
        y = x.double()
        y = y / (y.square().mean(-1, keepdim=True) + EPSILON).sqrt() * weight.double()
        n = case["rotary"]
        if case["layout"] == "half":
            z = torch.complex(y[..., :n // 2], y[..., n // 2:n])
        else:
            z = torch.complex(y[..., 0:n:2], y[..., 1:n:2])
        angle = positions.double()[:, None] * s["frequency"]
        z = z * torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]
        z = (torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else
             torch.view_as_real(z).flatten(-2))
        return torch.cat([z, y[..., n:]], -1)

    if case["op"] == "norm":
        found = []
        for name in ("query", "key"):
            x = s[name].double().requires_grad_()
            weight = s[name + "_weight"].double().requires_grad_()
            y = normed(x, weight, s["positions"])
            found.append(torch.autograd.grad(y, (x, weight), s["grad_" + name].double())
                         if case["backward"] else (y.detach(),))
        return tuple(x for pair in zip(*found) for x in pair)
    B, H, page = case["sequences"], case["kv_heads"], case["page"]
    rows, lengths = s["indptr"].tolist(), s["lengths"].tolist()

    def where(b, at):
        """Places of positions `at` of sequence b in the flattened cache."""
        return s["indices"][rows[b]:rows[b + 1]][at // page] * page + at % page

    if case["op"] == "evict":
        K, R, F = case["keep"], case["recent"], case["first"]
        names = ("key_cache", "value_cache") + (("weights",) if case["move_weights"] else ())
        out = {name: s[name].double() for name in names}
        kept = np.full((B, H, K), -1, dtype=np.int32)
        for b, length in enumerate(lengths):
            gone = max(0, length - K)
            mine = s["weights"].flatten(0, 1)[where(b, torch.arange(length, device=dev))]
            mine = mine.cpu().numpy()
            for h in range(H):
                to = np.arange(length - gone)
                if gone:
                    middle = np.arange(F, length - R)
                    heavy = middle[np.lexsort((middle, -mine[middle, h]))][:K - R - F]
                    stays = np.concatenate([np.arange(F), heavy])
                    holes = np.setdiff1d(np.arange(K - R), stays)
                    to[holes] = np.sort(stays[stays >= K - R])
                    to[K - R:] += gone
                kept[b, h, :to.size] = to
                source = where(b, torch.from_numpy(to).to(dev))
                target = where(b, torch.arange(to.size, device=dev))
                for name in names:
                    flat = out[name].flatten(0, 1)[:, h]
                    moved = flat[source]
                    out[name][target // page, target % page, h] = moved
        return dict(out, lengths=s["lengths"].clamp(max=K), kept=torch.from_numpy(kept).to(dev))
    ends = (s["query_indptr"] if s["query_indptr"] is not None else torch.arange(B + 1)).tolist()
    if case["op"] == "append":
        query, key = torch.empty_like(s["query"], dtype=torch.float64), s["key"]
        kc, vc = s["key_cache"].double(), s["value_cache"].double()
        for b in range(B):
            new = slice(ends[b], ends[b + 1])
            at = torch.arange(lengths[b] - (ends[b + 1] - ends[b]), lengths[b], device=dev)
            turn = case["offset"] + s["shift"][b] + at
            kc.flatten(0, 1)[where(b, at)] = normed(key[new], s["key_weight"], turn)
            vc.flatten(0, 1)[where(b, at)] = s["value"][new].double()
            query[new] = normed(s["query"][new], s["query_weight"], turn)
        return {"query": query, "key_cache": kc, "value_cache": vc}
    G, D = case["heads"] // H, case["dim"]
    weights = s["weights"].double()
    for b in range(B):
        new, n, length = slice(ends[b], ends[b + 1]), ends[b + 1] - ends[b], lengths[b]
        at = torch.arange(length, device=dev)
        places = where(b, at)
        last = length - n + torch.arange(n, device=dev)
        for h in range(H):
            heads = slice(h * G, (h + 1) * G)
            q, k = s["query"][new, heads].double(), s["key_cache"][:, :, h].flatten(0, 1)
            score = k[places].double() @ q.reshape(n * G, D).t().contiguous() * D ** -0.5
            prob = (score.reshape(length, n, G) - s["lse"][new, heads].double()).exp()
            got = (prob.sum(-1) * (at[:, None] <= last)).sum(-1)
            old = weights[places // page, places % page, h] * case["decay"]
            weights[places // page, places % page, h] = torch.where(at < length - n, old, 0) + got
    return weights