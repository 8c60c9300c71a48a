"""What the operators of attention over a paged cache are timed and compared on: rotary
positions with their gradient, appending keys and values to a paged cache with the rotation
applied on the way, and attention of a batch whose sequences share a long prefix.

A cache is an array of pages [pages, page, kv_heads, dim] for the keys and one for the values.
Which pages a sequence owns is a CSR structure, int64 ``indptr``/``indices`` as everywhere in
this repository; the pages of the shared prefix are a list of their own.

A case is {"name", "op", "dtype", "dim", ...}:
  op "rope"       tokens, heads, rotary (dims that are rotated), layout (half | interleaved),
                  scaling (none | linear | yarn), positions (the largest), backward
  op "append"     sequences, max_query (new tokens per sequence, 1 to that many), offset
                  (tokens before the sequence's first: the shared prefix), max_length (tokens
                  in a sequence's own pages, at most), page, heads (of the queries, rotated in
                  the same call), kv_heads, rotary, layout, scaling
  op "attention"  sequences, max_query, prefix (shared tokens), max_length, page, heads,
                  kv_heads
"""

import math
import random

import torch

own = False

BASE = 10000.0
TRAINED = 4096              # positions that the unscaled frequencies were made for
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # queries and keys of a decode step of 8 sequences, packed: one launch, latency alone
        {"name": "rope_decode", "op": "rope", "dtype": "bf16", "tokens": 8, "heads": 40,
         "dim": 128, "rotary": 128, "layout": "half", "scaling": "yarn", "positions": 131072,
         "backward": False},
        # a training step's queries and keys, forward
        {"name": "rope_train", "op": "rope", "dtype": "bf16", "tokens": 16384, "heads": 40,
         "dim": 128, "rotary": 128, "layout": "half", "scaling": "none", "positions": 4096,
         "backward": False},
        # its backward pass in single precision: part of an odd head size, an odd token count
        {"name": "rope_backward_part", "op": "rope", "dtype": "f32", "tokens": 8191, "heads": 25,
         "dim": 96, "rotary": 64, "layout": "interleaved", "scaling": "linear",
         "positions": 16384, "backward": True},
        # a decode step: one new token each behind a shared prompt
        {"name": "append_decode", "op": "append", "dtype": "bf16", "sequences": 32,
         "max_query": 1, "offset": 8192, "max_length": 1024, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "yarn"},
        # prompts of mixed lengths, small heads, interleaved pairs in half of each head
        {"name": "append_ragged", "op": "append", "dtype": "f16", "sequences": 17,
         "max_query": 700, "offset": 0, "max_length": 1500, "page": 24, "heads": 12,
         "kv_heads": 4, "dim": 64, "rotary": 32, "layout": "interleaved", "scaling": "none"},
        # the long prompt that a batch will share, filled in at once
        {"name": "append_prompt", "op": "append", "dtype": "bf16", "sequences": 1,
         "max_query": 16384, "offset": 0, "max_length": 16384, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "yarn"},
        # a handful of sequences behind a short prompt: latency alone
        {"name": "attention_small", "op": "attention", "dtype": "f16", "sequences": 4,
         "max_query": 1, "prefix": 500, "max_length": 60, "page": 16, "heads": 8, "kv_heads": 2,
         "dim": 64},
        # an ordinary decode step behind a system prompt
        {"name": "attention_decode", "op": "attention", "dtype": "bf16", "sequences": 32,
         "max_query": 1, "prefix": 8192, "max_length": 1024, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128},
        # several samples of one very long document
        {"name": "attention_long", "op": "attention", "dtype": "bf16", "sequences": 8,
         "max_query": 1, "prefix": 131072, "max_length": 256, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128},
        # many sequences with answers of their own behind a long prompt: prefix bound by the
        # matrix cores, answers by memory
        {"name": "attention_batch", "op": "attention", "dtype": "bf16", "sequences": 128,
         "max_query": 1, "prefix": 32768, "max_length": 2048, "page": 16, "heads": 64,
         "kv_heads": 8, "dim": 128},
        # draft tokens checked a few at a time, one shared kv head, odd head and page sizes
        {"name": "attention_drafts", "op": "attention", "dtype": "f16", "sequences": 24,
         "max_query": 7, "prefix": 6001, "max_length": 900, "page": 24, "heads": 16,
         "kv_heads": 1, "dim": 96},
        # chunks of new prompts behind the shared one: matrix products throughout
        {"name": "attention_chunks", "op": "attention", "dtype": "bf16", "sequences": 2,
         "max_query": 512, "prefix": 16384, "max_length": 700, "page": 64, "heads": 16,
         "kv_heads": 4, "dim": 128},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _rotary(rng, dim):
    return rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 2])


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    if op == "rope":
        heads = _between(rng, 1, 48)
        tokens = _between(rng, 1, min(16384, 16384 * 40 * 128 // (2 * heads * dim)))
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "tokens": tokens,
                "heads": heads, "dim": dim, "rotary": _rotary(rng, dim),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "yarn"]),
                "positions": _between(rng, tokens, 131072), "backward": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([g for g in (1, 2, 3, 4, 8, 16) if g * kv_heads <= 64])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "dim": dim,
            "heads": group * kv_heads, "kv_heads": kv_heads,
            "page": rng.choice([16, 16, 24, 32, 64, 128])}
    if op == "append":
        sequences = _between(rng, 1, 128)
        most = min(16384, 16384 * 48 * 128 // (2 * (case["heads"] + 2 * kv_heads) * dim))
        max_query = _between(rng, 1, max(1, most // sequences)) if rng.random() < 0.6 else 1
        return dict(case, dtype=rng.choice(["bf16", "f16", "f32"]), sequences=sequences,
                    max_query=max_query, offset=rng.choice([0, _between(rng, 1, 65536)]),
                    max_length=max_query + _between(rng, 1, 1024), rotary=_rotary(rng, dim),
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn"]))
    sequences = _between(rng, 1, 128)
    max_query = 1 if rng.random() < 0.6 else _between(rng, 2, max(3, 512 // sequences))
    rows = sequences * max_query * case["heads"]
    key = kv_heads * dim
    prefix = _between(rng, 1, min(131072, 1.3e11 / (4 * rows * dim), 2.6e8 / rows, 1.3e8 / key))
    most = min(2048, 2.6e8 / rows, 2 * (1.6e8 - prefix * key) / (sequences * key))
    return dict(case, sequences=sequences, max_query=max_query, prefix=prefix,
                max_length=max_query + _between(rng, 1, max(2, most)))


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
    """Of each sequence: its new tokens, and those already in its own pages when they come
    (some have none); in an order that has nothing to do with the seed."""
    before = _spread(case["sequences"], 0, case["max_length"] - case["max_query"])
    random.Random(1).shuffle(before)
    return list(zip(_spread(case["sequences"], 1, case["max_query"]), before))


def _indptr(counts, dev):
    return torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(dev)


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    state = {"case": case}
    if "rotary" in case:
        f, state["magnitude"] = _frequency(case, dev)
        state["frequency"] = f
        last = case["positions"] if case["op"] == "rope" else case["offset"] + case["max_length"]
        angle = torch.arange(last, dtype=torch.float64, device=dev)[:, None] * f
        # the tables that the plain form looks its rotations up in
        state["cos"] = (angle.cos() * state["magnitude"]).float()
        state["sin"] = (angle.sin() * state["magnitude"]).float()
    if case["op"] == "rope":
        n = case["tokens"]
        # a decode step's tokens stand anywhere; a longer call's follow one another, sequence
        # after sequence
        state["positions"] = torch.randint(case["positions"], (n if n <= 64 else 1,),
                                           generator=g, device=dev)
        if n > 64:
            state["positions"] = (state["positions"] + torch.arange(n, device=dev)) % (
                case["positions"])
        state["x"] = normal(n, case["heads"], case["dim"])
        return state
    rng = random.Random(seed)
    page, B = case["page"], case["sequences"]
    sequences = _sequences(case)
    rng.shuffle(sequences)
    counts = [new for new, _ in sequences]
    lengths = [new + before for new, before in sequences]
    owned = [-(-n // page) + i % 2 for i, n in enumerate(lengths)]   # every other holds a spare
    shared = -(-case.get("prefix", 0) // page)
    pages = shared + sum(owned) + 3
    order = torch.randperm(pages, generator=g, device=dev)
    state.update(
        prefix=order[:shared], indices=order[shared:shared + sum(owned)],
        indptr=_indptr(owned, dev), lengths=torch.tensor(lengths, dtype=torch.int64, device=dev),
        query_indptr=_indptr(counts, dev) if case["max_query"] > 1 else None,
        key_cache=normal(pages, page, case["kv_heads"], case["dim"]),
        value_cache=normal(pages, page, case["kv_heads"], case["dim"]),
        query=normal(sum(counts), case["heads"], case["dim"]))
    if case["op"] == "append":
        state["key"] = normal(sum(counts), case["kv_heads"], case["dim"])
        state["value"] = normal(sum(counts), case["kv_heads"], case["dim"])
    return state


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def _rotate(x, cos, sin, layout, back=False):
    """Pairs of x[..., :rotary] turned by their angles, in 32 bits; the rest as it is."""
    n = 2 * cos.shape[-1]
    cos, sin = cos[:, None], -sin[:, None] if back else sin[:, None]
    y = x.float()
    if layout == "half":
        a, b = y[..., :n // 2], y[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., n:]], -1).to(x.dtype)


def _tokens(s):
    """Each new token's sequence, its place among the sequence's new ones, and its position in
    the sequence's own pages."""
    n = s["query"].shape[0]
    at = torch.arange(n, device=s["query"].device)
    if s["query_indptr"] is None:
        return at, torch.zeros_like(at), s["lengths"] - 1
    seq = torch.searchsorted(s["query_indptr"], at, right=True) - 1
    nth = at - s["query_indptr"][seq]
    return seq, nth, (s["lengths"] - s["query_indptr"].diff())[seq] + nth


def _plain_append(s):
    case = s["case"]
    seq, _, position = _tokens(s)
    cos, sin = s["cos"][case["offset"] + position], s["sin"][case["offset"] + position]
    page = s["indices"][s["indptr"][seq] + position // case["page"]]
    slot = position % case["page"]
    s["key_cache"][page, slot] = _rotate(s["key"], cos, sin, case["layout"])
    s["value_cache"][page, slot] = s["value"]
    return _rotate(s["query"], cos, sin, case["layout"])


def _plain_attention(s):
    case = s["case"]
    B, H, D = case["sequences"], case["kv_heads"], case["dim"]
    G, n, L = case["heads"] // H, case["max_query"], case["max_length"]
    T = s["query"].shape[0]
    seq, nth, position = _tokens(s)
    q = s["query"].float().reshape(T, H, G, D) / math.sqrt(D)
    # the shared prefix: [H, T G, prefix]
    k = s["key_cache"][s["prefix"]].reshape(-1, H, D)[:case["prefix"]].float().transpose(0, 1)
    v = s["value_cache"][s["prefix"]].reshape(-1, H, D)[:case["prefix"]].float().transpose(0, 1)
    score = q.transpose(0, 1).reshape(H, T * G, D) @ k.transpose(1, 2)
    # each sequence's own pages, padded to the longest: [B, H, n G, L]
    at = torch.arange(L, device=q.device)
    listed_at = (s["indptr"][:-1, None] + at // case["page"]).clamp(max=s["indices"].numel() - 1)
    page = s["indices"][listed_at]
    k2 = s["key_cache"][page, at % case["page"]].float().transpose(1, 2)
    v2 = s["value_cache"][page, at % case["page"]].float().transpose(1, 2)
    padded = q.new_zeros(B, n, H, G, D)
    padded[seq, nth] = q
    seen = torch.full((B, n), -1, dtype=torch.int64, device=q.device)
    seen[seq, nth] = position
    score2 = padded.transpose(1, 2).reshape(B, H, n * G, D) @ k2.transpose(2, 3)
    hidden = (at > seen[:, :, None]).repeat_interleave(G, 1)[:, None]
    score2.masked_fill_(hidden, -math.inf)
    # one softmax over both
    score2 = score2.reshape(B, H, n, G, L)
    top2 = score2.amax(-1)[seq, :, nth].transpose(0, 1).reshape(H, T * G)
    top = torch.maximum(score.amax(-1), top2)
    score = (score - top[..., None]).exp_()
    back = q.new_zeros(B, n, H, G)
    back[seq, nth] = top.reshape(H, T, G).transpose(0, 1)
    score2 = (score2 - back.transpose(1, 2)[..., None]).exp_()
    total = score.sum(-1) + score2.sum(-1)[seq, :, nth].transpose(0, 1).reshape(H, T * G)
    out2 = (score2.reshape(B, H, n * G, L) @ v2).reshape(B, H, n, G, D)[seq, :, nth]
    out = score @ v + out2.transpose(0, 1).reshape(H, T * G, D)
    out = (out / total[..., None]).reshape(H, T, G, D).transpose(0, 1).reshape(T, H * G, D)
    lse = (top + total.log()).reshape(H, T, G).transpose(0, 1).reshape(T, H * G)
    return out.to(s["query"].dtype), lse


def run(state):
    s, case = state, state["case"]
    if own:
        from tilegen_amd import attention
    if case["op"] == "rope":
        if own:
            turn = attention.rope_backward if case["backward"] else attention.rope
            return turn(s["x"], s["positions"], s["frequency"], layout=case["layout"],
                        magnitude=s["magnitude"])
        return _rotate(s["x"], s["cos"][s["positions"]], s["sin"][s["positions"]],
                       case["layout"], case["backward"])
    if case["op"] == "append":
        if own:
            query = attention.paged_append(
                s["key"], s["value"], s["key_cache"], s["value_cache"], s["indptr"],
                s["indices"], s["lengths"], s["frequency"], query=s["query"],
                query_indptr=s["query_indptr"], offset=case["offset"], layout=case["layout"],
                magnitude=s["magnitude"])
        else:
            query = _plain_append(s)
        return {"query": query, "key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    if own:
        out, lse = attention.prefix_attention(
            s["query"], s["key_cache"], s["value_cache"], s["prefix"], case["prefix"],
            s["indptr"], s["indices"], s["lengths"], query_indptr=s["query_indptr"],
            max_query=case["max_query"], max_length=case["max_length"], return_lse=True)
    else:
        out, lse = _plain_attention(s)
    return {"out": out, "lse": lse}


# --------------------------------------------------------------------------- #
# what a pass cannot do without, and what it should give
# --------------------------------------------------------------------------- #
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + 8 * case["tokens"] + 4 * case["rotary"],
                "flops": 3 * n * case["rotary"]}
    sequences = _sequences(case)
    tokens = sum(new for new, _ in sequences)
    if case["op"] == "append":
        rows = tokens * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * rows * case["dim"] * size + 8 * case["sequences"] * 3,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    # each key is read once for all the queries that see it
    keys = case["prefix"] + sum(new + before for new, before in sequences)
    # a new token sees the prefix, what its sequence had, and the new ones up to itself
    pairs = sum(new * (case["prefix"] + before) + new * (new + 1) // 2
                for new, before in sequences)
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size
            + 2 * tokens * case["heads"] * case["dim"] * size + 4 * tokens * case["heads"]
            + 8 * keys // case["page"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def exact(case, seed):
    """From the definitions, in 64 bits: pairs as complex numbers; each sequence's keys and
    values as one list."""
    s = prepare(case, seed)
    dev = s["frequency"].device if "frequency" in s else s["query"].device

    def turned(x, positions, sign):
        n = case["rotary"]
        y = x.double().clone()
        z = (torch.complex(y[..., :n // 2], y[..., n // 2:n]) if case["layout"] == "half" else
             torch.view_as_complex(y[..., :n].unflatten(-1, (n // 2, 2)).contiguous()))
        angle = sign * positions.double()[:, None] * s["frequency"]
        z = z * torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]
        y[..., :n] = (torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else
                      torch.view_as_real(z).flatten(-2))
        return y

    if case["op"] == "rope":
        return turned(s["x"], s["positions"], -1 if case["backward"] else 1)
    B, page = case["sequences"], case["page"]
    ends = (s["query_indptr"] if s["query_indptr"] is not None else torch.arange(B + 1)).tolist()
    rows, lengths = s["indptr"].tolist(), s["lengths"].tolist()
    if case["op"] == "append":
        query, key = torch.empty_like(s["query"], dtype=torch.float64), s["key"]
        kc, vc = s["key_cache"].double(), s["value_cache"].double()
        for b in range(B):
            new = slice(ends[b], ends[b + 1])
            at = torch.arange(lengths[b] - (ends[b + 1] - ends[b]), lengths[b], device=dev)
            where = s["indices"][rows[b]:rows[b + 1]][at // page] * page + at % page
            kc.flatten(0, 1)[where] = turned(key[new], case["offset"] + at, 1)
            vc.flatten(0, 1)[where] = s["value"][new].double()
            query[new] = turned(s["query"][new], case["offset"] + at, 1)
        return {"query": query, "key_cache": kc, "value_cache": vc}
    H, D, P = case["kv_heads"], case["dim"], case["prefix"]
    G = case["heads"] // H
    out = torch.empty_like(s["query"], dtype=torch.float64)
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device=dev)
    for h in range(H):
        shared = [c[s["prefix"], :, h].flatten(0, 1)[:P].double()
                  for c in (s["key_cache"], s["value_cache"])]
        for b in range(B):
            new = slice(ends[b], ends[b + 1])
            n = ends[b + 1] - ends[b]
            mine = s["indices"][rows[b]:rows[b + 1]]
            k, v = (torch.cat([p, c[mine, :, h].flatten(0, 1)[:lengths[b]].double()])
                    for p, c in zip(shared, (s["key_cache"], s["value_cache"])))
            q = s["query"][new, h * G:(h + 1) * G].double()
            score = q.reshape(n * G, D).matmul(k.t().contiguous()).reshape(n, G, -1) * D ** -0.5
            at = torch.arange(k.shape[0], device=dev)
            last = P + lengths[b] - n + torch.arange(n, device=dev)
            score.masked_fill_((at > last[:, None])[:, None], -math.inf)
            lse[new, h * G:(h + 1) * G] = torch.logsumexp(score, -1)
            out[new, h * G:(h + 1) * G] = torch.softmax(score, -1).reshape(n * G, -1).matmul(
                v).reshape(n, G, D)
    return {"out": out, "lse": lse}
