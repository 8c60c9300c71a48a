"""Rotary positions, the append to a paged cache and attention behind a shared prefix
(tilegen_amd.attention) against the formulas in 64 bits.

Tolerances come from the arithmetic.  u is the unit roundoff of the operands' type (2^-8
bfloat16, 2^-11 float16, 2^-24 float32): a value rounded to it once is off by u of itself.

rope: a value is a cos - b sin in 32 bits, rounded once.  The angle's fraction of a turn is
exact to 2^-25 of itself, so the cosine and sine to about 2 pi 2^-26 + 2^-24; with the two
products and the sum: |error| <= u |y| + 2^-21 (|a| + |b|) magnitude.

attention: probabilities (up to 2^8 times the largest one's, see narrow.h) are rounded to the
operands' type (relative u, and half the smallest float16, 2^-25, where they are below its
normal range), the result once more; scores are off by at most dim 2^-23 scale sum |q k|, in the
numerator and in the denominator; sums of n terms by n 2^-24 of the sum of magnitudes."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tilegen_amd import attention as at

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


# --------------------------------------------------------------------------- #
# rope
# --------------------------------------------------------------------------- #
def _turned(x, positions, frequency, layout, magnitude=1.0, sign=1):
    """The formula in 64 bits, on the CPU."""
    y = x.detach().cpu().double().clone()
    f = frequency.cpu().double().numpy()
    p = positions.cpu().numpy().astype(np.float64)
    angle = torch.from_numpy(sign * p[:, None] * f)
    c, s = magnitude * torch.cos(angle)[:, None], magnitude * torch.sin(angle)[:, None]
    n = f.size
    first = slice(0, n) if layout == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if layout == "half" else slice(1, 2 * n, 2)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size = y.abs()
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * magnitude
    return y, size


def _check_turned(got, x, positions, frequency, layout, magnitude=1.0, sign=1):
    want, size = _turned(x, positions, frequency, layout, magnitude, sign)
    off = (got.cpu().double() - want).abs()
    tiny = 2.0 ** -25 if got.dtype == F16 else 0.0
    bound = U[got.dtype] * want.abs() + 2.0 ** -21 * size + tiny
    bound *= 1 + 2.0 ** -6
    assert (off <= bound).all(), float((off - bound).max())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [
    (1, 1, 2, 2), (3, 2, 7, 4), (5, 3, 64, 64), (4, 5, 80, 38), (2, 40, 128, 128), (9, 1, 96, 0),
    (1, 7, 256, 62), (4099, 2, 96, 64), (3, 1, 1024, 1024), (70, 3, 17, 16), (4, 300, 24, 24)])
def test_rope(hip_ready, layout, dtype, tokens, heads, dim, rotary):
    g = _gen(tokens + dim)
    x = _normal(g, tokens, heads, dim, dtype=dtype)
    positions = torch.randint(-1000, 10 ** 7, (tokens,), generator=g, device="cuda")
    frequency, magnitude = at.rope_frequencies(rotary, scaling="yarn", factor=8, trained=2048)
    keep = x.clone()
    y = at.rope(x, positions, frequency, layout=layout, magnitude=magnitude)
    _check_turned(y, x, positions, frequency, layout, magnitude)
    d = at.rope_backward(x, positions, frequency, layout=layout, magnitude=magnitude)
    _check_turned(d, x, positions, frequency, layout, magnitude, sign=-1)
    assert torch.equal(x, keep)
    assert at.rope(x, positions, frequency, layout=layout, magnitude=magnitude, out=x) is x
    assert torch.equal(x, y)    # in place: the same bits


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_on_views(hip_ready, layout):
    """Heads of a packed projection, odd offsets, transposed tokens and heads."""
    g = _gen(1)
    frequency, _ = at.rope_frequencies(48)
    packed = _normal(g, 11, 9, 65, dtype=BF16)
    positions = torch.arange(11, device="cuda") * 12345
    out = torch.zeros(9, 11, 77, device="cuda", dtype=BF16)
    x, y = packed[:, 2:7, 1:65], out[1:6, :, 5:69].transpose(0, 1)
    assert at.rope(x, positions, frequency, layout=layout, out=y) is y
    _check_turned(y, x, positions, frequency, layout)
    y.zero_()
    assert not out.any()        # nothing beside the view was written
    wide = x[:, :1].expand(11, 4, 64)
    _check_turned(at.rope(wide, positions, frequency, layout=layout), wide, positions, frequency,
                  layout)
    before = packed.clone()
    at.rope(x, positions, frequency, layout=layout, out=x)
    before[:, 2:7, 1:65] = x
    assert torch.equal(packed, before)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient(hip_ready, layout):
    """The gradient through autograd is the transposed map, and matches differences of the
    formula (linear in x: exact but for rounding)."""
    g = _gen(2)
    frequency, magnitude = at.rope_frequencies(24, scaling="yarn", factor=4, trained=512)
    positions = torch.tensor([0, 1, 77, 100000, 5], device="cuda")
    x = _normal(g, 5, 3, 30, dtype=F32).requires_grad_()
    w = _normal(g, 5, 3, 30, dtype=F32)
    y = at.rope(x, positions, frequency, layout=layout, magnitude=magnitude)
    (y * w).sum().backward()
    _check_turned(x.grad, w, positions, frequency, layout, magnitude, sign=-1)
    for t, h, i in ((0, 0, 0), (2, 1, 13), (3, 2, 23), (4, 0, 29), (3, 0, 12)):
        plus, minus = x.detach().clone(), x.detach().clone()
        plus[t, h, i] += 0.5
        minus[t, h, i] -= 0.5
        difference = sum(s * float((_turned(v, positions, frequency, layout, magnitude)[0]
                                    * w.cpu().double()).sum())
                         for s, v in ((1, plus), (-1, minus)))
        # the two steps are exact to 2^-23 of x, the gradient to the bound above
        assert abs(float(x.grad[t, h, i]) - difference) <= 2.0 ** -18 * magnitude
    x.grad = None
    at.rope(x, positions, frequency, layout=layout).sum().backward()   # a broadcast gradient
    _check_turned(x.grad, torch.ones_like(w), positions, frequency, layout, sign=-1)


# --------------------------------------------------------------------------- #
# a batch with its cache
# --------------------------------------------------------------------------- #
class Batch:
    """Random pages for a prefix and for each sequence, one page to spare on odd ones; cache
    slots that no token has hold NaN."""

    def __init__(self, dtype, heads, kv_heads, dim, page, prefix, lengths, counts, seed=0,
                 spare=True):
        g = self.g = _gen(seed)
        self.dtype, self.heads, self.kv_heads, self.dim = dtype, heads, kv_heads, dim
        self.page, self.prefix_length = page, prefix
        self.lengths_host, self.counts = list(lengths), list(counts)
        owned = [-(-max(0, n) // page) + (i % 2 if spare else 0) for i, n in enumerate(lengths)]
        shared = -(-prefix // page)
        self.pages = shared + sum(owned) + 2
        order = torch.randperm(self.pages, generator=g, device="cuda")
        self.prefix = order[:shared].contiguous()
        self.indices = order[shared:shared + sum(owned)].contiguous()
        self.indptr = self._ends(owned)
        self.lengths = torch.tensor(self.lengths_host, dtype=torch.int64, device="cuda")
        self.ends = self._ends(self.counts)
        self.ends_host = [0] + np.cumsum(self.counts).tolist()
        shape = (self.pages, page, kv_heads, dim)
        self.kc = torch.full(shape, math.nan, device="cuda", dtype=dtype)
        self.vc = torch.full(shape, math.nan, device="cuda", dtype=dtype)
        tokens = sum(self.counts)
        self.query = _normal(g, tokens, heads, dim, dtype=dtype)
        self.key = _normal(g, tokens, kv_heads, dim, dtype=dtype)
        self.value = _normal(g, tokens, kv_heads, dim, dtype=dtype)

    @staticmethod
    def _ends(n):
        return torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int64, device="cuda")

    def places(self, b=None):
        """(page, slot) of the prefix's keys, or of sequence b's."""
        if b is None:
            pages, n = self.prefix, self.prefix_length
        else:
            pages = self.indices[int(self.indptr[b]):int(self.indptr[b + 1])]
            n = min(max(0, self.lengths_host[b]), pages.numel() * self.page)
        at_ = torch.arange(n, device="cuda")
        return pages[at_ // self.page], at_ % self.page

    def fill(self):
        for b in [None] + list(range(len(self.counts))):
            page, slot = self.places(b)
            for c in (self.kc, self.vc):
                c[page, slot] = _normal(self.g, page.numel(), self.kv_heads, self.dim,
                                        dtype=self.dtype)
        return self

    def attend(self, **more):
        args = dict(query_indptr=self.ends, max_query=max(self.counts + [1]),
                    max_length=max(self.lengths_host + [1]), return_lse=True)
        if all(n == 1 for n in self.counts):
            args["query_indptr"] = None
        args.update(more)
        return at.prefix_attention(self.query, self.kc, self.vc, self.prefix,
                                   self.prefix_length, self.indptr, self.indices, self.lengths,
                                   **args)

    def want(self, scale=None):
        """(out, lse, bound of |out|'s error, bound of lse's), 64 bits, on the CPU."""
        scale = self.dim ** -0.5 if scale is None else scale
        G = self.heads // self.kv_heads
        T = sum(self.counts)
        u = U[self.dtype]
        out = torch.zeros(T, self.heads, self.dim, dtype=torch.float64)
        lse = torch.full((T, self.heads), -math.inf, dtype=torch.float64)
        eo, el = torch.zeros_like(out), torch.zeros_like(lse)
        kp, vp = (c[self.places()].cpu().double() for c in (self.kc, self.vc))
        q = self.query.cpu().double()
        for b, n in enumerate(self.counts):
            ko, vo = (c[self.places(b)].cpu().double() for c in (self.kc, self.vc))
            for j in range(n):
                t = self.ends_host[b] + j
                see = min(max(0, self.lengths_host[b] - n + j + 1), ko.shape[0])
                k, v = torch.cat([kp, ko[:see]]), torch.cat([vp, vo[:see]])
                if not len(k):
                    continue
                for h in range(self.heads):
                    kh, vh = k[:, h // G], v[:, h // G]
                    s = scale * (kh @ q[t, h])
                    es = self.dim * 2.0 ** -23 * scale * float((kh.abs() @ q[t, h].abs()).max())
                    p = torch.softmax(s, 0)
                    size = p @ vh.abs()
                    out[t, h], lse[t, h] = p @ vh, torch.logsumexp(s, 0)
                    el[t, h] = es + 2.0 ** -22 * (len(k) ** 0.5 + 4 + abs(float(lse[t, h])))
                    eo[t, h] = (u * (size + out[t, h].abs()) + (2 * es + 2.0 ** -22 * len(k) ** 0.5)
                                * size)
                    if self.dtype == F16:
                        eo[t, h] += 2.0 ** -25 * (vh.abs().sum(0) + 1)
        return out, lse, eo * (1 + 2.0 ** -6), el

    def check(self, got, scale=None):
        out, lse, eo, el = self.want(scale)
        o, e = got[0].cpu().double(), got[1].cpu().double()
        assert torch.isfinite(o).all()
        assert ((o - out).abs() <= eo).all(), float(((o - out).abs() / (eo + 1e-30)).max())
        empty = lse == -math.inf
        assert torch.equal(e == -math.inf, empty) and not o[empty].any()
        assert ((e - lse)[~empty].abs() <= el[~empty]).all(), float(
            ((e - lse).abs() / el)[~empty].max())


ATTENTION = [
    # heads, kv_heads, dim, page, prefix, lengths, counts
    (1, 1, 8, 1, 1, [1], [1]),
    (1, 1, 64, 16, 0, [1], [1]),
    (4, 1, 40, 7, 33, [5, 0, 64], [1, 1, 1]),
    (8, 2, 64, 16, 500, [60, 1, 17, 33], [1, 1, 1, 1]),
    (6, 2, 80, 24, 31, [100, 24, 25], [1, 1, 1]),
    (16, 1, 96, 24, 129, [40, 7, 90], [7, 1, 3]),
    (5, 5, 72, 3, 64, [12, 30], [2, 9]),
    (20, 1, 128, 16, 1000, [300, 2], [1, 2]),
    (8, 8, 128, 32, 0, [200, 31, 0, 129], [1, 1, 1, 1]),
    (3, 1, 136, 5, 77, [20, 41], [5, 0]),
    (4, 2, 192, 16, 65, [70, 3], [33, 3]),
    (2, 1, 256, 64, 700, [90, 200, 1], [17, 40, 1]),
    (32, 8, 128, 16, 2100, [40] * 9, [1] * 9),
    (16, 4, 128, 64, 600, [190, 77], [150, 70]),
    (12, 4, 64, 16, 300, [64, 200, 33, 1], [64, 130, 20, 1]),
    (8, 1, 64, 1, 40, [9, 4], [4, 4]),
    # wide over many tiles: pages of 8-key groups, of neither 8 nor 16, heads of all sizes
    (16, 1, 96, 24, 1501, [40, 7, 90], [7, 1, 3]),
    (9, 1, 64, 7, 1100, [600, 31], [9, 4]),
    (40, 2, 128, 20, 1300, [1, 140], [1, 1]),
    (24, 1, 256, 16, 1217, [700, 80], [1, 3]),
    (17, 1, 200, 8, 900, [33], [1]),
    # more workgroups than the chip holds: the longest sequences first, and more than are ranked
    (8, 8, 64, 16, 40, [(37 * i) % 90 for i in range(80)], [1] * 80),
    (2, 2, 40, 16, 0, [(11 * i) % 50 for i in range(300)], [1] * 300),
    # fewer tokens than new ones: the first see the prefix alone, or nothing
    (4, 2, 64, 16, 20, [2, 0], [5, 3]),
    (4, 2, 64, 16, 0, [2, 0], [5, 3]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,prefix,lengths,counts", ATTENTION)
def test_prefix_attention(hip_ready, dtype, heads, kv_heads, dim, page, prefix, lengths, counts):
    b = Batch(dtype, heads, kv_heads, dim, page, prefix, lengths, counts, seed=dim).fill()
    got = b.attend()
    b.check(got)
    # launch bounds below the truth are slower, not wrong; a run repeats bit for bit
    b.check(b.attend(max_query=1, max_length=1))
    again = b.attend()
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_hidden_keys_of_few_rows(hip_ready, dtype):
    """As below, where a sequence's new tokens fill less than one narrow tile."""
    b = Batch(dtype, 2, 1, 96, 24, 70, [33, 64], [4, 8], seed=14).fill()
    clean = b.want()
    page, slot = b.places(0)
    b.vc[page[-1], slot[-1]] = math.inf
    b.kc[page[-2], slot[-2]] = math.nan         # seen by tokens 2 and 3
    page, slot = b.places(1)
    b.vc[page[-4], slot[-4], 0, 95] = math.nan  # seen by the last four
    got, lse = (x.cpu().double() for x in b.attend())
    fine = torch.ones(12, 2, 96, dtype=torch.bool)
    fine[2:4] = False
    fine[8:, :, 95] = False
    assert ((got - clean[0]).abs() <= clean[2])[fine].all()
    assert torch.isnan(got[~fine]).all()
    rows = torch.tensor([i not in (2, 3) for i in range(12)])
    assert ((lse - clean[1]).abs() <= clean[3])[rows].all()


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (40, 1, 128, 8),
                                                     (20, 1, 96, 7), (17, 1, 256, 24)])
def test_lost_pages_inside_a_long_prefix(hip_ready, heads, kv_heads, dim, page):
    """Pages of the prefix that do not exist count as hidden, wherever their tiles stand, and what
    the first page of the cache holds does not matter."""
    b = Batch(BF16, heads, kv_heads, dim, page, 1200, [30, 9], [1, 1], seed=dim).fill()
    n = -(-1200 // page)
    lost = [0, 3, n // 2, n // 2 + 1, n - 2]
    whole = b.prefix.clone()
    b.prefix[lost] = torch.tensor([-1, b.pages, 2 ** 40, -2 ** 40, b.pages + 1], device="cuda")
    used = bool((whole == 0).any() or (b.indices == 0).any())
    if not used:
        b.kc[0], b.vc[0] = math.nan, math.inf
    got = b.attend()
    # the same keys as a prefix without those pages
    keep = torch.ones(n, dtype=torch.bool)
    keep[lost] = False
    short = Batch(BF16, heads, kv_heads, dim, page, 1200, [30, 9], [1, 1], seed=dim)
    short.kc, short.vc, short.query = b.kc, b.vc, b.query
    short.indptr, short.indices = b.indptr, b.indices
    short.prefix = whole[keep.cuda()].contiguous()
    short.prefix_length = 1200 - page * len(lost)
    short.check(got)
    short.check(short.attend())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_hidden_keys_hold_anything(hip_ready, dtype):
    """Infinities and NaN in keys and values that a row does not see, among them those of later
    tokens of its own sequence, change nothing; those that it sees do."""
    b = Batch(dtype, 4, 2, 64, 16, 40, [35, 9, 50], [6, 3, 20], seed=3).fill()
    page, slot = b.places(0)
    b.kc[page[-1], slot[-1]] = math.inf         # seen by the sequence's last token alone
    b.vc[page[-1], slot[-1]] = math.nan
    page, slot = b.places(2)
    b.vc[page[-8], slot[-8], 0, 3] = -math.inf  # by its last eight, one element, one kv head
    got, lse = b.attend()
    clean = Batch(dtype, 4, 2, 64, 16, 40, [35, 9, 50], [6, 3, 20], seed=3).fill()
    out, lse_want, eo, el = clean.want()
    tainted = torch.zeros(out.shape, dtype=torch.bool)
    tainted[5] = True
    tainted[21:, :2, 3] = True
    got = got.cpu().double()
    assert ((got - out).abs() <= eo)[~tainted].all()
    assert torch.isnan(got[5]).all()
    assert (got[21:, :2, 3] == -math.inf).all()
    rows = torch.arange(29) != 5
    assert ((lse.cpu().double() - lse_want).abs() <= el)[rows].all()


def test_scores_at_the_ends_of_the_range(hip_ready):
    """Keys of -inf leave rows with no weight (0 and -inf, as a row without keys), the lowest
    finite values do not; scores that climb through the whole range keep their softmax."""
    b = Batch(BF16, 2, 1, 64, 16, 96, [40], [1], seed=4).fill()
    b.query.fill_(1.0)
    b.kc[b.places()] = -math.inf
    b.kc[b.places(0)] = -math.inf
    out, lse = b.attend()
    assert not out.any() and (lse == -math.inf).all()
    page, slot = b.places(0)
    lowest = torch.finfo(BF16).min
    b.kc[page[7], slot[7]] = 0.0
    b.kc[page[7], slot[7], :, 0] = lowest       # one key with a finite score, far below all
    out, lse = b.attend()
    assert torch.equal(out[0], b.vc[page[7], slot[7], 0].expand(2, 64))
    climb = Batch(F16, 3, 1, 64, 16, 700, [300], [1], seed=5).fill()
    climb.query.fill_(1.0)
    for place, lo, hi in ((climb.places(), -60.0, 20.0), (climb.places(0), 20.0, 90.0)):
        n = place[0].numel()
        climb.kc[place] = torch.linspace(lo, hi, n, device="cuda").to(F16)[:, None, None]
    climb.check(climb.attend())
    falling = Batch(BF16, 3, 1, 64, 16, 700, [300], [1], seed=6).fill()
    falling.query.fill_(1.0)
    page, slot = falling.places()
    falling.kc[page, slot] = torch.linspace(90, -60, 700, device="cuda").to(BF16)[:, None, None]
    falling.check(falling.attend())


def test_pages_and_rows_that_point_nowhere(hip_ready):
    """Pages outside the cache count as hidden, row pointers outside the list as its ends; a
    length past a sequence's pages as their end; negative lengths as none."""
    b = Batch(BF16, 4, 2, 64, 16, 64, [64, 64, 20, 7], [1, 1, 1, 1], seed=7, spare=False).fill()
    b.prefix[1] = b.pages + 5
    b.indices[1], b.indices[6] = -1, 2 ** 40
    kc, vc = b.kc, b.vc
    got, lse = b.attend()
    # the same without those keys: all that is left stands on a prefix or a sequence of its own
    for i, n in enumerate([64, 64, 20, 7]):
        pages = torch.cat([b.prefix, b.indices[int(b.indptr[i]):int(b.indptr[i + 1])]]).cpu()
        keys = torch.arange(64 + n)
        page = pages[keys // 16]
        fine = (page >= 0) & (page < b.pages)
        k, v = (c.cpu()[page[fine], (keys % 16)[fine]].double() for c in (kc, vc))
        for h in range(4):
            s = k[:, h // 2] @ b.query[i, h].cpu().double() / 8
            o = torch.softmax(s, 0) @ v[:, h // 2]
            # the largest value is under 2^3: u of sums and results, twice
            assert (got[i, h].cpu().double() - o).abs().max() <= 2.0 ** -5
            assert abs(float(lse[i, h]) - float(torch.logsumexp(s, 0))) <= 2.0 ** -16
    c = Batch(BF16, 4, 2, 64, 16, 0, [64, 64], [1, 1], seed=8, spare=False).fill()
    c.lengths[0] = 1000         # 64 keys listed
    full = c.attend(max_length=1000)
    c.check(full)
    c.lengths[1] = -5
    out, lse = c.attend()
    assert torch.equal(out[0], full[0][0]) and not out[1].any() and (lse[1] == -math.inf).all()
    c.lengths[1] = 64
    c.indptr[2] = 10 ** 12
    assert torch.equal(c.attend()[0], full[0])
    c.indptr[1] = -3            # sequence 0 has no pages, sequence 1 all of them
    out, lse = c.attend()
    assert not out[0].any() and (lse[0] == -math.inf).all() and torch.isfinite(out[1]).all()


def test_strides_and_given_outputs(hip_ready):
    """Caches as [pages, kv_heads, page, dim] and as halves of one array, queries of a packed
    projection at odd offsets, an output with gaps."""
    b = Batch(F16, 6, 2, 72, 16, 50, [40, 9], [2, 1], seed=9).fill()
    want = b.attend()
    b.check(want)
    both = torch.zeros(b.pages, 2, b.kv_heads, 16, 74, device="cuda", dtype=F16)
    k, v = both[:, 0, :, :, 1:73].transpose(1, 2), both[:, 1, :, :, 2:74].transpose(1, 2)
    k.copy_(b.kc), v.copy_(b.vc)
    packed = torch.zeros(3, 9, 73, device="cuda", dtype=F16)
    packed[:, 1:7, 1:] = b.query
    room = torch.zeros(3, 8, 80, device="cuda", dtype=F16)
    out = room[:, 1:7, 3:75]
    b.kc, b.vc, b.query = k, v, packed[:, 1:7, 1:]
    got = b.attend(out=out)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    out.zero_()
    assert not room.any()
    b.check(b.attend(scale=0.5), scale=0.5)


@pytest.mark.parametrize("heads", [4, 16])     # narrow and wide
def test_offsets_past_32_bits(hip_ready, heads):
    """Pages whose elements lie past 2^31, and 2^32 bytes, of the cache."""
    pages, page, dim = 70000, 64, 256
    kc = torch.empty(pages, page, 2, dim, device="cuda", dtype=BF16)      # 2.3 G elements
    vc = torch.empty(pages, page, 2, dim, device="cuda", dtype=BF16)
    b = Batch(BF16, heads, 2, dim, page, 100, [90, 3], [3, 2], seed=10)
    b.prefix += pages - b.pages
    b.indices += pages - b.pages
    b.kc, b.vc, b.pages = kc, vc, pages
    b.fill()
    frequency, _ = at.rope_frequencies(dim)
    at.paged_append(b.key, b.value, kc, vc, b.indptr, b.indices, b.lengths, frequency,
                    query_indptr=b.ends, offset=100)
    for i in range(2):
        at_, n = b.places(i), b.counts[i]
        rows = slice(b.ends_host[i], b.ends_host[i + 1])
        position = 100 + torch.arange(b.lengths_host[i] - n, b.lengths_host[i])
        _check_turned(kc[at_][-n:], b.key[rows], position, frequency, "half")
        assert torch.equal(vc[at_][-n:], b.value[rows])
    b.check(b.attend())


# --------------------------------------------------------------------------- #
# append
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page,lengths,counts", [
    (1, 1, 64, 64, 16, [1], [1]),
    (0, 2, 128, 128, 16, [5, 33, 16], [1, 1, 1]),
    (12, 4, 80, 38, 7, [30, 8, 50, 9], [30, 1, 0, 9]),
    (3, 1, 17, 16, 1, [4, 9], [3, 2]),
    (8, 8, 64, 0, 24, [200, 77], [150, 3]),
    (4, 1, 256, 62, 64, [4200], [4200]),
    (2, 2, 96, 96, 16, [3] * 150, [2] * 150),
])
def test_paged_append(hip_ready, layout, dtype, heads, kv_heads, dim, rotary, page, lengths,
                      counts):
    b = Batch(dtype, max(heads, 1), kv_heads, dim, page, 0, lengths, counts, seed=dim + page)
    frequency, magnitude = at.rope_frequencies(rotary, scaling="linear", factor=2)
    offset = 4097
    kc, vc = b.kc.clone(), b.vc.clone()
    query = at.paged_append(
        b.key, b.value, kc, vc, b.indptr, b.indices, b.lengths, frequency if rotary else None,
        query=b.query if heads else None,
        query_indptr=None if set(counts) == {1} else b.ends, offset=offset, layout=layout)
    assert (query is None) == (heads == 0)
    for i, n in enumerate(counts):
        rows = slice(b.ends_host[i], b.ends_host[i + 1])
        where = tuple(x[lengths[i] - n:] for x in b.places(i))
        position = offset + torch.arange(lengths[i] - n, lengths[i])
        _check_turned(kc[where], b.key[rows], position, frequency, layout)
        assert torch.equal(vc[where], b.value[rows])
        if heads:
            _check_turned(query[rows], b.query[rows], position, frequency, layout)
        kc[where] = math.nan
        vc[where] = math.nan
    assert torch.isnan(kc).all() and torch.isnan(vc).all()      # nothing else was written


def test_paged_append_leaves_out_what_has_no_place(hip_ready):
    b = Batch(BF16, 2, 1, 64, 16, 0, [40, 20, 17], [3, 18, 2], seed=11, spare=False)
    frequency, _ = at.rope_frequencies(64)
    b.lengths[1] = 50           # two pages hold 32: positions 32 .. 49 have none
    b.indices[0] = -1           # not in use by the new tokens of sequence 0
    b.indices[2] = b.pages      # positions 37 .. 39 of sequence 0
    b.ends[3] = 22              # the last token belongs to no sequence
    kc, vc = b.kc.clone(), b.vc.clone()
    query = at.paged_append(b.key, b.value, kc, vc, b.indptr, b.indices, b.lengths, frequency,
                            query=b.query, query_indptr=b.ends)
    written = ~torch.isnan(kc).flatten(1).any(1)
    slots = (~torch.isnan(kc).any(-1).any(-1)).sum()
    assert int(slots) == 1 and int(written.sum()) == 0       # sequence 2's one token
    page = b.indices[int(b.indptr[2]) + 1]
    assert torch.equal(vc[page, 0, 0], b.value[21, 0])
    assert not query[22].any() and query[:22].any(-1).all()
    out, lse = at.prefix_attention(b.query, kc, vc, b.prefix, 0, b.indptr, b.indices, b.lengths,
                                   query_indptr=b.ends, max_query=18, max_length=50,
                                   return_lse=True)
    assert not out[22].any() and (lse[22] == -math.inf).all()


# --------------------------------------------------------------------------- #
# streams, graphs, refusals
# --------------------------------------------------------------------------- #
def _step(b, frequency):
    q = at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query, query_indptr=b.ends, offset=b.prefix_length)
    return at.prefix_attention(q, b.kc, b.vc, b.prefix, b.prefix_length, b.indptr, b.indices,
                               b.lengths, query_indptr=b.ends, max_query=2, max_length=80)


def test_other_streams(hip_ready):
    """Two streams at work at once, each with a batch of its own."""
    frequency, _ = at.rope_frequencies(64)
    batches = [Batch(BF16, 8, 2, 64, 16, 3000, [70, 33], [2, 1], seed=s).fill() for s in (1, 2)]
    want = [_step(b, frequency) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(20):
        for s, b, to in zip(streams, batches, got):
            with torch.cuda.stream(s):
                to.append(_step(b, frequency))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_in_a_graph(hip_ready):
    """A captured step replayed with longer sequences each time, eager work between."""
    frequency, _ = at.rope_frequencies(64)
    b = Batch(BF16, 8, 2, 64, 16, 100, [80, 80], [2, 1], seed=12).fill()
    eager = Batch(BF16, 8, 2, 64, 16, 100, [80, 80], [2, 1], seed=12).fill()
    b.lengths -= 60
    eager.lengths -= 60
    _step(b, frequency)
    _step(eager, frequency)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(b, frequency)
    for i in range(5):
        b.lengths += 9
        eager.lengths += 9
        b.query.normal_(generator=_gen(i))
        eager.query.copy_(b.query)
        graph.replay()
        want = _step(eager, frequency)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    assert torch.equal(b.kc.nan_to_num(), eager.kc.nan_to_num())


def test_nothing_to_do(hip_ready):
    frequency, _ = at.rope_frequencies(64)
    empty = torch.empty(0, 4, 64, device="cuda", dtype=BF16)
    none = torch.empty(0, device="cuda", dtype=torch.int64)
    assert at.rope(empty, none, frequency).shape == (0, 4, 64)
    cache = torch.zeros(2, 16, 4, 64, device="cuda", dtype=BF16)
    ends = torch.zeros(1, device="cuda", dtype=torch.int64)
    q = at.paged_append(empty, empty, cache, cache.clone(), ends, none, none, frequency,
                        query=empty)
    assert q.shape == (0, 4, 64)
    out, lse = at.prefix_attention(empty, cache, cache, none, 0, ends, none, none, max_length=1,
                                   return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    # a cache without pages: no row sees a key
    b = Batch(BF16, 4, 2, 64, 16, 0, [5, 5], [1, 1])
    b.kc, b.vc = b.kc[:0], b.vc[:0]
    out, lse = b.attend()
    assert not out.any() and (lse == -math.inf).all()


def test_refusals(hip_ready):
    frequency, _ = at.rope_frequencies(64)
    x = torch.zeros(4, 2, 64, device="cuda", dtype=BF16)
    pos = torch.arange(4, device="cuda")
    for args, more in [
            ((x.cpu(), pos, frequency), {}), ((x.double(), pos, frequency), {}),
            ((x[0], pos, frequency), {}), ((x, pos[:3], frequency), {}),
            ((x, pos.int(), frequency), {}), ((x, pos, frequency.float()), {}),
            ((x, pos.cpu(), frequency), {}), ((x, pos, frequency), dict(layout="both")),
            ((x[..., :32], pos, frequency), {}),                # rotary past the head
            ((x.transpose(1, 2), pos, frequency[:1]), {}),      # heads not contiguous
            ((x, pos, frequency), dict(out=x[:3])), ((x, pos, frequency), dict(out=x.float())),
            ((x, pos, frequency), dict(out=x[:, :1].expand(4, 2, 64))),
            ((x[:, :, :62], pos, frequency[:8]), dict(out=x[:, :, 2:])),    # overlaps
            ((torch.zeros(1, 1, 1025, device="cuda"), pos[:1], frequency), {}),
            ((x.float().requires_grad_(), pos, frequency), dict(out=x.float()))]:
        with pytest.raises(ValueError):
            at.rope(*args, **more)
    b = Batch(BF16, 4, 2, 64, 16, 32, [20, 9], [1, 1]).fill()

    def append(**change):
        a = dict(key=b.key, value=b.value, key_cache=b.kc, value_cache=b.vc, indptr=b.indptr,
                 indices=b.indices, lengths=b.lengths, frequency=frequency, query=b.query)
        a.update(change)
        return at.paged_append(**a)

    def attend(**change):
        a = dict(query=b.query, key_cache=b.kc, value_cache=b.vc, prefix=b.prefix,
                 prefix_length=32, indptr=b.indptr, indices=b.indices, lengths=b.lengths,
                 max_length=20)
        a.update(change)
        return at.prefix_attention(**a)

    append(), attend()
    for change in [dict(key=b.key[:1]), dict(value=b.value.half()), dict(value_cache=b.vc[:1]),
                   dict(key_cache=b.kc[..., :32]), dict(indptr=b.indptr[:2]),
                   dict(lengths=b.lengths[:1]), dict(lengths=b.lengths.int()),
                   dict(indices=b.indices.float()), dict(query=b.query[:1]),
                   dict(query_out=b.query[:1]), dict(query=None, query_out=b.query),
                   dict(query_indptr=b.indptr[:2]), dict(layout="neither"),
                   dict(key_cache=b.kc[:1].expand(b.kc.shape)),
                   dict(frequency=torch.zeros(40, device="cuda", dtype=torch.float64))]:
        with pytest.raises(ValueError):
            append(**change)
    for change in [dict(query=b.query.float()), dict(query=b.query[..., :32]),
                   dict(query=b.query[:, :3]), dict(key_cache=b.kc.half()),
                   dict(value_cache=b.vc[:, :8]), dict(prefix=b.prefix[:1]),
                   dict(prefix_length=33), dict(prefix_length=-1), dict(max_length=-1),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                   dict(scale=math.inf), dict(indptr=b.indptr[1:]), dict(lengths=b.lengths[:1]),
                   dict(out=b.query[:1]), dict(out=b.query[:, :1].expand(2, 4, 64)),
                   dict(query_indptr=b.indptr.int()), dict(max_length=2 ** 40),
                   dict(query=torch.zeros(2, 4, 12, device="cuda", dtype=BF16),
                        key_cache=b.kc[..., :12], value_cache=b.vc[..., :12]),
                   dict(query=torch.zeros(2, 4, 264, device="cuda", dtype=BF16),
                        key_cache=torch.zeros(9, 16, 2, 264, device="cuda", dtype=BF16),
                        value_cache=torch.zeros(9, 16, 2, 264, device="cuda", dtype=BF16))]:
        with pytest.raises(ValueError):
            attend(**change)
    append(), attend()


def test_the_sparse_kernels_give_the_same(hip_ready):
    """The same attention through this package's own SDDMM and SpMM, in 64 bits: the page
    table as a CSR pattern over cache slots, one row a token."""
    import scipy.sparse as sp

    from tilegen_amd.schedules import TUNED
    from tilegen_amd.variant import Variant
    b = Batch(BF16, 1, 1, 64, 16, 90, [50, 3, 0, 16], [1, 1, 1, 1], seed=13).fill()
    out, _ = b.attend()
    rows, cols = [], []
    for i in range(4):
        for page, slot in (b.places(), b.places(i)):
            cols.append((page * 16 + slot).cpu().numpy())
            rows.append(np.full(page.numel(), i))
    rows, cols = np.concatenate(rows), np.concatenate(cols)
    A = sp.csr_matrix((np.full(rows.size, 1 / 8), (rows, cols)), shape=(4, b.pages * 16))
    A.sort_indices()
    K, V = (np.nan_to_num(c.cpu().double().numpy()).reshape(-1, 64) for c in (b.kc, b.vc))
    Q = b.query[:, 0].cpu().double().numpy()
    S = Variant("sddmm", TUNED["c5"]).run(A, U=Q, V=K)
    P = A.copy()
    for i in range(4):
        s = S[A.indptr[i]:A.indptr[i + 1]]
        e = np.exp(s - s.max())
        P.data[A.indptr[i]:A.indptr[i + 1]] = e / e.sum()
    want = Variant("spmm", TUNED["c4"]).run(P, B=V)
    bound = b.want()[2][:, 0].numpy()
    assert (np.abs(out[:, 0].cpu().double().numpy() - want) <= bound).all()


def test_paged_decode(hip_ready):
    """The decode loop of tilegen_amd.paged_decode against attention over its unrotated inputs in
    64 bits.  The calls round rotated queries and keys to bfloat16: scores are off by 2 u scale
    sum |q k| (rotated) more than in the tests above."""
    from tilegen_amd import paged_decode
    heads, kv_heads, dim, prompt = 4, 2, 64, 90
    r = paged_decode.run(sequences=3, prompt=prompt, steps=20, heads=heads, kv_heads=kv_heads,
                         dim=dim, page=16, start=9, seed=3, keep=True)
    f, magnitude, counts, u = r["frequency"], r["magnitude"], r["counts"], U[BF16]

    def turn(x, position):
        return _turned(x, torch.tensor(position), f, "half", magnitude)[0]

    keys = [turn(r["prompt"][0], list(range(prompt)))] * 3
    values = [r["prompt"][1].cpu().double()] * 3
    lengths = [0, 0, 0]
    for call, (q, k, v, out) in enumerate(r["calls"]):
        n = counts if call == 0 else [1, 1, 1]
        row = 0
        for b in range(3):
            mine = slice(row, row + n[b])
            at_ = [prompt + lengths[b] + j for j in range(n[b])]
            keys[b] = torch.cat([keys[b], turn(k[mine], at_)])
            values[b] = torch.cat([values[b], v[mine].cpu().double()])
            qs = turn(q[mine], at_)
            lengths[b] += n[b]
            for j in range(n[b]):
                see = prompt + lengths[b] - n[b] + j + 1
                for h in range(heads):
                    kh, vh = keys[b][:see, h // 2], values[b][:see, h // 2]
                    p = torch.softmax(kh @ qs[j, h] / 8, 0)
                    es = float((kh.abs() @ qs[j, h].abs()).max()) / 8 * (2 * u + dim * 2.0 ** -23)
                    size = p @ vh.abs()
                    bound = 2 * u * size + (math.exp(2 * es) - 1) * size
                    off = (out[row + j, h].cpu().double() - p @ vh).abs()
                    assert (off <= bound).all(), (call, b, j, h)
            row += n[b]
    assert len(r["calls"]) == 21 and lengths == [n + 20 for n in counts]


# --------------------------------------------------------------------------- #
# workgroups of 128 rows: bounds above what the batch has make small batches take them
# --------------------------------------------------------------------------- #
WIDE = dict(max_query=10 ** 6, max_length=1100)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,prefix,lengths,counts", [
    # heads, kv_heads, dim, page, prefix, lengths, counts: 49 rows of a kv head or more
    (16, 1, 40, 7, 33, [40, 7, 90, 0], [7, 1, 3, 0]),
    (16, 4, 64, 16, 129, [300, 20, 64], [40, 9, 3]),
    (7, 1, 64, 1, 70, [66, 130, 5], [3, 64, 5]),
    (12, 4, 80, 24, 0, [200, 33, 1], [130, 20, 1]),
    (50, 1, 96, 16, 500, [65, 0, 40], [1, 1, 1]),
    (24, 2, 96, 3, 64, [140, 2], [9, 2]),
    (16, 4, 128, 64, 600, [190, 77], [150, 70]),
    (60, 1, 128, 16, 63, [63, 64, 129], [1, 1, 1]),
    (25, 1, 128, 20, 1, [300, 2], [1, 2]),
    (32, 1, 200, 8, 90, [33, 70], [1, 2]),
    (20, 1, 256, 5, 65, [120, 31], [5, 4]),
    (14, 2, 256, 64, 200, [90, 200, 1], [17, 40, 1]),
    # fewer tokens than new ones, and no key at all
    (32, 1, 64, 16, 20, [2, 0], [5, 3]),
    (32, 1, 128, 16, 0, [2, 0], [5, 3]),
])
def test_wide(hip_ready, dtype, heads, kv_heads, dim, page, prefix, lengths, counts):
    b = Batch(dtype, heads, kv_heads, dim, page, prefix, lengths, counts, seed=dim + 1).fill()
    got = b.attend(**WIDE)
    b.check(got)
    b.check(b.attend(max_query=10 ** 6, max_length=30000))
    again = b.attend(**WIDE)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,prefix,lengths,counts", [
    (8, 2, 64, 16, 2000, [(13 * i) % 70 for i in range(40)], [1] * 40),
    (6, 2, 96, 24, 1900, [(13 * i) % 70 for i in range(48)], [1] * 48),
    (8, 8, 40, 7, 700, [30] * 20, [1 + i % 3 for i in range(20)]),
    (8, 4, 256, 16, 1100, [(7 * i) % 40 for i in range(20)], [1] * 20),
])
def test_wide_prefix_and_narrow_own_pages(hip_ready, dtype, heads, kv_heads, dim, page, prefix,
                                          lengths, counts):
    b = Batch(dtype, heads, kv_heads, dim, page, prefix, lengths, counts, seed=dim + 2).fill()
    b.check(b.attend())


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(100, 2, 64, 16), (40, 1, 128, 8),
                                                     (52, 1, 96, 7), (50, 1, 256, 24)])
def test_wide_with_lost_pages(hip_ready, heads, kv_heads, dim, page):
    b = Batch(BF16, heads, kv_heads, dim, page, 700, [200, 9], [1, 1], seed=dim + 3,
              spare=False).fill()
    n = -(-700 // page)
    lost, own = [0, 3, n // 2, n // 2 + 1, n - 2], 1
    whole, mine = b.prefix.clone(), b.indices.clone()
    b.prefix[lost] = torch.tensor([-1, b.pages, 2 ** 40, -2 ** 40, b.pages + 1], device="cuda")
    b.indices[own] = -2 ** 33
    if not bool((whole == 0).any() or (mine == 0).any()):
        b.kc[0], b.vc[0] = math.nan, math.inf
    got = b.attend(**WIDE)
    keep = torch.ones(n, dtype=torch.bool)
    keep[lost] = False
    short = Batch(BF16, heads, kv_heads, dim, page, 700, [200 - page, 9], [1, 1], seed=0,
                  spare=False)
    short.kc, short.vc, short.query = b.kc, b.vc, b.query
    short.indices = torch.cat([mine[:own], mine[own + 1:]])
    short.prefix = whole[keep.cuda()].contiguous()
    short.prefix_length = 700 - page * len(lost)
    short.check(got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_wide_with_hidden_keys_that_hold_anything(hip_ready, dtype, dim):
    shape = (dtype, 4, 2, dim, 16, 40, [35, 9, 90], [6, 3, 60])
    b = Batch(*shape, seed=3).fill()
    page, slot = b.places(0)
    b.kc[page[-1], slot[-1]] = math.inf         # seen by the sequence's last token alone
    b.vc[page[-1], slot[-1]] = math.nan
    page, slot = b.places(2)
    b.vc[page[-8], slot[-8], 0, 3] = -math.inf  # by its last eight, one element, one kv head
    got, lse = b.attend(**WIDE)
    out, lse_want, eo, el = Batch(*shape, seed=3).fill().want()
    tainted = torch.zeros(out.shape, dtype=torch.bool)
    tainted[5] = True
    tainted[61:, :2, 3] = True
    got = got.cpu().double()
    assert ((got - out).abs() <= eo)[~tainted].all()
    assert torch.isnan(got[5]).all()
    assert (got[61:, :2, 3] == -math.inf).all()
    rows = torch.arange(69) != 5
    assert ((lse.cpu().double() - lse_want).abs() <= el)[rows].all()


def test_wide_at_the_ends_of_the_range(hip_ready):
    b = Batch(BF16, 50, 1, 64, 16, 96, [40], [1], seed=4).fill()
    b.query.fill_(1.0)
    b.kc[b.places()] = -math.inf
    b.kc[b.places(0)] = -math.inf
    out, lse = b.attend(**WIDE)
    assert not out.any() and (lse == -math.inf).all()
    page, slot = b.places(0)
    b.kc[page[7], slot[7]] = 0.0
    b.kc[page[7], slot[7], :, 0] = torch.finfo(BF16).min    # one finite score, far below all
    out, lse = b.attend(**WIDE)
    assert torch.equal(out[0], b.vc[page[7], slot[7], 0].expand(50, 64))
    for dtype, first, last in ((F16, -60.0, 90.0), (BF16, 90.0, -60.0)):
        for dim in (64, 128):
            c = Batch(dtype, 50, 1, dim, 16, 700, [300], [1], seed=5).fill()
            c.query.fill_(1.0)
            for place, lo, hi in ((c.places(), first, first + (last - first) / 2),
                                  (c.places(0), first + (last - first) / 2, last)):
                n = place[0].numel()
                c.kc[place] = torch.linspace(lo, hi, n, device="cuda").to(dtype)[:, None, None]
            c.check(c.attend(**WIDE))


@pytest.mark.parametrize("page,dim", [(16, 72), (10, 72), (16, 128), (6, 256)])
def test_wide_with_other_strides(hip_ready, page, dim):
    """Caches that are halves of one array with heads before slots, at odd offsets."""
    b = Batch(F16, 60, 2, dim, page, 150, [140, 9], [2, 1], seed=9).fill()
    want = b.attend(**WIDE)
    b.check(want)
    both = torch.zeros(b.pages, 2, b.kv_heads, page, dim + 2, device="cuda", dtype=F16)
    k = both[:, 0, :, :, 1:dim + 1].transpose(1, 2)
    v = both[:, 1, :, :, 2:].transpose(1, 2)
    k.copy_(b.kc), v.copy_(b.vc)
    packed = torch.zeros(3, 63, dim + 1, device="cuda", dtype=F16)
    packed[:, 1:61, 1:] = b.query
    b.query = packed[:, 1:61, 1:]
    kc, vc = b.kc, b.vc
    for b.kc, b.vc in ((k, v), (kc, v), (k, vc)):      # alike strides, and not
        got = b.attend(**WIDE)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_wide_past_32_bits(hip_ready):
    """test_offsets_past_32_bits for workgroups of 128 rows, pages of 64 and of 60 keys."""
    pages, dim = 70000, 256
    pool = torch.empty(2, pages * 64 * 2 * dim, device="cuda", dtype=BF16)
    for page in (64, 60):
        kc, vc = (x[:pages * page * 2 * dim].view(pages, page, 2, dim) for x in pool)
        b = Batch(BF16, 64, 2, dim, page, 100, [90, 3], [3, 2], seed=10)
        b.prefix += pages - b.pages
        b.indices += pages - b.pages
        b.kc, b.vc, b.pages = kc, vc, pages
        b.fill()
        frequency, _ = at.rope_frequencies(dim)
        at.paged_append(b.key, b.value, kc, vc, b.indptr, b.indices, b.lengths, frequency,
                        query_indptr=b.ends, offset=100)
        b.check(b.attend(**WIDE))


def test_gradients_that_do_not_exist_are_refused(hip_ready):
    frequency, _ = at.rope_frequencies(64)
    b = Batch(BF16, 4, 2, 64, 16, 32, [20, 9], [1, 1], seed=12).fill()
    query = b.query.clone().requires_grad_()
    for call in (lambda: at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths,
                                         frequency, query=query),
                 lambda: at.prefix_attention(query, b.kc, b.vc, b.prefix, 32, b.indptr, b.indices,
                                             b.lengths, max_length=20)):
        with pytest.raises(ValueError, match="backward"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("prefix", [32, 900])      # in one launch, and in parts
def test_attention_over_its_own_query(hip_ready, prefix):
    """out may be the query, and may share no other memory with the operands."""
    b = Batch(BF16, 4, 2, 64, 16, prefix, [40, 9], [30, 1], seed=13).fill()
    want = b.attend()[0]
    packed = torch.zeros(31, 6, 64, device="cuda", dtype=BF16)
    packed[:, :4] = b.query
    b.query = packed[:, :4]
    for out in (packed[:, 1:5], b.kc.view(-1, 4, 64)[:31]):
        with pytest.raises(ValueError, match="overlaps"):
            b.attend(out=out)
    assert torch.equal(b.attend(out=b.query)[0], want) and not packed[:, 4:].any()


# --------------------------------------------------------------------------- #
# row pointers, numbers and memory that calls must not mix up
# --------------------------------------------------------------------------- #
def _bits(t):
    return t.view(torch.int16)


@pytest.mark.parametrize("first,last", [(1, 3), (1, 2), (2, 3)])
@pytest.mark.parametrize("prefix", [32, 900])      # in one launch, and in parts
def test_a_block_of_row_pointers(hip_ready, prefix, first, last):
    """Sequences first .. last of a batch by slices of its row pointers: the tokens before and
    after theirs belong to no sequence."""
    lengths, counts = [40, 9, 33], [3, 1, 5]
    b = Batch(BF16, 4, 2, 64, 16, prefix, lengths, counts, seed=15).fill()
    out, lse, eo, el = b.want()
    indptr, ends = b.indptr[first:last + 1], b.ends[first:last + 1]
    rows = torch.zeros(9, dtype=torch.bool)
    rows[b.ends_host[first]:b.ends_host[last]] = True
    given = torch.full_like(b.query, math.nan)
    spoil = torch.full((1 << 22,), math.nan, device="cuda")     # what fresh memory may hold
    del spoil
    got, got_lse = at.prefix_attention(
        b.query, b.kc, b.vc, b.prefix, prefix, indptr, b.indices, b.lengths[first:last],
        query_indptr=ends, max_query=5, max_length=40, out=given, return_lse=True)
    got, got_lse = got.cpu().double(), got_lse.cpu().double()
    assert ((got - out).abs() <= eo)[rows].all() and ((got_lse - lse).abs() <= el)[rows].all()
    assert not got[~rows].any() and (got_lse[~rows] == -math.inf).all()
    frequency, _ = at.rope_frequencies(64)
    kc, vc = b.kc.clone(), b.vc.clone()
    query = at.paged_append(b.key, b.value, kc, vc, indptr, b.indices, b.lengths[first:last],
                            frequency, query=b.query, query_indptr=ends)
    assert not query[~rows.cuda()].any() and query[rows.cuda()].any(-1).all()
    for i in range(first, last):
        new = tuple(x[lengths[i] - counts[i]:] for x in b.places(i))
        mine = slice(b.ends_host[i], b.ends_host[i + 1])
        assert torch.equal(vc[new], b.value[mine])
        _check_turned(kc[new], b.key[mine],
                      torch.arange(lengths[i] - counts[i], lengths[i]), frequency, "half")
        kc[new], vc[new] = b.kc[new], b.vc[new]
    assert torch.equal(_bits(kc), _bits(b.kc)) and torch.equal(_bits(vc), _bits(b.vc))


def test_slices_of_one_array(hip_ready):
    """Outputs that lie between their operands without a byte in common."""
    b = Batch(BF16, 4, 4, 64, 16, 32, [20, 9], [1, 1], seed=12).fill()
    frequency, _ = at.rope_frequencies(64)
    pos = torch.arange(2, device="cuda")
    packed = torch.zeros(2, 13, 64, device="cuda", dtype=BF16)
    packed[:, :4] = b.query
    want = at.rope(b.query, pos, frequency)
    at.rope(packed[:, :4], pos, frequency, out=packed[:, 4:8])
    assert torch.equal(packed[:, 4:8], want)
    want = b.attend()[0]
    b.query = packed[:, :4]
    b.attend(out=packed[:, 8:12])
    assert torch.equal(packed[:, 8:12], want) and not packed[:, 12:].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 16), (128, 7), (256, 24)])
@pytest.mark.parametrize("wide", [False, True])
def test_an_infinity_at_the_end_of_the_prefix(hip_ready, dtype, dim, page, wide):
    """Places past the prefix's last key, in the tile that it ends in, have no part in the sums."""
    for prefix in (100, 900):
        b = Batch(dtype, 60 if wide else 2, 1, dim, page, prefix, [20, 9], [1, 1], seed=16).fill()
        out, lse, eo, el = b.want()
        pages, slots = b.places()
        b.vc[pages[-1], slots[-1], 0, 3] = math.inf
        b.vc[pages[-1], slots[-1], 0, 5] = -math.inf
        got, got_lse = (x.cpu().double() for x in b.attend(
            **dict(WIDE, query_indptr=b.ends) if wide else {}))
        assert (got[:, :, 3] == math.inf).all() and (got[:, :, 5] == -math.inf).all()
        got[:, :, [3, 5]] = out[:, :, [3, 5]]
        assert ((got - out).abs() <= eo).all() and ((got_lse - lse).abs() <= el).all()


@pytest.mark.parametrize("more", [{}, dict(max_length=1100, max_query=10 ** 6)])
def test_scores_that_are_not_numbers(hip_ready, more):
    """A NaN among a row's scores makes its result NaN, also where no other score is there to
    give a maximum: to the row, to a wave, to a part."""
    for heads in (2, 60):
        # all of a row's keys; those of one wave's tile; in one launch, and in parts
        for prefix, bad in ((0, 0), (96, 96), (900, 900), (900, 32), (128, 32)):
            b = Batch(BF16, heads, 1, 64, 16, prefix, [1, 0], [1, 1], seed=17).fill()
            page, slot = b.places()
            b.kc[page[:bad], slot[:bad]] = math.nan
            if bad == prefix:
                b.kc[b.places(0)] = math.nan
            out, lse = b.attend(**more)
            assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all(), (heads, prefix, bad)
            if bad:
                assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
            else:
                assert not out[1].any() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("heads,first", [(2, 128), (50, 128), (50, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_climb_by_their_last_bit(hip_ready, dtype, heads, first):
    """Past 2^27 neighbouring scores are 16 apart.  Probabilities are powers of two, which are
    exact, and the results, under 1, rounded once (twice u for the sums' order)."""
    b = Batch(dtype, heads, 1, 64, 16, 0, [640], [1], seed=18).fill()
    page, slot = b.places(0)
    b.query.zero_()
    b.query[..., 0], b.query[..., 1] = 32768.0, 16.0
    b.kc[page, slot] = 0.0
    b.kc[page, slot, 0, 0] = 4096.0
    b.kc[page[:first], slot[:first], 0, 1] = 1.0
    b.kc[page[first:], slot[first:], 0, 1] = 2.0
    out, lse = b.attend(scale=math.log(2.0), max_length=640 if heads < 50 else 30000,
                        max_query=10 ** 6, query_indptr=b.ends)
    weight = torch.ones(640, dtype=torch.float64)
    weight[:first] = 2.0 ** -16
    want = weight @ b.vc[page, slot, 0].cpu().double() / weight.sum()
    off = (out[0].cpu().double() - want).abs()
    assert (off <= 2.0 ** -7).all(), float(off.max())


def test_many_small_probabilities(hip_ready):
    """131071 keys 18 nats under one other, in one part for many rows: 0.2% of the weight.  Each
    probability is off by at most 2^-25 of the 2^7 that the largest is (float16's smallest number
    is 2^-24); 32-bit sums over 16 keys at a time, and the rounded result, by u."""
    n, kv = 131072, 64
    kc = torch.zeros(n // 64, 64, kv, 8, device="cuda", dtype=F16)
    vc = torch.ones(n // 64, 64, kv, 8, device="cuda", dtype=F16)
    kc[..., 0] = -18.0
    kc[0, 0, :, 0] = vc[0, 0] = 0.0
    q = torch.zeros(1024, kv, 8, device="cuda", dtype=F16)
    q[..., 0] = 1.0
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    zero = torch.zeros(2, dtype=torch.int64, device="cuda")
    small = (n - 1) * math.exp(-18)
    want = small / (1 + small)
    for tokens in (1024, 1):
        ends = torch.tensor([0, tokens], device="cuda")
        out = at.prefix_attention(q[:tokens], kc, vc, torch.arange(n // 64, device="cuda"), n, zero,
                                  none, zero[:1], query_indptr=ends, max_query=tokens,
                                  max_length=0, scale=1.0)
        off = float((out.double() - want).abs().max())
        assert off <= 2 * U[F16] * want + n * 2.0 ** -32, (tokens, off, want)


def test_second_derivatives_of_rope(hip_ready):
    """The gradient of a loss of the gradient.  Two turns after one another: the bound above
    twice, the first's error turned with the rest; |a| + |b| stays under 2^4."""
    g = _gen(21)
    frequency, magnitude = at.rope_frequencies(24, scaling="yarn", factor=4, trained=512)
    positions = torch.tensor([0, 1, 77, 100000, 5], device="cuda")
    x = _normal(g, 5, 3, 30, dtype=F32).requires_grad_()
    w = _normal(g, 5, 3, 30, dtype=F32)
    y = at.rope(x, positions, frequency, magnitude=magnitude)
    first, = torch.autograd.grad((y * y).sum() / 2, x, create_graph=True)
    assert first.requires_grad
    second, = torch.autograd.grad((first * w).sum(), x)
    # d/dx w . R'(R x) = R' R w
    there = _turned(w, positions, frequency, "half", magnitude)[0]
    want = _turned(there, positions, frequency, "half", magnitude, -1)[0]
    assert ((second.cpu().double() - want).abs() <= 2.0 ** -15 * magnitude ** 2).all()
    grad = w.clone().requires_grad_()
    back = at.rope_backward(grad, positions, frequency, magnitude=magnitude)
    back.backward(x.detach())
    _check_turned(grad.grad, x, positions, frequency, "half", magnitude)


def test_tangents_of_rope(hip_ready):
    """Forward mode: the tangent of the result is the map of x's."""
    import torch.autograd.forward_ad as fw
    g = _gen(22)
    frequency, _ = at.rope_frequencies(16)
    positions = torch.arange(4, device="cuda")
    x, t = (_normal(g, 4, 2, 20, dtype=F32) for _ in range(2))
    for turn, sign in ((at.rope, 1), (at.rope_backward, -1)):
        with fw.dual_level():
            y = fw.unpack_dual(turn(fw.make_dual(x, t), positions, frequency))
            assert y.tangent is not None
            _check_turned(y.primal, x, positions, frequency, "half", sign=sign)
            _check_turned(y.tangent, t, positions, frequency, "half", sign=sign)


def test_lost_derivatives(hip_ready):
    """Operands whose derivatives a call would drop, outputs that have a history of their own, and
    tangents of calls without derivatives are refused."""
    import torch.autograd.forward_ad as fw
    frequency, _ = at.rope_frequencies(64)
    b = Batch(BF16, 4, 2, 64, 16, 32, [20, 9], [1, 1], seed=12).fill()
    pos = torch.arange(2, device="cuda")
    needs = frequency.clone().requires_grad_()
    grad_out = torch.empty_like(b.query).requires_grad_()

    def append(**change):
        return at.paged_append(**dict(dict(
            key=b.key, value=b.value, key_cache=b.kc, value_cache=b.vc, indptr=b.indptr,
            indices=b.indices, lengths=b.lengths, frequency=frequency, query=b.query), **change))

    def attend(**change):
        return at.prefix_attention(**dict(dict(
            query=b.query, key_cache=b.kc, value_cache=b.vc, prefix=b.prefix, prefix_length=32,
            indptr=b.indptr, indices=b.indices, lengths=b.lengths, max_length=20), **change))

    calls = [lambda: at.rope(b.query, pos, needs), lambda: at.rope_backward(b.query, pos, needs),
             lambda: append(frequency=needs),
             lambda: at.rope(b.query, pos, frequency, out=grad_out),
             lambda: at.rope_backward(b.query, pos, frequency, out=grad_out),
             lambda: at.rope_backward(b.query.clone().requires_grad_(), pos, frequency,
                                      out=torch.empty_like(b.query)),
             lambda: append(query_out=grad_out), lambda: attend(out=grad_out)]
    for call in calls:
        with pytest.raises(ValueError):
            call()
        with torch.no_grad():
            call()
    with fw.dual_level():
        dual = fw.make_dual(b.query, b.query)
        for call in (lambda: append(query=dual), lambda: attend(query=dual),
                     lambda: at.rope(dual, pos, frequency, out=torch.empty_like(b.query))):
            with pytest.raises(ValueError):
                call()
        append(), attend()      # a level without tangents among the operands


def test_autograd_notices_what_is_written(hip_ready):
    """Tensors that a backward pass has saved and a call has written since make it fail, as torch's
    own writes do; inference tensors have no such count."""
    frequency, _ = at.rope_frequencies(64)
    pos = torch.arange(2, device="cuda")
    w = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    b = Batch(BF16, 4, 2, 64, 16, 32, [20, 9], [1, 1], seed=12).fill()

    def append(**more):
        at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query, **more)

    other = torch.zeros_like(b.query)
    for saved, call in ((b.query, lambda: at.rope(b.query, pos, frequency, out=b.query)),
                        (other, lambda: at.rope_backward(b.query, pos, frequency, out=other)),
                        (b.kc, append), (b.vc, append), (other, lambda: append(query_out=other)),
                        (other, lambda: b.attend(out=other))):
        loss = (saved * w).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    loss = (b.query * w).sum()      # read alone
    append(), b.attend(), at.rope(b.query, pos, frequency)
    loss.backward()
    with torch.inference_mode():
        made = torch.zeros_like(b.query)
    at.rope(b.query, pos, frequency, out=made)
    with torch.inference_mode():
        at.rope(b.query, pos, frequency, out=made)
        append(query_out=made)


def test_numbers_that_do_not_fit(hip_ready):
    """Bounds, offsets and factors that no field of the C structures holds are refused as others
    are."""
    frequency, _ = at.rope_frequencies(64)
    b = Batch(BF16, 4, 2, 64, 16, 32, [20, 9], [1, 1], seed=12).fill()
    pos = torch.arange(2, device="cuda")
    for more in (dict(max_length=2 ** 70), dict(max_query=-2 ** 70), dict(max_length=1.5),
                 dict(scale="one")):
        with pytest.raises(ValueError):
            b.attend(**more)
    for more in (dict(offset=2 ** 64), dict(offset=0.5), dict(magnitude="one")):
        with pytest.raises(ValueError):
            at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                            **more)
    with pytest.raises(ValueError):
        at.rope(b.query, pos, frequency, magnitude=None)
