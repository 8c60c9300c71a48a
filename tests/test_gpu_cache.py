"""Norms that turn, the append with them, the attention weight of cached keys and eviction by it
(tilegen_amd.attention) against the formulas in 64 bits.

Tolerances come from the arithmetic.  u is the unit roundoff of the operands' type (2^-8
bfloat16, 2^-11 float16, 2^-24 float32); e = 2^-24.

norm_rope: a sum of dim squares is off by at most (dim + 1) e of itself, its root's reciprocal by
half of that and 4 e; an element of the normed head, with its two products, by N = (dim / 2 + 8) e.
Turning adds 2^-21 of the pair (cosine and sine to about 2 pi 2^-26 + 2^-24, two products and a
sum), rounding u: |error| <= u |y| + (2^-21 + N) (|a| + |b|) magnitude.

backward: the gradient turned back is off by U = 2^-21 (|p| + |q|) magnitude, v = u w by U |w| + e
|v|, the sum v x by dim e sum |v x| + sum |x w| U; dx = r (v - x r^2 mean(v x)) follows, r to N; a
weight's gradient sums N terms in 32 bits, each off by its own error and at most N e of the sum of
magnitudes.

attention_weights: scores are off by S = dim 2^-23 scale sum |q k|, the exponent by e of score
and logarithm each more, an exponential by 2^-22 of itself, a sum of n terms by n e.

Eviction is exact."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tilegen_amd import attention as at

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
E = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPSILON = 1e-5


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cpu(x):
    return x.detach().cpu().double()


# --------------------------------------------------------------------------- #
# the formula
# --------------------------------------------------------------------------- #
def _angles(positions, frequency, magnitude):
    if frequency is None:
        return torch.ones(1, 1, 0, dtype=torch.float64), torch.zeros(1, 1, 0, dtype=torch.float64)
    angle = torch.from_numpy(positions.cpu().numpy().astype(np.float64)[:, None]
                             * frequency.cpu().double().numpy())
    return magnitude * torch.cos(angle)[:, None], magnitude * torch.sin(angle)[:, None]


def _parts(n, layout):
    return ((slice(0, n), slice(n, 2 * n)) if layout == "half" else
            (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))


def _turned(z, positions, frequency, layout, magnitude, sign=1):
    """(the turned heads, the sum of magnitudes that their pairs have)"""
    c, s = _angles(positions, frequency, magnitude)
    s = s * sign
    first, second = _parts(c.shape[-1], layout)
    y, size = z.clone(), z.abs()
    a, b = z[..., first], z[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(magnitude)
    return y, size


def _normed(x, weight, epsilon=EPSILON):
    x = _cpu(x)
    z = x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt()
    return z if weight is None else z * _cpu(weight)


def _check_normed(got, x, weight, positions, frequency, layout, magnitude=1.0, epsilon=EPSILON):
    want, size = _turned(_normed(x, weight, epsilon), positions, frequency, layout, magnitude)
    N = (x.shape[-1] / 2 + 8) * E
    bound = U[got.dtype] * want.abs() + (2.0 ** -21 + N) * size + TINY[got.dtype]
    off = (_cpu(got) - want).abs()
    assert (off <= bound * (1 + 2.0 ** -6)).all(), float((off - bound).max())


def _check_gradient(dx, dw, g, x, weight, positions, frequency, layout, magnitude=1.0):
    """Against the derivatives of the formula, with the bounds of the file's head."""
    D = x.shape[-1]
    u, size = _turned(_cpu(g), positions, frequency, layout, magnitude, sign=-1)
    eu = 2.0 ** -21 * size
    y, w = _cpu(x), torch.ones(D, dtype=torch.float64) if weight is None else _cpu(weight)
    r = (y.square().mean(-1, keepdim=True) + EPSILON).rsqrt()
    v, N = u * w, (D / 2 + 8) * E
    ev = eu * w.abs() + 2 * E * v.abs()
    mean = (v * y).mean(-1, keepdim=True)
    emean = ((D + 2) * E * (v * y).abs().mean(-1, keepdim=True)
             + (ev * y.abs()).mean(-1, keepdim=True))
    want = r * (v - y * r.square() * mean)
    each = r * v.abs() + y.abs() * r ** 3 * mean.abs()
    bound = (U[dx.dtype] * want.abs() + r * ev + y.abs() * r ** 3 * emean + 4 * N * each
             + TINY[dx.dtype])
    off = (_cpu(dx) - want).abs()
    assert (off <= bound * (1 + 2.0 ** -6)).all(), float((off - bound).max())
    if dw is None:
        return
    term, eterm = u * y * r, (eu * y.abs() + 2 * N * (u * y).abs()) * r
    axes = (0,) if weight.dim() == 2 else (0, 1)
    terms = x.shape[0] if weight.dim() == 2 else x.shape[0] * x.shape[1]
    want = term.sum(axes)
    bound = (U[dw.dtype] * want.abs() + eterm.sum(axes) + terms * E * term.abs().sum(axes)
             + TINY[dw.dtype])
    off = (_cpu(dw) - want).abs()
    assert dw.shape == weight.shape and dw.dtype == weight.dtype
    assert (off <= bound * (1 + 2.0 ** -6)).all(), float((off - bound).max())


def _weights(g, kind, heads, dim, dtype):
    """A norm's weight: none, one for all heads, one each; of the heads' type or in 32 bits."""
    if kind is None:
        return None
    shape = (heads, dim) if "each" in kind else (dim,)
    return (1 + 0.3 * _normal(g, *shape, dtype=F32)).to(F32 if "32" in kind else dtype)


NORMS = [
    # tokens, heads, kv_heads, dim, rotary, weights
    (1, 1, 0, 1, 0, "one"), (3, 2, 1, 7, 4, "one"), (5, 3, 2, 64, 64, "each"),
    (4, 5, 5, 80, 38, "each32"), (2, 32, 8, 128, 128, "one"), (9, 1, 1, 96, 0, None),
    (6, 7, 3, 256, 62, "one32"), (7, 5, 3, 256, 256, "each"), (1, 3, 1, 255, 100, "one"),
    (300, 2, 1, 96, 64, "one"), (70, 3, 2, 17, 16, "each"), (3, 150, 70, 24, 24, "one"),
    (2, 9, 9, 8, 8, "one32"), (515, 12, 4, 72, 24, "one"), (2100, 32, 8, 16, 16, "one32"),
    (1, 64, 1, 160, 80, "each"), (11, 3, 2, 192, 192, "one"), (2100, 8, 2, 66, 34, "each32"),
    (33, 3, 1, 18, 0, "one"), (5, 2, 2, 12, 10, "one32"), (2, 1, 3, 254, 254, "one"),
    (40, 2, 1, 9, 0, "each"), (7, 3, 3, 46, 20, "one")]


def _operands(layout, dtype, tokens, heads, kv_heads, dim, rotary, kind):
    g = _gen(tokens + dim + heads)
    q = 3 * _normal(g, tokens, heads, dim, dtype=dtype)
    k = _normal(g, tokens, kv_heads, dim, dtype=dtype) if kv_heads else None
    wq = _weights(g, kind, heads, dim, dtype)
    wk = _weights(g, kind, kv_heads, dim, dtype) if kv_heads else None
    positions = torch.randint(-1000, 10 ** 7, (tokens,), generator=g, device="cuda")
    frequency, magnitude = None, 1.0
    if rotary:
        frequency, magnitude = at.rope_frequencies(rotary, scaling="yarn", factor=8, trained=2048)
    return g, q, k, wq, wk, positions, frequency, magnitude


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,kind", NORMS)
def test_norm_rope(hip_ready, layout, dtype, tokens, heads, kv_heads, dim, rotary, kind):
    g, q, k, wq, wk, positions, frequency, magnitude = _operands(
        layout, dtype, tokens, heads, kv_heads, dim, rotary, kind)
    keep = q.clone()
    how = dict(epsilon=EPSILON, layout=layout, magnitude=magnitude)
    y, z = at.norm_rope(q, k, positions, frequency, wq, wk, **how)
    _check_normed(y, q, wq, positions, frequency, layout, magnitude)
    if k is None:
        assert z is None
    else:
        _check_normed(z, k, wk, positions, frequency, layout, magnitude)
    assert torch.equal(q, keep)
    # over their inputs: the same bits
    got = at.norm_rope(q, k, positions, frequency, wq, wk, query_out=q, key_out=k, **how)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, y) and (k is None or torch.equal(k, z))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,kind", NORMS)
def test_norm_rope_backward(hip_ready, layout, dtype, tokens, heads, kv_heads, dim, rotary, kind):
    g, q, k, wq, wk, positions, frequency, magnitude = _operands(
        layout, dtype, tokens, heads, kv_heads, dim, rotary, kind)
    gq = _normal(g, tokens, heads, dim, dtype=dtype)
    gk = _normal(g, tokens, kv_heads, dim, dtype=dtype) if kv_heads else None
    how = dict(epsilon=EPSILON, layout=layout, magnitude=magnitude)
    got = at.norm_rope_backward(gq, gk, q, k, positions, frequency, wq, wk, **how)
    _check_gradient(got[0], got[2], gq, q, wq, positions, frequency, layout, magnitude)
    if k is None:
        assert got[1] is None and got[3] is None
    else:
        _check_gradient(got[1], got[3], gk, k, wk, positions, frequency, layout, magnitude)
    if wq is None:
        assert got[2] is None
    again = at.norm_rope_backward(gq, gk, q, k, positions, frequency, wq, wk, **how)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_norm_rope_on_views(hip_ready, layout):
    """Heads of a packed projection, odd offsets, transposed tokens and heads, expanded weights."""
    g = _gen(1)
    frequency, _ = at.rope_frequencies(48)
    packed = _normal(g, 11, 9, 65, dtype=BF16)
    positions = torch.arange(11, device="cuda") * 12345
    w = _weights(g, "one", 1, 64, BF16)
    out = torch.zeros(9, 11, 77, device="cuda", dtype=BF16)
    q, k = packed[:, 2:7, 1:65], packed[:, 7:9, 1:65]
    y, z = out[1:6, :, 5:69].transpose(0, 1), out[6:8, :, 5:69].transpose(0, 1)
    at.norm_rope(q, k, positions, frequency, w, w.expand(2, 64), epsilon=EPSILON, layout=layout,
                 query_out=y, key_out=z)
    _check_normed(y, q, w, positions, frequency, layout)
    _check_normed(z, k, w, positions, frequency, layout)
    y.zero_(), z.zero_()
    assert not out.any()        # nothing beside the views was written
    before = packed.clone()
    at.norm_rope(q, k, positions, frequency, w, w, epsilon=EPSILON, layout=layout, query_out=q,
                 key_out=k)
    assert torch.equal(packed[:, :2], before[:, :2])
    _check_normed(q, before[:, 2:7, 1:65], w, positions, frequency, layout)
    wide = before[:, :1, :64].expand(11, 4, 64)
    got = at.norm_rope(wide, None, positions, frequency, w, epsilon=EPSILON, layout=layout)[0]
    _check_normed(got, wide, w, positions, frequency, layout)
    gq = _normal(g, 1, 1, 64, dtype=BF16).expand(11, 4, 64)
    dq, _, dw, _ = at.norm_rope_backward(gq, None, wide, None, positions, frequency,
                                         w.expand(4, 64), epsilon=EPSILON, layout=layout)
    _check_gradient(dq, dw, gq, wide, w.expand(4, 64), positions, frequency, layout)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_norm_rope_gradient(hip_ready, layout):
    """Through autograd, against the formula's derivatives and against its differences."""
    g = _gen(2)
    frequency, magnitude = at.rope_frequencies(24, scaling="yarn", factor=4, trained=512)
    positions = torch.tensor([0, 1, 77, 100000, 5], device="cuda")
    packed = _normal(g, 5, 5, 30, dtype=F32).requires_grad_()
    wq = _weights(g, "one", 3, 30, F32).requires_grad_()
    wk = _weights(g, "one", 2, 30, F32).requires_grad_()
    mine = _normal(g, 5, 3, 30, dtype=F32), _normal(g, 5, 2, 30, dtype=F32)
    how = dict(epsilon=EPSILON, layout=layout, magnitude=magnitude)
    y, z = at.norm_rope(packed[:, :3], packed[:, 3:], positions, frequency, wq,
                        wk.expand(2, 30), **how)
    ((y * mine[0]).sum() + (z * mine[1]).sum()).backward()
    x = packed.detach()
    _check_gradient(packed.grad[:, :3], wq.grad, mine[0], x[:, :3], wq.detach(), positions,
                    frequency, layout, magnitude)
    _check_gradient(packed.grad[:, 3:], wk.grad, mine[1], x[:, 3:], wk.detach(), positions,
                    frequency, layout, magnitude)

    def value(x, wq, wk):
        return sum(float((_turned(_normed(a, w), positions, frequency, layout, magnitude)[0]
                          * _cpu(m)).sum())
                   for a, w, m in ((x[:, :3], wq, mine[0]), (x[:, 3:], wk, mine[1])))

    # steps of 2^-10 along a direction: the difference is off by its third derivative / 6 * 2^-20,
    # at most about 2^-20 |grad| times the direction's size squared (heads are of size about 5)
    step = 2.0 ** -10
    for of in range(3):
        at_ = [_cpu(x), _cpu(wq), _cpu(wk)]
        way = torch.randn(at_[of].shape, generator=torch.Generator().manual_seed(of),
                          dtype=torch.float64)
        grad = (packed.grad, wq.grad, wk.grad)[of]
        plus, minus = list(at_), list(at_)
        plus[of], minus[of] = at_[of] + step * way, at_[of] - step * way
        difference = (value(*plus) - value(*minus)) / (2 * step)
        slope = float((_cpu(grad) * way).sum())
        size = float((_cpu(grad) * way).abs().sum())
        assert abs(slope - difference) <= 2.0 ** -14 * size, of
    # a broadcast gradient, keys alone unused, weights that need none
    packed.grad = None
    at.norm_rope(packed[:, :3], packed[:, 3:], positions, frequency, wq.detach(), wk.detach(),
                 **how)[0].sum().backward()
    _check_gradient(packed.grad[:, :3], None, torch.ones_like(mine[0]), x[:, :3], wq.detach(),
                    positions, frequency, layout, magnitude)
    assert not packed.grad[:, 3:].any()


def test_norm_rope_of_many_heads(hip_ready):
    """More groups of rows than a launch has waves: heads of one element, which norm to their sign."""
    x = torch.ones(1 << 20, 200, 1, device="cuda", dtype=BF16)
    x[::3], x[5, 7], x[-1, -1] = -2, 0, 3
    y, _ = at.norm_rope(x, None, None, None, epsilon=EPSILON)
    # 1 and 2 are off by epsilon / 2 and less of themselves, under the type's half step
    assert torch.equal(y, x.sign())


def test_norm_rope_gradient_in_a_graph(hip_ready):
    """A forward and backward pass captured and replayed, against eager ones."""
    g = _gen(8)
    frequency, _ = at.rope_frequencies(64)
    q, k = (_normal(g, 70, n, 64, dtype=BF16).requires_grad_() for n in (6, 2))
    wq, wk = (_weights(g, "one", 1, 64, F32).requires_grad_() for _ in range(2))
    positions = torch.arange(70, device="cuda")
    gq, gk = torch.ones_like(q), torch.ones_like(k)

    def step():
        y, z = at.norm_rope(q, k, positions, frequency, wq, wk)
        return torch.autograd.grad([y, z], [q, k, wq, wk], [gq, gk])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(_normal(g, *q.shape, dtype=BF16))
            wk.mul_(1.25)
        gk.copy_(_normal(g, *gk.shape, dtype=BF16))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


def test_norm_rope_at_the_ends(hip_ready):
    """Heads of zeros, of infinities and NaN; no tokens; sums past 32 bits' range."""
    frequency, _ = at.rope_frequencies(64)
    positions = torch.arange(4, device="cuda")
    x = torch.zeros(4, 1, 64, device="cuda", dtype=BF16)
    x[1] = 2.0
    x[2, 0, 5] = math.nan
    x[3, 0, 7] = math.inf
    w = torch.ones(64, device="cuda", dtype=BF16)
    y, _ = at.norm_rope(x, x, positions, frequency, w, w)
    assert not y[0].any() and torch.isfinite(y[1]).all()
    assert y[2].isnan().all() and y[3, 0, 7].isnan() and y[3, 0, 7 + 32].isnan()
    assert not y[3, 0, :7].any()
    none = torch.empty(0, 3, 64, device="cuda", dtype=BF16)
    y, z = at.norm_rope(none, none, positions[:0], frequency, w, w)
    assert y.shape == z.shape == none.shape
    got = at.norm_rope_backward(none, none, none, none, positions[:0], frequency, w, w)
    assert not got[2].any() and not got[3].any() and got[0].shape == none.shape


@pytest.mark.parametrize("tokens", [0, 1, 70])
@pytest.mark.parametrize("kind", ["one", "each32"])
@pytest.mark.parametrize("heads,kv_heads", [(3, 0), (40, 0), (0, 2), (0, 0)])
def test_norm_rope_backward_without_heads(hip_ready, monkeypatch, heads, kv_heads, kind, tokens):
    """A weight that no head reads has a gradient of zeros, whatever its memory held."""
    monkeypatch.setattr(at, "_like", lambda x: torch.full(x.shape, math.nan, dtype=x.dtype,
                                                          device=x.device))
    _, q, k, wq, wk, positions, frequency, magnitude = _operands("half", BF16, tokens, heads,
                                                                 kv_heads, 64, 64, kind)
    if k is None:
        k = torch.empty(tokens, 0, 64, device="cuda", dtype=BF16)
        wk = _weights(_gen(1), kind, 0, 64, BF16)
    g = _gen(2)
    gq, gk = (_normal(g, *x.shape, dtype=BF16) for x in (q, k))
    args, how = (q, k, positions, frequency, wq, wk), dict(epsilon=EPSILON, magnitude=magnitude)
    dq, dk, dwq, dwk = at.norm_rope_backward(gq, gk, *args, **how)
    _check_gradient(dq, dwq, gq, q, wq, positions, frequency, "half", magnitude)
    _check_gradient(dk, dwk, gk, k, wk, positions, frequency, "half", magnitude)
    y = at.norm_rope(q, k, positions, frequency, wq.requires_grad_(), wk.requires_grad_(), **how)
    again = torch.autograd.grad(y, [wq, wk], [gq, gk])
    assert torch.equal(again[0], dwq) and torch.equal(again[1], dwk)


# --------------------------------------------------------------------------- #
# a batch with its cache
# --------------------------------------------------------------------------- #
class Batch:
    """Random pages for each sequence, one to spare on odd ones; cache slots that no token has hold
    NaN.  Weights stand with a head's slots side by side, or as the caches do."""

    def __init__(self, dtype, heads, kv_heads, dim, page, lengths, counts=None, seed=0,
                 side_by_side=True):
        g = self.g = _gen(seed)
        counts = [0] * len(lengths) if counts is None else counts
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = (dtype, heads, kv_heads, dim,
                                                                      page)
        self.lengths_host, self.counts = list(lengths), list(counts)
        owned = [-(-max(0, n) // page) + i % 2 for i, n in enumerate(lengths)]
        self.pages = sum(owned) + 2
        order = torch.randperm(self.pages, generator=g, device="cuda")
        self.indices = order[:sum(owned)].contiguous()
        self.indptr, self.ends = self._ends(owned), self._ends(counts)
        self.ends_host = [0] + np.cumsum(counts).tolist()
        self.lengths = torch.tensor(self.lengths_host, dtype=torch.int64, device="cuda")
        shape = (self.pages, page, kv_heads, dim)
        self.kc = torch.full(shape, math.nan, device="cuda", dtype=dtype)
        self.vc = torch.full(shape, math.nan, device="cuda", dtype=dtype)
        shape = (self.pages, kv_heads, page) if side_by_side else shape[:3]
        self.w = torch.full(shape, math.nan, device="cuda")
        self.w = self.w.transpose(1, 2) if side_by_side else self.w
        self.query = _normal(g, sum(counts), heads, dim, dtype=dtype)
        self.key = _normal(g, sum(counts), kv_heads, dim, dtype=dtype)
        self.value = _normal(g, sum(counts), kv_heads, dim, dtype=dtype)

    @staticmethod
    def _ends(n):
        return torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int64, device="cuda")

    def places(self, b):
        pages = self.indices[int(self.indptr[b]):int(self.indptr[b + 1])]
        n = min(max(0, self.lengths_host[b]), pages.numel() * self.page)
        at_ = torch.arange(n, device="cuda")
        return pages[at_ // self.page], at_ % self.page

    def fill(self, weights=None):
        for b in range(len(self.counts)):
            page, slot = self.places(b)
            for c in (self.kc, self.vc):
                c[page, slot] = _normal(self.g, page.numel(), self.kv_heads, self.dim,
                                        dtype=self.dtype)
            self.w[page, slot] = _normal(self.g, page.numel(), self.kv_heads, dtype=F32).exp()
        return self

    def lse(self, scale=None):
        """Each row's logarithm of the sum of its exponentials, with a little more as a prefix
        would add; float32."""
        scale = self.dim ** -0.5 if scale is None else scale
        G = self.heads // self.kv_heads
        out = torch.full((sum(self.counts), self.heads), -math.inf, dtype=torch.float64)
        q = _cpu(self.query)
        for b, n in enumerate(self.counts):
            k = _cpu(self.kc[self.places(b)])
            for j in range(n):
                see = min(max(0, self.lengths_host[b] - n + j + 1), k.shape[0])
                if see:
                    s = torch.einsum("khd,hgd->hgk", k[:see], q[self.ends_host[b] + j].reshape(
                        self.kv_heads, G, -1)) * scale
                    out[self.ends_host[b] + j] = s.logsumexp(-1).flatten() + 0.1
        return out.float().cuda()

    def weigh(self, lse, **more):
        args = dict(query_indptr=self.ends, max_query=max(self.counts + [1]),
                    max_length=max(self.lengths_host + [1]))
        if all(n == 1 for n in self.counts):
            args["query_indptr"] = None
        args.update(more)
        return at.attention_weights(self.query, lse, self.kc, self.w, self.indptr, self.indices,
                                    self.lengths, **args)

    def check_weights(self, before, lse, scale=None, decay=1.0):
        """self.w against the formula from what it was before."""
        scale = self.dim ** -0.5 if scale is None else scale
        G = self.heads // self.kv_heads
        q, lse = _cpu(self.query), _cpu(lse)
        touched = torch.zeros(self.w.shape, dtype=torch.bool)
        for b, n in enumerate(self.counts):
            if n == 0:
                continue
            page, slot = self.places(b)
            k = _cpu(self.kc[page, slot])
            L = k.shape[0]
            p0 = self.lengths_host[b] - n
            at_ = torch.arange(L)
            old = torch.where((at_ < p0)[:, None], decay * _cpu(before[page, slot]), 0.0)
            sum_, bound = torch.zeros_like(old), 2 * E * old.abs()
            terms = 0
            for j in range(n):
                rows = q[self.ends_host[b] + j].reshape(self.kv_heads, G, -1)
                e = lse[self.ends_host[b] + j].reshape(self.kv_heads, G)
                s = torch.einsum("khd,hgd->khg", k, rows) * scale
                size = torch.einsum("khd,hgd->khg", k.abs(), rows.abs()) * scale
                got = (s - e).exp()
                off = got * (self.dim * 2.0 ** -23 * size + E * (s.abs() + 2 * e.abs() + 2)
                             + 2.0 ** -22)
                seen = (at_ <= p0 + j)[:, None, None] & (e > -math.inf)
                sum_ += torch.where(seen, got, 0.0).sum(-1)
                bound += torch.where(seen, off, 0.0).sum(-1)
                terms += G
            want = old + sum_
            bound += (terms + 2) * E * sum_ + E * want.abs()
            off = (_cpu(self.w[page, slot]) - want).abs()
            assert (off <= bound * (1 + 2.0 ** -6)).all(), (b, float((off - bound).max()))
            touched[page.cpu(), slot.cpu()] = True
        rest = ~touched.cuda()
        assert torch.equal(self.w[rest].nan_to_num(-7), before[rest].nan_to_num(-7))


# --------------------------------------------------------------------------- #
# append
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page,lengths,counts,kind", [
    (4, 2, 64, 64, 16, [5, 17, 32], [1, 1, 1], "one"),
    (3, 3, 7, 4, 3, [9, 4, 0, 10], [3, 4, 0, 1], "each"),
    (5, 1, 80, 38, 24, [100, 60], [70, 2], "one32"),
    (32, 8, 128, 128, 16, [700, 3], [600, 3], "one"),
    (2, 1, 256, 0, 5, [11, 12], [2, 7], "each32"),
    (0, 2, 96, 48, 8, [9, 20], [9, 3], "one"),
    (8, 4, 128, 62, 64, [65, 1, 1, 130], [1, 1, 1, 1], None),
])
def test_append_with_norms(hip_ready, layout, dtype, heads, kv_heads, dim, rotary, page, lengths,
                           counts, kind):
    b = Batch(dtype, heads, kv_heads, dim, page, lengths, counts, seed=dim)
    frequency, magnitude = (at.rope_frequencies(rotary, scaling="yarn", factor=4, trained=512)
                            if rotary else (None, 1.0))
    shift = torch.randint(10 ** 6, (len(lengths),), generator=b.g, device="cuda")
    wq = _weights(b.g, kind, heads, dim, dtype) if heads else None
    wk = _weights(b.g, kind, kv_heads, dim, dtype)
    one = all(n == 1 for n in counts)
    q = at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query if heads else None, query_indptr=None if one else b.ends,
                        offset=77, layout=layout, magnitude=magnitude, query_weight=wq,
                        key_weight=wk, epsilon=EPSILON, shift=shift)
    written = torch.zeros(b.pages, page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(counts):
        if not n:
            continue
        mine = slice(b.ends_host[s], b.ends_host[s] + n)
        at_ = torch.arange(lengths[s] - n, lengths[s], device="cuda")
        where = tuple(x[at_] for x in b.places(s))
        positions = 77 + shift[s] + at_
        _check_normed(b.kc[where], b.key[mine], wk, positions, frequency, layout, magnitude)
        assert torch.equal(b.vc[where], b.value[mine])
        if heads:
            _check_normed(q[mine], b.query[mine], wq, positions, frequency, layout, magnitude)
        written[where] = True
    assert b.kc[~written].isnan().all() and b.vc[~written].isnan().all()


def test_append_with_a_shift_alone(hip_ready):
    """Without norms: as paged_append at other positions; offsets past 32 bits."""
    b = Batch(BF16, 4, 2, 64, 16, [5, 17, 32], [1, 1, 1])
    frequency, _ = at.rope_frequencies(64)
    shift = torch.tensor([0, 2 ** 33, 12], device="cuda")
    q = at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query, shift=shift, offset=3)
    positions = b.lengths + 2 + shift
    want = at.rope(b.query, positions, frequency)
    assert ((q.float() - want.float()).abs() <= 2 * U[BF16] * want.float().abs() + 2.0 ** -19).all()
    keys = at.rope(b.key, positions, frequency)
    for s, n in enumerate(b.lengths_host):
        page, slot = (x[n - 1] for x in b.places(s))
        off = (b.kc[page, slot].float() - keys[s].float()).abs()
        assert (off <= 2 * U[BF16] * keys[s].float().abs() + 2.0 ** -19).all()


def test_append_of_nothing_with_norms(hip_ready):
    """A batch without tokens, and one without query heads: presence goes by the operand."""
    b = Batch(BF16, 4, 2, 64, 16, [20, 33], [0, 0]).fill()
    frequency, _ = at.rope_frequencies(64)
    wq, wk = (_weights(b.g, "one", 1, 64, BF16) for _ in range(2))
    how = dict(query_weight=wq, key_weight=wk, epsilon=EPSILON)
    before = b.kc.clone(), b.vc.clone()
    table = (b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency)
    q = at.paged_append(b.key, b.value, *table, query=b.query, query_indptr=b.ends, **how)
    assert q.shape == (0, 4, 64)
    none = b.ends[:1], b.indices[:0], b.lengths[:0]
    q = at.paged_append(b.key, b.value, b.kc, b.vc, *none, frequency, query=b.query, **how)
    assert q.shape == (0, 4, 64)
    for old, new in zip(before, (b.kc, b.vc)):
        assert torch.equal(old.nan_to_num(-7), new.nan_to_num(-7))
    key, value = (_normal(b.g, 2, 2, 64, dtype=BF16) for _ in range(2))
    q = at.paged_append(key, value, *table, query=key[:, :0], **how)
    assert q.shape == (2, 0, 64)
    got = b.kc.clone(), b.vc.clone()
    at.paged_append(key, value, *table, key_weight=wk, epsilon=EPSILON)
    for old, new in zip(got, (b.kc, b.vc)):
        assert torch.equal(old.nan_to_num(-7), new.nan_to_num(-7))
    assert not torch.equal(b.kc.nan_to_num(-7), before[0].nan_to_num(-7))


def test_append_leaves_out_what_has_no_place(hip_ready):
    """Rows of no sequence, positions past a sequence's pages, pages outside the cache."""
    b = Batch(F16, 4, 2, 64, 8, [9, 40, 8, 8], [2, 3, 1, 1])
    frequency, _ = at.rope_frequencies(64)
    w = _weights(b.g, "one", 1, 64, F16)
    query = torch.cat([b.query[:1], b.query, b.query[:2]])     # one row before, two behind
    key, value = (torch.cat([x[:1], x, x[:2]]) for x in (b.key, b.value))
    b.lengths[1] += 20          # its last token is past its pages
    indices = b.indices.clone()
    indices[b.indptr[2]], indices[b.indptr[3]] = -1, b.pages
    q = at.paged_append(key, value, b.kc, b.vc, b.indptr, indices, b.lengths, frequency,
                        query=query, query_indptr=b.ends + 1, query_weight=w, key_weight=w,
                        epsilon=0.0, shift=torch.zeros_like(b.lengths))
    assert not q[0].any() and not q[8:].any() and q[1:8].any(-1).all()
    assert int((~b.kc.isnan()).any(-1).any(-1).sum()) == 2      # the first sequence's two


# --------------------------------------------------------------------------- #
# the weight of keys
# --------------------------------------------------------------------------- #
MANY = dict(max_query=10 ** 6, max_length=1100)     # bounds that make workgroups of many rows

SHAPES = [
    # heads, kv_heads, dim, page, lengths, counts
    (4, 2, 64, 16, [70, 33, 1], [1, 1, 1]),
    (1, 1, 8, 1, [5, 1], [1, 1]),
    (7, 1, 40, 7, [40, 7, 90, 0], [7, 1, 3, 0]),
    (16, 4, 64, 16, [300, 20, 64, 31], [40, 9, 3, 0]),
    (12, 4, 80, 24, [200, 33, 1], [130, 20, 1]),
    (8, 8, 96, 3, [140, 2], [9, 2]),
    (32, 8, 128, 64, [190, 77, 1], [150, 70, 1]),
    (25, 1, 128, 20, [300, 2], [1, 2]),
    (4, 1, 200, 8, [33, 70], [1, 2]),
    (10, 2, 256, 5, [120, 31, 600], [5, 4, 300]),
    (6, 2, 128, 16, [1100, 513], [700, 513]),
    (4, 2, 64, 16, [2, 0, 9], [5, 3, 1]),       # fewer tokens than new ones
    # workgroups of many rows, and rows in parts
    (16, 1, 64, 16, [600, 300, 0, 257], [500, 20, 0, 2]),
    (16, 2, 96, 24, [520, 700], [300, 300]),
    (32, 1, 128, 64, [256, 900, 40], [70, 130, 40]),
    (32, 2, 256, 7, [300, 129, 128], [160, 1, 128]),
    (48, 1, 72, 16, [70, 33, 1], [1, 1, 1]),
    (40, 1, 128, 16, [20, 1], [33, 2]),
    # and heads that do not fill their tiles
    (16, 1, 40, 16, [200, 100], [60, 3]),
    (48, 1, 72, 16, [70, 33, 1], [9, 8, 1]),
    (20, 1, 104, 8, [150, 60], [30, 9]),
    (32, 1, 200, 8, [133, 70], [20, 2]),
]


@pytest.mark.parametrize("bounds", [dict(), MANY])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,lengths,counts", SHAPES)
def test_attention_weights(hip_ready, dtype, heads, kv_heads, dim, page, lengths, counts, bounds):
    b = Batch(dtype, heads, kv_heads, dim, page, lengths, counts, seed=dim,
              side_by_side=page != 16).fill()
    lse, before = b.lse(), b.w.clone()
    assert b.weigh(lse, decay=0.75, **bounds) is b.w
    b.check_weights(before, lse, decay=0.75)
    # the same bits again
    got, b.w = b.w, before.clone()
    b.weigh(lse, decay=0.75, **bounds)
    assert torch.equal(b.w.nan_to_num(-7), got.nan_to_num(-7))


@pytest.mark.parametrize("bounds", [dict(max_length=100), dict(max_query=40), dict(max_query=1),
                                    dict(max_length=1, max_query=130), dict(max_length=5000)])
def test_attention_weights_past_their_bounds(hip_ready, bounds):
    """max_length and max_query size the launch: what is longer is right all the same."""
    b = Batch(BF16, 32, 2, 128, 16, [900, 300, 77], [400, 5, 60]).fill()
    lse, before = b.lse(), b.w.clone()
    b.weigh(lse, **bounds)
    b.check_weights(before, lse)


@pytest.mark.parametrize("heads,kv_heads,dim,lengths,counts,max_length", [
    # parts of two sizes, most of what there might be absent
    (64, 1, 64, [900, 50, 40, 10, 300, 17], [520, 40, 3, 0, 20, 17], 8000),
    (128, 2, 128, [90, 600], [90, 510], 12000),
    # the same with more keys, and with more new tokens, than the bounds
    (64, 1, 64, [900, 50, 40, 10, 300, 17], [520, 40, 3, 0, 20, 17], 700),
    # more sequences than are looked over
    (1, 1, 64, [3 + i % 50 for i in range(1100)], [i % 3 for i in range(1100)], 1100),
])
def test_attention_weights_of_many_pieces(hip_ready, heads, kv_heads, dim, lengths, counts,
                                          max_length):
    b = Batch(BF16, heads, kv_heads, dim, 16, lengths, counts).fill()
    lse, before = b.lse(), b.w.clone()
    b.weigh(lse, max_query=10 ** 6, max_length=max_length, decay=0.5)
    b.check_weights(before, lse, decay=0.5)
    b.w = before.clone()
    b.weigh(lse, max_query=400, max_length=max_length, decay=0.5)
    b.check_weights(before, lse, decay=0.5)


def test_attention_weights_of_prompts_in_a_graph(hip_ready):
    """Parts joined through a workspace, captured twice and replayed in turn, beside eager calls."""
    b = Batch(BF16, 32, 2, 64, 16, [700, 90, 400], [600, 40, 300]).fill()
    other = Batch(BF16, 32, 2, 64, 16, [500, 300], [420, 300], seed=5).fill()
    sides = [(x, x.lse(), x.w.clone()) for x in (b, other)]
    graphs = []
    for x, lse, before in sides:
        x.weigh(lse)
    torch.cuda.synchronize()
    for x, lse, before in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            x.weigh(lse)
    for i in range(3):
        for (x, lse, before), graph in zip(sides, graphs):
            x.query.copy_(_normal(_gen(i), *x.query.shape, dtype=BF16))
            x.w.copy_(before)
            x.weigh(lse)
            want = x.w.clone()
            x.w.copy_(before)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(x.w.nan_to_num(-7), want.nan_to_num(-7)), i


@pytest.mark.parametrize("sequences", [2, 64, 65, 200, 256, 257])
@pytest.mark.parametrize("several", [False, True])
def test_attention_weights_of_many_sequences(hip_ready, sequences, several):
    lengths = [(37 * i) % 150 + 1 for i in range(sequences)]
    counts = [i % 3 if several else 1 for i in range(sequences)]
    b = Batch(F16, 4, 2, 64, 8, lengths, counts).fill()
    lse, before = b.lse(), b.w.clone()
    b.weigh(lse)
    b.check_weights(before, lse)
    b.w = before.clone()
    b.weigh(lse, max_length=40)     # the last piece of a sequence takes what is past the bound
    b.check_weights(before, lse)


@pytest.mark.parametrize("extra,at_", [(1, 0), (2, 1), (2, 2), (6, 4), (8, 0)])
def test_attention_weights_of_queries_anywhere(hip_ready, extra, at_):
    """Many rows whose heads start at any element."""
    b = Batch(BF16, 24, 2, 80, 16, [700, 90], [600, 40]).fill()
    loose = torch.full((642, 25, 80 + extra), math.nan, device="cuda", dtype=BF16)
    lse, before = b.lse(), b.w.clone()
    query = loose[1:641, :24, at_:at_ + 80]
    query.copy_(b.query)
    b.query = query
    b.weigh(lse)
    b.check_weights(before, lse)


def test_attention_weights_sum_to_one(hip_ready):
    """With prefix_attention's own logarithms, each row's weights sum to one."""
    b = Batch(BF16, 8, 2, 128, 16, [300, 77, 64], [9, 77, 1]).fill()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    _, lse = at.prefix_attention(b.query, b.kc, b.vc, none, 0, b.indptr, b.indices, b.lengths,
                                 query_indptr=b.ends, max_query=77, max_length=300,
                                 return_lse=True)
    before = b.w.clone()
    b.weigh(lse, decay=0.0)
    b.check_weights(before, lse, decay=0.0)
    for s, n in enumerate(b.counts):
        total = float(b.w[b.places(s)].double().sum())
        assert abs(total - n * 8) <= n * 8 * 2.0 ** -14


@pytest.mark.parametrize("heads", [4, 40])
def test_attention_weights_of_strange_rows_and_keys(hip_ready, heads):
    """Hidden keys may hold anything; rows without keys add nothing; a NaN that is seen is seen."""
    b = Batch(BF16, heads, 2, 64, 16, [40, 20], [3, 2] if heads == 4 else [7, 8]).fill()
    bounds = dict(max_query=10 ** 6, max_length=5000) if heads > 4 else {}
    lse, before = b.lse(), b.w.clone()
    lse[1, 2] = -math.inf
    b.weigh(lse, **bounds)
    b.check_weights(before, lse)
    # a later token's key is not seen by earlier rows, and stands for itself alone
    page, slot = b.places(0)
    b.kc[page[39], slot[39]] = math.nan
    want, b.w = b.w.clone(), before.clone()
    b.weigh(lse, **bounds)
    assert b.w[page[39], slot[39]].isnan().all()
    want[page[39], slot[39]] = math.nan
    assert torch.equal(b.w.nan_to_num(-7), want.nan_to_num(-7))
    # rows of no sequence hold anything
    query, b.query = b.query, torch.cat([b.query, torch.full_like(b.query, math.nan)])
    b.w = before.clone()
    b.weigh(torch.cat([lse, torch.full_like(lse, math.nan)]), **bounds)
    assert torch.equal(b.w.nan_to_num(-7), want.nan_to_num(-7))


@pytest.mark.parametrize("large", [1e38, -1e38])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("bounds", [dict(), dict(max_query=10 ** 6, max_length=5000)])
def test_attention_weights_of_hidden_scores_past_32_bits(hip_ready, bounds, dim, large):
    """A finite key whose scores with rows that do not see it pass 32 bits: what they are does not
    matter."""
    b = Batch(BF16, 40, 2, dim, 16, [40, 300], [7, 8]).fill()
    page, slot = b.places(0)
    b.kc[page[38], slot[38], :, 0] = large
    b.query[:5, :, 0] = 8.0          # positions 33 .. 37
    b.query[5:7, :, 0] = 0.0         # 38 and 39, which see it
    lse, before = b.lse(), b.w.clone()
    assert lse.isfinite().all()
    b.weigh(lse, **bounds)
    b.check_weights(before, lse)
    assert b.w[page, slot].isfinite().all()


@pytest.mark.parametrize("counts", [[3, 1, 4], [3, 1, 30]])
def test_attention_weights_of_lost_pages(hip_ready, counts):
    b = Batch(F16, 8, 2, 64, 8, [50, 40, 30], counts).fill()
    lse = b.lse()
    indices = b.indices.clone()
    indices[1], indices[int(b.indptr[1]) + 2] = -5, b.pages + 3
    kept = b.indices
    before, b.indices = b.w.clone(), indices
    b.weigh(lse, **(MANY if max(counts) > 4 else {}))
    got, b.w, b.indices = b.w.clone(), before.clone(), kept
    b.weigh(lse, **(MANY if max(counts) > 4 else {}))
    same = torch.ones(b.pages, dtype=torch.bool, device="cuda")
    lost = kept[[1, int(b.indptr[1]) + 2]]
    same[lost] = False
    assert torch.equal(got[same].nan_to_num(-7), b.w[same].nan_to_num(-7))
    assert torch.equal(got[lost].nan_to_num(-7), before[lost].nan_to_num(-7))


# --------------------------------------------------------------------------- #
# eviction
# --------------------------------------------------------------------------- #
def _kept(weights, length, keep, recent, first):
    """The definition: where the token at each position was, for one head."""
    if length <= keep:
        return list(range(length))
    key = [(-math.inf if math.isnan(w) else -w, p) for p, w in enumerate(weights)]
    heavy = sorted(range(first, length - recent), key=lambda p: key[p])[:keep - recent - first]
    stays = set(range(first)) | set(heavy)
    front = keep - recent
    later = iter(sorted(p for p in stays if p >= front))
    return [p if p in stays else next(later) for p in range(front)] + list(
        range(length - recent, length))


def _check_evicted(b, before, fewer, kept, keep, recent, first, move_weights=True):
    kc, vc, w = before
    ends = torch.zeros(b.pages, b.page, dtype=torch.bool, device="cuda")
    for s, length in enumerate(b.lengths_host):
        page, slot = b.places(s)
        length = page.numel()
        assert int(fewer[s]) == min(length, keep)
        for h in range(b.kv_heads):
            want = _kept(w[page, slot, h].tolist(), length, keep, recent, first)
            n = len(want)
            assert kept[s, h].tolist() == want + [-1] * (keep - n), (s, h)
            source = torch.tensor(want, dtype=torch.int64, device="cuda")
            for old, new in ((kc, b.kc), (vc, b.vc)) + (((w, b.w),) if move_weights else ()):
                x = old[page[source], slot[source], h]
                y = new[page[:n], slot[:n], h]
                assert torch.equal(x.nan_to_num(-7), y.nan_to_num(-7)), (s, h)
        if length:
            ends[page, slot] = True
    for old, new in ((kc, b.kc), (vc, b.vc), (w, b.w)):     # other pages' slots are left alone
        rest = ~ends if old is not w or move_weights else torch.ones_like(ends)
        assert torch.equal(old[rest].nan_to_num(-7), new[rest].nan_to_num(-7))


def _evict(b, keep, recent, first, **more):
    before = [x.clone() for x in (b.kc, b.vc, b.w)]
    args = dict(keep=keep, recent=recent, first=first, max_length=max(b.lengths_host))
    fewer, kept = at.paged_evict(b.w, b.kc, b.vc, b.indptr, b.indices, b.lengths,
                                 **dict(args, **more))
    _check_evicted(b, before, fewer, kept, keep, recent, first, more.get("move_weights", True))
    return fewer, kept


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv_heads,dim,page,lengths,keep,recent,first", [
    (2, 64, 16, [70, 33, 1, 0], 20, 5, 2), (1, 8, 1, [5, 1, 7], 3, 0, 0),
    (3, 96, 24, [210, 90, 101], 101, 17, 3), (2, 17, 5, [64, 65, 63], 64, 64, 0),
    (1, 1, 3, [40, 9], 7, 0, 7), (2, 7, 4, [300], 1, 1, 0), (2, 40, 8, [100, 30], 0, 0, 0),
    (1, 200, 16, [1300, 900], 700, 650, 1), (5, 128, 64, [4500, 5000, 100], 4096, 100, 4),
    (2, 24, 16, [9000, 4097], 5000, 0, 0), (1, 16, 128, [40000, 33000], 11000, 3000, 10),
    (1, 256, 16, [130, 140], 128, 100, 4), (1, 1000, 16, [50], 30, 11, 2),
    (2, 128, 16, [4000, 3500], 1500, 200, 4), (2, 128, 24, [700, 701, 3], 600, 590, 0),
    (1, 128, 16, [17000], 16000, 15000, 1), (100, 16, 16, [90, 70, 33], 40, 9, 0),
    # workgroups of 512 and of 256 threads
    (128, 24, 16, [90, 700, 33], 60, 9, 1), (350, 40, 8, [300, 41], 40, 17, 3),
    (170, 128, 16, [1100, 90, 1200, 1030], 1000, 260, 2), (130, 8, 4, [4000, 20], 1500, 300, 0),
    # fours of positions that start before the candidates, and as many as threads hold
    (2, 64, 4, [33, 47, 64], 20, 6, 5), (1, 32, 16, [4161, 4160], 1000, 64, 1),
    (1, 8, 16, [16394, 16395], 3000, 8, 3), (1, 8, 64, [32780], 3000, 10, 2),
])
def test_paged_evict(hip_ready, dtype, kv_heads, dim, page, lengths, keep, recent, first):
    b = Batch(dtype, kv_heads, kv_heads, dim, page, lengths, seed=keep,
              side_by_side=page != 16).fill()
    _evict(b, keep, recent, first)


def test_evict_ties_and_strange_weights(hip_ready):
    b = Batch(BF16, 2, 2, 32, 16, [200, 150, 120, 90, 5000]).fill()
    w = b.w
    w.copy_(torch.randint(0, 4, w.shape, generator=b.g, device="cuda").float())  # many ties
    page, slot = b.places(1)
    w[page, slot] = 0.0
    w[page[::2], slot[::2]] = -0.0            # the same weight
    page, slot = b.places(2)
    w[page, slot] = torch.tensor([math.nan, math.inf, -math.inf, -1.5, 1e-45, -1e-45, 3e38, 0.0],
                                 device="cuda").repeat(15)[:, None]
    page, slot = b.places(3)
    w[page, slot] = -math.inf
    _evict(b, 70, 10, 3)


def test_evict_without_the_weights(hip_ready):
    b = Batch(F16, 2, 2, 64, 16, [300, 170]).fill()
    fewer, kept = _evict(b, 100, 20, 4, move_weights=False)
    b.lengths_host = fewer.tolist()
    b.lengths.copy_(fewer)
    fewer, kept = _evict(b, 100, 20, 4)       # nothing left to do
    assert kept.tolist() == [[list(range(100))] * 2] * 2


@pytest.mark.parametrize("kv_heads,lengths,keep", [(2, [300, 170], 100), (100, [90, 33], 40),
                                                   (2, [5000, 4097, 20], 1500)])
def test_evict_by_weights_that_heads_share(hip_ready, kv_heads, lengths, keep):
    """Weights that are only read may share memory: one for all kv heads, one for all of a page."""
    b = Batch(BF16, kv_heads, kv_heads, 24, 16, lengths).fill()
    w, kc, vc = b.w, b.kc.clone(), b.vc.clone()
    for shared in (w[:, :, :1], w[:, :1]):
        b.kc.copy_(kc), b.vc.copy_(vc)
        b.w = shared.expand(w.shape)
        _evict(b, keep, 20, 4, move_weights=False)
        with pytest.raises(ValueError, match="share memory"):
            at.paged_evict(b.w, b.kc, b.vc, b.indptr, b.indices, b.lengths, keep=keep,
                           max_length=5000)


@pytest.mark.parametrize("lengths,keep,max_length", [([6000, 300], 128, 10), ([6000, 300], 5000, 10),
                                                     ([20000], 9000, 10), ([40000], 12000, 12000),
                                                     ([7000], 3000, 3300)])
def test_evict_past_its_bound(hip_ready, lengths, keep, max_length):
    """max_length sizes the launch: longer sequences are cut all the same."""
    b = Batch(BF16, 2, 2, 64, 16, lengths).fill()
    _evict(b, keep, 30, 2, max_length=max_length)


@pytest.mark.parametrize("kv_heads", [140, 350])
def test_evict_many_heads_past_the_bound(hip_ready, kv_heads):
    b = Batch(BF16, kv_heads, kv_heads, 8, 16, [4700, 50]).fill()
    _evict(b, 3000, 30, 1, max_length=3300)


def test_evict_lengths_past_the_pages(hip_ready):
    """Tokens that a sequence's pages do not hold are not among those that it has: lengths end with
    the pages, whether or not that is past `keep`."""
    b = Batch(BF16, 2, 2, 64, 16, [70, 90, 33], seed=3).fill()
    b.lengths_host = [1000, 91, 33]         # 5, 7 and 3 pages
    b.lengths.copy_(torch.tensor(b.lengths_host, device="cuda"))
    fewer, _ = _evict(b, 85, 9, 2)
    assert fewer.tolist() == [80, 85, 33]
    fewer, _ = _evict(b, 40, 9, 2, max_length=5000)
    assert fewer.tolist() == [40, 40, 33]


def test_evict_lost_pages(hip_ready):
    """Slots of pages outside the cache weigh least, and nothing is read or written there."""
    b = Batch(BF16, 1, 1, 16, 8, [80, 64]).fill()
    kc = b.kc.clone()
    w = b.w.clone()
    indices = b.indices.clone()
    indices[4], indices[1] = b.pages, -1          # positions 32 .. 39, 8 .. 15 of the first
    fewer, kept = at.paged_evict(b.w, b.kc, b.vc, b.indptr, indices, b.lengths, keep=40, recent=8,
                                 max_length=80)
    assert fewer.tolist() == [40, 40]
    page, slot = b.places(0)
    weights = w[page, slot, 0].tolist()
    for p in list(range(8, 16)) + list(range(32, 40)):
        weights[p] = -math.inf
    want = _kept(weights, 80, 40, 8, 0)
    assert kept[0, 0].tolist() == want
    for i, p in enumerate(want):
        if i // 8 not in (1, 4) and p // 8 not in (1, 4):
            assert torch.equal(b.kc[page[i], slot[i]], kc[page[p], slot[p]]), i
    assert torch.equal(b.kc[b.indices[[1, 4]]].nan_to_num(-7), kc[b.indices[[1, 4]]].nan_to_num(-7))


def test_a_cache_without_pages(hip_ready):
    """Nothing is read or written; what is kept are the first, the recent and the first between."""
    b = Batch(BF16, 2, 2, 16, 8, [80, 5], [3, 1]).fill()
    lse = b.lse()
    kc, vc, w = b.kc[:0], b.vc[:0], b.w[:0]
    at.attention_weights(b.query, lse, kc, w, b.indptr, b.indices, b.lengths, max_length=80,
                         query_indptr=b.ends, max_query=3)
    fewer, kept = at.paged_evict(w, kc, vc, b.indptr, b.indices, b.lengths, keep=20, recent=4,
                                 first=2, max_length=80)
    assert fewer.tolist() == [20, 5]
    assert kept[0, 0].tolist() == list(range(16)) + [76, 77, 78, 79]
    assert kept[1, 1].tolist() == list(range(5)) + [-1] * 15
    frequency, _ = at.rope_frequencies(16)
    q = at.paged_append(b.key, b.value, kc, vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query, query_indptr=b.ends, epsilon=EPSILON)
    assert q.any()


def test_strides_of_weights_and_caches(hip_ready):
    """Caches and weights inside larger arrays; what lies between is left alone."""
    b = Batch(BF16, 4, 2, 64, 16, [90, 33], [2, 1]).fill()
    wide = [torch.zeros(b.pages, 2, 19, 70, device="cuda", dtype=BF16) for _ in range(2)]
    kc, vc = (x[:, :, 1:17, 3:67].transpose(1, 2) for x in wide)
    kc.copy_(b.kc), vc.copy_(b.vc)
    loose = torch.zeros(16, b.pages, 5, device="cuda")
    w = loose[:, :, 1:4:2].transpose(0, 1)
    w.copy_(b.w)
    lse = b.lse()
    wide_lse = torch.zeros(3, 9, device="cuda")[:, 1::2]
    wide_lse.copy_(lse)
    args = (b.indptr, b.indices, b.lengths)
    at.attention_weights(b.query, wide_lse, kc, w, *args, max_length=90, query_indptr=b.ends,
                         max_query=2)
    b.weigh(lse)
    assert torch.equal(w.nan_to_num(-7), b.w.nan_to_num(-7))
    got = at.paged_evict(w, kc, vc, *args, keep=30, recent=7, max_length=90)
    want = at.paged_evict(b.w, b.kc, b.vc, *args, keep=30, recent=7, max_length=90)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    for x, y in ((w, b.w), (kc, b.kc), (vc, b.vc)):
        assert torch.equal(x.nan_to_num(-7), y.nan_to_num(-7))
    kc.zero_(), vc.zero_(), w.zero_()
    assert not any(x.any() for x in wide + [loose])


def test_cache_past_32_bits(hip_ready):
    """Pages whose elements, and weights, stand past 2^32 bytes."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("not enough memory")
    page, kv_heads, dim = 16, 2, 128
    pages = (1 << 32) // (page * kv_heads * dim) + 4
    kc = torch.zeros(pages, page, kv_heads, dim, device="cuda", dtype=BF16)
    vc = torch.zeros_like(kc)
    far = torch.zeros(pages, 1 << 9, device="cuda")           # 2^20 pages, 2^11 bytes each
    w = far[:, :page * kv_heads].reshape(pages, page, kv_heads)
    if w.data_ptr() != far.data_ptr():
        w = far.as_strided((pages, page, kv_heads), (1 << 9, kv_heads, 1))
    b = Batch(BF16, 4, 2, 128, 16, [90, 33], [2, 1]).fill()
    last = torch.arange(pages - b.pages, pages, device="cuda")
    kc[last], vc[last] = b.kc, b.vc
    w[last] = b.w
    lse = b.lse()
    indices = last[b.indices]
    at.attention_weights(b.query, lse, kc, w, b.indptr, indices, b.lengths, max_length=90,
                         query_indptr=b.ends, max_query=2)
    b.weigh(lse)
    assert torch.equal(w[last].nan_to_num(-7), b.w.nan_to_num(-7))
    at.paged_evict(w, kc, vc, b.indptr, indices, b.lengths, keep=30, recent=7, max_length=90)
    at.paged_evict(b.w, b.kc, b.vc, b.indptr, b.indices, b.lengths, keep=30, recent=7,
                   max_length=90)
    assert torch.equal(kc[last].nan_to_num(-7), b.kc.nan_to_num(-7))
    assert torch.equal(w[last].nan_to_num(-7), b.w.nan_to_num(-7))
    assert not kc[0].any()
    frequency, _ = at.rope_frequencies(dim)
    at.paged_append(b.key, b.value, kc, vc, b.indptr, indices, b.lengths, frequency,
                    query_indptr=b.ends, epsilon=EPSILON)
    at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                    query_indptr=b.ends, epsilon=EPSILON)
    assert torch.equal(kc[last].nan_to_num(-7), b.kc.nan_to_num(-7))
    assert torch.equal(vc[last].nan_to_num(-7), b.vc.nan_to_num(-7))


def _far(near, pages, stride):
    """The same values with pages `stride` elements apart, in memory that nothing else needs."""
    far = torch.empty((pages - 1) * stride + near[0].numel(), dtype=near.dtype, device="cuda")
    far = far.as_strided(near.shape, (stride,) + near[0].contiguous().stride())
    far.copy_(near)
    return far


@pytest.mark.parametrize("bounds,group", [(dict(max_query=1), 20), (dict(), 20),
                                          (dict(max_query=1, max_length=10), 1)])
def test_cache_past_2_to_the_32_elements(hip_ready, bounds, group):
    """Keys, values and weights past 2^32 elements: few rows and many, rows in parts, eviction in two
    launches and in one, the append."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    b = Batch(BF16, 2 * group, 2, 64, 512, [5000, 4300, 600], [40, 30, 1], side_by_side=False)
    b.fill()
    stride = (1 << 28) + 1024
    assert (b.pages - 1) * stride > 1 << 32
    lse = b.lse()
    kc, vc, w = (_far(x, b.pages, stride) for x in (b.kc, b.vc, b.w))
    frequency, _ = at.rope_frequencies(64)

    def both(call):
        table = (b.indptr, b.indices, b.lengths)
        return call(kc, vc, w, *table), call(b.kc, b.vc, b.w, *table)

    def same():
        for x, y in ((kc, b.kc), (vc, b.vc), (w, b.w)):
            assert torch.equal(x.nan_to_num(-7), y.nan_to_num(-7))

    how = dict(dict(max_query=40, max_length=5000), **bounds)
    both(lambda kc, vc, w, *table: at.attention_weights(b.query, lse, kc, w, *table,
                                                        query_indptr=b.ends, **how))
    same()
    both(lambda kc, vc, w, *table: at.paged_append(b.key, b.value, kc, vc, *table, frequency,
                                                   query_indptr=b.ends, epsilon=EPSILON))
    same()
    for keep in (4200, 1500, 700):
        (fewer, kept), (want, moved) = both(lambda kc, vc, w, *table: at.paged_evict(
            w, kc, vc, *table, keep=keep, recent=100, first=3, max_length=int(b.lengths.max())))
        assert torch.equal(fewer, want) and torch.equal(kept, moved)
        same()
        b.lengths.copy_(fewer)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotary", [64, 22])
def test_norm_rope_past_2_to_the_32_elements(hip_ready, rotary, layout):
    """Rows of tokens, and of heads, that far apart: forward into such rows, backward, the append."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    far, g = (1 << 30) + 512, _gen(5)
    frequency, _ = at.rope_frequencies(rotary)
    positions = torch.arange(6, device="cuda")
    q, k, gq, gk = (_normal(g, 6, 6, 64, dtype=BF16) for _ in range(4))
    wq, wk = (_weights(g, "one", 1, 64, F32) for _ in range(2))
    how = dict(layout=layout, epsilon=EPSILON)
    # (one array for all, so that each starts elsewhere in it)
    space = torch.empty(5 * far + (1 << 17), device="cuda", dtype=BF16)

    def apart(x, tokens, start):
        strides = (far, 64, 1) if tokens else (64, far, 1)
        y = space[start << 14:].as_strided(x.shape, strides)
        return y.copy_(x)

    for tokens in (True, False):
        want = at.norm_rope(q, k, positions, frequency, wq, wk, **how)
        out = tuple(apart(torch.zeros_like(x), tokens, i) for i, x in enumerate((q, k)))
        x, y = apart(q, tokens, 2), apart(k, tokens, 3)
        at.norm_rope(x, y, positions, frequency, wq, wk, query_out=out[0], key_out=out[1], **how)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        gx, gy = apart(gq, tokens, 4), apart(gk, tokens, 5)
        want = at.norm_rope_backward(gq, gk, q, k, positions, frequency, wq, wk, **how)
        got = at.norm_rope_backward(gx, gy, x, y, positions, frequency, wq, wk, **how)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        b = Batch(BF16, 6, 6, 64, 16, [9, 5, 1, 40, 2, 17], [1] * 6).fill()
        table = (b.indptr, b.indices, b.lengths, frequency)
        kc, vc = b.kc.clone(), b.vc.clone()
        append = dict(how, query_weight=wq, key_weight=wk)
        got = at.paged_append(y, gy, kc, vc, *table, query=x, query_out=out[0], **append)
        want = at.paged_append(k, gk, b.kc, b.vc, *table, query=q, **append)
        assert torch.equal(got, want)
        for u, v in ((kc, b.kc), (vc, b.vc)):
            assert torch.equal(u.nan_to_num(-7), v.nan_to_num(-7))


# --------------------------------------------------------------------------- #
# together
# --------------------------------------------------------------------------- #
def _loop(b, frequency, wq, wk, shift, none, keep):
    """One step of a bounded cache: append, attend, weigh, evict."""
    q = at.paged_append(b.key, b.value, b.kc, b.vc, b.indptr, b.indices, b.lengths, frequency,
                        query=b.query, query_weight=wq, key_weight=wk, epsilon=EPSILON,
                        shift=shift)
    out, lse = at.prefix_attention(q, b.kc, b.vc, none, 0, b.indptr, b.indices, b.lengths,
                                   max_length=64, return_lse=True)
    at.attention_weights(q, lse, b.kc, b.w, b.indptr, b.indices, b.lengths, max_length=64)
    fewer, kept = at.paged_evict(b.w, b.kc, b.vc, b.indptr, b.indices, b.lengths, keep=keep,
                                 recent=5, first=2, max_length=64)
    shift += b.lengths - fewer
    b.lengths.copy_(fewer)
    return out, kept


def _bounded():
    b = Batch(BF16, 8, 2, 64, 16, [64, 64, 64], [1, 1, 1], seed=4)
    b.kc.zero_(), b.vc.zero_(), b.w.zero_()
    b.lengths.copy_(torch.tensor([0, 3, 11], device="cuda"))
    frequency, _ = at.rope_frequencies(64)
    wq, wk = (_weights(b.g, "one", 1, 64, BF16) for _ in range(2))
    return (b, frequency, wq, wk, torch.zeros_like(b.lengths),
            torch.empty(0, dtype=torch.int64, device="cuda"))


def test_a_bounded_cache(hip_ready):
    """The loop against lists of tokens: what is kept, and attention over it.  The lists follow the
    device's own weights (they are tested above), so that every choice is theirs."""
    b, frequency, wq, wk, shift, none = _bounded()
    keep, G = 17, 4
    g = _gen(9)
    lists = [[[] for _ in range(2)] for _ in range(3)]     # (key, value) of each position
    start = b.lengths.tolist()
    for s, n in enumerate(start):
        page, slot = (x[:n] for x in b.places(s))
        for h in range(2):
            lists[s][h] = [(_cpu(b.kc[p, t, h]), _cpu(b.vc[p, t, h])) for p, t in zip(page, slot)]
    for step in range(40):
        for x in (b.query, b.key, b.value):
            x.copy_(_normal(g, *x.shape, dtype=BF16))
        b.lengths += 1
        position = (b.lengths - 1 + shift).clone()
        out, kept = _loop(b, frequency, wq, wk, shift, none, keep)
        keys = _turned(_normed(b.key, wk), position, frequency, "half", 1.0)[0]
        queries = _turned(_normed(b.query, wq), position, frequency, "half", 1.0)[0]
        for s in range(3):
            for h in range(2):
                tokens = lists[s][h]
                tokens.append((keys[s, h], _cpu(b.value[s, h])))
                k, v = (torch.stack([t[i] for t in tokens]) for i in range(2))
                for q in range(h * G, (h + 1) * G):
                    score = k @ queries[s, q] / 8
                    # queries and keys are rounded to bfloat16, probabilities too
                    es = float((k.abs() @ queries[s, q].abs()).max()) / 8 * (
                        2 * U[BF16] + 2.0 ** -16)
                    p = torch.softmax(score, 0)
                    size = p @ v.abs()
                    bound = 2 * U[BF16] * size + (math.exp(2 * es) - 1) * size
                    assert ((_cpu(out[s, q]) - p @ v).abs() <= bound).all(), (step, s, q)
                lists[s][h] = [tokens[i] for i in kept[s, h].tolist() if i >= 0]
    assert b.lengths.tolist() == [keep] * 3
    assert shift.tolist() == [max(0, n + 40 - keep) for n in start]


def test_a_bounded_cache_in_a_graph(hip_ready):
    b, *rest = _bounded()
    eager, *others = _bounded()
    for x in (b, eager):
        x.lengths += 1
    _loop(b, *rest, 17)
    _loop(eager, *others, 17)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, kept = _loop(b, *rest, 17)
    for i in range(25):
        for x in (b, eager):
            x.lengths += 1
            x.query.copy_(_normal(_gen(i), *x.query.shape, dtype=BF16))
            x.key.copy_(_normal(_gen(100 + i), *x.key.shape, dtype=BF16))
        graph.replay()
        want, places = _loop(eager, *others, 17)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kept, places), i
        assert torch.equal(b.lengths, eager.lengths) and torch.equal(b.w, eager.w)
    assert torch.equal(b.kc, eager.kc)


@pytest.mark.parametrize("norm,bound,recent,first", [(True, 0, None, 0), (False, 12, 4, 1),
                                                     (True, 10, None, 2)])
def test_paged_decode_with_norms_and_a_bound(hip_ready, norm, bound, recent, first):
    """The decode loop of tilegen_amd.paged_decode, against attention over what each kv head has kept
    of its unrotated inputs in 64 bits.  Keys and queries are rounded once, to bfloat16 (and off by
    the norm's and the rotation's errors): a score is off by at most S = scale sum (dk |q| + |k| dq +
    dk dq) + dim 2^-23 scale sum |k q|, an output, with probabilities and itself rounded, by 2 u + exp
    2 S - 1 of its sum of magnitudes.  A key's weight is off by exp(2 S + 2^-16) - 1 of itself: its at
    most 60 terms, the exponents' size below 64 and the exponential come to less than 2^-16."""
    from tilegen_amd import paged_decode
    heads, kv_heads, dim, prompt, every, steps = 4, 2, 64, 50, 5, 21
    r = paged_decode.run(sequences=3, prompt=prompt, steps=steps, heads=heads, kv_heads=kv_heads,
                         dim=dim, page=16, start=20, seed=5, keep=True, norm=norm, bound=bound,
                         recent=recent, first=first, every=every)
    f, magnitude, counts, u = r["frequency"], r["magnitude"], r["counts"], U[BF16]
    learned = r["norm"] or {}
    recent = bound // 4 if recent is None else recent
    assert (r["norm"] is not None) == norm and len(r["calls"]) == steps + 1
    assert [call for call, _ in r["stayed"]] == ([0, 5, 10, 15, 20] if bound else [])

    def made(x, which, positions):
        """(normed and turned in 64 bits, by how much the calls' may be off)"""
        z, N = _cpu(x), 0.0
        if norm:
            z, N = _normed(x, learned[which], learned["epsilon"]), (dim / 2 + 8) * E
        y, size = _turned(z, torch.tensor(positions), f, "half", magnitude)
        return y, u * y.abs() + (2.0 ** -21 + N) * size

    shared, eshared = made(r["prompt"][0], "key_weight", list(range(prompt)))
    vshared = _cpu(r["prompt"][1])
    own = [[(torch.empty(0, dim, dtype=torch.float64),) * 3] * kv_heads for _ in range(3)]
    weight = [[torch.zeros(2, 0, dtype=torch.float64)] * kv_heads for _ in range(3)]  # and bounds
    seen, stayed = [0, 0, 0], dict(r["stayed"])
    for call, (q, k, v, out) in enumerate(r["calls"]):
        n = counts if call == 0 else [1, 1, 1]
        row = 0
        for b in range(3):
            mine = slice(row, row + n[b])
            at_ = [prompt + seen[b] + j for j in range(n[b])]
            (ks, eks), (qs, eqs) = made(k[mine], "key_weight", at_), made(q[mine], "query_weight", at_)
            vs = _cpu(v[mine])
            for h in range(kv_heads):
                key, ekey, value = (torch.cat([a, x[:, h]])
                                    for a, x in zip(own[b][h], (ks, eks, vs)))
                own[b][h] = key, ekey, value
                weight[b][h] = torch.cat([weight[b][h], torch.zeros(2, n[b])], 1)
                for j in range(n[b]):
                    see = key.shape[0] - n[b] + j + 1
                    kh = torch.cat([shared[:, h], key[:see]])
                    ek = torch.cat([eshared[:, h], ekey[:see]])
                    vh = torch.cat([vshared[:, h], value[:see]])
                    for g in range(2 * h, 2 * h + 2):
                        qh, eq = qs[j, g], eqs[j, g]
                        p = torch.softmax(kh @ qh / 8, 0)
                        S = float((ek @ qh.abs() + kh.abs() @ eq + ek @ eq
                                   + dim * 2.0 ** -23 * (kh.abs() @ qh.abs())).max()) / 8
                        size = p @ vh.abs()
                        bound_ = (2 * u + math.exp(2 * S) - 1) * size
                        off = (_cpu(out[row + j, g]) - p @ vh).abs()
                        assert (off <= bound_ * (1 + 2.0 ** -6)).all(), (call, b, j, g)
                        weight[b][h][0, :see] += p[prompt:]
                        weight[b][h][1, :see] += p[prompt:] * (math.exp(2 * S + 2.0 ** -16) - 1)
            row += n[b]
            seen[b] += n[b]
            length = own[b][0][0].shape[0]
            if call not in stayed:
                continue
            for h in range(kv_heads):
                where = stayed[call][b, h].tolist()
                there = [p for p in where if p >= 0]
                assert len(there) == min(length, bound) and where[len(there):] == [-1] * (
                    bound - len(there))
                kept = set(there)
                assert len(kept) == len(there) and max(there) < length
                if length > bound:
                    always = set(range(first)) | set(range(length - recent, length))
                    w, e = weight[b][h]
                    left = [p for p in range(length) if p not in kept]
                    chosen = [p for p in there if p not in always]
                    assert always <= kept and chosen
                    assert float((w + e)[chosen].min()) >= float((w - e)[left].max())
                own[b][h] = tuple(x[there] for x in own[b][h])
                weight[b][h] = weight[b][h][:, there]
    cache = r["cache"]
    assert seen == [n + steps for n in counts]
    if bound:
        assert cache.capacity == 20 and cache.lengths.tolist() == [bound + steps % every] * 3
        assert (cache.lengths + cache.shift).tolist() == seen
    else:
        assert cache.lengths.tolist() == seen and cache.shift is None


def test_norms_in_a_graph_and_on_streams(hip_ready):
    """Forward and backward calls captured, replayed, and two streams at once."""
    g = _gen(3)
    frequency, _ = at.rope_frequencies(128)
    q, k = _normal(g, 600, 12, 128, dtype=BF16), _normal(g, 600, 4, 128, dtype=BF16)
    gq, gk = _normal(g, 600, 12, 128, dtype=BF16), _normal(g, 600, 4, 128, dtype=BF16)
    wq, wk = (_weights(g, "one", 1, 128, BF16) for _ in range(2))
    positions = torch.arange(600, device="cuda")

    def both():
        return at.norm_rope(q, k, positions, frequency, wq, wk) + at.norm_rope_backward(
            gq, gk, q, k, positions, frequency, wq, wk)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(4):
        q.copy_(_normal(g, *q.shape, dtype=BF16))
        gk.copy_(_normal(g, *gk.shape, dtype=BF16))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r in results for x, y in zip(r, want))


# --------------------------------------------------------------------------- #
# refusals
# --------------------------------------------------------------------------- #
def test_refusals(hip_ready):
    frequency, _ = at.rope_frequencies(64)
    x = torch.zeros(3, 4, 64, device="cuda", dtype=BF16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=BF16)
    n = torch.arange(3, device="cuda")
    w = torch.ones(64, device="cuda", dtype=BF16)

    def no(words, call, *args, **more):
        with pytest.raises(ValueError, match=words):
            call(*args, **more)

    norm = at.norm_rope
    no("query", norm, x.double(), k, n, frequency)
    no("key", norm, x, k.float(), n, frequency)
    no("key", norm, x, k[:2], n, frequency)
    no("query_weight", norm, x, k, n, frequency, w[:32])
    no("query_weight", norm, x, k, n, frequency, w.half())
    no("query_weight", norm, x, k, n, frequency, w.expand(3, 64))
    no("key_weight", norm, x, k, n, frequency, w, w.float())
    no("key_weight", norm, x, None, n, frequency, w, w)
    no("positions", norm, x, k, None, frequency)
    no("positions", norm, x, k, n[:2], frequency)
    no("epsilon", norm, x, k, n, frequency, epsilon=-1e-6)
    no("epsilon", norm, x, k, n, frequency, epsilon=math.nan)
    no("layout", norm, x, k, n, frequency, layout="thirds")
    no("number", norm, x, k, n, frequency, epsilon=None)
    no("rotary", norm, x[..., :32], k[..., :32], n, frequency)
    wide = torch.zeros(3, 4, 264, device="cuda", dtype=BF16)
    no("dim", norm, wide, None, n, frequency)
    no("query_out", norm, x, k, n, frequency, query_out=x[:2])
    no("overlaps", norm, x, k, n, frequency, key_out=x[:, :2])
    no("overlaps", norm, x[:, 1:], k, n, frequency, query_out=x[:, :3])
    no("share memory", norm, x, k, n, frequency, key_out=k[:, :1].expand(3, 2, 64))
    no("grad_query", at.norm_rope_backward, x[:2], k, x, k, n, frequency)
    no("grad_key", at.norm_rope_backward, x, k, x, None, n, frequency)
    leaf = x.clone().requires_grad_()
    no("out", norm, leaf, k, n, frequency, query_out=torch.empty_like(x))
    no("norm_rope", norm, x, k, n, frequency.clone().requires_grad_())
    no("backward", at.norm_rope_backward, leaf, k, x, k, n, frequency)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        no("forward", norm, dual, k, n, frequency)
    y = norm(leaf, None, n, frequency, w)[0]
    grad, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()

    b = Batch(BF16, 4, 2, 64, 16, [5, 17, 32], [1, 1, 1]).fill()
    table = (b.indptr, b.indices, b.lengths)

    def append(**more):
        return at.paged_append(b.key, b.value, b.kc, b.vc, *table, frequency, query=b.query,
                               **more)

    no("epsilon", append, query_weight=w)
    no("epsilon", append, query_weight=w, shift=b.lengths)
    no("shift", append, shift=b.lengths[:2])
    no("shift", append, shift=b.lengths.int())
    no("epsilon", append, epsilon=-1.0)
    no("key_weight", append, epsilon=1e-6, key_weight=w[:3])
    no("query_weight", at.paged_append, b.key, b.value, b.kc, b.vc, *table, frequency,
       query_weight=w, epsilon=1e-6)
    no("backward", append, epsilon=1e-6, key_weight=w.clone().requires_grad_())

    lse = b.lse()

    def weigh(query=b.query, lse=lse, kc=b.kc, w=b.w, **more):
        return at.attention_weights(query, lse, kc, w, *table, **dict(dict(max_length=32), **more))

    no("query", weigh, query=b.query.float(), kc=b.kc.float())
    no("lse", weigh, lse=lse[:, :2])
    no("lse", weigh, lse=lse.double())
    no("weights", weigh, w=b.w.half())
    no("weights", weigh, w=b.w[:, :8])
    no("share memory", weigh, w=b.w[:, :1].expand(b.w.shape))
    no("cache", weigh, query=b.query[..., :32])
    no("scale", weigh, scale=0.0)
    no("scale", weigh, scale=1e-60)
    no("decay", weigh, decay=-0.5)
    no("decay", weigh, decay=math.inf)
    no("negative", weigh, max_length=-1)
    no("backward", weigh, query=b.query.clone().requires_grad_())
    inside = b.kc.view(torch.float32)[..., 0]
    no("overlaps", weigh, w=inside)

    def evict(w=b.w, kc=b.kc, vc=b.vc, **more):
        return at.paged_evict(w, kc, vc, *table, **dict(dict(keep=10, max_length=32), **more))

    no("weights", evict, w=b.w.double())
    no("keep", evict, keep=-1)
    no("keep", evict, keep=1 << 23)
    no("more than keep", evict, recent=11)
    no("more than keep", evict, recent=6, first=5)
    no("negative", evict, recent=-1)
    no("value_cache", evict, vc=b.vc[:-1])
    no("overlaps", evict, vc=b.kc)
    no("overlaps", evict, w=inside)
    no("2\\^30", evict, max_length=1 << 40)
    no("backward", evict, vc=b.vc.clone().requires_grad_())


def test_autograd_notices_what_the_calls_write(hip_ready):
    b = Batch(BF16, 4, 2, 64, 16, [40, 17], [1, 1]).fill()
    versions = [x._version for x in (b.w, b.kc, b.vc)]
    b.weigh(b.lse())
    at.paged_evict(b.w, b.kc, b.vc, b.indptr, b.indices, b.lengths, keep=9, max_length=40)
    now = [x._version for x in (b.w, b.kc, b.vc)]
    assert now[0] >= versions[0] + 2 and now[1] > versions[1] and now[2] > versions[2]
