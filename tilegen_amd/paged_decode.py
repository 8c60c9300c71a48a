"""Decoding behind a shared prompt, with the cache and attention of ``tilegen_amd.attention``:
``python -m tilegen_amd.paged_decode [--sequences 32 --prompt 8192 --steps 64 ...]``.

One layer of attention with random projections.  The prompt's keys and values go to the pages of
the shared prefix once; then every step projects the sequences' last vectors, appends their
keys and values to each sequence's own pages, rotated, with the queries, attends over prefix and own
pages, and feeds the result on.  Sequences start with answers of different lengths, and all pages
come from one pool in random order, as a server's do.
"""

from __future__ import annotations

import argparse
from typing import Dict, List

import torch

from . import attention

__all__ = ["Cache", "run"]


class Cache:
    """Pages of keys and values, the shared prefix's list and the page table (CSR) of sequences
    that may grow to ``capacity`` tokens of their own each."""

    def __init__(self, sequences: int, prompt: int, capacity: int, page: int, kv_heads: int,
                 dim: int, dtype: torch.dtype, generator: torch.Generator):
        shared, each = -(-prompt // page), -(-capacity // page)
        pool = torch.randperm(shared + sequences * each, generator=generator, device="cuda")
        shape = (pool.numel(), page, kv_heads, dim)
        self.keys = torch.zeros(shape, dtype=dtype, device="cuda")
        self.values = torch.zeros(shape, dtype=dtype, device="cuda")
        self.prefix, self.prompt = pool[:shared].contiguous(), prompt
        self.indices = pool[shared:].contiguous()
        self.indptr = torch.arange(sequences + 1, device="cuda") * each
        self.lengths = torch.zeros(sequences, dtype=torch.int64, device="cuda")
        self.capacity = capacity

    def fill_prompt(self, key, value, frequency, magnitude):
        """The prompt as one sequence whose pages are the prefix's."""
        ends = torch.tensor([0, self.prompt], device="cuda")
        attention.paged_append(
            key, value, self.keys, self.values,
            torch.tensor([0, self.prefix.numel()], device="cuda"), self.prefix, ends[1:],
            frequency, query_indptr=ends, magnitude=magnitude)

    def append(self, key, value, query, frequency, magnitude, query_indptr=None):
        return attention.paged_append(
            key, value, self.keys, self.values, self.indptr, self.indices, self.lengths,
            frequency, query=query, query_indptr=query_indptr, offset=self.prompt,
            magnitude=magnitude)

    def attend(self, query, query_indptr=None, max_query=1):
        return attention.prefix_attention(
            query, self.keys, self.values, self.prefix, self.prompt, self.indptr, self.indices,
            self.lengths, query_indptr=query_indptr, max_query=max_query,
            max_length=self.capacity)


def run(sequences: int = 32, prompt: int = 8192, steps: int = 64, heads: int = 32,
        kv_heads: int = 8, dim: int = 128, page: int = 16, start: int = 24, seed: int = 0,
        keep: bool = False) -> Dict[str, object]:
    """Decodes ``steps`` tokens for each sequence after first answers of 1 to ``start`` tokens;
    {"us_per_step"} and, with ``keep``, what went in and came out: the prompt's keys and values, the
    first answers' counts, and every call's (query, key, value, result), none rotated."""
    for name, n, least in (("sequences", sequences, 1), ("start", start, 1), ("prompt", prompt, 0),
                           ("steps", steps, 0)):
        if n < least:
            raise ValueError("%s is %d, expected at least %d" % (name, n, least))
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    width = heads * dim
    project = normal(width, (heads + 2 * kv_heads) * dim, scale=width ** -0.5)
    frequency, magnitude = attention.rope_frequencies(dim, scaling="yarn", factor=8, trained=4096)
    cache = Cache(sequences, prompt, start + steps, page, kv_heads, dim, dtype, g)
    kept: List[tuple] = []

    def split(x):
        y = (x.reshape(-1, width) @ project).view(-1, heads + 2 * kv_heads, dim)
        return y[:, :heads], y[:, heads:heads + kv_heads], y[:, heads + kv_heads:]

    _, key, value = split(normal(prompt, width))
    cache.fill_prompt(key, value, frequency, magnitude)
    # the first answers' tokens, all at once
    counts = [1 + i * (start - 1) // max(1, sequences - 1) for i in range(sequences)]
    ends = torch.tensor([0] + counts, device="cuda").cumsum(0)
    cache.lengths += ends.diff()
    q, k, v = split(normal(sum(counts), width))
    out = cache.attend(cache.append(k, v, q, frequency, magnitude, ends), ends, max(counts))
    if keep:
        kept.append((q, k, v, out))
    x = out[ends[1:] - 1]
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(steps):
        cache.lengths += 1
        q, k, v = split(x)
        out = cache.attend(cache.append(k, v, q, frequency, magnitude))
        if keep:
            kept.append((q, k, v, out))
        # the next input: the result, at the size that the projection expects
        x = (out.float() * (dim ** 0.5 / out.float().norm(dim=-1, keepdim=True))).to(dtype)
    end.record()
    end.synchronize()
    result: Dict[str, object] = {"us_per_step": 1e3 * begin.elapsed_time(end) / max(1, steps)}
    if keep:
        result.update(prompt=(key, value), counts=counts, calls=kept, frequency=frequency,
                      magnitude=magnitude)
    return result


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("sequences", 32), ("prompt", 8192), ("steps", 64), ("heads", 32),
                          ("kv-heads", 8), ("dim", 128), ("page", 16), ("start", 24)):
        ap.add_argument("--" + name, type=int, default=default)
    a = vars(ap.parse_args(argv))
    print("%(sequences)d sequences behind %(prompt)d shared tokens" % a, end=": ", flush=True)
    run(**dict(a, steps=2))     # loads the library and the projection's kernels
    print("%.1f us a step" % run(**a)["us_per_step"], flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
