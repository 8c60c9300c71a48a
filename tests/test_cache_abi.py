"""libtgcache.so without a GPU: its exports, the structures that the binding packs, refusals and
spills."""

from __future__ import annotations

import math
import os
import re
import subprocess

import pytest
import torch

from tilegen_amd import attention as at
from tilegen_amd import build, runtime

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "tilegen_cache.h")
PACKED = {"tg_norm_rope": at._NORM, "tg_norm_rope_backward": at._NORM_BACKWARD,
          "tg_paged_append_normed": at._APPEND_NORMED, "tg_attention_weights": at._WEIGHTS,
          "tg_paged_evict": at._EVICT}
MOST = (1 << 63) - 1


def _fields(name):
    """[(field, struct code)] of a structure in the header."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
    fields = []
    for line in body.split(";"):    # no field list mixes pointers and numbers
        if line.strip():
            kind = "P" if "*" in line else "d" if "double" in line else "q"
            fields += [(re.search(r"(\w+)\s*$", f).group(1), kind) for f in line.split(",")]
    return fields


class Call:
    """A structure by its fields' names."""

    def __init__(self, struct, entry, **base):
        self.struct, self.entry, self.base = struct, entry, base
        self.names = [f for f, _ in _fields(struct)]

    def pack(self, **change):
        values = dict.fromkeys(self.names, 0)
        values.update(self.base)
        assert set(change) <= set(values), change
        values.update(change)
        return PACKED[self.struct].pack(*(values[n] for n in self.names))

    def __call__(self, **change):
        """(status, message)"""
        rc = getattr(at._cache_lib(), self.entry)(self.pack(**change), None)
        return rc, runtime.last_error()


NORM = Call("tg_norm_rope", "launch_norm_rope", tokens=4, heads=2, kv_heads=1, dim=64, rotary=64,
            query_token=128, query_head=64, key_token=64, key_head=64, qout_token=128, qout_head=64,
            kout_token=64, kout_head=64, magnitude=1.0, epsilon=1e-6)
BACK = Call("tg_norm_rope_backward", "launch_norm_rope_backward", tokens=40, heads=2, kv_heads=1,
            dim=64, rotary=64, query_token=128, query_head=64, key_token=64, key_head=64,
            grad_query_token=128, grad_query_head=64, grad_key_token=64, grad_key_head=64,
            qout_token=128, qout_head=64, kout_token=64, kout_head=64, magnitude=1.0, epsilon=1e-6)
APPEND = Call("tg_paged_append_normed", "launch_paged_append_normed", tokens=4, sequences=4,
              heads=2, kv_heads=1, dim=64, rotary=64, pages=9, page=16, n_indices=9, normed=1,
              key_token=64, key_head=64, value_token=64, value_head=64, query_token=128,
              query_head=64, out_token=128, out_head=64, kc_page=1024, kc_slot=64, kc_head=64,
              vc_page=1024, vc_slot=64, vc_head=64, magnitude=1.0, epsilon=1e-6)
WEIGHTS = Call("tg_attention_weights", "launch_attention_weights", tokens=2, sequences=2, heads=4,
               kv_heads=2, dim=64, pages=9, page=16, n_indices=4, max_query=1, max_length=20,
               query_token=256, query_head=64, lse_token=4, lse_head=1, kc_page=2048, kc_slot=128,
               kc_head=64, w_page=32, w_slot=2, w_head=1, scale=0.125, decay=1.0)
EVICT = Call("tg_paged_evict", "launch_paged_evict", sequences=2, kv_heads=2, dim=64, pages=9,
             page=16, n_indices=4, max_length=20, keep=10, recent=2, first=1, kc_page=2048,
             kc_slot=128, kc_head=64, vc_page=2048, vc_slot=128, vc_head=64, w_page=32, w_slot=2,
             w_head=1)


def test_exports_what_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(\w+)\(const tg_\w+\*", text))
    assert declared == {"launch_norm_rope", "launch_norm_rope_backward",
                        "norm_rope_backward_workspace", "launch_paged_append_normed",
                        "launch_attention_weights", "attention_weights_workspace",
                        "launch_paged_evict"}
    out = subprocess.run(["nm", "-D", "--defined-only",
                          os.path.join(runtime.lib_dir(), "libtgcache.so")],
                         capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert declared <= exported
    assert all(s in declared or s.startswith("_") for s in exported), exported


def test_packed_fields_follow_the_header():
    for name, packed in PACKED.items():
        codes = "".join(kind for _, kind in _fields(name))
        flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Pqd])", packed.format))
        assert codes == flat, name
        assert packed.size == 8 * len(codes)


@pytest.mark.parametrize("call,changes", [
    (NORM, [(dict(), "null"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
            (dict(weight_dtype=1), "weights"), (dict(dim=0), "dim"), (dict(dim=257), "dim"),
            (dict(rotary=66), "rotary"), (dict(rotary=7), "rotary"), (dict(layout=2), "layout"),
            (dict(tokens=-1), "negative"), (dict(heads=-1), "negative"),
            (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=math.nan), "epsilon"),
            (dict(epsilon=math.inf), "epsilon"),
            (dict(query=4096, query_out=4098), "overlaps"),
            (dict(query_out=4096, key_out=4096 + 64), "overlaps"),
            (dict(query=4096, key_out=4096), "overlaps"),
            (dict(key=4096, query_out=4096), "overlaps"),
            (dict(query_out=4096, qout_head=32), "share memory")]),
    (BACK, [(dict(), "null"), (dict(dim=257), "dim"), (dict(epsilon=-1.0), "epsilon"),
            (dict(query_weight_out=4096), "without the weight"),
            (dict(grad_query=4096, query_out=4098), "overlaps"),
            (dict(grad_key=4096, query_out=4096), "overlaps"),
            (dict(query=4096, key_out=4096), "overlaps"),
            (dict(key_out=4096, kout_token=32), "share memory")]),
    (APPEND, [(dict(), "null"), (dict(kv_heads=0), "kv_heads"), (dict(normed=2), "normed"),
              (dict(normed=0, key_weight=4096), "without a norm"), (dict(page=0), "page"),
              (dict(sequences=-1), "negative"), (dict(pages=-1), "negative"),
              (dict(sequences=3), "query_indptr"), (dict(dim=300), "dim"),
              (dict(key_cache=1 << 20, value_cache=(1 << 20) + 1024), "overlaps"),
              (dict(query_out=1 << 20, key_cache=1 << 20), "overlaps"),
              (dict(key_cache=1 << 20, kc_slot=32), "share memory")]),
    (WEIGHTS, [(dict(dtype=2), "dtype"), (dict(dim=12), "dim"), (dict(dim=264), "dim"),
               (dict(kv_heads=3), "heads"), (dict(kv_heads=0), "heads"), (dict(page=0), "page"),
               (dict(scale=0.0), "scale"), (dict(scale=1e-60), "scale"),
               (dict(scale=math.nan), "scale"), (dict(decay=-1.0), "decay"),
               (dict(decay=math.nan), "decay"), (dict(tokens=3), "query_indptr"),
               (dict(sequences=-1), "negative"), (dict(max_query=-1), "negative"),
               (dict(max_length=-1), "negative"), (dict(), "null"),
               (dict(weights=1 << 20, key_cache=1 << 20), "overlaps"),
               (dict(weights=1 << 20, lse=(1 << 20) + 4), "overlaps"),
               (dict(weights=1 << 20, query=1 << 20), "overlaps"),
               (dict(weights=1 << 20, w_slot=1), "share memory")]),
    (EVICT, [(dict(dtype=3), "dtype"), (dict(dim=0), "dim"), (dict(dim=1025), "dim"),
             (dict(kv_heads=0), "kv_heads"), (dict(keep=-1), "negative"),
             (dict(recent=-1), "negative"), (dict(first=-1), "negative"),
             (dict(recent=11), "more than keep"), (dict(first=9), "more than keep"),
             (dict(recent=MOST), "more than keep"), (dict(first=MOST), "more than keep"),
             (dict(move_weights=2), "move_weights"), (dict(page=0), "page"), (dict(), "null"),
             (dict(key_cache=1 << 20, value_cache=1 << 20), "overlaps"),
             (dict(key_cache=1 << 20, weights=(1 << 20) + 256), "overlaps"),
             (dict(lengths=1 << 20, lengths_out=(1 << 20) + 8), "overlaps"),
             (dict(value_cache=1 << 20, vc_head=32), "share memory"),
             (dict(weights=1 << 20, w_slot=1, move_weights=1), "share memory")]),
])
def test_bad_arguments(call, changes):
    """Refused on the host, before any HIP call."""
    assert getattr(at._cache_lib(), call.entry)(None, None) == -1
    assert "null" in runtime.last_error()
    for change, word in changes:
        rc, message = call(**change)
        assert rc == -1 and word in message, (change, rc, message)


def test_sizes_beyond_one_launch():
    for call, change in [
            (NORM, dict(tokens=1 << 40)), (NORM, dict(heads=MOST)), (NORM, dict(kv_heads=1 << 20)),
            (BACK, dict(tokens=1 << 40)), (BACK, dict(heads=1 << 30)),
            (APPEND, dict(tokens=1 << 40, sequences=1 << 40)), (APPEND, dict(pages=MOST)),
            (APPEND, dict(sequences=1 << 30)), (WEIGHTS, dict(max_length=1 << 40)),
            (WEIGHTS, dict(tokens=1 << 25, sequences=1 << 25)), (WEIGHTS, dict(pages=1 << 40)),
            (WEIGHTS, dict(heads=1 << 40)), (WEIGHTS, dict(kc_page=MOST)),
            (WEIGHTS, dict(w_slot=-MOST)), (WEIGHTS, dict(tokens=1 << 20, sequences=1 << 20,
                                                          max_length=1 << 20)),
            (EVICT, dict(max_length=1 << 40)), (EVICT, dict(keep=1 << 23)),
            (EVICT, dict(sequences=1 << 30)), (EVICT, dict(w_page=1 << 62)),
            (EVICT, dict(kv_heads=0x10000, sequences=1 << 20, keep=0, recent=0, first=0,
                         indptr=8, lengths=8, lengths_out=1 << 50, indices=8, pages=0))]:
        rc, message = call(**change)
        assert rc == -2, (call.entry, change, rc, message)
    for call, entry in ((BACK, "norm_rope_backward_workspace"),
                        (WEIGHTS, "attention_weights_workspace")):
        ask = getattr(at._cache_lib(), entry)
        assert ask(None) < 0 and ask(call.pack(tokens=-1)) < 0
        assert ask(call.pack(tokens=1 << 40, **({"sequences": 1 << 40} if call is WEIGHTS else {}))
                   ) < 0


def test_nothing_to_do():
    for call, change in [(NORM, dict(tokens=0)), (NORM, dict(heads=0, kv_heads=0)),
                         (BACK, dict(tokens=0)), (BACK, dict(heads=0, kv_heads=0)),
                         (APPEND, dict(tokens=0)), (WEIGHTS, dict(tokens=0, sequences=0)),
                         (WEIGHTS, dict(pages=0)), (WEIGHTS, dict(n_indices=0)),
                         (EVICT, dict(sequences=0))]:
        assert call(**change)[0] == 0, (call.entry, change)


def test_workspaces():
    """Asked for by the sums of the weights' gradients alone."""
    ask = at._cache_lib().norm_rope_backward_workspace
    every = dict(query=1 << 20, key=2 << 20, grad_query=3 << 20, grad_key=4 << 20,
                 query_out=5 << 20, key_out=6 << 20, positions=8, frequency=8, query_weight=8,
                 key_weight=8)
    assert ask(BACK.pack(**every)) == 0
    need = ask(BACK.pack(query_weight_out=8, key_weight_out=8, **every))
    assert need > 0 and need % 4 == 0
    for change, word in [(dict(workspace=4096, workspace_bytes=need - 1), "too small"),
                         (dict(workspace_bytes=need), "too small"),
                         (dict(workspace=4100, workspace_bytes=need), "aligned")]:
        rc, message = BACK(query_weight_out=8, key_weight_out=8, **every, **change)
        assert rc == -1 and word in message


def test_operands_on_the_host_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int64)
    f = torch.zeros(32, dtype=torch.float64)
    cache, w = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2)
    for call in (lambda: at.norm_rope(x, x, n, f), lambda: at.norm_rope_backward(x, x, x, x, n, f),
                 lambda: at.paged_append(x, x, cache, cache, n, n, n, f, epsilon=1e-6),
                 lambda: at.attention_weights(x, w, cache, w, n, n, n, max_length=1),
                 lambda: at.paged_evict(w, cache, cache, n, n, n, keep=1, max_length=1)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_calls_go_by_the_operands_device(monkeypatch):
    """Workspaces' sizes and launches are asked for with the operands' device current, on its stream
    (a stand-in library; host tensors count as device -1)."""
    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.before, current[0] = current[0], self.device

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        def __getattr__(self, name):
            def entry(packed, *stream):
                seen.append((name, current[0]) + stream)
                return 0 if stream else 64
            return entry

    monkeypatch.setattr(at, "_cache_lib", Library)
    monkeypatch.setattr(at, "_operand", lambda name, t, dtypes: (t.get_device(), t.dtype))
    monkeypatch.setattr(at, "_raw_stream", lambda device: 1000 + device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    n, f = torch.zeros(3, dtype=torch.int64), torch.zeros(32, dtype=torch.float64)
    cache, w = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2)
    calls = [
        (lambda: at.norm_rope(x, x, n[:2], f), ["launch_norm_rope"]),
        (lambda: at.norm_rope_backward(x, x, x, x, n[:2], f),
         ["norm_rope_backward_workspace", "launch_norm_rope_backward"]),
        (lambda: at.paged_append(x, x, cache, cache, n, n, n[:2], f, shift=n[:2]),
         ["launch_paged_append_normed"]),
        (lambda: at.attention_weights(x, w[:, 0], cache, w, n, n, n[:2], max_length=1),
         ["attention_weights_workspace", "launch_attention_weights"]),
        (lambda: at.paged_evict(w, cache, cache, n, n, n[:2], keep=1, max_length=1),
         ["launch_paged_evict"])]
    for call, entries in calls:
        for current[0] in (0, -1):
            seen.clear()
            call()
            assert [(e[0], e[1]) for e in seen] == [(name, -1) for name in entries]
            assert seen[-1][2] == 999


def test_append_of_nothing_with_norms(monkeypatch):
    """Whether there is a query is not for its address to say: a batch without tokens, or without
    query heads, has none (a stand-in library; host tensors count as device -1)."""
    seen = []

    class Library:
        def launch_paged_append_normed(self, packed, stream):
            seen.append(dict(zip((f for f, _ in _fields("tg_paged_append_normed")),
                                 at._APPEND_NORMED.unpack(packed))))
            return 0

    monkeypatch.setattr(at, "_cache_lib", Library)
    monkeypatch.setattr(at, "_operand", lambda name, t, dtypes: (t.get_device(), t.dtype))
    monkeypatch.setattr(at, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    n, f = torch.zeros(3, dtype=torch.int64), torch.zeros(32, dtype=torch.float64)
    cache, w = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), torch.ones(64)
    how = dict(query_weight=w, key_weight=w, epsilon=1e-6)
    for key, query, table in ((x[:0], x[:0], (n[:1], n[:0], n[:0])), (x, x[:, :0], (n, n, n[:2]))):
        got = at.paged_append(key, key, cache, cache, *table, f, query=query, **how)
        assert got.shape == query.shape
        assert (seen[-1]["tokens"], seen[-1]["heads"]) == query.shape[:2]
        assert seen[-1]["query_weight"] == seen[-1]["key_weight"] == w.data_ptr()
    with pytest.raises(ValueError, match="query_weight without query"):
        at.paged_append(x, x, cache, cache, n, n, n[:2], f, **how)


def test_backward_needs_both_gradients(monkeypatch):
    monkeypatch.setattr(at, "_operand", lambda name, t, dtypes: (t.get_device(), t.dtype))
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for gq, gk, key in ((None, x, x), (x, None, x), (None, None, None)):
        with pytest.raises(ValueError, match="grad_query" if gq is None else "grad_key"):
            at.norm_rope_backward(gq, gk, x, key, None, None)


def test_kernels_do_not_spill(tmp_path):
    readelf = "/opt/rocm/llvm/bin/llvm-readelf"
    if not os.path.exists(readelf):
        pytest.skip("llvm-readelf not available")
    found = 0
    for co in build.cache_code_objects(str(tmp_path)):
        notes = subprocess.run([readelf, "--notes", co], capture_output=True, text=True,
                               check=True).stdout
        for k in re.split(r"\n\s+- \.", notes):
            name = re.search(r"\.name:\s+(\S+)", k)
            if not name or ".vgpr_spill_count" not in k:
                continue
            used = tuple(int(re.search(r"\.%s:\s+(\d+)" % f, k).group(1))
                         for f in ("private_segment_fixed_size", "vgpr_spill_count"))
            assert used == (0, 0), (name.group(1), used)
            found += 1
    assert found >= 80      # norms by type, layout and lanes, forward, append and backward, ...


def test_paged_decode_refuses_bounds_it_cannot_keep():
    """Before it asks for a device."""
    from tilegen_amd import paged_decode
    for sizes in (dict(bound=-1), dict(every=0), dict(first=-1), dict(recent=9, bound=8),
                  dict(recent=-1, bound=8), dict(recent=6, first=3, bound=8)):
        with pytest.raises(ValueError, match=list(sizes)[0]):
            paged_decode.run(**sizes)
