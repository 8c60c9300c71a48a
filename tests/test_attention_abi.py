"""libtgattn.so without a GPU: its exports, the structures that the binding packs, refusals,
spills, and the frequencies of rotary positions."""

from __future__ import annotations

import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from tilegen_amd import attention as at
from tilegen_amd import build, runtime

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "tilegen_attention.h")
PACKED = {"tg_rope": at._ROPE, "tg_paged_append": at._APPEND, "tg_prefix_attention": at._ATTENTION}


def test_exports_what_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(\w+)\(const tg_\w+\*", text))
    assert declared == {"launch_rope", "launch_paged_append", "launch_prefix_attention",
                        "prefix_attention_workspace"}
    out = subprocess.run(["nm", "-D", "--defined-only",
                          os.path.join(runtime.lib_dir(), "libtgattn.so")],
                         capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert declared <= exported
    assert all(s in declared or s.startswith("_") for s in exported), exported


def test_packed_fields_follow_the_header():
    """The header's field types in order, as struct codes."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, packed in PACKED.items():
        body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
        codes = ""
        for line in body.split(";"):    # no field list mixes pointers and numbers
            if line.strip():
                kind = "P" if "*" in line else "d" if "double" in line else "q"
                codes += kind * len(line.split(","))
        flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Pqd])", packed.format))
        assert codes == flat, name
        assert packed.size == 8 * len(codes)


def test_refusals_without_a_device():
    """Refused on the host, before any HIP call."""
    L = at._lib()

    def message(rc, code):
        assert rc == code
        return runtime.last_error()

    assert "null" in message(L.launch_rope(None, None), -1)
    rope = dict(x=0, y=0, positions=0, frequency=0, dtype=0, tokens=4, heads=2, dim=64,
                rotary=64, layout=0, xt=128, xh=64, yt=128, yh=64, magnitude=1.0, sign=1)
    for change, word in [(dict(), "null"), (dict(dtype=3), "dtype"), (dict(dim=0), "dim"),
                         (dict(dim=1025), "dim"), (dict(rotary=66), "rotary"),
                         (dict(rotary=7), "rotary"), (dict(layout=2), "layout"),
                         (dict(tokens=-1), "negative"), (dict(sign=0), "sign")]:
        args = at._ROPE.pack(*{**rope, **change}.values())
        assert word in message(L.launch_rope(args, None), -1)
    assert "tokens" in message(L.launch_rope(at._ROPE.pack(*{**rope, "tokens": 1 << 40}.values()),
                                             None), -2)
    assert L.launch_rope(at._ROPE.pack(*{**rope, "tokens": 0}.values()), None) == 0
    names = [f for f in ("query kc vc prefix indptr indices lengths ends out lse workspace bytes "
                         "dtype tokens sequences heads kv_heads dim pages page n_prefix "
                         "prefix_length n_indices max_query max_length").split()]
    base = dict.fromkeys(names, 0)
    base.update(tokens=2, sequences=2, heads=4, kv_heads=2, dim=64, pages=999, page=16,
                n_prefix=200, prefix_length=3200, n_indices=4, max_query=1, max_length=20)
    base.update({"s%d" % i: 64 for i in range(10)}, scale=0.125)

    def attend(**change):
        return at._ATTENTION.pack(*{**base, **change}.values())

    need = L.prefix_attention_workspace(attend())
    assert L.prefix_attention_workspace(attend(prefix_length=32)) == 0   # one launch, no parts
    assert need > 0 and "null" in message(L.launch_prefix_attention(attend(), None), -1)
    every = {n: 4096 for n in names[:10]}
    assert "workspace" in message(L.launch_prefix_attention(
        attend(**every, workspace=4096, bytes=need - 1), None), -1)
    assert "aligned" in message(L.launch_prefix_attention(
        attend(**every, workspace=4100, bytes=need), None), -1)
    for change, code in [(dict(dtype=2), -1), (dict(dim=12), -1), (dict(dim=264), -1),
                         (dict(kv_heads=3), -1), (dict(kv_heads=0), -1), (dict(page=0), -1),
                         (dict(scale=0.0), -1), (dict(scale=math.nan), -1),
                         (dict(prefix_length=3201), -1), (dict(tokens=3), -1),
                         (dict(max_length=1 << 40), -2), (dict(sequences=-1), -1),
                         (dict(tokens=1 << 25, sequences=1 << 25), -2)]:
        assert L.prefix_attention_workspace(attend(**change)) < 0, change
        assert L.launch_prefix_attention(attend(**change), None) == code, change
    assert L.prefix_attention_workspace(attend(tokens=0, sequences=0)) == 0
    assert L.launch_prefix_attention(attend(tokens=0, sequences=0), None) == 0


def test_operands_on_the_host_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int64)
    f = torch.zeros(32, dtype=torch.float64)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        at.rope(x, n, f)
    with pytest.raises(ValueError):
        at.paged_append(x, x, cache, cache, n, n, n, f)
    with pytest.raises(ValueError):
        at.prefix_attention(x, cache, cache, n, 0, n, n, n, max_length=1)


def test_rope_frequencies():
    """Against the formulas; kept, divided and ramped pairs."""
    n = 64
    plain = np.array([10000.0 ** (-i / n) for i in range(0, n, 2)])
    f, m = at.rope_frequencies(n, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    np.testing.assert_allclose(f.numpy(), plain, rtol=1e-15)
    f, m = at.rope_frequencies(n, scaling="linear", factor=8, device="cpu")
    np.testing.assert_allclose(f.numpy(), plain / 8, rtol=1e-15)
    f, m = at.rope_frequencies(n, scaling="ntk", factor=8, device="cpu")
    np.testing.assert_allclose(f.numpy()[[0, -1]], plain[[0, -1]] / [1, 8], rtol=1e-12)
    f, m = at.rope_frequencies(n, scaling="yarn", factor=8, trained=4096, device="cpu")
    turns = 4096 * plain / (2 * np.pi)
    assert (f.numpy()[turns >= 32] == plain[turns >= 32]).all() and (turns >= 32).any()
    np.testing.assert_allclose(f.numpy()[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    assert (np.diff(f.numpy()) < 0).all() and m == pytest.approx(0.1 * math.log(8) + 1)
    for bad in (dict(rotary=3), dict(rotary=4, scaling="x"), dict(rotary=4, factor=0.5),
                dict(rotary=4, scaling="yarn")):
        with pytest.raises(ValueError):
            at.rope_frequencies(device="cpu", **bad)


def test_sizes_at_the_ends_of_64_bits():
    """Refused, or used as the bounds they are, without overflow on the way."""
    L = at._lib()
    names = ("query kc vc prefix indptr indices lengths ends out lse workspace bytes dtype tokens "
             "sequences heads kv_heads dim pages page n_prefix prefix_length n_indices max_query "
             "max_length").split()
    base = dict.fromkeys(names, 0)
    base.update(tokens=2, sequences=2, heads=4, kv_heads=2, dim=64, pages=999, page=16,
                n_prefix=200, prefix_length=3200, n_indices=4, max_query=1, max_length=20)
    base.update({"s%d" % i: 64 for i in range(10)}, scale=0.125)
    most = (1 << 63) - 1

    def workspace(**change):
        return L.prefix_attention_workspace(at._ATTENTION.pack(*{**base, **change}.values()))

    for change in (dict(prefix_length=most), dict(max_length=most), dict(pages=1 << 31),
                   dict(heads=1 << 62, kv_heads=1 << 61), dict(heads=1 << 17),
                   dict(sequences=most)):
        assert workspace(**change) < 0, change
    # a bound on new tokens above all tokens is all tokens
    for tokens in (2, 40):
        sizes = dict(tokens=tokens, ends=4096)
        assert workspace(**sizes, max_query=most) == workspace(**sizes, max_query=tokens) > 0


def _append_args(**change):
    names = ("key value query kc vc out indptr indices lengths ends frequency dtype tokens sequences "
             "heads kv_heads dim rotary layout pages page n_indices offset key_token key_head "
             "value_token value_head query_token query_head out_token out_head kc_page kc_slot "
             "kc_head vc_page vc_slot vc_head magnitude").split()
    base = dict.fromkeys(names, 0)
    base.update(dtype=0, tokens=5, sequences=5, heads=4, kv_heads=2, dim=64, rotary=64, pages=9,
                page=16, n_indices=5, magnitude=1.0)
    for token, head in (("key_token", "key_head"), ("value_token", "value_head"),
                        ("query_token", "query_head"), ("out_token", "out_head")):
        base.update({token: 512, head: 64})
    for c in ("kc", "vc"):
        base.update({c + "_page": 2048, c + "_slot": 128, c + "_head": 64})
    base.update(key=1 << 20, value=2 << 20, query=3 << 20, out=4 << 20, kc=5 << 20, vc=6 << 20)
    base.update(change)
    return at._APPEND.pack(*base.values())


def test_append_over_its_own_operands():
    """Refused where what is written shares memory with what is read or written beside it, and
    there alone: slices of one array may lie between one another.  (The row pointers are null, so
    that calls without a fault end in that refusal and nothing is launched.)"""
    L = at._lib()

    def message(**change):
        assert L.launch_paged_append(_append_args(**change), None) == -1
        return runtime.last_error()

    q, k, v = 3 << 20, (3 << 20) + 4 * 128, (3 << 20) + 6 * 128     # packed, 8 heads a token
    packed = dict(query=q, key=k, value=v)
    for fine in (dict(), packed, dict(packed, out=q), dict(out=3 << 20),
                 dict(vc=(5 << 20) + 2048, kc_page=2048, vc_page=2048, page=8),
                 # keys by slots, values by heads, in halves of a page
                 dict(vc=(5 << 20) + 4096, kc_page=4096, vc_page=4096, vc_slot=64, vc_head=1024),
                 dict(heads=0, query=0, out=0), dict(kc=5 << 20, vc=5 << 20, rotary=0, value=1 << 20),
                 dict(key=(5 << 20) + 4096)):       # a key from the cache
        assert "null" in message(**fine), fine
    for change, out, other in [
            (dict(out=q + 128), "query_out", "query"), (dict(packed, out=k - 2), "query_out", "query"),
            (dict(packed, out=k), "query_out", "key"),
            (dict(packed, heads=2, out=v), "query_out", "value"),
            (dict(out=(1 << 20) + 2), "query_out", "key"), (dict(out=2 << 20), "query_out", "value"),
            (dict(out=(1 << 20) + 4 * 1024 + 254), "query_out", "key"),
            (dict(out=(5 << 20) + 9 * 4096 - 2), "query_out", "key_cache"),
            (dict(out=6 << 20), "query_out", "value_cache"),
            (dict(out=3 << 20, out_head=128), "query_out", "query"),
            (dict(vc=5 << 20), "value_cache", "key_cache"),
            (dict(vc=(5 << 20) + 4094, kc_page=4096, vc_page=4096), "value_cache", "key_cache"),
            (dict(vc=5 << 20, rotary=0), "value_cache", "key_cache")]:
        want = "%s overlaps %s" % (out, other)
        assert message(**change).endswith(want), (change, runtime.last_error())
    assert "null" in message(out=(1 << 20) + 4 * 1024 + 256)    # past the last key's second head


def test_more_sequences_than_the_search_can_count():
    """The search for a token's sequence looks up to 64 steps past the last one, in 32 bits."""
    L = at._lib()
    for sequences in ((1 << 31) - 1, (1 << 31) - 64, (1 << 30) + 1):
        assert L.launch_paged_append(_append_args(sequences=sequences, ends=4096), None) == -1
        assert "sequences" in runtime.last_error()
    assert L.launch_paged_append(_append_args(sequences=1 << 30, ends=4096), None) == -1
    assert "null" in runtime.last_error()


def test_launches_that_hip_would_refuse():
    """A grid has under 2^32 threads: calls beyond are refused before anything is enqueued, in the
    parts' launch (here 4096 row tiles of the prefix for each of 32 kv heads beside 2^24 - 32
    workgroups of own pages) and in the joining's, four rows a workgroup."""
    L = at._lib()
    base = dict.fromkeys(("query kc vc prefix indptr indices lengths ends out lse workspace bytes "
                          "dtype").split(), 0)
    base.update(tokens=0, sequences=0, heads=32, kv_heads=32, dim=64, pages=999, page=16,
                n_prefix=200, prefix_length=3200, n_indices=4, max_query=1, max_length=20)
    base.update({"s%d" % i: 64 for i in range(10)}, scale=0.125)

    def workspace(**change):
        return L.prefix_attention_workspace(at._ATTENTION.pack(*{**base, **change}.values()))

    many = (1 << 19) - 1
    assert workspace(tokens=many, sequences=many) < 0
    assert "workgroups" in runtime.last_error()
    assert workspace(tokens=many, sequences=many, prefix_length=0) > 0
    assert workspace(tokens=many - 4096, sequences=many - 4096) > 0
    rows = dict(ends=4096, sequences=1, heads=16, kv_heads=1, max_query=1 << 22)
    assert workspace(**rows, tokens=1 << 22) < 0
    assert "rows" in runtime.last_error()
    assert workspace(**rows, tokens=(1 << 22) - 1) > 0


def test_scales_that_are_0_in_32_bits():
    L = at._lib()
    base = [0] * 12 + [0, 2, 2, 4, 2, 64, 999, 16, 200, 3200, 4, 1, 20] + [64] * 10
    for scale, fine in ((1e-46, False), (5e-324, False), (1e-44, True), (1.0, True)):
        assert (L.prefix_attention_workspace(at._ATTENTION.pack(*base, scale)) > 0) == fine, scale


def test_plans_and_launches_go_by_the_operands_device(monkeypatch):
    """The workspace's size and the launch are asked for with the operands' device current,
    whichever was before (a stand-in library; host tensors count as device -1)."""
    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.before, current[0] = current[0], self.device

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        def prefix_attention_workspace(self, packed):
            seen.append(("workspace", current[0]))
            return 64

        def launch_prefix_attention(self, packed, stream):
            seen.append(("launch", current[0], stream))
            return 0

    monkeypatch.setattr(at, "_lib", Library)
    monkeypatch.setattr(at, "_operand", lambda name, t, dtypes: (t.get_device(), t.dtype))
    monkeypatch.setattr(at, "_raw_stream", lambda device: 1000 + device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(3, dtype=torch.int64)
    for current[0] in (0, -1):
        seen.clear()
        at.prefix_attention(q, cache, cache, n, 0, n, n, n[:2], max_length=1)
        assert seen == [("workspace", -1), ("launch", -1, 999)]


def test_paged_decode_refuses_what_it_cannot_run():
    """Before it asks for a device."""
    from tilegen_amd import paged_decode
    for sizes in (dict(sequences=0), dict(start=0), dict(prompt=-1), dict(steps=-1)):
        with pytest.raises(ValueError, match=list(sizes)[0]):
            paged_decode.run(**sizes)


# (head size, rows of a prefix workgroup, of an own pages' one): bytes of scratch a lane, vector
# registers spilled.  The first reserves its bytes and touches none.
SPILLS = {(64, 128, 16): (68, 0), (128, 128, 128): (184, 45), (256, 128, 128): (336, 111)}


def test_kernels_that_spill(tmp_path):
    """Kernels keep their values in registers, but for those listed, and those to that extent.
    (Scalar registers go to lanes of vector registers, not to memory.)"""
    readelf = "/opt/rocm/llvm/bin/llvm-readelf"
    if not os.path.exists(readelf):
        pytest.skip("llvm-readelf not available")
    found, most = 0, {}
    for co in build.attention_code_objects(str(tmp_path)):
        notes = subprocess.run([readelf, "--notes", co], capture_output=True, text=True,
                               check=True).stdout
        for k in re.split(r"\n\s+- \.", notes):
            name = re.search(r"\.name:\s+(\S+)", k)
            if not name or ".vgpr_spill_count" not in k:
                continue
            used = tuple(int(re.search(r"\.%s:\s+(\d+)" % f, k).group(1))
                         for f in ("private_segment_fixed_size", "vgpr_spill_count"))
            sizes = re.search(r"6attend\w*?Li(\d+)ELi(\d+)ELi(\d+)E", name.group(1))
            at_most = SPILLS.get(tuple(map(int, sizes.groups()))) if sizes else None
            at_most = at_most or (0, 0)
            assert used[0] <= at_most[0] and used[1] <= at_most[1], (name.group(1), used)
            found += 1
            if at_most != (0, 0):
                key = tuple(map(int, sizes.groups()))
                most[key] = max(most.get(key, (0, 0)), used)
    # attend by prefix and own rows and attend_whole for 4 head sizes and 2 types; joins of 3 widths
    # for 2 types, in one wave and four; rotations by type, layout, whole chunks, append
    assert found == 4 * 8 + 12 + 24
    assert most == SPILLS       # a list that is out of date says so


def test_outputs_whose_elements_share_memory():
    """Refused whatever the strides are that make them; layouts that only interleave are not.
    (Null arrays end the calls that pass.)"""
    L = at._lib()

    def append(**change):
        assert L.launch_paged_append(_append_args(**change), None) == -1
        return runtime.last_error()

    def rope(token, head, tokens=5, heads=4, dim=64):
        args = at._ROPE.pack(0, 1 << 20, 0, 0, 0, tokens, heads, dim, 0, 0, 0, 0, token, head, 1.0, 1)
        assert L.launch_rope(args, None) == -1
        return runtime.last_error()

    for fine in (dict(), dict(out_token=64, out_head=320), dict(kc_page=64, kc_slot=18 * 64,
                                                                kc_head=9 * 64)):
        assert "null" in append(**fine), fine
    for change, name in [(dict(out_head=32), "query_out"), (dict(out_head=0), "query_out"),
                         (dict(out_token=192), "query_out"), (dict(out_head=63), "query_out"),
                         (dict(out_token=-192), "query_out"), (dict(kc_page=0), "key_cache"),
                         (dict(vc_slot=64), "value_cache"), (dict(vc_page=2047), "value_cache")]:
        assert name + " is written" in append(**change), change
    assert "null" in rope(256, 64) and "null" in rope(64, 320) and "null" in rope(0, 64, tokens=1)
    # 2 heads 64 and 160 apart under 2 tokens; three tokens 4 apart are one step of heads 6 apart
    # twice, but there have to be four tokens for it
    assert "share" in rope(96, 64, tokens=2, heads=2) and "null" in rope(64, 160, tokens=2, heads=2)
    assert "share" in rope(4, 6, tokens=4, heads=3, dim=2) and "null" in rope(
        4, 6, tokens=3, heads=3, dim=2)
