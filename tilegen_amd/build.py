"""Build everything native, in-tree: ``python -m tilegen_amd.build``.

1. ``tilegen_amd/_lib/libtgrt.so`` (the runtime, include/tgrt.h) with the host
   C++ compiler against the ROCm HIP runtime and hipRTC;
2. ``libtg_vendor.so``, the rocSPARSE comparison (when rocSPARSE is installed),
   ``tilegen_bench``, the native host harness (TGM1 matrix + variant library),
   ``libtgna.so`` (hipcc), the SpMV entry point that allocates nothing, and
   ``libtgattn.so`` (hipcc), attention over a paged cache;
3. the test oracle (``oracle/Makefile``: the C restatement, and the
   reference's own ref.cpp where its sources are present);
4. the hipRTC code objects and C launchers of every named schedule
   (``schedules.TUNED`` and ``TEST_SCHEDULES``) into the kernel cache, so GPU
   runs load prebuilt variants instead of compiling, and the code objects of
   the hardware probes (``tilegen_amd.probes``).  hipRTC needs no GPU.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import time
from concurrent.futures import ThreadPoolExecutor
from typing import List, Optional

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def _run(cmd: List[str], cwd: Optional[str] = None) -> None:
    res = subprocess.run(cmd, cwd=cwd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("command failed (%d): %s\n%s%s" % (res.returncode, " ".join(cmd),
                                                              res.stdout, res.stderr))


def build_runtime() -> str:
    out_dir = os.path.join(PKG, "_lib")
    os.makedirs(out_dir, exist_ok=True)
    out = os.path.join(out_dir, "libtgrt.so")
    tmp = out + ".tmp%d" % os.getpid()
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    _run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__",
          "-I", os.path.join(REPO, "include"), "-I", os.path.join(ROCM, "include"),
          os.path.join(PKG, "csrc", "tgrt.cpp"), "-o", tmp, "-Wl,-soname,libtgrt.so",
          "-L", os.path.join(ROCM, "lib"), "-lamdhip64", "-lhiprtc",
          "-Wl,-rpath," + os.path.join(ROCM, "lib")])
    os.replace(tmp, out)
    return out


def build_vendor() -> Optional[str]:
    """libtg_vendor.so (rocSPARSE comparison); skipped when rocSPARSE is absent."""
    if not os.path.exists(os.path.join(ROCM, "include", "rocsparse", "rocsparse.h")):
        return None
    out = os.path.join(PKG, "_lib", "libtg_vendor.so")
    tmp = out + ".tmp%d" % os.getpid()
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    _run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
          "-Wno-deprecated-declarations", "-I", os.path.join(ROCM, "include"),
          os.path.join(PKG, "csrc", "vendor.cpp"), "-o", tmp, "-L", os.path.join(ROCM, "lib"),
          "-lrocsparse", "-lamdhip64", "-Wl,-rpath," + os.path.join(ROCM, "lib")])
    os.replace(tmp, out)
    return out


def build_harness() -> str:
    """tilegen_bench, the native host harness (csrc/bench_main.cpp)."""
    lib_dir = os.path.join(PKG, "_lib")
    out = os.path.join(lib_dir, "tilegen_bench")
    tmp = out + ".tmp%d" % os.getpid()
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    _run([cxx, "-std=c++17", "-O2", "-Wall", "-I", os.path.join(REPO, "include"),
          os.path.join(PKG, "csrc", "bench_main.cpp"), "-o", tmp, "-L", lib_dir, "-ltgrt",
          "-ldl", "-Wl,-rpath," + lib_dir])
    os.replace(tmp, out)
    return out


def noalloc_kernel_source() -> str:
    """spmv_noalloc_kernel.inc: the hybrid SpMV kernel of schedules.NOALLOC_SCHEDULE
    with its row-piece slots as a kernel argument, and the TG_NA_* geometry the
    host side of libtgna launches it with."""
    from .codegen import MERGE_CAP, _lowering, _plan, emit_hip, launch_geometry
    from .dsl import standard_kernels
    from .passes import run_pipeline
    from .schedules import NOALLOC_SCHEDULE
    cfg = NOALLOC_SCHEDULE
    k = run_pipeline(standard_kernels()["spmv"], cfg, backend="hip")
    geo = launch_geometry(_plan(k), _lowering(k))
    if not geo.nnz_chunk or geo.stream:
        raise RuntimeError("the no-alloc SpMV needs a hybrid-tile schedule, got %s" % cfg.short())
    head = [
        "// generated by tilegen_amd.build from the schedule %s -- DO NOT EDIT" % cfg.short(),
        "#define TG_NA_ROWS_PER_BLOCK %d" % geo.rows_per_block,
        "#define TG_NA_BLOCK %d" % geo.block,
        "#define TG_NA_CHUNK %d  // nonzeros per long-row range" % geo.nnz_chunk,
        "#define TG_NA_SLOTS %d  // two per range, for %d ranges" % (2 * MERGE_CAP, MERGE_CAP),
        "#define TG_NA_MAX_NNZ %dLL" % (MERGE_CAP * geo.nnz_chunk),
        "",
    ]
    return "\n".join(head) + emit_hip(k, cfg, scratch_arg=True)


def _noalloc_compile(gen_dir: str) -> List[str]:
    """hipcc and the compile flags of libtgna.so, with its generated kernel written
    into gen_dir."""
    from .verify import hip_arch
    os.makedirs(gen_dir, exist_ok=True)
    inc = os.path.join(gen_dir, "spmv_noalloc_kernel.inc")
    with open(inc + ".tmp", "w") as fh:
        fh.write(noalloc_kernel_source())
    os.replace(inc + ".tmp", inc)
    return [os.path.join(ROCM, "bin", "hipcc"), "--offload-arch=%s" % hip_arch(), "-O3",
            "-std=c++17", "-fPIC", "-fvisibility=hidden",
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-I", os.path.join(REPO, "include"), "-I", gen_dir,
            os.path.join(PKG, "csrc", "spmv_noalloc.hip")]


def build_noalloc() -> str:
    """libtgna.so: launch_spmv_noalloc (include/tilegen_noalloc.h), hipcc for gfx950."""
    lib_dir = os.path.join(PKG, "_lib")
    out = os.path.join(lib_dir, "libtgna.so")
    tmp = out + ".tmp%d" % os.getpid()
    _run(_noalloc_compile(os.path.join(REPO, "build", "noalloc")) +
         ["-shared", "-o", tmp, "-L", lib_dir, "-ltgrt", "-Wl,-rpath," + lib_dir])
    os.replace(tmp, out)
    return out


def noalloc_code_object(out: str) -> str:
    """libtgna's device code object alone (the same source and flags as the library,
    device pass only), for checks of its kernels' registers and spills."""
    _run(_noalloc_compile(os.path.join(os.path.dirname(out), "noalloc_gen")) +
         ["--offload-device-only", "--no-gpu-bundle-output", "-o", out])
    return out


def attention_sources() -> List[str]:
    src = os.path.join(PKG, "csrc", "attention")
    return [os.path.join(src, f) for f in sorted(os.listdir(src)) if f.endswith(".hip")]


def _attention_compile(source: str) -> List[str]:
    """hipcc and the compile flags of one of libtgattn.so's sources."""
    from .verify import hip_arch
    return [os.path.join(ROCM, "bin", "hipcc"), "--offload-arch=%s" % hip_arch(), "-O3",
            "-std=c++17", "-fPIC", "-fvisibility=hidden",
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-I", os.path.join(REPO, "include"), "-c", source]


def build_attention() -> str:
    """libtgattn.so: attention over a paged cache (include/tilegen_attention.h), hipcc for
    gfx950, its sources side by side."""
    lib_dir = os.path.join(PKG, "_lib")
    obj_dir = os.path.join(REPO, "build", "attention")
    os.makedirs(obj_dir, exist_ok=True)
    out = os.path.join(lib_dir, "libtgattn.so")
    tmp = out + ".tmp%d" % os.getpid()

    def one(source: str) -> str:
        obj = os.path.join(obj_dir, os.path.basename(source)[:-len(".hip")] + ".o")
        _run(_attention_compile(source) + ["-o", obj])
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objects = list(pool.map(one, attention_sources()))
    _run([os.path.join(ROCM, "bin", "hipcc"), "-shared", "-o", tmp] + objects +
         ["-L", lib_dir, "-ltgrt", "-Wl,-rpath," + lib_dir])
    os.replace(tmp, out)
    return out


def attention_code_objects(out_dir: str) -> List[str]:
    """libtgattn's device code objects alone (the same sources and flags as the library, device
    pass only), for checks of their kernels' registers and spills."""
    def one(source: str) -> str:
        out = os.path.join(out_dir, os.path.basename(source)[:-len(".hip")] + ".co")
        _run(_attention_compile(source) +
             ["--offload-device-only", "--no-gpu-bundle-output", "-o", out])
        return out

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        return list(pool.map(one, attention_sources()))


def build_oracle(force: bool = False) -> None:
    _run(["make", "-s"] + (["-B"] if force else []) + ["-C", os.path.join(REPO, "oracle")])


def warm_cache(verbose: bool = False) -> int:
    """Compile every named schedule for every kernel it applies to, and the
    one-pass-skipped variants the pass ablation times."""
    from . import runtime
    runtime._LIB = None  # pick up a freshly built library
    from .ablation import DEFAULT_CASES
    from .codegen import Config, generate
    from .dsl import standard_kernels
    from .matrices import baseline_case
    from .passes import PASS_NAMES
    from .schedules import (HYBRID_TEST_SCHEDULES, MERGE_TEST_SCHEDULES, NOALLOC_SCHEDULE,
                            ODD_BLOCK_SCHEDULES, SORTED_TEST_SCHEDULES, STREAM_TEST_SCHEDULES,
                            TEST_KERNELS, TEST_SCHEDULES, TUNED)
    from .verify import compile_generated

    kernels = standard_kernels()
    todo = []
    for case_id, cfg in TUNED.items():
        todo.append((baseline_case(case_id).kernel, cfg, ()))
    todo.append(("spmv", NOALLOC_SCHEDULE, ()))  # launch_spmv beside launch_spmv_noalloc
    for name in TEST_KERNELS:
        for cfg in TEST_SCHEDULES + ODD_BLOCK_SCHEDULES:
            todo.append((name, cfg, ()))
        todo.append((name, Config(tile_size=32, threads_per_row=4, unroll=2, vector_width=1,
                                  block_size=256, inject_bug=True), ()))
    for name in ("spmv", "fused_spmv_axpy"):
        for cfg in (MERGE_TEST_SCHEDULES + HYBRID_TEST_SCHEDULES + STREAM_TEST_SCHEDULES
                    + SORTED_TEST_SCHEDULES):
            todo.append((name, cfg, ()))
        for cfg in SORTED_TEST_SCHEDULES:  # the direct twins they are checked against
            todo.append((name, Config(**{**cfg.to_dict(), "gather": "direct"}), ()))
        for balance in ("nnz", "hybrid", "stream"):
            todo.append((name, Config(tile_size=32, threads_per_row=4, unroll=2, vector_width=1,
                                      block_size=256, inject_bug=True, balance=balance), ()))
    for name, cases in DEFAULT_CASES.items():
        for case_id in cases:
            todo += [(name, TUNED[case_id], skip) for skip in [()] + [(p,) for p in PASS_NAMES]]
    workdir = os.path.join(REPO, "build", "generated")
    n, seen = 0, set()
    for name, cfg, skip in todo:
        gen = generate(kernels[name], cfg, "hip", outdir=workdir, skip_passes=skip)
        if gen.filename in seen:
            continue
        seen.add(gen.filename)
        if skip:
            full = generate(kernels[name], cfg, "hip", write=False)
            if gen.abi_args != full.abi_args:
                continue  # the ablation reports these as invalid and never runs them
        compile_generated(gen, "hip", workdir)
        n += 1
        if verbose:
            print("[build] %s %s %s" % (name, cfg.short(), " ".join(skip)))
    return n


def build_all(verbose: bool = True, force: bool = False) -> None:
    """Build everything; ``force`` also recompiles the oracle and every cached
    kernel variant instead of reusing up-to-date outputs."""
    t0 = time.time()
    path = build_runtime()
    if verbose:
        print("[build] runtime %s (%.1fs)" % (path, time.time() - t0))
    build_vendor()
    build_harness()
    build_noalloc()
    if verbose:
        print("[build] no-alloc SpMV library (%.1fs)" % (time.time() - t0))
    build_attention()
    if verbose:
        print("[build] attention library (%.1fs)" % (time.time() - t0))
    build_oracle(force)
    if force:
        from .verify import cache_dir
        shutil.rmtree(cache_dir(), ignore_errors=True)
    if verbose:
        print("[build] oracle (%.1fs)" % (time.time() - t0))
    n = warm_cache()
    if verbose:
        print("[build] %d HIP variants cached (%.1fs)" % (n, time.time() - t0))
    from .probes import build as build_probes
    n = build_probes()
    if verbose:
        print("[build] %d probe kernels cached (%.1fs)" % (n, time.time() - t0))


if __name__ == "__main__":
    build_all(verbose=True, force="--force" in sys.argv[1:])
    sys.exit(0)
