"""Builds libccglib_amd.so (HIP kernels + C ABI) for gfx950 with hipcc, in tree.

    python -m ccglib_amd.build            # compile what changed, link
    python -m ccglib_amd.build --force    # recompile everything
"""
import concurrent.futures
import os
import re
import shutil
import subprocess
import sys
import time

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "_build")
LIB_PATH = os.path.join(HERE, "libccglib_amd.so")
# (gemm_mfma.hip is compiled in parts, one per input type, and type of C and kind of rows for 16 bits, so that they build in
# parallel; those that take longest come first)
SOURCES = ["gemm_mfma_f16_f32.hip", "gemm_mfma_bf16_f32.hip", "gemm_mfma_f32.hip", "gemm_mfma_f16_f16.hip",
           "gemm_mfma_bf16_bf16.hip", "gemm_mfma_fp8.hip", "gemm_mfma_f16_f32_pairs.hip", "gemm_mfma_bf16_f32_pairs.hip",
           "gemm_mfma_f16_f16_pairs.hip", "gemm_mfma_bf16_bf16_pairs.hip", "scaled_gemm_e8m0.hip", "scaled_gemm_wide_rows.hip",
           "scaled_gemm_wide_blocks.hip", "scaled_gemm_wide_e8m0.hip", "quantize.hip", "scaled_gemm_rows.hip",
           "scaled_gemm_blocks.hip", "orthogonalize.hip", "linear_f16_output.hip",
           "linear_bf16_output.hip", "linear_f16_weights.hip", "linear_bf16_weights.hip", "linear_f16_input.hip",
           "linear_bf16_input.hip", "gemm_mfma_int1.hip", "linear_f16_backward.hip",
           "linear_bf16_backward.hip", "linear_rows.hip", "transpose.hip", "combine.hip", "route.hip", "linear.hip",
           "gemm_int1.hip", "packing.hip", "capi.hip", "operators_capi.hip", "linear_capi.hip", "scaled_gemm.hip",
           "gemm_mfma_dispatch.hip", "host_copy.hip"]
# Packed-fp32 instruction selection is switched off for all device code.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _defines():
    """Build options taken from the environment: CCGLIB_AMD_STATIC_SCRATCH_BYTES, the size
    of the static device array of ccglib_pipeline_run_static (default in the header)."""
    v = os.environ.get("CCGLIB_AMD_STATIC_SCRATCH_BYTES")
    return ["-DCCGLIB_AMD_STATIC_SCRATCH_BYTES=((size_t)%d)" % int(v)] if v else []


def _hipcc():
    return shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def _jobs():
    """How many sources are compiled at a time: a processor each, and not more than 16 (one takes up to 0.6 GB)."""
    return max(1, min(16, len(os.sched_getaffinity(0)), len(SOURCES)))


def _run(cmd):
    """Runs the compiler or the linker. One that ends without an error in the source to report (it was killed, or ran out of
    something) is run once more; what it said the first time stays in the output."""
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0 and not re.search(r"^\S+:\d+(:\d+)?: (fatal )?error:|undefined symbol|undefined reference", r.stdout + r.stderr, re.M):
        again = subprocess.run(cmd, capture_output=True, text=True)
        again.stderr = "%s\nended with status %d and was run again\n%s" % ((r.stdout + r.stderr).rstrip(), r.returncode, again.stderr)
        return again
    return r


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _with_includes(path, found=None):
    """The source and every file of this tree that it includes, directly or not."""
    found = [] if found is None else found
    if path not in found and os.path.exists(path):
        found.append(path)
        with open(path) as f:
            for name in re.findall(r'^#include "([^"]+)"', f.read(), re.M):
                _with_includes(os.path.normpath(os.path.join(os.path.dirname(path), name)), found)
    return found


def _object(src):
    return os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")


def _compiler_version():
    r = subprocess.run([_hipcc(), "--version"], capture_output=True, text=True)
    return "; ".join(r.stdout.splitlines()[:2])


def _compile(src, force):
    obj = _object(src)
    path = os.path.join(CSRC, src)
    if not force and not _stale(obj, _with_includes(path)):
        return obj, ""
    cmd = [_hipcc()] + HIPCC_FLAGS + _defines() + ["-Rpass-analysis=kernel-resource-usage", "-c", path,
                                                   "-o", obj]
    r = _run(cmd)
    lines = (r.stdout + r.stderr).splitlines()
    kept, includes, skip = [], [], 0
    for l in lines:      # (the remarks, each with its source line, caret and includes, stay out of the log)
        if l.startswith("In file included from"):
            includes.append(l)
        elif "kernel-resource-usage" in l:
            includes, skip = [], 2
        elif skip and (l.lstrip()[:1].isdigit() or l.strip().startswith("|")):
            skip -= 1
        elif "packed-fp32-ops" not in l:
            kept += includes + [l]
            includes, skip = [], 0
    log = "\n".join(kept)
    if r.returncode != 0:
        raise RuntimeError("hipcc failed for %s:\n%s" % (src, log))
    _no_scratch_in_gemm_kernels(src, lines)
    return obj, log


def _no_scratch_in_gemm_kernels(src, remarks):
    """The MFMA GEMM kernels wait for their copies with explicit `s_waitcnt vmcnt(n)` counts,
    which only hold while the compiler adds no memory instructions of its own inside the K
    loop. The compiler's resource remarks say whether a kernel spills registers to scratch
    memory. The one-wave-per-SIMD kernels (complex_gemm_mfma_wide) run at the edge of the
    register file and must not spill at all: the build stops if one does. Of the others, the
    1-bit 256 x 128 and 128 x 128 kernels spill four to eight values at set-up and in the epilogue, the four-wave 128 x 128
    ones of ragged 16-bit pairs two or three, and reload them where a block moves
    to its next C tile (the compiler waits for all memory operations there), and those of 32-bit pairs
    to 16-bit C one address while they look for NaN behind the K loop; anything beyond
    those few bytes stops the build as well. The real products (gemm_real, gemm_linear) count their
    copies too and must not spill."""
    name = None
    for l in remarks:
        if "Function Name:" in l:
            name = l.split("Function Name:")[1].split("[")[0].strip()
        elif "ScratchSize [bytes/lane]:" in l and name and any(n in name for n in ("complex_gemm_mfma", "gemm_real", "gemm_linear")):
            size = int(l.split("ScratchSize [bytes/lane]:")[1].split("[")[0])
            if size > (0 if any(n in name for n in ("complex_gemm_mfma_wide", "gemm_real", "gemm_linear")) else 32):
                os.remove(_object(src))
                raise RuntimeError("%s: kernel %s spills %d bytes per lane to scratch memory; its "
                                   "explicit vmcnt counts would not hold" % (src, name, size))


def build(force=False, verbose=False):
    """Compile every HIP source for gfx950 and link the shared library.

    A source's outcome is reported when it is known: its time (verbose), or what is wrong with it,
    upon which nothing further is started."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    began = time.monotonic()
    with concurrent.futures.ThreadPoolExecutor(max_workers=_jobs()) as ex:
        sources = {ex.submit(_compile, s, force): s for s in SOURCES}
        for done in concurrent.futures.as_completed(sources):
            try:
                _, log = done.result()
            except Exception:
                for other in sources:
                    other.cancel()
                print("%s: failed, %.0f s; compiler: %s" % (sources[done], time.monotonic() - began, _compiler_version()),
                      file=sys.stderr, flush=True)
                raise
            if verbose:
                print("%s%s: %.0f s" % (log.strip() + "\n" if log.strip() else "", sources[done], time.monotonic() - began),
                      flush=True)
    objs = [_object(s) for s in SOURCES]
    if force or _stale(LIB_PATH, objs):
        cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs
        r = _run(cmd)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
