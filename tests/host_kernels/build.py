"""Builds the kernels of the many-class loss and of the 8-bit checkpoints for the CPU (host_hip.h): the sources in maxstyle_amd/csrc as they are, but for what only the
GPU's assembler reads - inline assembly (waits, the LDS DMA: a function in its place) and the LDS address space.

`limits` replaces constants that set the size of a piece, so that small inputs are cut into several."""
import ctypes
import hashlib
import os
import re
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(ROOT, "maxstyle_amd", "csrc")
CLANG = "/opt/rocm/llvm/bin/clang++"
SOURCES = [s for s in ("ms_class_ce.hip", "ms_class_ce_narrow.hip", "ms_act8.hip", "ms_logit_ce.hip") if os.path.exists(os.path.join(CSRC, s))]
HEADERS = ("ms_common.h", "ms_class_ce.h", "ms_class_ce_narrow.h")


def _prepare(text, limits):
    text = text.replace("#include <hip/hip_runtime.h>", '#include "host_hip.h"')
    text = re.sub(r'asm volatile\("s_mov_b32 m0, %0\\n\\ts_nop 0\\n\\tbuffer_load_dwordx4 [^;]*;', "host::dma16(rsrc, lds_byte_addr, voff, soff);", text)
    text = re.sub(r"(?s)__device__ __forceinline__ unsigned ms_lds_addr\(const void\* p\) \{.*?\n\}", "inline unsigned ms_lds_addr(const void* p) { return host::lds_addr(p); }", text)
    text = re.sub(r'asm (volatile)?\s*\([^;]*;|asm\([^;]*;', ";", text)
    text = text.replace("__attribute__((address_space(3)))", "")
    for old, new in limits.items():
        text = text.replace(old, new)
    return text


def build(limits=None):
    """Path of the library; compiled once for its sources."""
    limits = limits or {}
    out = {}
    for name in HEADERS + tuple(SOURCES):
        with open(os.path.join(CSRC, name)) as f:
            out[name] = _prepare(f.read(), limits)
    found = "".join(out[s] for s in SOURCES)
    for old, new in limits.items():
        if new not in found:
            raise ValueError(f"host kernels: {old!r} is not in the sources")
    heads = "".join(open(os.path.join(HERE, n)).read() for n in ("host_hip.h", "host_hip.cpp")) + "".join(out[n] for n in HEADERS)
    cache = os.path.join(HERE, "build")
    keyed = lambda text: hashlib.sha256((heads + text).encode()).hexdigest()[:16]
    lib = os.path.join(cache, "libhost_kernels_%s.so" % keyed(repr(sorted(out.items()))))
    if os.path.exists(lib):
        return lib
    flags = ["-O1", "-march=x86-64-v3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-w", "-I", HERE, "-I", os.path.join(ROOT, "include")]
    objects, jobs = [], []
    for name in SOURCES + ["host_hip.cpp"]:
        where = os.path.join(cache, "%s_%s" % (name.split(".")[0], keyed(out.get(name, ""))))      # (a source and its headers: one object)
        obj = os.path.join(where, "a.o")
        objects.append(obj)
        if os.path.exists(obj):
            continue
        os.makedirs(where, exist_ok=True)
        for n in HEADERS + ((name,) if name in out else ()):
            with open(os.path.join(where, n), "w") as f:
                f.write(out[n])
        src = ["-x", "c++", os.path.join(where, name)] if name in out else [os.path.join(HERE, name)]
        tmp = "%s.%d" % (obj, os.getpid())
        jobs.append((subprocess.Popen([CLANG] + flags + ["-I", where, "-c", "-o", tmp] + src, stderr=subprocess.PIPE, text=True), tmp, obj))
    for proc, tmp, obj in jobs:
        err = proc.communicate()[1]
        if proc.returncode:
            raise RuntimeError(err[-4000:])
        os.replace(tmp, obj)
    tmp = "%s.%d" % (lib, os.getpid())
    subprocess.run([CLANG, "-shared", "-o", tmp] + objects, check=True)
    os.replace(tmp, lib)
    return lib


def load(limits=None):
    lib = ctypes.CDLL(build(limits))
    lib.host_last_error.restype = ctypes.c_char_p
    return lib
