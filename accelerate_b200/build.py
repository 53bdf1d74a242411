"""Build the backend's shared library in-tree.

``libaccb200.so`` holds the host side (program parser, scalar code generator,
NVRTC kernel cache, runtime, C ABI) and the text of the hand-written sm_100a
skeletons (``csrc/skeletons/*.cuh``), which NVRTC compiles together with the
generated scalar code at run time.  Ahead-of-time CUDA sources (``csrc/*.cu``)
are compiled by nvcc for sm_100a and linked in.  ``_binding.*.so`` is the CPython module
that makes a run's calls.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libaccb200.so")
BINDING = os.path.join(HERE, "_binding" + sysconfig.get_config_var("EXT_SUFFIX"))      # one for every Python version
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC_ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _embed_skeletons():
    """Turn every skeleton into a C++ raw string (skeleton_data.cpp)."""
    parts = ['// generated by build.py from csrc/skeletons/*.cuh\n#include <cstring>\n#include <string>\n#include "codegen.hpp"\n',
             '#include "ir.hpp"\nnamespace accb200 {\nnamespace {\n']
    names = []
    for path in sorted(glob.glob(os.path.join(CSRC, "skeletons", "*.cuh"))):
        name = os.path.splitext(os.path.basename(path))[0]
        names.append(name)
        text = open(path).read()
        assert ')ACCSK"' not in text
        # raw string literals are limited in some compilers: split into chunks
        chunks = [text[i:i + 12000] for i in range(0, len(text), 12000)]
        parts.append(f"const char* const sk_{name} =\n" + "\n".join(f'R"ACCSK({c})ACCSK"' for c in chunks) + ";\n")
    parts.append("}  // namespace\nconst char* prelude_source() { return sk_prelude; }\n")
    parts.append("const char* skeleton_source(const std::string& name) {\n")
    for n in names:
        parts.append(f'  if (name == "{n}") return sk_{n};\n')
    parts.append('  throw Error(B200_ERR_ARG, "unknown skeleton " + name);\n}\n}  // namespace accb200\n')
    out = os.path.join(CSRC, "skeleton_data.cpp")
    text = "".join(parts)
    if not os.path.exists(out) or open(out).read() != text:
        open(out, "w").write(text)
    return out


def _newer(target, sources):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _build_binding(force, verbose):
    """The CPython module for the calls that every run makes (csrc/python/binding.cpp)."""
    src = os.path.join(CSRC, "python", "binding.cpp")
    untagged = os.path.join(HERE, "_binding.so")
    if os.path.exists(untagged):         # every version would load this one, whichever it was built for
        os.remove(untagged)
    if not force and not _newer(BINDING, [src, os.path.abspath(__file__)]):
        return
    include = sysconfig.get_paths()["include"]
    if not os.path.exists(os.path.join(include, "Python.h")):
        warnings.warn(f"no Python.h in {include}: the backend's calls go through ctypes, which takes longer", RuntimeWarning, stacklevel=3)
        return
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-I{include}", src, "-o", BINDING]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)


def build(force=False, verbose=False):
    _build_binding(force, verbose)
    _embed_skeletons()
    cpps = sorted(glob.glob(os.path.join(CSRC, "*.cpp")))
    cus = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    deps = cpps + cus + glob.glob(os.path.join(CSRC, "*.hpp")) + glob.glob(os.path.join(CSRC, "skeletons", "*.cuh")) + \
        [os.path.join(HERE, "..", "include", "accelerate_b200.h"), os.path.abspath(__file__)]
    if not force and not _newer(OUT, deps):
        return OUT
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for src in cpps:
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", f"-I{CUDA}/include", "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        subprocess.check_call(cmd)
        objs.append(obj)
    for src in cus:
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = ["nvcc", *NVCC_ARCH, "-lineinfo", "-O3", "-std=c++17", "--fmad=false", "-Xcompiler", "-fPIC",
               "-Xptxas", "-v", f"-I{os.path.join(CSRC, 'skeletons')}", "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError("nvcc failed for " + src)
        objs.append(obj)
    link = ["g++", "-shared", "-o", OUT, *objs, f"-L{CUDA}/lib64", "-lcudart_static", "-lnvrtc", "-ldl", "-lrt", "-lpthread",
            f"-Wl,-rpath,{CUDA}/lib64"]
    if verbose:
        print(" ".join(link))
    subprocess.check_call(link)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
