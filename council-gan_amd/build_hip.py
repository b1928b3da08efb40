"""Builds the gfx950 shared library IN-TREE: council-gan_amd/lib/libcouncilgan_hip.so, and the host extension cg_nodes.so beside it
(autograd nodes of the channel-MLP operators: C++ against torch's headers, no device code).

    python council-gan_amd/build_hip.py [--force]

hipcc cross-compiles without a GPU; the .so is git-ignored but travels with gpurun snapshots.  Every translation unit is
compiled to its own object (in parallel, cached by a digest of the file, the shared headers and the flags under lib/obj/) and
the objects are linked: an edit to one kernel file recompiles that file only."""
import hashlib
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
UNITS = ("conv_gemm.hip", "conv_x3.hip", "norm.hip", "elementwise.hip", "collective.hip", "head.hip", "channel_mlp.hip",
         "gated.hip")
SRC = [os.path.join(CSRC, f) for f in UNITS if os.path.exists(os.path.join(CSRC, f))]
# headers / include files every unit may see (a change recompiles everything)
SHARED = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".h", ".inc")) and f != "cg_vec.h"] + \
         [os.path.join(HERE, "..", "include", "council_gan_hip.h")]
CHANNEL_UNITS = ("channel_mlp.hip", "gated.hip")       # the units that include cg_vec.h
EXTRA = {u: [os.path.join(CSRC, "cg_vec.h")] for u in CHANNEL_UNITS}
DEPS = SRC + SHARED + [os.path.join(CSRC, "cg_vec.h")]
OUT_DIR = os.path.join(HERE, "lib")
OBJ_DIR = os.path.join(OUT_DIR, "obj")
OUT = os.path.join(OUT_DIR, "libcouncilgan_hip.so")
STAMP = OUT + ".stamp"
# no packed fp32 arithmetic: some of its forms have given wrong results on this hardware now and then
CFLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang",
          "-packed-fp32-ops"] + os.environ.get("CG_HIPCC_FLAGS", "").split()
FLAGS = CFLAGS + ["-shared"]
UNIT_FLAGS = {u: ["-Wno-inline-asm"] for u in CHANNEL_UNITS}


def _digest(paths=DEPS):
    h = hashlib.sha256()
    for p in paths:
        h.update(open(p, "rb").read())
    h.update(" ".join(FLAGS).encode())
    for u in UNITS:
        if os.path.join(CSRC, u) in paths and u in UNIT_FLAGS:
            h.update(" ".join(UNIT_FLAGS[u]).encode())
    return h.hexdigest()


def _compile(hipcc, src, verbose):
    dig = _digest([src] + EXTRA.get(os.path.basename(src), []) + SHARED)
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    tag = obj + ".stamp"
    if os.path.exists(obj) and os.path.exists(tag) and open(tag).read() == dig:
        return obj
    cmd = [hipcc] + CFLAGS + UNIT_FLAGS.get(os.path.basename(src), []) + ["-c", src, "-o", obj]
    if verbose:
        print("[build_hip]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    open(tag, "w").write(dig)
    return obj


NODES_SRC = os.path.join(CSRC, "nodes.cpp")
NODES = os.path.join(OUT_DIR, "cg_nodes.so")


def build_nodes(force=False, verbose=True):
    torch_dir = list(importlib.util.find_spec("torch").submodule_search_locations)[0]      # located, not imported
    inc, lib = os.path.join(torch_dir, "include"), os.path.join(torch_dir, "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I/opt/rocm/include", "-I" + inc,
           "-I" + os.path.join(inc, "torch", "csrc", "api", "include"), "-I" + sysconfig.get_paths()["include"], NODES_SRC, "-o", NODES,
           "-L" + lib, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
    h = hashlib.sha256(" ".join(cmd).encode())
    for p in (NODES_SRC, SHARED[-1], os.path.join(torch_dir, "version.py")):
        h.update(open(p, "rb").read())
    tag, dig = os.path.join(OBJ_DIR, "cg_nodes.so.stamp"), h.hexdigest()
    if not force and os.path.exists(NODES) and os.path.exists(tag) and open(tag).read() == dig:
        return NODES
    if verbose:
        print("[build_hip]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    open(tag, "w").write(dig)
    return NODES


def build(force=False, verbose=True):
    os.makedirs(OBJ_DIR, exist_ok=True)
    build_library(force, verbose)
    build_nodes(force, verbose)
    return OUT


def build_library(force=False, verbose=True):
    dig = _digest()
    if not force and os.path.exists(OUT) and os.path.exists(STAMP) and open(STAMP).read() == dig:
        return OUT
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if force:
        for f in os.listdir(OBJ_DIR):
            os.remove(os.path.join(OBJ_DIR, f))
    with ThreadPoolExecutor(max_workers=min(len(SRC), os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(hipcc, s, verbose), SRC))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC"] + objs + ["-ldl", "-o", OUT]
    if verbose:
        print("[build_hip]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    open(STAMP, "w").write(dig)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(OUT)
