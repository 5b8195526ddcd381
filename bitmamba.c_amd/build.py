"""Builds libbitmamba_hip.so (gfx950 HIP kernels + C ABI + C11 host code).

Run directly (``python bitmamba.c_amd/build.py``) or through
``__graft_entry__.build()``.  Always recompiles: objects go to
``bitmamba.c_amd/_build`` and the library next to this file.
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libbitmamba_hip.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17",
    # parity: no a*b+c contraction anywhere in the device code; the device
    # code divides and takes square roots only through bm_fp.h, which spells
    # out the correctly rounded sequences (the option below is the compiler's
    # default and only matters for a plain `/` or sqrtf, of which there are
    # none; tests/test_fp_build.py checks the equivalence)
    "-ffp-contract=off", "-fhip-fp32-correctly-rounded-divide-sqrt",
    # packed fp32 instructions off (wrong results seen on this hardware)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]
# of single files
FILE_FLAGS = {
    # results of matrix instructions in vector registers: with more than 256 in
    # use the compiler puts them into accumulation registers otherwise, and
    # copies them for every other instruction
    "bm_delta.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
}
C_FLAGS = ["-std=gnu11", "-O2", "-fPIC", "-fopenmp", "-ffp-contract=off",
           "-Wall", "-Wextra"]
INCLUDES = ["-I" + os.path.join(ROOT, "include"),
            "-I" + os.path.join(HERE, "host"),
            "-I" + os.path.join(HERE, "csrc")]


def _run(cmd):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError("build step failed:\n%s\n%s" % (" ".join(cmd), r.stdout))
    out = "\n".join(l for l in r.stdout.splitlines()
                    if "packed-fp32-ops" not in l and l.strip())
    return out


def build(verbose=False):
    obj_dir = os.path.join(HERE, "_build")
    if os.path.isdir(obj_dir):
        shutil.rmtree(obj_dir)
    os.makedirs(obj_dir)
    hipcc = os.path.join(ROCM, "bin", "hipcc")
    jobs = []
    for f in sorted(os.listdir(os.path.join(HERE, "csrc"))):
        if f.endswith(".hip"):
            src = os.path.join(HERE, "csrc", f)
            obj = os.path.join(obj_dir, f[:-4] + ".o")
            jobs.append([hipcc] + HIP_FLAGS + FILE_FLAGS.get(f, []) + INCLUDES +
                        ["-c", src, "-o", obj])
    for f in sorted(os.listdir(os.path.join(HERE, "host"))):
        if f.endswith(".c"):
            src = os.path.join(HERE, "host", f)
            obj = os.path.join(obj_dir, f[:-2] + ".c.o")
            jobs.append(["gcc"] + C_FLAGS + INCLUDES + ["-c", src, "-o", obj])
    with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
        outs = list(ex.map(_run, jobs))
    if verbose:
        for o in outs:
            if o:
                print(o)
    objs = sorted(os.path.join(obj_dir, f) for f in os.listdir(obj_dir) if f.endswith(".o"))
    tmp = LIB + ".tmp"
    _run(["g++", "-shared", "-o", tmp] + objs +
         ["-L" + os.path.join(ROCM, "lib"), "-Wl,-rpath," + os.path.join(ROCM, "lib"),
          "-lamdhip64", "-fopenmp", "-lm"])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
