"""Builds librlx_adamw.so (HIP kernels + C ABI) for gfx950 with hipcc, in-tree."""
import hashlib
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = [os.path.join(HERE, "csrc", f) for f in ("rlx_adamw.hip", "rlx_losses.hip")]
OUT = os.path.join(HERE, "librlx_adamw.so")

# -ffp-contract=off: every FP32 operation of the update rounds once, as in the CPU restatement
# the results are checked against.  Packed FP32 instructions are switched off for device code.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-command-line-argument",
]


HEADERS = [os.path.join(ROOT, "include", "rlx_adamw.h"), os.path.join(HERE, "csrc", "rlx_internal.h")]
STAMP = OUT + ".srchash"


def source_hash():
    """Hash of everything the library is built from (kernel sources, headers, compiler flags)."""
    h = hashlib.sha256()
    for path in SOURCES + HEADERS:
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(HIPCC_FLAGS).encode())
    return h.hexdigest()


def is_current():
    """True if the built library was made from the sources as they are now."""
    try:
        return os.path.exists(OUT) and open(STAMP).read().strip() == source_hash()
    except OSError:
        return False


def is_stale():
    """True if the library carries a source stamp and the stamp differs from the sources in the tree.  A library
    without a stamp was built by other means (the documented hipcc line, CMake) and is not judged here."""
    try:
        return os.path.exists(OUT) and os.path.exists(STAMP) and open(STAMP).read().strip() != source_hash()
    except OSError:
        return False


def hipcc_path():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


def build_library(verbose=False):
    """Compiles the library every time it is called; returns the path of the .so."""
    hipcc, objects, jobs = hipcc_path(), [], []
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"] + ["-I", os.path.join(ROOT, "include"), "-c"]
    try:
        for src in SOURCES:                       # side by side: the loss kernels alone take a minute and a half
            objects.append("%s.%d.%s.o" % (OUT, os.getpid(), os.path.basename(src)))
            jobs.append(subprocess.Popen([hipcc] + compile_flags + ["-o", objects[-1], src], stdout=subprocess.DEVNULL,
                                         stderr=subprocess.PIPE, text=True))
        stderr = [j.communicate()[1] for j in jobs]
        failed = any(j.returncode != 0 for j in jobs)
        if not failed:
            res = subprocess.run([hipcc, "--offload-arch=gfx950", "-shared", "-o", OUT + ".tmp"] + objects,
                                 capture_output=True, text=True)
            stderr.append(res.stderr)
            failed = res.returncode != 0
    finally:
        for path in objects:
            if os.path.exists(path):
                os.remove(path)
    noise = "packed-fp32-ops"
    err = "\n".join(l for l in "".join(stderr).splitlines() if noise not in l)
    if failed:
        raise RuntimeError("hipcc failed:\n" + err)
    if verbose and err.strip():
        print(err)
    os.replace(OUT + ".tmp", OUT)
    with open(STAMP, "w") as f:
        f.write(source_hash() + "\n")
    return OUT


if __name__ == "__main__":
    print(build_library(verbose=True))
