"""Build libs2t_hip.so (all HIP kernels + the C-ABI) in-tree for gfx950 with hipcc.

The built library lives at ``s2t_amd/lib/libs2t_hip.so`` (git-ignored, shipped to the GPU box by gpurun).
Objects are cached by source mtime and by the command that made them (kept beside each as ``*.cmd``), so that a rebuild after touching one
kernel takes seconds and none of another set of flags is ever linked.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libs2t_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-result",
         # no packed fp32 instructions: some of their forms have given wrong results on MI355X now and then, without an error
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# Per-file extras.  attention_fused.hip: hipcc puts the MFMA results of the fused attention kernels into AccVGPRs and copies
# every one of them out again for the softmax arithmetic (64 v_accvgpr moves per 16 x 64 step in kernels that are bound by
# vector issue); with the results in ordinary VGPRs the copies are gone and the kernels need FEWER registers (dQ 224 -> 208,
# the decoder's dK/dV 180 -> 168): dQ 44.1 -> 43.3 us, dK/dV 46.6 -> 44.4 us per launch on MI355X.
# paged.hip: the same (one tile row of 64-wide bf16 heads: 172 -> 148 registers, three waves of a SIMD instead of two).
FILE_FLAGS = {"attention_fused.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"], "paged.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}


def flags_of(src):
    return FLAGS + FILE_FLAGS.get(os.path.basename(src), [])


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _deps_mtime():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    hs.append(os.path.join(os.path.dirname(HERE), "include", "s2t_hip.h"))
    return max(os.path.getmtime(h) for h in hs)


def _record(cmd):
    """``cmd`` as it is kept: the same wherever the tree lies."""
    return "\n".join(cmd).replace(os.path.dirname(HERE), ".")


def _current(out, cmd, inputs_mtime):
    """Whether ``out`` is there, made by ``cmd`` and no older than what it was made of."""
    try:
        with open(out + ".cmd") as f:
            return f.read() == _record(cmd) and os.path.getmtime(out) >= inputs_mtime
    except FileNotFoundError:
        return False


def _make(out, cmd, failed):
    """Runs ``cmd``, which makes ``out``; the record of the command is there only while both are whole."""
    if os.path.exists(out + ".cmd"):
        os.remove(out + ".cmd")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("%s:\n%s" % (failed, r.stderr[-4000:]))
    with open(out + ".cmd", "w") as f:
        f.write(_record(cmd))


def build(force=False, verbose=True):
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    hdr = _deps_mtime()
    jobs = []
    objs = []
    for src in _sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        cmd = [HIPCC] + flags_of(src) + ["-c", src, "-o", obj]
        if force or not _current(obj, cmd, max(os.path.getmtime(src), hdr)):
            jobs.append((src, obj, cmd))

    def cc(job):
        src, obj, cmd = job
        _make(obj, cmd, "hipcc failed for " + src)
        return src

    if jobs:
        with ThreadPoolExecutor(max_workers=min(6, len(jobs))) as ex:
            for done in ex.map(cc, jobs):
                if verbose:
                    print("[s2t_amd.build] compiled", os.path.basename(done), flush=True)
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if jobs or not _current(LIB, cmd, max(os.path.getmtime(o) for o in objs)):
        _make(LIB, cmd, "link failed")
        if verbose:
            print("[s2t_amd.build] linked", LIB, flush=True)
    return LIB


if __name__ == "__main__":
    if len(sys.argv) == 3 and sys.argv[1] == "--flags":  # of one source, for a script that compiles a variant of it
        print(" ".join(flags_of(sys.argv[2])))
    else:
        build(force="--force" in sys.argv)
