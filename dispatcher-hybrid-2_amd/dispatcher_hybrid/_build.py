"""Build libdh_mixer.so (gfx950) in-tree from ``csrc/*.hip``, and the torch extension of ``csrc/host`` beside it.

    python -m dispatcher_hybrid._build

Compiles every translation unit with ``hipcc --offload-arch=gfx950`` in parallel, links one shared
library into ``dispatcher_hybrid/_lib/``, and replaces the old file atomically. Needs only hipcc
(no GPU): the code objects are embedded in the library.
"""

import glob
import os
import shutil
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
PROJECT_DIR = os.path.dirname(PKG_DIR)                      # dispatcher-hybrid-2_amd/
CSRC_DIR = os.path.join(PROJECT_DIR, "csrc")
REPO_DIR = os.path.dirname(PROJECT_DIR)
INCLUDE_DIRS = [os.path.join(REPO_DIR, "include"), CSRC_DIR]
OUT_DIR = os.path.join(PKG_DIR, "_lib")
LIB = os.path.join(OUT_DIR, "libdh_mixer.so")
NODES_SRC = os.path.join(CSRC_DIR, "host", "vocab_nodes.cpp")
NODES_LIB = os.path.join(OUT_DIR, "_vocab_nodes.so")

ARCH = os.environ.get("DH_OFFLOAD_ARCH", "gfx950")
HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")

# Packed-fp32 VALU ops stay off: hipcc may only use scalar fp32 instructions.
COMMON_FLAGS = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
                "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                "-Wno-unused-command-line-argument"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC_DIR, "*.hip")))


def nodes_command(out):
    """The host compiler's command for the torch extension (no device code; it finds the kernels at run time)."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(HIPCC)))
    system = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
              os.path.join(rocm, "include"), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    return ([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall",
             "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f'-DDH_TORCH_VERSION="{torch.__version__}"',
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
            + [a for d in system for a in ("-isystem", d)] + [f"-I{d}" for d in INCLUDE_DIRS]
            + [NODES_SRC, "-o", out, f"-L{os.path.join(root, 'lib')}"]
            + [f"-l{n}" for n in ("c10", "c10_hip", "torch_cpu", "torch_hip", "torch", "torch_python")])


def _quiet(out):
    return "\n".join(l for l in out.decode(errors="replace").splitlines() if "packed-fp32-ops" not in l)


def _start_nodes():
    """(command, process) of the extension's compilation, the process None and the reason in the command's place where it cannot
    begin (no torch, no host compiler)."""
    try:
        cmd = nodes_command(NODES_LIB + ".tmp")
        return " ".join(cmd), subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    except (ImportError, OSError) as e:
        return f"{type(e).__name__}: {e}", None


def _end_nodes(cmd, process, verbose):
    """Put the extension in place. Where it does not compile (no Python or torch headers, say) the kernel library stays as it
    is: importing fused_vocab raises ImportError, and nothing else needs the extension."""
    out = "" if process is None else _quiet(process.communicate()[0])
    if process is not None and process.returncode == 0 and "warning:" not in out:
        os.replace(NODES_LIB + ".tmp", NODES_LIB)
        if verbose and out.strip():
            print(out)
        return
    for path in (NODES_LIB, NODES_LIB + ".tmp"):               # (an older one would be of other sources)
        if os.path.exists(path):
            os.remove(path)
    print(f"the torch extension of csrc/host was not built; dispatcher_hybrid.fused_vocab needs it:\n$ {cmd}\n{out}",
          file=sys.stderr, flush=True)


def build(verbose=False):
    srcs = sources()
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC_DIR}")
    os.makedirs(OUT_DIR, exist_ok=True)
    inc = [f"-I{d}" for d in INCLUDE_DIRS]
    with tempfile.TemporaryDirectory(prefix="dh_build_") as tmp:
        nodes = _start_nodes()
        procs = []
        objs = []
        for src in srcs:
            obj = os.path.join(tmp, os.path.basename(src) + ".o")
            objs.append(obj)
            cmd = [HIPCC] + COMMON_FLAGS + inc + ["-c", src, "-o", obj]
            procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        failed = []
        for cmd, p in procs:
            out = _quiet(p.communicate()[0])
            if p.returncode != 0 or "warning:" in out:
                # warnings fail the build too (an inline-asm clobber of a reserved register is one)
                failed.append(f"$ {' '.join(cmd)}\n{out}")
            elif verbose and out.strip():
                print(out)
        if failed:
            if nodes[1] is not None:
                nodes[1].kill()
                nodes[1].communicate()
            raise RuntimeError("hipcc failed:\n" + "\n".join(failed))
        tmp_lib = LIB + ".tmp"
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp_lib] + objs
        p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
        if p.returncode != 0:
            raise RuntimeError(f"link failed:\n$ {' '.join(cmd)}\n{p.stdout.decode(errors='replace')}")
        os.replace(tmp_lib, LIB)
        _end_nodes(*nodes, verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
