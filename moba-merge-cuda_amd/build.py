"""Build libmoba_hip.so (gfx950) and the host path _calls.so in-tree.

Every ``csrc/*.hip`` (device code) and ``csrc/*.cpp`` (host-only runtime:
page pool, prepared-decode driver) file is compiled to an object under ``_build/`` and
linked into ``moba_hip/libmoba_hip.so``.  ``csrc/python/calls.cpp`` (host-only,
against torch's headers) becomes the extension ``moba_hip/_calls.so``, for the
torch and Python that build it; without torch the library alone is built, which is
all that callers of the C-ABI need.  Objects are rebuilt when their source or any
header changed, the extension's also when its torch or Python did.  ``python
build.py`` builds; ``--force`` rebuilds everything.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
OUT_DIR = ROOT / "_build"
LIB = ROOT / "moba_hip" / "libmoba_hip.so"
CALLS = ROOT / "moba_hip" / "_calls.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-ffp-contract=off",
    # packed fp32 ops are disabled on this pool (device-side flag; the host
    # pass warns that it does not know the feature).
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in VGPRs: no accumulator round trips through AGPRs for
    # the short-lived S / dP tiles
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-Wall", "-Wno-unused-result",
]


def _headers():
    hs = list(CSRC.glob("*.h")) + list((ROOT.parent / "include").glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _flags(src: Path):
    if src.suffix == ".cpp":  # host-only sources: the host compiler, HIP runtime API only
        return ["-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-result", "-D__HIP_PLATFORM_AMD__",
                "-I/opt/rocm/include"]
    return FLAGS


def _compile(src: Path, force: bool) -> Path:
    obj = OUT_DIR / (src.name + ".o")  # suffix kept: foo.hip and foo.cpp get distinct objects
    if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, _headers()):
        cc = os.environ.get("CXX", "g++") if src.suffix == ".cpp" else HIPCC
        cmd = [cc, *_flags(src), "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError(f"hipcc failed on {src.name}")
    return obj


def _calls_target():
    """(what _calls.so is built for, include paths, library folder), or None
    without torch, whose headers it needs."""
    try:
        import torch
        from torch.utils.cpp_extension import include_paths
    except ImportError:
        return None
    import sysconfig
    dirs = [*include_paths(), sysconfig.get_paths()["include"]]
    flags = [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             *[f"-I{d}" for d in dirs]]
    built_for = f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"
    return built_for, flags, Path(torch.__file__).parent / "lib"


def _compile_calls(force: bool):
    target = _calls_target()
    if target is None:
        return None
    built_for, flags, _ = target
    src, obj, stamp = CSRC / "python" / "calls.cpp", OUT_DIR / "calls.cpp.o", OUT_DIR / "calls.cpp.for"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-w", *flags,
           f'-DMOBA_BUILT_FOR="{built_for}"', "-c", str(src), "-o", str(obj)]
    made = stamp.read_text() if stamp.exists() else None
    if force or made != " ".join(cmd) or not obj.exists() or \
            obj.stat().st_mtime < max(src.stat().st_mtime, _headers()):
        stamp.unlink(missing_ok=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("g++ failed on calls.cpp")
        stamp.write_text(" ".join(cmd))
    return obj


def _link_calls(obj: Path, force: bool) -> None:
    if not force and CALLS.exists() and CALLS.stat().st_mtime >= obj.stat().st_mtime:
        return
    libs = _calls_target()[2]
    tmp = CALLS.with_suffix(f".so.{os.getpid()}")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-shared", str(obj), "-o", str(tmp),
                           f"-L{LIB.parent}", "-l:libmoba_hip.so", "-Wl,-rpath,$ORIGIN",
                           f"-L{libs}", "-ltorch_python", "-ltorch_cpu", "-lc10"])
    os.replace(tmp, CALLS)


def build(force: bool = False, jobs: int = 8) -> Path:
    OUT_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip")) + sorted(CSRC.glob("*.cpp"))
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        calls = ex.submit(_compile_calls, force)
        objs = list(ex.map(lambda s: _compile(s, force), sources))
    newest = max(o.stat().st_mtime for o in objs)
    if force or not LIB.exists() or LIB.stat().st_mtime < newest:
        tmp = LIB.with_suffix(f".so.{os.getpid()}")
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
        subprocess.check_call(cmd)
        os.replace(tmp, LIB)
    if calls.result() is None:
        sys.stderr.write("no torch: libmoba_hip.so alone is built, without the Python host path\n")
    else:
        _link_calls(calls.result(), force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
