"""In-tree hipcc build of the CDNA4 extensions (gfx950 only, no JIT cache).

Built .so files live next to this file (git-ignored), so that a copy of the
tree carries them to machines that do not build.
"""
from __future__ import annotations

import os
import subprocess
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent
CSRC = PKG / "csrc"
OUT = PKG / "ops"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CXX = os.environ.get("CXX", "g++")
ARCH = os.environ.get("RLS_OFFLOAD_ARCH", "gfx950")

# Packed FP32 instructions stay off: hipcc -O3 forms them from ordinary float
# code, and some of their forms have given wrong results on this part.
# (hipcc's host pass warns that it does not know the feature; harmless.)
FLAGS = ["-O3", "-std=c++17", "-fPIC", "-shared",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# of the torch bindings, beside the paths of torch and ROCm
BIND_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared",
              "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
              "-Wl,-rpath,$ORIGIN", "-Wl,--no-as-needed"]
BIND_LIBS = ["-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip",
             "-ltorch_python"]

# name -> sources
_LIBS = {
    "librlsched_env.so": ["env_step.hip"],
    "librlsched_nn.so": ["nn_kernels.hip"],
    "librlsched_train.so": ["train_kernels.hip"],
    "librlsched_gru.so": ["gru_train.hip"],
    "librlsched_mega.so": ["rollout_mega.hip"],
    "librlsched_norm.so": ["layer_norm.hip"],
    "librlsched_scan.so": ["gated_scan.hip"],
    "librlsched_logp.so": ["logprob.hip"],
    "librlsched_seq.so": ["seq_bind.cpp"],
}

# torch bindings: host code, linked with the kernel libraries beside them
_BINDS = {
    "librlsched_seq.so": ["librlsched_norm.so", "librlsched_scan.so",
                          "librlsched_logp.so"],
}


def _bind_flags(name: str) -> list[str]:
    import sysconfig

    import torch
    root = Path(torch.__file__).resolve().parent
    rocm = Path(HIPCC).resolve().parent.parent
    abi = int(torch.compiled_with_cxx11_abi())
    return ([*BIND_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
             f"-I{sysconfig.get_paths()['include']}"]
            + [f"-isystem{d}" for d in
               (root / "include", root / "include/torch/csrc/api/include",
                rocm / "include")]
            + [f"-L{root / 'lib'}", f"-L{OUT}"]
            + [f"-l:{lib}" for lib in _BINDS[name]] + BIND_LIBS)


def source_hash(name: str) -> str:
    """sha256-prefix over this lib's sources + all shared headers + the
    compile flags. Embedded at compile time (-DRLS_SOURCE_HASH) and checked
    at load: a .so whose sources changed can never silently test old
    kernels."""
    import hashlib
    h = hashlib.sha256(" ".join(FLAGS).encode())
    if name in _BINDS:
        import torch
        h.update(torch.__version__.encode())
        h.update(" ".join(BIND_FLAGS + _BINDS[name] + BIND_LIBS).encode())
    srcs = [CSRC / s for s in _LIBS[name]] + sorted(CSRC.glob("*.h"))
    for p in sorted(srcs):
        h.update(p.name.encode())
        h.update(p.read_bytes())
    return h.hexdigest()[:16]


def embedded_hash(so: Path) -> str | None:
    """Read the RLSHASH marker from the binary without dlopen (dlopen
    caches handles per path, so a load-check-rebuild-reload cycle would
    see the stale mapping)."""
    data = so.read_bytes()
    i = data.find(b"RLSHASH:")
    if i < 0:
        return None
    return data[i + 8:i + 24].decode(errors="replace")


def _needs_build(so: Path, srcs: list[Path], name: str) -> bool:
    if not so.exists():
        return True
    # content-addressed: rebuild IFF the embedded source hash disagrees
    # (mtimes are unreliable across clones/snapshots)
    return embedded_hash(so) != source_hash(name)


def build_lib(name: str, verbose: bool = False, force: bool = False) -> Path:
    srcs = [CSRC / s for s in _LIBS[name]]
    missing = [s for s in srcs if not s.exists()]
    if missing:
        raise FileNotFoundError(f"missing sources for {name}: {missing}")
    so = OUT / name
    if not force and not _needs_build(so, srcs, name):
        return so
    h = source_hash(name)
    tmp = so.with_suffix(f".{os.getpid()}.tmp")   # replaced whole, when done
    head = ([CXX] if name in _BINDS
            else [HIPCC, f"--offload-arch={ARCH}", *FLAGS])
    cmd = [*head, f'-DRLS_SOURCE_HASH="{h}"', "-o", str(tmp),
           *(str(s) for s in srcs)]
    if name in _BINDS:
        for lib in _BINDS[name]:
            build_lib(lib, verbose)
        cmd += _bind_flags(name)
    if verbose:
        print("+", " ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        tmp.unlink(missing_ok=True)
        raise RuntimeError(f"{cmd[0]} failed for {name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, so)
    got = embedded_hash(so)
    if got != h:
        raise RuntimeError(f"{name}: embedded hash {got!r} != expected {h!r} "
                           "after build")
    return so


def verify_loaded(lib, name: str) -> None:
    """Assert a dlopen'ed lib carries the hash of the current sources.
    Called by every ops loader right after CDLL."""
    import ctypes
    try:
        fn = lib.rlsched_source_hash
    except AttributeError:
        raise RuntimeError(
            f"{name} has no rlsched_source_hash export — stale pre-round-2 "
            "binary; delete it and rebuild (python -m "
            "rlgpuschedule_amd.ops.build)") from None
    fn.restype = ctypes.c_char_p
    got = fn().decode(errors="replace").split("RLSHASH:")[-1]
    want = source_hash(name)
    if got != want:
        raise RuntimeError(
            f"{name} is stale: embedded source hash {got} != computed "
            f"{want}; the mapped binary does not match csrc/ — rebuild")


def build_all(verbose: bool = False, force: bool = False) -> list[Path]:
    """Build every library (force: also those whose binary is current),
    a few compilers at a time, and then the bindings linked with them."""
    from concurrent.futures import ThreadPoolExecutor
    names = [name for name, srcs in _LIBS.items()
             if all((CSRC / s).exists() for s in srcs)]
    kernels = [n for n in names if n not in _BINDS]
    with ThreadPoolExecutor(max_workers=4) as pool:
        out = list(pool.map(lambda n: build_lib(n, verbose, force), kernels))
    return out + [build_lib(n, verbose, force) for n in names if n in _BINDS]


if __name__ == "__main__":
    for p in build_all(verbose=True):
        print("built", p)
