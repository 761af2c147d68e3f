"""Build ``libtoktier_hip.so`` and ``libtoktier_head.so`` for gfx950 with
hipcc (in-tree).

The library holds the device code object (gfx950) and the C-ABI host
engine. A manifest beside it records the sha256 of the library, the
offload architecture, the hipcc version and the exported ``tk_*`` symbols
(the role of the reference's ``tools/build_fatbin.py`` manifest).
"""

from __future__ import annotations

import ctypes as C
import hashlib
import json
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
ABI_HEADER = ROOT / "include" / "toktier_hip.h"
LIBDIR = PKG / "_lib"
LIB = LIBDIR / "libtoktier_hip.so"
MANIFEST = LIBDIR / "manifest.json"
ARCH = "gfx950"

SOURCES = ["tk_device.hip", "tk_added.hip", "tk_engine.cpp"]

# The answering end (include/toktier_head.h) is a library of its own, so that
# its sources are no part of the encode library's build key: the route
# evidence and the counter summaries stay those of the encode path.
HEAD_SRC = CSRC / "head"
HEAD_LIB = LIBDIR / "libtoktier_head.so"
HEAD_ABI_HEADER = ROOT / "include" / "toktier_head.h"
HEAD_SOURCES = ["head_norm.hip", "head_matmul.hip", "head_sample.hip",
                "head_api.cpp"]


def hashed_files() -> dict[str, Path]:
    """Every file the code object depends on, by the name the manifest
    records: all of ``csrc/`` (the compiled sources and the headers they
    include) and the C-ABI header."""
    files = {f"csrc/{f.name}": f for f in sorted(CSRC.iterdir())
             if f.is_file() and f.suffix in (".hip", ".cpp", ".h")}
    files["include/toktier_hip.h"] = ABI_HEADER
    return files


def source_digests() -> dict[str, str]:
    return {name: hashlib.sha256(f.read_bytes()).hexdigest()
            for name, f in hashed_files().items()}


def library_digest(lib: Path | None = None) -> str:
    lib = LIB if lib is None else lib
    return hashlib.sha256(b"toktier-hip-lib\0" + lib.read_bytes()).hexdigest()


HIPCC_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-Wall", "-Wno-unused-function",
    # packed FP32 instructions stay off, as a precaution
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.sep not in cand or Path(cand).exists()):
            return cand
    return "hipcc"


def exported_symbols(lib: Path) -> list[str]:
    nm = "/opt/rocm/llvm/bin/llvm-nm"
    if not Path(nm).exists():
        nm = "nm"
    out = subprocess.run([nm, "-D", "--defined-only", str(lib)],
                         capture_output=True, text=True, check=True).stdout
    return sorted({line.split()[-1] for line in out.splitlines()
                   if line.split() and line.split()[-1].startswith("tk_")})


def build_key(sources: dict, flags: list, hipcc: list) -> str:
    """Digest of what determines the code object: the sources, the flags
    and the compiler version. hipcc gives each compile a random unit id,
    so two builds of the same sources differ in a few bytes of the library
    and its own sha256 cannot name a build across rebuilds; this key can
    (the committed counter summaries are matched on it)."""
    body = json.dumps({"sources": sources, "flags": flags, "hipcc": hipcc,
                       "arch": ARCH}, sort_keys=True)
    return hashlib.sha256(b"toktier-hip-build\0" + body.encode()).hexdigest()


def build(verbose: bool = False) -> Path:
    LIBDIR.mkdir(exist_ok=True)
    tmp = LIB.with_suffix(f".so.tmp{os.getpid()}")
    cmd = [_hipcc(), *HIPCC_FLAGS, "-o", str(tmp),
           *[str(CSRC / s) for s in SOURCES]]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("hipcc build of libtoktier_hip.so failed")
    os.replace(tmp, LIB)
    ver = subprocess.run([_hipcc(), "--version"], capture_output=True,
                         text=True).stdout.strip().splitlines()
    digest = library_digest()
    sources = source_digests()
    MANIFEST.write_text(json.dumps({
        "library": LIB.name,
        "sha256_domain": "toktier-hip-lib",
        "sha256": digest,
        "build_key": build_key(sources, HIPCC_FLAGS, ver[:2]),
        "architecture": ARCH,
        "hipcc": ver[:2],
        "flags": HIPCC_FLAGS,
        "sources": sources,
        "symbols": exported_symbols(LIB),
    }, indent=1) + "\n")
    return LIB


def head_digest() -> str:
    """Digest of what ``libtoktier_head.so`` is built from: its sources, its
    header and the flags. The library holds the one that it was built from."""
    files = [f for f in sorted(HEAD_SRC.iterdir()) if f.suffix in (".hip", ".cpp", ".h")]
    body = json.dumps({"sources": {f.name: hashlib.sha256(f.read_bytes()).hexdigest()
                                   for f in (*files, HEAD_ABI_HEADER)},
                       "flags": HIPCC_FLAGS}, sort_keys=True)
    return hashlib.sha256(b"toktier-head-build\0" + body.encode()).hexdigest()


def build_head(verbose: bool = False) -> Path:
    """Build ``libtoktier_head.so`` (one compiler per source, then a link)."""
    LIBDIR.mkdir(exist_ok=True)
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    compile_flags.append(f'-DTKH_SOURCES="{head_digest()}"')
    objs, running = [], []
    for src in HEAD_SOURCES:
        obj = LIBDIR / f"{src}.{os.getpid()}.o"
        lang = ["-x", "hip"] if src.endswith(".cpp") else []
        cmd = [_hipcc(), *compile_flags, "-c", *lang, str(HEAD_SRC / src),
               "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        objs.append(obj)
        running.append(subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                        stderr=subprocess.STDOUT, text=True))
    logs = [(p.communicate()[0], p.returncode) for p in running]
    tmp = HEAD_LIB.with_suffix(f".so.tmp{os.getpid()}")
    try:
        if not any(rc for _, rc in logs):
            res = subprocess.run(
                [_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o",
                 str(tmp), *map(str, objs)], capture_output=True, text=True)
            logs.append((res.stdout + res.stderr, res.returncode))
        if any(rc for _, rc in logs):
            sys.stderr.write("".join(out for out, rc in logs if rc))
            raise RuntimeError("hipcc build of libtoktier_head.so failed")
    finally:
        for obj in objs:
            obj.unlink(missing_ok=True)
    os.replace(tmp, HEAD_LIB)
    return HEAD_LIB


def verify(manifest: dict | None = None) -> str | None:
    """None when the library on disk is the one the manifest describes and
    the sources it was built from are unchanged; else what differs (a
    stale library, or sources edited after the build)."""
    try:
        m = manifest if manifest is not None else json.loads(MANIFEST.read_text())
    except (OSError, ValueError) as err:
        return f"manifest unreadable: {err}"
    if not LIB.exists():
        return "library missing"
    if library_digest() != m.get("sha256"):
        return "library bytes differ from the manifest"
    now = source_digests()
    was = m.get("sources", {})
    changed = sorted(k for k in set(now) | set(was) if now.get(k) != was.get(k))
    if changed:
        return "sources changed since the build: " + ", ".join(changed)
    return None


def verify_head(lib: Path | None = None) -> str | None:
    """None when ``libtoktier_head.so`` is there and was built from the
    present sources, or where no sources are; else what differs."""
    lib = HEAD_LIB if lib is None else lib
    if not lib.exists():
        return "library missing"
    if not HEAD_SRC.is_dir() or not HEAD_ABI_HEADER.exists():
        return None
    sources = getattr(C.CDLL(str(lib)), "tk_head_sources", None)
    if sources is not None:
        sources.restype = C.c_char_p
    if sources is None or sources().decode() != head_digest():
        return "sources or flags changed since the build"
    return None


if __name__ == "__main__":
    build(verbose=True)
    print(LIB)
    build_head(verbose=True)
    print(HEAD_LIB)
