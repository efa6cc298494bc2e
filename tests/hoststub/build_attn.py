"""Builds the host-only library (build.py) with the attention's host code (attn_host.cpp) and its launchers' stand-ins
(attn_stub.cpp): tests/hoststub/_build/libijah_hoststub_attn.so. TEST INFRASTRUCTURE ONLY."""
import importlib.util
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent
OUT = HERE / "_build" / "libijah_hoststub_attn.so"


def build():
    spec = importlib.util.spec_from_file_location("hoststub_build", HERE / "build.py")
    base = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(base)
    csrc = base.ROOT / "ijah_amd" / "csrc"
    sources = base.SOURCES + [csrc / "attn_host.cpp", HERE / "attn_stub.cpp"]
    newer = sources + [csrc / "attn.h", csrc / "common.h", base.ROOT / "include" / "ijah_attn.h"]
    if OUT.exists() and all(s.stat().st_mtime < OUT.stat().st_mtime for s in newer):
        return OUT
    OUT.parent.mkdir(exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-Wno-format-truncation", "-I/opt/rocm/include", f"-I{base.ROOT / 'include'}", *map(str, sources),
                    "-o", str(OUT)], check=True, capture_output=True, text=True)
    return OUT
