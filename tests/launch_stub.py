"""Builds the stub of the HIP launch (launch_order_stub.cpp) that tests on the CPU preload under the library."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
LIB = HERE.parent / "efficient-inference-system_amd" / "libpaged_hip.so"


def build(folder: Path) -> Path:
    gxx = shutil.which("g++")
    if gxx is None or not LIB.exists() or not Path("/opt/rocm/include/hip/hip_runtime_api.h").exists():
        pytest.skip("needs g++, the HIP headers and the built library")
    out = folder / "libstub.so"
    subprocess.run([gxx, "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(HERE / "launch_order_stub.cpp"), "-o", str(out), "-pthread"], check=True, timeout=120)
    return out
