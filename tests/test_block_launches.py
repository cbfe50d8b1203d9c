"""The block operators' launches (CPU only): the built library driven by the programs of tests/cpp, which record the kernels it
would launch, their grids and arguments."""
from __future__ import annotations

import os
import subprocess
from pathlib import Path

import ascq

ROOT = Path(__file__).resolve().parent.parent
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _run(tmp_path, name):
    exe = tmp_path / name
    libdir = Path(ascq.LIB_PATH).parent
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-x", "hip", "-std=c++17", "-O1",
                    "-I", str(ROOT / "include"), "-I", str(libdir / "csrc"), str(ROOT / "tests" / "cpp" / f"{name}.cpp"),
                    "-rdynamic", "-L", str(libdir), "-lascq", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib", "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]


def test_rows_past_k_are_past_the_range(tmp_path):
    """w [K, N] of large row pitches: what the tiles read past K is nothing of w"""
    _run(tmp_path, "linear_pitches")


def test_norm_of_very_many_rows(tmp_path):
    """up to 2^31 rows: every row once, no grid of 2^32 threads"""
    _run(tmp_path, "norm_rows")


def test_routing_and_rows_of_very_many_tokens(tmp_path):
    """up to 2^31 rows: every token once, no grid of 2^32 threads"""
    _run(tmp_path, "moe_tokens")


def test_linear_of_very_many_tiles(tmp_path):
    """outputs of more tiles than a grid has room for"""
    _run(tmp_path, "linear_grids")
