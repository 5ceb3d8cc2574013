"""The build rules of mamba_unet_amd/csrc/Makefile, as `make -n` prints them (nothing is compiled)."""
import os
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "mamba_unet_amd", "csrc")
SCALAR = ("ss2d_linattn_fwd", "ss2d_linattn_bwd", "ss2d_linattn_step", "ss2d_blocknorm", "ss2d_gradclip", "ss2d_colsum")


def commands(*args):
    out = subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], check=True, capture_output=True, text=True)
    return out.stdout.splitlines()


@pytest.mark.parametrize("args", [(), ("CXXFLAGS=-O1 --offload-arch=gfx950",)], ids=["default", "own flags"])
def test_no_packed_fp32_in_the_operators_beside_the_scan(args):
    lines = commands(*args)
    for name in SCALAR:
        line, = [x for x in lines if f"-c {name}.hip" in x]
        assert "-packed-fp32-ops" in line, name


@pytest.mark.parametrize("name", SCALAR)
def test_a_variant_is_compiled_as_the_file_itself(name):
    line = [x for x in commands("variant", f"SRC={name}", "NAME=other", "DEFS=-DX") if f"-c {name}.hip" in x and "-DX" in x]
    assert len(line) == 1 and "-packed-fp32-ops" in line[0]


def test_the_library_alone_is_built_without_torch():
    host, library = "host_ops.cpp", "-shared -o ../libss2d_hip.so"
    both = "\n".join(commands())
    assert host in both and library in both
    for args in (("PYTHON=false",), ("lib",)):
        only = "\n".join(commands(*args))
        assert host not in only and library in only
