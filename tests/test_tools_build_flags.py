"""The tools that compile kernels by themselves compile them as the library's Makefile does: a sheet or a variant of other code says nothing about it."""
import importlib.util
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def read(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def test_tools_leave_packed_fp32_out_as_the_makefile_does():
    flags = " ".join(re.search(r"^CXXFLAGS \+= (-Xclang .*)$", read("gs-sdf_amd", "csrc", "Makefile"), re.M).group(1).split())
    assert flags == "-Xclang -target-feature -Xclang -packed-fp32-ops"
    compiles = [line for line in read("tools", "build_variants.sh").splitlines() if "hipcc" in line and " -c " in line]
    assert compiles and all(flags in line for line in compiles)


def test_resource_sheet_compiles_each_kernel_as_the_makefile_does(monkeypatch):
    spec = importlib.util.spec_from_file_location("kernel_resources", os.path.join(ROOT, "tools", "kernel_resources.py"))
    tool = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(tool)
    seen = []
    monkeypatch.setattr(tool.subprocess, "run", lambda cmd, **kw: seen.append(cmd))
    make = read("gs-sdf_amd", "csrc", "Makefile")
    strict = set(re.search(r"^STRICT_SRCS := (.*)$", make, re.M).group(1).split())
    no_slp = set(re.findall(r"\$\(OBJ\)/(\w+)\.o", re.search(r"^(.*): CXXFLAGS \+= -fno-slp-vectorize$", make, re.M).group(1)))
    for src in sorted(strict) + ["raster_fwd.hip", "raster_bwd.hip", "lowrank_bf16.hip", "mlp.hip"]:
        tool.assemble(src, "out.s")
        cmd = " ".join(seen[-1])
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in cmd and "-O3" in cmd and "--offload-arch=gfx950" in cmd
        assert ("-ffp-contract=off" in cmd) == (src in strict) and ("-fno-slp-vectorize" in cmd) == (src[:-4] in no_slp)
