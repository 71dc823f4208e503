"""The generated code of the 8-bit kernels: what fits on a compute unit is what the launches assume."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> what the metadata says of it"""
    src = os.path.join(ROOT, "neurondb_amd", "csrc", "ndbhip_int8.hip")
    make = open(os.path.join(os.path.dirname(src), "Makefile")).read()
    flags = re.search(r"^CXXFLAGS \?= (.*?[^\\])$", make, re.S | re.M).group(1).replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    flags += re.search(r"ndbhip_int8.o: CXXFLAGS \+= (.*)", make).group(1).split()
    out = str(tmp_path_factory.mktemp("asm") / "i8.s")
    subprocess.run(["/opt/rocm/bin/hipcc", *flags, "--cuda-device-only", "-S", src, "-o", out], check=True, stderr=subprocess.DEVNULL)
    found = {}
    for part in open(out).read().split("  - .agpr_count:")[1:]:
        found[re.search(r"\.name:\s+(\S+)", part).group(1)] = {k: int(v) for k, v in re.findall(r"\.(\w+):\s+(\d+)\n", part)}
    return found


def test_blocks_of_a_tile_that_fit_a_compute_unit(kernels):
    """the launch deals the narrow tile two blocks a compute unit without biases and masks, and every other tile one: what LDS and
    registers have room for, so that no block waits for another to end"""
    tiles = {n: k for n, k in kernels.items() if "k_i8_tile" in n}
    assert len(tiles) == 2 * (4 + 2 * 2 * 3)
    for name, k in tiles.items():
        width, bias, mask = re.search(r"k_i8_tileILi(\d)E6I8KindILi\dELb(\d)ELb(\d)", name).groups()
        waves = k["max_flat_workgroup_size"] // 64
        per_simd = 512 // (-(-k["vgpr_count"] // 8) * 8)
        fit = min(160 * 1024 // k["group_segment_fixed_size"], per_simd * 4 // waves)
        assert fit == (2 if (width, bias, mask) == ("2", "0", "0") else 1), (name, k["vgpr_count"], k["group_segment_fixed_size"])
