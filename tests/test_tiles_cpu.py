"""The rule that gives a block operator's products their tiles and splits (csrc/ec_gemm.h, ec_ff.hip, ec_ortho.hip), for
the sizes of the GPU tests, compiled for the host."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from test_gpu_block_tiles import FF, ORTHO

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_sizes_take_the_tiles_that_they_are_for(tmp_path):
    exe, none = tmp_path / "tiles", tmp_path / "none"
    none.write_bytes(b"")   # in the place of the device code
    subprocess.run([HIPCC, "-O1", "-std=c++17", "--offload-arch=gfx950", "--offload-host-only",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "megatron-lm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "tiles_driver.hip"), "-Xclang", "-fcuda-include-gpubinary", "-Xclang", str(none),
                    "-o", str(exe)], check=True)
    sizes = [(f"ff {'bf16' if kind == 'narrow' else kind} {n} {width} {inner} 1", tiles) for kind, n, width, inner, tiles in FF]
    sizes += [(f"ff fp16 {n} {width} {inner} 1", tiles) for kind, n, width, inner, tiles in FF if kind == "narrow"]
    sizes += [(f"ortho {kind} {batch} {rows} {cols}", tiles) for kind, batch, rows, cols, tiles in ORTHO]
    got = subprocess.run([str(exe)], input="\n".join(line for line, _ in sizes), capture_output=True, text=True, timeout=60)
    assert got.returncode == 0
    assert got.stdout.splitlines() == [tiles for _, tiles in sizes]
    # each kind of product takes every shape, split and not, that is built for it
    for rows, types, products in ((FF, ("narrow", "fp32"), 3), (ORTHO, ("fast", "exact"), 3)):
        for kind in types:
            for at in range(products):
                shapes = {row[-1].split()[at].split("/")[0] for row in rows if row[0] == kind}
                assert shapes == ({"middle", "least"} if kind == "exact" else {"large", "middle", "least"}), (kind, at)
