"""CPU (hipcc cross-compiles gfx950): the flags that the device units are built
with reach their code, and the hash that ties a counter profile to a kernel
build changes with them."""
import json
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from gene2vec_amd import build as B

PACKED = re.compile(r"\bv_pk_(add|mul|fma)_f32\b")
UNITS = [("g2v_sgns_atomic.hip", ["-DG2V_K=5"]), ("g2v_sgns.hip", ["-DG2V_K=5"]),
         ("g2v_kernels.hip", []), ("g2v_api.hip", []), ("g2v_coexpr.hip", []),
         ("g2v_embed.hip", []), ("g2v_gradnorm.hip", [])]


def assembly(out, src, defs, flags):
    cmd = [B.hipcc(), *B.COMPILE_FLAGS, *flags, "-I", os.path.join(B.ROOT, "include"), "-I", B.CSRC,
           *defs, "--cuda-device-only", "-S", os.path.join(B.CSRC, src), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    return open(out).read()


def test_every_device_unit_is_listed():
    assert {u[0] for u in UNITS} == {u[0] for u in B.UNITS if u[0].endswith(".hip")}
    for src, _, _ in B.UNITS:
        flags = " ".join(B.unit_flags(src))
        assert ("-packed-fp32-ops" in flags) == src.endswith(".hip")


@pytest.mark.timeout(900)
def test_no_packed_fp32_arithmetic(tmp_path):
    def packed(i):
        src, defs = UNITS[i]
        asm = assembly(str(tmp_path / f"{i}.s"), src, defs, B.unit_flags(src))
        assert "s_endpgm" in asm or src == "g2v_api.hip", src  # (host code only)
        return src, len(PACKED.findall(asm))
    with ThreadPoolExecutor(4) as pool:
        assert all(n == 0 for _, n in pool.map(packed, range(len(UNITS))))
    # what the flag is for: without it the same source has them
    src, defs = UNITS[0]
    assert PACKED.search(assembly(str(tmp_path / "without.s"), src, defs, B.SGNS_KERNEL_FLAGS[4:]))


def test_kernel_hash_covers_the_flags(monkeypatch):
    here = B.kernel_source_hash()
    assert re.fullmatch("[0-9a-f]{16}", here)
    for name, value in (("DEVICE_FLAGS", ()), ("SGNS_KERNEL_FLAGS", B.DEVICE_FLAGS),
                        ("COMPILE_FLAGS", (*B.COMPILE_FLAGS, "-O2"))):
        with monkeypatch.context() as m:
            m.setattr(B, name, value)
            if name == "DEVICE_FLAGS":
                m.setattr(B, "SGNS_KERNEL_FLAGS", B.SGNS_KERNEL_FLAGS[4:])
            assert B.kernel_source_hash() != here
    assert B.kernel_source_hash() == here
    # counters of the kernels with packed arithmetic are of another build
    old = json.load(open(os.path.join(B.ROOT, "profiles", "r06", "traffic_r06.json")))
    assert old["kernel_src_sha16"] != here


def test_norm_and_clip_workgroups_are_all_resident(tmp_path):
    """their grids are sized to 8 waves a SIMD"""
    src = "g2v_gradnorm.hip"
    cmd = [B.hipcc(), *B.COMPILE_FLAGS, *B.unit_flags(src), "-I", os.path.join(B.ROOT, "include"),
           "-I", B.CSRC, "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c",
           os.path.join(B.CSRC, src), "-o", str(tmp_path / "x.o")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    found = 0
    for part in r.stderr.split("Function Name: ")[1:]:
        if re.match(r"\S*(k_square_sum|k_clip)", part):
            found += 1
            assert re.search(r"Occupancy \[waves/SIMD\]: 8\b", part), part
            assert re.search(r"VGPRs Spill: 0\b", part), part
    assert found == 6
