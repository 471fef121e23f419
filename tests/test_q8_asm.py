"""The 8-bit cache's and the tables' kernels as gfx950 assembly, with the library's flags: none spills, none keeps
anything in scratch memory, and the decode of up to 8 heads a kv head keeps its registers below what lets two workgroups
share a CU (8 waves) or one of 12 waves run."""
import re
import subprocess

import pytest

from test_kernel_asm import _flags, _hipcc_or_skip

SOURCES = ("atf_decode_q8.hip", "atf_kv_write_q8.hip", "atf_tables.hip")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> (spills, scratch bytes, vector registers)."""
    B = _hipcc_or_skip()
    out = {}
    for src in B.sources():
        if not src.endswith(SOURCES):
            continue
        path = tmp_path_factory.mktemp("asm") / "k.s"
        subprocess.run([B.HIPCC, *_flags(B, src), "-I", B.CSRC, "--cuda-device-only", "-S", src, "-o", str(path)], check=True,
                       capture_output=True, text=True)
        for block in path.read_text().split("- .agpr_count")[1:]:
            get = lambda key: int(re.search(r"\.%s:\s+(\d+)" % key, block).group(1))  # noqa: E731
            name = re.search(r"\.name:\s+(\S+)", block).group(1)
            out[name] = (get("vgpr_spill_count") + get("sgpr_spill_count"), get("private_segment_fixed_size"), get("vgpr_count"))
    return out


def test_nothing_spills(kernels):
    assert len(kernels) >= 14
    for name, (spills, scratch, _) in kernels.items():
        assert spills == 0 and scratch == 0, name


def test_decode_registers_leave_room_for_the_waves(kernels):
    names = [n for n in kernels if "decode_q8_kernel" in n]
    assert len(names) == 8
    for n in names:
        wide, waves = re.search(r"ILb[01]ELb([01])ELi(\d+)E", n).groups()
        regs = kernels[n][2]
        # 512 registers a SIMD lane, in steps of 8: 4 waves at 128, 3 at 168
        assert regs <= (168 if waves == "12" else 256 if wide == "1" else 128), (n, regs)
