"""The kernels of norms, log probabilities and shared pages as gfx950 assembly, with the library's flags: none spills or keeps anything in
scratch memory, and the log probabilities' keep to the registers that their waves share a SIMD with."""
import re
import subprocess

import pytest

from test_kernel_asm import _flags, _hipcc_or_skip

SOURCES = ("atf_qk_norm.hip", "atf_logprobs.hip", "atf_pages.hip")


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
    assert len(kernels) >= 15
    for name, (spills, scratch, _) in kernels.items():
        assert spills == 0 and scratch == 0, name


def test_log_probabilities_leave_room_for_four_waves_a_simd(kernels):
    names = [n for n in kernels if "token_logprobs_kernel" in n]
    assert len(names) == 6
    for n in names:
        assert kernels[n][2] <= 128, (n, kernels[n][2])
