"""What the kernels over 16-bit pages must not pay for the 4-bit ones, read off the
registers that the compiler gives them."""
import re
import subprocess

import pytest

from prismkv_amd import build


def registers(source, tmp_path):
    """Kernel -> (vector registers, scalar registers spilled)."""
    hipcc = build._hipcc("/opt/rocm")
    try:
        subprocess.run([hipcc, "--version"], capture_output=True, check=True)
    except OSError:
        pytest.skip("no hipcc")
    out = tmp_path / "source.s"
    subprocess.run([hipcc, *build.HIP_FLAGS, f"-I{build.CSRC}", f"-I{build.INCLUDE}", "--cuda-device-only", "-S",
                    str(build.CSRC / source), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    found = {}
    for entry in text[text.index("amdhsa.kernels:"):].split("\n  - ")[1:]:
        value = {key: re.search(rf"\.{key}: +(\S+)", entry) for key in ("name", "vgpr_count", "sgpr_spill_count")}
        if all(value.values()):
            found[value["name"][1]] = int(value["vgpr_count"][1]), int(value["sgpr_spill_count"][1])
    return found


def test_cuts_of_16_bit_pages_move_no_scales(tmp_path):
    found = registers("paged.hip", tmp_path)
    for name in ("paged_select_kernel", "paged_move_kernel"):
        (plain,) = [x for key, x in found.items() if name in key and "ILb0E" in key]
        (four,) = [x for key, x in found.items() if name in key and "ILb1E" in key]
        assert plain[0] < four[0], name
        assert plain[1] == 0, name
