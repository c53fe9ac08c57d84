"""The prompt attention's copies into LDS take their address from M0, which an asm statement cannot declare as clobbered:
the compiler itself must have no use for it in these kernels (read from their assembly, no GPU)."""
import re
import subprocess

from mnemocuda_amd import build as mbuild


def test_compiler_leaves_m0_alone(tmp_path):
    out = tmp_path / "paged_prompt.s"
    subprocess.run([str(mbuild.ROCM / "bin" / "hipcc"), *mbuild.HIPCC_FLAGS, "-S", "--offload-device-only",
                    str(mbuild.CSRC / "paged_prompt.hip"), "-o", str(out)], check=True, capture_output=True)
    asm, own = False, 0
    for line in out.read_text().splitlines():
        asm = (asm or "ASMSTART" in line) and "ASMEND" not in line
        if re.search(r"\bm0\b", line.split(";")[0]):
            assert asm, line
            own += 1
    assert own
