"""Vector registers that the built attention kernels take: how many waves a SIMD
holds (512 registers) hangs on them.  Decode over the 16-bit cache with heads of 64
is made for three."""
import os
import re
import shutil
import subprocess

LLVM = "/opt/rocm/llvm/bin/"


def kernels(tmp_path):
    """name: (vector registers, those spilled) of the library's kernels."""
    from inferflux_amd import _lib
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([LLVM + "llvm-objdump", "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    out = {}
    for f in sorted(os.listdir(tmp_path)):
        if f.endswith("gfx950"):
            notes = subprocess.run([LLVM + "llvm-readelf", "--notes", f], cwd=tmp_path, check=True, capture_output=True,
                                   text=True).stdout
            for k in notes.split("  - .agpr_count")[1:]:
                name = re.search(r"\.name:\s+(\S+)", k).group(1)
                out[name] = tuple(int(re.search(rf"\.{x}:\s+(\d+)", k).group(1)) for x in ("vgpr_count", "vgpr_spill_count"))
    return out


def test_waves_of_16_bit_decode(tmp_path):
    found = {k: v for k, v in kernels(tmp_path).items() if "11k_attn_rowsI" in k and "ELb0E" in k}
    assert len(found) == 8
    for name, (registers, spilled) in found.items():
        D = int(re.search(r"ELi(\d+)ELb0", name).group(1))
        assert registers <= {64: 168, 96: 256, 128: 256, 256: 512}[D], (name, registers)
        assert spilled == 0 or D == 256, (name, spilled)
