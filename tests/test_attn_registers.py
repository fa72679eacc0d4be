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


def reloads_among_products(tmp_path, kernel):
    """name: scratch loads between a kernel's first and last matrix instruction.  They
    wait for the copies to LDS that are on their way, and the products wait for them."""
    from inferflux_amd import _lib
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([LLVM + "llvm-objdump", "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    out = {}
    for f in sorted(os.listdir(tmp_path)):
        if not f.endswith("gfx950") or kernel.encode() not in (tmp_path / f).read_bytes():
            continue
        text = subprocess.run([LLVM + "llvm-objdump", "-d", "--no-show-raw-insn", f], cwd=tmp_path, check=True,
                              capture_output=True, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <(?=_Z)", text, flags=re.M)[1:]:
            name, body = part.split(">:", 1)
            if kernel in name:
                ops = re.findall(r"^\s+(v_mfma|scratch_load)", body, re.M)
                last = len(ops) - 1 - ops[::-1].index("v_mfma")
                out[name] = ops[ops.index("v_mfma"):last].count("scratch_load")
    return out


def test_chunks_and_prompts_of_heads_of_256(tmp_path):
    """Their 512 registers do not hold all of Q, accumulators and fragments.  With 28
    (chunks) and 66 (prompts) such loads in fp16 they were up to 12 % slower than with
    26 and 54."""
    found = {k: n for k, n in reloads_among_products(tmp_path, "11k_attn_tileI").items() if "ELi256E" in k}
    assert len(found) == 6
    for name, n in found.items():
        assert n <= (54 if "ELb0ELb0E" in name else 26), (name, n)
