"""What the built kernels must not contain, read from their own code: a 64-bit
shift whose amount is in the last register of the wave's allocation.  Such a
shift gave wrong bits now and then (with 120 registers and the amount in v119,
tails of rows came out with bits of other values in them)."""
import concurrent.futures as cf
import re
import struct
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LLVM = Path("/opt/rocm/llvm/bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
GRANULE = 8  # registers are allocated eight at a time


def code_objects(data):
    """The gfx950 code objects in a library's bytes."""
    at = data.find(MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            triple = data[entry + 24 : entry + 24 + length]
            entry += 24 + length
            if b"gfx950" in triple and size:
                yield data[at + offset : at + offset + size]
        at = data.find(MAGIC, at + 1)


def last_register_shifts(kernel_registers, assembly):
    """Shifts of a kernel with that many registers whose amount is in the last one."""
    last = -(-kernel_registers // GRANULE) * GRANULE - 1
    return [m.group(0) for m in re.finditer(r"v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* v\[\d+:\d+\], v(\d+),", assembly) if int(m.group(1)) == last]


def test_the_reader():
    text = "v_lshlrev_b64 v[4:5], v119, v[6:7]\nv_lshrrev_b64 v[4:5], v118, v[6:7]\nv_lshlrev_b64 v[4:5], 1, v[118:119]"
    assert len(last_register_shifts(120, text)) == len(last_register_shifts(113, text)) == 1
    assert not last_register_shifts(121, text) and not last_register_shifts(112, text)


def scan(path):
    notes = subprocess.run([LLVM / "llvm-readelf", "--notes", path], capture_output=True, text=True, check=True).stdout
    registers = {re.search(r"\.name:\s+(\S+)", k).group(1): int(re.search(r"\.vgpr_count:\s+(\d+)", k).group(1)) for k in notes.split("- .agpr_count")[1:]}
    text = subprocess.run([LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
    found, seen = [], 0
    for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
        head = re.match(r"[0-9a-f]{16} <(.*)>:", part)
        if head and head.group(1) in registers:
            seen += 1
            found += [(head.group(1), s) for s in last_register_shifts(registers[head.group(1)], part)]
    return seen, len(registers), found


def test_no_shift_by_the_last_register(lib, tmp_path):
    if not (LLVM / "llvm-objdump").exists():
        pytest.skip("no llvm-objdump")
    paths = []
    for i, code in enumerate(code_objects((ROOT / "nerf_amd" / "libnerf.so").read_bytes())):
        paths.append(tmp_path / f"{i}.co")
        paths[-1].write_bytes(code)
    assert paths
    with cf.ThreadPoolExecutor(4) as pool:
        results = list(pool.map(scan, paths))
    assert sum(seen for seen, _, _ in results) == sum(named for _, named, _ in results) > 0
    assert not [f for _, _, found in results for f in found]
