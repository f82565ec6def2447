"""What the library's own gfx950 code must not hold, read from the built library: no GPU needed."""
import os
import re
import struct
import subprocess

import pytest

from mference_amd import _capi

TOOLS = "/opt/rocm/llvm/bin/"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(tmp_path):
    """the gfx950 code objects in the library's fat binaries, one a source file"""
    _capi.lib()
    sections = subprocess.run([TOOLS + "llvm-readelf", "-S", "--wide", _capi.LIB_PATH], capture_output=True, text=True, check=True).stdout
    _, at, size = (int(v, 16) for v in re.search(r"\.hip_fatbin\s+PROGBITS\s+(\w+)\s+(\w+)\s+(\w+)", sections).groups())
    with open(_capi.LIB_PATH, "rb") as fh:
        fh.seek(at)
        data = fh.read(size)
    paths = []
    for start in (m.start() for m in re.finditer(MAGIC, data)):
        place = start + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", data, place - 8)[0]):
            off, length, name = struct.unpack_from("<QQQ", data, place)
            if b"gfx950" in data[place + 24:place + 24 + name] and length:
                paths.append(tmp_path / f"{len(paths)}.elf")
                paths[-1].write_bytes(data[start + off:start + off + length])
            place += 24 + name
    return paths


@pytest.mark.skipif(not os.path.exists(TOOLS + "llvm-objdump"), reason="no disassembler")
def test_no_64_bit_shift_by_a_vector_register(tmp_path):
    """Masks of lanes are made without a 64-bit shift by a lane's own amount: where the amount lay in the last register of a wave, single waves
    got a wrong mask, and where the compiler puts it changes with every edit."""
    objects = code_objects(tmp_path)
    assert len(objects) > 10
    found = []
    for path in objects:
        listing = subprocess.Popen([TOOLS + "llvm-objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], stdout=subprocess.PIPE, text=True)
        kernel = ""
        for line in listing.stdout:
            if line.startswith("<"):
                kernel = line.strip()
            elif "64 v[" in line and re.match(r"\s*v_(lshlrev_b64|lshrrev_b64|ashrrev_i64)(_e64)?\s+v\[\d+:\d+\], v\d+,", line):
                found.append(f"{kernel} {line.split('//')[0].strip()}")
        assert listing.wait() == 0
    assert not found, found


@pytest.mark.skipif(not os.path.exists(TOOLS + "llvm-readelf"), reason="no reader of code objects")
def test_row_grouping_has_the_instances_that_are_launched(tmp_path):
    """rows a lane takes in turn: 1, 4 or 16 (AdapterPlan::turns_of), counting runs or placing rows"""
    names = set()
    for path in code_objects(tmp_path):
        symbols = subprocess.run([TOOLS + "llvm-readelf", "--symbols", "--wide", str(path)], capture_output=True, text=True, check=True).stdout
        names |= set(re.findall(r"adapter_group_kernelILi(\d+)ELb(\d)E\w+(?!\w|\.kd)", symbols))
    # a batch of one run (up to 4096 rows) has 1 or 4 turns and is not counted; longer ones have 1, 4 or 16 and are
    assert names == {(turns, count) for turns in ("1", "4", "16") for count in ("0", "1")}
