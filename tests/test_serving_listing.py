"""not-gpu: what the built library's own machine code of the sampling kernel has to show, read from its listing (llvm-objdump of the gfx950 code
objects in libdsrg_hip.so)."""
import os
import re
import struct
import subprocess

from dsrg_amd import _lib

OBJDUMP = os.path.join(os.environ.get('ROCM_PATH', '/opt/rocm'), 'llvm', 'bin', 'llvm-objdump')


def _code_objects():
    """the gfx950 code objects of the library: one offload bundle a source (magic, count, then offset, size and a counted name an entry)"""
    data, magic = open(_lib.LIB_PATH, 'rb').read(), b'__CLANG_OFFLOAD_BUNDLE__'
    for at in (m.start() for m in re.finditer(magic, data)):
        pos = at + len(magic) + 8
        for _ in range(struct.unpack_from('<Q', data, at + len(magic))[0]):
            off, size, named = struct.unpack_from('<QQQ', data, pos)
            name = data[pos + 24:pos + 24 + named]
            pos += 24 + named
            if b'gfx950' in name:
                yield data[at + off:at + off + size]


def _listing(kernel, tmp_path):
    (obj,) = [o for o in _code_objects() if kernel.encode() in o]
    path = tmp_path / 'code.o'
    path.write_bytes(obj)
    return subprocess.run([OBJDUMP, '-d', '--no-show-raw-insn', str(path)], check=True, capture_output=True, text=True).stdout


def test_sample_rows_loads_have_their_whole_offset_checked(tmp_path):
    """A buffer load's scalar offset is not (or not for certain, when it passes the row's size by itself) part of what the hardware checks against
    the row: it has to be 0 in every load, with the position in the lane's offset and the constant, so that nothing past the row is read."""
    loads = re.findall(r'\bbuffer_load_\w+ .*', _listing('sample_rows_kernel', tmp_path))
    assert len(loads) >= 100                              # (eight instantiations that hold their row in registers, two that walk it)
    for line in loads:
        m = re.match(r'buffer_load_(?:dword|ushort|short_d16(?:_hi)?) v\d+, v\d+, s\[\d+:\d+\], (\S+) offen', line)
        assert m and m.group(1) == '0', line
