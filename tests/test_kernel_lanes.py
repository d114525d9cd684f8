"""Kernels whose scalar registers do not suffice: copies of vector registers must not lie between the label that a skipped branch jumps to and the
instruction that brings the branch's lanes back, where lanes that skipped it would keep old values.  (hipcc of ROCm 7.2 has put them there, behind
scalar registers that it reads back in the same place.)  Read from the instructions of the library's own code objects."""

import re
import struct
import subprocess

import pytest

from lighthouse_amd import _lib

READELF = "/opt/rocm/llvm/bin/llvm-readelf"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"

COPY = re.compile(r"(v_mov_b32_e32 v\d+, v\d+|v_mov_b64_e32 v\[\d+:\d+\], v\[|v_accvgpr_(read|write)_b32 [av]\d+, [av]\d+)")
OTHER_LANES = ("s_cbranch", "s_branch", "s_endpgm", "s_and_saveexec", "s_andn2_saveexec", "s_xor_saveexec", "s_or_saveexec", "s_mov_b64 exec", "s_and_b64 exec", "s_andn2_b64 exec")


def misplaced(lines):
    """Copies between a label that s_cbranch_execz jumps to and the `s_or_b64 exec` behind it.  lines: (offset, instruction, offset that it jumps to)."""
    skipped_to = {to for _, text, to in lines if text.startswith("s_cbranch_execz")}
    found, since = [], None
    for offset, text, _ in lines:
        if offset in skipped_to:
            since = []
        if since is None:
            continue
        if text.startswith("s_or_b64 exec, exec"):
            found += since
            since = None
        elif text.startswith(OTHER_LANES):
            since = None
        elif COPY.match(text):
            since.append((hex(offset), text))
    return found


def test_the_search_finds_what_it_is_for():
    line = lambda at, text, to=None: (at, text, to)  # noqa: E731
    good = [line(0, "s_and_saveexec_b64 s[4:5], vcc"), line(4, "s_cbranch_execz 3", 16), line(8, "v_mov_b32_e32 v1, v2"), line(12, "s_nop 0"),
            line(16, "v_readlane_b32 s6, v9, 0"), line(20, "s_or_b64 exec, exec, s[4:5]"), line(24, "v_mov_b32_e32 v3, v4")]
    assert misplaced(good) == []
    bad = good[:5] + [line(18, "v_mov_b32_e32 v3, v4")] + good[5:]
    assert misplaced(bad) == [("0x12", "v_mov_b32_e32 v3, v4")]
    assert misplaced([line(0, "s_cbranch_execnz 3", 16)] + bad[2:]) == []  # (lanes of the branch jump there themselves)


@pytest.fixture(scope="module")
def spilling(tmp_path_factory):
    """{mangled name: lines} of the kernels of attention that keep scalar registers in vector registers."""
    _lib.load()
    blob = _lib.library_path().read_bytes()
    folder = tmp_path_factory.mktemp("code")
    found, at = {}, blob.find(MAGIC)
    while at >= 0:
        pos = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", blob, pos - 8)[0]):
            offset, size, length = struct.unpack_from("<QQQ", blob, pos)
            target, pos = blob[pos + 24:pos + 24 + length], pos + 24 + length
            if not size or b"gfx950" not in target:
                continue
            obj = folder / f"object{at + offset}"
            obj.write_bytes(blob[at + offset:at + offset + size])
            notes = subprocess.run([READELF, "--notes", str(obj)], capture_output=True, text=True, check=True).stdout
            names = [re.search(r"\.name: +(\S+)", k).group(1) for k in re.split(r"\n +- \.agpr_count", notes)[1:]
                     if int(re.search(r"\.sgpr_spill_count: +(\d+)", k).group(1)) > 0]
            for name in (n for n in names if re.search(r"(paged|chunk)_attention_kernel", n)):
                text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f"--disassemble-symbols={name}", str(obj)], capture_output=True, text=True, check=True).stdout
                lines = []
                for line in text.splitlines():
                    m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(?:[^<]*<[^>]*\+0x([0-9a-f]+)>)?", line)
                    if m:
                        lines.append((int(m.group(2), 16), m.group(1), m.group(3)))
                first = lines[0][0]
                found[name] = [(o - first, t, None if to is None else int(to, 16)) for o, t, to in lines]
        at = blob.find(MAGIC, at + 1)
    return found


def test_no_copies_for_lanes_that_are_not_back_yet(spilling):
    assert spilling and all(any(t.startswith("s_or_b64 exec") for _, t, _ in lines) for lines in spilling.values())
    assert any(to is not None for lines in spilling.values() for _, _, to in lines)
    assert {name: found for name, found in ((n, misplaced(lines)) for n, lines in spilling.items()) if found} == {}
