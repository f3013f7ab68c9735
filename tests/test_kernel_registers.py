"""Kernels whose registers are budgeted to the last one keep nothing in scratch memory: read from the metadata that the
compiler put beside each kernel in the built library."""
import re
import struct

import pytest

from channelestimationtransformer_amd import _cabi

msgpack = pytest.importorskip("msgpack")


def code_objects(blob):
    """The gfx950 code objects in the library's offload bundles."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = blob.find(magic)
    while at >= 0:
        n, p = struct.unpack_from("<Q", blob, at + len(magic))[0], at + len(magic) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", blob, p)
            if b"gfx950" in blob[p + 24:p + 24 + length] and size:
                yield blob[at + offset:at + offset + size]
            p += 24 + length
        at = blob.find(magic, at + 1)


def kernels(elf):
    """{name: metadata} from the note of one code object."""
    shoff, = struct.unpack_from("<Q", elf, 40)
    size, count = struct.unpack_from("<HH", elf, 58)
    out = {}
    for s in range(count):
        kind, = struct.unpack_from("<I", elf, shoff + s * size + 4)
        offset, length = struct.unpack_from("<QQ", elf, shoff + s * size + 24)
        at = offset
        while kind == 7 and at < offset + length:  # notes
            name, desc, note = struct.unpack_from("<III", elf, at)
            at += 12 + -(-name // 4) * 4
            if note == 32:
                for k in msgpack.unpackb(elf[at:at + desc], strict_map_key=False)["amdhsa.kernels"]:
                    out[k[".name"]] = k
            at += -(-desc // 4) * 4
    return out


@pytest.fixture(scope="module")
def metadata():
    with open(_cabi.LIB_PATH, "rb") as f:
        blob = f.read()
    out = {}
    for elf in code_objects(blob):
        out.update(kernels(elf))
    return out


@pytest.mark.parametrize("pattern, least", [("rnn_mid_kernel", 30), ("2la6chunks", 100), ("5gated7product", 54), ("narrow_(for|back)ward", 24),
                                            ("rotary_kernel", 20), ("8few_rows", 9)])
def test_nothing_in_scratch_memory(metadata, pattern, least):
    found = {n: k for n, k in metadata.items() if re.search(pattern, n)}
    assert len(found) >= least
    spilled = {n: k[".private_segment_fixed_size"] for n, k in found.items() if k[".private_segment_fixed_size"]}
    assert not spilled
