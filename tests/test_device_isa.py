"""What the gfx950 code of the built libraries may not contain, read from its disassembly (CPU only: the compiler's own choices count
as much as what the sources spell out)."""
import os
import shutil
import struct
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def device_objects(blob):
    """The gfx950 code objects inside a shared library: clang's offload bundles, one per translation unit."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    out, at = [], blob.find(magic)
    while at >= 0:
        n, = struct.unpack_from("<Q", blob, at + len(magic))
        p = at + len(magic) + 8
        for _ in range(n):
            off, size, idlen = struct.unpack_from("<QQQ", blob, p)
            triple = blob[p + 24:p + 24 + idlen].decode()
            p += 24 + idlen
            if size and triple.endswith("gfx950"):
                out.append(blob[at + off:at + off + size])
        at = blob.find(magic, at + len(magic))
    return out


@pytest.fixture(scope="module", params=["libbgt_hip.so", "libbgt_hip_bench.so"])
def mnemonics(request, tmp_path_factory):
    """The set of instruction names in the device code of one library."""
    import bgt_amd
    lib = os.path.join(os.path.dirname(bgt_amd.library_path()), request.param)
    if not os.path.exists(lib):
        bgt_amd.build_library()
    tool = OBJDUMP if os.path.exists(OBJDUMP) else shutil.which("llvm-objdump")
    assert tool, "llvm-objdump is part of ROCm's compiler"
    objs = device_objects(open(lib, "rb").read())
    assert objs, "no gfx950 code object in " + request.param
    tmp = tmp_path_factory.mktemp("isa")
    files = []
    for i, o in enumerate(objs):
        files.append(str(tmp / ("%d.co" % i)))
        with open(files[-1], "wb") as f:
            f.write(o)
    names = set()
    with subprocess.Popen([tool, "-d", "--mcpu=gfx950", "--no-show-raw-insn", "--no-leading-addr"] + files, stdout=subprocess.PIPE, text=True) as p:
        for line in p.stdout:
            if line[:1] in (" ", "\t"):                       # (labels and file headers start in the first column)
                names.add(line.split(None, 1)[0])
    assert p.returncode == 0
    for f in files:
        os.remove(f)
    assert "s_endpgm" in names and any(n.startswith("global_store") for n in names), "not a disassembly"
    return names


def test_no_write_through_the_scalar_data_cache(mnemonics):
    """Scalar memory instructions only read: what a kernel writes leaves through vector stores and vector atomics."""
    scalar = {n for n in mnemonics if n.startswith("s_")}
    bad = sorted(n for n in scalar if "store" in n or "atomic" in n or ("cache" in n and not n.endswith(("_inv", "_inv_vol"))))
    assert not bad, bad


def test_no_packed_fp32_arithmetic(mnemonics):
    """The device code is built without the packed-FP32 feature (bgt_amd/csrc/Makefile): neither written by hand, which the assembler
    then refuses, nor made by the compiler out of ordinary float code."""
    bad = sorted(n for n in mnemonics if n.startswith("v_pk_") and n.split("_e")[0].endswith("_f32"))
    assert not bad, bad
