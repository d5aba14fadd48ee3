"""The compiled cross-attention kernels are those that a call can ask for: the rule of the launch (waves per block and ranges by type, width and lengths), walked over
its whole range of sizes, against the kernels in the library."""
import re
import shutil
import subprocess

import pytest

COMPUTE_UNITS = 256


def waves(kind, bf16, hd, rows, other):
    if rows <= 32:
        return 1
    if not bf16:
        return 4
    if hd <= 64:
        return 1 if rows <= 128 or other <= 256 else 4
    if kind == "dkv" and hd > 96 and other <= 128:
        return 2
    if rows > 128:
        return 8
    return 1 if kind == "dq" else 4


def in_ranges(kind, bf16, hd, rows, other, pairs):
    rw = waves(kind, bf16, hd, rows, other)
    three = kind == "fwd" and bf16 and hd <= 64 and rw == 4 and other >= 2048
    step = 1024 if three else 128 if kind == "fwd" else 256
    blocks, want = -(-rows // (32 * rw)) * pairs, COMPUTE_UNITS * ((12 if three else 8) // rw)
    return min(1 if blocks >= want else want // blocks, -(-other // step), 64) > 1


def asked_for():
    out = set()
    sizes = [1, 31, 32, 33, 64, 65, 96, 127, 128, 129, 160, 255, 256, 257, 300, 512, 513, 1024, 1500, 2047, 2048, 2049, 4096, 10000]
    for bf16 in (False, True):
        for hd in range(8, 129, 8):
            width, tile = -(-hd // 32) * 32, "unsigned short" if bf16 else "float"
            for kind in ("fwd", "dq", "dkv"):
                for rows in sizes:
                    for other in sizes:
                        rw = waves(kind, bf16, hd, rows, other)
                        bn = 32 if rw == 1 or not bf16 else 64
                        for pairs in (1, 100000):
                            split = in_ranges(kind, bf16, hd, rows, other, pairs)
                            if kind == "fwd":
                                out.add("xattn_fwd_kernel<%s, %d, %d, %d, %s>" % (tile, width, rw, bn, str(split).lower()))
                            elif kind == "dkv":
                                out.add("xattn_dkv_kernel<%s, %d, %d, %s>" % (tile, width, rw, str(split).lower()))
                            else:
                                for part in ((1, 2) if bf16 else (1,)) if split else (0,):
                                    out.add("xattn_dq_kernel<%s, %d, %d, %d, (Part)%d>" % (tile, width, rw, bn, part))
    return out


def test_every_compiled_block_shape_is_asked_for_and_every_shape_asked_for_is_compiled():
    from declip_amd import lib as L
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("no nm")
    L.load()
    names = subprocess.run([nm, "-C", L.LIB_PATH], capture_output=True, text=True, check=True).stdout.replace("(anonymous namespace)::", "")
    built = set(re.findall(r"__device_stub__(xattn_(?:fwd|dq|dkv)_kernel<[^>]*>)", names))
    assert built, "the library's local symbols are gone"
    assert built == asked_for(), (sorted(built - asked_for()), sorted(asked_for() - built))
