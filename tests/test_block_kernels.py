"""The decoder block's kernels as they are built, from the library's own code objects: the waits of the tiles' products."""
import os
import re
import shutil
import struct
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"
TOOLS = {t: os.path.join(LLVM, "llvm-" + t) for t in ("readelf", "objcopy", "objdump")}
PRODUCTS = r"product_kernel|gate_kernel|gate_backward_kernel"


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """The gfx950 code objects that hold kernels of the gated feed-forward block: [(path, symbols)]."""
    from nest_splat import _lib
    if not all(os.path.exists(t) for t in TOOLS.values()):
        pytest.skip("the ROCm LLVM tools are not installed")
    d = tmp_path_factory.mktemp("co")
    so = shutil.copy(os.path.join(os.path.dirname(_lib.__file__), "libnest_splat.so"), d)
    subprocess.run([TOOLS["objcopy"], f"--dump-section=.hip_fatbin={d / 'fat'}", so, str(d / "out.so")], check=True, capture_output=True)
    blob, found = (d / "fat").read_bytes(), []
    for m in re.finditer(rb"__CLANG_OFFLOAD_BUNDLE__", blob):
        at = m.end()
        (n,), at = struct.unpack_from("<Q", blob, at), at + 8
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", blob, at)
            ident, at = blob[at + 24:at + 24 + length], at + 24 + length
            if size == 0 or b"gfx950" not in ident:
                continue
            path = d / f"{len(found)}.elf"
            path.write_bytes(blob[m.start() + off:m.start() + off + size])
            names = subprocess.run([TOOLS["readelf"], "--symbols", "--wide", str(path)], check=True, capture_output=True, text=True).stdout
            found.append((path, sorted(set(re.findall(r"FUNC .* (_Z\S+)", names)))))
    assert found
    return found


def instructions(path, symbols):
    """{symbol: [instruction]}."""
    out = subprocess.run([TOOLS["objdump"], "-d", "--no-show-raw-insn", "--no-leading-addr", f"--disassemble-symbols={','.join(symbols)}",
                          str(path)], check=True, capture_output=True, text=True).stdout
    found = {}
    for line in out.splitlines():
        m = re.match(r"^(?:[0-9a-f]+ )?<(\S+)>:", line)
        if m:
            found[m.group(1)] = code = []
        elif re.match(r"^\s+[a-z]", line):
            code.append(line.split("//")[0].strip())
    return found


def test_waits_of_the_products(objects):
    """Between a tile's first product and its last each barrier comes after a wait that counts direct loads, with no access
    to memory between, and no other wait is for all of them: the loads of the steps ahead stay in flight over a step."""
    memory = ("buffer_", "global_", "flat_", "scratch_", "ds_")
    seen = 0
    for path, symbols in objects:
        names = [s for s in symbols if re.search(PRODUCTS, s)]
        if not names:
            continue
        for name, code in instructions(path, names).items():
            products = [i for i, c in enumerate(code) if c.startswith("v_mfma")]
            assert products, name
            loop = code[products[0]:products[-1] + 1]
            assert any("buffer_load" in c and c.endswith("lds") for c in loop), name
            waited = held = None   # a wait with nothing loaded since; one for all, before its barrier
            for i, c in enumerate(loop):
                if c.startswith("s_waitcnt") and "vmcnt" in c:
                    waited = i
                    held = i if "vmcnt(0)" in c else held
                elif c.startswith("s_barrier"):
                    assert waited is not None, (name, loop[max(i - 3, 0):i + 1])
                    held = None
                elif c.startswith(memory):
                    assert held is None, (name, loop[held:held + 4])
                    waited = None
            seen += 1
    assert seen >= 3 * 4 * 5   # types, tiles, products


def test_no_kernel_spills(objects):
    """Registers hold all that the kernels of these files keep: none has scratch memory."""
    seen = 0
    for path, symbols in objects:
        if not any(re.search(PRODUCTS + r"|layer_norm|dropout_kernel|narrow_|few_kernel", s) for s in symbols):
            continue
        notes = subprocess.run([TOOLS["readelf"], "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        for k in re.split(r"\n  - \.", notes)[1:]:
            name = re.search(r"\.name: +(_Z\w+)", k)
            if name:
                seen += 1
                spilled = [int(v) for v in re.findall(r"\.(?:private_segment_fixed_size|vgpr_spill_count): +(\d+)", k)]
                assert len(spilled) == 2 and not any(spilled), (name.group(1), spilled)
    assert seen > 100
