"""CPU check of the machine code that the build left: the distances between instructions that the hardware does not keep by
itself, over every path of every kernel.

    results   an instruction that reads or overwrites a matrix product's result stands far enough behind the product: the
              compiler keeps that distance in a straight line, and may miss it where ways fork and join again
    copies    a copy from memory into LDS is inline assembly, no memory instruction to the compiler: an address in scalar
              registers that a vector instruction wrote may be read 5 wait states later at the earliest, M0 one

Needs the library that the build makes and the disassembler beside the compiler; skipped without either.
"""
import os
import re
import struct
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-thresholded-attention_amd")
LIB = os.path.join(PKG, "libsta_hip.so")
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")

# wait states of a product before its result is there: what the compiler keeps for this target between a product and the
# next instruction in a straight line
RESULT = {"v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_32x32x16_f16": 12, "v_mfma_f32_16x16x32_bf16": 8,
          "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_32x32x2_f32": 18,
          "v_mfma_scale_f32_32x32x64_f8f6f4": 20}


def _device_objects():
    """The device code of every source, as the bundles in the library hold it."""
    data = open(LIB, "rb").read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    for m in re.finditer(magic, data):
        at = m.start() + len(magic)
        n, = struct.unpack_from("<Q", data, at)
        at += 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + length].decode()
            at += 24 + length
            if "gfx950" in name and size:
                yield data[m.start() + offset:m.start() + offset + size]


def _kernels(tmp_path):
    """(name, instructions): an instruction is (text, index of its branch's target or None)."""
    path = str(tmp_path / "device.o")
    for code in _device_objects():
        with open(path, "wb") as f:
            f.write(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
        for name, body in re.findall(r"^[0-9a-f]+ <(\w+)>:\n(.*?)(?=^\S|\Z)", text, re.S | re.M):
            lines = re.findall(r"^\t(.*?)\s*// ([0-9A-F]+):.*?(?:<\w+\+0x([0-9a-f]+)>|<\w+>)?$", body, re.M)
            if not lines:
                continue
            first = int(lines[0][1], 16)
            index = {int(at, 16) - first: i for i, (_, at, _) in enumerate(lines)}
            yield name, [(op.strip(), index[int(to or "0", 16)] if op.startswith(("s_branch", "s_cbranch")) else None)
                         for op, _, to in lines]


def _registers(operand):
    operand = operand.strip().strip("-|")
    m = re.match(r"^([avs])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"^([avs])(\d+)\b", operand)
    return {(m.group(1), int(m.group(2)))} if m else set()


def _operands(text):
    return [x.split()[0] for x in text.split(None, 1)[1].split(",") if x.split()] if " " in text else []


def _behind(code, start, states, stop):
    """Instructions on any path behind `start`, fewer than `states` wait states away, with their distance; a path ends where
    stop(text) says so."""
    nearest, todo, seen = {}, [(start + 1, 0)], []
    while todo:
        i, waits = todo.pop()
        while i < len(code) and waits < states and nearest.get(i, states) > waits:
            nearest[i] = waits
            text, target = code[i]
            seen.append((waits, text))
            if stop(text):
                break
            waits += int(text.split()[1], 0) + 1 if text.startswith("s_nop") else 1
            if target is not None:
                todo.append((target, waits))
            if text.startswith(("s_branch", "s_endpgm", "s_setpc")):
                break
            i += 1
    return seen


def _early_results(code):
    for at, (text, _) in enumerate(code):
        if not text.startswith(("v_mfma", "v_smfma")):
            continue
        op = text.split()[0]
        out = _registers(_operands(text)[0])

        def touches(other):
            if not other.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                return False
            operands = _operands(other)
            # a product that adds to this one's result is given it in time
            return any(_registers(x) & out for x in (operands[1:3] if other.startswith("v_mfma") else operands))

        def ends(other):
            return touches(other) or other.startswith("v_mfma") and bool(_registers(_operands(other)[0]) & out)
        for waits, other in _behind(code, at, RESULT[op], ends):
            if touches(other):
                yield f"{other} {waits} wait states behind {text}, which needs {RESULT[op]}"


def _early_addresses(code):
    for at, (text, _) in enumerate(code):
        vector = text.startswith(("v_readfirstlane", "v_readlane", "v_cmp"))
        m0 = re.match(r"s_\w+ m0,", text) is not None
        if not vector and not m0:
            continue
        out = set() if m0 else _registers(_operands(text)[0])
        copy = re.compile(r"(global|buffer)_load_(lds_)?\w*.*\blds\b|global_load_lds")
        for waits, other in _behind(code, at, 1 if m0 else 5, lambda _: False):
            if copy.match(other) and (m0 or any(_registers(x) & out for x in _operands(other))):
                yield f"{other} {waits} wait states behind {text}"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no disassembler")
    return list(_kernels(tmp_path_factory.mktemp("device")))


def test_the_search_finds_what_it_looks_for():
    product = "v_mfma_f32_32x32x16_bf16 v[2:17], a[0:3], v[20:23], v[2:17]"
    read, other = "v_add_f32_e32 v1, v2, v3", "v_add_f32_e32 v1, v30, v31"
    #        product, a fork over 12 wait states to a join, and the reader behind it
    code = [(product, None), ("s_cbranch_scc1 2", 3), ("s_nop 11", None), ("s_nop 7", None), (read, None), ("s_endpgm", None)]
    assert len(list(_early_results(code))) == 1
    assert not list(_early_results(code[:3] + [("s_nop 10", None)] + code[4:]))
    assert not list(_early_results([(product, None), (product, None), ("s_nop 11", None), (read, None)]))
    assert not list(_early_results([(product, None), (other, None), ("s_endpgm", None), (read, None)]))
    copy = "global_load_lds_dwordx4 v4, s[6:7]"
    for first, near, far in (("v_readfirstlane_b32 s7, v1", "s_nop 3", "s_nop 4"), ("s_mov_b32 m0, s3", None, "s_nop 0")):
        assert len(list(_early_addresses([(first, None)] + ([(near, None)] if near else []) + [(copy, None)]))) == 1
        assert not list(_early_addresses([(first, None), (far, None), (copy, None)]))


def test_no_result_of_a_matrix_product_is_touched_too_early(kernels):
    assert sum("v_mfma" in text for _, code in kernels for text, _ in code) > 10000
    early = [f"{name}: {x}" for name, code in kernels for x in _early_results(code)]
    assert not early, f"{len(early)} in all, the first {early[:4]}"


def test_no_copy_into_lds_reads_its_scalar_operands_too_early(kernels):
    assert sum("_lds_" in text for _, code in kernels for text, _ in code) > 1000
    early = [f"{name}: {x}" for name, code in kernels for x in _early_addresses(code)]
    assert not early, f"{len(early)} in all, the first {early[:4]}"


def test_copies_into_lds_wait_for_their_scalar_operands_themselves():
    """Whatever is built around them: a copy with a scalar base waits 5 states, any other one for M0."""
    found = 0
    for name in sorted(os.listdir(os.path.join(PKG, "csrc"))):
        text = open(os.path.join(PKG, "csrc", name)).read()
        for wait, operands in re.findall(r'asm volatile\("(?:s_nop (\d+)\\n\\t)?global_load_lds_\w+ [^"]*"\s*:[^:]*:([^;]*);', text):
            found += 1
            assert wait and int(wait) >= (4 if '"s"(' in operands else 0), (name, operands)
        assert text.count("global_load_lds_dword") - len(re.findall(r"//.*global_load_lds_dword|\(global_load_lds_dword", text)) \
            == len(re.findall(r'asm volatile\("s_nop \d\\n\\tglobal_load_lds_dword', text)), name
    assert found >= 5
