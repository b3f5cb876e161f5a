"""The built library's matrix instructions, read from its own code: none reads a register within two wait
states of the vector instruction that writes it. The compiler sees to that for its builtins; products
written as asm have to keep it themselves."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from collections import defaultdict
from pathlib import Path

import pytest

WAIT_STATES = 2
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
REGISTERS = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
INSTRUCTION = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):(.*)$")
TARGET = re.compile(r"<[^>]*?(?:\+0x([0-9a-f]+))?>")


def _code_objects(data):
    at = data.find(MAGIC)
    while at >= 0:
        p = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(MAGIC))[0]):
            offset, size, chars = struct.unpack_from("<QQQ", data, p)
            triple = data[p + 24 : p + 24 + chars]
            p += 24 + chars
            if b"gfx950" in triple and size:
                yield data[at + offset : at + offset + size]
        at = data.find(MAGIC, at + 1)


def _functions(listing):
    """{name: [(operation, operands, address, branch target)]} of a disassembly."""
    out, body = {}, None
    for line in listing.splitlines():
        head = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if head:
            body = out.setdefault(head[1], [])
            continue
        m = INSTRUCTION.match(line)
        if m and body is not None:
            body.append((m[1], m[2], int(m[3], 16), m[4]))
    return {name: body for name, body in out.items() if body}


def _registers(operands):
    regs = set()
    for m in REGISTERS.finditer(operands):
        lo, hi = (int(m[2]),) * 2 if m[2] else (int(m[3]), int(m[4]))
        regs |= {(m[1], r) for r in range(lo, hi + 1)}
    return regs


def _before(body):
    """For each instruction the ones that may run right before it."""
    index = {addr: i for i, (_, _, addr, _) in enumerate(body)}
    before = defaultdict(list)
    for i, (op, _, _, rest) in enumerate(body):
        if op.startswith(("s_branch", "s_cbranch")):
            m = TARGET.search(rest)
            if m:
                before[index[body[0][2] + int(m[1] or "0", 16)]].append(i)
        if i + 1 < len(body) and op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[i + 1].append(i)
    return before


def _too_near(body):
    """(matrix instruction, writer) pairs with fewer wait states between them."""
    before, found = _before(body), []
    for i, (op, operands, _, _) in enumerate(body):
        if not op.startswith("v_mfma"):
            continue
        read = _registers(operands.split(",", 1)[1])
        work = [(j, 0) for j in before[i]]
        while work:
            j, states = work.pop()
            if states >= WAIT_STATES:
                continue
            name, args = body[j][:2]
            if name.startswith("v_") and not name.startswith("v_mfma"):
                written = _registers(args if "swap" in name else args.split(",", 1)[0])
                if written & read:
                    found.append((f"{op} {operands}", f"{name} {args}"))
            states += int(args, 0) + 1 if name == "s_nop" else 1
            work += [(k, states) for k in before[j]]
    return found


def test_the_search_finds_a_missing_wait():
    line = "\t{} // {:012X}: 00000000"
    def listing(*ops):
        return "0000000000001000 <f>:\n" + "\n".join(line.format(o, 0x1000 + 8 * i) for i, o in enumerate(ops))

    shift = "v_lshrrev_b32_e32 v105, v82, v108"
    mfma = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[18:25], v[34:41], a[0:3], v95, v105 op_sel_hi:[0,0,0]"
    for between, wrong in (((), 1), (("v_mov_b32_e32 v1, v2",), 1), (("s_nop 0",), 1), (("s_nop 1",), 0),
                           (("s_nop 0", "s_barrier"), 0)):
        assert len(_too_near(_functions(listing(shift, *between, mfma))["f"])) == wrong, between
    loop = listing(mfma, "v_mov_b32_e32 v20, 0", "s_cbranch_scc1 65533") + " <f>"  # back to the first
    assert len(_too_near(_functions(loop)["f"])) == 1


def test_matrix_instructions_wait_for_their_operands(pkg, tmp_path):
    lib = Path(pkg._lib.LIB_PATH)
    tool = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
    if not lib.exists() or not Path(tool).exists():
        pytest.skip("no built library or no llvm-objdump")
    products, wrong = 0, []
    for n, obj in enumerate(_code_objects(lib.read_bytes())):
        path = tmp_path / f"{n}.o"
        path.write_bytes(obj)
        listing = subprocess.run([tool, "-d", "--mcpu=gfx950", "-C", str(path)], capture_output=True, text=True,
                                 check=True).stdout
        for name, body in _functions(listing).items():
            products += sum(op.startswith("v_mfma") for op, *_ in body)
            wrong += [(name, *pair) for pair in _too_near(body)]
    assert products > 1000  # the listing was read
    assert not wrong, wrong[:5]
