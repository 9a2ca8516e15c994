"""Wait states between a matrix product and what reads its result, looked for in the library's own machine code along every jump.

A vector instruction or a store that reads a product's result has to stand behind it by the product's passes and three more (bf16 and fp16
operands) or two more (fp32): CDNA3 instruction set guide, "Manually Inserted Wait States".  The compiler puts them there, but where a branch
stands right behind a product and its two ways meet again in front of the reader, it has been seen to count them along the longer
way alone; which source makes it do that is not predictable, so what it made is looked at.  The rules of
test_wait_states.py are applied along jumps here as well."""
import os
import re
import subprocess

import pytest

import test_wait_states as W

_JUMP = re.compile(r"<([^>+]+)(?:\+0x([0-9a-f]+))?>\s*$")
_PASSES = {"32x32x16": 8, "16x16x32": 4, "32x32x8": 8, "16x16x16": 4, "32x32x2": 16, "16x16x4": 8}


def wanted(op):
    passes = _PASSES[re.search(r"_(\d+x\d+x\d+)_?", op).group(1)]
    return passes + (2 if op.endswith("_f32") else 3)


def read(op, operands):
    """Vector registers that an instruction reads; none for a product's own addend, which may follow at once."""
    if op.startswith("v_mfma"):
        return set()
    writes_first = op.startswith("v_") or "_load" in op or op.startswith(("ds_read", "ds_bpermute"))
    return {r for o in operands[1 if writes_first else 0:] for r in W.registers(o) if r[0] in "va"}


def too_near(listing):
    code, labels = W.parse(listing)
    at_address = {c[0]: i for i, c in enumerate(code)}
    bad, products = [], 0
    for i, (address, op, operands, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        products += 1
        result, states = W.registers(operands[0]), wanted(op)
        todo, nearest = [(i + 1, 0)], {}
        while todo:
            j, waited = todo.pop()
            if j >= len(code) or waited >= states or nearest.get(j, states) <= waited:
                continue
            nearest[j] = waited
            _, name, args, target = code[j]
            if name.startswith("v_mfma") and W.registers(args[0]) & result:
                continue  # (from here on its own result counts)
            if read(name, args) & result:
                bad.append((address, op, waited, states, name, args))
                continue
            if name in ("s_endpgm", "s_setpc_b64", "s_swappc_b64"):
                continue
            waited += int(args[0]) + 1 if name == "s_nop" else 1
            if target and target[0] in labels:
                goal = at_address.get(code[labels[target[0]]][0] + target[1])
                if goal is not None:
                    todo.append((goal, waited))
                if name == "s_branch":
                    continue
            todo.append((j + 1, waited))
    return products, bad


@pytest.fixture
def jumps(monkeypatch):
    monkeypatch.setattr(W, "_TARGET", _JUMP)


def test_the_rule_is_seen(jumps):
    def listing(*lines):
        rows = [(*line.split(" -> "), "")[:2] for line in lines]
        return "<k>:\n" + "".join(f"\t{text} // {4 * i:012X}: 00000000 {goal}\n" for i, (text, goal) in enumerate(rows))

    product, reader = "v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], 0", "v_accvgpr_read_b32 v9, a3"
    assert too_near(listing(product, "s_nop 9", reader))[1]
    assert not too_near(listing(product, "s_nop 10", reader))[1]
    assert not too_near(listing(product, "v_accvgpr_read_b32 v9, a16"))[1]
    assert not too_near(listing(product, "s_branch 1 -> <k+0xc>", reader, "s_endpgm"))[1]
    # a way round the wait states
    ways = [product, "s_cbranch_vccnz 1 -> <k+0xc>", "s_nop 12", reader, "s_endpgm"]
    assert too_near(listing(*ways))[1]
    assert not too_near(listing(ways[0], "s_nop 10", *ways[1:]))[1]
    assert too_near(listing(product, "v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]", "s_nop 4", "buffer_store_dword a5, v1, s[0:3], 0 offen"))[1]
    assert not too_near(listing("v_mfma_f32_16x16x4_f32 v[0:3], v4, v5, v[0:3]", "s_nop 9", "v_add_f32_e32 v6, v0, v1"))[1]


@pytest.mark.skipif(not os.path.exists(W.OBJDUMP), reason="no disassembler")
def test_products_of_the_library(tmp_path, jumps):
    assert os.path.exists(W.LIB), "not built"
    products = 0
    for i, content in enumerate(W.code_objects(W.LIB)):
        path = tmp_path / f"{i}.co"
        path.write_bytes(content)
        listing = subprocess.run([W.OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True, capture_output=True,
                                 text=True).stdout
        n, bad = too_near(listing)
        products += n
        assert not bad, f"{len(bad)} places, the first ones: " + "; ".join(f"{op} at {a:#x}, {w} of {s} states, {r}" for a, op, w, s, *r in bad[:8])
        _, bad = W.violations(listing)
        assert not bad, f"{len(bad)} places, the first ones: " + "; ".join(f"{w} at {a:#x}: {op} then {b}" for w, a, op, b in bad[:8])
    assert products > 1000
