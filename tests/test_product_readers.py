"""Wait states between a matrix product and the readers that test_product_wait_states.py does not count: another product's operands and
addend, and instructions that add to their own destination.

In wait states behind a product of n passes (CDNA3 instruction set guide, "Manually Inserted Wait States"): n + 3 (bf16 and fp16 operands) or
n + 2 (fp32) for a vector instruction that reads one of the result's registers and for a product that has one among its first two operands;
n + 1 or n for a product whose addend shares registers with the result without being it.  The same registers as addend may follow at once."""
import os
import re
import subprocess

import pytest

import test_product_wait_states as P
import test_wait_states as W

_IN_PLACE = re.compile(r"v_(pk_)?(fmac|mac|dot\dc|madmk|smfmac)")


def wanted(op, result, name, args):
    """Wait states that instruction `name` has to stay behind product `op`; 0 where they have nothing to do with each other."""
    full = P.wanted(op)
    if name.startswith("v_mfma"):
        addend = W.registers(args[3]) if len(args) > 3 else set()
        if result & (W.registers(args[1]) | W.registers(args[2])):
            return full
        return full - 2 if addend & result and addend != result else 0
    if not name.startswith("v_"):
        return 0
    return full if result & {r for a in args[0 if _IN_PLACE.match(name) else 1:] for r in W.registers(a)} else 0


def too_near(listing):
    code, labels = W.parse(listing)
    at_address = {c[0]: i for i, c in enumerate(code)}
    bad, fed = [], 0
    for i, (address, op, operands, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result, most = W.registers(operands[0]), P.wanted(op)
        todo, nearest = [(i + 1, 0)], {}
        while todo:
            j, waited = todo.pop()
            if j >= len(code) or waited >= most or nearest.get(j, most) <= waited:
                continue
            nearest[j] = waited
            _, name, args, target = code[j]
            states = wanted(op, result, name, args)
            if waited < states:
                bad.append((address, op, waited, states, name, args))
                continue
            if name.startswith("v_mfma") and W.registers(args[0]) & result:
                fed += 1
                continue  # (from here on its own result counts)
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
    return fed, bad


def test_the_rule_is_seen():
    def bad(*lines):
        rows = [(*line.split(" -> "), "")[:2] for line in lines]
        return too_near("<k>:\n" + "".join(f"\t{text} // {4 * i:012X}: 00000000 {goal}\n" for i, (text, goal) in enumerate(rows)))[1]

    wide, small = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], 0", "v_mfma_f32_16x16x4_f32 v[0:3], v4, v5, v[0:3]"
    # another product's operands, first and second
    assert bad(wide, "s_nop 9", "v_mfma_f32_32x32x16_bf16 v[40:55], v[0:3], v[24:27], 0")
    assert bad(wide, "s_nop 9", "v_mfma_f32_32x32x16_bf16 v[40:55], v[20:23], v[12:15], 0")
    assert not bad(wide, "s_nop 10", "v_mfma_f32_32x32x16_bf16 v[40:55], v[0:3], v[24:27], 0")
    assert bad(small, "s_nop 8", "v_mfma_f32_16x16x4_f32 v[8:11], v2, v5, v[8:11]")
    assert not bad(small, "s_nop 9", "v_mfma_f32_16x16x4_f32 v[8:11], v2, v5, v[8:11]")
    # its addend: the result itself at once, others not
    assert not bad(small, "v_mfma_f32_16x16x4_f32 v[0:3], v6, v7, v[0:3]")
    assert not bad(small, "v_mfma_f32_16x16x4_f32 v[8:11], v6, v7, v[0:3]")
    assert bad(small, "s_nop 6", "v_mfma_f32_16x16x4_f32 v[8:11], v6, v7, v[2:5]")
    # instructions that add to their destination
    assert bad(wide, "s_nop 9", "v_fmac_f32_e32 v3, v30, v31") and bad(wide, "s_nop 9", "v_dot2c_f32_bf16 v3, v30, v31")
    assert not bad(wide, "s_nop 10", "v_fmac_f32_e32 v3, v30, v31") and not bad(wide, "v_fmac_f32_e32 v16, v30, v31")
    assert not bad(wide, "s_branch 1 -> <k+0xc>", "v_fmac_f32_e32 v3, v30, v31", "s_endpgm")


@pytest.mark.skipif(not os.path.exists(W.OBJDUMP), reason="no disassembler")
def test_products_of_the_library(tmp_path):
    assert os.path.exists(W.LIB), "not built"
    fed = 0
    for i, content in enumerate(W.code_objects(W.LIB)):
        path = tmp_path / f"{i}.co"
        path.write_bytes(content)
        listing = subprocess.run([W.OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True, capture_output=True,
                                 text=True).stdout
        n, bad = too_near(listing)
        fed += n
        assert not bad, f"{len(bad)} places, the first ones: " + "; ".join(f"{op} at {a:#x}, {w} of {s} states, {r}" for a, op, w, s, *r in bad[:8])
    assert fed > 1000  # (chains of products are seen at all)
