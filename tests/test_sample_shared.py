"""What the sampling kernels read from shared memory, looked for in the library's own machine code.

Until a workgroup has met at a barrier, a word of shared memory that some wavefront writes may not be there for the others, and no run shows it: they
are mostly done by then.  So up to the first barrier, along every way through the code, nothing is read from shared memory."""
import os
import subprocess

import pytest

import test_wait_states as W

KERNELS = ("sample_row_kernel", "sample_scan_kernel", "sample_pick_kernel")


def far_jump(code, i):
    """Where `s_getpc, s_add_u32, s_addc_u32, s_setpc` goes; None for a jump of another kind."""
    if i < 3 or code[i - 3][1] != "s_getpc_b64" or code[i - 3][2] != code[i][2] or code[i - 2][1] != "s_add_u32":
        return None
    by = int(code[i - 2][2][2], 0) & 0xFFFFFFFF
    return code[i - 2][0] + by - (by >> 31 << 32)


def reads_before_barrier(code, labels, start):
    """(address, instruction) of what reads shared memory, or leaves for other code, on a way from `start` to the first barrier."""
    at_address = {c[0]: i for i, c in enumerate(code)}
    todo, seen, bad = [start], set(), []
    while todo:
        i = todo.pop()
        if i in seen or i >= len(code):
            continue
        seen.add(i)
        address, op, operands, target = code[i]
        if op == "s_barrier" or op == "s_endpgm":
            continue
        if op.startswith("ds_") and not op.startswith(("ds_write", "ds_bpermute", "ds_permute", "ds_swizzle")):
            if "_rtn" in op or op.startswith("ds_read"):
                bad.append((address, op, operands))
        if op in ("s_setpc_b64", "s_swappc_b64"):
            goal = at_address.get(far_jump(code, i)) if op == "s_setpc_b64" else None
            if goal is None:
                bad.append((address, op, operands))
            else:
                todo.append(goal)
            continue
        if target and target[0] in labels:
            todo.append(at_address[code[labels[target[0]]][0] + target[1]])
            if op == "s_branch":
                continue
        todo.append(i + 1)
    return bad


def test_the_rule_is_seen():
    def bad(*lines):
        rows = [(*line.split(" -> "), "")[:2] for line in lines]
        code, labels = W.parse("<k>:\n" + "".join(f"\t{text} // {4 * i:012X}: 00000000 {goal}\n" for i, (text, goal) in enumerate(rows)))
        return reads_before_barrier(code, labels, 0)

    write, read = "ds_write_b64 v0, v[2:3]", "ds_read_b64 v[4:5], v1"
    assert bad(write, read, "s_barrier", "s_endpgm")
    assert not bad(write, "ds_bpermute_b32 v4, v1, v2", "s_barrier", read, "s_endpgm")
    assert bad(write, "s_cbranch_execz 1 -> <k+0xc>", "s_barrier", read, "s_endpgm")
    assert not bad(write, "s_cbranch_execz 1 -> <k+0x10>", "s_barrier", read, "s_endpgm")
    assert not bad(write, "s_branch 1 -> <k+0xc>", read, "s_barrier", "s_endpgm")
    far = ["s_getpc_b64 s[8:9]", "s_add_u32 s8, s8, 16", "s_addc_u32 s9, s9, 0", "s_setpc_b64 s[8:9]"]  # from 4 to 20
    assert bad(*far, "s_barrier", read) and not bad(*far, read, "s_barrier", "s_endpgm") and bad("s_setpc_b64 s[30:31]")
    assert bad("ds_add_rtn_u32 v4, v1, v2", "s_barrier", "s_endpgm")


@pytest.mark.skipif(not os.path.exists(W.OBJDUMP), reason="no disassembler")
def test_nothing_shared_is_read_before_the_workgroup_has_met(tmp_path):
    assert os.path.exists(W.LIB), "not built"
    found = set()
    for i, content in enumerate(W.code_objects(W.LIB)):
        path = tmp_path / f"{i}.co"
        path.write_bytes(content)
        listing = subprocess.run([W.OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True, capture_output=True,
                                 text=True).stdout
        code, labels = W.parse(listing)
        for name, start in labels.items():
            if not any(k in name for k in KERNELS):
                continue
            found.add(name)
            bad = reads_before_barrier(code, labels, start)
            assert not bad, f"{name}: " + "; ".join(f"{op} {' '.join(args)} at {a:#x}" for a, op, args in bad[:8])
    assert len(found) == 12, found  # 3 types: the row, the chunks in two widths, the picks
