"""The wait states of the wave-per-slot DP's hand-written interior block (SW_BLOCK_ASM in falcon_unzip_amd/csrc/fzp_align.hip).

Some results reach a later instruction only after a number of other instructions have been issued, and the compiler, which pads its own code for that, does not look into inline asm.  On gfx950:
  an SGPR or vcc written by a VALU instruction (compare, readlane), read by a VALU instruction        2 between them
  the same as the lane select of v_readlane / v_writelane                                             4
  a VGPR written by a VALU instruction, read through DPP                                              2
  a VGPR written by a VALU instruction, read by v_readlane                                            1
The block's eight step variants are expanded from the source as the preprocessor would and every step is checked together with each step that can follow it, in both bands."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "falcon_unzip_amd", "csrc", "fzp_align.hip")


def _literals(text):
    """the string literals and bare names of a macro body, in order"""
    return re.findall(r'"((?:[^"\\]|\\.)*)"|([A-Za-z_][A-Za-z_0-9]*)', text)


def _macro(src, name):
    m = re.search(r"#define %s\b(?:\(([^)]*)\))?((?:[^\n]*\\\n)*[^\n]*)" % name, src)
    return [a.strip() for a in (m.group(1) or "").split(",") if a.strip()], m.group(2).replace("\\\n", "\n")


def _text(src, body, env):
    return "".join(lit if not nm else env[nm] if nm in env else _text(src, _macro(src, nm)[1], {}) for lit, nm in _literals(body))


def _instructions(text):
    return [i.strip() for i in text.replace("\\n", "\n").replace("\\t", " ").split("\n") if i.strip() and not i.strip().endswith(":")]


def _steps(src, st, ln):
    """label -> (its instructions, the labels that can follow)"""
    block = _macro(src, "SW_BLOCK_ASM")[1]
    out = {}
    for kind, args in re.findall(r"SWB_(DOWN|RIGHT)\(((?:[^()\"]|\"[^\"]*\")*)\)", block):
        pars, body = _macro(src, "SWB_" + kind)
        parts = [a.strip() for a in re.findall(r'(?:"[^"]*"|[^,"])+', args)]
        env = {p: (st if p == "ST" else ln if p == "LN" else _text(src, a, {})) for p, a in zip(pars, parts)}
        assert len(parts) == len(pars)
        ins = _instructions(_text(src, body, env))
        nxt = {m.group(1) for i in ins for m in [re.match(r"s_c?branch\S*\s+Lsw%=_(p\w+)", i)] if m}
        out[env["LBL"]] = (ins, nxt)
    return out


def _regs(op):
    """the registers an operand names, one 32-bit register each"""
    op = op.strip().split(" ")[0]
    m = re.match(r"s\[(\d+):(\d+)\]$", op)
    if m:
        return {"s%d" % k for k in range(int(m.group(1)), int(m.group(2)) + 1)}
    return {op} if re.match(r"(s\d+|vcc|m0|%\[\w+\])$", op) else set()


SGPR_OPS = {"%[top]", "%[bot]", "%[gap]", "%[mv]", "%[qb]", "%[tb]", "%[qsel]", "%[tsel]"}


def _is_sgpr(r):
    return r in ("vcc", "m0") or re.match(r"s\d+$", r) is not None or r in SGPR_OPS


def hazards(ins):
    """what in a straight run of instructions is read too early"""
    bad, written = [], {}                       # register -> index of the VALU instruction that wrote it last
    for k, i in enumerate(ins):
        op, _, rest = i.partition(" ")
        ops = rest.split(",")
        if not op.startswith("v_"):
            for r in _regs(ops[0]):             # a scalar instruction's result is waited for by the hardware
                written.pop(r, None)
            continue
        dst, src = _regs(ops[0]), [_regs(o) for o in ops[1:]]
        for n, rs in enumerate(src):
            for r in rs & set(written):
                between = k - written[r] - 1
                need = 0
                if _is_sgpr(r):
                    need = 4 if op in ("v_readlane_b32", "v_writelane_b32") and n == 1 else 2
                elif "wave_sh" in i and n == 0:
                    need = 2
                elif op == "v_readlane_b32":
                    need = 1
                if between < need:
                    bad.append("%s  (%s from `%s`: %d between, %d needed)" % (i, r, ins[written[r]], between, need))
        for r in dst:
            written[r] = k
    return bad


def test_the_checker_finds_what_it_is_for():
    cmp, cnd = "v_cmp_eq_u32_e32 vcc, %[a], %[b]", "v_cndmask_b32_e32 %[sc], %[x], %[y], vcc"
    assert hazards([cmp, cnd]) and hazards([cmp, "s_nop 0", cnd]) and not hazards([cmp, "s_nop 0", "s_nop 0", cnd])
    mx, dpp = "v_max_i32_e32 %[X], %[hd], %[mm]", "v_mov_b32_dpp %[y], %[X] wave_shl:1 row_mask:0xf bank_mask:0xf"
    assert hazards([mx, "s_nop 0", dpp]) and not hazards([mx, "s_nop 0", "s_nop 0", dpp])
    rl = "v_readlane_b32 %[top], %[X], 0"
    assert hazards([mx, rl]) and not hazards([mx, "s_nop 0", rl])
    c64 = "v_cmp_eq_i32_e64 s[60:61], %[X], %[hd]"
    assert hazards([c64, "s_nop 0", "v_writelane_b32 %[r], s61, m0"]) and not hazards([c64, "s_nop 0", "s_nop 0", "v_writelane_b32 %[r], s60, m0"])
    assert hazards([c64, "s_nop 0", "s_nop 0", "s_nop 0", "v_writelane_b32 %[r], s3, s60"])


@pytest.mark.parametrize("band", ["63", "31"])
def test_interior_block_keeps_its_wait_states(band):
    with open(SRC) as f:
        src = f.read()
    forms = re.findall(r'SW_BLOCK_ASM\((\w+|""), "%s"\)' % band, src)
    assert len(forms) == 2                      # with and without the masks' records
    for form in forms:
        st = "" if form == '""' else _text(src, _macro(src, form)[1], {})
        steps = _steps(src, st, band)
        assert sorted(steps) == ["p0DD", "p0DR", "p0RD", "p0RR", "p1DD", "p1DR", "p1RD", "p1RR"]
        for lbl, (ins, nxt) in steps.items():
            assert len(ins) >= 18 and len(nxt) == 2, (lbl, nxt)
            for n in nxt:
                assert not hazards(ins + steps[n][0]), (lbl, n, hazards(ins + steps[n][0]))
