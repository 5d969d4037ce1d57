"""Wait states in the built kernels, counted on their machine code.

The compiler inserts the wait states that gfx950's matrix pipes and LDS copies need, but it does not look into inline
asm: an asm statement that reads an MFMA's result too early, or that starts an LDS copy right behind the write of M0,
gets no help and reads stale values.  This walks the control flow of every kernel in the library's own machine code and
counts the wait states on all paths, by the numbers that the compiler itself keeps for builtins:

* a scalar write of M0, then a copy into LDS: 1;
* an MFMA's result, then a vector instruction, a store or an LDS write that reads or overwrites it: 8 for
  16x16x32 and smaller, 12 for the scaled 16x16x128, 20 for everything larger;
* a vector instruction's result, then an MFMA, a lane swap or a DPP operand that reads it: 2;
* the result of a transcendental, then any other vector instruction that reads it: 1;
* a scalar register that a vector instruction wrote, then a load, copy or store that takes its address from it: 5.
"""
import os
import re
import shutil
import subprocess

import pytest

from mlc_decode_amd import build as B

TOOL = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
_LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<\S+?(?:\+0x([0-9a-f]+))?>)?$")
_HEAD = re.compile(r"^([0-9a-f]+) <(\S+)>:$")
_REG = re.compile(r"(?<![\w.])([vas])(?:(\d+)\b|\[(\d+):(\d+)\])")
TRANS = ("v_exp_", "v_log_", "v_rcp_", "v_rsq_", "v_sqrt_", "v_sin_", "v_cos_")
MEMORY = ("global_", "buffer_", "flat_", "scratch_")
STORES = ("global_store", "buffer_store", "flat_store", "scratch_store", "ds_write", "global_atomic", "buffer_atomic", "flat_atomic")


def registers(text):
    for f, one, lo, hi in _REG.findall(text):
        for i in range(int(one or lo), int(one or hi) + 1):
            yield f, i


class Instruction:
    __slots__ = ("op", "text", "at", "target", "writes", "reads", "mfma", "valu", "m0", "copy", "states", "special", "base")

    def __init__(self, op, rest, at, target):
        self.op, self.text, self.at, self.target = op, f"{op} {rest}", at, target
        first, _, others = rest.partition(",")
        self.mfma = op.startswith("v_mfma") or op.startswith("v_smfma")
        self.valu = op.startswith("v_") and not self.mfma and op != "v_nop"
        self.copy = op.startswith(("global_load_lds", "buffer_load")) and ("_lds_" in op or " lds" in rest)
        self.m0 = op.startswith("s_") and first == "m0"
        self.states = int(rest, 0) + 1 if op == "s_nop" else 1
        self.special = "swap" if op.startswith("v_permlane") else "dpp" if self.valu and "_dpp" in op else "trans" if op.startswith(TRANS) else None
        self.base = frozenset(r for r in registers(rest) if r[0] == "s") if op.startswith(MEMORY) else frozenset()
        if self.mfma or self.valu:
            swaps = "swap" in op  # both operands are read and written
            self.writes = frozenset(registers(rest if swaps else first))
            self.reads = frozenset(registers(rest if swaps else others))
        else:
            self.writes = frozenset()
            self.reads = frozenset(registers(rest)) if op.startswith(STORES) else frozenset()

    def result_wait(self):
        if "16x16x128" in self.op:
            return 12
        return 8 if re.search(r"16x16x(32|16|8|4)_|4x4x4", self.op) else 20


def kernels(listing):
    """{name: instructions} of a disassembly."""
    out, start, body = {}, 0, None
    for line in listing.splitlines():
        head = _HEAD.match(line)
        if head:
            start, body = int(head[1], 16), out.setdefault(head[2], [])
            continue
        m = _LINE.match(line)
        if m and body is not None:
            branch = m[1].startswith(("s_branch", "s_cbranch"))
            body.append(Instruction(m[1], m[2], int(m[3], 16), start + int(m[4] or "0", 16) if branch else None))
    return out


def advance(ins, pending, found):
    """`pending`: wait states still missing, by ("m0",) or (what wrote it, register); updated in place."""
    def too_early(kind, regs, rule, verb):
        for r in regs:
            if (kind, r) in pending:
                found.add((rule, ins.at, f"{ins.text}: {verb} {r[0]}{r[1]} {pending[kind, r]} wait states too early"))

    if pending:
        if ins.copy and ("m0",) in pending:
            found.add(("copy", ins.at, f"{ins.text}: right behind the write of m0"))
        too_early("scalar", ins.base, "address", "takes its address from")
        if ins.mfma:
            too_early("valu", ins.reads, "operand", "reads")
        else:
            too_early("mfma", ins.reads | ins.writes, "result", "meets the result")
        if ins.special in ("swap", "dpp"):
            too_early("valu", ins.reads, "lanes", "reads")
        if ins.valu and ins.special != "trans":
            too_early("trans", ins.reads, "transcendental", "reads")
        for k in list(pending):
            pending[k] -= ins.states
            if pending[k] <= 0:
                del pending[k]
    if ins.m0:
        pending[("m0",)] = 1
    for r in ins.writes:
        for kind in ("mfma", "valu", "trans", "scalar"):
            pending.pop((kind, r), None)
        if ins.mfma:
            pending["mfma", r] = ins.result_wait()
        elif r[0] == "s":
            pending["scalar", r] = 5
        else:
            pending["valu", r] = 2
            if ins.special == "trans":
                pending["trans", r] = 1


def violations(body):
    at = {ins.at: i for i, ins in enumerate(body)}
    starts = {0} | {at[i.target] for i in body if i.target in at} | {n + 1 for n, i in enumerate(body) if i.target is not None}
    entry, todo, found = {}, [(0, {})], set()
    while todo:
        i, pending = todo.pop()
        seen = entry.get(i)
        if seen is not None:
            more = {k: v for k, v in pending.items() if seen.get(k, 0) < v}
            if not more:
                continue
            pending = {**seen, **more}
        entry[i] = dict(pending)
        pending = dict(pending)
        while i < len(body):
            ins = body[i]
            advance(ins, pending, found)
            if ins.target is not None:
                if ins.target in at:
                    todo.append((at[ins.target], dict(pending)))
                if ins.op == "s_branch":
                    break
            elif ins.op.startswith(("s_endpgm", "s_setpc")):
                break
            i += 1
            if i in starts:
                todo.append((i, pending))
                break
    return sorted(found)


def test_rules_on_small_listings():
    """On listings written by hand: each rule, the count across a branch, and code that keeps it."""
    def run(*lines):
        text = "0000000000001000 <k>:\n" + "".join(f"\t{t:50s} // {0x1000 + 4 * n:012X}: BF800000{f' <k+0x{b:x}>' if b is not None else ''}\n"
                                                   for n, (t, b) in enumerate((l if isinstance(l, tuple) else (l, None)) for l in lines))
        return {(rule, at) for rule, at, _ in violations(kernels(text)["k"])}  # the instructions that come too early

    mfma, scaled = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], 0", "v_mfma_scale_f32_16x16x128_f8f6f4 v[0:3], v[8:11], v[12:19], 0, v4, v5"
    assert len(run("s_mov_b32 m0, s2", "global_load_lds_dwordx4 v2, s[4:5]")) == 1
    assert len(run("s_add_u32 m0, s2, 0x400", "global_load_lds_dword v[2:3], off nt")) == 1
    assert not run("s_mov_b32 m0, s2", "s_nop 0", "global_load_lds_dwordx4 v2, s[4:5]")
    for op, need in ((mfma, 8), (scaled, 12)):
        assert not run(op, f"s_nop {min(need, 8) - 1}", f"s_nop {max(need - 9, 0)}", "v_max3_f32 v1, v2, v3, v4")
        assert len(run(op, f"s_nop {need - 2}", "v_max3_f32 v9, v2, v7, v6")) == 1
        assert len(run(op, "v_mov_b32_e32 v3, 0")) == 1 and len(run(op, "ds_write_b128 v20, v[0:3]")) == 1
        assert not run(op, "v_mov_b32_e32 v20, v21", op)
    assert not run(mfma, "s_nop 6", ("s_cbranch_scc1 1", 16), "s_nop 0", "v_add_f32_e32 v9, v0, v0")
    assert len(run(mfma, "s_nop 5", ("s_cbranch_scc1 1", 16), "s_nop 0", "v_add_f32_e32 v9, v0, v0")) == 1  # on the taken path alone
    assert len(run("v_mov_b32_e32 v8, v20", "s_nop 0", mfma)) == 1 and not run("v_mov_b32_e32 v8, v20", "s_nop 1", mfma)
    assert len(run("v_permlane16_swap_b32 v20, v8", mfma)) == 1
    assert len(run("v_max_f32_e32 v7, v6, v5", "v_mov_b32_e32 v8, v9", "v_permlane32_swap_b32_e32 v7, v1")) == 1
    assert len(run("v_max_f32_e32 v7, v6, v5", "v_mov_b32_dpp v1, v7 row_ror:8")) == 1 and not run("v_max_f32_e32 v7, v6, v5", "s_nop 1", "v_mov_b32_dpp v1, v7 row_ror:8")
    assert len(run("v_exp_f32_e32 v7, v6", "v_mul_f32_e32 v1, v7, v7")) == 1 and not run("v_exp_f32_e32 v7, v6", "v_exp_f32_e32 v8, v7")
    assert len(run("v_readfirstlane_b32 s5, v1", "s_nop 3", "global_load_dword v1, v0, s[4:5]")) == 1
    assert not run("v_readfirstlane_b32 s5, v1", "s_nop 4", "global_load_dword v1, v0, s[4:5]")
    assert not run("v_readfirstlane_b32 s5, v1", "s_add_u32 s4, s5, s6", "global_load_dword v1, v0, s[2:3]")


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    """[(kernel, instructions)] of the built library."""
    if not os.path.exists(TOOL) or not os.path.exists(B.LIB_PATH):
        pytest.skip("needs llvm-objdump and the built library")
    tmp = tmp_path_factory.mktemp("isa")
    lib = shutil.copy(B.LIB_PATH, tmp)
    subprocess.run([TOOL, "--offloading", lib], check=True, capture_output=True, cwd=tmp)
    units = sorted(f for f in os.listdir(tmp) if f.endswith(B.ARCH))
    assert len(units) == len(B.SOURCES)
    out = []
    for unit in units:
        out += kernels(subprocess.run([TOOL, "-d", f"--mcpu={B.ARCH}", os.path.join(tmp, unit)], check=True, capture_output=True, text=True).stdout).items()
    assert sum(i.copy for _, body in out for i in body) > 100 and sum(i.mfma for _, body in out for i in body) > 1000  # it was understood
    return out


@pytest.fixture(scope="module")
def early(library):
    return [(rule, f"{name}+{at:x}: {what}") for name, body in library for rule, at, what in violations(body)]


@pytest.mark.parametrize("rule", ["copy", "operand", "result", "address", "lanes", "transcendental"])
def test_wait_states_of_every_kernel(early, rule):
    bad = [what for r, what in early if r == rule]
    assert not bad, f"{len(bad)} places, first:\n" + "\n".join(bad[:20])
