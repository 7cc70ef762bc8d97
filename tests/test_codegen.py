"""Device code of the built libraries, looked over for a fault that the compiler has made in it.

A vector whose elements are changed behind a branch, one at a time, while it lives in accumulation registers, has been copied back with its first element in place
of each of the others: `v_accvgpr_write a65, v102; v_accvgpr_write a66, v102; v_accvgpr_write a67, v102` for v102, v103, v104.  No source that is wrong stands behind
it, so tests of values see it only where a call takes that branch.  Adjacent accumulation registers that are written from one vector register are it, or a vector of
equal constants."""
import re
import subprocess
from pathlib import Path

import pytest

from moshi_amd import build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
WRITE = re.compile(r"v_accvgpr_write_b32 a(\d+), (v\d+)\b")
DEFINED = re.compile(r"(v_\w+|global_\w+|buffer_\w+|flat_\w+|scratch_\w+|ds_\w+) (v\d+|v\[\d+:\d+\])(?:, (\S+))?")


def copies_of_one(lines):
    """Lines of adjacent accumulation registers written from one vector register that does not hold a constant."""
    found, run, constant, where = [], [], {}, None

    def end():
        if len(run) > 1 and not constant.get(run[0][1]):
            found.append((where, [t for _, _, t in run]))
        run.clear()

    for line in lines:
        t = line.split("//")[0].split(";")[0].strip()
        m = re.match(r"[0-9a-f]+ <(\w+)>:", t) or re.match(r"(_Z\w+):", t)
        if m:
            end()
            where, constant = m.group(1), {}
            continue
        if not t:
            continue
        m = WRITE.match(t)
        if m:
            a, v = int(m.group(1)), m.group(2)
            if run and (a != run[-1][0] + 1 or v != run[-1][1]):
                end()
            run.append((a, v, t))
            continue
        end()
        m = DEFINED.match(t)
        if m:
            regs = [m.group(2)]
            if "[" in regs[0]:
                lo, hi = map(int, re.findall(r"\d+", regs[0]))
                regs = [f"v{i}" for i in range(lo, hi + 1)]
            for r in regs:
                constant[r] = m.group(1).startswith("v_mov_b32") and re.fullmatch(r"-?[0-9a-fx.]+", m.group(3) or "") is not None
    end()
    return found


SPILL = re.compile(r"scratch_store_dword(?:x\d)? off, v(?:\[(\d+):(\d+)\]|(\d+)), off(?: offset:(\d+))?$")
RELOAD = re.compile(r"scratch_load_dword(?:x\d)? ([av])(?:\[(\d+):(\d+)\]|(\d+)), off, off(?: offset:(\d+))?$")


def lost_elements(lines):
    """Reloads of a part of a vector whose next element waits in an accumulation register and is not fetched beside them."""
    functions, code = [], None
    for line in lines:
        t = line.split("//")[0].split(";")[0].strip()
        m = re.match(r"[0-9a-f]+ <(\w+)>:", t) or re.match(r"(_Z\w+):", t)
        if m:
            code = []
            functions.append((m.group(1), code))
        elif t and code is not None:
            code.append(t)
    found = []
    for name, code in functions:
        waiting = {}                                       # (place, elements): the accumulation registers that hold the element behind them
        for k, t in enumerate(code):
            m = SPILL.match(t)
            if m:
                lo, hi = (int(m.group(1)), int(m.group(2))) if m.group(1) else (int(m.group(3)),) * 2
                for near in code[max(0, k - 4):k + 5]:
                    w = WRITE.match(near)
                    if w and w.group(2) == f"v{hi + 1}":
                        waiting.setdefault((m.group(4), hi - lo), set()).add(w.group(1))
        for k, t in enumerate(code):
            m = RELOAD.match(t)
            if not m:
                continue
            lo, hi = (int(m.group(2)), int(m.group(3))) if m.group(2) else (int(m.group(4)),) * 2
            held = waiting.get((m.group(5), hi - lo))
            fetch = held and re.compile(rf"v_accvgpr_(?:read|mov)_b32 {m.group(1)}{hi + 1}, a(?:{'|'.join(held)})$")
            if held and not any(fetch.match(near) for near in code[max(0, k - 6):k + 7]):
                found.append((name, t))
    return found


def test_the_lost_element_is_seen():
    spill = ["_Zk:", "v_accvgpr_write_b32 a255, v7", "scratch_store_dwordx3 off, v[4:6], off", "scratch_store_dwordx4 off, v[4:7], off offset:16"]
    bad = ["scratch_load_dwordx4 a[16:19], off, off offset:16", "scratch_load_dwordx3 a[170:172], off, off", "v_mfma_f32_32x32x16_f16 a[16:31], v[0:3], a[170:173], a[16:31]"]
    assert lost_elements(spill + bad) == [("_Zk", bad[1])]
    assert not lost_elements(spill + ["v_accvgpr_read_b32 v57, a255", "scratch_load_dwordx3 v[54:56], off, off"])
    assert not lost_elements(spill + ["v_accvgpr_mov_b32 a173, a255"] + bad) and not lost_elements(["_Zk:", spill[3]] + bad[:1])


def test_the_fault_is_seen():
    bad = ["_Zk:", "v_accvgpr_read_b32 v102, a64", "v_cndmask_b32_e32 v103, v4, v103, vcc", "v_accvgpr_write_b32 a65, v102", "v_accvgpr_write_b32 a66, v102",
           "v_accvgpr_write_b32 a67, v102", "s_branch 12"]
    assert copies_of_one(bad) == [("_Zk", bad[3:6])]
    right = bad[:4] + ["v_accvgpr_write_b32 a66, v103", "v_accvgpr_write_b32 a67, v104", "s_branch 12"]
    assert not copies_of_one(right)
    assert not copies_of_one(["_Zk:", "v_mov_b32_e32 v7, 0", "v_accvgpr_write_b32 a0, v7", "v_accvgpr_write_b32 a1, v7", "v_accvgpr_write_b32 a2, 0", "v_accvgpr_write_b32 a3, 0"])
    assert copies_of_one(["_Zk:", "v_mov_b32_e32 v7, 0", "global_load_dwordx2 v[6:7], v[0:1], off", "v_accvgpr_write_b32 a0, v7", "v_accvgpr_write_b32 a1, v7"])


@pytest.mark.parametrize("which", sorted(build.LIBS))
def test_no_vector_is_copied_back_as_its_first_element(which, tmp_path):
    build.build(verbose=False, which=which)
    lib = build.LIBS[which][0]
    (tmp_path / lib.name).symlink_to(lib)
    subprocess.run([OBJDUMP, "--offloading", lib.name], cwd=tmp_path, check=True, capture_output=True)
    code = [p for p in tmp_path.iterdir() if p.name.endswith(build.ARCH)]
    assert code
    seen = 0
    for p in code:
        with subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", p.name], cwd=tmp_path, stdout=subprocess.PIPE, text=True) as dump:
            lines = dump.stdout.readlines()
        assert dump.returncode == 0
        seen += sum("v_accvgpr_write" in x for x in lines)
        assert not copies_of_one(lines) and not lost_elements(lines)
    assert seen


def test_no_element_is_cast_where_it_stands():
    """An element is read into a variable before its bits are taken (of arrays that would be right, but nothing tells them from vectors here)."""
    bare = re.compile(r"__builtin_bit_cast\((?:unsigned|int|float|u?int\d+_t|_Float16), [\w.]+(?:\[[^\[\]]*\])+\)")
    assert bare.search("__builtin_bit_cast(unsigned, x[2])") and not bare.search("__builtin_bit_cast(float, w[0] << 16)")
    for p in sorted(build.CSRC.glob("*.h")) + sorted(build.CSRC.glob("*.hip")):
        assert not bare.findall(p.read_text()), p
