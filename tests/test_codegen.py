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
        assert not copies_of_one(lines)
    assert seen


def test_no_element_is_cast_where_it_stands():
    """An element is read into a variable before its bits are taken (of arrays that would be right, but nothing tells them from vectors here)."""
    bare = re.compile(r"__builtin_bit_cast\((?:unsigned|int|float|u?int\d+_t|_Float16), [\w.]+(?:\[[^\[\]]*\])+\)")
    assert bare.search("__builtin_bit_cast(unsigned, x[2])") and not bare.search("__builtin_bit_cast(float, w[0] << 16)")
    for p in sorted(build.CSRC.glob("*.h")) + sorted(build.CSRC.glob("*.hip")):
        assert not bare.findall(p.read_text()), p
