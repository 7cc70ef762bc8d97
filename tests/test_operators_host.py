"""The operators' binding, and beam search from the command line (the kernels on the CPU simulator)."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from moshi_amd import _capi, loaders
from tests import operator_cases as oc
from tests import tlm_cases as tc
from tests.test_tlm_host import BIBAPEL, _save
from tests.test_tlm_sim import tlm_lib  # noqa: F401  (fixture)

ROOT = Path(__file__).resolve().parents[1]


def _header():
    return (ROOT / "include" / "moshi_tlm.h").read_text()


def test_binding_covers_the_header_and_the_library_exports_it():
    declared = set(re.findall(r"\b(mmi_(?:kv|beam)_[a-z0-9_]+)\s*\(", _header()))
    assert len(declared) == 7 and declared == {n for n in _capi.TLM_SIGNATURES if n.startswith(("mmi_kv_", "mmi_beam_"))}
    from moshi_amd import build
    build.build(verbose=False, which="tlm")
    lib = _capi.load_tlm()
    assert all(hasattr(lib.cdll, n) for n in declared)


def test_structs_equal_the_binding(tmp_path):
    structs = {"mmi_kv_cache": _capi.KVCacheDesc, "mmi_kv_seqs": _capi.KVSeqs, "mmi_tlm_cfg": _capi.TLMCfg}
    lines = ['#include "moshi_tlm.h"', "#include <stdio.h>", "#include <stddef.h>", "int main(void) {"]
    for s, cls in structs.items():
        lines.append(f'  printf("{s} . %zu\\n", sizeof({s}));')
        lines += [f'  printf("{s} {f} %zu\\n", offsetof({s}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "t.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    for line in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = line.split()
        assert (ctypes.sizeof(structs[s]) if f == "." else getattr(structs[s], f).offset) == int(v), line


def test_public_names():
    import moshi_amd
    assert {"PagedKVCache", "BeamChoice", "BeamHypothesis", "beam_reorder", "beam_search", "beam_select"} <= set(moshi_amd.__all__)
    assert all(hasattr(moshi_amd, n) for n in moshi_amd.__all__)


def _run(tlm_lib, tmp_path, monkeypatch, prompts, *args):  # noqa: F811
    from moshi_amd import run_inference
    load, made = loaders.get_token_lm, []
    monkeypatch.setattr(loaders, "get_token_lm", lambda path, **kw: made.append(load(path, **{**kw, "device": "cpu", "lib": tlm_lib})) or made[-1])
    (tmp_path / "in.txt").write_text("\n".join(" ".join(map(str, p)) for p in prompts) + "\n")
    run_inference.main(["--checkpoint-dir", str(tmp_path), "--dtype", "float32", "--batch-size", "2", "--step-tokens", "16", "--max-new-tokens", "4", *args,
                        str(tmp_path / "in.txt"), str(tmp_path / "out.txt")])
    return made[0], [[int(t) for t in ln.split()] for ln in (tmp_path / "out.txt").read_text().splitlines()]


@pytest.mark.parametrize("codes", ["like-dtype", "int8"])
def test_command_line_searches_with_beams(tlm_lib, tmp_path, monkeypatch, codes):  # noqa: F811
    _save(tmp_path, BIBAPEL)
    cfg = loaders.token_lm_config_from_dict(BIBAPEL)
    prompts = [tc.tokens_of(cfg, n, seed=n) for n in (7, 40, 2)]
    lm, got = _run(tlm_lib, tmp_path, monkeypatch, prompts, "--beams", "3", "--stop-token", "1", "--length-penalty", "0.5", "--kv-cache", codes)
    assert lm.kv_cache == (None if codes == "like-dtype" else codes) and lm.max_slots == 6 and lm.free_pages == lm.total_pages
    want = oc.beam_search(lm, prompts, 3, 4, eos=1, length_penalty=0.5, step_tokens=16)
    assert got == [h[0].tokens for h in want] and all(len(t) == 4 or t[-1] == 1 for t in got)


def test_command_line_takes_one_end_token_for_beams(tlm_lib, tmp_path, monkeypatch):  # noqa: F811
    _save(tmp_path, BIBAPEL)
    with pytest.raises(SystemExit):
        _run(tlm_lib, tmp_path, monkeypatch, [[1, 2]], "--beams", "2", "--stop-token", "1", "--stop-token", "2")
