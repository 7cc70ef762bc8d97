"""The token language models' operators on a real MI355X: the cases of tests/operator_cases.py, captured graphs, other streams."""
import pytest
import torch

from tests import operator_cases as oc
from tests import tlm_cases as tc

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="session")
def lib():
    assert torch.cuda.is_available(), "-m gpu tests need a GPU"
    from moshi_amd import _capi
    return _capi.load_tlm()


def test_refusals(lib):
    oc.check_refusals(DEV, lib)


def test_select_refusals(lib):
    oc.check_select_refusals(DEV, lib)


def test_reorder_refusals(lib):
    oc.check_reorder_refusals(DEV, lib)


@pytest.mark.parametrize("name", sorted(oc.APPENDS))
def test_append(lib, name):
    oc.check_append(name, DEV, lib)


@pytest.mark.parametrize("name", ["single_tokens", "portions", "rotated_part_of_odd_sizes"])
def test_append_unaligned(lib, name):
    oc.check_append(name, DEV, lib, strided=True)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_append_in_any_order(lib, codes):
    oc.check_append_order(DEV, lib, codes)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_not_finite(lib, codes):
    oc.check_not_finite(DEV, lib, codes)


@pytest.mark.parametrize("name", sorted(oc.ATTENDS))
def test_attend(lib, name):
    oc.check_attend(name, DEV, lib)


@pytest.mark.parametrize("name", ["single_fp32", "rotated", "portions"])
def test_attend_unaligned(lib, name):
    oc.check_attend(name, DEV, lib, strided=True)


def test_extreme_scores(lib):
    oc.check_extreme_scores(DEV, lib)


@pytest.mark.parametrize("name", sorted(oc.SELECTS))
def test_select(lib, name):
    oc.check_select(name, DEV, lib)


@pytest.mark.parametrize("beams", [1, 3, 8, 13, 32])
def test_reorder(lib, beams):
    oc.check_reorder(DEV, lib, beams)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [oc.F32, oc.BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", sorted(n for n in tc.MECHANISMS if n.startswith("grouped_attention")) + ["bibapel", "two_kept_windows"])
def test_token_lm(lib, name, dtype, codes):
    oc.check_token_lm(name, DEV, lib, dtype, codes)


@pytest.mark.parametrize("dtype", [oc.F32, oc.BF16], ids=["fp32", "bf16"])
def test_token_lm_longer_than_its_pool(lib, dtype):
    oc.check_token_lm("two_kept_windows", DEV, lib, dtype, "int8", n=700, cut_sets=((130, 1),), max_slots=2, max_tokens=320)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_token_lm_batch(lib, codes):
    oc.check_token_lm_batch(DEV, lib, oc.F32, codes)


def _decode(lib, seqs=3, steps=40):
    """What a decoding loop keeps: cache, page table, positions, and the tokens' queries, keys and values of every step."""
    from moshi_amd.kv_cache import PagedKVCache
    g = torch.Generator().manual_seed(1)
    cache = PagedKVCache.empty(2 * seqs, 2, 64, codes="int8", device=DEV, rot_dim=64, lib=lib)
    table = torch.randperm(2 * seqs, generator=g).to(torch.int32).view(seqs, 2).to(DEV)
    rows = [[torch.randn((seqs, n, 64), generator=g).to(torch.bfloat16).to(DEV) for n in (8, 2, 2)] for _ in range(steps)]
    return cache, table, torch.full((seqs,), 50, dtype=torch.int32, device=DEV), rows


def test_captured_decoding(lib):
    """append, attend, select and reorder in one graph, positions advanced between its replays: every replay gives what eager calls give."""
    from moshi_amd.beam import beam_reorder, beam_select
    eager, table, pos, rows = _decode(lib)
    graphed, _, gpos, _ = _decode(lib)
    q, k, v = [t.clone() for t in rows[0]]
    logits, scores, state = torch.randn((4, 500), device=DEV), torch.zeros((1, 4), device=DEV), torch.randn((4, 33), device=DEV)

    def step(cache, p):
        cache.append(k, v, table, p)
        r = beam_select(logits, scores, lib=lib)
        beam_reorder([state], r.parents, lib=lib)
        return cache.attend(q, table, p, window=60, keep_first=2), r

    keep = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(_decode(lib)[0], gpos)                           # (allocations and code, outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, r = step(graphed, gpos)
    g = torch.Generator().manual_seed(8)
    for i, (a, b, c) in enumerate(rows):
        q.copy_(a), k.copy_(b), v.copy_(c)
        logits.copy_(torch.randn((4, 500), generator=g))
        state.copy_(keep)
        want, wr = step(eager, pos)
        moved = state.clone()
        state.copy_(keep)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(r.tokens, wr.tokens) and torch.equal(r.scores, wr.scores) and torch.equal(state, moved), i
        pos += 1
        gpos += 1
    assert torch.equal(eager.k, graphed.k) and torch.equal(eager.v_scale, graphed.v_scale)


def test_streams_of_their_own(lib):
    """Two loops on two streams at once, many splits each, beside the same loops one after the other."""
    def loop(seed):
        c = oc.Case([1300, 700], [1, 1], single=True, kv_heads=2, rep=4, seed=seed, dim=128, vdim=128)
        cache, q, k, v, args = oc.build(c, DEV, lib)
        def run():
            for _ in range(20):
                cache.append(k, v, *args)
                out = cache.attend(q, *args)
            return out
        return run
    loops = [loop(1), loop(2)]
    want = [f().clone() for f in loops]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in loops], [None, None]
    for i, (s, f) in enumerate(zip(streams, loops)):
        with torch.cuda.stream(s):
            got[i] = f()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_offsets_past_32_bits(lib):
    """A pool above 4 GiB of codes, its last pages in use."""
    from moshi_amd.kv_cache import PagedKVCache
    pages = (1 << 32) // (8 * 64 * 128) + 70
    cache = PagedKVCache.empty(pages, 8, 128, codes="int8", device=DEV, lib=lib)
    small = PagedKVCache.empty(4, 8, 128, codes="int8", device=DEV, lib=lib)
    g = torch.Generator().manual_seed(2)
    k, v = [torch.randn((200, 8, 128), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    q = torch.randn((200, 16, 128), generator=g).to(torch.bfloat16).to(DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = []
    for c, table in ((cache, i32([pages - 1, 3, pages - 2, pages - 60])), (small, i32([3, 2, 1, 0]))):
        c.append(k, v, table, i32(0), i32(0, 200))
        out.append((c.attend(q, table, i32(0), i32(0, 200)), c.attend(q[-1:], table, i32(199))))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("name, codes", [("mixed", None), ("bibapel", None), ("bibapel", "int8"), ("two_kept_windows", "e4m3"), ("bigram", None), ("delta_widest", None),
                                         ("projected_passes", None)])
@pytest.mark.parametrize("dtype", [oc.F32, oc.BF16], ids=["fp32", "bf16"])
def test_token_lm_reorder(lib, name, codes, dtype):
    oc.check_token_lm_reorder(name, DEV, lib, dtype, codes)


def test_token_lm_reorder_pool(lib):
    oc.check_token_lm_reorder_pool(DEV, lib)


@pytest.mark.parametrize("name, codes, alpha", [("mixed", None, 0.0), ("bibapel", None, 0.7), ("grouped_attention", "int8", 1.0), ("bibapel", "e4m3", 0.0)])
@pytest.mark.parametrize("dtype", [oc.F32, oc.BF16], ids=["fp32", "bf16"])
def test_beam_search(lib, name, codes, alpha, dtype):
    oc.check_beam_search(DEV, lib, name, dtype, codes, alpha=alpha)


def test_beam_search_of_one(lib):
    oc.check_beam_search_of_one(DEV, lib)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_position_past_the_table(lib, codes):
    oc.check_position_past_the_table(DEV, lib, codes)


def test_rows_in_no_order(lib):
    oc.check_rows_in_no_order(DEV, lib)


@pytest.mark.parametrize("name", sorted(oc.FAR | oc.FAR_LARGE))
def test_blocks_far_apart(lib, name):
    oc.check_blocks_far_apart(name, DEV, lib)


def test_select_penalties(lib):
    oc.check_select_penalties(DEV, lib)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_keeps_everything(lib, codes):
    oc.check_keeps_everything(DEV, lib, codes)


@pytest.mark.parametrize("codes", [None, "int8", "e4m3"])
def test_token_lm_keeps_everything(lib, codes):
    oc.check_token_lm_keeps_everything(DEV, lib, codes)


@pytest.mark.parametrize("name", sorted(oc.RESTS))
def test_rows_that_no_sequence_brings(lib, name):
    oc.check_rest(name, DEV, lib)


def test_flags(lib):
    oc.check_flags(DEV, lib)


def test_reorder_views(lib):
    oc.check_reorder_views(DEV, lib)


def test_output_rows(lib):
    oc.check_output_rows(DEV, lib)


def test_wide_integers(lib):
    oc.check_wide_integers(DEV, lib)


@pytest.mark.parametrize("name, codes, alpha", [("mixed", None, 0.0), ("bibapel", None, 0.7), ("grouped_attention", "int8", 1.0), ("bibapel", "e4m3", 0.0), ("two_kept_windows", "int8", -0.5)])
@pytest.mark.parametrize("dtype", [oc.F32, oc.BF16], ids=["fp32", "bf16"])
def test_beam_search_choices(lib, name, codes, alpha, dtype):
    oc.check_beam_search_choices(DEV, lib, name, dtype, codes, alpha=alpha)


def test_wide_negative_integers(lib):
    oc.check_wide_negative_integers(DEV, lib)


def test_reorder_of_too_long_rows(lib):
    oc.check_reorder_of_too_long_rows(DEV, lib)
