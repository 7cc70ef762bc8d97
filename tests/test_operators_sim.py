"""The token language models' operators on the kernel simulator: the cases of tests/operator_cases.py."""
import pytest

from tests import operator_cases as oc
from tests.test_tlm_sim import tlm_lib  # noqa: F401  (fixture)

DEV = "cpu"


@pytest.mark.parametrize("name", sorted(oc.APPENDS))
def test_append(tlm_lib, name):  # noqa: F811
    oc.check_append(name, DEV, tlm_lib)


@pytest.mark.parametrize("name", ["single_tokens", "portions", "rotated_part_of_odd_sizes"])
def test_append_unaligned(tlm_lib, name):  # noqa: F811
    oc.check_append(name, DEV, tlm_lib, strided=True)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_append_in_any_order(tlm_lib, codes):  # noqa: F811
    oc.check_append_order(DEV, tlm_lib, codes)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_not_finite(tlm_lib, codes):  # noqa: F811
    oc.check_not_finite(DEV, tlm_lib, codes)


@pytest.mark.parametrize("name", sorted(oc.ATTENDS))
def test_attend(tlm_lib, name):  # noqa: F811
    oc.check_attend(name, DEV, tlm_lib)


@pytest.mark.parametrize("name", ["single_fp32", "rotated", "portions"])
def test_attend_unaligned(tlm_lib, name):  # noqa: F811
    oc.check_attend(name, DEV, tlm_lib, strided=True)


def test_extreme_scores(tlm_lib):  # noqa: F811
    oc.check_extreme_scores(DEV, tlm_lib)


def test_refusals(tlm_lib):  # noqa: F811
    oc.check_refusals(DEV, tlm_lib)


@pytest.mark.parametrize("name", sorted(oc.SELECTS))
def test_select(tlm_lib, name):  # noqa: F811
    oc.check_select(name, DEV, tlm_lib)


def test_select_refusals(tlm_lib):  # noqa: F811
    oc.check_select_refusals(DEV, tlm_lib)


@pytest.mark.parametrize("beams", [1, 3, 8, 13, 32])
def test_reorder(tlm_lib, beams):  # noqa: F811
    oc.check_reorder(DEV, tlm_lib, beams)


def test_reorder_refusals(tlm_lib):  # noqa: F811
    oc.check_reorder_refusals(DEV, tlm_lib)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("name", ["grouped_attention", "grouped_attention_own_heads", "grouped_attention_wide", "grouped_attention_keeps_more_than_it_sees", "bibapel"])
def test_token_lm(tlm_lib, name, codes):  # noqa: F811
    oc.check_token_lm(name, DEV, tlm_lib, oc.F32, codes)


def test_token_lm_bf16(tlm_lib):  # noqa: F811
    oc.check_token_lm("grouped_attention", DEV, tlm_lib, oc.BF16, "int8")


def test_token_lm_longer_than_its_pool(tlm_lib):  # noqa: F811
    oc.check_token_lm("two_kept_windows", DEV, tlm_lib, oc.F32, "int8", n=330, cut_sets=((130, 1),), max_slots=2, max_tokens=320)


def test_token_lm_batch(tlm_lib):  # noqa: F811
    oc.check_token_lm_batch(DEV, tlm_lib, oc.F32, "int8")


def test_token_lm_refusals(tlm_lib):  # noqa: F811
    oc.check_token_lm_refusals(DEV, tlm_lib)


@pytest.mark.parametrize("name, codes", [("mixed", None), ("bibapel", None), ("bibapel", "int8"), ("two_kept_windows", "e4m3"), ("bigram", None), ("delta", None)])
def test_token_lm_reorder(tlm_lib, name, codes):  # noqa: F811
    oc.check_token_lm_reorder(name, DEV, tlm_lib, codes=codes, lengths=((20, 64, 1, 70, 63), (65, 7, 30, 30, 66)), tail=6)


def test_token_lm_reorder_pool(tlm_lib):  # noqa: F811
    oc.check_token_lm_reorder_pool(DEV, tlm_lib)


@pytest.mark.parametrize("name, codes, alpha", [("mixed", None, 0.0), ("bibapel", None, 0.7), ("grouped_attention", "int8", 1.0)])
def test_beam_search(tlm_lib, name, codes, alpha):  # noqa: F811
    oc.check_beam_search(DEV, tlm_lib, name, codes=codes, alpha=alpha, beams=3, steps=5)


def test_beam_search_of_one(tlm_lib):  # noqa: F811
    oc.check_beam_search_of_one(DEV, tlm_lib)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_position_past_the_table(tlm_lib, codes):  # noqa: F811
    oc.check_position_past_the_table(DEV, tlm_lib, codes)


def test_rows_in_no_order(tlm_lib):  # noqa: F811
    oc.check_rows_in_no_order(DEV, tlm_lib)


@pytest.mark.parametrize("name", sorted(oc.FAR))
def test_blocks_far_apart(tlm_lib, name):  # noqa: F811
    oc.check_blocks_far_apart(name, DEV, tlm_lib)


def test_select_penalties(tlm_lib):  # noqa: F811
    oc.check_select_penalties(DEV, tlm_lib)


def test_large_lds_is_asked_for_on_every_device(tlm_lib):  # noqa: F811
    """How much LDS a kernel may have is an attribute of the kernel on ONE device: the operators, and the engine's kernels, ask again on another."""
    c, dll, asked = oc.ATTENDS["portions_fp32"], tlm_lib.cdll, []
    cfg = oc.tc.MECHANISMS["delta"]
    sd = oc.random_token_lm_state_dict(cfg, seed=5)
    for device in (51, 52, 51):
        dll.hipsim_set_device(device)
        try:
            cache, q, k, v, args = oc.build(c, DEV, tlm_lib)
            cache.append(k, v, *args)
            before = dll.hipsim_attributes(device)
            cache.attend(q, *args)
            both = dll.hipsim_attributes(device)
            lm = oc.TokenLM(sd, cfg, device=DEV, dtype=oc.F32, lib=tlm_lib, max_slots=2, max_tokens=256)
            lm.step([(lm.open(), oc.tc.tokens_of(cfg, 80), [79])])
        finally:
            dll.hipsim_set_device(0)
        asked.append((both - before, dll.hipsim_attributes(device)))
    assert asked[0][0] == 1 and asked[0][1] > 1 and asked[1] == asked[0] and asked[2] == (0, asked[0][1]), asked


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_keeps_everything(tlm_lib, codes):  # noqa: F811
    oc.check_keeps_everything(DEV, tlm_lib, codes)


@pytest.mark.parametrize("codes", [None, "int8", "e4m3"])
def test_token_lm_keeps_everything(tlm_lib, codes):  # noqa: F811
    oc.check_token_lm_keeps_everything(DEV, tlm_lib, codes)


@pytest.mark.parametrize("name", sorted(oc.RESTS))
def test_rows_that_no_sequence_brings(tlm_lib, name):  # noqa: F811
    oc.check_rest(name, DEV, tlm_lib)


def test_flags(tlm_lib):  # noqa: F811
    oc.check_flags(DEV, tlm_lib)


def test_reorder_views(tlm_lib):  # noqa: F811
    oc.check_reorder_views(DEV, tlm_lib)


def test_output_rows(tlm_lib):  # noqa: F811
    oc.check_output_rows(DEV, tlm_lib)


def test_wide_integers(tlm_lib):  # noqa: F811
    oc.check_wide_integers(DEV, tlm_lib)


@pytest.mark.parametrize("name, codes, alpha, dtype", [("mixed", None, 0.0, oc.F32), ("bibapel", None, 0.7, oc.BF16), ("grouped_attention", "int8", 1.0, oc.F32),
                                                       ("two_kept_windows", "e4m3", 0.0, oc.BF16)])
def test_beam_search_choices(tlm_lib, name, codes, alpha, dtype):  # noqa: F811
    oc.check_beam_search_choices(DEV, tlm_lib, name, dtype, codes, beams=3, steps=4, alpha=alpha)


def test_long_tables(tlm_lib):  # noqa: F811
    oc.check_long_tables(DEV, tlm_lib)


def test_wide_negative_integers(tlm_lib):  # noqa: F811
    oc.check_wide_negative_integers(DEV, tlm_lib)


def test_reorder_of_too_long_rows(tlm_lib):  # noqa: F811
    oc.check_reorder_of_too_long_rows(DEV, tlm_lib)
