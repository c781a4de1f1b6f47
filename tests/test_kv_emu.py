"""The operators on the paged cache in the host-side kernel build, on tensors that end at an inaccessible page (tests/emu): rows
with several rotation axes, attention over packed prompts and drafted trees, the pages' books, and a serving sequence of all of
them, against the oracle in float64.  Rows that no sequence holds are NaN, so a kernel that looks at one shows it."""
import numpy as np
import pytest

import emu_util
import kv_cases as KC


@pytest.fixture(scope="module")
def emu(qk):
    with emu_util.emulated(qk) as pool:
        yield pool


@pytest.mark.parametrize("case", KC.PREP, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-r{c[5]}")
def test_prep_axes(qk, emu, case):
    KC.prep_case(qk, emu.tensor, case)


@pytest.mark.parametrize("case", KC.ATT, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-b{c[9]}")
def test_attention(qk, emu, case):
    KC.att_case(qk, emu.tensor, emu.workspace, case)


@pytest.mark.parametrize("name,case,edit,behind", KC.ODD, ids=[c[0] for c in KC.ODD])
def test_attention_odd(qk, emu, name, case, edit, behind):
    KC.att_case(qk, emu.tensor, emu.workspace, case, edit=edit, behind=behind, l2=KC.ODD_L2.get(name, 4e-6))


@pytest.mark.parametrize("seed,page", [(0, 16), (1, 16), (2, 32), (3, 0)])
def test_books(qk, emu, seed, page):
    KC.books_case(qk, emu.tensor, emu.workspace, type_=("f32", "f16")[seed % 2], dh=(128, 256)[seed // 2], page=page, seed=seed, steps=14)


@pytest.mark.parametrize("type_,dh,hq,hkv,page", [("f32", 256, 4, 2, 16), ("f16", 128, 4, 1, 0)])
def test_serving_sequence(qk, emu, type_, dh, hq, hkv, page):
    KC.serve_case(qk, emu.tensor, emu.workspace, type_, dh, hq, hkv, page)


def test_calls_without_work(qk, emu):
    KC.nothing_case(qk, emu.tensor, emu.workspace)


def test_results_do_not_depend_on_the_order_of_the_threads(qk, emu):
    """The same bits whatever order the threads of a workgroup run in between two barriers (a missing barrier shows)."""
    L = emu_util.emu_lib(qk)
    got = []
    try:
        for mode, seed in ((0, 0), (1, 0), (2, 5), (2, 6)):
            L.emu_set_schedule(mode, seed)
            outs = [KC.att_case(qk, emu.tensor, emu.workspace, case)[0] for case in (KC.ATT[0], KC.ATT[3], KC.ATT[4], KC.ATT[7])]
            KC.prep_case(qk, emu.tensor, KC.PREP[1])
            KC.books_case(qk, emu.tensor, emu.workspace, seed=4, steps=6)
            got.append(outs)
    finally:
        L.emu_set_schedule(0, 0)
    for other in got[1:]:
        assert all(KC.same(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("name,case,edit", KC.RANGE_SCORE, ids=[c[0] for c in KC.RANGE_SCORE])
def test_scores_of_far_keys_and_queries(qk, emu, name, case, edit):
    KC.range_case(qk, emu.tensor, emu.workspace, case, edit, "row")


@pytest.mark.parametrize("name,case,edit", KC.RANGE_SUM, ids=[c[0] for c in KC.RANGE_SUM])
def test_value_rows_of_any_size_keep_their_weight(qk, emu, name, case, edit):
    KC.range_case(qk, emu.tensor, emu.workspace, case, edit, "row")


@pytest.mark.parametrize("name,case,edit,per", KC.RANGE_SPLIT, ids=[c[0] for c in KC.RANGE_SPLIT])
def test_small_elements_beside_large_ones(qk, emu, name, case, edit, per):
    KC.range_case(qk, emu.tensor, emu.workspace, case, edit, per)


@pytest.mark.parametrize("case", KC.MANY_RUNS, ids=lambda c: f"{c[0]}-{len(c[6])}-b{c[9]}")
def test_attention_of_many_runs(qk, emu, case):
    KC.att_case(qk, emu.tensor, emu.workspace, case, behind=1)


@pytest.mark.parametrize("case", KC.MANY_RUNS_PREP, ids=lambda c: f"{c[0]}-{len(c[9])}")
def test_prep_of_many_runs(qk, emu, case):
    KC.prep_case(qk, emu.tensor, case)
