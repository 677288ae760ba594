"""Every form of the sequence operators' kernels is run by a test on the GPU: the lists of cases there, put through the library's own rules.  A
change of a rule that leaves a form without a case fails here."""
import ctypes

import pytest

from tests import _sequence_forms as F
from tests import test_gpu_sequence as T
from tests import test_gpu_sequence_edges as E
from tests import test_gpu_sequence_forms as L
from tests import test_sequence_cpu as C
from turboae_amd import _lib


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    if F.compiler() is None:
        pytest.skip("no C++ compiler")
    return F.Forms(str(tmp_path_factory.mktemp("forms")))


def test_every_form_of_the_scan_has_a_case(forms):
    cases = [(("bf16", "f32", "f16")[sum(c) % 3], *c) for c in E.FORMS] + [c[:5] for c in T.SCAN] + L.SCANS
    want = {("lane", full, cut) for full in (False, True) for cut in (False, True)}
    want |= {("tile", lanes, per_lane, cut, V) for lanes, per_lane in F.TILES for cut in (False, True) for V in (1, 4)}
    want |= {("short", 4, 1 << i) for i in range(5)} | {("short", 1, 1 << i) for i in range(7)}
    want |= {("step", 4, 1 << i, each) for i in range(5) for each in (1, 4)} | {("step", 1, 1 << i, each) for i in range(7) for each in (1, 4)}
    assert set(forms.scan(cases)) == want


def test_every_form_of_the_scan_meets_infinities(forms):
    """With states that fill its lanes and with states that do not; pieces only matter to the latter."""
    found = {form[:-1] + ("cut" if form[-1] else "whole",) if form[0] == "lane" else form + (c[4] == form[1] * form[2],) if form[0] == "tile" else form[:3] for form, c in
             zip(forms.scan(L.INFINITE), L.INFINITE)}
    tiles = {("tile", *split, cut, V, False) for split in F.TILES for cut in (False, True) for V in (1, 4)} | {("tile", *split, False, V, True) for split in F.TILES for V in (1, 4)}
    assert found >= tiles | {("lane", False, "whole"), ("lane", False, "cut"), ("lane", True, "whole")}
    halves = {c[4] > 12 for form, c in zip(forms.scan(L.INFINITE), L.INFINITE) if form[0] == "lane" and c[4] < 16}
    assert halves == {False, True}                                # with and without states in the last quarter of a lane
    assert found >= {("short", 4, 1 << i) for i in (2, 3, 4)} | {("short", 1, 1 << i) for i in range(2, 7)} | {("step", 4, 4), ("step", 1, 8)}


def test_every_form_of_int8_linear_has_a_case(forms):
    small, large = forms.int8(T.INT8), forms.int8(L.INT8_LARGE)
    assert set(small + large) == set(F.INT8_FORMS)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    for form in ("tiles128", "tiles128_two", "tiles256"):         # aligned rows of 16-bit and of 32-bit outputs, and others
        aligned = {(size[dt], N * size[dt] % 16 == 0) for (dt, M, K, N), f in zip(T.INT8 + L.INT8_LARGE, small + large) if f == form}
        assert aligned >= {(2, True), (2, False), (4, True)}, (form, aligned)
    tiles = [-(-M // 256) * -(-N // 256) for (dt, M, K, N), f in zip(L.INT8_LARGE, large) if f == "tiles256"]
    assert tiles and all(t > 256 for t in tiles)                  # more than the workgroups that run at once


def test_every_form_of_token_logprobs_has_a_case(forms):
    cases = [(*c, aligned) for c in T.LOGP + L.LOGP_LARGE for aligned in (False, True)]
    found = {(lanes, elements, parts > 1) for lanes, elements, parts in forms.logprobs(cases)}
    assert found >= {(8, 8, False), (64, 8, False), (64, 32, False), (64, 32, True), (256, 32, False), (256, 32, True), (256, 64, False), (256, 64, True)}


def test_short_rows_of_logits_are_one_part_wherever_they_start(forms):
    """Rows that are read by single elements need no room for a granule that they start inside: one launch, no workspace."""
    rows = [(dt, 1000, V, top, aligned) for dt in F.DTYPE for V in (33, 56, 57, 60, 61, 63, 64) for top in (0, 1, V // 2, 32) for aligned in (False, True)]
    for case, (lanes, elements, parts) in zip(rows, forms.logprobs(rows)):
        assert (lanes, elements, parts) == (8, 8, 1), case
        a = C.build(_lib.TaeLogprobsArgs, dtype=F.DTYPE[case[0]], rows=case[1], vocab=case[2], top=case[3])
        assert _lib.load().tae_token_logprobs_workspace(ctypes.byref(a)) == 0, case
