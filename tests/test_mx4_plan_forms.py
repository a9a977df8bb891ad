"""The shapes of test_gpu_mx4_forms.py take every form that a product of mx4 rows has, and the limits that the header states are the
plan's; no GPU."""
import os
import re

import test_gpu_mx4_forms as forms
from test_mx4_plan import BATCH, ROWS, TILES, form, plan  # noqa: F401  (plan: a fixture)


def held_deep(m, k, words):
    """Whether a ring of three turns of four steps leaves room for the rows of x (linear_mx4_rows.hip)."""
    blocks = k // 32
    turn = 4 * 1024 + (256 if words else 4 * 256)
    return m * (blocks * 16 + 16 + (blocks + 15) // 16 * 16) <= 160 * 1024 - 8 * 3 * turn - 2 * 8 * 1024


def test_few_rows_have_every_turn_and_ring(plan):  # noqa: F811
    seen = set()
    for m, n, k in forms.ROWS:
        assert form(plan, m, n, k)[0] == ROWS and n % 2 == 0
        steps, words = (k + 127) // 128, k % 128 == 0
        seen.add((4 if steps > 16 else 2 if steps > 8 else 1, steps <= 16 or held_deep(m, k, words), words))
    assert seen == {(u, deep, words) for u in (1, 2, 4) for deep in (True, False) for words in (True, False) if deep or u == 4}
    assert any(n > 16 * 256 for _, n, _ in forms.ROWS)      # several pieces a workgroup


def test_batches_have_both_sizes(plan):  # noqa: F811
    seen = {(m <= 32, k % 128 == 0) for m, n, k in forms.BATCH}
    assert all(form(plan, *shape)[0] == BATCH and shape[1] % 2 == 0 for shape in forms.BATCH)
    assert len(seen) == 4 and {m <= 32 for m, n, _ in forms.BATCH if n > 16 * 256} == {True, False}


def test_tiles_have_every_size_depth_and_share(plan):  # noqa: F811
    seen = set()
    for m, n, k in forms.TILES:
        kernel, rows, parts, deep, whole = form(plan, m, n, k)
        assert kernel == TILES and n % 2 == 0
        share = "none" if parts == 1 else f"last of {parts}" if whole else "all"
        several = "one run" if k <= 512 else "runs"
        seen.add((rows, bool(deep), share, several, k % 128 == 0))
    for words in (True, False):
        want = {(rows, deep, "none", runs, words) for rows, deep in ((64, True), (64, False), (128, True), (128, False), (256, False))
                for runs in ("one run", "runs")} - {(64, False, "none", "one run", words), (128, False, "none", "one run", words)}
        want |= {(rows, rows < 256, "all", "runs", words) for rows in (64, 128, 256)}
        want |= {(128, False, f"last of {parts}", "runs", words) for parts in (2, 3)}
        assert want <= {s for s in seen if s[-1] == words}, want - seen


def test_the_published_limits_of_few_rows(plan):  # noqa: F811
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "karume_hip.h")).read()
    sixteen, one = map(int, re.search(r"16 of k = (\d+), one of (\d+)\)", text).groups())
    assert plan.fits(16, sixteen) and not plan.fits(16, sixteen + 32) and not plan.fits(17, 32)
    assert plan.fits(1, one) and not plan.fits(1, one + 32)
