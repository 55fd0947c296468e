"""What a page plan says of the pages that it lacks: d_missing is, step by step, the number of pages that a sequence's new
tokens lie in and have no entry for.  CPU only: the index rule and the plain form."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import long_context as L

ROOT = Path(__file__).resolve().parents[1]


def test_index_rule(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "plan_lacks"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "plan_lacks.cpp"), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def lost(plan, S, page):
    """Pages of each sequence's rows without a slot."""
    got = np.zeros(S, np.int64)
    for s in range(S):
        rows = (plan["sequences"] == s) & (plan["slots"] < 0)
        got[s] = len(set(plan["positions"][rows] // page))
    return got


def test_missing_is_what_the_rows_lack():
    rng = np.random.default_rng(1)
    S, width, page, count = 6, 9, 16, 40
    pages, lengths = np.full((S, width), -1, np.int32), np.zeros(S, np.int64)
    free, free_count = rng.permutation(count).astype(np.int32), count
    kinds = set()
    for step in range(200):
        new = None if step % 3 else rng.integers(0, 60, S) * (rng.random(S) < 0.5)
        keep = np.where(rng.random(S) < 0.04, -1, 0)
        if step % 20 == 7:  # some entries come to name nothing
            pages[rng.random(pages.shape) < 0.1] = -1
        before = np.where(keep < 0, 0, lengths)
        got = L.plan(pages, lengths, new, keep, free, free_count, page, count, 400)
        assert np.array_equal(got["missing"], lost(got, S, page))
        for s in np.flatnonzero(got["missing"]):
            kinds.add(("begun", before[s] % page != 0 and got["pages"][s, min(before[s] // page, width - 1)] < 0))
            kinds.add(("beyond", got["lengths"][s] > width * page))
        pages, lengths, free, free_count = got["pages"], got["lengths"], got["free"], got["free_count"]
    assert kinds == {(k, b) for k in ("begun", "beyond") for b in (False, True)}


def test_a_shortage_is_told_until_the_page_is_passed():
    """A token that opens a page and finds none: the other fifteen are dropped too, whatever comes free meanwhile."""
    pages, lengths = np.array([[0, -1, -1]], np.int32), np.array([16])
    free, free_count = np.array([2, 1, -1], np.int32), 0
    told = []
    for step in range(20):
        got = L.plan(pages, lengths, None, None, free, free_count, 16, 3, 1)
        told.append((int(got["missing"][0]), int(got["slots"][0]) < 0))
        pages, lengths, free_count = got["pages"], got["lengths"], 2 if step >= 5 else 0
    assert told == [(1, True)] * 16 + [(0, False)] * 4
