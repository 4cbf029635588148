"""CPU: from how many rows on a sequence takes the tensor map of a long tensor is found in the driver's own maps; a layout of them that is not
understood ends the call with an error, and does not get lengths put into it."""
import os
import subprocess

import pytest

from conftest import ROOT

FOUND, NOT_ENCODED, NOT_UNDERSTOOD = range(3)
ONE_BIT, NO_BORDER, TWO_BORDERS, ROWS_TWICE, TWO_WORDS, NO_ENCODER = 0, 1, 2, 3, 4, 5


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("map_kind") / "driver")
    src = os.path.join(ROOT, "tests", "cxx", "map_kind_driver.cpp")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", src, "-o", out], check=True)

    def run(layout, rows, border=0, guess=0):
        r = subprocess.run([out, *map(str, (layout, rows, border, guess))], capture_output=True, text=True)
        assert r.returncode == 0, r
        return tuple(map(int, r.stdout.split()))
    return run


@pytest.mark.parametrize("layout", [ONE_BIT, TWO_WORDS])
@pytest.mark.parametrize("rows,border", [(2, 2), (3, 2), (3, 3), (500, 64), (500, 500), (500, 2), (2 ** 31 - 1, 2 ** 30 + 7)])
def test_the_border_is_found(driver, layout, rows, border):
    assert driver(layout, rows, border, border) == (FOUND, border, 2)  # as a rule: two maps
    for guess in (1, border - 1, border + 1, rows + 1, 2 ** 40):
        found, n, calls = driver(layout, rows, border, guess)
        assert (found, n) == (FOUND, border) and calls <= 31 + 4


@pytest.mark.parametrize("rows", [1, 2, 500])
def test_one_kind_of_map(driver, rows):
    assert driver(NO_BORDER, rows, 0, 64) == (FOUND, 1, 0)
    assert driver(ONE_BIT, rows, rows + 1, rows + 1) == (FOUND, 1, 0)  # a tensor that is not long


@pytest.mark.parametrize("guess", [1, 64, 500, 501])
def test_what_is_not_understood(driver, guess):
    """More than one border, or the rows in more than one word: every length would look like a kind of its own."""
    assert driver(TWO_BORDERS, 500, 64, guess)[0] == NOT_UNDERSTOOD
    found, _, calls = driver(ROWS_TWICE, 500, 0, guess)
    assert found == NOT_UNDERSTOOD and calls <= 31 + 4
    assert driver(ROWS_TWICE, 3, 0, guess)[0] == NOT_UNDERSTOOD
    assert driver(ROWS_TWICE, 2, 0, guess)[:2] == (FOUND, 2)  # (its two lengths have maps of their own)


def test_a_driver_that_refuses(driver):
    assert driver(NO_ENCODER, 500, 0, 64)[0] == NOT_ENCODED
