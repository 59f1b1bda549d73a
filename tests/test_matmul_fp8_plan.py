"""The planner of the 8-bit products (gsp_matmul_fp8_plan.cpp, plain C++), built with g++ and asked on the host."""
import subprocess
from pathlib import Path

import pytest

from fp8_forms import CUS, PIECES, STREAM32, STREAMS, TILES

NATIVE = Path(__file__).resolve().parent / "native"


@pytest.fixture(scope="module")
def plan():
    subprocess.run(["make", "-C", str(NATIVE), "_build/matmul_fp8_plan"], check=True, capture_output=True, text=True)

    def ask(sizes, aligned, cus=CUS):
        lines = "".join(f"{i} {o} {b} {int(aligned and i % 256 == 0)} {cus}\n" for i, o, b in sizes)
        out = subprocess.run([str(NATIVE / "_build" / "matmul_fp8_plan")], input=lines, check=True, capture_output=True,
                             text=True).stdout.split("\n")[:-1]
        assert len(out) == len(sizes)
        rows = [r.split() for r in out]
        return [(r[0], *(int(v) for v in r[1:])) for r in rows]  # form, ranges, units of a range, waves, bytes

    return ask


@pytest.mark.parametrize("aligned", [True, False])
def test_sizes_reach_their_forms(plan, aligned):
    cases = TILES + PIECES + (STREAM32 if aligned else STREAMS)
    got = plan([c[:3] for c in cases], aligned)
    assert [(c, g[:3]) for c, g in zip(cases, got) if g[:3] != c[3:]] == []


def test_every_form_is_reached(plan):
    """Each tile form: whole K, an odd first unit behind the first range, a last range shorter than the others, and K that
    ends inside a unit; ragged rows and outputs."""
    for form in ("wide", "tile64", "tile32"):
        mine = [c for c in TILES if c[3] == form]
        units = {c: c[0] // 256 + (c[0] % 256 != 0) for c in mine}
        assert any(c[4] == 1 for c in mine) and any(c[4] > 1 and c[5] % 2 for c in mine)
        assert any(c[4] * c[5] > units[c] for c in mine) and any(c[0] % 256 for c in mine)
        assert any(c[0] % 256 == 0 and c[4] > 1 for c in mine)
    assert {g[3] for g in plan([c[:3] for c in STREAM32], True)} == {4, 8}


def test_ranges_cover_k(plan):
    """Over many sizes: every range has a unit, and together they are K."""
    sizes = [(64 * i, o, b) for i in (1, 3, 4, 5, 14, 41, 56, 76, 296, 2048) for o in (1, 130, 896, 3584, 18944, 100000)
             for b in (1, 17, 64, 65, 128, 200, 512, 1300, 9000)]
    for (i, o, b), (form, ranges, per, waves, _) in zip(sizes, plan(sizes, True)):
        units = i // 256 + (i % 256 != 0)
        assert ranges >= 1 and (ranges - 1) * per < units <= ranges * per
        assert (form == "stream32") == (waves > 0)
        assert ranges == 1 or b > 64  # a first call of up to 64 rows may be captured: no workspace


def test_converted_activations_stay_within_a_gigabyte(plan):
    """Whatever K is: where one workgroup's 128 rows alone would pass it, another form is taken."""
    ks = [64, 3584, 18944, 131072, 1 << 20, 3947520, 3947584, 1 << 22, 1 << 23, (1 << 24) - 64, 1 << 24]
    sizes = [(k, o, b) for k in ks for o in (64, 1000, 4096, 100000) for b in (65, 128, 129, 1024, 4097, 100000)]
    got = plan(sizes, True)
    assert max(g[4] for g in got) <= 1 << 30
    assert all(g[4] == 0 and g[0] != "wide" for s, g in zip(sizes, got) if s[0] > 3947520)
    assert any(g[0] == "wide" and g[4] > 1 << 29 for s, g in zip(sizes, got) if s[0] <= 3947520)


def test_pieces_are_pieces(plan):
    for (k, _, batch, *_), got in zip(PIECES, plan([c[:3] for c in PIECES], True)):
        assert got[4] == 896 // 32 * 2048 * (16384 + 1024) and batch > 896
