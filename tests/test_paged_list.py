"""The list of tiles that attention over a paged cache deals to its CTAs: its limits, compiled by the host compiler or read from the sources. Runs without a GPU."""
import os
import re
import subprocess

import pytest

import helpers

CSRC = os.path.join(helpers.PKG_DIR, "csrc")


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """Compiles C++ lines that print one number each, and returns those."""
    def run(lines):
        folder = tmp_path_factory.mktemp("list")
        (folder / "ask.cpp").write_text('#include <cstdio>\n#include "%s"\nint main() {\n%s\n}\n' % (os.path.join(CSRC, "paged_list.cuh"), "\n".join(lines)))
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-o", str(folder / "ask"), str(folder / "ask.cpp")], check=True)
        return [int(x) for x in subprocess.run([str(folder / "ask")], check=True, capture_output=True, text=True).stdout.split()]
    return run


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


# CTAs per SM and warps of a CTA, as the kernels' launches have them: heads of 64 and of 128 on tiles, lanes of four, two and one warp
FORMS = [(3, 4), (2, 4), (2, 2), (2, 1)]


@pytest.mark.parametrize("per_sm,warps", FORMS)
def test_a_join_takes_the_parts_of_all_ctas(ask, per_sm, warps):
    """One long row of one kv head has a part of every warp of every CTA, whatever the device."""
    sms = [1, 2, 132, 148, 149, 150, 160, 264, 1000, 100000]
    most, *ctas = ask(['printf("%u\\n", PAGED_PARTS_MOST);'] + [f'printf("%u\\n", paged_list_ctas({n}, {per_sm}, {warps}));' for n in sms])
    for n, c in zip(sms, ctas):
        assert 0 < c * warps <= most and c <= n * per_sm, n
        assert c == n * per_sm or n >= 150, "all CTAs that are resident, where the join takes them"


def test_ctas_of_a_list_are_never_more():
    """Every number of CTAs goes through that limit, and the join has room for it."""
    tiles, lanes = source("attention_paged.cu"), source("attention_paged_lanes.cu")
    assert re.findall(r"\bctas = ([^;]*);", tiles) == [
        "by_lanes ? lanes.ctas : paged_list_ctas((uint32_t)ctx->sm_count, hd == 64u ? TilesCfg<64, false>::CTAS : TilesCfg<128, false>::CTAS, TILES_WARPS)"]
    assert re.findall(r"\bctas = ([^;]*);", lanes) == ["paged_list_ctas((uint32_t)ctx->sm_count, 2u, out->warps)"]
    assert re.search(r"MOST = PAGED_PARTS_MOST\b", tiles) and "sw[MOST]" in tiles


def test_tiles_before_a_row_do_not_wrap():
    """32 rows of the most entries that a slot may have, in tiles of one warp's eight: their number takes 33 bits, and so does what is added up over a warp's lanes."""
    most = 1 << 30
    assert "> (1ull << 30)" in source("paged.cuh") and 32 * (most // 8) == 1 << 32
    make = source("attention_paged.cuh")
    make = make[make.index("void paged_list_make("):make.index("void paged_list_enter(")]
    added = re.findall(r"(\w+) (?:sum|u|before) =", make)
    assert len(added) == 3 and set(added) == {"uint64_t"}


def test_runs_are_counted_in_32_bits(ask):
    """The longest run of every list that is taken fits, and lists are refused only where it would not."""
    cases = [(rows, units, tiles, ctas) for rows in (1, 31, 32, 255, 256) for units in (1, 37, 512, 65535) for tiles in (1, 1 << 20, (1 << 27) - 1, 1 << 27)
             for ctas in (1, 148, 296, 444)]
    cases += [(1, 1, (1 << 27), 1), (256, 60, 1 << 27, 296), (256, 1, 1 << 24, 1), (256, 1, (1 << 24) - 1, 1)]
    got = ask([f'printf("%d\\n", paged_list_fits({r}u, {u}ull, {t}u, {c}u));' for r, u, t, c in cases])
    for (r, u, t, c), fits in zip(cases, got):
        assert fits == (-(-r * u * t // c) < 1 << 32), (r, u, t, c)
        assert fits or r * u * t * 8 >> 32 >= c * 8 - 8
    assert "!paged_list_fits(" in source("attention_paged.cu") and 0 < sum(got) < len(got)
