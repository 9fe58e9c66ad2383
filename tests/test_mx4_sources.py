"""The rules of test_kernel_sources.py for the kernels on 4-bit values, whose bodies are functions of headers."""

import re

import pytest

from test_kernel_sources import CSRC, roles

HEADERS = {"mx4_gemm.h": "product_block", "mx4_few.h": "few_block", "mx4_pair.h": "pair_block"}


def block(header):
    text = re.sub(r"//[^\n]*", "", (CSRC / header).read_text())
    body = text[text.index(f"void {HEADERS[header]}("):]
    return body[:body.index("\n}\n")]


def test_every_kernel_with_tensor_memory_is_known():
    found = {p.name for p in CSRC.glob("mx4*") if "tmem_alloc" in p.read_text()}
    assert found == set(HEADERS)


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_successors_start_behind_the_allocation(header):
    body = block(header)
    assert body.count("chain_release();") == 1
    assert re.search(r"if \(warp == \d\) \{\s*tmem_alloc(_pair)?\([^;]*;\s*chain_release\(\);\s*\}", body)
    assert body.count("tmem_dealloc") == 1


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_lanes_leave_a_loop_together(header):
    for role in roles(block(header)):
        if not re.search(r"mbar_wait\w*\(", role):
            continue
        together = re.search(r"elect_one|tmem_ld|store_unit|store_rows|_sync\(0xffffffffu|__syncwarp", role)
        if together and "lane == 0) {\n" not in role[:250]:
            assert not re.search(r"mbar_wait(_cluster)?\(", role), "a wait that each lane judges by itself"


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_copies_land_before_the_block_ends(header):
    parts = re.split(r"\n    (?:if|\} else if) \(warp ", block(header))
    role = next(r for r in parts if re.search(r"tma_load_[23]d", r))
    behind = role[max(m.end() for m in re.finditer(r"(tma_load_[23]d\w*|load_weights|load_rows)\(", role)):]
    assert re.search(r"for \(int \w+ = [^;]*;[^)]*\)\s*if \(!mbar_wait\w*\([^;]*full[^;]*timed_out = true;", behind)


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_bounded_waits_begin_behind_the_kernel_before(header):
    """A wait's time does not run while the kernel in front, however long it takes, still does."""
    common, *parts = re.split(r"\n    (?:if|\} else if|\} else) (?:\(warp == [01]\) )?\{\n", block(header))
    if re.search(r"\n    chain_wait\(\);", block(header).split("// ----")[0].split("bool timed_out")[0]):
        return
    waiting = [p for p in parts if "mbar_wait" in p]
    assert len(waiting) == 3
    for part in waiting:
        assert "chain_wait();" in part and part.index("chain_wait();") < part.index("mbar_wait")


def test_every_wait_is_bounded():
    for p in CSRC.glob("mx4*"):
        text = re.sub(r"//[^\n]*", "", p.read_text())
        assert not re.search(r"while \(!?\s*mbar_|for \(;;\)|__nanosleep", text), p.name
        assert "multicast::cluster" not in text, p.name


def test_long_quantisations_release_nobody_early():
    """A kernel whose blocks come in several rounds lets its successors start only at its end: those with tensor memory and
    clusters would else take SMs one by one while its last round drains."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "mx4.cu").read_text())
    releases = re.findall(r"[^;{}]*chain_release\(\);", text)
    assert len(releases) == 2 and all("if (tasks.at_once)" in r for r in releases)
    assert len(re.findall(r"__launch_bounds__\(256, (?:2 \* )?RESIDENT\)\s*mx4_(?:quantize|values)_kernel", text)) == 2
    assert re.search(r"tasks = \{[^;]*blocks <= RESIDENT \* \(unsigned\)sm_count\(\)\};", text)
