"""What the order of the 4-bit attention's copies and reads rests on, looked up in the source: no run shows it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-candle_b200", "csrc")


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name), encoding="utf-8").read())


def _between(src, begin, end):
    at = src.index(begin)
    return src[at:src.index(end, at)]


def test_the_lane_that_counts_a_stage_s_bytes_arrives_for_it():
    """An arrival by another lane could come in front of the expected bytes and end the phase with nothing copied: which lane elect.sync picks is not promised."""
    issue = _between(_source("fp4_decode.cuh"), "auto issue = [&](int stage)", "absent = (absent")
    whole, halves = issue.split("page_left -= 2;")
    assert "mbar_arrive_expect_tx" in whole                                     # one instruction for both
    assert "ptx::elect_one()" in halves and halves.count("elect_one") == 1      # one choice for the expected bytes, the copies and the arrival
    assert "lane == 0" not in halves
    assert re.search(r"if \(one\) \{\s*asm volatile\(\"mbarrier\.expect_tx", halves) and re.search(r"if \(one\) ptx::mbar_arrive\(stage_bar\)", halves)


def test_a_stage_is_read_in_front_of_its_release():
    """Shared loads that the compiler may move could come behind the warp's barrier, and so behind the copies that fill their stage again."""
    loads = re.findall(r"asm[^;]*?ld\.shared[^;]*;[^;]*;", _source("fp4_decode.cuh"))
    assert len(loads) == 4 and all(x.startswith("asm volatile(") and re.search(r":\s*\"memory\"\);$", x) for x in loads), loads
