"""Waits of the attention kernels have a time limit, after which a lane goes on without the data.
A phase can complete just as the limit passes, so that some lanes of a warp give up and others do
not.  They have to stay on one path as long as the warp executes anything together (TMEM loads and
stores, shuffles, __syncwarp): a lane that left its loop would leave the others waiting for it, and
the limit would not bound anything.  No wait is made to run out on a GPU; the sources say whether a
lane can leave."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "deepseek-v4-flash-sm120_b200", "csrc")
KERNELS = ["dense_attn_sm100.cu", "shared_prefix_sm100.cu"]


def source(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    # one lane alone loads in the dense kernel: it may stop (its block, up to the brace at its own indentation)
    return re.sub(r"\n( *)if \(elect_one\(\)\) \{\n.*?\n\1\}", "", text, flags=re.S)


@pytest.mark.parametrize("name", KERNELS)
def test_no_lane_leaves_a_loop_when_its_wait_gives_up(name):
    text = source(name)
    assert "gave_up(" in text and "mbar_wait_fast(" in text
    for m in re.finditer(r"gave_up\([A-Za-z_]+\);", text):
        rest = text[m.end():m.end() + 80].split("}")[0]
        assert not re.search(r"\b(break|return|continue)\b", rest), text[m.start() - 80:m.end() + 80]
    assert not re.search(r"if \(!ok\) (break|return)", text)
    for head in re.findall(r"for \(([^{]*?)\) ", text):
        assert not re.search(r"\bok\b", head), head
    for head in re.findall(r"while \(([^{]*?)\) \{", text):
        assert not re.search(r"\bok\b", head) or "__all_sync" in head, head


@pytest.mark.parametrize("name", KERNELS)
def test_every_wait_is_skipped_after_one_has_given_up(name):
    text = source(name)
    for m in re.finditer(r"!mbar_wait_fast\(", text):
        assert text[:m.start()].rstrip().endswith("ok &&"), text[m.start() - 60:m.end() + 60]


def test_a_lane_that_gave_up_reports_nothing_to_the_other_cta():
    """The leader's barriers count arrivals of both CTAs: one that no longer waits could arrive in the other's place."""
    text = source("shared_prefix_sm100.cu")
    calls = re.findall(r"if \(([^\n]*)\) arrive_leader\(", text)
    assert len(calls) == 3 and all(c == "lane == 0 && ok" for c in calls)
    assert len(re.findall(r"arrive_leader\(bar\(", text)) == 3


def test_a_cta_that_gave_up_makes_the_whole_cluster_s_result_nan():
    """Each CTA of a cluster writes columns of the merged row, and one of them its log-sum-exp."""
    body = re.search(r"void cluster_merge\(.*?\n\}", source("sparse_attn_sm100.cu"), re.S).group(0)
    assert re.search(r"const float lv = ctrl\.fail \? NAN : l_own;", body)
    assert "st_cluster_b32(map_to_rank(a_l, r), __float_as_uint(lv));" in body
