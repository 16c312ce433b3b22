"""The cached attention's waits, in its source: a wait that can give up is taken by a
warp as a whole (ac_wait votes on its lanes' verdicts).  A lane that left its
steps alone could not be shown on a GPU without risking the hang it would cause."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_lane_gives_up_a_wait_alone():
    text = open(os.path.join(ROOT, "glassboxai-transformer_b200", "csrc", "attn_cached.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    vote = re.search(r"bool ac_wait\([^)]*\)\s*\{\s*return __all_sync\(0xffffffffu, tc::mbar_wait\(bar, parity, abort, limit_ns\)\);\s*\}", text)
    assert vote
    rest = text[:vote.start()] + text[vote.end():]
    alone = re.findall(r"tc::mbar_wait\(.*", rest)
    # what is left waits for copies that are in flight and has no verdict
    assert len(alone) == 2 and all("nullptr, kDeviceWaitNs);" in x for x in alone), alone
    assert len(re.findall(r"\bac_wait\(", rest)) == 5
