"""CPU: what the build makes again when something that it is made of changes (make is asked, nothing is compiled)."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dualvgr-videoqa_amd", "csrc")


def would_compile(changed):
    out = subprocess.run(["make", "-n", "-W", changed], cwd=CSRC, capture_output=True, text=True, check=True).stdout
    return set(re.findall(r"-c (\w+\.hip)", out)), "dvgr_torch.cpp" in out


def test_new_flags_reach_every_object():
    objects, nodes = would_compile("Makefile")
    assert objects == {f for f in os.listdir(CSRC) if f.endswith(".hip")} and nodes


def test_shared_headers_reach_their_objects():
    assert {"dvgr_attn.hip", "dvgr_attn_bwd.hip", "dvgr_embed.hip", "dvgr_distill.hip"} <= would_compile("dvgr_elem.h")[0]
    assert {"dvgr_attn.hip", "dvgr_attn_bwd.hip"} <= would_compile("dvgr_attn_few.h")[0]
    objects, nodes = would_compile("../../include/dvgr_attn.h")
    assert {"dvgr_attn.hip", "dvgr_attn_bwd.hip"} <= objects and nodes
