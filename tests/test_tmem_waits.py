"""CPU: a TMEM load is asynchronous and its results are plain registers to the compiler.  Arithmetic on them is only kept
behind the wait if the wait names them, so every load of the ragged attention is followed by one that does, before
anything else touches its registers."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferno_b200", "csrc")


def test_every_tmem_load_is_awaited_by_name():
    lines = [s.strip() for s in open(os.path.join(CSRC, "ragged_attention.cu"))]
    loads = [(i, re.match(r"tmem_ld\w+\(.*, (\w+)(?: \+ \d+)?\);$", s)) for i, s in enumerate(lines) if re.match(r"tmem_ld\w*\(", s)]
    assert len(loads) >= 12
    for i, m in loads:
        assert m, lines[i]
        waited = next(s for s in lines[i + 1:] if s.startswith("tc_wait_ld"))
        assert re.match(rf"tc_wait_ld(32|64)\({m.group(1)}\);$", waited), f"line {i + 1}: {lines[i]} ... {waited}"
