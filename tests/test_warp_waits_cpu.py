"""A lane that waits for a whole warp: a shuffle tells the other lanes that the wait is over but orders no memory, so they look at the barrier
too, or meet the first lane at a warp barrier, before they read what was waited for."""
import re

import pytest

import test_dependent_launches_cpu as rules

SOURCES = sorted(p for p in rules.CSRC.rglob("*") if p.suffix in (".cu", ".cuh") and re.search(r"__shfl_sync\(0xffffffffu, (ok|okw|there)\b", p.read_text()))


def broadcasts(text):
    """What follows each broadcast of a wait's outcome, as far as the end of its function or loop body's next twelve statements."""
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    for m in re.finditer(r"__shfl_sync\(0xffffffffu, (ok|okw|there), 0\)", code):
        rest, depth = code[m.end():], 0
        for i, c in enumerate(rest):
            depth += (c == "{") - (c == "}")
            if depth < 0:
                break
        yield code[max(0, m.start() - 160):m.end()], ";".join(rest[:i].split(";")[:12])


def reads_meet_first(text) -> bool:
    """Every read of tensor memory, the first thing that is read behind a wait, comes directly behind a warp barrier."""
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    return all(re.search(r"__syncwarp\(\);\s*$", code[:m.start()]) for m in re.finditer(r"tmem_ld_32x32\(", code))


def ordered(after: str) -> bool:
    at = re.search(r"mbar_wait\(|__syncwarp\(\)", after)
    use = re.search(r"tmem_ld|ld_stream|load_acc|return (?!false)", after)
    return at is not None and (use is None or at.start() < use.start())


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_every_lane_is_ordered_behind_the_wait(path):
    found = list(broadcasts(path.read_text()))
    assert found
    for before, after in found:
        assert ordered(after) or (path.name == "orthogonal_small.cu" and reads_meet_first(path.read_text())), before[-80:] + after[:200]


def test_the_rule_sees_what_it_is_for():
    assert len(SOURCES) >= 4
    for body, fine in (("return there != 0;", False), ("tc_fence(); __syncwarp(); return there != 0;", True), ("if (!x) return false; mbar_wait(b, p, t); return true;", True),
                       ("tmem_ld_32x32(a, r); __syncwarp();", False)):
        assert ordered(body) is fine
    assert reads_meet_first("__syncwarp();\n  tmem_ld_32x32(a, r);") and not reads_meet_first("f(); tmem_ld_32x32(a, r);")
