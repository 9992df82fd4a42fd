"""Rules for the sources of the long-context operators, all of whose kernels are launched as programmatic dependents: every one waits for
the grids before it once, where every thread comes by, and touches nothing that they may have written, or that they may still read,
before.  Each rule is shown to fail on sources that break it."""
import re

import pytest

import test_dependent_launches_cpu as rules

SOURCES = {p.name: re.sub(r"//[^\n]*|/\*.*?\*/", "", p.read_text(), flags=re.S)
           for p in (rules.CSRC / "ops" / n for n in ("rotary.cu", "distill.cu", "window_decode.cu", "window_attention.cu"))}
# what reads or writes memory of the GPU, by name
ACCESS = re.compile(r"\b(?:copy16|cp_async16|hold|fetch|load_tile|load_half|bulk_g2s|tma_load\w*|ld_stream|__ld\w+|__st\w+|atomic\w+|"
                    r"read_entries|window_bwd_run|warp_store_box)\s*(?:<[^>;]*>)?\(|cp\.async|\b(?:ld|st|red|atom)\.global")


def uncalled(code):
    """``code`` without the bodies of its lambdas, which run where they are called."""
    out, at = "", 0
    for m in re.finditer(r"\[&?\]\s*\([^()]*\)\s*(?:->\s*\w+\s*)?\{", code):
        if m.start() >= at:
            out += code[at:m.start()]
            at = rules._matching(code, m.end() - 1, "{}") + 1
    return out + code[at:]


def problems(text):
    kernels = rules.functions(text, "__global__")
    found = [] if kernels else ["no kernel"]
    if "<<<" in text or re.search(r"cudaLaunchKernel\w*\(", text):
        found.append("a plain launch")
    if not re.search(r"\blaunch_dependent(_clusters)?\(", text):
        found.append("no dependent launch")
    for name, (_, body) in kernels.items():
        tops = []
        for m in re.finditer(r"grid_wait\(\);", body):
            before = body[:m.start()]
            if re.search(r"[;{}]\s*$", before) and before.count("{") - before.count("}") == 1:
                tops.append(before)
        if len(tops) != 1:
            found.append(f"{name}: {len(tops)} waits that every thread comes to")
            continue
        early = uncalled(tops[0])
        if re.search(r"\breturn\b", re.sub(r"grid_wait\(\);[^{}]*return;", "", early)):
            found.append(f"{name}: leaves without a wait")
        if ACCESS.search(early):
            found.append(f"{name}: {ACCESS.search(early).group(0)} before the wait")
        # pointers of the arguments, and pointers made of them, that are looked into
        made = re.findall(r"\*\s*(\w+)\s*=\s*[^;]*?\b\w+\.\w+", early)
        for p in [r"\b\w+\.\w+"] + [r"\b" + v for v in made]:
            hit = re.search(p + r"\s*\[|(?<=[=(,;{}!])\s*\*\s*" + p + r"\b|(?<=[=(,;{}!])\s*\*\s*reinterpret_cast<[^()]*>\(\s*" + p, early)
            if hit:
                found.append(f"{name}: {hit.group(0).strip()} before the wait")
    return found


@pytest.mark.parametrize("name", SOURCES)
def test_sources_follow_the_rules(name):
    assert problems(SOURCES[name]) == []


KERNELS = [(n, k) for n, t in SOURCES.items() for k in rules.functions(t, "__global__")]


def mutated(name, kernel, change):
    text = SOURCES[name]
    body = rules.functions(text, "__global__")[kernel][1]
    assert text.count(body) == 1
    return text.replace(body, change(body))


def test_every_kernel_is_known():
    assert {k for _, k in KERNELS} >= {"rotary_kernel", "distill_row_kernel", "distill_partial_kernel", "distill_grad_kernel", "window_decode_kernel",
                                       "window_fwd_kernel", "window_delta_kernel", "window_rows_kernel", "window_parts_kernel",
                                       "window_bwd_kernel"}


def _at_top(body):
    """Where the wait is that every thread comes to."""
    return next(m.start() for m in re.finditer(r"grid_wait\(\);", body)
                if body[:m.start()].count("{") - body[:m.start()].count("}") == 1)


CHANGES = {
    "no wait": lambda b, w: b[:w] + b[w + len("grid_wait();"):],
    "a wait of some": lambda b, w: b[:w] + "if (threadIdx.x == 0) " + b[w:],
    "a wait inside a block": lambda b, w: b[:w] + "{ grid_wait(); }" + b[w + len("grid_wait();"):],
    "two waits": lambda b, w: b[:w] + "grid_wait(); " + b[w:],
    "an argument's element": lambda b, w: b[:w] + "const auto early = a.positions[0]; " + b[w:],
    "an element of a pointer": lambda b, w: b[:w] + "const float* early = a.stats + 3; const float e0 = early[1]; " + b[w:],
    "what a pointer points to": lambda b, w: b[:w] + "const float* early = a.stats + 3; const float e0 = *early; " + b[w:],
    "what a cast points to": lambda b, w: b[:w] + "const uint4 early = *reinterpret_cast<const uint4*>(a.qkv); " + b[w:],
    "a copy": lambda b, w: b[:w] + "copy16(0u, nullptr, true); " + b[w:],
    "a helper that reads": lambda b, w: b[:w] + "Held early = hold(a, 0); " + b[w:],
    "a tile": lambda b, w: b[:w] + "load_tile(sQ, &tm_qkv, q_full, 0, 0, 0); " + b[w:],
    "a coherent load": lambda b, w: b[:w] + "const auto early = __ldcg(p); " + b[w:],
    "leaving": lambda b, w: b[:w] + "if (blockIdx.x > 3) return; " + b[w:],
}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("name,kernel", KERNELS)
def test_rules_can_fail(name, kernel, change):
    assert any(kernel in p for p in problems(mutated(name, kernel, lambda b: CHANGES[change](b, _at_top(b)))))


def test_launch_rules_can_fail():
    text = SOURCES["rotary.cu"]
    assert problems(text.replace("return launch_dependent(kernel", "kernel<<<1, 1>>>(w); return launch_dependent(kernel")) == ["a plain launch"]
    assert problems(text.replace("launch_dependent(", "launched(")) == ["no dependent launch"]
