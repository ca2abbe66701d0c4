"""The order of the two programmatic-launch calls in the kernels, read from their source.

The fused decode step with HKV_APPEND_EARLY reads its cache before it has waited for the
grid before it. That is safe only if every grid further back has completed, so each kernel
that is launched with the programmatic attribute lets the next grid in after its own wait,
never before. (The kernels that do it the other way round are launched in plain order.)"""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hetero_kvcache_optimizer_b200", "csrc")


def sources():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            with open(os.path.join(CSRC, name)) as f:
                yield name, re.sub(r"//[^\n]*", "", f.read())


def body(text, at):
    """The braces that follow position `at`."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError("unbalanced braces")


def kernels():
    found = {}
    for _, text in sources():
        for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\s*\(", text):
            found[m.group(1)] = body(text, m.end())
    return found


def test_programmatic_launches_let_the_next_grid_in_after_their_own_wait():
    found = kernels()
    launched = {k for _, text in sources() for k in re.findall(r"launch_pdl\(\d+,\s*hkv::(\w+_kernel)", text)}
    assert {"decode_kernel", "quantize_pack_kernel", "append_kv_kernel", "norm_rope_kernel", "pages_fork_map_kernel"} <= launched
    for name in sorted(launched):
        calls = re.findall(r"griddep_(wait|launch_dependents)\(\)", found[name])
        assert calls and calls[0] == "wait", (name, calls)
        for i, c in enumerate(calls):
            if c == "launch_dependents":
                assert calls[i - 1] == "wait", (name, calls)
    for name, text in found.items():  # the others have no wait of their own to be ahead of
        if name not in launched:
            assert "griddep_wait()" not in text, name
