"""What the sources of kernels that may start before the kernel ahead of them has finished have to keep to.

Such a kernel (programmatic dependent launch) is resident while the kernel ahead still writes its inputs. So it reads none of them through
the read-only path, whose data nobody may write while the kernel runs and whose loads the compiler may move above the wait, and none
of its warps begins a wait that has a limit before the kernel ahead has finished, which may take longer.
"""

import re

import pytest

from feather_ops_b200 import _build

SOURCES = ["fp8_block_mm_sm100.cu", "fp8_block_quantize_sm100.cu", "int8_mm_sm100.cu"]
WAITS = re.compile(r"\b(grid_dependency_wait|start_after_kernel_ahead)\(\)")


def without_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", "", re.sub(r"//[^\n]*", "", text), flags=re.S)


def closing(text: str, at: int) -> int:
    """The end of the bracket that opens at `at`."""
    pairs = {"(": ")", "{": "}"}
    depth = 0
    for i in range(at, len(text)):
        depth += {text[at]: 1, pairs[text[at]]: -1}.get(text[i], 0)
        if depth == 0:
            return i
    raise AssertionError("brackets do not match")


def kernels(name: str) -> dict[str, tuple[str, str]]:
    """Parameters and body of every kernel of a source file."""
    text = without_comments((_build.CSRC / name).read_text())
    found = {}
    for head in re.finditer(r"__global__\s+void\s+", text):
        at = head.end()
        while True:   # attributes with brackets of their own, then the name and its parameters
            word = re.compile(r"\s*(\w+)\s*\(").match(text, at)
            end = closing(text, word.end() - 1)
            if not word[1].startswith("__"):
                break
            at = end + 1
        body = text.index("{", end)
        found[word[1]] = text[word.end() : end], text[body : closing(text, body) + 1]
    return found


def dependents() -> list[tuple[str, str]]:
    return [(name, kernel) for name in SOURCES for kernel, (_, body) in kernels(name).items() if WAITS.search(body)]


def test_every_source_that_launches_programmatically_is_looked_at():
    launching = {p.name for p in _build.CSRC.glob("*.cu") if "cudaLaunchAttributeProgrammaticStreamSerialization" in p.read_text()}
    assert launching == set(SOURCES)
    assert {k for _, k in dependents()} == {
        "small_kernel", "pair_kernel", "tile_quantize_kernel", "silu_mul_dgrad_kernel", "rms_norm_fp8_kernel", "rms_norm_dgrad_few_kernel",
        "column_sum_kernel", "int8_mm_pair_kernel",
    }


@pytest.mark.parametrize("name,kernel", dependents())
def test_inputs_are_not_read_through_the_read_only_path(name, kernel):
    parameters, body = kernels(name)[kernel]
    assert not re.search(r"\bconst\b[^,]*__restrict__", parameters)
    assert "__ldg" not in body and "load16_readonly" not in body
    assert not re.search(r"load_weight<[^>]*\btrue>", body)
    # ... nor by what it calls
    text = without_comments((_build.CSRC / "fp8_block.cuh").read_text())
    load16 = re.search(r"\bload16\(const uint16_t\* p\)\s*(\{[^}]*\})", text)[1]
    assert "__ldg" not in load16


def waits_for_the_kernel_ahead_first(body: str, at: int) -> bool:
    """Whether the code on the way to `at` (the blocks that are open there, without those closed before) has the dependency wait."""
    way = [""]
    for c in body[:at]:
        if c == "{":
            way.append("")
        elif c == "}":
            way.pop()
        else:
            way[-1] += c
    return any(WAITS.search(part) for part in way)


@pytest.mark.parametrize("name,kernel", dependents())
def test_no_limited_wait_begins_before_the_kernel_ahead_has_finished(name, kernel):
    body = kernels(name)[kernel][1]
    waits = [m.start() for m in re.finditer(r"\b(guard\.wait|warp_wait)\(", body)]
    assert waits or not kernel.endswith(("small_kernel", "pair_kernel"))
    early = [body[at : at + 70] for at in waits if not waits_for_the_kernel_ahead_first(body, at)]
    assert not early
