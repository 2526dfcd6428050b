"""Named barriers and loads of tensor memory are instructions of a whole warp (bar.sync and bar.arrive are the aligned forms): the lanes have to
arrive together, and behind a branch or loop of single lanes only a warp barrier says that they do.  Read off the sources, since lanes that do
not meet leave the instruction undefined."""
import re
from pathlib import Path

import pytest

KERNELS = Path(__file__).resolve().parents[1] / "aginfer_b200" / "csrc" / "kernels"
WHOLE_WARP = r'asm volatile\("bar\.(?:sync|arrive)|(?<!void )\btmem_load\w*\('
# whole warps get there by branches on the warp alone, straight from the barrier in front
UNIFORM = r"(?:__syncwarp\(\);\s*|__syncwarp\(\);\s*if \(warp == kMmaWarp\) \{\s*|__syncwarp\(\);\s*if \(warp == kMmaWarp\) \{[^{}]*\} else \{\s*)$"


def apart(source: str) -> list[str]:
    """Instructions of whole warps that no warp barrier stands directly in front of."""
    text = re.sub(r"//[^\n]*", "", source)
    return [text[m.start():text.find("\n", m.start())].strip() for m in re.finditer(WHOLE_WARP, text)
            if not re.search(UNIFORM, text[:m.start()])]


@pytest.mark.parametrize("name", ["gemm_w4.cuh", "gemm_tk.cuh", "paged_few.cuh"])
def test_the_lanes_meet_before_instructions_of_the_whole_warp(name):
    text = (KERNELS / name).read_text()
    assert re.search(WHOLE_WARP, text) and apart(text) == []


def test_the_reading_sees_a_missing_barrier():
    bar = 'asm volatile("bar.sync 1, 128;" ::: "memory");'
    assert apart(f"if (lane == 0) ask(s);\n{bar}\n") == [bar]
    assert apart(f"if (lane == 0) ask(s);\n__syncwarp();  // together\n{bar}\n") == []
    assert apart("if (row < rows) store();\ntmem_load16_nowait(a, r);\n") == ["tmem_load16_nowait(a, r);"]
