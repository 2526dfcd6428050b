"""Loads and stores of tensor memory are instructions of a whole warp: its lanes have to arrive together, and after a branch that depends
on the lane only a warp barrier (or a shuffle or vote of all lanes) says that they do.  Read off the kernel's source, since lanes that
do not meet leave the instruction undefined."""
import re
from pathlib import Path

KERNEL = Path(__file__).resolve().parents[1] / "aginfer_b200" / "csrc" / "kernels" / "paged_many.cuh"
LANES = r"if \([^{};]*\b(?:merges|is_live|stays|at|lane == 0|r == 0|row < live)\b|\? __ldcg|row < live \?"
TOGETHER = r"__syncwarp\(|__syncthreads\(|__shfl_sync\(|__any_sync\("
WHOLE_WARP = r"\btmem_load\w*\(|\btmem_store\w*\(|\"bar\.(?:sync|arrive)"
EVENTS = re.compile(f"(?P<lanes>{LANES})|(?P<together>{TOGETHER})|(?P<warp>{WHOLE_WARP})")


def body() -> str:
    source = re.sub(r"//[^\n]*", "", KERNEL.read_text())
    start = source.index("setmaxnreg.inc")
    return source[start:source.index("grid_dependency_only_wait();", source.index("note.pieces", start))]


def apart(text: str) -> list[str]:
    """Warp instructions that follow a branch by lanes with nothing between that brings the lanes together."""
    found, split = [], False
    for m in EVENTS.finditer(text):
        if m.lastgroup == "lanes":
            split = True
        elif m.lastgroup == "together":
            split = False
        elif split:
            end = text.find("\n", m.end())
            line = text[text.rfind("\n", 0, m.start()) + 1:len(text) if end < 0 else end].strip()
            found.append(line)
    return found


def test_the_lanes_meet_before_instructions_of_the_whole_warp():
    text = body()
    loop = text.index("for (unsigned c0")
    again = text[loop:text.index("tc::mbar_arrive(&o_empty", loop)]      # the output loop's second turn follows its first one
    assert "merges" in again and "is_live" in again and "tmem_load32" in again
    assert apart(text) == []
    assert apart(again + again) == []


def test_the_reading_sees_a_missing_barrier():
    assert apart("if (merges) { x = y; } tmem_load32(a, v);") == ["if (merges) { x = y; } tmem_load32(a, v);"]
    assert apart("if (merges) { x = y; } __syncwarp(); tmem_load32(a, v);") == []
