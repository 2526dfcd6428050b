"""The many-row kernel's schedule keeps 16 bytes a sequence in dynamic shared memory, in front of what goes there later.  With 64-wide heads
the sequences that the builder accepts reach past the queries into the ring of keys, which bulk copies (another proxy) then write: a
proxy fence has to stand between.  Read off the source, since a race on shared memory must not be run."""
import re
from pathlib import Path

from aginfer_b200.recipes.builder import PAGED_MAX_SEQUENCES, PagedCache, paged_many_tiling
from aginfer_b200.recipes import Arena

KERNEL = Path(__file__).resolve().parents[1] / "aginfer_b200" / "csrc" / "kernels" / "paged_many.cuh"


def test_every_thread_fences_the_schedules_memory_before_copies_go_there():
    source = re.sub(r"//[^\n]*", "", KERNEL.read_text())
    written, read = source.index("places[i] = "), source.rindex("places[seq]")
    handed_on = source.index("auto give_up", read)          # the roles begin behind it
    between = source[read:handed_on]
    assert written < read and re.search(r"(\bif \(!kPrefix\) )?tc::fence_async_shared\(\);\s*__syncthreads\(\);", between)


def test_the_schedule_fits_where_it_is_kept():
    at = Arena(0)
    for d in (64, 128):
        cache = PagedCache(k=at, v=at, table=at, lengths=at, starts=at, sequences=PAGED_MAX_SEQUENCES, pages=1, page=16, pages_per_sequence=1,
                           kv_heads=1, head_dim=d)
        queries, ring = 2 * 128 * d * 2, paged_many_tiling(cache, 1, 16)["shared_bytes"] - 1024 - 20480
        assert 16 * PAGED_MAX_SEQUENCES <= ring
        assert d == 128 or 16 * PAGED_MAX_SEQUENCES > queries      # what the fence is there for
