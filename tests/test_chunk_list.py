"""The chunk kernel's work list without a GPU: the code that lists a CTA's segments, run on the host for all CTAs."""
import subprocess
from pathlib import Path

import pytest

from q3s import build

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def listed(tmp_path_factory):
    exe = tmp_path_factory.mktemp("chunk_list") / "chunk_list"
    subprocess.run([build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", f"-I{HERE.parent / 'qwen3tts-streaming_b200' / 'csrc'}",
                    f"-I{build.INCLUDE}", "-o", str(exe), str(HERE / "chunk_list.cu")], check=True, capture_output=True)

    def run(seed, rows, active, new, own, heads, group, prefix=0, window=0):
        r = subprocess.run([str(exe), *map(str, (seed, rows, active, new, own, heads, group, prefix, window))], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout
        return dict(zip(("segments", "batches", "cuts", "operations"), map(int, r.stdout.split())))

    return run


@pytest.mark.parametrize("rows,active,new,own,heads,group,prefix,window", [
    (1, 1, 1, 0, 1, 1, 0, 0), (1, 1, 1, 0, 1, 1, 1, 0), (1, 1, 5, 700, 8, 2, 200, 0), (2, 1, 4096, 3500, 8, 2, 150, 0),
    (13, 1, 700, 3000, 4, 4, 0, 512), (48, 1, 9, 1500, 8, 4, 333, 0), (48, 3, 9, 1500, 8, 4, 333, 100), (3, 1, 90, 4000, 2, 5, 129, 1),
    (20, 2, 300, 500, 1, 128, 7, 64), (400, 5, 40, 300, 2, 3, 0, 0), (900, 1, 3, 100, 2, 1, 20, 0)])
def test_every_step_is_listed_once_and_its_parts_are_joined(listed, rows, active, new, own, heads, group, prefix, window):
    got = listed(rows, rows, active, new, own, heads, group, prefix, window)
    assert got["segments"] > 0


@pytest.mark.parametrize("rows,heads", [(600, 32), (300, 64)])
def test_cut_items_are_defined_after_every_batch_of_segments(listed, rows, heads):
    """A CTA whose waits give up lists no more segments: what it has written of its cut item by then is what the joining
    kernel reads, from a workspace that needs no initial value.  More segments a CTA than it lists at a time."""
    got = listed(rows, rows, 1, 3, 20, heads, 1)
    assert got["batches"] > 148 and got["segments"] > 64 * 148


@pytest.mark.parametrize("rows,active,new", [(8000, 0, 300), (8000, 500, 300), (60000, 0, 2000), (2000, 1999, 5)])
def test_rows_without_tokens_are_passed_over(listed, rows, active, new):
    """Rows behind the last with tokens cost a CTA nothing, rows between them an operation of its lanes for 32 rows, not the
    dozen that a row of its own takes: what a CTA does before its first copy goes by the rows that bring tokens."""
    got = listed(rows, rows, active, new, 2000, 8, 2)
    ranges = 1 if active == 0 else -(-rows // active)  # rows with tokens
    assert got["operations"] <= 100 + 40 * ranges + (0 if active == 0 else rows // 32 + 2 * ranges)
