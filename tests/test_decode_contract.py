"""What the decode step's operators promise about order, resources and reports,
as far as it can be checked without a GPU."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen3tts-streaming_b200" / "csrc"


def kernel_bodies(name):
    """{kernel: body} of the __global__ functions of a source file, comments removed."""
    text = re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S))
    out = {}
    for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\(", text):
        start = text.index("{", m.end())
        depth, i = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        out[m.group(1)] = text[start:i]
    return out


@pytest.mark.parametrize("kernel", ["quantize_rows_kernel", "quantize_warps_kernel", "int8_gemv_kernel", "int8_split_kernel",
                                    "int8_pair_kernel"])
def test_8_bit_kernels_read_no_operand_before_they_wait(kernel):
    """Rows, scales and weights may all have been written by the kernel before."""
    body = kernel_bodies("q3s_int8.cuh")[kernel]
    before = body[:body.index("grid_wait()")]
    assert not re.search(r"ld_stream16|tma_load|reinterpret_cast<const|a_scales|w_scales|bias", before), before
