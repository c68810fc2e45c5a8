"""What the decode step's operators promise about order, resources and reports,
as far as it can be checked without a GPU."""
import re
import subprocess
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


TENSOR_MEMORY_PROGRAM = r"""
#include <cstdio>
#include <set>
#include <utility>
#include "q3s_attn_prefix.cuh"
#include "q3s_int8.cuh"
int main() {
  std::set<std::pair<int, int>> cuts;  // the cluster product's shared memory and columns, over its range of shapes
  for (int M : {1, 2, 9, 16, 31, 32, 33, 64, 65, 96, 97, 128, 129, 160, 161, 192, 200, 224, 225, 256, 257, 300, 400, 513, 1000, 3000, 9400})
    for (int N : {1, 128, 257, 1000, 2048, 5000, 9000, 18000})
      for (int K : {16, 128, 144, 256, 272, 512, 528, 1024, 2048, 4096, 6144, 16384, 131056}) {
        const q3s::I8Cut c = q3s::int8_cut(M, N, K, 148);
        cuts.insert({c.smem, c.tmem});
      }
  for (const auto& c : cuts) printf("split %d %d\n", c.first, c.second);
  printf("pair %d 512\n", q3s::I8P_SMEM);
  printf("prefix %d 512\nprefix %d 512\n", q3s::PrefixTile<64>::SMEM, q3s::PrefixTile<128>::SMEM);
  printf("head %d %d\n", q3s::HeadTile<4, 64>::SMEM_BYTES, q3s::HeadTile<4, 64>::TMEM_COLS);
  printf("head %d %d\n", q3s::HeadTile<4, 96>::SMEM_BYTES, q3s::HeadTile<4, 96>::TMEM_COLS);
  printf("head %d %d\n", q3s::HeadTile<4, 128>::SMEM_BYTES, q3s::HeadTile<4, 128>::TMEM_COLS);
  printf("head %d %d\n", q3s::HeadTile<8, 128>::SMEM_BYTES, q3s::HeadTile<8, 128>::TMEM_COLS);
  printf("head %d %d\n", q3s::HeadTile<8, 192>::SMEM_BYTES, q3s::HeadTile<8, 192>::TMEM_COLS);
}
"""


def test_kernels_on_one_multiprocessor_never_wait_for_each_others_tensor_memory(tmp_path):
    """CTAs that fit a SM together, by shared memory alone (228 KB, 1 KB of it reserved a CTA), need 512 columns at most:
    a CTA of a cluster that waited for another grid's columns could wait for good."""
    from q3s import build

    src, exe = tmp_path / "columns.cu", tmp_path / "columns"
    src.write_text(TENSOR_MEMORY_PROGRAM)
    subprocess.run([build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", f"-I{CSRC}", f"-I{build.INCLUDE}",
                    "-o", str(exe), str(src)], check=True, capture_output=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    kinds = {}
    for kind, smem, columns in (ln.split() for ln in lines if ln):
        kinds.setdefault(int(columns), []).append((int(smem), kind))
    assert sum(len(v) for v in kinds.values()) > 20
    unit = 128  # shared memory is handed out in pieces of this size
    room = 228 * 1024 // unit
    need = {c: (min(v)[0] + 1024) // unit for c, v in kinds.items()}  # a kernel's least shared memory decides
    most = [0] * (room + 1)  # columns that CTAs within so much shared memory can ask for
    for x in range(room + 1):
        most[x] = max([0] + [most[x - n] + c for c, n in need.items() if n <= x])
    assert most[room] <= 512, (most[room], {c: min(v) for c, v in kinds.items()})


def test_every_operator_with_device_waits_takes_an_error_word():
    import q3s

    q3s.load_torch_ops()
    import torch

    for name in ("cache_append", "prefix_attention", "int8_matmul", "int8_linear"):
        arg = {a.name: a for a in getattr(torch.ops.q3s, name).default._schema.arguments}["error_word"]
        assert arg.alias_info is not None and arg.alias_info.is_write and arg.default_value is None


def test_cache_tables_descriptor_of_before_the_flags_is_taken():
    import ctypes as C

    from q3s import _lib
    from test_decode_host import GOOD

    lib, (cls, good) = _lib.load(), GOOD["q3s_cache_tables"]
    old = cls.flags.offset
    for size, kw, message in ((old, dict(flags=77), "ring_size"), (C.sizeof(cls), dict(flags=2), "flags"), (old + 4, {}, "struct_size"),
                              (C.sizeof(cls), dict(flags=_lib.TABLES_WHOLE_ROWS), "ring_size")):
        d = cls(**{**good, "struct_size": size, "ring_size": 0, **kw})
        assert lib.q3s_cache_tables(C.byref(d), None) == _lib.ERR_INVALID_ARGUMENT and message in _lib.last_error()


def test_attention_descriptor_of_before_the_slot_map_is_taken():
    import ctypes as C

    from q3s import _lib
    from test_decode_host import GOOD

    lib, (cls, good) = _lib.load(), GOOD["q3s_prefix_attention"]
    n = C.c_int64()
    for size, status in ((cls.slot_map.offset, _lib.OK), (C.sizeof(cls), _lib.OK), (cls.slot_map.offset - 8, _lib.ERR_INVALID_ARGUMENT)):
        assert lib.q3s_prefix_attention_workspace(C.byref(cls(**{**good, "struct_size": size})), C.byref(n)) == status
