"""The paged kernels' arithmetic of tiles and positions at sizes that no GPU test reaches: the device functions are compiled
for the host and run there."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMPAT = os.path.join(ROOT, "framework-torch-paras_b200", "csrc", "compat")

MAIN = r"""
#include "paged_attn.cuh"
#include <cstdio>
#include <cstdlib>
using namespace pb;
int main(int argc, char** argv) {
    PagedParams p{};
    PagedSeq s{};
    auto arg = [&](int i) { return std::atoi(argv[i]); };
    if (argc == 6) {          // causal, new tokens, positions, position of the first token, tokens of a query tile
        p.causal = arg(1); s.nq = arg(2); s.kv = arg(3); s.pos0 = arg(4);
        std::printf("%lld\n", (long long)head_tiles(p, s, arg(5)));
    }
    if (argc == 7) {          // causal, tokens in all, cu[b], cu[b+1], kv_lens[b], a row of the sequence: first row, count, keys the row attends
        p.causal = arg(1); p.T = p.max_q = p.q_max = arg(2); p.q_min = 1; p.cap = 1 << 30;
        s = paged_place(p, arg(3), arg(4), arg(5));
        std::printf("%d %d %d\n", s.row0, s.nq, paged_keys(p, s, arg(6) - s.row0));
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("arithmetic")
    src, exe = d / "main.cu", d / "main"
    src.write_text(MAIN)
    nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    subprocess.run([nvcc if os.path.exists(nvcc) else "nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-diag-suppress", "177,550",
                    "-I", COMPAT, "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True, timeout=600)
    return lambda *a: [int(x) for x in subprocess.run([str(exe), *map(str, a)], check=True, capture_output=True, text=True).stdout.split()]


def tiles(causal, nq, kv, pos0, pt):
    n = 0
    for first in range(0, nq, 2 * pt):
        last = min(nq, first + 2 * pt) - 1
        keys = max(0, min(kv, pos0 + last + 1)) if causal else kv
        n += max(1, -(-keys // 128))
    return n


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("nq,kv,pt", [(0, 100, 32), (1, 0, 128), (300, 1000, 32), (700, 701, 42), (512, 2 ** 30, 1), (16384, 2 ** 30, 32),
                                      (4096, 2 ** 31 - 256, 16), (1 << 20, 1 << 20, 1)])
def test_tiles_of_a_head(program, causal, nq, kv, pt):
    # 512 tokens of 128 heads that share a kv head are 256 items, which attend 2^23 tiles each at 2^30 positions
    pos0 = kv - nq
    assert program(causal, nq, kv, pos0, pt) == [tiles(causal, nq, kv, pos0, pt)]


@pytest.mark.parametrize("T,c0,c1,kv,row", [(10, 0, 4, 100, 2), (10, 4, 10, 6, 4), (10, 4, 10, 3, 4), (10, 4, 10, 3, 9), (10, 4, 14, 100, 6), (10, 4, 14, 9, 9),
                                            (10, 4, 1 << 30, 100, 9), (10, -3, 6, 20, 0), (10, 0, 10, -5, 9), (10, 0, 10, -2 ** 31, 9), (10, 0, 10, 2 ** 31 - 1, 3),
                                            (2 ** 30 + 500, 0, 2 ** 30 + 500, 1, 2 ** 30 + 498), (2 ** 30 + 500, 0, 2 ** 30 + 500, 1, 2 ** 30 + 499),
                                            (2 ** 30 + 500, 0, 2 ** 30 + 500, 600, 2 ** 30 + 100)])
@pytest.mark.parametrize("causal", [0, 1])
def test_a_rows_position(program, causal, T, c0, c1, kv, row):
    # row r of a sequence stands at kv_lens[b] - (cu[b+1] - cu[b]) + (r - cu[b]), wherever the sequence's rows end
    first, end = max(0, c0), min(c1, T)
    held = max(0, min(kv, 1 << 30))
    keys = max(0, min(held, kv - c1 + row + 1)) if causal else held
    assert program(causal, T, c0, c1, kv, row) == [first, end - first, keys]
