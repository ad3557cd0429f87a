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
