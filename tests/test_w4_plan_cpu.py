"""The plan of the 4-bit products with few rows, on the host: what a CTA holds fits
its shared memory, whatever the width, and the parts cover all columns."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "lc_w4_few.cuh"
using namespace lc;
template <typename T, int GROUP, int NT>
void one(long long cols, long long rows, int batch) {
    W4 w = {};
    w.rows = (int)rows, w.cols = (int)cols, w.group = GROUP;
    w.tiles = (int)((rows + kW4Rows - 1) / kW4Rows), w.blocks = (int)((cols + kW4Cols - 1) / kW4Cols);
    using S = FewShape<T, GROUP, NT>;
    const FewPlan p = few_plan<S>(w, batch, 148);
    std::printf("%d %d %d %d %d %d %d %d %d %zu\n", (int)sizeof(T), GROUP, NT, w.blocks, batch, p.cluster, p.phases, p.split, p.blocks,
                S::smem(p, batch));
}
template <typename T, int GROUP>
void all(long long cols, long long rows) {
    const int half = sizeof(T) == 4 ? 4 : 8;
    for (int batch = 1; batch <= 2 * half; ++batch)
        batch <= half ? one<T, GROUP, 1>(cols, rows, batch) : one<T, GROUP, 2>(cols, rows, batch);
}
int main() {
    long long cols, rows;
    while (std::scanf("%lld %lld", &cols, &rows) == 2) {
        all<float, 32>(cols, rows), all<float, 64>(cols, rows), all<float, 128>(cols, rows);
        all<__half, 32>(cols, rows), all<__half, 64>(cols, rows), all<__half, 128>(cols, rows);
    }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    import build
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cu").write_text(PROGRAM)
    subprocess.run([build._nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", build.CSRC, "-I", build.INCLUDE,
                    "-cudart", "static", str(at / "plan.cu"), "-o", str(at / "plan")], check=True, capture_output=True)

    def run(sizes):
        text = "\n".join(f"{c} {r}" for c, r in sizes)
        out = subprocess.run([str(at / "plan")], input=text, capture_output=True, text=True, check=True, timeout=120).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def held(elem, group, nt, batch, cluster, split, blocks):
    """Bytes of a CTA, counted apart: rings of 8 warps x 3 blocks of two tiles, the
    columns of x and one of zeros, factors and largest sizes, the warps' sums, and what
    a cluster's CTAs send, twice."""
    groups, rows = 128 // group, (4 if elem == 4 else 8) * nt
    columns = batch * (2 if elem == 4 else 1) + 1
    runs = -(-8 // split * 2 * rows // cluster)
    ring = 8 * 3 * 2 * (1024 + 16 * groups * 3)
    return (ring + columns * (256 * blocks + 64) + 9 * rows * 4 + 8 * 2 * rows * 24 * 4 +
            (2 * cluster * runs * 16 * 4 if cluster > 1 else 0))


# From one block to the widest matrix; the last ones are some whose sums, in 32 bits,
# are those of a few kilobytes.
WIDTHS = [1, 128, 2048, 8192, 40000, 140000, 1 << 20, 63 << 20, 1 << 28, 977000000, 2 ** 31 - 1 - (1 << 20)]


@pytest.mark.parametrize("rows", [1, 300])
def test_shared_memory_holds_what_the_plan_says(plans, rows):
    cluster = 8
    wrap = [932049 * cluster * 128, 932100 * cluster * 128, 958682 * cluster * 128, 979677 * cluster * 128, 986875 * cluster * 128]
    for elem, group, nt, width, batch, cs, phases, split, blocks, smem in plans([(c, rows) for c in WIDTHS + wrap]):
        what = f"{elem}-byte rows, groups of {group}, {batch} x {width} blocks: {blocks} blocks of {cs} CTAs and {phases} phases"
        assert blocks * cs * phases >= width, what
        assert smem == held(elem, group, nt, batch, cs, split, blocks), what
        assert smem <= 226 * 1024, what
