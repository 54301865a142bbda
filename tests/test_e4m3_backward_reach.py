"""On the host: how far the weight gradient's product of phonlp_linear_e4m3_backward reaches into dY where it reads dY itself (bf16, no ReLU,
whole steps of 32).  The kernel's own address arithmetic (csrc/e4m3_backward.h) runs over all tiles, lanes and rows of a step."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "phonlp_amd", "csrc")

DRIVER = r"""
#include <stdio.h>
#include <stdlib.h>
#include "e4m3_backward.h"
using namespace phonlp;

template <int TI>
static long reach(const BwOperand &a, int M, int N, long *behind) {
    long most = 0;
    for (int i0 = 0; i0 < N; i0 += TI)
        for (int u = 0; u < 32 * TI * 2 / 1024; ++u)
            for (int lane = 0; lane < 64; ++lane) {
                const long off = tr_offset<TI * 2>(u, lane, a.pitch, a.width - i0 * 2L), in_row = (i0 * 2L + off) % a.pitch + 16;
                const long end = (M / 32 - 1) * 32 * a.pitch + i0 * 2L + off + 16;
                if (end > most) most = end;
                if (in_row > N * 2L) ++*behind;
            }
    return most;
}

int main(int argc, char **argv) {
    const int M = atoi(argv[1]), N = atoi(argv[2]);
    const long ld = atol(argv[3]);
    if (!bw_direct((const void *)16, PHONLP_BF16, ld, nullptr, M, N)) return 3;
    const BwOperand a = bw_dz(true, (const void *)16, ld, nullptr, N, M, N);
    long behind = 0;
    const long small = reach<128>(a, M, N, &behind), large = reach<256>(a, M, N, &behind);
    printf("%ld %ld %ld\n", small, large, behind);
    return a.at == (const uint8_t *)16 ? 0 : 4;
}
"""


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("reach")
    (d / "reach.cpp").write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-isystem", "/opt/rocm/include", "-I", CSRC,
                           "-o", str(d / "reach"), str(d / "reach.cpp")])
    return str(d / "reach")


@pytest.mark.parametrize("M,N,ld", [(32, 32, 32), (32, 32, 64), (64, 32, 4096), (64, 160, 320), (96, 160, 168), (32768, 2368, 4736), (64, 2464, 2472),
                                    (64, 256, 512), (32, 384, 392), (64, 128, 256)])
def test_the_weight_gradients_product_stays_inside_dY(driver, M, N, ld):
    """A right-hand slice of wider rows, the last one of which ends N columns after its first: nothing may be read behind it."""
    small, large, behind = map(int, subprocess.check_output([driver, str(M), str(N), str(ld)]).split())
    last = (M - 1) * ld * 2 + N * 2
    assert small == large == last and behind == 0
