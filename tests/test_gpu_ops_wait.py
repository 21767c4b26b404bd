"""The operators' bounded waits (csrc/ops_wait.cuh) on the B200: a wait for what nothing does ends after its limit, with a status."""

import ctypes
import subprocess

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from conftest import PKG      # noqa: E402

SOURCE = r"""
#include <cuda_runtime.h>
#include "ops_wait.cuh"

/* warps 0 to 2 wait for one barrier, the other one, and both; with `arrive` warp 3 arrives on them */
__global__ void waits(unsigned *status, unsigned *passed, uint64_t limit, int arrive) {
    __shared__ uint64_t barrier[2];
    __shared__ volatile unsigned abort;
    const int warp = threadIdx.x >> 5;
    const uint32_t a = shared_address(&barrier[0]), b = shared_address(&barrier[1]);
    if (threadIdx.x == 0) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(a));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(b));
        abort = 0;
    }
    __syncthreads();
    if (threadIdx.x & 31) return;
    if (warp == 3) {
        const uint64_t start = now_ns();
        if (!arrive) wait_for_end(a, 0, start, limit);
        if (arrive) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(a) : "memory");
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
        }
        return;
    }
    passed[warp] = warp == 0   ? wait_for(a, 0, &abort, status, 1, limit)
                   : warp == 1 ? wait_for(b, 0, &abort, status, 2, limit)
                               : wait_for_both(a, 0, b, 0, &abort, status, 4, limit);
}

extern "C" int run(unsigned *status, unsigned *passed, uint64_t limit, int arrive, uint64_t stream) {
    waits<<<1, 128, 0, (cudaStream_t)stream>>>(status, passed, limit, arrive);
    return (int)cudaGetLastError();
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    d = tmp_path_factory.mktemp("waits")
    (d / "waits.cu").write_text(SOURCE)
    subprocess.run(["nvcc", "-O2", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a",
                    f"-I{PKG / 'csrc'}", str(d / "waits.cu"), "-o", str(d / "waits.so"), "-cudart", "static"], check=True)
    fn = ctypes.CDLL(str(d / "waits.so")).run
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int, ctypes.c_uint64]

    def call(limit, arrive):
        status, passed = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((3,), 9, dtype=torch.int32, device="cuda")
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        assert fn(status.data_ptr(), passed.data_ptr(), limit, arrive, torch.cuda.current_stream().cuda_stream) == 0
        end.record()
        torch.cuda.synchronize()
        return status.item(), passed.tolist(), start.elapsed_time(end)
    return call


def test_a_wait_for_nothing_ends(run):
    for _ in range(3):
        status, passed, ms = run(20_000_000, 0)
        assert passed == [0, 0, 0]
        assert status & 7 and status & ~7 == 0          # whoever gave up first told the others, which need not
        assert 19 <= ms < 5000
        assert run(20_000_000, 1)[:2] == (0, [1, 1, 1])  # and the context works on


def test_a_wait_that_ends_in_time_has_no_status(run):
    for limit in (20_000_000, 2_000_000_000):
        assert run(limit, 1)[:2] == (0, [1, 1, 1])
