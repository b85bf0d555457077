"""GPU test of the exponential that the sampler's weights are taken with, by itself, against CUDA's ``exp``.

Bound.  With |r| <= ln 2 / 128: the polynomial leaves out r^6 / 720 <= 0.31 x 2^-53 of the value; its last fma and the product
with the table round by 2^-53 each, the earlier steps by at most |r| 2^-53 < 0.01 x 2^-53 each (four of them); the table's
exp2 is off by at most 1 ulp, 2 x 2^-53.  Together 4.4 x 2^-53.  CUDA documents 1 ulp for exp, 2 x 2^-53: the two differ by
at most 6.4 x 2^-53 of the value, 6.5 with second-order terms.
"""
import ctypes
import os
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include <cuda_runtime.h>
#include "sample_exp.cuh"
__global__ void both(const double* z, double* mine, double* theirs, int n) {
  __shared__ double table[fa::SA_EXP_TABLE];
  if (threadIdx.x < fa::SA_EXP_TABLE) table[threadIdx.x] = exp2((double)threadIdx.x / fa::SA_EXP_TABLE);
  __syncthreads();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) mine[i] = fa::sa_exp(z[i], table), theirs[i] = exp(z[i]);
}
extern "C" int run(const double* z, double* mine, double* theirs, int n) {
  both<<<(n + 255) / 256, 256>>>(z, mine, theirs, n);
  return (int)cudaDeviceSynchronize();
}
"""


@pytest.fixture(scope="module")
def both(tmp_path_factory):
    d = tmp_path_factory.mktemp("exp")
    (d / "t.cu").write_text(SOURCE)
    nvcc = "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc"
    subprocess.check_call([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
                           "-I", os.path.join(ROOT, "fourierattention_b200", "csrc"), str(d / "t.cu"), "-o", str(d / "t.so")])
    lib = ctypes.CDLL(str(d / "t.so"))
    lib.run.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int]

    def f(z):
        z = z.contiguous()
        mine, theirs = torch.empty_like(z), torch.empty_like(z)
        torch.cuda.synchronize()
        assert lib.run(z.data_ptr(), mine.data_ptr(), theirs.data_ptr(), z.numel()) == 0
        return mine, theirs
    return f


@pytest.mark.parametrize("low", [700.0, 40.0, 1.0, 2.0 ** -6, 2.0 ** -30])
def test_against_cuda(both, low):
    g = torch.Generator("cuda").manual_seed(int(low))
    z = -low * torch.rand(1 << 21, dtype=torch.float64, device="cuda", generator=g)
    mine, theirs = both(z)
    assert float(((mine - theirs).abs() / theirs).max()) <= 6.5 * 2.0 ** -53


def test_borders(both):
    """Exactly 1 at 0 (min_p = 1 keeps the largest), at the borders of the reduction, 0 from e^-700 down."""
    step = torch.arange(0, 64600, dtype=torch.float64, device="cuda") * (-0.6931471805599453 / 128.0)     # halves of a step too
    step = step[step >= -700.0]
    mine, theirs = both(torch.cat([step, step.nextafter(torch.zeros_like(step)), torch.tensor([0.0, -700.0], device="cuda", dtype=torch.float64)]))
    assert float(((mine - theirs).abs() / theirs).max()) <= 6.5 * 2.0 ** -53
    far = torch.tensor([0.0, -0.0, -700.0001, -745.2, -1e6, -1e83, -1e300, float("-inf")], dtype=torch.float64, device="cuda")
    assert both(far)[0].tolist() == [1.0, 1.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0]
