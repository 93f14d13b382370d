"""GPU: the serving operators' kernels at the sizes where each of their forms is chosen, against 64 bits or exact values,
and what a call owes the framework around it. Tolerances as in test_serving_ops_gpu.py."""
import pytest
import torch

from actalker_amd import ops
from tests.test_serving_ops_gpu import _seed, act      # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ product
@pytest.mark.parametrize("M,N,K", [(1, 8200, 528), (1, 16, 128), (16, 70, 640), (5, 8200, 517), (17, 300, 640), (32, 1030, 333),
                                   (300, 320, 272), (130, 1030, 144), (700, 640, 512), (700, 640, 509)])
def test_gemm_fp8_few_rows_keep_small_products(dev, M, N, K):
    """Large products that cancel beside one small one: every partial sum has at most 23 bits between its first and last
    (2^15 .. 2^-7), so fp32 sums are exact in any order, and what is left is a power of two times 1 or 1.5, exact in 16 bits."""
    a, w = torch.zeros(M, K), (2.0 ** (torch.arange(N) % 3))[:, None].repeat(1, K)
    n16 = K // 16
    a[:, 0:16 * n16:16], a[:, 8:16 * n16:16] = 256.0, -256.0
    m = torch.arange(M)
    a[m, 16 * (m % n16) + 1 + m % 7] = (1 + 0.5 * (m % 2)) * 2.0 ** -6
    want = ((1 + 0.5 * (m % 2)) * 2.0 ** -6)[:, None] * w[:, 0]
    s, ws = torch.ones(M, -(-K // 128)), torch.ones(-(-N // 128), -(-K // 128))
    for f32 in (False, True):
        out = ops.gemm_fp8(a.to(ops.FP8).to(dev), s.to(dev), w.to(ops.FP8).to(dev), ws.to(dev), out_f32=f32)
        assert torch.equal(out.float().cpu(), want)
