"""Weight gradients where a batch carries a few adapters of a large table, or as many segments as a call
takes at the largest rank (a ring of one stage), against float64."""
import pytest
import torch

from test_gpu_lora import STEP, _status, close, cuda_i32, make, reference, row_adapters  # noqa: F401

pytestmark = pytest.mark.gpu


def check(M, K, N, R, L, ends, adapter, grad_w_dtype=torch.float32):
    import kernels
    x, a, b, s, _ = make(M, K, N, R, L, seed=M + L)
    go = torch.randn(M, N, generator=torch.Generator().manual_seed(L)).bfloat16().cuda()
    rows = row_adapters(M, ends, adapter, L)
    oi, ai = cuda_i32(ends), cuda_i32(adapter)
    _, v = kernels.lora_grouped_mm(x, a, b, oi, ai, s, return_v=True)
    _, ga, gb = kernels.lora_grouped_mm_backward(go, x, a, b, v, oi, ai, s, grad_w_dtype=grad_w_dtype)
    vref, verr, _, _ = reference(x, a, b, s, None, rows)
    dv, dverr, _, _ = reference(go, b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous(), s, None, rows)
    used = sorted({int(l) for l in rows.tolist() if l >= 0})
    for l in used:
        m = (rows == l).nonzero().reshape(-1)
        n = 2 * m.numel() + 2
        for got, u, uerr, z in ((ga[l], dv[m], dverr[m], x[m].double()), (gb[l].t(), vref[m], verr[m], go[m].double())):
            close(got, u.t() @ z, uerr.t() @ z.abs() + n * STEP * (u.abs().t() @ z.abs()), f"adapter {l}")
    rest = torch.ones(L, dtype=torch.bool)
    rest[used] = False
    assert not bool(ga[rest.cuda()].any()) and not bool(gb[rest.cuda()].any())


@pytest.mark.parametrize("R", [8, 32, 72])
@pytest.mark.parametrize("M,ends,adapter", [
    (700, [100, 100, 350, 420, 690], [499, 3, 77, 498, 77]),
    (4000, [1, 2, 3000, 3100, 4000], [0, 499, 250, 0, 499]),
    (130, [130], [321]),
    (900, [200, 500, 900], [-1, 500, 7])])
def test_a_few_adapters_of_many(M, ends, adapter, R):
    check(M, 264, 520, R, 500, ends, adapter)


@pytest.mark.parametrize("L", [3, 1023, 1024, 1025])
def test_as_many_segments_as_a_call_takes_at_the_largest_rank(L):
    M = 2500
    ends = [min(M, 2 * i + i % 3) for i in range(1, 1025)]
    check(M, 64, 136, 128, L, ends, [(37 * i + 5) % (L + 1) for i in range(1024)])
