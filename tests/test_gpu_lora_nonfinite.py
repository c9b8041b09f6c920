"""Infinite values in the adapters' operands: the formula's infinities, in the elements the formula puts
them in, at ranks that are no multiple of 16 as well.  Everything else is positive, so that no infinity
meets a zero or one of the other sign and the formula has no NaN anywhere."""
import pytest
import torch

from test_gpu_lora import _status, cuda_i32, make  # noqa: F401

pytestmark = pytest.mark.gpu

INF = float("inf")
RANKS = [8, 16, 24, 40, 72, 128]


def positive(M, K, N, R, L, seed=3):
    x, a, b, s, base = make(M, K, N, R, L, seed=seed)
    go = torch.randn(M, N, generator=torch.Generator().manual_seed(seed + 1)).bfloat16().cuda()
    return [t.abs() + 0.0625 for t in (x, a, b)] + [s, base, go.abs() + 0.0625]


def only_at(t, rows, cols):
    """+inf in the given rows and columns (all of a dimension where None) and finite elsewhere."""
    want = torch.zeros(t.shape, dtype=torch.bool, device=t.device)
    want[rows if rows is not None else slice(None), cols if cols is not None else slice(None)] = True
    return torch.equal(t == INF, want) and bool(t[~want].isfinite().all())


# 300 rows take 128-row tiles, 20 rows the row form; 1024 columns split a tile's contraction
@pytest.mark.parametrize("M,K,N", [(20, 64, 72), (300, 64, 1032), (300, 1024, 72)])
@pytest.mark.parametrize("R", RANKS)
def test_infinite_input(M, K, N, R):
    """One infinite x: its row of the output; one infinite grad_out: its row of grad_x.  v's padding stays 0."""
    import kernels
    x, a, b, s, base, go = positive(M, K, N, R, 2)
    ends, ad = cuda_i32([M - 8, M]), cuda_i32([0, 1])
    _, v = kernels.lora_grouped_mm(x, a, b, ends, ad, s, return_v=True)
    bad = go.clone()
    bad[M - 3, 7] = INF
    gx, _, _ = kernels.lora_grouped_mm_backward(bad, x, a, b, v, ends, ad, s, need=(True, False, False))
    assert only_at(gx, [M - 3], None)
    x[M - 3, 5] = INF
    out, v = kernels.lora_grouped_mm(x, a, b, ends, ad, s, base=base, return_v=True)
    assert only_at(out, [M - 3], None)
    assert not bool(v[:, :, R:].any())
    rows = torch.zeros(M, dtype=torch.int32, device="cuda")
    rows[M - 8:] = 1
    out, v = kernels.lora_grouped_mm(x, a, b, None, rows, s, base=base, return_v=True)
    assert only_at(out, [M - 3], None)
    assert not bool(v[:, :, R:].any())
