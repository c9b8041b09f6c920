"""Segment ends of 64 bits: one that 32 bits do not hold lies past the rows (or before them) and must not wrap
into their range."""
import pytest
import torch

from test_gpu_lora import _status, cuda_i32, make  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [50, 300])
@pytest.mark.parametrize("ends", [[40, (1 << 32) + 10], [-(1 << 32) + 20, 45], [10, 1 << 40], [1 << 31, 1 << 33]])
def test_ends_do_not_wrap(M, ends):
    import kernels
    x, a, b, s, base = make(M, 64, 72, 8, 2)
    go = torch.randn(M, 72, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    cut = cuda_i32([min(max(e, 0), M) for e in ends])
    wide = torch.tensor(ends, dtype=torch.int64, device="cuda")
    got, want = base.clone(), base.clone()
    v = kernels.lora_grouped_mm(x, a, b, wide, None, s, out=got, return_v=True)[1]
    u = kernels.lora_grouped_mm(x, a, b, cut, None, s, out=want, return_v=True)[1]
    assert torch.equal(got, want)
    live = int(cut.max())
    assert torch.equal(v[:live], u[:live])
    gx = [kernels.lora_grouped_mm_backward(go, x, a, b, u, e, None, s) for e in (wide, cut)]
    assert torch.equal(gx[0][0][:live], gx[1][0][:live])
    assert torch.equal(gx[0][1], gx[1][1]) and torch.equal(gx[0][2], gx[1][2])
