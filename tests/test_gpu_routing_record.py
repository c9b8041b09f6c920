"""The router's gradient is that of the record route_topk wrote, whatever tensors a Routing carries in the
fields' places."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (333, 40, 3), (70, 256, 8)])
def test_replaced_fields_do_not_change_the_gradient(T, E, k):
    """Half-precision weights, int64 choices and strided counts in the fields, as a user's program may keep
    them: read as fp32 and int32 they would be other numbers, and end before the tensors' ends."""
    from mxgg.moe import route_topk, route_topk_backward
    g = torch.Generator().manual_seed(T)
    x, gw = torch.randn(T, E, generator=g).cuda(), torch.randn(T, k, generator=g).cuda()
    r = route_topk(x, k)
    want = route_topk_backward(x, r, gw, 0.5, 0.25)
    spread = torch.zeros(E, 2, dtype=torch.int32, device="cuda")
    spread[:, 0] = r.counts
    other = r._replace(experts=r.experts.long(), weights=r.weights.half(), counts=spread[:, 0])
    assert torch.equal(route_topk_backward(x, other, gw, 0.5, 0.25), want)
    scaled = r._replace(weights=r.weights * 2.5)
    assert torch.equal(route_topk_backward(x, scaled, gw, 0.5, 0.25), want)


def test_weights_scaled_in_place_are_refused():
    from mxgg.moe import route_topk, route_topk_backward
    x = torch.randn(50, 8, generator=torch.Generator().manual_seed(1)).cuda()
    r = route_topk(x, 2)
    route_topk_backward(x, r, torch.ones(50, 2, device="cuda"))
    r.weights.mul_(2.5)
    with pytest.raises(ValueError, match="in place"):
        route_topk_backward(x, r, torch.ones(50, 2, device="cuda"))


def test_inference_mode():
    from mxgg.moe import route_topk, route_topk_backward
    x = torch.randn(50, 8, generator=torch.Generator().manual_seed(1)).cuda()
    want = route_topk_backward(x, route_topk(x, 2), None, 1.0, 1.0)
    with torch.inference_mode():
        assert torch.equal(route_topk_backward(x, route_topk(x, 2), None, 1.0, 1.0), want)
