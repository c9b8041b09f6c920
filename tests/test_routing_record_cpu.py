"""The router's gradient refuses a Routing whose record is not the one route_topk wrote.  The checks come
before the device is touched, so they run on CPU tensors."""
import pytest
import torch

from mxgg import _lib
from mxgg.moe import Routing, _routing_parts, route_topk_backward

T, K, E = 6, 2, 8


def size(tokens):
    return _routing_parts(tokens, K, E)[5] + _lib.load().mxgg_route_workspace_size(tokens, E) // 4


def routing(**other):
    at = _routing_parts(T, K, E)
    ints = torch.zeros(size(T), dtype=torch.int32)
    floats = ints.view(torch.float32)
    r = Routing(ints.as_strided((T, K), (K, 1), 0), floats.as_strided((T, K), (K, 1), at[1]),
                ints.as_strided((E,), (1,), at[3]), floats.as_strided((), (), at[4]),
                floats.as_strided((), (), at[4] + 1), ints, True)
    return r._replace(**other)


def call(r):
    return route_topk_backward(torch.zeros(T, E), r)


def test_a_good_record_comes_as_far_as_the_device():
    with pytest.raises(RuntimeError, match="CUDA"):
        call(routing())


@pytest.mark.parametrize("buffer", [
    lambda n: torch.zeros(n, dtype=torch.int64), lambda n: torch.zeros(n, dtype=torch.float32),
    lambda n: torch.zeros(n - 4, dtype=torch.int32), lambda n: torch.zeros(2 * n, dtype=torch.int32)[::2],
    lambda n: torch.zeros(1, n, dtype=torch.int32)], ids=["int64", "fp32", "short", "strided", "2-D"])
def test_other_buffers_are_refused(buffer):
    with pytest.raises(ValueError, match="buffer"):
        call(routing(buffer=buffer(size(T))))


def test_a_record_of_another_size_than_its_fields_is_refused():
    """More tokens or experts in the fields than the record has: what lies behind it must not be read.  Fewer:
    its parts lie elsewhere."""
    with pytest.raises(ValueError, match="buffer"):
        route_topk_backward(torch.zeros(3, E), routing(experts=torch.zeros(3, K, dtype=torch.int32)))
    with pytest.raises(ValueError, match="buffer"):
        call(routing(experts=torch.zeros(1000, K, dtype=torch.int32)))
    with pytest.raises(ValueError, match="buffer"):
        call(routing(counts=torch.zeros(1000, dtype=torch.int32)))
    with pytest.raises(ValueError, match="choices|experts"):
        call(routing(experts=torch.zeros(T * K, dtype=torch.int32)))


@pytest.mark.parametrize("name", ["experts", "weights", "counts", "balance_loss"])
def test_a_record_changed_in_place_is_refused(name):
    r = routing()
    getattr(r, name).add_(1)
    with pytest.raises(ValueError, match="in place"):
        call(r)


def test_records_made_in_inference_mode_have_no_version():
    with torch.inference_mode():
        r = routing()
        with pytest.raises(RuntimeError, match="CUDA"):
            call(r)
