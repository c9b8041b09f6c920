"""The documented way through a routed layer with adapters, forward and backward, run as it is written."""
import glob
import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def recipe():
    """The one python block of the documents that takes adapters' gradients on a dispatch plan."""
    found = []
    for path in glob.glob(os.path.join(ROOT, "*.md")):
        with open(path) as f:
            found += [b for b in re.findall(r"```python\n(.*?)```", f.read(), re.S)
                      if "lora_grouped_mm_backward(" in b and "dispatch_plan(" in b]
    assert len(found) == 1
    return found[0]


def run(last_token):
    import utils
    E, T, K, N, R = 4, 70, 64, 128, 8
    g = torch.Generator().manual_seed(6)
    w_s, w_q = utils.to_mx((torch.randn(E, N, K, generator=g) * K ** -0.5).bfloat16().cuda())
    x = torch.randn(T, K, generator=g).bfloat16()
    logits = torch.randn(T, E, generator=g)
    x[-1] = last_token
    mask = torch.ones(T, dtype=torch.bool)
    mask[-1] = False
    rows = (2 * T + E * 31) // 32 * 32
    names = {"E": E, "x": x.cuda(), "logits": logits.cuda(), "mask": mask.cuda(), "w_q": w_q, "w_s": w_s,
             "lora_a": (torch.randn(E, R, K, generator=g) * K ** -0.5).bfloat16().cuda(),
             "lora_b": (torch.randn(E, N, R, generator=g) * R ** -0.5).bfloat16().cuda(),
             "grad_out": torch.randn(T, N, generator=g).bfloat16().cuda(),
             "dgrad_rows": torch.randn(rows, K, generator=g).bfloat16().cuda(), "torch": torch}
    import kernels
    names["triton_mxfp8_grouped_mm"] = kernels.triton_mxfp8_grouped_mm
    exec(compile(recipe(), "recipe", "exec"), names)
    return {k: names[k] for k in ("out", "gw", "g_a", "g_b", "g_x", "g_logits")}


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1e30])
def test_a_masked_token_may_hold_anything(value):
    """The last token, masked, changes nothing: padding rows are no token's."""
    want, got = run(0.5), run(value)
    for name in want:
        assert bool(want[name].isfinite().all()), name
        assert torch.equal(got[name], want[name]), name
