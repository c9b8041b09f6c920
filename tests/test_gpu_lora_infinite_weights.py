"""Infinite operands of the adapters' second products, which multiply v's two halves: the formula's infinities
and no NaN.  Everything else is positive, so that the formula has no NaN anywhere; the low half has either sign."""
import pytest
import torch

from test_gpu_lora import _status, cuda_i32  # noqa: F401
from test_gpu_lora_nonfinite import INF, RANKS, only_at, positive

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [20, 300])
@pytest.mark.parametrize("R", RANKS)
def test_infinite_weight(M, R, out_dtype):
    """One infinite element of B: a column of its adapter's rows; one of A: a column of grad_x."""
    import kernels
    K, N = 72, 136
    x, a, b, s, base, go = positive(M, K, N, R, 2)
    base = base.to(out_dtype)
    ends, ad = cuda_i32([M - 8, M]), cuda_i32([0, 1])
    mine = list(range(M - 8, M))
    b2 = b.clone()
    b2[1, 69, R - 1] = INF
    out, v = kernels.lora_grouped_mm(x, a, b2, ends, ad, s, base=base, return_v=True)
    assert only_at(out, mine, [69])
    rows = torch.zeros(M, dtype=torch.int32, device="cuda")
    rows[M - 8:] = 1
    assert only_at(kernels.lora_grouped_mm(x, a, b2, None, rows, s, base=base), mine, [69])
    clean, _ = kernels.lora_grouped_mm(x, a, b, ends, ad, s, base=base, return_v=True)
    keep = [c for c in range(N) if c != 69]
    assert torch.equal(out[:, keep], clean[:, keep])
    # the halves' sum is exact in the high half: the low one is 0
    a2 = torch.zeros_like(a)
    a2[:, :, 0] = 1.0
    ones = torch.ones_like(x)
    assert only_at(kernels.lora_grouped_mm(ones, a2, b2, ends, ad, None, base=base), mine, [69])
    assert only_at(kernels.lora_grouped_mm(ones, a2, b2, None, rows, None, base=base), mine, [69])
    a2 = a.clone()
    a2[1, 2, 66] = INF
    gx, _, _ = kernels.lora_grouped_mm_backward(go, x, a2, b, v, ends, ad, s, grad_x_dtype=out_dtype,
                                                need=(True, False, False))
    assert only_at(gx, mine, [66])


@pytest.mark.parametrize("R", RANKS)
def test_infinite_value_in_a_weight_gradient(R):
    """One infinite x: a column of its adapter's grad_a; one infinite grad_out: a row of grad_b (and, through
    dv, all of its adapter's grad_a).  Above rank 32 NaNs may take the infinities' places, and no others."""
    import kernels
    M, K, N = 400, 200, 136
    x, a, b, s, _, go = positive(M, K, N, R, 3)
    ends, ad = cuda_i32([100, 300, 400]), cuda_i32([0, 2, 1])
    _, v = kernels.lora_grouped_mm(x, a, b, ends, ad, s, return_v=True)

    def only(t, rows, cols):
        return only_at(t if R <= 32 else torch.where(t.isnan(), INF, t), rows, cols)

    x2 = x.clone()
    x2[220, 130] = INF
    gx, ga, gb = kernels.lora_grouped_mm_backward(go, x2, a, b, v, ends, ad, s)
    assert only(ga[2], None, [130]) and bool(ga[:2].isfinite().all())
    assert bool(gx.isfinite().all()) and bool(gb.isfinite().all())
    go2 = go.clone()
    go2[310, 133] = INF
    gx, ga, gb = kernels.lora_grouped_mm_backward(go2, x, a, b, v, ends, ad, s)
    assert only(gb[1], [133], None) and bool(gb[0].isfinite().all()) and bool(gb[2].isfinite().all())
    assert bool((ga[1] == INF).all()) and bool(ga[0].isfinite().all()) and bool(ga[2].isfinite().all())
    assert only_at(gx, [310], None)


def test_nan_weights_stay_in_their_columns():
    """NaNs are taken again and stay NaN; a whole adapter of them is slow, not wrong."""
    import kernels
    x, a, b, s, base, _ = positive(500, 64, 1032, 40, 2)
    ends, ad = cuda_i32([200, 500]), cuda_i32([0, 1])
    clean = kernels.lora_grouped_mm(x, a, b, ends, ad, s, base=base)
    b2 = b.clone()
    b2[1, 700] = float("nan")
    b2[0] = float("nan")
    out = kernels.lora_grouped_mm(x, a, b2, ends, ad, s, base=base)
    assert bool(out[:200].isnan().all()) and bool(out[200:, 700].isnan().all())
    keep = [c for c in range(1032) if c != 700]
    assert torch.equal(out[200:, keep], clean[200:, keep])


def signs(M, K, N, R, seed=9):
    """Operands of both signs, and which of v's elements are far enough from 0 to have a sign beyond doubt."""
    from test_gpu_lora import make, reference
    x, a, b, s, base = make(M, K, N, R, 2, seed=seed)
    rows = torch.zeros(M, dtype=torch.int64, device="cuda")
    rows[M // 2:] = 1
    v, verr, _, _ = reference(x, a, b, s, None, rows)
    return x, a, b, s, base, rows, v, v.abs() > 2 * verr


@pytest.mark.parametrize("M", [24, 300])
@pytest.mark.parametrize("R", RANKS)
def test_signs_of_infinities(M, R):
    """An infinite weight in every column, of either sign and at every rank: the infinity has v's sign times the
    weight's.  Two of them in a column: an infinity where their signs agree, NaN where they do not."""
    import kernels
    K, N = 64, 200
    x, a, b, s, base, rows, v, sure = signs(M, K, N, R)
    ends, ad = cuda_i32([M // 2, M]), cuda_i32([0, 1])
    cols = torch.arange(N, device="cuda")
    first, second = cols % R, (7 * cols + 3) % R
    one, two = b.clone(), b.clone()
    up = torch.where(cols % 3 == 0, -INF, INF)
    for l in range(2):
        one[l, cols, first] = up.bfloat16()
        two[l, cols, first] = up.bfloat16()
        two[l, cols, second] = INF
    p, q = v[:, first] * up, v[:, second] * INF
    known, both = sure[:, first], sure[:, first] & sure[:, second]
    p2 = torch.where(first == second, q, p)
    for w, want, ok in ((one, p, known), (two, p2 + q, both)):
        for out in (kernels.lora_grouped_mm(x, a, w, ends, ad, s, base=base),
                    kernels.lora_grouped_mm(x, a, w, None, rows.int(), s, base=base, out_dtype=base.dtype)):
            got = out.double()
            same = (got == want) | (got.isnan() & want.isnan())
            assert bool(same[ok].all()), int((~same & ok).sum())


@pytest.mark.parametrize("R", [8, 24, 32])
def test_signs_of_infinities_in_a_weight_gradient(R):
    """An infinite x in every seventh column: grad_a's infinity has dv's sign times its own."""
    import kernels
    M, K, N = 400, 200, 136
    x, a, b, s, _, rows, _, _ = signs(M, K, N, R)
    from test_gpu_lora import reference
    ends, ad = cuda_i32([M // 2, M]), cuda_i32([0, 1])
    go = torch.randn(M, N, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    dv, err, _, _ = reference(go, b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous(), s, None, rows)
    _, v = kernels.lora_grouped_mm(x, a, b, ends, ad, s, return_v=True)
    x2 = x.clone()
    for c in range(0, K, 7):
        m = M // 2 + 3 * c // 7 % 200
        x2[m, c] = INF if c % 2 else -INF
    _, ga, _ = kernels.lora_grouped_mm_backward(go, x2, a, b, v, ends, ad, s, need=(False, True, False))
    for c in range(0, K, 7):
        m = M // 2 + 3 * c // 7 % 200
        ok = dv[m].abs() > 2 * err[m]
        assert torch.equal(ga[1, :, c].double()[ok], (dv[m] * (INF if c % 2 else -INF))[ok])
    rest = [c for c in range(K) if c % 7]
    assert bool(ga[:, :, rest].isfinite().all()) and bool(ga[0].isfinite().all())
