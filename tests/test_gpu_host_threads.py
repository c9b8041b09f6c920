"""Calls of several host threads at once, each on a stream of its own: no call's launch depends on another's
sizes, and every result is the one a lone thread gets."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

ROUNDS = 2000


def both(jobs):
    """Runs every job in a thread of its own, all at once; the first exception of each."""
    errors, start = [], threading.Barrier(len(jobs))

    def work(job):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(ROUNDS):
                    job()
                stream.synchronize()
        except Exception as e:  # noqa: BLE001 - handed to the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


def adapters(M, R, S, dtype, rows):
    """A job of one rank, row count, segment count and type, and a check of its last result."""
    import kernels
    g = torch.Generator().manual_seed(R + M)
    K, N, L = 128, 136, 3
    x, go = torch.randn(M, K, generator=g).bfloat16().cuda(), torch.randn(M, N, generator=g).bfloat16().cuda()
    a = (torch.randn(L, R, K, generator=g) * K ** -0.5).bfloat16().cuda()
    b = (torch.randn(L, N, R, generator=g) * R ** -0.5).bfloat16().cuda()
    ends = torch.tensor([M * (i + 1) // S for i in range(S)], dtype=torch.int32, device="cuda")
    ad = (torch.arange(M if rows else S, dtype=torch.int32) % L).cuda()
    last = []

    def job():
        if rows:
            got = [kernels.lora_grouped_mm(x, a, b, None, ad, out_dtype=dtype)]
        else:
            out, v = kernels.lora_grouped_mm(x, a, b, ends, ad, out_dtype=dtype, return_v=True)
            got = [out, *kernels.lora_grouped_mm_backward(go, x, a, b, v, ends, ad, grad_x_dtype=dtype,
                                                          grad_w_dtype=dtype)]
        last[:] = got

    job()
    want = [t.clone() for t in last]
    return job, lambda: all(torch.equal(p, q) for p, q in zip(last, want))


CALLS = [
    # the same kernels with different shared memory: row counts, ranks, segment counts
    [(3, 64, 3, torch.bfloat16, True), (40, 64, 40, torch.bfloat16, True), (40, 48, 40, torch.bfloat16, True)],
    [(300, 16, 2, torch.bfloat16, False), (300, 64, 2, torch.bfloat16, False), (300, 128, 2, torch.bfloat16, False),
     (600, 32, 300, torch.bfloat16, False)],
    [(300, 8, 2, torch.float32, False), (300, 96, 2, torch.float32, False), (300, 64, 5, torch.float16, False)],
]


@pytest.mark.parametrize("calls", CALLS, ids=["rows", "ranks", "types"])
def test_adapters(calls):
    import mxgg
    mxgg.device_status(clear=True)
    jobs = [adapters(*c) for c in calls]
    torch.cuda.synchronize()
    errors = both([j for j, _ in jobs])
    assert not errors, errors[0]
    assert all(same() for _, same in jobs)
    assert mxgg.device_status(clear=True) == 0


def test_plans():
    from mxgg.moe import dispatch_plan
    jobs, wants, lasts = [], [], []
    for E in (700, 800, 1024):
        e = torch.randint(0, E, (3000, 2), generator=torch.Generator().manual_seed(E), dtype=torch.int32).cuda()
        last = []
        lasts.append(last)

        def job(e=e, E=E, last=last):
            last[:] = dispatch_plan(e, E)

        job()
        wants.append([t.clone() for t in last])
        jobs.append(job)
    torch.cuda.synchronize()
    errors = both(jobs)
    assert not errors, errors[0]
    for last, want in zip(lasts, wants):
        assert all(torch.equal(p, q) for p, q in zip(last, want))
