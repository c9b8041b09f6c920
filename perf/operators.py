"""The operators a routed layer needs around its grouped products, each as a case to run and time.

Four operators of this framework, in two forms.  With ``own`` false ``run`` computes them in
elementary torch operations, in 32 bits; with ``own`` true it makes the calls a user makes:

* ``route``: ``mxgg.moe.route_topk`` (top-k router with per-expert counts, a balance loss and a
  z loss) and, for training, ``mxgg.moe.route_topk_backward``;
* ``plan``: ``mxgg.moe.dispatch_plan`` (rows sorted by expert, padded groups, all on the GPU);
* ``combine``: ``mxgg.moe.combine_topk_backward`` (gradients of the weighted top-k combine);
* ``lora``: ``kernels.lora_grouped_mm`` (low-rank adapters beside a shared projection) and, for
  training, ``kernels.lora_grouped_mm_backward``.
"""

import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# weights of the two losses in the training objective
BALANCE, ZLOSS = 1e-2, 1e-3


def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grouped-gemms_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import kernels
    import mxgg.moe
    return mxgg.moe, kernels


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of a few requests through the benchmark's MoE layer (8 experts, top-2): latency only
        {"name": "route_decode", "op": "route", "tokens": 7, "experts": 8, "k": 2, "dtype": "fp32",
         "masked": False, "train": False},
        # one training step of the benchmark's MoE layer: 16384 tokens on one GPU
        {"name": "route_train", "op": "route", "tokens": 16384, "experts": 8, "k": 2, "dtype": "fp32",
         "masked": False, "train": True},
        # many small experts, low-precision logits, a padded batch
        {"name": "route_train_wide", "op": "route", "tokens": 65521, "experts": 256, "k": 8, "dtype": "bf16",
         "masked": True, "train": True},
        # the plan of a decode step
        {"name": "plan_decode", "op": "plan", "tokens": 61, "experts": 8, "k": 2, "masked": False},
        # the plan of the benchmark's largest MoE step: 64 experts, 131072 tokens
        {"name": "plan_large", "op": "plan", "tokens": 131072, "experts": 64, "k": 2, "masked": True},
        # gradients of the combine: a short odd batch, then the benchmark's MoE layer
        {"name": "combine_small", "op": "combine", "tokens": 1021, "experts": 8, "k": 2, "width": 2048},
        {"name": "combine_train", "op": "combine", "tokens": 16384, "experts": 8, "k": 2, "width": 5120},
        # a decode batch, every request with an adapter of its own, beside the up projection
        {"name": "lora_decode", "op": "lora", "form": "rows", "rows": 64, "segments": 64, "adapters": 64,
         "d_in": 5120, "d_out": 8192, "rank": 16},
        # one request alone, a large rank
        {"name": "lora_single", "op": "lora", "form": "rows", "rows": 1, "segments": 1, "adapters": 4,
         "d_in": 8192, "d_out": 5120, "rank": 64},
        # prompts of eight requests (or eight experts' groups) in one ragged batch, the sweep's row count
        {"name": "lora_prefill", "op": "lora", "form": "segments", "rows": 16640, "segments": 8, "adapters": 8,
         "d_in": 5120, "d_out": 8192, "rank": 32},
        # fine-tuning, a short odd batch whose segments share adapters
        {"name": "lora_train_small", "op": "lora", "form": "train", "rows": 1001, "segments": 5, "adapters": 3,
         "d_in": 2048, "d_out": 2048, "rank": 8},
        # fine-tuning every expert's up projection of the benchmark's MoE layer
        {"name": "lora_train", "op": "lora", "form": "train", "rows": 16384, "segments": 8, "adapters": 8,
         "d_in": 5120, "d_out": 8192, "rank": 16},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "plan", "combine", "lora", "lora"])
    if op == "route":
        experts = _log(rng, 2, 256)
        return {"op": op, "tokens": _log(rng, 1, 65521), "experts": experts, "k": rng.randint(1, min(8, experts)),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]) if experts <= 128 else rng.choice(["bf16", "fp16"]),
                "masked": rng.random() < 0.5, "train": rng.random() < 0.7}
    if op == "plan":
        experts = _log(rng, 2, 256)
        return {"op": op, "tokens": _log(rng, 1, 32768), "experts": experts, "k": rng.randint(1, min(8, experts)),
                "masked": rng.random() < 0.5}
    if op == "combine":
        k = rng.randint(1, 8)
        return {"op": op, "tokens": _log(rng, 1, 32768 // (k + 1)), "experts": _log(rng, k, 64), "k": k,
                "width": 8 * _log(rng, 16, 640)}
    form = rng.choice(["rows", "segments", "train"])
    case = {"op": op, "form": form, "d_in": 8 * _log(rng, 16, 640), "d_out": 8 * _log(rng, 16, 1024),
            "rank": rng.choice([8, 16, 24, 32, 48, 64])}
    if form == "rows":
        rows = _log(rng, 1, 256)
        case.update(rows=rows, segments=rows, adapters=_log(rng, 1, 64))
    else:
        rows = _log(rng, 32, 16000)
        if form == "train":
            case["rank"] = min(case["rank"], 16)
        case.update(rows=rows, segments=rng.randint(1, min(32, rows)), adapters=_log(rng, 1, 16))
    return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _experts(case, g):
    """Top-k choices of seeded logits; with `masked` the batch's padding tokens have none."""
    T, E, k = case["tokens"], case["experts"], case["k"]
    logits = torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    if case.get("masked"):
        experts[torch.rand(T, generator=g, device="cuda") < 0.1] = -1
    return experts.contiguous()


def _segments(case, seed):
    """Jagged cumulative ends that fill all rows (empty segments among them) and their adapters, on the host."""
    M, S, L = case["rows"], case["segments"], case["adapters"]
    rng = np.random.RandomState(seed % (1 << 31))
    if case["form"] == "rows":
        ends = np.arange(1, M + 1)
        adapter = rng.randint(0, L, M)
        adapter[1:][rng.rand(M - 1) < 0.05] = -1    # some requests have no adapter
    else:
        ends = np.sort(np.append(rng.randint(0, M + 1, S - 1), M))
        adapter = np.arange(S) % L
    return ends.astype(np.int32), adapter.astype(np.int32)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        logits = 1.5 * torch.randn(T, E, generator=g, device="cuda") + torch.randn(E, generator=g, device="cuda")
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        st["mask"] = (torch.rand(T, generator=g, device="cuda") < 0.9) if case["masked"] else None
        st["grad_w"] = torch.randn(T, k, generator=g, device="cuda")
    elif case["op"] == "plan":
        st["experts"] = _experts(case, g)
    elif case["op"] == "combine":
        T, k, N, E = case["tokens"], case["k"], case["width"], case["experts"]
        experts = _experts(case, g)
        w = torch.rand(T, k, generator=g, device="cuda") + 0.1
        st["weights"] = w / w.sum(1, keepdim=True)
        offs, counts, row_index, pair_pos = _plain_plan(experts, E)
        st["plan"] = (offs, counts, row_index, pair_pos)
        st["y"] = torch.randn(row_index.numel(), N, generator=g, device="cuda", dtype=torch.bfloat16)
        st["grad_out"] = torch.randn(T, N, generator=g, device="cuda", dtype=torch.bfloat16)
    else:
        M, L, K, N, R = case["rows"], case["adapters"], case["d_in"], case["d_out"], case["rank"]
        bf = torch.bfloat16
        st["x"] = torch.randn(M, K, generator=g, device="cuda", dtype=bf)
        st["a"] = (torch.randn(L, R, K, generator=g, device="cuda") * K ** -0.5).to(bf)
        st["b"] = (torch.randn(L, N, R, generator=g, device="cuda") * R ** -0.5).to(bf)
        st["scaling"] = 0.5 + torch.rand(L, generator=g, device="cuda")
        st["base"] = torch.randn(M, N, generator=g, device="cuda", dtype=bf)
        ends, adapter = _segments(case, seed)
        st["ends"], st["adapter"] = ends.tolist(), adapter.tolist()
        st["offs_d"] = torch.from_numpy(ends).cuda()
        st["adapter_d"] = torch.from_numpy(adapter).cuda()
        if case["form"] == "train":
            st["grad_out"] = torch.randn(M, N, generator=g, device="cuda", dtype=bf)
            st["grad_base"] = torch.randn(M, K, generator=g, device="cuda", dtype=bf)
    return st


# ------------------------------------------------------------- plain forms
def _plain_route(st):
    c = st["case"]
    E, k = c["experts"], c["k"]
    x = st["logits"].float()
    T = x.shape[0]
    on = st["mask"] if st["mask"] is not None else torch.ones(T, dtype=torch.bool, device=x.device)
    experts = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total)).squeeze(1)
    chosen = torch.gather(p, 1, experts)
    w = chosen / chosen.sum(1, keepdim=True)
    picks = torch.zeros(E + 1, dtype=torch.int64, device=x.device)
    slot = torch.where(on[:, None], experts, torch.full_like(experts, E)).reshape(-1)
    picks.index_add_(0, slot, torch.ones_like(slot))
    counts = picks[:E]
    n = on.sum().float().clamp(min=1)
    zero = torch.zeros((), device=x.device)
    mean = torch.where(on[:, None], p, zero).sum(0) / n
    frac = counts.float() / (n * k)
    balance = E * (frac * mean).sum()
    z = torch.where(on, lse * lse, zero).sum() / n
    out = {"experts": torch.where(on[:, None], experts, torch.full_like(experts, -1)).to(torch.int32),
           "weights": torch.where(on[:, None], w, zero), "counts": counts.to(torch.int32),
           "balance": balance, "z": z}
    if c["train"]:
        gw = st["grad_w"]
        dp = (BALANCE * E / n) * frac
        d = p * (dp - (p * dp).sum(1, keepdim=True)) + p * (ZLOSS * 2 * lse / n)[:, None]
        d = d.scatter_add(1, experts, w * (gw - (w * gw).sum(1, keepdim=True)))
        out["grad"] = torch.where(on[:, None], d, zero).to(st["logits"].dtype)
    return out


def _plain_plan(experts, E, pad=32):
    """(offs, counts, row_index, pair_pos): choices sorted by expert, every group padded to `pad` rows;
    row_index as long as the worst case, -1 in padding."""
    T, k = experts.shape
    pairs = T * k
    rows = (pairs + min(E, pairs) * (pad - 1)) // pad * pad
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    total = torch.zeros(E + 1, dtype=torch.int64, device=experts.device)
    total.index_add_(0, key, torch.ones_like(key))
    counts = total[:E]
    padded = (counts + pad - 1) // pad * pad
    offs = torch.cumsum(padded, 0)
    # a sentinel group for the choices that take no part
    start_pad = torch.cat([offs - padded, offs.new_zeros(1)])
    start = torch.cumsum(total, 0) - total
    by = key[order]
    pos = start_pad[by] + torch.arange(pairs, device=experts.device) - start[by]
    pos = torch.where(by == E, torch.full_like(pos, -1), pos)
    pair_pos = torch.empty_like(flat)
    pair_pos[order] = pos
    row_index = torch.full((rows + 1,), -1, dtype=torch.int32, device=experts.device)
    row_index[torch.where(pos < 0, torch.full_like(pos, rows), pos)] = (order // k).to(torch.int32)
    return offs.to(torch.int32), counts.to(torch.int32), row_index[:rows].clone(), pair_pos.reshape(T, k)


def _plain_combine(st):
    k = st["case"]["k"]
    _, _, row_index, pos = st["plan"]
    g, w = st["grad_out"].float(), st["weights"]
    grad_w = torch.stack([(g * st["y"][pos[:, j]].float()).sum(1) for j in range(k)], 1)
    grad_y = torch.zeros(row_index.numel(), g.shape[1], dtype=torch.bfloat16, device=g.device)
    for j in range(k):
        grad_y[pos[:, j]] = (w[:, j:j + 1] * g).to(torch.bfloat16)
    return {"grad_y": grad_y, "grad_weights": grad_w}


def _lora(st, dt, round_out):
    """The operator in the type `dt`, every output through `round_out` once."""
    c = st["case"]
    x, base = st["x"], st["base"]
    train = c["form"] == "train"
    out = torch.empty(base.shape, dtype=round_out or dt, device=x.device)
    if train:
        gx = torch.empty(x.shape, dtype=round_out or dt, device=x.device)
        ga = torch.zeros(st["a"].shape, dtype=dt, device=x.device)
        gb = torch.zeros(st["b"].shape, dtype=dt, device=x.device)
    if c["form"] == "rows":
        # one adapter a row: batched products over the gathered adapters
        sel = st["adapter_d"].long()
        step = max(1, (1 << 26) // (c["rank"] * max(c["d_in"], c["d_out"])))
        for i in range(0, c["rows"], step):
            s = sel[i:i + step]
            a, b = st["a"][s.clamp(min=0)].to(dt), st["b"][s.clamp(min=0)].to(dt)
            scale = torch.where(s < 0, torch.zeros_like(st["scaling"][:1]), st["scaling"][s.clamp(min=0)]).to(dt)
            u = torch.bmm(a, x[i:i + step].to(dt)[:, :, None]) * scale[:, None, None]
            out[i:i + step] = (base[i:i + step].to(dt) + torch.bmm(b, u)[:, :, 0]).to(out.dtype)
        return {"out": out}
    begin = 0
    scales = st["scaling"].to(dt)
    for end, l in zip(st["ends"], st["adapter"]):
        if end > begin:
            r = slice(begin, end)
            a, b, xs = st["a"][l].to(dt), st["b"][l].to(dt), x[r].to(dt)
            u = scales[l] * (xs @ a.t())
            out[r] = (base[r].to(dt) + u @ b.t()).to(out.dtype)
            if train:
                dy = st["grad_out"][r].to(dt)
                du = scales[l] * (dy @ b)
                gx[r] = (st["grad_base"][r].to(dt) + du @ a).to(gx.dtype)
                ga[l] += du.t() @ xs
                gb[l] += dy.t() @ u
        begin = end
    res = {"out": out}
    if train:
        res.update(grad_x=gx, grad_a=ga.to(round_out or dt), grad_b=gb.to(round_out or dt))
    return res


def run(st):
    c = st["case"]
    if own:
        moe, kernels = _package()
        if c["op"] == "route":
            r = moe.route_topk(st["logits"], c["k"], token_mask=st["mask"])
            out = {"experts": r.experts, "weights": r.weights, "counts": r.counts,
                   "balance": r.balance_loss, "z": r.z_loss}
            if c["train"]:
                out["grad"] = moe.route_topk_backward(st["logits"], r, st["grad_w"], BALANCE, ZLOSS)
            return out
        if c["op"] == "plan":
            p = moe.dispatch_plan(st["experts"], c["experts"])
            return {"offs": p.offs, "counts": p.counts, "row_index": p.row_index, "pair_pos": p.pair_pos}
        if c["op"] == "combine":
            _, _, row_index, pos = st["plan"]
            gy, gw = moe.combine_topk_backward(st["grad_out"], st["y"], pos, st["weights"], row_index)
            return {"grad_y": gy, "grad_weights": gw}
        if c["form"] == "rows":
            return {"out": kernels.lora_grouped_mm(st["x"], st["a"], st["b"], None, st["adapter_d"], st["scaling"],
                                                   base=st["base"])}
        if c["form"] == "segments":
            return {"out": kernels.lora_grouped_mm(st["x"], st["a"], st["b"], st["offs_d"], st["adapter_d"],
                                                   st["scaling"], base=st["base"])}
        out, v = kernels.lora_grouped_mm(st["x"], st["a"], st["b"], st["offs_d"], st["adapter_d"], st["scaling"],
                                         base=st["base"], return_v=True)
        gx, ga, gb = kernels.lora_grouped_mm_backward(st["grad_out"], st["x"], st["a"], st["b"], v, st["offs_d"],
                                                      st["adapter_d"], st["scaling"], grad_base=st["grad_base"])
        return {"out": out, "grad_x": gx, "grad_a": ga, "grad_b": gb}
    if c["op"] == "route":
        return _plain_route(st)
    if c["op"] == "plan":
        offs, counts, row_index, pair_pos = _plain_plan(st["experts"], c["experts"])
        return {"offs": offs, "counts": counts, "row_index": row_index, "pair_pos": pair_pos}
    if c["op"] == "combine":
        return _plain_combine(st)
    return _lora(st, torch.float32, torch.bfloat16)


# ------------------------------------------------------------------- exact
def _exact_route(case, st):
    """From the definition, in float64 on the host: softmax, the k largest (lowest index first among
    equals), their weights, both losses and the derivative of the objective to every logit."""
    x = st["logits"].double().cpu().numpy()
    T, E = x.shape
    k = case["k"]
    on = np.ones(T, bool) if st["mask"] is None else st["mask"].cpu().numpy()
    rows = np.arange(T)[:, None]
    experts = np.argsort(-x, axis=1, kind="stable")[:, :k]
    m = x.max(1)
    lse = m + np.log(np.exp(x - m[:, None]).sum(1))
    p = np.exp(x - lse[:, None])
    # the renormalised weights are a softmax over the chosen logits alone
    xc = x[rows, experts]
    w = np.exp(xc - xc[:, :1])
    w /= w.sum(1, keepdims=True)
    counts = np.bincount(experts[on].reshape(-1), minlength=E)
    n = max(1, int(on.sum()))
    frac = counts / (n * k)
    balance = E * float(frac @ p[on].sum(0)) / n
    z = float((lse[on] ** 2).sum()) / n
    out = {"experts": np.where(on[:, None], experts, -1).astype(np.int32), "weights": np.where(on[:, None], w, 0.0),
           "counts": counts.astype(np.int32), "balance": np.float64(balance), "z": np.float64(z)}
    if case["train"]:
        gw = st["grad_w"].double().cpu().numpy()
        grad = (BALANCE * E / n) * p * (frac[None, :] - (p @ frac)[:, None]) + (2 * ZLOSS / n) * lse[:, None] * p
        grad[rows, experts] += w * (gw - (w * gw).sum(1, keepdims=True))
        grad[~on] = 0.0
        out["grad"] = grad
    return out


def _exact_combine(case, st):
    _, _, row_index, pos = st["plan"]
    g = st["grad_out"].double()
    k = case["k"]
    y = st["y"].double()
    rows = row_index.numel()
    grad_y = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device)
    grad_w = torch.empty(g.shape[0], k, dtype=torch.float64, device=g.device)
    for j in range(k):
        grad_w[:, j] = torch.einsum("tn,tn->t", g, y.index_select(0, pos[:, j]))
        grad_y.index_copy_(0, pos[:, j], g * st["weights"][:, j].double()[:, None])
    return {"grad_y": grad_y, "grad_weights": grad_w}


def _exact_lora(case, st):
    """One adapter after another over the rows that carry it."""
    M = case["rows"]
    row_adapter = np.full(M, -1)
    begin = 0
    for end, l in zip(st["ends"], st["adapter"]):
        row_adapter[begin:end] = l
        begin = max(begin, end)
    out = st["base"].double()
    train = case["form"] == "train"
    if train:
        grad_x = st["grad_base"].double()
        grad_a = torch.zeros(st["a"].shape, dtype=torch.float64, device="cuda")
        grad_b = torch.zeros(st["b"].shape, dtype=torch.float64, device="cuda")
    for l in range(case["adapters"]):
        rows = torch.from_numpy(np.flatnonzero(row_adapter == l)).cuda()
        if rows.numel() == 0:
            continue
        a, b = st["a"][l].double(), st["b"][l].double()
        s = st["scaling"][l].double()
        x = st["x"].index_select(0, rows).double()
        u = torch.einsum("mk,rk->mr", x, a)
        out.index_add_(0, rows, s * torch.einsum("mr,nr->mn", u, b))
        if train:
            dy = st["grad_out"].index_select(0, rows).double()
            dyb = torch.einsum("mn,nr->mr", dy, b)
            grad_x.index_add_(0, rows, s * torch.einsum("mr,rk->mk", dyb, a))
            grad_a[l] = s * torch.einsum("mr,mk->rk", dyb, x)
            grad_b[l] = s * torch.einsum("mn,mr->nr", dy, u)
    res = {"out": out}
    if train:
        res.update(grad_x=grad_x, grad_a=grad_a, grad_b=grad_b)
    return res


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, st)
    if case["op"] == "plan":
        return None                                   # whole numbers: the plain form is the definition
    if case["op"] == "combine":
        return _exact_combine(case, st)
    return _exact_lora(case, st)


# -------------------------------------------------------------------- work
def work(case):
    """Bytes each input and output once, and the floating-point operations of the formulas."""
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        es = 4 if case["dtype"] == "fp32" else 2
        n = T * E * es + T * k * 8 + E * 4 + (T if case["masked"] else 0)
        f = 5 * T * E
        if case["train"]:
            n += T * E * es + T * k * 4
            f += 6 * T * E
        return {"bytes": n, "flops": f}
    if case["op"] == "plan":
        T, E, k = case["tokens"], case["experts"], case["k"]
        pairs = T * k
        rows = (pairs + min(E, pairs) * 31) // 32 * 32
        return {"bytes": pairs * 4 + pairs * 8 + rows * 4 + E * 8, "flops": 0}
    if case["op"] == "combine":
        T, E, k, N = case["tokens"], case["experts"], case["k"], case["width"]
        pairs = T * k
        rows = (pairs + min(E, pairs) * 31) // 32 * 32
        return {"bytes": 2 * N * (T + pairs + rows) + pairs * 16 + rows * 4, "flops": 3 * pairs * N}
    M, L, K, N, R = case["rows"], case["adapters"], case["d_in"], case["d_out"], case["rank"]
    used = min(L, case["segments"])
    n = 2 * (M * K + 2 * M * N + used * R * (K + N))
    f = 2 * M * R * (K + N)
    if case["form"] == "train":
        n += 2 * (M * N + 2 * M * K + L * R * (K + N))
        f *= 3
    return {"bytes": n, "flops": f}
