"""Cases of the operators beside frozen MXFP4 weights: low-rank adapters of many requests, the input gradient of a linear layer, the
router of an expert MLP with its balance loss, and the weighted sum of the experts' rows.

`own` false: `run` is the operator in elementary torch operations (32-bit arithmetic, rounded once). `own` true: the calls that a user of
wave_b200 makes. `exact` is the definition in 64 bits.
"""

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "f32": F32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # serving: one token of one request, the smallest call of a decode step
        dict(name="adapters one token", op="adapters", train=False, rows=1, K=4096, N=4096, rank=16, pool=8, ids="mixed", y="bf16"),
        # serving: a decode step of 32 requests with an adapter each, some without, beside a wide projection
        dict(name="adapters decode of 32", op="adapters", train=False, rows=32, K=4096, N=14336, rank=16, pool=64, ids="mixed", y="bf16"),
        # serving: a ragged prefill of several short requests, odd output width and rank, f32 output
        dict(name="adapters ragged f32", op="adapters", train=False, rows=600, K=1024, N=4001, rank=12, pool=9, ids="runs", y="f32"),
        # serving: a long prefill of a few requests with adapters of high rank
        dict(name="adapters prefill", op="adapters", train=False, rows=8192, K=8192, N=8192, rank=64, pool=6, ids="runs", y="bf16"),
        # fine-tuning one adapter: forward and the gradients of x, a and b
        dict(name="adapters training", op="adapters", train=True, rows=4096, K=4096, N=4096, rank=16, pool=1, ids="runs", y="bf16"),
        # fine-tuning several adapters in one batch, ragged
        dict(name="adapters training of 5", op="adapters", train=True, rows=1111, K=2048, N=5120, rank=32, pool=5, ids="runs", y="bf16"),
        # fine-tuning: the gradient through a frozen layer, a short batch over an odd number of rows
        dict(name="input gradient ragged", op="input_grad", rows=600, N=4000, K=2048),
        # the same for a large batch and weight
        dict(name="input gradient large", op="input_grad", rows=8192, N=8192, K=8192),
        # routing of a decode step: latency
        dict(name="router decode", op="router", train=False, rows=16, experts=8, top_k=2, logits="bf16", padded=False, renormalize=False),
        # routing of a training batch with many experts, padded sequences, with the gradient of weights and balance loss
        dict(name="router training", op="router", train=True, rows=8192, experts=256, top_k=8, logits="f32", padded=True, renormalize=True),
        # the sum of the experts' rows of a training batch, with the gradient of the routing weights
        dict(name="combine training", op="combine", rows=4096, N=4096, top_k=2),
        # the same for few tokens and more experts a token, with pairs that were dropped
        dict(name="combine short", op="combine", rows=130, N=2048, top_k=6),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(("adapters", "adapters", "adapters", "input_grad", "router", "combine"))
    if op == "adapters":
        train = rng.random() < 0.4
        K = 32 * _spread(rng, 4, 256)
        N = _spread(rng, 64, 14336)
        if rng.random() < 0.6:
            N = -(-N // 32) * 32
        rows = min(_spread(rng, 16 if train else 1, 8192), (8192 * 8192) // max(K, N))
        rank = rng.choice((4, 8, 8, 12, 16, 16, 16, 32, 32, 64, 64, 100, 128))
        pool = _spread(rng, 1, max(1, min(64, 300000 // (rows * rank) if rows > 512 else 64)))
        if train:
            rows, pool = min(rows, 4096), min(pool, 8)
            rows = min(rows, (4096 * 4096) // max(K, N) * 2)
            rank = min(rank, 64)
        return dict(op=op, train=train, rows=rows, K=K, N=N, rank=rank, pool=pool, ids=rng.choice(("runs", "mixed")),
                    y="bf16" if train else rng.choice(("bf16", "bf16", "f32")))
    if op == "input_grad":
        rows, N, K = _spread(rng, 1, 8192), 8 * _spread(rng, 16, 1024), 32 * _spread(rng, 4, 256)
        return dict(op=op, rows=rows, N=N, K=K)
    if op == "router":
        experts = _spread(rng, 2, 256)
        return dict(op=op, train=rng.random() < 0.6, rows=_spread(rng, 1, 16384), experts=experts, top_k=min(experts, rng.choice((1, 2, 2, 4, 6, 8))),
                    logits=rng.choice(("f32", "bf16")), padded=rng.random() < 0.5, renormalize=rng.random() < 0.5)
    N = _spread(rng, 64, 8192)
    if rng.random() < 0.7:
        N = -(-N // 8) * 8
    return dict(op=op, rows=_spread(rng, 1, 4096), N=N, top_k=rng.choice((1, 2, 2, 4, 6)))


def _ids(case, gen):
    """Adapter of every row, -1 for none: sequences one behind another ("runs"), or a choice for each row ("mixed")."""
    rows, pool = case["rows"], case["pool"]
    if case["ids"] == "mixed":
        ids = torch.randint(0, pool, (rows,), generator=gen, device="cuda")
        return torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.1, -1 if rows > 1 else ids, ids).to(torch.int32)
    cuts = torch.sort(torch.randint(0, rows + 1, (pool - 1,), generator=gen, device="cuda")).values
    order = torch.randperm(pool, generator=gen, device="cuda")
    at = (torch.arange(rows, device="cuda")[:, None] >= cuts[None, :]).sum(1)
    return order[at].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, dtype=BF16, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    op, rows = case["op"], case["rows"]
    state = dict(case=case)
    if op == "adapters":
        K, N, r, pool = case["K"], case["N"], case["rank"], case["pool"]
        state.update(x=normal(rows, K), y=normal(rows, N, dtype=DTYPES[case["y"]]), a=normal(pool, r, K, std=K ** -0.5), b=normal(pool, N, r, std=0.3),
                     scale=torch.rand(pool, generator=gen, device="cuda") * 1.5 + 0.5, ids=_ids(case, gen))
        if case["train"]:
            state.update(g=normal(rows, N, std=1e-2))
            for name in ("x", "a", "b"):
                state[name].requires_grad_()
    elif op == "input_grad":
        K, N = case["K"], case["N"]
        # a weight of normal values, quantised: per 32 values of a row a power of two, and the nearest of the sixteen values
        w = normal(N, K // 32, 32, dtype=F32, std=K ** -0.5)
        exponent = torch.floor(torch.log2(w.abs().amax(-1, keepdim=True))) - 2
        size = (w / torch.exp2(exponent)).abs()
        codes = torch.bucketize(size, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")) + 8 * (w < 0)
        codes = codes.to(torch.uint8).reshape(N, K // 2, 2)
        state.update(codes=(codes[..., 0] | codes[..., 1] << 4).contiguous(), scales=(exponent.reshape(N, K // 32) + 127).to(torch.uint8),
                     g=normal(rows, N, std=1e-2))
    elif op == "router":
        E, k = case["experts"], case["top_k"]
        logits = normal(rows, E, dtype=DTYPES[case["logits"]]) + normal(E, dtype=DTYPES[case["logits"]], std=0.5)
        mask = None
        if case["padded"]:  # eight sequences of one padded length each
            length = -(-rows // 8)
            kept = torch.randint(length // 2, length + 1, (8,), generator=gen, device="cuda")
            mask = (torch.arange(length, device="cuda")[None, :] < kept[:, None]).reshape(-1)[:rows].contiguous()
        state.update(logits=logits, mask=mask)
        if case["train"]:
            logits.requires_grad_()
            state.update(g_weight=normal(rows, k, dtype=F32), g_loss=torch.rand((), generator=gen, device="cuda") + 0.01)
    else:
        N, k = case["N"], case["top_k"]
        n = rows * k
        row_of = torch.randperm(n + n // 4 + 8, generator=gen, device="cuda")[:n]
        row_of = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.02, -1, row_of).to(torch.int32).reshape(rows, k)
        state.update(y=normal(n + n // 4 + 8, N), row_of=row_of, weight=torch.rand(rows, k, generator=gen, device="cuda").requires_grad_(),
                     g=normal(rows, N, std=1e-2))
    return state


def _plain_adapters(s):
    case = s["case"]
    pool, r, K, N = case["pool"], case["rank"], case["K"], case["N"]
    x, a, b = s["x"].detach().float(), s["a"].detach().float().reshape(pool * r, K), s["b"].detach().float()
    b = b.permute(0, 2, 1).reshape(pool * r, N)
    # every adapter's rows of a and b side by side; a row of x keeps the columns of its own adapter
    chosen = (s["ids"][:, None] == torch.arange(pool, device="cuda")[None, :]).float() * s["scale"][None, :]
    chosen = chosen[:, :, None].expand(-1, -1, r).reshape(-1, pool * r)
    v = (x @ a.T) * chosen
    out = (s["y"].float() + v @ b).to(s["y"].dtype)
    if not case["train"]:
        return out
    g = s["g"].float()
    u = (g @ b.T) * chosen
    return dict(out=out, x=(u @ a).to(BF16), a=(u.T @ x).reshape(pool, r, K).to(BF16), b=(g.T @ v).reshape(N, pool, r).permute(1, 0, 2).contiguous().to(BF16))


def _plain_input_grad(s):
    case = s["case"]
    table = torch.tensor(E2M1, device="cuda")
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=-1).int()
    w = table[codes].reshape(case["N"], case["K"] // 32, 32) * torch.exp2(s["scales"].float() - 127)[:, :, None]
    return (s["g"].float() @ w.reshape(case["N"], case["K"])).to(BF16)


def _plain_router(s):
    case = s["case"]
    E, k = case["experts"], case["top_k"]
    z = s["logits"].detach().float()
    valid = torch.ones(case["rows"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    e = torch.exp(z - z.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True) * valid[:, None]
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    ids = torch.where(valid[:, None], order, -1)
    chosen = torch.gather(p, 1, order)
    total = chosen.sum(1, keepdim=True)
    weight = torch.where(valid[:, None], chosen / total, 0.0) if case["renormalize"] else chosen
    picked = torch.zeros_like(p).scatter_(1, order, 1.0) * valid[:, None]
    counts = picked.sum(0).to(torch.int32)
    tokens = valid.sum().clamp(min=1).float()
    share = counts.float() / (k * tokens)
    loss = E * (share * p.sum(0) / tokens).sum()
    out = dict(weight=weight, ids=ids.to(torch.int32), counts=counts, loss=loss)
    if not case["train"]:
        return out
    # gradient by the probabilities, then through the softmax
    gp = (s["g_loss"] * E / tokens * share)[None, :].expand_as(p).clone()
    gw = s["g_weight"]
    if case["renormalize"]:
        gw = torch.where(valid[:, None], (gw - (gw * weight).sum(1, keepdim=True)) / total, 0.0)
    gp = gp + torch.zeros_like(p).scatter_(1, order, gw)
    out["logits"] = (p * (gp - (p * gp).sum(1, keepdim=True))).to(s["logits"].dtype)
    return out


def _plain_combine(s):
    row_of, weight = s["row_of"].long(), s["weight"].detach()
    kept = row_of >= 0
    rows = s["y"].float()[row_of.clamp(min=0)] * kept[:, :, None]
    out = (rows * weight[:, :, None]).sum(1).to(BF16)
    return dict(out=out, weight=(rows * s["g"].float()[:, None, :]).sum(2))


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        with torch.no_grad():
            return dict(adapters=_plain_adapters, input_grad=_plain_input_grad, router=_plain_router, combine=_plain_combine)[op](s)
    import wave_b200 as wb

    if op == "adapters":
        out = wb.apply_adapters(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scale"])
        if not case["train"]:
            return out
        gx, ga, gb = torch.autograd.grad(out, (s["x"], s["a"], s["b"]), s["g"])
        return dict(out=out, x=gx, a=ga, b=gb)
    if op == "input_grad":
        return wb.mxfp4_input_grad(s["g"], s["codes"], s["scales"])
    if op == "router":
        r = wb.router(s["logits"], case["top_k"], mask=s["mask"], renormalize=case["renormalize"])
        out = dict(weight=r.weight, ids=r.ids, counts=r.counts, loss=r.balance_loss)
        if case["train"]:
            out["logits"], = torch.autograd.grad((r.weight, r.balance_loss), s["logits"], (s["g_weight"], s["g_loss"]))
        return out
    out = wb.combine_rows(s["y"], s["row_of"], s["weight"])
    return dict(out=out, weight=torch.autograd.grad(out, s["weight"], s["g"])[0])


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "adapters":
        K, N, r, pool = case["K"], case["N"], case["rank"], case["pool"]
        used = pool * (1 - (1 - 1 / pool) ** rows)  # adapters that some row asks for, on average
        size = 2 if case["y"] == "bf16" else 4
        data = rows * (2 * K + 2 * size * N) + 2 * used * r * (K + N) + 4 * rows
        flops = 2 * rows * r * (K + N)
        if case["train"]:
            data += rows * (2 * K + 2 * N) + 2 * pool * r * (K + N)
            flops *= 3
        return dict(bytes=data, flops=flops)
    if op == "input_grad":
        N, K = case["N"], case["K"]
        return dict(bytes=2 * rows * (N + K) + N * K // 2 + N * K // 32, flops=2 * rows * N * K)
    if op == "router":
        E, k = case["experts"], case["top_k"]
        size = 2 if case["logits"] == "bf16" else 4
        data = rows * (E * size + 8 * k) + 4 * E
        if case["train"]:
            data += rows * (E * size + 4 * k)
        return dict(bytes=data, flops=rows * E * (10 if case["train"] else 4))
    N, k = case["N"], case["top_k"]
    return dict(bytes=2 * rows * N * (k + 2) + 12 * rows * k, flops=4 * rows * N * k)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "adapters":
            x, out = s["x"].double(), s["y"].double()
            gx, ga, gb = torch.zeros_like(x), torch.zeros_like(s["a"], dtype=F64), torch.zeros_like(s["b"], dtype=F64)
            for i in range(case["pool"]):
                at = (s["ids"] == i).nonzero()[:, 0]
                a, b, scale = s["a"][i].double(), s["b"][i].double(), s["scale"][i].double()
                v = x[at] @ a.T
                out[at] += scale * (v @ b.T)
                if case["train"]:
                    u = scale * (s["g"][at].double() @ b)
                    gx[at] = u @ a
                    ga[i] = u.T @ x[at]
                    gb[i] = scale * (s["g"][at].double().T @ v)
            return dict(out=out, x=gx, a=ga, b=gb) if case["train"] else out
        if op == "input_grad":
            N, K = case["N"], case["K"]
            w = torch.empty(N, K, dtype=F64, device="cuda")
            for half, nibble in enumerate((s["codes"] & 15, s["codes"] >> 4)):
                w[:, half::2] = torch.tensor(E2M1, dtype=F64, device="cuda")[nibble.int()]
            w *= torch.repeat_interleave(torch.pow(2.0, s["scales"].double() - 127), 32, dim=1)
            return s["g"].double() @ w
        if op == "router":
            E, k = case["experts"], case["top_k"]
            z = s["logits"].detach().double()
            valid = torch.ones(case["rows"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
            z.requires_grad_()
            with torch.enable_grad():
                p = torch.softmax(z, dim=1)
                # k times the largest of what is left, the lowest index first among equals
                left, ids = z.detach().clone(), []
                for _ in range(k):
                    best = left.amax(1, keepdim=True)
                    first = torch.where(left == best, torch.arange(E, device="cuda")[None, :], E).amin(1, keepdim=True)
                    ids.append(first)
                    left = left.scatter(1, first, float("-inf"))
                ids = torch.cat(ids, 1)
                weight = torch.gather(p, 1, ids)
                if case["renormalize"]:
                    weight = weight / weight.sum(1, keepdim=True)
                weight = weight * valid[:, None]
                counts = torch.bincount(ids[valid].reshape(-1), minlength=E)
                tokens = max(1, int(valid.sum()))
                loss = E * ((counts.double() / (k * tokens)) * (p * valid[:, None]).sum(0) / tokens).sum()
                out = dict(weight=weight.detach(), ids=None, counts=None, loss=loss.detach())
                if case["train"]:
                    total = (weight * s["g_weight"].double()).sum() + loss * s["g_loss"].double()
                    out["logits"], = torch.autograd.grad(total, z)
            return out
        y, g, weight = s["y"].double(), s["g"].double(), s["weight"].detach().double()
        out, gw = torch.zeros(case["rows"], case["N"], dtype=F64, device="cuda"), torch.zeros_like(weight)
        for j in range(case["top_k"]):
            row = s["row_of"][:, j].long()
            part = y[row.clamp(min=0)]
            part[row < 0] = 0
            out += weight[:, j, None] * part
            gw[:, j] = (part * g).sum(1)
        return dict(out=out, weight=gw)
