"""What is measured of the gated expert layer, its backward pass and the projection with low-rank adapters.

Three operators, each with a plain form (elementary torch operations in 32 bits) and the calls a user makes:

  gated   out = sum over a token's picks of gate * (act(x Wg) * (x Wu)) Wd            (serving)
  train   the same forward, then the gradients of x, the gates and the three weights  (a training step)
  lora    out = x W + scale[a] * (x A[a]^T) B[a], every token with the adapter a of its request, or none

Sizes follow the layer configurations of sparsebench_b200/workloads.py and, for the projection, the widths of the
same models.
"""

import math

import torch

own = False

ZIPF_EXPONENT = 1.2  # of the framework's skewed routing


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One new token of one sequence, fine-grained experts: latency of the smallest call.
        dict(name="gated_1_fine", op="gated", T=1, D=1024, F=4096, E=64, k=2, routing="random", act="silu"),
        # One decoding step of 37 sequences: every expert that is picked has one or two rows.
        dict(name="gated_37_fine", op="gated", T=37, D=1024, F=4096, E=64, k=2, routing="random", act="silu"),
        # A prefill batch of the headline layer.
        dict(name="gated_4096_fine", op="gated", T=4096, D=1024, F=4096, E=64, k=2, routing="random", act="silu"),
        # A ragged prefill batch over few large experts, with the erf GELU as the gate.
        dict(name="gated_1999_mixtral_like", op="gated", T=1999, D=4096, F=14336, E=8, k=2, routing="random", act="gelu"),
        # A small training step (the CPU-sized configuration with an odd batch).
        dict(name="train_333_small", op="train", T=333, D=256, F=1024, E=8, k=2, routing="random", act="silu"),
        # Training steps of the three benchmark layers: uniform, skewed with many experts, few large experts.
        dict(name="train_4096_fine", op="train", T=4096, D=1024, F=4096, E=64, k=2, routing="random", act="silu"),
        dict(name="train_4096_zipf", op="train", T=4096, D=2048, F=2048, E=128, k=2, routing="zipf", act="silu"),
        dict(name="train_4096_mixtral_like", op="train", T=4096, D=4096, F=14336, E=8, k=2, routing="random", act="silu"),
        # One new token of one request with an adapter.
        dict(name="lora_1", op="lora", T=1, D=4096, N=4096, r=16, L=8, requests=1, fp32=False),
        # One decoding step of 64 requests, most with an adapter of their own, into the wide projection.
        dict(name="lora_64_wide", op="lora", T=64, D=4096, N=14336, r=16, L=32, requests=64, fp32=False),
        # The router's projection of a prefill batch: few columns, logits in 32 bits.
        dict(name="lora_4096_router", op="lora", T=4096, D=1024, N=64, r=8, L=16, requests=23, fp32=True),
        # A prefill batch of 31 requests of very different lengths.
        dict(name="lora_8191", op="lora", T=8191, D=4096, N=4096, r=64, L=24, requests=31, fp32=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["gated", "gated", "train", "train", "lora", "lora"])
    if op == "lora":
        T = _spread(rng, 1, 8191)
        return dict(op=op, T=T, D=8 * _spread(rng, 32, 512), N=8 * _spread(rng, 4, 1792 if T < 2048 else 512),
                    r=8 * rng.choice([1, 2, 3, 4, 8]), L=_spread(rng, 1, 48), requests=_spread(rng, 1, min(T, 64)),
                    fp32=rng.random() < 0.25)
    E, D = _spread(rng, 2, 128), 128 * _spread(rng, 2, 32)
    F = 128 * _spread(rng, 2, max(2, min(112, (8 * 4096 * 14336) // (E * D * 128))))
    k = min(E, rng.choice([1, 2, 2, 3, 4]))
    return dict(op=op, T=_spread(rng, 1, 8192 // k), D=D, F=F, E=E, k=k, routing=rng.choice(["random", "zipf"]),
                act=rng.choice(["silu", "gelu"]))


# ---- inputs ------------------------------------------------------------------------------------------------------

def _popularity(case):
    E = case["E"]
    return torch.ones(E) if case["routing"] == "random" else torch.arange(1, E + 1, dtype=torch.float64) ** -ZIPF_EXPONENT


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16) * scale)

    T, D = case["T"], case["D"]
    if case["op"] == "lora":
        N, r, L, R = case["N"], case["r"], case["L"], case["requests"]
        # A batch is its requests' tokens one after another; a few requests have no adapter (-1).
        cuts = torch.randperm(T - 1, generator=g, device="cuda")[: R - 1].sort().values + 1 if T > 1 else torch.empty(0, device="cuda", dtype=torch.int64)
        request = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True)
        adapter = torch.randint(0, L, (R,), generator=g, device="cuda")
        adapter = torch.where(torch.rand(R, generator=g, device="cuda") < 0.1, torch.full_like(adapter, -1), adapter)
        return dict(case=case, x=normal(T, D), w=normal(D, N, scale=D**-0.5), a=normal(L, r, D, scale=D**-0.5),
                    b=normal(L, r, N, scale=r**-0.5), scale=torch.rand(L, generator=g, device="cuda") + 0.5,
                    adapter=adapter[request])
    E, F, k = case["E"], case["F"], case["k"]
    perm = torch.randperm(E, generator=g, device="cuda")
    chance = _popularity(case).to("cuda", torch.float32)[perm]
    # k picks without replacement with these chances: the k largest of log chance plus Gumbel noise.
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
    idx = (chance.log() + noise).topk(k, dim=-1).indices
    gate = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), dim=-1).bfloat16()
    return dict(case=case, x=normal(T, D), idx=idx, gate=gate, wg=normal(E, D, F, scale=D**-0.5),
                wu=normal(E, D, F, scale=D**-0.5), wd=normal(E, F, D, scale=F**-0.5),
                grad=normal(T, D) if case["op"] == "train" else None)


# ---- plain forms -------------------------------------------------------------------------------------------------

def _act(v, name):
    """(activation, its derivative) of v."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-v))
        return v * s, s * (1 + v * (1 - s))
    cdf = 0.5 * (1 + torch.erf(v * 0.5**0.5))
    return v * cdf, cdf + v * torch.exp(-0.5 * v * v) * (2 * math.pi) ** -0.5


def _plain_gated(s, train):
    x, gate, k, act = s["x"], s["gate"].float(), s["case"]["k"], s["case"]["act"]
    E = s["wg"].shape[0]
    flat = s["idx"].reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=E).tolist()
    token = order // k
    rows, w = x[token].float(), gate.reshape(-1)[order, None]
    y = torch.empty(rows.shape, device=x.device)
    if train:
        go = s["grad"][token].float()
        dx_rows, dgate_rows = torch.empty_like(y), torch.empty_like(w)
        dwg, dwu, dwd = (torch.zeros_like(s[n]) for n in ("wg", "wu", "wd"))
    at = 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        here = slice(at, at + n)
        at += n
        wg, wu, wd = s["wg"][e].float(), s["wu"][e].float(), s["wd"][e].float()
        u = rows[here] @ wu
        a, slope = _act(rows[here] @ wg, act)
        h = a * u
        y[here] = h @ wd
        if train:
            dgate_rows[here] = (go[here] * y[here]).sum(1, keepdim=True)
            dy = go[here] * w[here]
            dh = dy @ wd.T
            dg, du = dh * u * slope, dh * a
            dwd[e] = h.T @ dy
            dwg[e] = rows[here].T @ dg
            dwu[e] = rows[here].T @ du
            dx_rows[here] = dg @ wg.T + du @ wu.T
    back = torch.empty_like(order)
    back[order] = torch.arange(order.numel(), device=order.device)
    T, D = x.shape
    out = (y[back].view(T, k, D) * gate[..., None]).sum(1).to(x.dtype)
    if not train:
        return out
    return dict(out=out, dx=dx_rows[back].view(T, k, D).sum(1).to(x.dtype),
                dgate=dgate_rows[back].view(T, k).to(s["gate"].dtype), dwg=dwg, dwu=dwu, dwd=dwd)


def _plain_lora(s):
    x, a, b, ad = s["x"].float(), s["a"], s["b"], s["adapter"]
    L, r, _ = a.shape
    base = x @ s["w"].float()
    factor = torch.where(ad >= 0, s["scale"][ad.clamp(min=0)], torch.zeros_like(ad, dtype=torch.float32))[:, None]
    if x.shape[0] <= 64:  # few tokens: each with its own adapter's rows
        pick = ad.clamp(min=0)
        v = (a[pick].float() * x[:, None, :]).sum(-1) * factor
        low = (v[..., None] * b[pick].float()).sum(1)
    else:  # many: all adapters side by side, those of other requests masked
        v = (x @ a.reshape(L * r, -1).float().T).view(-1, L, r) * factor[..., None]
        mine = ad[:, None] == torch.arange(L, device=ad.device)
        v = torch.where(mine[..., None], v, torch.zeros_like(v))
        low = v.reshape(-1, L * r) @ b.reshape(L * r, -1).float()
    return (base + low).to(torch.float32 if s["case"]["fp32"] else s["x"].dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        import sparsebench_b200 as sb

        if case["op"] == "lora":
            return sb.lora_linear(s["x"], s["w"], s["a"], s["b"], s["adapter"], scale=s["scale"],
                                  out_dtype=torch.float32 if case["fp32"] else torch.bfloat16)
        if case["op"] == "gated":
            return sb.moe_forward_gated(s["x"], s["idx"], s["gate"], s["wg"], s["wu"], s["wd"], activation=case["act"])
        out, saved = sb.moe_forward_gated_saved(s["x"], s["idx"], s["gate"], s["wg"], s["wu"], s["wd"],
                                                activation=case["act"])
        g = sb.moe_backward_gated(s["grad"], saved)
        return dict(out=out, dx=g.x, dgate=g.expert_weight, dwg=g.w_gate, dwu=g.w_up, dwd=g.w_down)
    if case["op"] == "lora":
        return _plain_lora(s)
    return _plain_gated(s, case["op"] == "train")


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    T, D = case["T"], case["D"]
    if case["op"] == "lora":
        N, r = case["N"], case["r"]
        used = min(case["L"], case["requests"])
        return {"bytes": 2 * (T * D + D * N + used * r * (D + N)) + T * N * (4 if case["fp32"] else 2) + 8 * T,
                "flops": 2 * T * D * N + 2 * T * r * (D + N)}
    E, F, k = case["E"], case["F"], case["k"]
    p = _popularity(case)
    p = (p / p.sum() * k).clamp(max=1.0)
    used = float((1 - (1 - p.double()) ** T).sum())  # experts that some token picks, about
    weights, flops = 2 * 3 * used * D * F, 6 * T * k * D * F
    if case["op"] == "gated":
        return {"bytes": weights + 2 * 2 * T * D + T * k * 10, "flops": flops}
    return {"bytes": weights + 2 * 3 * E * D * F + 2 * 4 * T * D + T * k * 12, "flops": 3 * flops}


# ---- the operators' definitions in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        x, w = s["x"].double(), s["w"].double()
        out = x @ w
        for a in range(case["L"]):
            rows = torch.nonzero(s["adapter"] == a).flatten()
            out[rows] += s["scale"][a].double() * (x[rows] @ s["a"][a].double().T @ s["b"][a].double())
        return out
    train = case["op"] == "train"
    leaves = [s[n].double().requires_grad_(train) for n in ("x", "gate", "wg", "wu", "wd")]
    x, gate = leaves[:2]
    wg, wu, wd = (w.unbind() for w in leaves[2:])
    act = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
    out = torch.zeros_like(x)
    for e in range(case["E"]):
        t, j = torch.nonzero(s["idx"] == e, as_tuple=True)
        if t.numel():
            h = act(x[t] @ wg[e]) * (x[t] @ wu[e])
            out = out.index_add(0, t, gate[t, j, None] * (h @ wd[e]))
    if not train:
        return out
    names = ("dx", "dgate", "dwg", "dwu", "dwd")
    return dict(zip(names, torch.autograd.grad(out, leaves, s["grad"].double())), out=out.detach())
