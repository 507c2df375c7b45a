"""Cases of the products whose rows choose their own weights: a projection with low-rank adapters, and a
mixture-of-experts layer for a few tokens. Each is written here in plain torch operations, too, which need
nothing of the package.

    lora   D = X W^T + scale[s] (X A_s^T) B_s^T with s = the row's adapter, -1 for none
    moe    y_t = sum_j w_tj W2_e (silu(G_e x_t) * (U_e x_t)) over the top_k experts e of token t's router logits;
           G_e and U_e are the halves of W13[e]

Inputs and outputs have 16 bits, sums 32 or more.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_PRODUCT = 4096 * 8192 * 8192     # rows x columns x depth of the largest projection
MOST_EXPERT_WEIGHTS = 64 * 3 * 2048 * 4096
_package = None


def package():
    global _package
    if _package is None:
        from __graft_entry__ import load_package
        _package = load_package()
    return _package


def lora(name, rows, n, k, rank, adapters, mix, dtype):
    return {"name": name, "op": "lora", "rows": rows, "n": n, "k": k, "rank": rank, "adapters": adapters, "mix": mix, "dtype": dtype}


def moe(name, tokens, hidden, inner, experts, top_k, normalise, logits, dtype):
    return {"name": name, "op": "moe", "tokens": tokens, "hidden": hidden, "inner": inner, "experts": experts, "top_k": top_k,
            "normalise": normalise, "logits": logits, "dtype": dtype}


def listed():
    return [
        # one user, one token: a square projection, where the latency of the call is what counts
        lora("lora_one_row", 1, 4096, 4096, 16, 8, "rows", "bf16"),
        # a decode step of 16 requests against the wide projection of a large model; any request may have any adapter
        lora("lora_decode_16", 16, 28672, 8192, 16, 32, "rows", "bf16"),
        # the same step on one of eight devices that share the columns, with a larger rank
        lora("lora_decode_16_shard", 16, 3584, 8192, 64, 32, "rows", "fp16"),
        # a decode step of 128 requests
        lora("lora_decode_128", 128, 28672, 8192, 32, 64, "rows", "bf16"),
        # odd sizes: no extent is a multiple of a tile
        lora("lora_odd", 77, 4104, 2056, 8, 5, "rows", "fp16"),
        # the prompts of eight requests behind one another
        lora("lora_prompts", 4096, 8192, 8192, 64, 8, "segments", "bf16"),
        # the smallest layer: two tokens, eight experts
        moe("moe_small", 2, 1024, 512, 8, 2, True, "fp32", "fp16"),
        # one token of a model with many narrow experts
        moe("moe_one_token", 1, 2048, 768, 128, 8, True, "fp32", "bf16"),
        # a decode step of 16 requests, wide experts, weights not normalised over the chosen ones
        moe("moe_decode_16", 16, 4096, 2048, 64, 6, False, "fp32", "bf16"),
        # odd sizes; the router's logits come from 16 bits, so some of them are equal
        moe("moe_odd", 37, 1000, 360, 20, 3, True, "bf16", "bf16"),
        # a decode step of 64 requests: every expert has a few tokens
        moe("moe_decode_64", 64, 4096, 1408, 64, 6, True, "bf16", "fp16"),
        # the most tokens that the layer takes at once
        moe("moe_decode_256", 256, 2048, 768, 128, 8, True, "fp32", "bf16"),
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    if rng.random() < 0.5:
        while True:
            rows, n, k = _log(rng, 1, 4096), _log(rng, 256, 28672, 8), _log(rng, 256, 8192, 8)
            if rows * n * k <= MOST_PRODUCT:
                break
        rank, adapters = _log(rng, 8, 128, 8), _log(rng, 1, 64)
        mix = "rows" if rows <= 256 and rng.random() < 0.8 else "segments"
        case = lora("", rows, n, k, rank, adapters, mix, dtype)
    else:
        while True:
            hidden, inner, experts = _log(rng, 256, 4096, 8), _log(rng, 128, 2048, 8), _log(rng, 4, 256)
            if experts * 3 * inner * hidden <= MOST_EXPERT_WEIGHTS:
                break
        case = moe("", _log(rng, 1, 256), hidden, inner, experts, rng.randint(1, min(8, experts)), rng.random() < 0.5,
                   rng.choice(["fp32", "bf16"]), dtype)
    del case["name"]
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=t).mul_(std)

    if case["op"] == "lora":
        m, n, k, r, s = case["rows"], case["n"], case["k"], case["rank"], case["adapters"]
        if case["mix"] == "rows":     # any row any adapter, or none
            ids = torch.randint(-1, s, (m,), generator=g, device="cuda", dtype=torch.int32)
        else:                         # one stretch of rows for each adapter, of odd lengths
            cuts = torch.randint(0, m + 1, (s - 1,), generator=g, device="cuda", dtype=torch.int32).sort()[0]
            ids = torch.searchsorted(cuts, torch.arange(m, device="cuda", dtype=torch.int32), right=True).to(torch.int32)
        return {"op": "lora", "x": normal(m, k), "w": normal(n, k, std=k ** -0.5), "a": normal(s, r, k, std=k ** -0.5),
                "b": normal(s, n, r, std=0.5 * r ** -0.5), "scale": torch.rand(s, generator=g, device="cuda") + 0.5, "ids": ids}
    n, h, i, e = case["tokens"], case["hidden"], case["inner"], case["experts"]
    logits = torch.randn(n, e, generator=g, device="cuda").mul_(1.5)
    if case["logits"] == "bf16":
        logits = logits.bfloat16().float()
    return {"op": "moe", "x": normal(n, h), "logits": logits, "w13": normal(e, 2 * i, h, std=h ** -0.5), "w2": normal(e, h, i, std=i ** -0.5),
            "top_k": case["top_k"], "normalise": case["normalise"]}


def run(state):
    if own:
        p = package()
        if state["op"] == "lora":
            return p.gemm_lora(state["x"], state["w"], state["a"], state["b"], state["ids"], state["scale"])
        return p.moe(state["x"], state["logits"], state["w13"], state["w2"], state["top_k"], normalise=state["normalise"])
    return plain_lora(state) if state["op"] == "lora" else plain_moe(state)


def plain_lora(state):
    """Every row against every adapter; what is not the row's own is masked out between the two products."""
    x, a, b, ids = state["x"].float(), state["a"], state["b"], state["ids"]
    s, r, k = a.shape
    u = (x @ a.reshape(s * r, k).float().t()).reshape(-1, s, r)
    mine = ids[:, None] == torch.arange(s, device=ids.device)[None]
    u = torch.where(mine[:, :, None], u * state["scale"][None, :, None], 0.0).reshape(-1, s * r)
    d = x @ state["w"].float().t() + u @ b.permute(0, 2, 1).reshape(s * r, -1).float()
    return d.to(state["x"].dtype)


def plain_moe(state):
    """With fewer picks than experts each pick's weights are gathered, else every expert sees every token."""
    x, logits, w13, w2, top_k = state["x"].float(), state["logits"], state["w13"], state["w2"], state["top_k"]
    tokens, experts, inner = x.shape[0], w13.shape[0], w2.shape[2]
    p = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    ids = logits.sort(dim=1, descending=True, stable=True)[1][:, :top_k]
    weights = p.gather(1, ids)
    if state["normalise"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    if tokens * top_k < experts:
        pick = ids.reshape(-1)
        z = torch.matmul(w13[pick].float(), x.repeat_interleave(top_k, dim=0)[:, :, None])[:, :, 0]
        h = z[:, :inner] / (1.0 + torch.exp(-z[:, :inner])) * z[:, inner:]
        o = torch.matmul(w2[pick].float(), h[:, :, None])[:, :, 0].reshape(tokens, top_k, -1)
        y = (o * weights[:, :, None]).sum(dim=1)
    else:
        z = torch.matmul(x[None], w13.float().transpose(1, 2))
        h = z[..., :inner] / (1.0 + torch.exp(-z[..., :inner])) * z[..., inner:]
        o = torch.matmul(h, w2.float().transpose(1, 2))
        mine = torch.zeros(tokens, experts, device=x.device).scatter_(1, ids, weights)
        y = (o * mine.t()[:, :, None]).sum(dim=0)
    return y.to(state["x"].dtype), ids.to(torch.int32), weights


def work(case):
    """Each input that the result depends on once, each output once. Which experts and adapters are used depends on the
    inputs: counted is the number expected of independent choices."""
    if case["op"] == "lora":
        m, n, k, r, s = case["rows"], case["n"], case["k"], case["rank"], case["adapters"]
        used = s * (1.0 - (1.0 - 1.0 / (s + 1)) ** m) if case["mix"] == "rows" else min(s, m)
        return {"bytes": 2.0 * (m * k + n * k + m * n + used * r * (n + k)) + 4.0 * (m + used), "flops": 2.0 * m * (n * k + r * (n + k))}
    n, h, i, e, k = case["tokens"], case["hidden"], case["inner"], case["experts"], case["top_k"]
    used = e * (1.0 - (1.0 - k / e) ** n)
    return {"bytes": 2.0 * (used * 3 * i * h + 2 * n * h) + 4.0 * n * e + 8.0 * n * k, "flops": 6.0 * n * k * i * h}


def exact(case, seed):
    """The definition in 64 bits, one adapter or expert after the other."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "lora":
        d = x @ s["w"].double().t()
        for j in range(case["adapters"]):
            rows = (s["ids"] == j).nonzero()[:, 0]
            d[rows] += s["scale"][j].double() * ((x[rows] @ s["a"][j].double().t()) @ s["b"][j].double().t())
        return d
    logits, top_k, inner = s["logits"].double().cpu(), case["top_k"], case["inner"]
    ids = torch.tensor([sorted(range(case["experts"]), key=lambda e: (-row[e], e))[:top_k] for row in logits.tolist()])
    chosen = logits.gather(1, ids)
    # log-sum-exp over what the weights are normalised over
    weights = torch.exp(chosen - torch.logsumexp(chosen if case["normalise"] else logits, dim=1, keepdim=True)).cuda()
    ids = ids.cuda()
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            z = x[t] @ s["w13"][e].double().t()
            y[t] += weights[t, j, None] * ((z[:, :inner] * torch.sigmoid(z[:, :inner]) * z[:, inner:]) @ s["w2"][e].double().t())
    return y, None, weights
