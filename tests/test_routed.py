"""Products whose rows choose their own weights: a projection with low-rank adapters (b200_gemm_lora) and a
mixture-of-experts layer for a few tokens (b200_moe), against their definitions in 64 bits.

Tolerances. A result is rounded once to 16 bits: at most eps/2 of its value (2^-25 absolute below fp16's normal range).
An fp32 sum of n products errs by at most (n/16 + 64) * 2^-22 of the sum of their magnitudes: the tensor core adds 16
products per step, each step loses at most two units of 2^-23 of the magnitudes summed so far, and 64 covers the
additions outside (splits of the depth, warps, the few steps of the joins). Intermediate values kept as a pair of 16-bit
numbers err by at most eps^2/4 of their value (a rounding of a rounding), bounded here by 2^-16 for bf16 and fp16 alike."""
import numpy as np
import pytest

from helpers import Guarded

EPS = {"bf16": 2.0 ** -7, "fp16": 2.0 ** -10}


def dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def gamma(n):
    return (n / 16 + 64) * 2.0 ** -22


def check_close(got, want, slack, name):
    """|got - want| <= slack + half a step of the rounding, everywhere."""
    got, half = got.double(), EPS[name] / 2
    bound = slack * (1 + half) + half * want.abs() + 2.0 ** -25
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{float(((got - want).abs() / bound).nan_to_num(float('inf')).max()):.3g} times the bound, first at {bad.nonzero()[0].tolist()}")


# ------------------------------------------------------------------------------------------------ adapters

def lora_inputs(torch, name, m, n, k, r, s, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    t = dt(torch, name)
    rnd = lambda *sh, std=1.0: (torch.randn(*sh, generator=g, device=device) * std).to(t)
    return rnd(m, k), rnd(n, k, std=k ** -0.5), rnd(s, r, k, std=k ** -0.5), rnd(s, n, r, std=r ** -0.5), torch.rand(s, generator=g, device=device) + 0.5


def lora_want(torch, x, w, a, b, ids, scale):
    """The definition in 64 bits, and a bound of what fp32 sums may lose."""
    x, w, (s, r, k) = x.double(), w.double(), a.shape
    d, mag = x @ w.t(), x.abs() @ w.t().abs()
    slack = gamma(k) * mag
    for j in range(s):
        rows = (ids == j).nonzero()[:, 0]
        if rows.numel():
            f = 1.0 if scale is None else float(scale[j])
            aj, bj = a[j].double(), b[j].double()
            u, um = x[rows] @ aj.t(), x[rows].abs() @ aj.t().abs()
            d[rows] += f * (u @ bj.t())
            slack[rows] += f * ((gamma(k) + gamma(r) + 2.0 ** -16) * um) @ bj.t().abs()
    return d, slack


def run_lora(pkg, torch, x, w, a, b, ids, scale):
    (m, k), n, (s, r) = x.shape, w.shape[0], a.shape[:2]
    D = Guarded(torch, (m, n), x.dtype)
    W = Guarded(torch, (pkg.gemm_lora_workspace_bytes(m, n, k, s, r),), torch.uint8, fill=0xFF, band_bytes=1 << 16)
    out = pkg.gemm_lora(x, w, a, b, ids, scale, D=D.t, workspace=W.t)
    assert out is D.t
    st, info = pkg.device_status()
    assert st == pkg.OK, (st, info)
    D.check("D")
    W.check("workspace")
    return out


LORA = [  # m, n, k, rank, adapters, order of the ids
    (1, 8, 8, 8, 1, "all"), (1, 264, 72, 8, 3, "mixed"), (1, 4096, 1024, 16, 4, "mixed"), (2, 136, 4104, 128, 2, "mixed"),
    (5, 1000, 520, 24, 7, "mixed"), (16, 2048, 2048, 16, 16, "each"), (17, 328, 264, 40, 3, "none"), (31, 512, 1032, 8, 2, "stretches"),
    (33, 1544, 136, 72, 5, "mixed"), (64, 776, 968, 64, 64, "each"), (65, 256, 512, 16, 3, "stretches"), (100, 2056, 264, 8, 9, "mixed"),
    (128, 1032, 2048, 32, 128, "each"), (129, 640, 328, 16, 2, "mixed"), (200, 264, 1096, 56, 6, "stretches"), (256, 520, 64, 128, 4, "mixed"),
    (257, 384, 456, 24, 3, "mixed"), (300, 1288, 712, 16, 5, "stretches"), (513, 904, 1024, 64, 4, "stretches"), (1000, 256, 264, 8, 300, "mixed"),
    (1030, 2056, 520, 32, 3, "stretches"),
]


def lora_ids(torch, order, m, s, seed):
    g = torch.Generator().manual_seed(seed)
    if order == "all":
        ids = torch.zeros(m, dtype=torch.int32)
    elif order == "none":
        ids = torch.tensor([-1, s, -2 ** 31, 2 ** 31 - 1], dtype=torch.int64).repeat(m // 4 + 1)[:m].to(torch.int32)
    elif order == "each":
        ids = torch.randperm(s, generator=g)[torch.arange(m) % s].to(torch.int32)
    elif order == "stretches":
        ids = (torch.randint(0, s + 1, (m,), generator=g).sort()[0] - 1).to(torch.int32)
    else:
        ids = torch.randint(-1, s + 1, (m,), generator=g).to(torch.int32)      # s itself: out of range, no adapter
    return ids.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("case", LORA, ids=lambda c: "x".join(map(str, c)))
def test_lora_against_64_bits(pkg, cuda, case, name):
    m, n, k, r, s, order = case
    x, w, a, b, scale = lora_inputs(cuda, name, m, n, k, r, s, m + n)
    ids = lora_ids(cuda, order, m, s, m * 7 + r)
    scale = scale if m % 2 else None
    got = run_lora(pkg, cuda, x, w, a, b, ids, scale)
    check_close(got, *lora_want(cuda, x, w, a, b, ids, scale), name)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 300])
def test_lora_reads_nothing_of_adapters_and_rows_that_are_not_a_rows_own(pkg, cuda, m):
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, "bf16", m, 520, 264, 16, 5, 3)
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % 2 + 1               # adapters 1 and 2 only
    ids[m // 2] = -1
    clean = run_lora(pkg, torch, x, w, a, b, ids, scale)
    for j in (0, 3, 4):
        a[j], b[j], scale[j] = float("nan"), float("inf"), float("nan")
    assert torch.equal(run_lora(pkg, torch, x, w, a, b, ids, scale), clean)
    # an adapter's infinity stays with its rows, an input's NaN with its row
    b[2, 7] = float("inf")
    x[0, 5] = float("nan")
    got = run_lora(pkg, torch, x, w, a, b, ids, scale)
    assert got[0].isnan().all()
    rows = torch.arange(m, device="cuda")
    own = (ids == 2) & (rows > 0)
    assert not got[own, 7].isfinite().any()
    got[own, 7] = clean[own, 7]
    assert torch.equal(got[1:], clean[1:])


@pytest.mark.gpu
def test_lora_without_adapters_is_the_plain_product_and_calls_repeat_bit_for_bit(pkg, cuda):
    torch = cuda
    for m in (4, 90, 400):
        x, w, a, b, scale = lora_inputs(torch, "fp16", m, 648, 904, 32, 3, m)
        none = torch.full((m,), -1, dtype=torch.int32, device="cuda")
        base = run_lora(pkg, torch, x, w, a, b, none, scale)
        zero = torch.zeros_like(b)
        ids = lora_ids(torch, "mixed", m, 3, m)
        assert torch.equal(run_lora(pkg, torch, x, w, a, zero, ids, scale), base)
        first = run_lora(pkg, torch, x, w, a, b, ids, scale)
        for _ in range(5):
            assert torch.equal(run_lora(pkg, torch, x, w, a, b, ids, scale), first)


# ------------------------------------------------------------------------------------------------ experts

def moe_inputs(torch, name, tokens, hidden, inner, experts, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *sh, std=1.0: (torch.randn(*sh, generator=g, device="cuda") * std).to(dt(torch, name))
    logits = torch.randn(tokens, experts, generator=g, device="cuda") * 1.5
    return rnd(tokens, hidden), logits, rnd(experts, 2 * inner, hidden, std=hidden ** -0.5), rnd(experts, hidden, inner, std=inner ** -0.5)


def route_want(torch, logits, top_k, normalise):
    """One token after the other, in Python's numbers."""
    ids, weights = [], []
    for row in logits.double().cpu().tolist():
        row = [min(v, float(np.finfo(np.float32).max)) if v == v else -np.inf for v in row]
        pick = [e for e in sorted(range(len(row)), key=lambda e: (-row[e], e))[:top_k] if row[e] > -np.inf]
        top = max(row)
        total = sum(np.exp(row[e] - top) for e in (pick if normalise else range(len(row))) if row[e] > -np.inf)
        ids.append(pick + [-1] * (top_k - len(pick)))
        weights.append([np.exp(row[e] - top) / total for e in pick] + [0.0] * (top_k - len(pick)))
    return torch.tensor(ids, dtype=torch.int32).cuda(), torch.tensor(weights, dtype=torch.float64).cuda()


def moe_want(torch, x, w13, w2, ids, weights):
    x, inner = x.double(), w2.shape[2]
    y, slack = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(w13.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        a, b, p = w13[e].double(), w2[e].double(), weights[t, j, None]
        z, dz = x[t] @ a.t(), gamma(x.shape[1]) * (x[t].abs() @ a.t().abs())
        g, u, dg, du = z[:, :inner], z[:, inner:], dz[:, :inner], dz[:, inner:]
        silu = g * torch.sigmoid(g)
        # the slope of silu is at most 1.1; its exponential and division err by a few units of 2^-23
        dh = 1.1 * dg * (u.abs() + du) + silu.abs() * du + (2.0 ** -16 + 2.0 ** -20) * (silu * u).abs()
        y[t] += p * ((silu * u) @ b.t())
        # weights: exp, sum and division of fp32 values, 2^-20 at most
        slack[t] += p * (dh @ b.t().abs() + (gamma(inner) + 2.0 ** -20) * ((silu * u).abs() @ b.t().abs()))
    return y, slack


def run_moe(pkg, torch, x, logits, w13, w2, top_k, normalise):
    (tokens, hidden), (experts, _, inner) = x.shape, w2.shape
    Y = Guarded(torch, (tokens, hidden), x.dtype)
    ids, weights = Guarded(torch, (tokens, top_k), torch.int32, fill=77), Guarded(torch, (tokens, top_k), torch.float32)
    W = Guarded(torch, (pkg.moe_workspace_bytes(tokens, hidden, inner, experts, top_k),), torch.uint8, fill=0xFF, band_bytes=1 << 16)
    out = pkg.moe(x, logits, w13, w2, top_k, normalise, Y=Y.t, ids=ids.t, weights=weights.t, workspace=W.t)
    assert out[0] is Y.t and out[1] is ids.t and out[2] is weights.t
    st, info = pkg.device_status()
    assert st == pkg.OK, (st, info)
    for what, gd in (("Y", Y), ("ids", ids), ("weights", weights), ("workspace", W)):
        gd.check(what)
    return out


def check_moe(pkg, torch, name, x, logits, w13, w2, top_k, normalise):
    y, ids, weights = run_moe(pkg, torch, x, logits, w13, w2, top_k, normalise)
    want_ids, want_weights = route_want(torch, logits, top_k, normalise)
    assert torch.equal(ids, want_ids)
    # The fp32 difference d of a logit and the largest is rounded by at most 2^-24 |d|, which its exponential takes over as a
    # relative error; and |d| <= -ln w, since w = exp(d) / total with a total of at least 1. All else: 2^-20 at most.
    rel = 2.0 ** -20 - 2.0 ** -24 * want_weights.clamp(min=1e-300).log()
    assert ((weights.double() - want_weights).abs() <= rel * want_weights).all()
    check_close(y, *moe_want(torch, x, w13, w2, want_ids, want_weights), name)
    return y, ids, weights


MOE = [  # tokens, hidden, inner, experts, top_k, normalise
    (1, 8, 8, 1, 1, True), (1, 72, 40, 3, 2, False), (1, 2048, 768, 32, 8, True), (2, 1024, 512, 8, 2, True), (3, 264, 136, 5, 5, False),
    (7, 520, 1032, 4, 1, True), (8, 1032, 64, 40, 4, True), (16, 512, 256, 16, 16, False), (17, 328, 200, 2, 1, True), (31, 640, 72, 100, 6, True),
    (33, 136, 456, 3, 2, False), (37, 1000, 360, 20, 3, True), (64, 768, 128, 8, 2, True), (65, 256, 328, 2, 2, True), (100, 392, 264, 1, 1, False),
    (129, 128, 64, 4, 3, True), (200, 520, 136, 512, 8, True), (256, 264, 72, 1, 1, True), (256, 512, 192, 6, 2, False), (255, 1288, 88, 130, 10, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("case", MOE, ids=lambda c: "x".join(map(str, c)))
def test_moe_against_64_bits(pkg, cuda, case, name):
    tokens, hidden, inner, experts, top_k, normalise = case
    x, logits, w13, w2 = moe_inputs(cuda, name, tokens, hidden, inner, experts, tokens + hidden)
    check_moe(pkg, cuda, name, x, logits, w13, w2, top_k, normalise)


@pytest.mark.gpu
@pytest.mark.parametrize("normalise", [True, False])
def test_moe_ties_and_masks(pkg, cuda, normalise):
    """Equal logits go to the lower index (zeros of either sign are equal); -infinity and NaN are never chosen, a token with
    nothing left gets zeros; the lowest finite value and +infinity are numbers like others."""
    torch = cuda
    tokens, experts, top_k = 12, 40, 4
    x, logits, w13, w2 = moe_inputs(torch, "bf16", tokens, 264, 72, experts, 5)
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    logits[0] = 1.25                                     # all equal
    logits[1, ::2], logits[1, 1::2] = -0.0, 0.0
    logits[2] = -inf                                     # nothing left
    logits[3] = nan
    logits[4] = -inf
    logits[4, 33] = -2.0                                 # one left
    logits[5] = nan
    logits[5, [39, 3]] = torch.tensor([0.5, 0.25], device="cuda")
    logits[6] = low                                      # a mask of the type's lowest value, all equal
    logits[7] = low
    logits[7, 20] = 3.0                                  # the masked ones fill up, with weight 0
    logits[8, 17] = inf
    logits[9, [30, 11]] = inf                            # two of them share
    logits[10] = (logits[10] * 2).round() / 2            # many ties
    logits[11, :20] = -inf
    y, ids, weights = check_moe(pkg, torch, "bf16", x, logits, w13, w2, top_k, normalise)
    assert ids[0].tolist() == ids[1].tolist() == ids[6].tolist() == [0, 1, 2, 3]
    assert ids[2].tolist() == ids[3].tolist() == [-1] * 4 and ids[4].tolist() == [33, -1, -1, -1] and ids[5].tolist() == [39, 3, -1, -1]
    assert not y[2:4].any() and not weights[2:4].any() and float(weights[4, 0]) == 1.0
    assert ids[7, 0] == 20 and float(weights[7, 0]) == 1.0 and ids[8, 0] == 17 and float(weights[8, 0]) == 1.0
    assert ids[9, :2].tolist() == [11, 30] and weights[9, :2].tolist() == [0.5, 0.5]


@pytest.mark.gpu
def test_moe_all_tokens_masked_or_all_on_one_expert(pkg, cuda):
    torch = cuda
    for tokens in (1, 20, 256):
        x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 392, 136, 12, tokens)
        y, ids, weights = run_moe(pkg, torch, x, torch.full_like(logits, -float("inf")), w13, w2, 3, True)
        assert not y.any() and (ids == -1).all() and not weights.any()
        logits[:, 7] = 50.0
        only = logits.clone()
        only[:, :7] = only[:, 8:] = -float("inf")
        check_moe(pkg, torch, "fp16", x, only, w13, w2, 3, True)
        check_moe(pkg, torch, "fp16", x, logits, w13, w2, 2, False)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 9, 70])
def test_moe_reads_nothing_of_experts_and_tokens_that_are_not_a_tokens_own(pkg, cuda, tokens):
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "bf16", tokens, 328, 72, 10, 9)
    logits[:, [0, 4, 9]] = -float("inf")
    clean = [t.clone() for t in run_moe(pkg, torch, x, logits, w13, w2, 3, True)]
    for e in (0, 4, 9):
        w13[e], w2[e] = float("nan"), float("inf")
    for got, want in zip(run_moe(pkg, torch, x, logits, w13, w2, 3, True), clean):
        assert torch.equal(got, want)
    x[0, 3] = float("nan")
    y = run_moe(pkg, torch, x, logits, w13, w2, 3, True)[0]
    assert y[0].isnan().all() and torch.equal(y[1:], clean[0][1:])


@pytest.mark.gpu
def test_moe_repeats_bit_for_bit_and_optional_outputs(pkg, cuda):
    torch = cuda
    for tokens in (1, 30, 256):
        x, logits, w13, w2 = moe_inputs(torch, "bf16", tokens, 776, 264, 24, 11)
        y = run_moe(pkg, torch, x, logits, w13, w2, 6, True)[0]
        for _ in range(5):
            assert torch.equal(run_moe(pkg, torch, x, logits, w13, w2, 6, True)[0], y)
        ws = torch.empty(pkg.moe_workspace_bytes(tokens, 776, 264, 24, 6), dtype=torch.uint8, device="cuda")
        Y = torch.empty_like(x)
        st = pkg.lib().b200_moe(pkg.BF16, x.data_ptr(), logits.data_ptr(), w13.data_ptr(), w2.data_ptr(), Y.data_ptr(), None, None, tokens, 776, 264, 24,
                                6, 1, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert st == pkg.OK and pkg.device_status()[0] == pkg.OK and torch.equal(Y, y)


# ------------------------------------------------------------------------------------------------ together

def block(pkg, torch, s, stream=None):
    """A block as a decode step runs it: the router's logits from the framework's product, the experts, then a projection with
    every request's adapter."""
    logits = pkg.gemm(s["x"], s["router"], stream=stream)
    y, ids, weights = pkg.moe(s["x"], logits, s["w13"], s["w2"], 3, stream=stream)
    return logits, y, ids, weights, pkg.gemm_lora(y, s["w"], s["a"], s["b"], s["ids"], s["scale"], stream=stream)


def block_state(torch, tokens, seed):
    x, _, w13, w2 = moe_inputs(torch, "bf16", tokens, 520, 136, 16, seed)
    _, w, a, b, scale = lora_inputs(torch, "bf16", tokens, 264, 520, 16, 4, seed + 1)
    router = (torch.randn(16, 520, generator=torch.Generator(device="cuda").manual_seed(seed + 2), device="cuda") * 520 ** -0.5).bfloat16()
    return {"x": x, "router": router, "w13": w13, "w2": w2, "w": w, "a": a, "b": b, "scale": scale, "ids": lora_ids(torch, "mixed", tokens, 4, seed)}


def check_block(torch, s, out):
    logits, y, ids, weights, d = out
    want_ids, want_weights = route_want(torch, logits, 3, True)
    assert torch.equal(ids, want_ids)
    check_close(y, *moe_want(torch, s["x"], s["w13"], s["w2"], want_ids, want_weights), "bf16")
    check_close(d, *lora_want(torch, y, s["w"], s["a"], s["b"], s["ids"], s["scale"]), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 13, 96])
def test_a_block_of_router_experts_and_adapters(pkg, cuda, tokens):
    s = block_state(cuda, tokens, tokens)
    out = block(pkg, cuda, s)
    assert pkg.device_status()[0] == pkg.OK
    check_block(cuda, s, out)


@pytest.mark.gpu
def test_a_block_captured_and_replayed_with_new_inputs(pkg, cuda):
    """Two graphs of different sizes, replayed side by side on two streams and in turn."""
    torch = cuda
    states = [block_state(torch, n, 40 + n) for n in (6, 70)]
    for s in states:
        block(pkg, torch, s)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = block(pkg, torch, s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in states]
    for seed in range(3):
        for s in states:
            new = block_state(torch, s["x"].shape[0], 100 * seed + s["x"].shape[0])
            for key in new:
                s[key].copy_(new[key])
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert pkg.device_status()[0] == pkg.OK
        for s in states:
            check_block(torch, s, s["out"])


@pytest.mark.gpu
def test_calls_on_other_streams_follow_their_streams_work(pkg, cuda):
    """Operands that a side stream is still writing, the call given that stream by handle or by torch's current stream;
    two calls of each kind in flight at once."""
    torch = cuda
    states = [block_state(torch, 24, 7), block_state(torch, 24, 8)]
    want = [block(pkg, torch, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for by_handle in (True, False):
        late = [{k: torch.zeros_like(v) for k, v in s.items()} for s in states]
        torch.cuda.synchronize()
        outs = []
        for s, l, st in zip(states, late, streams):
            with torch.cuda.stream(st):
                torch.cuda._sleep(20_000_000)
                for k in s:
                    l[k].copy_(s[k])
                if not by_handle:
                    outs.append(block(pkg, torch, l))
            if by_handle:
                outs.append(block_by_handle(pkg, torch, l, st))
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            for a, b in zip(w, o):
                assert torch.equal(a, b)


def block_by_handle(pkg, torch, s, st):
    D = torch.empty(s["x"].shape[0], 16, dtype=torch.float32, device="cuda")
    D.record_stream(st)
    torch.cuda.current_stream().synchronize()
    logits = pkg.gemm(s["x"], s["router"], D=D, workspace=torch.empty(0, dtype=torch.uint8, device="cuda"), stream=st.cuda_stream)
    y, ids, weights = pkg.moe(s["x"], logits, s["w13"], s["w2"], 3, stream=st.cuda_stream)
    return logits, y, ids, weights, pkg.gemm_lora(y, s["w"], s["a"], s["b"], s["ids"], s["scale"], stream=st.cuda_stream)


@pytest.mark.gpu
def test_chains_without_pauses_keep_their_order(pkg, cuda):
    """Each call's output feeds the next call, a hundred calls deep, in one stream: overlapped launches must not read early."""
    torch = cuda
    for tokens in (1, 20):
        x, _, w13, w2 = moe_inputs(torch, "bf16", tokens, 256, 64, 8, 3)
        logits = torch.randn(tokens, 8, device="cuda")
        _, w, a, b, scale = lora_inputs(torch, "bf16", tokens, 256, 256, 8, 3, 4)
        ids = lora_ids(torch, "mixed", tokens, 3, 5)

        def step(v):
            y = pkg.moe(v, logits, w13, w2, 2)[0]
            d = pkg.gemm_lora(y, w, a, b, ids, scale).float()
            return (d * d.square().mean().rsqrt()).bfloat16()      # the gate makes a step quadratic: kept at one size

        slow, fast = x, x
        for _ in range(50):
            slow = step(slow)
            torch.cuda.synchronize()
        for _ in range(50):
            fast = step(fast)
        assert torch.equal(slow, fast) and bool(slow.isfinite().all())


# ------------------------------------------------------------------------------------------------ far corners

@pytest.mark.gpu
@pytest.mark.parametrize("m", [20, 100, 400])
def test_lora_first_product_beyond_the_range_of_fp16(pkg, cuda, m):
    """u is held in fp32: values that fp16 has no number for (here up to some 10^6) meet small weights and give ordinary results."""
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, "fp16", m, 264, 512, 16, 2, m)
    x, a, b = x * 30.0, a * 8000.0, b * 1e-4
    ids = (torch.arange(m, device="cuda") >= m // 2).to(torch.int32)
    u = torch.stack([x[i].double() @ a[ids[i]].double().t() for i in range(0, m, 7)])
    assert float(u.abs().max()) > 2 * 65504
    got = run_lora(pkg, torch, x, w, a, b, ids, scale)
    check_close(got, *lora_want(torch, x, w, a, b, ids, scale), "fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 150])
def test_moe_gated_values_beyond_the_range_of_fp16(pkg, cuda, tokens):
    """A gated value travels as a pair of 16-bit numbers: up to twice the largest fp16 in that type."""
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 264, 72, 6, tokens)
    w13, w2 = w13 * 50.0, w2 * 1e-3
    x[:, 0] = 8.0
    w13[:, 5, :] = 0
    w13[:, 5, 0] = 40.0                      # gate of inner row 5: 320
    w13[:, 72 + 5, :] = 0
    w13[:, 72 + 5, 0] = 50.0                 # its other half: 400, so the gated value is 128000
    check_moe(pkg, torch, "fp16", x, logits, w13, w2, 2, True)


@pytest.mark.gpu
def test_lora_more_rows_than_one_pass_and_offsets_past_32_bits(pkg, cuda):
    """70000 rows are two passes of the library; D has more than 2^31 elements."""
    torch = cuda
    m, n, k, r, s = 70000, 32768, 64, 8, 5
    x, w, a, b, scale = lora_inputs(torch, "bf16", m, n, k, r, s, 3)
    ids = ((torch.arange(m, device="cuda") // 97) % (s + 1) - 1).to(torch.int32)
    D = torch.empty(m, n, dtype=x.dtype, device="cuda")
    D[-1, -8:] = float("nan")
    assert D.numel() > 2 ** 31
    pkg.gemm_lora(x, w, a, b, ids, scale, D=D)
    assert pkg.device_status()[0] == pkg.OK
    rows = torch.cat([torch.arange(0, m, 1999, device="cuda"), torch.arange(65500, 65600, device="cuda"), torch.arange(m - 40, m, device="cuda")])
    check_close(D[rows], *lora_want(torch, x[rows], w, a, b, ids[rows], scale), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [65536 + 7, 65536 + 300])
def test_lora_a_short_last_pass(pkg, cuda, m):
    x, w, a, b, scale = lora_inputs(cuda, "fp16", m, 72, 136, 8, 4, m)
    ids = ((cuda.arange(m, device="cuda") // 501) % 5 - 1).to(cuda.int32)
    got = run_lora(pkg, cuda, x, w, a, b, ids, scale)
    check_close(got, *lora_want(cuda, x, w, a, b, ids, scale), "fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [150, 256])
def test_lora_few_adapters_with_many_rows_each(pkg, cuda, m):
    """Up to 256 rows whose first product goes by lists of adapters: a large rank, few adapters, a long K."""
    for order in ("mixed", "stretches", "none", "all"):
        x, w, a, b, scale = lora_inputs(cuda, "bf16", m, 392, 8200, 128, 2, m)
        ids = lora_ids(cuda, order, m, 2, m)
        got = run_lora(pkg, cuda, x, w, a, b, ids, scale)
        check_close(got, *lora_want(cuda, x, w, a, b, ids, scale), "bf16")
        assert cuda.equal(run_lora(pkg, cuda, x, w, a, b, ids, scale), got)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("m, n, k, r, s, order", [(17, 8, 72, 8, 3, "mixed"), (33, 264, 8200, 16, 33, "each"), (90, 520, 1032, 72, 4, "mixed"), (225, 672, 1544, 40, 14, "stretches"),
                                                  (300, 136, 200, 24, 7, "mixed"), (535, 312, 360, 72, 43, "stretches"), (700, 1160, 264, 128, 5, "mixed"), (1025, 8, 2056, 8, 2, "all"),
                                                  (2232, 320, 936, 56, 5, "stretches"), (1100, 264, 1032, 32, 200, "stretches"), (4600, 136, 136, 16, 9, "none")])
def test_lora_blocks_of_rows(pkg, cuda, name, m, n, k, r, s, order):
    """Few columns of D: several blocks of rows, each with its own stretch of K blocks; a row's infinite input stays its own."""
    x, w, a, b, scale = lora_inputs(cuda, name, m, n, k, r, s, m)
    ids = lora_ids(cuda, order, m, s, m)
    got = run_lora(pkg, cuda, x, w, a, b, ids, scale)
    check_close(got, *lora_want(cuda, x, w, a, b, ids, scale), name)
    x[m // 2, 3] = float("nan")
    again = run_lora(pkg, cuda, x, w, a, b, ids, scale)
    assert again[m // 2].isnan().all()
    rest = cuda.arange(m, device="cuda") != m // 2
    assert cuda.equal(again[rest], got[rest])


@pytest.mark.gpu
def test_lora_workspace_of_each_number_of_adapters(pkg, cuda):
    """Few adapters need more workspace than many at the same sizes; the calls that allocate it themselves notice."""
    m, n, k, r = 256, 64, 1032, 128
    assert pkg.gemm_lora_workspace_bytes(m, n, k, 2, r) > pkg.gemm_lora_workspace_bytes(m, n, k, 256, r)
    for s in (256, 2, 256, 2):
        x, w, a, b, scale = lora_inputs(cuda, "bf16", m, n, k, r, s, s)
        ids = lora_ids(cuda, "mixed", m, s, s)
        check_close(pkg.gemm_lora(x, w, a, b, ids, scale), *lora_want(cuda, x, w, a, b, ids, scale), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40])
def test_moe_weights_past_32_bits(pkg, cuda, tokens):
    """W13 has more than 2^32 elements, W2 more than 2^31; the chosen experts lie at both ends."""
    torch = cuda
    experts, inner, hidden = 512, 1040, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    w13 = torch.empty(experts, 2 * inner, hidden, dtype=torch.bfloat16, device="cuda").normal_(0, hidden ** -0.5, generator=g)
    w2 = torch.empty(experts, hidden, inner, dtype=torch.bfloat16, device="cuda").normal_(0, inner ** -0.5, generator=g)
    assert w13.numel() > 2 ** 32 and w2.numel() > 2 ** 31
    x = torch.randn(tokens, hidden, generator=g, device="cuda").bfloat16()
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    logits[:, [0, 300, 511]] += 20.0
    y, ids, weights = run_moe(pkg, torch, x, logits, w13, w2, 3, True)
    assert sorted(set(ids.flatten().tolist())) == [0, 300, 511]
    want_ids, want_weights = route_want(torch, logits, 3, True)
    assert torch.equal(ids, want_ids)
    used = [0, 300, 511]
    place = torch.full((experts,), -1, dtype=torch.int32, device="cuda")
    place[used] = torch.arange(3, dtype=torch.int32, device="cuda")
    check_close(y, *moe_want(torch, x, w13[used], w2[used], place[want_ids.long()], want_weights), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["lora 8", "lora 100", "lora 600", "moe 2", "moe 200"])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(pkg, cuda, op):
    """With a budget of a nanosecond some bounded wait of the call expires: the launch ends by itself, the status record says so, and the
    same call with the usual budget is correct. The sizes make a wait longer than the hardware suspends a warp for on its own."""
    torch = cuda
    name, rows = op.split()
    if name == "lora":
        x, w, a, b, scale = lora_inputs(torch, "bf16", int(rows), 8192, 131072, 16, 3, 5)
        ids = lora_ids(torch, "stretches", int(rows), 3, 6)
        call = lambda: pkg.gemm_lora(x, w, a, b, ids, scale)
    else:
        x, logits, w13, w2 = moe_inputs(torch, "bf16", int(rows), 16384, 16384, 2, 5)
        call = lambda: pkg.moe(x, logits, w13, w2, 1)[0]
    want = call()
    assert pkg.device_status()[0] == pkg.OK
    pkg.set_wait_budget_ns(1)
    try:
        call()
        status, info = pkg.device_status()
    finally:
        pkg.set_wait_budget_ns(2_000_000_000)
    assert status == pkg.DEVICE_TIMEOUT and 1000 <= info[2] < 3400, (status, info)
    assert torch.equal(call(), want) and pkg.device_status()[0] == pkg.OK


# ------------------------------------------------------------------------------------------------ refusals

def test_lora_refusals(pkg):
    L = pkg.lib()
    p = lambda i: 0x10000000 * i     # never read: each call is refused before that
    good = dict(dtype=pkg.BF16, A=p(1), Bt=p(2), D=p(3), M=16, N=64, K=64, a=p(4), b=p(5), scale=p(6), ids=p(7), S=4, rank=8, ws=p(8), bytes=1 << 20, stream=None)

    def call(**change):
        return L.b200_gemm_lora(*{**good, **change}.values())

    for change in (dict(dtype=2), dict(dtype=-1), dict(rank=0), dict(rank=12), dict(rank=136), dict(rank=-8)):
        assert call(**change) == pkg.INVALID_CONFIG, change
    for change in (dict(M=0), dict(M=-1), dict(N=0), dict(K=0), dict(N=60), dict(K=68), dict(S=0), dict(S=-1), dict(M=1 << 31), dict(N=1 << 31), dict(K=1 << 31), dict(S=1 << 31)):
        assert call(**change) == pkg.INVALID_SHAPE, change
    for name in ("A", "Bt", "D", "a", "b", "ids"):
        assert call(**{name: None}) == pkg.INVALID_POINTER, name
    for name in ("A", "Bt", "D", "a", "b", "ws"):
        assert call(**{name: good[name] + 8}) == pkg.INVALID_POINTER, name
    assert call(ids=p(7) + 2) == call(scale=p(6) + 1) == pkg.INVALID_POINTER
    for name in ("A", "Bt", "a", "b", "ids", "ws"):       # D written over an operand or the workspace
        assert call(D=good[name]) == pkg.INVALID_POINTER, name
    need = pkg.gemm_lora_workspace_bytes(16, 64, 64, 4, 8)
    assert need > 0
    assert call(ws=None) == call(bytes=need - 1) == call(bytes=0) == pkg.WORKSPACE_TOO_SMALL
    for bad in ((0, 64, 64, 4, 8), (16, 60, 64, 4, 8), (16, 64, 64, 0, 8), (16, 64, 64, 4, 9)):
        assert pkg.gemm_lora_workspace_bytes(*bad) == -1


def test_moe_refusals(pkg):
    L = pkg.lib()
    p = lambda i: 0x10000000 * i
    good = dict(dtype=pkg.F16, X=p(1), logits=p(2), W13=p(3), W2=p(4), Y=p(5), ids=p(6), weights=p(7), T=8, H=64, I=32, E=4, k=2, norm=1, ws=p(8), bytes=1 << 24,
                stream=None)

    def call(**change):
        return L.b200_moe(*{**good, **change}.values())

    for change in (dict(dtype=3), dict(k=0), dict(k=5), dict(k=17, E=100), dict(norm=2), dict(norm=-1)):
        assert call(**change) == pkg.INVALID_CONFIG, change
    for change in (dict(T=0), dict(T=257), dict(T=-1), dict(H=0), dict(H=60), dict(I=0), dict(I=20), dict(E=0), dict(E=513), dict(H=1 << 30), dict(I=1 << 30)):
        assert call(**change) == pkg.INVALID_SHAPE, change
    for name in ("X", "logits", "W13", "W2", "Y"):
        assert call(**{name: None}) == pkg.INVALID_POINTER, name
    for name in ("X", "W13", "W2", "Y", "ws"):
        assert call(**{name: good[name] + 8}) == pkg.INVALID_POINTER, name
    for name in ("logits", "ids", "weights"):
        assert call(**{name: good[name] + 2}) == pkg.INVALID_POINTER, name
    for out in ("Y", "ids", "weights"):
        for name in ("X", "logits", "W13", "W2", "ws"):
            assert call(**{out: good[name]}) == pkg.INVALID_POINTER, (out, name)
    assert call(ids=p(5)) == call(weights=p(6)) == pkg.INVALID_POINTER
    need = pkg.moe_workspace_bytes(8, 64, 32, 4, 2)
    assert need > 0
    assert call(ws=None) == call(bytes=need - 1) == pkg.WORKSPACE_TOO_SMALL
    for bad in ((0, 64, 32, 4, 2), (8, 60, 32, 4, 2), (8, 64, 32, 4, 5), (257, 64, 32, 4, 2)):
        assert pkg.moe_workspace_bytes(*bad) == -1


def test_tensors_that_do_not_fit_are_refused(pkg):
    torch = pytest.importorskip("torch")
    x, ids = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.gemm_lora(x, torch.zeros(64, 64, dtype=torch.bfloat16), torch.zeros(1, 8, 64), torch.zeros(1, 64, 8), ids)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.moe(x, torch.zeros(4, 2), torch.zeros(2, 64, 64), torch.zeros(2, 64, 32), 1)


@pytest.mark.gpu
def test_tensors_that_do_not_fit_are_refused_on_the_gpu(pkg, cuda):
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, "bf16", 4, 64, 128, 8, 2, 1)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (dict(w=w.half()), dict(w=w[:, :64]), dict(a=a.transpose(1, 2)), dict(b=b[:1]), dict(ids=ids.long()), dict(ids=ids[:3]), dict(scale=scale.double()),
                dict(x=x[:, ::2]), dict(x=x.float()), dict(ids=ids.cpu()), dict(D=torch.empty(4, 64, device="cuda")), dict(D=torch.empty(64, 4, device="cuda", dtype=x.dtype).t())):
        v = {**dict(x=x, w=w, a=a, b=b, ids=ids, scale=scale, D=None), **bad}
        with pytest.raises(ValueError):
            pkg.gemm_lora(v["x"], v["w"], v["a"], v["b"], v["ids"], v["scale"], D=v["D"])
    with pytest.raises(pkg.B200Error, match="status 2"):
        pkg.gemm_lora(x[:0], w, a, b, ids[:0], scale)
    x, logits, w13, w2 = moe_inputs(torch, "fp16", 4, 64, 32, 4, 1)
    for bad in (dict(logits=logits.half()), dict(logits=logits[:, :3]), dict(w13=w13[:, :32]), dict(w2=w2.transpose(1, 2)), dict(x=x.bfloat16()), dict(Y=x.float())):
        v = {**dict(x=x, logits=logits, w13=w13, w2=w2, Y=None), **bad}
        with pytest.raises(ValueError):
            pkg.moe(v["x"], v["logits"], v["w13"], v["w2"], 2, Y=v["Y"])
    for bad, status in (((x, logits, w13, w2, 5), 1), ((x[:0], logits[:0], w13, w2, 2), 2)):
        with pytest.raises(pkg.B200Error, match=f"status {status}"):
            pkg.moe(*bad)
