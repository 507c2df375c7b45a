"""b200_moe where its gated values are very small, very large or of very different sizes. They pass through the tensor core as
pairs of 16-bit numbers, and fp16 has neither numbers beyond 65504 nor steps below 2^-24.

The layers of `one_number_each` make every element of Y a single gated value times a power of two, with a gate and an up
product that are exact in fp32, so that what the layer does to the gated value can be bounded tightly:

    exponential e = exp(-gate): 2 + 1.173 |gate| units of 2^-23 (the documented bound of the quick one), of which
    the part e / (1 + e) = sigmoid(-gate) reaches 1 + e                                   (2 + 1.173 |gate|) sigmoid(-gate) 2^-23
    quotient: 2 units of 2^-23 (documented)                                               2^-22
    1 + e, product with the up value: two roundings                                       2 * 2^-24
    value + remainder: a rounding of a rounding, (eps / 2)^2                              2^-22 (fp16), 2^-16 (bf16)
    their sum in the tensor core: two units of 2^-23                                      2^-22
    all but the exponential, relative to the gated value                                  3.5 * 2^-22, or 2.5 * 2^-22 + 2^-16

and, where the pair is scaled to its slot's largest value (to 2^14 at least), half of fp16's smallest step 2^-24: 2^-39 of that
largest value. The result is then rounded once."""
import pytest

from test_routed import check_close, check_moe, dt, moe_inputs, moe_want, route_want, run_moe

SIZES = [(1, 264, 72, 6, 2), (24, 264, 136, 5, 3), (64, 328, 1032, 4, 2), (150, 264, 72, 6, 2), (256, 136, 4168, 3, 1)]   # tokens, hidden, inner, experts, top_k


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("x_size, w2_size", [(3e-3, 30.0), (1e-3, 100.0), (1.0, 1.0)])
@pytest.mark.parametrize("size", SIZES, ids=lambda c: "x".join(map(str, c)))
def test_moe_small_activations(pkg, cuda, size, x_size, w2_size, name):
    """The gate makes the gated values quadratic in the activations; large weights behind them give ordinary results."""
    tokens, hidden, inner, experts, top_k = size
    x, logits, w13, w2 = moe_inputs(cuda, name, tokens, hidden, inner, experts, tokens)
    check_moe(pkg, cuda, name, x * x_size, logits, w13, w2 * w2_size, top_k, True)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 150])
def test_moe_gated_values_far_beyond_the_range_of_fp16(pkg, cuda, tokens):
    """A gated value of 3.6e7 in one place, ordinary results."""
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 264, 72, 6, tokens)
    x[:, 0] = 64.0
    w13[:, 5, :] = 0
    w13[:, 5, 0] = 93.75                     # gate of inner row 5: 6000
    w13[:, 72 + 5, :] = 0
    w13[:, 72 + 5, 0] = 93.75                # its other half as much
    y, _, _ = check_moe(pkg, torch, "fp16", x, logits, w13, w2 * 1e-3, 2, True)
    assert bool(y.isfinite().all())


# what the gates are (x's first coordinate times a weight of about this size), the up value, the weight behind them
REGIMES = {"ordinary": (1.0, 1.0, 2.0 ** 6, 1.0), "small": (2.0 ** -8, 2.0 ** -3, 2.0 ** -8, 2.0 ** 13), "smallest": (2.0 ** -6, 2.0 ** -4, 2.0 ** -12, 2.0 ** 15),
           "large": (2.0 ** 7, 2.0 ** 7, 2.0 ** 16, 2.0 ** -20), "closed": (1.0, -36.0, 2.0 ** 36, 2.0 ** 15)}


def one_number_each(torch, name, tokens, regime, seed):
    """x, logits, w13, w2, and in 64 bits: Y, the size of a token's largest gated value times the weight, the gates."""
    experts, width = 3, 72
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = dt(torch, name)
    gate_x, gate_w, up, back = REGIMES[regime]
    x, w13, w2 = torch.zeros(tokens, width, device="cuda", dtype=t), torch.zeros(experts, 2 * width, width, device="cuda", dtype=t), torch.zeros(experts, width, width, device="cuda", dtype=t)
    spread = 1.0 if regime == "closed" else 2.0 ** -(torch.arange(width, device="cuda") % 11)    # sizes of the gates within a token
    x[:, 0] = gate_x * (1.0 + 0.04 * torch.rand(tokens, generator=g, device="cuda"))
    w13[:, :width, 0] = gate_w * (1.0 + 0.04 * torch.rand(experts, width, generator=g, device="cuda")) * spread
    root = 2.0 ** -3 * up ** 0.5                                 # 64 products of two of them: the up value
    assert float(torch.tensor(root).log2()) % 1 == 0
    x[:, 1:65] = root
    w13[:, width:, 1:65] = root
    w2[:, range(width), range(width)] = back
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    e = logits.argmax(dim=1)
    gate = x[:, :1].double() * w13[e, :width, 0].double()
    h = gate * torch.sigmoid(gate) * up
    return x, logits, w13, w2, h * back, h.abs().amax(dim=1, keepdim=True) * back, gate


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("regime", REGIMES)
@pytest.mark.parametrize("tokens", [1, 40, 64, 256])
def test_moe_one_number_each(pkg, cuda, tokens, regime, name):
    x, logits, w13, w2, want, largest, gate = one_number_each(cuda, name, tokens, regime, tokens)
    got = run_moe(pkg, cuda, x, logits, w13, w2, 1, True)[0]
    rel = (3.5 * 2.0 ** -22 if name == "fp16" else 2.5 * 2.0 ** -22 + 2.0 ** -16) + (2 + 1.173 * gate.abs()) * cuda.sigmoid(-gate) * 2.0 ** -23
    check_close(got, want, rel * want.abs() + 2.0 ** -39 * largest, name)


# ------------------------------------------------------------------------------------------------ the kernels that fp16 takes

@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 130])
@pytest.mark.parametrize("inner", [8200, 20008])
def test_moe_many_inner_rows(pkg, cuda, tokens, inner):
    """More gated values of a slot than its cluster of blocks keeps in registers (16384), small ones among them."""
    x, logits, w13, w2 = moe_inputs(cuda, "fp16", tokens, 72, inner, 3, inner)
    check_moe(pkg, cuda, "fp16", x * 3e-3, logits, w13, w2 * 10.0, 2, True)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 9, 70])
def test_moe_fp16_reads_nothing_of_experts_and_tokens_that_are_not_a_tokens_own(pkg, cuda, tokens):
    """Nor does a slot's scale follow another's values, or values that are not finite."""
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 328, 72, 10, 9)
    logits[:, [0, 4, 9]] = -float("inf")
    clean = [t.clone() for t in run_moe(pkg, torch, x, logits, w13, w2, 3, True)]
    for e in (0, 4, 9):
        w13[e], w2[e] = float("nan"), float("inf")
    for got, want in zip(run_moe(pkg, torch, x, logits, w13, w2, 3, True), clean):
        assert torch.equal(got, want)
    x[0] *= 1000.0
    others = run_moe(pkg, torch, x, logits, w13, w2, 3, True)[0]
    assert torch.equal(others[1:], clean[0][1:])
    x[0, 3] = float("nan")
    y = run_moe(pkg, torch, x, logits, w13, w2, 3, True)[0]
    assert y[0].isnan().all() and torch.equal(y[1:], clean[0][1:])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 30, 200])
def test_moe_an_infinite_gated_value_beside_finite_ones(pkg, cuda, tokens):
    """An infinity of UP gives infinities of its weights' signs, whatever the finite values beside it are."""
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 72, 72, 2, 5)
    x[:, 0] = 60000.0
    w13[:, :, 0] = 0
    w13[:, 5, 0], w13[:, 72 + 5, 0] = 60000.0, float("inf")       # gate 3.6e9, up infinite
    w13[:, 6, 0], w13[:, 72 + 6, 0] = 60000.0, 60000.0            # a finite gated value of 1.3e19
    w2[w2 == 0] = 1.0
    y = run_moe(pkg, torch, x, logits, w13, w2, 1, True)[0]
    e = logits.argmax(dim=1)
    assert y.isinf().all() and torch.equal(y > 0, w2[e, :, 5] > 0)


@pytest.mark.gpu
def test_moe_fp16_chains_without_pauses_keep_their_order(pkg, cuda):
    torch = cuda
    for tokens in (1, 20, 100):
        x, _, w13, w2 = moe_inputs(torch, "fp16", tokens, 256, 64, 8, 3)
        logits = torch.randn(tokens, 8, device="cuda")
        workspace = torch.empty(pkg.moe_workspace_bytes(tokens, 256, 64, 8, 2), dtype=torch.uint8, device="cuda")

        def run(pause):
            v = x
            for _ in range(40):
                d = pkg.moe(v, logits, w13, w2, 2, workspace=workspace)[0]
                d = pkg.moe(d, logits, w13, w2 * 30.0, 2, workspace=workspace)[0].float()
                v = (d * d.square().mean(dim=1, keepdim=True).rsqrt()).half()      # the gate makes a step quadratic: each row is kept at one size
                if pause:
                    torch.cuda.synchronize()
            return v

        slow = run(True)
        assert bool(slow.isfinite().all()) and torch.equal(run(False), slow) and pkg.device_status()[0] == pkg.OK


@pytest.mark.gpu
def test_moe_fp16_graphs_replayed_side_by_side(pkg, cuda):
    """Captured calls of the two ways, on two streams, with new inputs of other sizes each time."""
    torch = cuda
    states = []
    for tokens in (6, 70):
        x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 520, 4168, 5, tokens)
        states.append(dict(x=x, logits=logits, w13=w13, w2=w2))
    graphs, streams = [], [torch.cuda.Stream() for _ in states]
    for s in states:
        pkg.moe(s["x"], s["logits"], s["w13"], s["w2"], 3)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = pkg.moe(s["x"], s["logits"], s["w13"], s["w2"], 3)
        graphs.append(g)
    for seed, size in enumerate((1.0, 1e-2, 30.0)):
        for s in states:
            x, logits, _, _ = moe_inputs(torch, "fp16", s["x"].shape[0], 520, 8, 5, seed)
            s["x"].copy_(x * size), s["logits"].copy_(logits)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert pkg.device_status()[0] == pkg.OK
        for s in states:
            y, ids, weights = s["out"]
            want_ids, want_weights = route_want(torch, s["logits"], 3, True)
            assert torch.equal(ids, want_ids)
            check_close(y, *moe_want(torch, s["x"], s["w13"], s["w2"], want_ids, want_weights), "fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 200])
def test_moe_fp16_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(pkg, cuda, tokens):
    torch = cuda
    x, logits, w13, w2 = moe_inputs(torch, "fp16", tokens, 16384, 16384, 2, 5)
    call = lambda: pkg.moe(x, logits, w13, w2, 1)[0]
    want = call()
    assert pkg.device_status()[0] == pkg.OK
    pkg.set_wait_budget_ns(1)
    try:
        call()
        status, info = pkg.device_status()
    finally:
        pkg.set_wait_budget_ns(2_000_000_000)
    assert status == pkg.DEVICE_TIMEOUT and 1000 <= info[2] < 1500, (status, info)
    assert torch.equal(call(), want) and pkg.device_status()[0] == pkg.OK
