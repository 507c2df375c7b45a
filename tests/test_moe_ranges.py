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

from test_routed import check_close, check_moe, dt, moe_inputs, run_moe

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
