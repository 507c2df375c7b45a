"""b200_gemm_lora in waves of whole 256 x 256 tiles, the form for more than 256 rows and more than 18 such tiles: there whole groups
of 32 rows with one adapter take their second product on the tensor core, with u as a pair of 16-bit numbers."""
import pytest

from test_routed import check_close, dt, lora_ids, lora_inputs, lora_want, run_lora

M, N, K = 600, 2056, 264        # 27 tiles


def in_waves(pkg, m, n, k, r, s):
    """In waves no sums of parts are kept, so the workspace does not grow with the columns; in the other forms it does."""
    return pkg.gemm_lora_workspace_bytes(m, n, k, s, r) == pkg.gemm_lora_workspace_bytes(m, 2 * n, k, s, r)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [8, 72, 128])
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-6])
@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_small_first_products(pkg, cuda, name, size, r):
    """Small u (by small scales) before large lora_b: below 2^-14 fp16 loses bits, below 2^-24 all of them."""
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, name, M, N, K, r, 3, r)
    assert in_waves(pkg, M, N, K, r, 3)
    w, b, scale = w * 1e-4, b * 100.0, scale * size
    ids = lora_ids(torch, "stretches", M, 3, r)
    check_close(run_lora(pkg, torch, x, w, a, b, ids, scale), *lora_want(torch, x, w, a, b, ids, scale), name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_ranks_and_rows_of_different_sizes(pkg, cuda, name):
    """Adapters stacked along the rank, one with small lora_a and large lora_b; rows of very different sizes."""
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, name, M, N, K, 32, 3, 9)
    a[:, 16:] *= 2.0 ** -9
    b[:, :, 16:] *= 2.0 ** 9
    x[1::2] *= 2.0 ** -7
    w = w * 1e-3
    ids = lora_ids(torch, "stretches", M, 3, 9)
    check_close(run_lora(pkg, torch, x, w, a, b, ids, scale), *lora_want(torch, x, w, a, b, ids, scale), name)


def test_which_sizes_are_in_waves(pkg):
    """The sizes that the tests of this file rest on; a change of the rule that takes them elsewhere has to show here."""
    for m, n, k, r, s in [(M, N, K, r, s) for r in (8, 32, 72, 128) for s in (1, 3, 5, 300)] + [(600, 2056, 2056, 72, 3), (1000, 2568, 136, 72, 300)]:
        assert in_waves(pkg, m, n, k, r, s), (m, n, k, r, s)
    for m, n, k, r, s in [(256, 2056, 264, 8, 3), (400, 264, 264, 8, 3), (513, 904, 1024, 64, 4), (1000, 256, 264, 8, 300)]:
        assert not in_waves(pkg, m, n, k, r, s), (m, n, k, r, s)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("m, n, k, r, s, order", [(M, N, K, 8, 3, "stretches"), (M, N, K, 72, 5, "stretches"), (M, N, K, 128, 1, "all"), (M, N, K, 128, 3, "mixed"), (M, N, K, 72, 300, "each"),
                                                  (M, N, K, 32, 3, "none"), (1000, 2568, 136, 72, 300, "stretches"), (257, 4872, 520, 104, 2, "all"), (4100, 520, 72, 24, 6, "stretches")])
def test_against_64_bits(pkg, cuda, m, n, k, r, s, order, name):
    """Ranks below, between and beyond the 64 of one turn of the tensor core, whole groups, mixed groups and none."""
    assert in_waves(pkg, m, n, k, r, s)
    x, w, a, b, scale = lora_inputs(cuda, name, m, n, k, r, s, m + r)
    ids = lora_ids(cuda, order, m, s, m + r)
    scale = scale if r % 16 else None
    first = run_lora(pkg, cuda, x, w, a, b, ids, scale)
    check_close(first, *lora_want(cuda, x, w, a, b, ids, scale), name)
    for _ in range(3):
        assert cuda.equal(run_lora(pkg, cuda, x, w, a, b, ids, scale), first)


@pytest.mark.gpu
def test_groups_of_every_kind_in_one_tile(pkg, cuda):
    """Whole groups of one adapter beside mixed ones, rows without an adapter, and neighbours of another adapter."""
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, "bf16", M, N, K, 72, 4, 5)
    ids = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    ids[:64] = 1                        # a run of two groups
    ids[64:96] = 2                      # a run of one, another adapter
    ids[96:128] = torch.arange(32, device="cuda") % 2
    ids[128:160] = 3
    ids[140] = -1                       # one row of a whole group without
    ids[192:256] = 0
    ids[256:500] = torch.arange(244, device="cuda") // 40 % 4
    ids[M - 30:] = 2                    # the last rows
    check_close(run_lora(pkg, torch, x, w, a, b, ids, scale), *lora_want(torch, x, w, a, b, ids, scale), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("order", ["stretches", "mixed"])
def test_reads_nothing_of_adapters_and_rows_that_are_not_a_rows_own(pkg, cuda, name, order):
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, name, M, N, K, 72, 5, 3)
    rows = torch.arange(M, device="cuda")
    ids = (rows >= M // 2).to(torch.int32) + 1 if order == "stretches" else rows.to(torch.int32) % 2 + 1       # adapters 1 and 2 only
    ids[M // 4] = -1
    clean = run_lora(pkg, torch, x, w, a, b, ids, scale)
    for j in (0, 3, 4):
        a[j], b[j], scale[j] = float("nan"), float("inf"), float("nan")      # never read below: lora_want leaves out what no row has
    assert torch.equal(run_lora(pkg, torch, x, w, a, b, ids, scale), clean)
    # an adapter's infinity stays with its rows, an input's NaN with its row, a first product's infinity too
    b[2, 7] = float("inf")
    x[0, 5] = float("nan")
    x[3, 5] = float("inf")
    got = run_lora(pkg, torch, x, w, a, b, ids, scale)
    assert got[0].isnan().all() and not got[3].isfinite().any()
    own = ids == 2
    assert not got[own, 7].isfinite().any()
    got[own, 7] = clean[own, 7]
    assert torch.equal(got[32:], clean[32:])
    # the neighbours in the first group may have come another way, with another rounding
    rest = (rows < 32) & (rows != 0) & (rows != 3) & ~own
    check_close(got[rest], *lora_want(torch, x[rest], w, a[:3], b[:3], ids[rest], scale), name)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [32, 128])
def test_first_product_beyond_the_range_of_fp16(pkg, cuda, r):
    """Values of u that fp16 has no number for keep a group off the tensor core."""
    torch = cuda
    x, w, a, b, scale = lora_inputs(torch, "fp16", M, N, K, r, 2, r)
    x, a, b = x * 30.0, a * 8000.0, b * 1e-4
    ids = (torch.arange(M, device="cuda") >= M // 2).to(torch.int32)
    u = torch.stack([x[i].double() @ a[ids[i]].double().t() for i in range(0, M, 7)])
    assert float(u.abs().max()) > 2 * 65504
    check_close(run_lora(pkg, torch, x, w, a, b, ids, scale), *lora_want(torch, x, w, a, b, ids, scale), "fp16")


@pytest.mark.gpu
def test_chain_without_pauses_keeps_its_order(pkg, cuda):
    """Each call's output is the next call's input, without a pause: none of a call's four overlapped kernels may read early."""
    torch = cuda
    m, n, r = 600, 2056, 72
    assert in_waves(pkg, m, n, n, r, 3)
    x, w, a, b, scale = lora_inputs(torch, "bf16", m, n, n, r, 3, 4)
    ids = lora_ids(torch, "stretches", m, 3, 5)
    workspace = torch.empty(pkg.gemm_lora_workspace_bytes(m, n, n, 3, r), dtype=torch.uint8, device="cuda")

    def run(pause):
        v = x
        for _ in range(20):
            v = pkg.gemm_lora(v, w, a, b, ids, scale, workspace=workspace)
            v = (v.float() * v.float().square().mean().rsqrt()).bfloat16()
            v = pkg.gemm_lora(v, w, a, b, ids, scale, workspace=workspace)      # one call directly behind the other
            v = pkg.gemm_lora(v, w, a, b, ids, scale, workspace=workspace)
            v = (v.float() * v.float().square().mean().rsqrt()).bfloat16()
            if pause:
                torch.cuda.synchronize()
        return v

    slow = run(True)
    assert bool(slow.isfinite().all()) and torch.equal(run(False), slow) and pkg.device_status()[0] == pkg.OK


@pytest.mark.gpu
def test_graphs_replayed_side_by_side(pkg, cuda):
    """Two captured calls on two streams with new inputs, each with the workspace that its capture allocated."""
    torch = cuda
    sizes = [(600, 2056, 264, 72), (700, 2312, 520, 16)]
    states = []
    for m, n, k, r in sizes:
        assert in_waves(pkg, m, n, k, r, 3)
        x, w, a, b, scale = lora_inputs(torch, "fp16", m, n, k, r, 3, m)
        states.append(dict(x=x, w=w, a=a, b=b, scale=scale, ids=lora_ids(torch, "stretches", m, 3, m)))
    call = lambda s: pkg.gemm_lora(s["x"], s["w"], s["a"], s["b"], s["ids"], s["scale"])
    graphs, streams = [], [torch.cuda.Stream() for _ in states]
    for s in states:
        call(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = call(s)
        graphs.append(g)
    for seed in range(3):
        for s, (m, n, k, r) in zip(states, sizes):
            x, _, a, b, _ = lora_inputs(torch, "fp16", m, n, k, r, 3, 10 * seed + m)
            s["x"].copy_(x), s["a"].copy_(a), s["b"].copy_(b), s["ids"].copy_(lora_ids(torch, "mixed" if seed == 1 else "stretches", m, 3, seed))
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert pkg.device_status()[0] == pkg.OK
        for s in states:
            check_close(s["out"], *lora_want(torch, s["x"], s["w"], s["a"], s["b"], s["ids"], s["scale"]), "fp16")
