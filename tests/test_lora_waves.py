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
