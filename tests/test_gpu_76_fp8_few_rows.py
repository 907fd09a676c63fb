"""The kernel that 8-bit products take on groups of few rows, forced on groups of any size: the checks of the products and the MLP
against their definitions, at the edges of its tiles (128 weight rows, 64 tokens, boxes of 16)."""
import pytest
import torch

from . import test_gpu_73_fp8 as products

pytestmark = pytest.mark.gpu


@pytest.fixture
def few_rows():
    from qwen3_moe_fused import _lib

    prev = _lib.set_gemm_path(_lib.PATH_TC_SINGLE)
    yield "few rows"
    _lib.set_gemm_path(prev)
    torch.cuda.synchronize()
    assert _lib.read_error_flag() == 0


SIZES = [[3], [0, 1, 16, 17, 0], [64, 65, 0, 31, 130], [5, 300, 2]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("K,N", [(256, 384), (16, 256), (720, 1008), (2048, 208), (128, 16), (1536, 144)])
def test_linear(cuda, few_rows, dtype, sizes, K, N):
    products.test_linear_forward_and_gradient(cuda, few_rows, dtype, sizes, K, N)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("H,I", [(256, 128), (400, 208), (2048, 768), (208, 1008)])
def test_mlp(cuda, few_rows, dtype, sizes, H, I):
    products.test_mlp_forward_and_gradient(cuda, few_rows, dtype, sizes, H, I)


def test_rows_next_to_nan_keep_their_bits(cuda, few_rows):
    products.test_rows_next_to_nan_keep_their_bits(cuda, few_rows)


def test_rows_behind_the_last_group_are_left(cuda, few_rows):
    products.test_rows_behind_the_last_group_are_left(cuda, few_rows)


def test_many_experts_of_few_rows(cuda):
    """The size where the two kernels take turns, on the path that the library chooses."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8

    gen = products.gen_for(cuda, 31)
    E, H, I = 40, 512, 384
    ws = [t for shape in ((E, I, H), (E, I, H), (E, H, I)) for t in products.fp8_weight(*shape, gen, cuda)]
    for rows in (1, 40, 32 * E, 32 * E + 1, 64 * E, 64 * E + 1):
        sizes = torch.bincount(torch.randint(0, E, (rows,), generator=gen, device=cuda), minlength=E).int()
        x = torch.randn(rows, H, generator=gen, device=cuda).to(torch.bfloat16)
        with torch.no_grad():
            got = moe_mlp_fp8(x, *ws, sizes)
            prev = _lib.set_gemm_path(_lib.PATH_TC)
            want = moe_mlp_fp8(x, *ws, sizes)
            _lib.set_gemm_path(prev)
        # the same codes but where h crosses a border between two: see the tolerances of the MLP, twice (two results)
        assert (got.double() - want.double()).norm() <= 2 * (2.0 ** -9 + 2.0 ** -8) * want.double().norm()
    assert _lib.read_error_flag() == 0
