"""quant_mx8 at rows whose length needs more than 32 bits: refused, not cut."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import paired_nvfp4_kernels  # noqa: F401
    return torch.ops.paired_nvfp4


@pytest.mark.parametrize("k", [2 ** 31, 2 ** 32 + 64])
def test_rows_too_long_are_refused(ops, k):
    """(2^32 + 64 elements were taken for 64.)"""
    x = torch.empty((1, k), dtype=torch.bfloat16, device="cuda")
    try:
        with pytest.raises(RuntimeError, match="below 2\\^31"):
            ops.quant_mx8(x)
    finally:
        del x
        torch.cuda.empty_cache()


def test_a_long_row_is_quantized_to_its_end(ops):
    """Its last 2048 elements are those of a row that has only them, their scales the last 16 atoms."""
    k = 2 ** 30 + 128
    x = torch.empty((1, k), dtype=torch.bfloat16, device="cuda")
    x.view(-1)[: 2 ** 30].view(-1, 2 ** 20)[:] = torch.randn(2 ** 20, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[0, 2 ** 30:] = torch.arange(1, 129, device="cuda")
    q, sf = ops.quant_mx8(x)
    tail, tail_sf = ops.quant_mx8(x[:, -2048:].contiguous())
    assert torch.equal(q[:, -2048:].view(torch.uint8), tail.view(torch.uint8))
    assert torch.equal(sf.view(torch.uint8)[-16 * 512:], tail_sf.view(torch.uint8))
    del x, q, sf
    torch.cuda.empty_cache()
