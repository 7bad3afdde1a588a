"""linear_plan says what a call takes, under an SM margin too."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(1, 256, 4096), (64, 2048, 2048), (64, 28672, 1024), (128, 4096, 4096), (777, 2880, 512), (3000, 2304, 256), (2048, 7168, 2048)]


def plan_for(sms, t, n, k, mx8, float_out, gated):
    from paired_nvfp4_kernels import _cabi
    v = [ctypes.c_int() for _ in range(3)]
    _cabi.check(_cabi.lib.pnv_linear_plan(mx8, t, n, k, float_out, gated, sms, *[ctypes.byref(x) for x in v]))
    tokens, split, width = (x.value for x in v)
    return ("split", tokens, split) if tokens else ("pair", width)


@pytest.mark.parametrize("margin", [0, 8, 20, 100, 146, 147, 1000])
def test_plan_is_that_of_the_call(margin):
    """The operators hand the device's SM count less the margin to the library, one SM at least."""
    from paired_nvfp4_kernels import ops
    sms = max(1, torch.cuda.get_device_properties(0).multi_processor_count - margin)
    try:
        ops.set_sm_margin(margin)
        for size in SIZES:
            for mx8, float_out, gated in ((0, 0, 0), (1, 0, 0), (0, 1, 0), (1, 0, 1)):
                assert ops.linear_plan(*size, mx8=mx8, float_out=float_out, gated=gated) == plan_for(sms, *size, mx8, float_out, gated), size
    finally:
        ops.set_sm_margin(0)


def test_a_margin_changes_plans():
    """Otherwise the test above compares nothing."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert any(plan_for(sms, *s, 0, 0, 0) != plan_for(sms - 100, *s, 0, 0, 0) for s in SIZES)


@pytest.mark.parametrize("margin", [0, 20, 100])
def test_call_and_plan_agree_in_their_bits(margin):
    """A call through the operator under a margin has the bits of the C entry's with that many SMs."""
    from paired_nvfp4_kernels import _cabi, ops
    sms = torch.cuda.get_device_properties(0).multi_processor_count - margin
    g = torch.Generator(device="cuda").manual_seed(margin)
    for t, n, k in ((1, 256, 4096), (64, 2048, 2048), (128, 4096, 4096)):
        x, w = (torch.randn((r, k), generator=g, device="cuda").to(torch.bfloat16) for r in (t, n))
        want = torch.empty((t, n), device="cuda")
        _cabi.check(_cabi.lib.pnv_linear(want.data_ptr(), 1, x.data_ptr(), k, w.data_ptr(), None, 0, None, 0, t, n, k, 2, 0, 1.0, -1.0, sms,
                                         torch.cuda.current_stream().cuda_stream))
        try:
            ops.set_sm_margin(margin)
            assert torch.equal(torch.ops.paired_nvfp4.linear(x, w, float_out=True), want)
        finally:
            ops.set_sm_margin(0)
