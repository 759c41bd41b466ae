"""Language-model operators at the edges of what their documents allow, without a GPU."""
import pytest
import torch

import lm_oracle as oracle
from aiforearth_api_platform_amd.ops import _ext
from aiforearth_api_platform_amd.ops.mx import mx_dequantize
from aiforearth_api_platform_amd.ops.norm import rms_norm_mx8


def kernels():
    if not _ext.available():
        pytest.skip("kernel library not built")
    return _ext.lib()


def test_c_entries_take_no_rows_at_null():
    """A tensor without elements has no memory: every pointer is null, and there is nothing to do (no GPU is touched)."""
    lib = kernels()
    assert lib.ai4e_mx_quantize(None, 40, 0, 40, 0, 0, None, None, None) == 0
    assert lib.ai4e_mx_dequantize(None, None, 0, 40, 0, 1, None, None) == 0
    assert lib.ai4e_rms_norm_mx8(None, 40, None, 0, 16, 1e-6, 0, 40, 0, None, None, None, None) == 0
    assert lib.ai4e_label_logprobs(None, 40, 0, 40, 0, None, 0, 0, 5, None, None, None, None, None) == 0
    assert lib.ai4e_mx_linear(None, None, 0, 16, 16, None, 0, 8, 128, None, 0, None) == 0
    # what else is wrong with such a call is still refused
    assert lib.ai4e_mx_quantize(None, 40, 0, 41, 0, 0, None, None, None) == 1
    assert lib.ai4e_rms_norm_mx8(None, 40, None, 0, 16, 0.0, 0, 40, 0, None, None, None, None) == 1
    assert lib.ai4e_mx_linear(None, None, 0, 16, 16, None, 0, 8, 64, None, 0, None) == 1


@pytest.mark.parametrize("eps", [0.0, -1e-6, 1e-46, float("nan")])
def test_rms_norm_refuses_an_eps_that_32_bits_do_not_hold(eps):
    with pytest.raises(ValueError):
        rms_norm_mx8(torch.ones(2, 64), torch.ones(64), eps=eps)


def test_rms_norm_reference_rounds_once():
    """y lies below the border 1.1875 of 1.125 and 1.25 by less than 32 bits hold: it becomes 1.125."""
    eps = 2.0 ** -20 * (1 + 2.0 ** -25)
    x, gamma = torch.full((2, 40), 2.0 ** -40), torch.full((40,), 1.1875)
    x[1] *= -1
    want = oracle.mx_values(oracle.rms_norm(x, gamma, None, eps), "e4m3")
    assert want[0].eq(1.125 * 2.0 ** -30).all()
    assert torch.equal(mx_dequantize(rms_norm_mx8(x, gamma, None, eps)[0]).double(), want)
    # above the border between 1 and 1.125, which falls to 1; at one it stays there
    gamma[:] = 1.0625
    for e, value in ((2.0 ** -20 * (1 - 2.0 ** -25), 1.125), (2.0 ** -20, 1.0)):
        assert mx_dequantize(rms_norm_mx8(x, gamma, None, e)[0])[0].eq(value * 2.0 ** -30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rms_norm_reference_takes_the_kernels_sums(dtype):
    """Sums of 16-bit rows are 32-bit numbers: 4.25 + 2^-23 is 4.25, the border of 4 and 4.5, and falls to 4."""
    x, r = torch.full((2, 64), 4.25, dtype=dtype), torch.full((2, 64), 2.0 ** -23, dtype=dtype)
    q, h = rms_norm_mx8(x, torch.ones(64), r, 2.0 ** 40)
    assert mx_dequantize(q).eq(4 * 2.0 ** -20).all() and h.eq(4.25).all()
