"""Language-model operators at the edges of what their documents allow, without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import lm_oracle as oracle
from aiforearth_api_platform_amd.ops import _ext, mx
from aiforearth_api_platform_amd.ops.head import label_logprobs
from aiforearth_api_platform_amd.ops.mx import MxTensor, mx_dequantize, mx_linear, mx_quantize
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
    """y lies next to a border, 1.1875 of 1.125 and 1.25 or 1.0625 of 1 and 1.125, by less than 32 bits hold."""
    x = torch.full((2, 40), 2.0 ** -24)  # the squares are 2^-28 of eps
    x[1] *= -1
    for gamma, eps, value in ((1.1875, 2.0 ** -20, 1.125), (1.0625, 2.0 ** -20 * (1 - 2.0 ** -24), 1.125), (1.0625, 2.0 ** -20, 1.0)):
        g = torch.full((40,), gamma)
        want = oracle.mx_values(oracle.rms_norm(x, g, None, eps), "e4m3")
        assert want[0].eq(value * 2.0 ** -14).all()
        assert torch.equal(mx_dequantize(rms_norm_mx8(x, g, None, eps)[0]).double(), want)


def test_rms_norm_eps_is_a_32_bit_number():
    """As it is in the kernel: what 32 bits do not hold of it moves no element."""
    x, gamma = torch.full((2, 40), 2.0 ** -40), torch.full((40,), 1.1875)  # at the border, which falls to 1.25
    for eps in (2.0 ** -20, 2.0 ** -20 * (1 + 2.0 ** -25), 2.0 ** -20 * (1 - 2.0 ** -26)):
        assert mx_dequantize(rms_norm_mx8(x, gamma, None, eps)[0]).eq(1.25 * 2.0 ** -30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rms_norm_reference_takes_the_kernels_sums(dtype):
    """Sums of 16-bit rows are 32-bit numbers: 4.25 + 2^-23 is 4.25, the border of 4 and 4.5, and falls to 4."""
    x, r = torch.full((2, 64), 4.25, dtype=dtype), torch.full((2, 64), 2.0 ** -23, dtype=dtype)
    q, h = rms_norm_mx8(x, torch.ones(64), r, 2.0 ** 40)
    assert mx_dequantize(q).eq(4 * 2.0 ** -20).all() and h.eq(4.25).all()


def shapes_only(rows, k):
    """An e2m1 MxTensor without memory behind it."""
    kp = mx.padded(k)
    return MxTensor(torch.empty(rows, kp // 2, dtype=torch.uint8, device="meta"),
                    torch.empty(rows, kp // 32, dtype=torch.uint8, device="meta"), k)


@pytest.mark.parametrize("m,n,k", [(1, 1, (1 << 23) + 1),           # deeper than 2^23
                                   ((1 << 29) + 1, 1, 512),         # over 2^22 tiles of 128 x 128
                                   (1 << 20, 1 << 17, 128),
                                   ((1 << 31) + 7, 1, 128), ((1 << 32) + 7, 1, 128),
                                   (1 << 28, 3, 100),               # 2^23 or more slices of 32 x 64
                                   (32, 1 << 29, 384)])
def test_linear_refuses_more_than_a_launch_holds(m, n, k):
    with pytest.raises(ValueError):
        mx_linear(shapes_only(m, k), shapes_only(n, k))
    if m < 1 << 31 and n < 1 << 31:
        assert kernels().ai4e_mx_linear(16, 16, 1, 16, 16, None, m, n, mx.padded(k), 16, 0, None) == 1


@pytest.mark.parametrize("m,n,k", [(1, 3, 1 << 23), (1 << 29, 4, 128), ((1 << 28) - 32, 3, 100), (32, (1 << 29) - 64, 384)])
def test_linear_takes_what_a_launch_holds(m, n, k):
    assert mx._linear_fits(m, n, mx.padded(k))


def test_quantize_refuses_more_than_a_launch_holds():
    rows = ((1 << 33) - 512) // 16  # of 16 groups of 8 values
    lib = kernels()
    x = torch.empty(rows + 1, 100, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError):
        mx_quantize(x)
    with pytest.raises(ValueError):
        mx_dequantize(shapes_only(rows + 1, 100))
    assert mx_quantize(x[1:]).shape == mx_dequantize(shapes_only(rows, 100)).shape == (rows, 100)
    assert lib.ai4e_mx_quantize(16, 100, rows + 1, 100, 0, 1, 16, 16, None) == 1
    assert lib.ai4e_mx_dequantize(16, 16, rows + 1, 100, 0, 1, 16, None) == 1


def test_label_logprobs_refuses_more_labels_than_an_int_counts():
    for n in ((1 << 30) + 1, (1 << 32) + 3):
        with pytest.raises(ValueError):
            label_logprobs(torch.empty(8, device="meta"), torch.empty(n, dtype=torch.int32, device="meta"), 1)
    assert kernels().ai4e_label_logprobs(16, 8, 1, 8, 0, 16, 0, (1 << 30) + 1, 1, 16, 16, 16, 16, None) == 1


def test_forward_mode_derivatives_are_refused():
    """No operator has a derivative, in either direction: a tangent would be lost without a word."""
    x, ones = torch.randn(2, 64), torch.ones(64)
    q, w = mx_quantize(x), mx_quantize(torch.randn(64, 64))
    with forward_ad.dual_level():
        dual, dual1 = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(ones, ones.clone())
        for call in (lambda: mx_quantize(dual), lambda: rms_norm_mx8(dual, ones), lambda: rms_norm_mx8(x, dual1),
                     lambda: rms_norm_mx8(x, ones, dual), lambda: mx_linear(q, w, dual1), lambda: label_logprobs(dual)):
            for grad in (torch.enable_grad, torch.no_grad):  # no_grad stops the other direction only
                with grad(), pytest.raises(ValueError):
                    call()
        # a tensor without a tangent, and one that was detached from it
        rms_norm_mx8(x, ones, dual.detach())
        label_logprobs(x, None, 1)


def test_codes_that_require_a_gradient_are_refused():
    q, w = mx_quantize(torch.randn(2, 64), "e4m3"), mx_quantize(torch.randn(5, 64))
    leaf = [MxTensor(q.data.clone().requires_grad_(), q.scale, 64), MxTensor(q.data, q.scale.clone().requires_grad_(), 64)]
    scaled = MxTensor(w.data, w.scale.clone().requires_grad_(), 64)
    for call in (*[lambda t=t: mx_dequantize(t) for t in leaf], *[lambda t=t: mx_linear(t, w) for t in leaf],
                 lambda: mx_linear(q, scaled)):
        with pytest.raises(ValueError):
            call()
        with torch.no_grad():
            call()


def test_c_entry_refuses_32_bit_results_of_8_bit_operands():
    """As the public function does: such products are added to about 17 bits."""
    assert kernels().ai4e_mx_linear(16, 16, 0, 16, 16, None, 1, 4, 128, 16, 2, None) == 1
