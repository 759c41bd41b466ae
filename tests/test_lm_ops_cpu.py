"""Language-model operators on the CPU: the PyTorch paths against 64-bit oracles, and what the entry points refuse."""
import math

import pytest
import torch

import lm_oracle as oracle
from aiforearth_api_platform_amd.ops import _ext, mx
from aiforearth_api_platform_amd.ops.head import label_logprobs
from aiforearth_api_platform_amd.ops.mx import MxTensor, mx_dequantize, mx_linear, mx_quantize
from aiforearth_api_platform_amd.ops.norm import rms_norm_mx8


def special_rows(k, seed=0):
    """Rows that reach every rounding and scale border: ties, zeros, tiny, huge, not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(12, k, generator=g)
    x[1] = 0
    x[2] *= 1e-38
    x[3] *= 2.0 ** 100
    x[4] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0])[torch.randint(0, 9, (k,), generator=g)]
    x[5] = (torch.randint(0, 1 << 9, (k,), generator=g) - 256).float() * 0.875  # halves of the 8-bit grid
    x[6, 0] = math.nan
    x[7, k - 1] = -math.inf
    x[8] = 7.0  # between 6 and 8: the scale needs its extra step
    x[9] = 449.0
    x[10] = 2.0 ** -133
    x[11, ::2] = -0.0
    return x


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("k", [1, 31, 32, 33, 127, 128, 129, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_reference_matches_64_bit_oracle(fmt, k, dtype):
    x = special_rows(k).to(dtype)
    q = mx_quantize(x, fmt)
    assert q.shape == x.shape and q.scale.shape == (12, mx.padded(k) // 32)
    el, e = oracle.mx(x, fmt)
    code = q.scale.view(torch.uint8).double()[:, :e.shape[1]]
    assert torch.equal(code, torch.where(torch.isnan(e), torch.full_like(e, 255), e + 127))
    got = mx_dequantize(q).double()
    want = oracle.mx_values(x, fmt)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])
    assert not q.data.view(torch.uint8)[:, (mx.padded(k) // 2 if fmt == "e2m1" else mx.padded(k)):].numel()


def test_padding_is_zero():
    q = mx_quantize(torch.ones(2, 33), "e2m1")
    assert q.data[:, 17:].eq(0).all() and q.scale.view(torch.uint8)[:, 2:].eq(0).all()


def test_linear_reference_and_leading_axes():
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(2, 3, 70, generator=g), torch.randn(5, 70, generator=g), torch.randn(5, generator=g)
    for fmt in ("e4m3", "e2m1"):
        xq, wq = mx_quantize(x, fmt), mx_quantize(w, "e2m1")
        y = mx_linear(xq, wq, b, torch.bfloat16)
        want = oracle.mx_values(x.view(6, 70), fmt) @ oracle.mx_values(w, "e2m1").T + b.double()
        assert y.shape == (2, 3, 5) and y.dtype == torch.bfloat16
        # one rounding to bf16 and 32-bit sums of 70 products
        assert ((y.view(6, 5).double() - want).abs() <= want.abs() * 2 ** -8 + 70 * 2 ** -23 * 6 * 20).all()


@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_reference(residual):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 3, 50, generator=g).bfloat16()
    r = torch.randn(4, 3, 50, generator=g).bfloat16() if residual else None
    gamma = torch.rand(50, generator=g) + 0.5
    q, h = rms_norm_mx8(x, gamma, r, 1e-6)
    y = oracle.rms_norm(x, gamma, r, 1e-6).view(12, 50)
    assert torch.equal(mx_dequantize(q).view(12, 50).double(), oracle.mx_values(y.float(), "e4m3"))
    assert (h is None) == (r is None)
    if residual:
        assert torch.equal(h, (x.float() + r.float()).bfloat16())


def test_label_logprobs_reference():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 40, generator=g) * 3
    x[1, 5:] = -math.inf
    x[2] = -math.inf
    x[3, ::3] = x[3].max()
    x[4] = torch.finfo(torch.float32).min
    labels = torch.tensor([[0, 3], [9, 1], [0, 0], [-1, 2], [7, 7], [39, 0]])
    got = label_logprobs(x, labels, 7)
    logp, ent, idx, top = oracle.logprobs(x, labels, 7)
    assert torch.equal(got.top_idx.long(), idx)
    for a, b in ((got.logp, logp), (got.entropy, ent), (got.top_logp, top)):
        assert torch.allclose(a.double(), b, rtol=2 ** -23, atol=2 ** -23)
    bad = x.clone()
    bad[0, 3], bad[5, 1] = math.nan, math.inf
    got = label_logprobs(bad, labels, 7)
    for r in (0, 5):
        assert got.entropy[r].isnan() and got.logp[r].isnan().all() and got.top_logp[r].isnan().all()
        assert got.top_idx[r].eq(-1).all()
    assert label_logprobs(x, torch.full((6,), 40), 0).logp.isnan().all()
    assert label_logprobs(x, None, 1).logp is None


def test_refusals():
    x = torch.randn(4, 64)
    q4, q8 = mx_quantize(x, "e2m1"), mx_quantize(x, "e4m3")
    bad = [
        lambda: mx_quantize(x, "e5m2"),
        lambda: mx_quantize(x.double()),
        lambda: mx_quantize(x[:, :0]),
        lambda: mx_quantize(torch.tensor(1.0)),
        lambda: mx_quantize(x.clone().requires_grad_()),
        lambda: mx_dequantize(q4, torch.float64),
        lambda: mx_dequantize(MxTensor(q4.data, q4.scale, 129)),
        lambda: mx_dequantize(MxTensor(q4.data, q4.scale, 0)),
        lambda: mx_dequantize(MxTensor(q4.data[:, ::2], q4.scale, 64)),
        lambda: mx_dequantize(MxTensor(q4.data.int(), q4.scale, 64)),
        lambda: mx_dequantize(MxTensor(q4.data, q4.scale[:2], 64)),
        lambda: mx_linear(q8, q8),                                            # 8-bit weights
        lambda: mx_linear(q4, mx_quantize(torch.randn(4, 65))),               # another width
        lambda: mx_linear(q4, mx_quantize(torch.randn(2, 2, 64))),            # weights of three axes
        lambda: mx_linear(q8, q4, out_dtype=torch.float32),
        lambda: mx_linear(q4, q4, out_dtype=torch.float64),
        lambda: mx_linear(q4, q4, bias=torch.randn(5)),
        lambda: mx_linear(q4, q4, bias=torch.ones(4, dtype=torch.int32)),
        lambda: mx_linear(q4, q4, bias=torch.randn(4, requires_grad=True)),
        lambda: rms_norm_mx8(x.double(), torch.ones(64)),
        lambda: rms_norm_mx8(x, torch.ones(63)),
        lambda: rms_norm_mx8(x, torch.ones(64), x[:2]),
        lambda: rms_norm_mx8(x, torch.ones(64), x.bfloat16()),
        lambda: rms_norm_mx8(x, torch.ones(64), eps=0.0),
        lambda: rms_norm_mx8(x, torch.ones(64, requires_grad=True)),
        lambda: label_logprobs(x.double(), None, 1),
        lambda: label_logprobs(x, None, 65),
        lambda: label_logprobs(x, None, -1),
        lambda: label_logprobs(x, torch.zeros(4), 1),
        lambda: label_logprobs(x, torch.zeros(3, dtype=torch.int64), 1),
        lambda: label_logprobs(x[:, :0], None, 0),
        lambda: label_logprobs(x.clone().requires_grad_(), None, 1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():  # a parameter is fine where nothing records
        rms_norm_mx8(x, torch.ones(64, requires_grad=True))


def test_no_rows():
    for fmt in ("e2m1", "e4m3"):
        q = mx_quantize(torch.empty(0, 40), fmt)
        assert mx_dequantize(q).shape == (0, 40)
        assert mx_linear(q, mx_quantize(torch.randn(3, 40))).shape == (0, 3)
    q, h = rms_norm_mx8(torch.empty(2, 0, 40), torch.ones(40), torch.empty(2, 0, 40))
    assert q.shape == (2, 0, 40) and h.shape == (2, 0, 40)


def test_c_entries_refuse_bad_arguments():
    """Status 1, before anything is launched (no GPU is touched)."""
    if not _ext.available():
        pytest.skip("kernel library not built")
    lib, p = _ext.lib(), 16
    assert lib.ai4e_mx_quantize(p, 10, 1, 11, 0, 0, p, p, None) == 1      # row stride below the width
    assert lib.ai4e_mx_quantize(p, 10, 1, 10, 3, 0, p, p, None) == 1      # type
    assert lib.ai4e_mx_quantize(p, 10, 1, 10, 0, 2, p, p, None) == 1      # format
    assert lib.ai4e_mx_quantize(None, 10, 1, 10, 0, 0, p, p, None) == 1
    assert lib.ai4e_mx_quantize(p, 10, 1 << 40, 10, 0, 0, p, p, None) == 1  # more threads than a launch holds
    assert lib.ai4e_mx_dequantize(p, p, 1, 0, 0, 0, p, None) == 1
    assert lib.ai4e_mx_linear(p, p, 0, p, p, None, 1, 1, 64, p, 0, None) == 1  # width not stored up to 128
    assert lib.ai4e_mx_linear(p, p, 2, p, p, None, 1, 1, 128, p, 0, None) == 1
    assert lib.ai4e_mx_linear(p, p, 0, p, None, None, 1, 1, 128, p, 0, None) == 1
    assert lib.ai4e_rms_norm_mx8(p, 4, None, 0, p, 0.0, 1, 4, 0, None, p, p, None) == 1
    assert lib.ai4e_rms_norm_mx8(p, 4, p, 3, p, 1e-6, 1, 4, 0, p, p, p, None) == 1
    assert lib.ai4e_label_logprobs(p, 8, 1, 8, 0, p, 1, 1, 9, p, p, p, p, None) == 1   # k over the classes
    assert lib.ai4e_label_logprobs(p, 8, 1, 8, 0, None, 1, 1, 0, p, p, None, None, None) == 1


def test_refusals_of_other_tensors_and_of_rows_past_the_limit():
    x = mx_quantize(torch.ones(2, 64))
    for call in (lambda: mx_dequantize(torch.ones(3)), lambda: mx_linear(torch.ones(3, 64), x), lambda: mx_linear(x, x.data)):
        with pytest.raises(TypeError):
            call()
    wide = torch.zeros(1).expand((1 << 30) + 1)  # no memory behind it
    codes = MxTensor(torch.zeros(1, dtype=torch.uint8).expand(1 << 29), torch.zeros(1, dtype=torch.uint8).expand(1 << 25), 1 << 32)
    for call in (lambda: mx_quantize(wide), lambda: label_logprobs(wide), lambda: rms_norm_mx8(wide, wide),
                 lambda: mx_dequantize(codes)):
        with pytest.raises(ValueError):
            call()
