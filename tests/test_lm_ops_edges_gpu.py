"""Language-model operators on the GPU at the edges of what their documents allow, against 64-bit oracles."""
import math

import pytest
import torch

import lm_oracle as oracle
from aiforearth_api_platform_amd.ops import mx
from aiforearth_api_platform_amd.ops.head import label_logprobs
from aiforearth_api_platform_amd.ops.mx import mx_dequantize, mx_linear, mx_quantize
from aiforearth_api_platform_amd.ops.norm import rms_norm_mx8
from test_lm_ops_gpu import DEV, check_logprobs, gen

pytestmark = pytest.mark.gpu

# finite fills that stand for a mask, and logits of any size
FILLS = [-1e5, -1e9, -3e9, -1e10, -1e12, -1e20, -1e30, -1e38, -2.36e38, -3e38]
# a wave per row, a workgroup of 4 waves (few and many classes), one of 16 waves
FORMS = [(24, 1500, 10), (24, 1500, 20), (24, 2600, 10), (300, 9001, 10), (24, 40001, 10)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c,k", FORMS)
def test_logprobs_rows_of_one_finite_value(dtype, rows, c, k):
    """Nothing but one value, however large: uniform."""
    values = torch.tensor(FILLS + [-v for v in FILLS] + [torch.finfo(dtype).max, torch.finfo(dtype).min, 65535.996, -65536.0])
    x = values.repeat(-(-rows // len(values)))[:rows, None].expand(rows, c).to(dtype).contiguous()
    check_logprobs(x, torch.arange(rows) * 61 % c, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c,k", FORMS)
@pytest.mark.parametrize("where", ["most", "prefix", "suffix"])
def test_logprobs_masked_by_finite_values(dtype, rows, c, k, where):
    """A few ordinary logits among fills: the fills have probability 0, whichever lanes see nothing else."""
    g = gen(c)
    x = (torch.randn(rows, c, generator=g) * 3).to(dtype)
    at = torch.arange(c).expand(rows, c)
    masked = {"most": torch.rand(rows, c, generator=g) < 0.95, "prefix": at < c - 40, "suffix": at >= 40}[where]
    fill = torch.tensor(FILLS).repeat(-(-rows // len(FILLS)))[:rows, None].to(dtype)
    x = torch.where(masked, fill.expand(rows, c), x)
    check_logprobs(x, torch.randint(0, c, (rows, 4), generator=g), k)


@pytest.mark.parametrize("rows,c,k", FORMS)
def test_logprobs_of_large_logits(rows, c, k):
    """Distributions far from 0, where neighbouring values still differ by a few nats or by fractions of one; logits on both
    sides of 2^16 and next to the type's ends."""
    g = gen(rows + c)
    x = torch.randn(rows, c, generator=g) * 3
    x[0] += 60000
    x[1] += 65536
    x[2] -= 65536
    x[3] += 1e6
    x[4] -= 1e7
    x[5] = 1e10 + 1024 * torch.randint(0, 3, (c,), generator=g)
    x[6] = -65536 - 2.0 ** -8 * torch.randint(0, 4, (c,), generator=g)
    x[7] = torch.tensor([-65536.0, -65535.996])[torch.randint(0, 2, (c,), generator=g)]
    x[8] = -1e30
    x[8, c - 2] = torch.finfo(torch.float32).max
    x[9, 5] = torch.finfo(torch.float32).max
    x[10, ::2] = 2.5e38
    x[10, 7] = 3e38
    x[11] = torch.randn(c, generator=g) * 1e5
    check_logprobs(x, torch.randint(0, c, (rows, 2), generator=g), k)


def test_logprobs_not_finite_among_large_logits():
    """A NaN or +inf is found beside any finite logit; -inf among them stays a mask."""
    for c in (1500, 30000):
        for value in (1e5, -1e10, 3e38, -3e38):
            x = torch.full((4, c), value)
            x[0, c // 3] = math.nan
            x[1, c - 1] = math.inf
            x[2, 100:] = -math.inf
            got = label_logprobs(x.to(DEV), torch.zeros(4, dtype=torch.int64, device=DEV), 3)
            for r in (0, 1):
                assert got.logp[r].isnan() and got.entropy[r].isnan() and got.top_logp[r].isnan().all()
                assert got.top_idx[r].eq(-1).all()
            assert got.top_idx[2:].cpu().tolist() == [[0, 1, 2]] * 2
            # 32-bit sums of up to c / 256 + 64 equal terms, and a logarithm
            for r, n in ((2, 100), (3, c)):
                assert abs(got.logp[r].item() + math.log(n)) <= (c / 256 + 64) * 2.0 ** -24 + math.log(n) * 2.0 ** -22


@pytest.mark.parametrize("shape", [(0, 40), (0, 3000), (2, 0, 600), (0, 0, 128)])
def test_no_rows(shape):
    """A batch without rows goes through every operator, alone and in their order."""
    lead, c = shape[:-1], shape[-1]
    x = torch.empty(shape, device=DEV)
    w = mx_quantize(torch.randn(30, c, device=DEV))
    for fmt in ("e2m1", "e4m3"):
        q = mx_quantize(x.bfloat16(), fmt)
        assert q.shape == shape and q.scale.shape == (*lead, mx.padded(c) // 32)
        assert mx_dequantize(q).shape == shape
        assert mx_linear(q, w).shape == (*lead, 30)
    for residual in (None, x):
        q, h = rms_norm_mx8(x, torch.ones(c, device=DEV), residual)
        assert q.shape == shape and (h is None if residual is None else h.shape == shape)
        y = mx_linear(q, w)
        got = label_logprobs(y, torch.empty(lead, dtype=torch.int64, device=DEV), 5)
        assert got.logp.shape == got.entropy.shape == lead and got.top_idx.shape == got.top_logp.shape == (*lead, 5)


@pytest.mark.parametrize("c", [64, 3000, 20000])
def test_rms_norm_where_eps_outweighs_the_squares(c):
    """y is next to a border by less than 32 bits hold, below it and above. eps itself is a 32-bit number on both devices."""
    x = torch.full((3, c), 2.0 ** -24)  # the squares are 2^-28 of eps
    x[1] = -x[1]
    for gamma, eps, value in ((1.1875, 2.0 ** -20, 1.125), (1.0625, 2.0 ** -20 * (1 - 2.0 ** -24), 1.125), (1.0625, 2.0 ** -20, 1.0)):
        g = torch.full((c,), gamma)
        assert oracle.mx_values(oracle.rms_norm(x, g, None, eps), "e4m3")[0].eq(value * 2.0 ** -14).all()
        for dev in ("cpu", DEV):
            for e in (eps, eps * (1 + 2.0 ** -27), eps * (1 - 2.0 ** -27)):
                q, _ = rms_norm_mx8(x.to(dev), g.to(dev), None, e)
                assert mx_dequantize(q)[[0, 2]].eq(value * 2.0 ** -14).all() and mx_dequantize(q)[1].eq(-value * 2.0 ** -14).all()
    tiny = x * 2.0 ** -46
    q, _ = rms_norm_mx8(tiny, g, None, 2.0 ** -149)
    p, _ = rms_norm_mx8(tiny.to(DEV), g.to(DEV), None, 2.0 ** -149)
    assert torch.equal(mx_dequantize(p).cpu(), mx_dequantize(q))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("c", [64, 500, 3000, 8192, 20000])
def test_rms_norm_of_sums_past_32_bits(dtype, c):
    """x + residual lies above 4.25, of which 1.0625 is the border between 1 and 1.125, by less than 32 bits hold. Sums of
    16-bit rows are 32-bit numbers (4.25, which falls to 4); of 32-bit rows what the sum lost counts (4.5). So on both devices."""
    x, r = torch.full((2, c), 4.25), torch.full((2, c), 2.0 ** -23)
    r[1] = 0
    eps = 2.0 ** 40  # y is the sum times 2^-20, less 2^-37 of it
    x, r, gamma = x.to(dtype), r.to(dtype), torch.ones(c)
    first = 4.5 if dtype == torch.float32 else 4.0
    want = torch.tensor([first, 4.0])[:, None].expand(2, c) * 2.0 ** -20
    for dev in ("cpu", DEV):
        q, h = rms_norm_mx8(x.to(dev), gamma.to(dev), r.to(dev), eps)
        assert torch.equal(mx_dequantize(q).cpu(), want) and h.eq(4.25).all(), dev
