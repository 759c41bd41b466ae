"""Language-model operators on the GPU against 64-bit oracles: MX quantisation, MX product, RMS norm to e4m3, label
log-probabilities; then the four in a row, on streams and in graphs."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import lm_oracle as oracle
from aiforearth_api_platform_amd.ops import _ext, mx
from aiforearth_api_platform_amd.ops.head import label_logprobs
from aiforearth_api_platform_amd.ops.mx import MxTensor, mx_dequantize, mx_linear, mx_quantize
from aiforearth_api_platform_amd.ops.norm import rms_norm_mx8
from test_lm_ops_cpu import special_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes(q):
    return q.data.view(torch.uint8).cpu(), q.scale.view(torch.uint8).cpu()


# ---------------------------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("k", [1, 31, 32, 33, 127, 128, 129, 1000, 4096, 4103])
def test_quantize(dtype, fmt, k):
    x = special_rows(k, seed=k).to(dtype)
    q = mx_quantize(x.to(DEV), fmt)
    want = mx.quantize_reference(x.float(), fmt)  # equal to the 64-bit oracle on the same rows (CPU test)
    assert all(torch.equal(a, b) for a, b in zip(codes(q), codes(want)))
    values = oracle.mx_values(x, fmt)
    for out in DTYPES:
        got, ref = mx_dequantize(q, out).cpu(), values.float().to(out)
        assert got.shape == x.shape and torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got[~ref.isnan()], ref[~ref.isnan()])


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quantize_every_16_bit_value(fmt):
    """Every bf16 and fp16 value in a block whose scale another value sets: all roundings of the formats."""
    for dtype in (torch.bfloat16, torch.float16):
        v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
        v = v[torch.isfinite(v)].sort().values
        v = torch.nn.functional.pad(v, (0, -v.numel() % 31)).view(-1, 31)
        x = torch.cat((v, v.abs().amax(1, keepdim=True)), 1)
        got = mx_quantize(x.to(DEV), fmt)
        assert all(torch.equal(a, b) for a, b in zip(codes(got), codes(mx.quantize_reference(x.float(), fmt))))


def test_quantize_strided_and_unaligned_rows():
    base = torch.randn(40, 515, generator=gen(1)).bfloat16()
    d = base.to(DEV)
    for a, b in ((d[:, 3:203], base[:, 3:203]), (d[::3, 1:514], base[::3, 1:514]), (d.t()[5:50], base.t()[5:50]),
                 (d[:1].expand(7, 515), base[:1].expand(7, 515)), (d.view(8, 5, 515)[:, 2], base.view(8, 5, 515)[:, 2])):
        for fmt in ("e2m1", "e4m3"):
            assert all(torch.equal(x, y) for x, y in zip(codes(mx_quantize(a, fmt)), codes(mx.quantize_reference(b.float(), fmt))))


def test_quantize_writes_its_rows_only():
    x = torch.randn(5, 200, generator=gen(2)).bfloat16().to(DEV)
    data = torch.full((5 * 256 + 512,), 0x5A, dtype=torch.uint8, device=DEV)
    scale = torch.full((5 * 8 + 64,), 0x5A, dtype=torch.uint8, device=DEV)
    _ext.call_on(x.get_device(), "ai4e_mx_quantize", x.data_ptr(), 200, 5, 200, 0, 0, data[256:].data_ptr(), scale[32:].data_ptr())
    torch.cuda.synchronize()
    assert data[:256].eq(0x5A).all() and data[256 + 5 * 256:].eq(0x5A).all()
    assert scale[:32].eq(0x5A).all() and scale[32 + 40:].eq(0x5A).all()


# ---------------------------------------------------------------------------------------------- product

def linear_error_bound(xv, wv, want, dtype, fmt):
    """Half a step of the result, and 32-bit accumulators: one rounding per matrix instruction of 64 and one per part of
    a split sum, 2^-24 of at most the sum of the absolute products. Sums of e4m3 products inside an instruction keep
    about 17 bits: 2^-14 of the absolute products is five times the largest that was measured."""
    s = xv.abs() @ wv.abs().T
    steps = xv.shape[1] / 64 + 16
    return want.abs() * U[dtype] + s * (steps * 2.0 ** -24 + (2.0 ** -14 if fmt == "e4m3" else 0)) + 1e-37


def check_linear(m, n, k, fmt, dtype, bias, seed=0, scale=1.0):
    g = gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))
    w = torch.randn(n, k, generator=g) * scale / math.sqrt(k)
    b = torch.randn(n, generator=g) if bias else None
    xq, wq = mx.quantize_reference(x, fmt), mx.quantize_reference(w, "e2m1")
    y = mx_linear(xq.to(DEV), wq.to(DEV), None if b is None else b.to(DEV), dtype)
    xv, wv = mx.dequantize_reference(xq).double(), mx.dequantize_reference(wq).double()
    want = xv @ wv.T + (0 if b is None else b.double())
    got = y.cpu().double()
    assert y.shape == (m, n) and y.dtype == dtype
    err, bound = (got - want).abs(), linear_error_bound(xv, wv, want, dtype, fmt)
    assert (err <= bound).all(), f"{(err / bound).max().item()} at {(err / bound).argmax().item()}"


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("e4m3", torch.float16), ("e2m1", torch.bfloat16),
                                       ("e2m1", torch.float16), ("e2m1", torch.float32)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 33, 129), (1, 1000, 4096), (2, 64, 512), (5, 100, 640), (15, 257, 1000),
                                   (16, 48, 8192), (17, 32, 128), (31, 31, 384), (33, 65, 300), (64, 128, 1024),
                                   (65, 200, 257), (100, 1000, 2048), (129, 255, 512), (255, 257, 769), (300, 520, 1100)])
def test_linear(m, n, k, fmt, dtype):
    check_linear(m, n, k, fmt, dtype, bias=(m + n) % 2 == 1, seed=m + n + k)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("m,n,k", [(512, 768, 256), (1024, 1024, 4096), (777, 1300, 2000), (2048, 512, 1024)])
def test_linear_large(m, n, k, fmt):
    check_linear(m, n, k, fmt, torch.bfloat16, bias=True, seed=m)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("e4m3", torch.float16), ("e2m1", torch.bfloat16),
                                       ("e2m1", torch.float32)])
@pytest.mark.parametrize("m,n,k", [(70, 12500, 1000), (1600, 2001, 640), (3500, 3699, 520), (2500, 300, 200),
                                   (3300, 4100, 1664), (20, 24601, 1024), (32, 24600, 640), (70, 4201, 1024),
                                   (128, 4096, 1536), (16, 14000, 512), (64, 12300, 2048)])
def test_linear_every_tile(m, n, k, fmt, dtype):
    """Every tile kernel, slices of many rows, odd counts of steps."""
    check_linear(m, n, k, fmt, dtype, bias=True, seed=m)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("m", [1, 16, 40, 200, 600])
def test_linear_not_finite_blocks_stay_in_their_row(m, fmt):
    g = gen(m)
    x, w = torch.randn(m, 320, generator=g), torch.randn(600, 320, generator=g)
    x[m // 2, 77] = math.nan
    w[10, 300] = math.inf
    y = mx_linear(mx_quantize(x.to(DEV), fmt), mx_quantize(w.to(DEV)), out_dtype=torch.bfloat16).cpu()
    want = torch.zeros(m, 600, dtype=torch.bool)
    want[m // 2] = True
    want[:, 10] = True
    assert torch.equal(y.isnan(), want)


@pytest.mark.parametrize("m,n", [(3, 37), (130, 130), (300, 515)])
def test_linear_writes_its_rows_only(m, n):
    g = gen(7)
    xq, wq = mx_quantize(torch.randn(m, 256, generator=g).to(DEV), "e4m3"), mx_quantize(torch.randn(n, 256, generator=g).to(DEV))
    buf = torch.full((m * n + 2048,), 7.0, dtype=torch.bfloat16, device=DEV)
    _ext.call_on(buf.get_device(), "ai4e_mx_linear", xq.data.data_ptr(), xq.scale.data_ptr(), 0, wq.data.data_ptr(),
                 wq.scale.data_ptr(), None, m, n, 256, buf[1024:].data_ptr(), 0)
    torch.cuda.synchronize()
    assert buf[:1024].eq(7).all() and buf[1024 + m * n:].eq(7).all()
    assert torch.equal(buf[1024:1024 + m * n].view(m, n), mx_linear(xq, wq))


def test_linear_scales_at_the_ends_of_their_range():
    x = torch.ones(4, 128) * 2.0 ** -126
    w = torch.ones(3, 128) * 2.0 ** 100
    y = mx_linear(mx_quantize(x.to(DEV), "e2m1"), mx_quantize(w.to(DEV)), out_dtype=torch.float32)
    assert y.cpu().eq(128 * 2.0 ** -26).all()
    big = torch.ones(4, 128) * 2.0 ** 120
    y = mx_linear(mx_quantize(big.to(DEV), "e4m3"), mx_quantize(w.to(DEV)), out_dtype=torch.bfloat16)
    assert y.cpu().eq(math.inf).all()


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("e2m1", torch.float32)])
@pytest.mark.parametrize("m,n,k", [(1793, 1700, 384), (1700, 1793, 200), (2000, 1650, 100), (833, 1030, 384), (40, 12300, 7),
                                   (12289, 4, 300), (24577, 5, 128), (30000, 3, 128), (33, 12289, 256),
                                   (4097, 4100, 130), (131073, 4, 384)])
def test_linear_short_rows(m, n, k, fmt, dtype):
    """Fewer than 4 steps of k: tiles whose last rows' scales end with the tensor, and the slices where no tile fits."""
    check_linear(m, n, k, fmt, dtype, bias=True, seed=m)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("e2m1", torch.float32)])
@pytest.mark.parametrize("m,n,k", [(1, 33000, 512), (32, 24600, 2500), (17, 65700, 640), (9, 40001, 1152), (31, 33300, 896)])
def test_linear_few_rows(m, n, k, fmt, dtype):
    """Up to 32 rows over several tiles of a workgroup, the last one ragged; a last group of k that shares steps."""
    check_linear(m, n, k, fmt, dtype, bias=True, seed=n)


def test_linear_same_call_same_bits():
    g = gen(9)
    for m, n, k in ((1, 512, 4096), (16, 1024, 8192), (200, 300, 4096)):
        xq, wq = mx_quantize(torch.randn(m, k, generator=g).to(DEV), "e4m3"), mx_quantize(torch.randn(n, k, generator=g).to(DEV))
        y = mx_linear(xq, wq)
        for _ in range(5):
            assert torch.equal(y, mx_linear(xq, wq))


# ---------------------------------------------------------------------------------------------- RMS norm

def check_norm(x, gamma, residual, eps=1e-6):
    q, h = rms_norm_mx8(x.to(DEV), gamma.to(DEV), None if residual is None else residual.to(DEV), eps)
    c = x.shape[-1]
    x2, r2 = x.reshape(-1, c), None if residual is None else residual.reshape(-1, c)
    want = oracle.rms_norm(x2, gamma, r2, eps)
    got = mx_dequantize(q).cpu().double().view(-1, c)
    code = q.scale.view(torch.uint8).cpu().view(got.shape[0], -1)
    bad = ~torch.isfinite(want)
    blocks = torch.nn.functional.pad(bad, (0, -c % 32)).view(bad.shape[0], -1, 32).any(-1)
    assert torch.equal(code[:, :blocks.shape[1]] == 255, blocks)
    assert code[:, blocks.shape[1]:].eq(0).all()
    e = code.double()[:, :blocks.shape[1]] - 127
    # y within a few roundings to 32 bits of the sum x + residual, the squares' sum and the two products
    near = 2.0 ** -21
    amax = torch.nn.functional.pad(torch.where(bad, 0.0, want.abs()), (0, -c % 32)).view(bad.shape[0], -1, 32).amax(-1)
    pow2 = torch.pow(torch.tensor(2.0, dtype=torch.float64), e)
    ok = blocks | ((amax * (1 - near) <= 448 * pow2) & ((amax * (1 + near) > 224 * pow2) | (e == -127)))
    assert ok.all()
    s = pow2.repeat_interleave(32, 1)[:, :c]
    tol = oracle.half_step(want / s, "e4m3") * s * (1 + 2.0 ** -10) + want.abs() * near
    fine = ~blocks.repeat_interleave(32, 1)[:, :c]
    assert ((got - want).abs() <= tol)[fine].all()
    flips = (got != oracle.mx_values(torch.where(bad, 0.0, want), "e4m3"))[fine].sum().item()
    assert flips <= 2 + fine.sum().item() * 2.0 ** -12  # a value falls within 2^-21 of a border, 2^-4 apart, that rarely
    if residual is None:
        assert h is None
    else:
        assert torch.equal(h.cpu().nan_to_num(77.0), (x.float() + residual.float()).to(x.dtype).nan_to_num(77.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [1, 8, 31, 32, 33, 128, 200, 500, 512, 513, 2048, 2050, 4096, 5000, 8192, 8193, 20000])
def test_rms_norm(dtype, c):
    g = gen(c)
    for rows, with_residual in ((1, True), (3, False), (37, True)):
        x = (torch.randn(rows, c, generator=g) * torch.exp(torch.randn(c, generator=g))).to(dtype)
        r = torch.randn(rows, c, generator=g).to(dtype) if with_residual else None
        check_norm(x, torch.randn(c, generator=g), r)


@pytest.mark.parametrize("c", [64, 3000, 10000])
def test_rms_norm_ranges_and_not_finite(c):
    g = gen(c)
    x = torch.randn(9, c, generator=g)
    x[0] *= 1e30          # squares over 32 bits
    x[1] *= 1e-25
    x[2] = 0
    x[3, c // 2] = math.nan
    x[4, 1] = math.inf    # the others of its row are 0 by the formula, inf / inf is nan
    x[5] = 3e38 * torch.sign(x[5])
    check_norm(x, torch.rand(c, generator=g) + 0.5, None)
    check_norm(x.bfloat16(), torch.rand(c, generator=g) + 0.5, torch.zeros(9, c).bfloat16())


@pytest.mark.parametrize("dtype,c,with_residual", [(torch.float32, 2500, True), (torch.float32, 700, False),
                                                   (torch.bfloat16, 4096, True), (torch.float16, 20000, True)])
def test_rms_norm_elements_are_the_exact_values_neighbours(dtype, c, with_residual):
    """y is held to some 2^-40 of itself: of a million elements, whose borders are 2^-4 apart, none falls to the other side."""
    g = gen(c)
    x = torch.randn(1 << 20, generator=g)[:(1 << 20) // c * c].view(-1, c).to(dtype)
    r = torch.randn(x.shape, generator=g).to(dtype) if with_residual else None
    gamma = torch.rand(c, generator=g) + 0.5
    q, _ = rms_norm_mx8(x.to(DEV), gamma.to(DEV), None if r is None else r.to(DEV))
    assert torch.equal(mx_dequantize(q).cpu().double(), oracle.mx_values(oracle.rms_norm(x, gamma, r, 1e-6), "e4m3"))


def test_rms_norm_sum_past_the_type():
    """A 32-bit sum that overflows is an infinity: its block is not finite, what else is in the row becomes 0."""
    x = torch.ones(2, 96)
    x[0, 40] = 3e38
    for dev in ("cpu", DEV):
        q, h = rms_norm_mx8(x.to(dev), torch.ones(96, device=dev), x.to(dev))
        assert q.scale.view(torch.uint8).cpu()[0].tolist() == [0, 255, 0, 0] and math.isinf(h[0, 40].item())
        assert q.data.view(torch.uint8)[0].eq(0).all() and torch.equal(mx_dequantize(q)[1].cpu(), torch.ones(96))


def test_rms_norm_strided_and_leading_axes():
    g = gen(4)
    x, r = torch.randn(6, 5, 333, generator=g).half(), torch.randn(6, 5, 333, generator=g).half()
    gamma = torch.randn(333, generator=g)
    check_norm(x, gamma, r)
    a, b = torch.randn(12, 700, generator=g).bfloat16(), torch.randn(12, 640, generator=g).bfloat16()
    q, h = rms_norm_mx8(a.to(DEV)[:, 7:340], gamma.to(DEV), b.to(DEV)[:, 1:334])
    q2, h2 = rms_norm_mx8(a[:, 7:340].contiguous().to(DEV), gamma.to(DEV), b[:, 1:334].contiguous().to(DEV))
    assert all(torch.equal(u, v) for u, v in zip(codes(q), codes(q2))) and torch.equal(h, h2)
    q3, _ = rms_norm_mx8(a.to(DEV)[:1, :333].expand(4, 333), gamma.to(DEV).bfloat16())
    assert torch.equal(codes(q3)[0][0], codes(q3)[0][3])


# ---------------------------------------------------------------------------------------------- log-probabilities

def check_logprobs(x, labels, k):
    got = label_logprobs(x.to(DEV), None if labels is None else labels.to(DEV), k)
    c = x.shape[-1]
    lab = None if labels is None else labels.reshape(x.shape[0], -1)
    logp, ent, idx, top = oracle.logprobs(x, lab, k)
    assert got.top_idx.shape == (x.shape[0], k) and torch.equal(got.top_idx.cpu().long(), idx)
    # a lane adds at most c / 256 + 8 terms, then 6 + 2 + 6 joins, each a rounding or two of 2^-24; e^u is good to 2^-22
    s_err = (c / 256 + 64) * 2.0 ** -24
    for a, b in ((got.top_logp, top), (got.logp, None if logp is None else logp.view(labels.shape))):
        if b is not None:
            a = a.cpu().double()
            assert torch.equal(torch.isinf(a), torch.isinf(b)) and not a.isnan().any()
            fine = ~torch.isinf(b)
            assert ((a - b).abs() <= s_err + b.abs() * 2.0 ** -22)[fine].all()
    assert ((got.entropy.cpu().double() - ent).abs() <= s_err * 3 * (1 + math.log(c))).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,k", [(1, 1, 1), (1, 7, 3), (3, 8, 8), (250, 1000, 5), (5, 63, 63), (2, 2047, 64),
                                      (4, 4099, 20), (3, 50001, 20), (1, 32768, 5), (1, 131072, 64), (600, 9000, 1),
                                      (1500, 300, 0), (2, 262147, 10)])
def test_logprobs(dtype, rows, c, k):
    g = gen(rows + c)
    x = (torch.randn(rows, c, generator=g) * 3).to(dtype)
    check_logprobs(x, torch.randint(0, c, (rows,), generator=g), k)
    check_logprobs(x, torch.randint(-1, c, (rows, 3), generator=g, dtype=torch.int32), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(9, 100), (9, 5000), (1400, 2600), (9, 40000)])
def test_logprobs_masks_and_ties(dtype, rows, c):
    g = gen(c)
    x = torch.randn(rows, c, generator=g).to(dtype)
    lowest = torch.finfo(dtype).min
    x[0, torch.rand(c, generator=g) < 0.9] = -math.inf
    x[1] = -math.inf                       # nothing left
    x[2] = lowest                          # all masked by the type's lowest value: uniform
    x[3, 3:] = -math.inf                   # fewer than k left
    x[4] = 1.5                             # every class ties
    x[5, : c // 2] = lowest
    x[6] = torch.arange(c, 0, -1).to(dtype)  # descending, with ties in 16 bits
    x[7] = torch.where(torch.rand(c, generator=g) < 0.5, 0.0, -0.0).to(dtype)  # 0 and -0 tie
    x[8, c - 1] = 200.0                    # all probability on one class
    labels = torch.randint(0, c, (rows,), generator=g)
    labels[0], labels[3] = int(x[0].float().argmin()), c - 1  # masked labels
    check_logprobs(x, labels, 10)


@pytest.mark.parametrize("c", [8192, 60000])
def test_logprobs_more_candidates_than_room(c):
    """Ten lanes see all large logits: the candidates overflow LDS and the rounds find the best."""
    g = gen(c)
    x = torch.randn(1100, c, generator=g)
    chunk = torch.arange(c) // 8
    x[3] = torch.where(chunk % 256 < 10, 50 + torch.rand(c, generator=g), x[3])
    x[3] += torch.where((chunk % 256 >= 10) & (chunk % 256 < 30) & (chunk < 256) & (torch.arange(c) % 8 == 0), 45.0, 0.0)
    x[5, :] = -math.inf
    x[5, (chunk % 256 < 19)] = torch.randn(int((chunk % 256 < 19).sum()), generator=g)
    labels = torch.randint(0, c, (1100,), generator=g)
    check_logprobs(x, labels, 20)
    check_logprobs(x[:8].contiguous(), labels[:8], 20)


@pytest.mark.parametrize("dtype,rows,c,k", [(torch.bfloat16, 2100, 130001, 20), (torch.float16, 9000, 30000, 64)])
def test_logprobs_more_than_caches_hold(dtype, rows, c, k):
    """Rows of a call of over 512 MB, against the same rows called by themselves and a few of them against the oracle."""
    g = torch.Generator(DEV).manual_seed(c)
    x = torch.empty(rows, c, device=DEV, dtype=dtype).normal_(0, 3, generator=g)
    x[0, 100:] = -math.inf
    x[1] = 1.0
    x[2] = -math.inf
    x[rows - 1, ::3] = torch.finfo(dtype).min
    labels = torch.randint(0, c, (rows,), generator=g, device=DEV)
    got = label_logprobs(x, labels, k)
    for at in (0, rows // 2, rows - 300):
        part = label_logprobs(x[at:at + 300], labels[at:at + 300], k)
        assert torch.equal(got.top_idx[at:at + 300], part.top_idx)
        for a, b in ((got.logp, part.logp), (got.entropy, part.entropy), (got.top_logp, part.top_logp)):
            assert torch.equal(a[at:at + 300], b)
    pick = [0, 1, 2, rows // 2, rows - 1]
    check_logprobs(x[pick].cpu(), labels[pick].cpu(), k)


def test_logprobs_not_finite_rows():
    for c in (500, 30000):
        x = torch.randn(6, c, generator=gen(c))
        x[1, c // 3] = math.nan
        x[2, c - 1] = math.inf
        x[4] = math.nan
        x[5] = -math.inf
        x[5, 3] = math.nan
        labels = torch.tensor([0, 1, 2, c, -1, 3])
        got = label_logprobs(x.to(DEV), labels.to(DEV), 6)
        ref = label_logprobs(x, labels, 6)
        assert torch.equal(got.top_idx.cpu(), ref.top_idx)
        for a, b in ((got.logp, ref.logp), (got.entropy, ref.entropy), (got.top_logp, ref.top_logp)):
            assert torch.allclose(a.cpu(), b, rtol=1e-5, atol=1e-5, equal_nan=True)
        assert got.logp[3].isnan() and got.logp[4] == 0


def test_logprobs_strided_and_leading_axes():
    g = gen(11)
    base = torch.randn(6, 777, generator=g).bfloat16()
    labels = torch.randint(0, 700, (6,), generator=g)
    want = label_logprobs(base[:, 5:705].contiguous().to(DEV), labels.to(DEV), 4)
    for v in (base.to(DEV)[:, 5:705], base.to(DEV).t().contiguous().t()[:, 5:705]):
        assert all(torch.equal(a, b) for a, b in zip(label_logprobs(v, labels.to(DEV), 4), want))
    three = label_logprobs(base.to(DEV).view(2, 3, 777)[..., 5:705], labels.view(2, 3).to(DEV), 4)
    assert three.top_idx.shape == (2, 3, 4) and torch.equal(three.logp.view(6), want.logp)
    wide = torch.stack((labels, labels + 1), 1).to(DEV)
    two = label_logprobs(base.to(DEV)[:, 5:705], wide.t().contiguous().t(), 4)  # labels of another order
    assert torch.equal(two.logp[:, 0], want.logp)


# ---------------------------------------------------------------------------------------------- together

def tail(x, r, gamma, wq, labels, k=5):
    q, h = rms_norm_mx8(x, gamma, r)
    return (h, *label_logprobs(mx_linear(q, wq, out_dtype=torch.float16), labels, k))


def tail_inputs(rows, seed, c=512, n=3000):
    g = gen(seed)
    return (torch.randn(rows, c, generator=g).bfloat16().to(DEV), torch.randn(rows, c, generator=g).bfloat16().to(DEV),
            (torch.rand(c, generator=g) + 0.5).to(DEV), mx_quantize((torch.randn(n, c, generator=g) / 8).to(DEV)),
            torch.randint(0, n, (rows,), generator=g).to(DEV))


@pytest.mark.parametrize("rows", [1, 5, 130])
def test_norm_projection_logprobs(rows):
    x, r, gamma, wq, labels = tail_inputs(rows, rows)
    h, logp, ent, idx, top = tail(x, r, gamma, wq, labels)
    y = oracle.rms_norm(x, gamma, r, 1e-6)
    logits = oracle.mx_values(y, "e4m3") @ mx_dequantize(wq).cpu().double().T
    rl, re, ri, rt = oracle.logprobs(logits, labels.cpu()[:, None], 5)
    # logits of up to 40 rounded to 11 bits (2^-11 of 40), and a flipped 8-bit value now and then
    tol = 40 * 2.0 ** -11 + 0.02
    assert (logp.cpu().double() - rl[:, 0]).abs().max() <= 2 * tol
    assert (top.cpu().double() - rt).abs().max() <= 2 * tol and (ent.cpu().double() - re).abs().max() <= 8 * tol
    assert (logits.gather(1, idx.cpu().long()) - logits.gather(1, ri)).abs().max() <= 2 * tol
    assert torch.equal(h.cpu(), (x.float() + r.float()).bfloat16().cpu())


def test_on_another_stream():
    x, r, gamma, wq, labels = tail_inputs(64, 3)
    want = tail(x, r, gamma, wq, labels)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tail(x, r, gamma, wq, labels)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [2, 70])
def test_two_captured_graphs(rows):
    """Two graphs of the same operators replayed in turns and on two streams at once, with eager calls between."""
    sets = [tail_inputs(rows, 20 + i, n=9000) for i in range(2)]
    want = [tail(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    graphs, outs = [], []
    for s, st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            tail(*s)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(tail(*s))
        graphs.append(g)
    for turn in range(4):
        for o in outs:
            for t in o:
                t.fill_(7)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w, s in zip(outs, want, sets):
            assert all(torch.equal(a, b) for a, b in zip(o, w)), turn
            assert all(torch.equal(a, b) for a, b in zip(tail(*s), w))


FIRST_CALL = """
import torch
from aiforearth_api_platform_amd.ops.head import label_logprobs
from aiforearth_api_platform_amd.ops.mx import mx_linear, mx_quantize, mx_dequantize
from aiforearth_api_platform_amd.ops.norm import rms_norm_mx8
x, w = torch.randn(300, 640, device="cuda"), torch.randn(4100, 640, device="cuda")
gamma, labels = torch.ones(640, device="cuda"), torch.arange(300, device="cuda")

def run(rows):
    q, h = rms_norm_mx8(x[:rows], gamma, x[:rows])
    y = mx_linear(q, mx_quantize(w))
    return [h, y, mx_dequantize(q), *label_logprobs(y, labels[:rows], 3)]

rows = (1, 16, 60, 300)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = [run(r) for r in rows]
for _ in range(3):
    g.replay()
    torch.cuda.synchronize()
    for r, out in zip(rows, outs):
        assert all(torch.equal(a, b) for a, b in zip(out, run(r))), r
print("same")
"""


def test_first_calls_in_a_capture():
    """A process whose first calls of the operators are captured: nothing is set up at a first eager call."""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr[-2000:]


def test_gpu_refusals():
    x = torch.randn(4, 64, device=DEV)
    with pytest.raises(ValueError):
        rms_norm_mx8(x, torch.ones(64))
    with pytest.raises(ValueError):
        rms_norm_mx8(x, torch.ones(64, device=DEV), torch.zeros(4, 64))
    with pytest.raises(ValueError):
        label_logprobs(x, torch.zeros(4, dtype=torch.int64), 1)
    with pytest.raises(ValueError):
        mx_linear(mx_quantize(x, "e4m3"), mx_quantize(torch.randn(4, 64)))
    q = mx_quantize(x)
    with pytest.raises(ValueError):
        mx_linear(MxTensor(q.data.view(-1)[8:8 + 64 * 3].view(3, 64), q.scale[:3], 64), q)  # not 16-byte aligned
