"""64-bit oracles of the MX formats, the RMS norm and the label log-probabilities, written from their definitions."""
import math

import torch

BLOCK = 32
LARGEST = {"e2m1": 6.0, "e4m3": 448.0}
GRID = {"e2m1": (0, 1), "e4m3": (-6, 3)}  # lowest exponent of a normal value, fraction bits


def _pow2(e):
    return torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())


def _exponent(v):
    """floor(log2 v) of positive 64-bit values, exact."""
    m, e = torch.frexp(v)
    return (e - 1).double()


def half_step(v, fmt):
    """Half the distance between neighbours of ``fmt`` at the scaled value ``v``."""
    lowest, fraction = GRID[fmt]
    e = torch.where(v == 0, torch.full_like(v, lowest), _exponent(v.abs().clamp_min(2.0 ** -200))).clamp_min(lowest)
    return _pow2(e - fraction - 1)


def mx(y, fmt):
    """[R, W] -> (elements [R, W], scale exponents [R, blocks]; nan where a block is not finite), 64 bits."""
    y = y.double().cpu()
    r, w = y.shape
    b = torch.nn.functional.pad(y, (0, -w % BLOCK)).view(r, -1, BLOCK)
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    amax = torch.where(bad, torch.ones_like(amax), amax)
    e = torch.where(amax > 0, _exponent(amax.clamp_min(2.0 ** -200)) - 9, torch.full_like(amax, -127))
    for _ in range(12):
        e = torch.where(amax > LARGEST[fmt] * _pow2(e), e + 1, e)
    e = e.clamp_min(-127)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    step = 2 * half_step(b / _pow2(e)[..., None], fmt)
    q = torch.round(b / _pow2(e)[..., None] / step) * step  # halves to even, as the elements are rounded
    return q.view(r, -1)[:, :w], torch.where(bad, torch.full_like(e, math.nan), e)


def mx_values(y, fmt):
    q, e = mx(y, fmt)
    return q * _pow2(e).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def rms_norm(x, gamma, residual, eps):
    h = x.double().cpu() if residual is None else x.double().cpu() + residual.double().cpu()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * gamma.double().cpu()


def logprobs(x, labels, k):
    """(logp, entropy, top classes, their logp) of [N, C] and labels [N, L]; rows with +inf or NaN are not handled."""
    x = x.double().cpu()
    m = x.amax(1, keepdim=True)
    none = torch.isneginf(m)[:, 0]
    d = x - torch.where(none[:, None], torch.zeros_like(m), m)
    log_s = torch.log(torch.exp(d).sum(1, keepdim=True))
    lp = torch.where(none[:, None], torch.full_like(d, -math.inf), d - log_s)
    term = torch.where(torch.isneginf(lp), torch.zeros_like(lp), torch.exp(lp) * lp)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    top = lp.gather(1, order)
    logp = None
    if labels is not None:
        labels = labels.cpu().long()
        logp = lp.gather(1, labels.clamp(0, x.shape[1] - 1))
        logp = torch.where(labels < 0, torch.zeros_like(logp), logp)
    return logp, -term.sum(1), torch.where(torch.isneginf(top), torch.full_like(order, -1), order), top
