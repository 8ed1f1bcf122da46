"""Oracles in 64 bits of the per-row-id operators and the error bounds of their fp32 arithmetic."""
import numpy as np
import torch

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
EPS32 = torch.finfo(torch.float32).eps / 2      # one fp32 rounding, relative


def half_step(dtype):
    """One rounding to ``dtype``: relative error."""
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """One rounding of values below the normal range: half of fp16's smallest step, which is kept; fp32 and bf16 results
    below 2^-126 may be flushed."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound elementwise; non-finite values have to be the same ones."""
    got, want = got.double(), want.double().to(got.device)
    bound = torch.as_tensor(bound, dtype=torch.float64, device=got.device).expand_as(want)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: other infinities"
    off = (got - want).abs()[fine] - bound[fine]
    assert off.numel() == 0 or float(off.max()) <= 0.0, f"{what}: over its bound by {float(off.max()):.3g}"


def group_order(index, count):
    """numpy: (order, offsets) of the rows by id, ids outside 0 .. count - 1 last."""
    index = np.asarray(index).reshape(-1).astype(np.int64)
    key = np.where((index >= 0) & (index < count), index, count)
    sizes = np.bincount(key, minlength=count + 1)[:count]
    return np.argsort(key, kind="stable"), np.concatenate([[0], np.cumsum(sizes)])


def grouped_linear(x, w, index, bias=None, gy=None):
    """y (and with gy: d_x, d_w, d_b) in 64 bits, with the sums of absolute products that bound their rounding."""
    x, w = x.double(), w.double()
    (m, _), (g, n, _) = x.shape, w.shape
    out = {"y": x.new_zeros(m, n)}
    size = {"y": x.new_zeros(m, n)}
    if gy is not None:
        gy = gy.double()
        out.update(d_x=torch.zeros_like(x), d_w=torch.zeros_like(w), d_b=x.new_zeros(g, n))
        size.update({k: torch.zeros_like(v) for k, v in out.items() if k != "y"})
    for e in range(g):
        r = torch.nonzero(index == e)[:, 0]
        xe, we = x[r], w[e]
        out["y"][r] = xe @ we.T + (0 if bias is None else bias[e].double())
        size["y"][r] = xe.abs() @ we.abs().T + (0 if bias is None else bias[e].double().abs())
        if gy is not None:
            ge = gy[r]
            out["d_x"][r], size["d_x"][r] = ge @ we, ge.abs() @ we.abs()
            out["d_w"][e], size["d_w"][e] = ge.T @ xe, ge.abs().T @ xe.abs()
            out["d_b"][e], size["d_b"][e] = ge.sum(0), ge.abs().sum(0)
    return out, size


def product_bound(want, size, terms, dtype):
    """A sum of ``terms`` products in fp32 in any order: each of its at most terms + 8 roundings (the split of fp32
    operands drops up to 3 parts of 2^-24 per product, joins of partial sums are counted) is off by at most 2^-24 of
    the sum of absolute products - doubled for a matrix unit that truncates; then one rounding to ``dtype``."""
    return size * (terms + 8) * 2 * EPS32 + want.abs() * half_step(dtype) + least(dtype)


def distill(logits, index, teacher, temperature):
    """(loss per row, d loss / d logits per row, counts, size of the logarithms) in 64 bits."""
    s, t = logits.double() / temperature, teacher.double() / temperature
    m, v = s.shape
    has = (index >= 0) & (index < v) & ~(t == -torch.inf)
    counts = has.any(1)
    at = index.long().clamp(0, v - 1)
    t = torch.where(has, t, torch.full_like(t, -torch.inf))
    t = torch.where(counts[:, None], t, torch.zeros_like(t))
    # (relative to the largest: at the type's lowest value even 64 bits lose the logarithm of a sum)
    t = t - t.amax(1, keepdim=True)
    s = s - s.amax(1, keepdim=True)
    log_p = t - torch.logsumexp(t, 1, keepdim=True)
    p = torch.where(has, log_p.exp(), torch.zeros_like(t))
    log_q = s - torch.logsumexp(s, 1, keepdim=True)
    log_qe = torch.gather(log_q, 1, at)
    # 0 log 0 = 0 (the kernel's p is an fp32 number: below 2^-126 it is 0)
    terms = torch.where(p < 2.0 ** -126, torch.zeros_like(p), p * (log_p - log_qe))
    loss = torch.where(counts, terms.sum(1), torch.zeros(m, dtype=torch.float64, device=s.device)) * temperature ** 2
    target = torch.zeros_like(s).scatter_add_(1, at, p)
    q = log_q.exp()
    grad = torch.where(counts[:, None], (q - target) * temperature, torch.zeros_like(s))
    big = torch.where(p >= 2.0 ** -126, torch.maximum(log_p.abs(), log_qe.abs()), torch.zeros_like(p))
    return loss, grad, counts, big, q, target
