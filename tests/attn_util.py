"""Plain attention in 64 bits and the error bound that the kernels are held to.

With u the unit roundoff of the 16-bit type (2^-11 F16, 2^-8 BF16), a result
out_c = sum_j p_j v_jc may differ from the exact one by
    u |out_c|                 its own rounding (none for F32 results), and
    (u + 2e) sum_j p_j |v_jc| each weight rounded to the type, and off by the
                              relative error e of exp(score - max), and
    n 2^-31 max |v|           F16 weights below its normal range,
where e = (dim + 8) 2^-23 max_j sum_c |q_c k_jc| scale + 2^-20 covers fp32 sums
of dim products and the exponential.  A log-sum-exp may differ by 2e plus 2^-20
of its size.
"""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend64(q, k, v, scale, visible):
    """q [rows, d], k and v [n, d] doubles, visible [rows]: keys each row sees.
    Returns out, lse, sum p|v|, e per row."""
    n = k.shape[0]
    rows = q.shape[0]
    if n == 0:
        z = torch.zeros(rows, v.shape[1], dtype=torch.float64, device=q.device)
        return z, torch.full((rows,), float("-inf"), dtype=torch.float64, device=q.device), z, z[:, :1]
    s = (q @ k.T) * scale
    mask = torch.arange(n, device=q.device)[None, :] >= visible[:, None]
    s = s.masked_fill(mask, float("-inf"))
    lse = torch.logsumexp(s, 1)
    p = torch.where(mask, torch.zeros_like(s), (s - lse[:, None]).exp())
    p = torch.where(visible[:, None] > 0, p, torch.zeros_like(p))
    mag = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(mask, 0.0).amax(1, keepdim=True)
    e = (q.shape[1] + 8) * 2.0 ** -23 * mag + 2.0 ** -20
    return p @ v, lse, p @ v.abs(), e


def bound(dtype, out_dtype, out, weighted, e, n, vmax):
    u = U[dtype]
    own = 0.0 if out_dtype == torch.float32 else u
    return own * out.abs() + (u + 2 * e) * weighted + n * 2.0 ** -31 * vmax + 2.0 ** -24


def check_rows(got, dtype, q, k, v, scale, visible, lse=None):
    """One head of one sequence: got [rows, d] against the definition."""
    out, want_lse, weighted, e = attend64(q.double(), k.double(), v.double(), scale, visible)
    vmax = v.double().abs().max().item() if v.numel() else 0.0
    tol = bound(dtype, got.dtype, out, weighted, e, k.shape[0], vmax)
    diff = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (diff <= tol).all(), f"off by {(diff / tol).max().item():.2f} bounds"
    if lse is not None:
        empty = visible <= 0
        assert torch.equal(torch.isneginf(lse), empty)
        ok = ~empty
        err = (lse.double() - want_lse)[ok].abs()
        assert (err <= (2 * e[:, 0] + 2.0 ** -20 * (1 + want_lse.abs()))[ok]).all()
