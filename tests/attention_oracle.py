"""Attention from its definition in 64 bits, and how far a kernel may be from it.

The kernel's result o~ of a query row differs from o = sum_j p_j v_j / l by
  - the rounding of each probability to the inputs' type: u A with A = sum_j
    p_j |v_j| / l and u half the type's step at 1 (2^-8 for bf16, 2^-11 for
    fp16); a probability that is not normal in fp16 is off by up to 2^-25
    where the largest is at least 1: 2^-25 sum_j |v_j|;
  - the scores: a sum of dim products in fp32 is off by up to dim 2^-24 sum_x
    |q_x k_x|, which enters p_j and l (twice) as a factor, and the base-2
    exponential with its argument by some 2^-22 |s|: 2 (dim + 8) 2^-24 S A
    with S the largest scale * sum_x |q_x k_x|, at least 1;
  - the sums of n terms in fp32: n 2^-24 A, twice;
  - the result's own rounding: u |o|, or 2^-25 where that is not normal.
"""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def attend(q, k, v, visible, scale):
    """(o, bound, lse) in 64 bits for q [n, heads, dim], k and v [m, kv_heads,
    dim], visible [n, m]; rows that see nothing: zeros and -inf."""
    dtype = q.dtype
    n, heads, dim = q.shape
    m, kv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    k, v = (x.repeat_interleave(heads // kv, 1) for x in (k, v))
    s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0)) * scale          # [heads, n, m]
    size = (torch.matmul(q.abs().transpose(0, 1), k.abs().permute(1, 2, 0)) * scale).masked_fill(~visible, 0.0)
    s = s.masked_fill(~visible, float("-inf"))
    if m == 0:
        return torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device), torch.zeros_like(q), \
            torch.full((n, heads), float("-inf"), dtype=torch.float64, device=q.device)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == float("-inf"), 0.0)[..., None])
    vt = v.transpose(0, 1)
    o = torch.matmul(p, vt).transpose(0, 1)
    a = torch.matmul(p, vt.abs()).transpose(0, 1)
    u = UNIT[dtype]
    most = size.amax(-1).clamp_min(1.0).t()[..., None]
    bound = (u + 2.0 ** -24 * (2 * (dim + 8) * most + 2 * m)) * a + u * o.abs()
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (1 + torch.matmul(visible.double(), vt.abs()).transpose(0, 1))
    return o, bound, lse.t()


def check(got, o, bound, where=""):
    """got within the bound (slightly above it: the bound leaves out products of small factors)."""
    off = (got.double() - o).abs() - 1.05 * bound
    assert bool((off <= 0).all()), "%s: off by %.3g more than %.3g" % (where, off.max().item(), bound.flatten()[off.argmax()].item())
