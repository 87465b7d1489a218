"""Attention and its gradient in 64 bits on the CPU, written from the formulas, with bounds of what a
kernel may be off that rounds its weights once and its results once to 16 bits.

u is the unit roundoff of the type (half a step at 1: 2^-8 for bfloat16, 2^-11 for float16) and tiny the
error of its smallest steps.  To first order, element by element:

* out: u |out| from its own rounding, u sum_j P_ij |v_j| from the weights', with 2^-20 of the
  latter for sums in 32 bits, times 1 + max scale |q| . |k|, which scales a 32-bit score's error;
* grad_v: the same with P^T and grad_out;
* dS = P (dP - delta): its own rounding u |dS|, and delta = grad_out . out of an out that was
  rounded: u P sum |grad_out| |out|.  grad_q and grad_k: u of themselves, and those summed with
  |scale k| or |scale q|.
"""

import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}
SLACK = 1.05  # second order


def seen(nq, nk, causal, window):
    i = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)
    m = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        m &= j <= i
    if window:
        m &= j > i - window
    return m


def one(q, k, v, mask, scale, grad=None):
    """One head of one sequence, all [n, dim] in float64: dict of results and their bounds' parts."""
    s = q @ k.T * scale
    s = torch.where(mask, s, torch.full_like(s, float("-inf")))
    if k.shape[0] == 0:
        s = torch.full((q.shape[0], 1), float("-inf"), dtype=torch.float64)
        k, v, mask = torch.zeros_like(q[:1]), torch.zeros_like(q[:1]), s == 0
        if q.shape[0] == 0:
            k, v = torch.zeros(1, q.shape[1]).double(), torch.zeros(1, q.shape[1]).double()
    lse = torch.logsumexp(s, 1)
    p = torch.where(mask, torch.exp(s - lse[:, None]), torch.zeros_like(s))
    size = 1 + ((q.abs() @ k.abs().T).max() * abs(scale) if s.numel() else 0)
    r = {"out": p @ v, "lse": lse, "abs_out": p @ v.abs(), "size": size}
    if grad is not None:
        delta = (grad * r["out"]).sum(1, keepdim=True)
        rough = (grad.abs() * r["out"].abs()).sum(1, keepdim=True)
        dp = grad @ v.T
        ds = p * (dp - delta) * scale
        scale = abs(scale)
        # what 32-bit sums may cost, in units of their own roundoff
        sums = p * (grad.abs() @ v.abs().T + rough) * scale
        r |= {"q": ds @ k, "k": ds.T @ q, "v": p.T @ grad, "abs_v": p.T @ grad.abs(),
              "abs_q": ds.abs() @ k.abs(), "abs_k": ds.abs().T @ q.abs(),
              "rough_q": (p * rough * scale) @ k.abs(), "rough_k": (p * rough * scale).T @ q.abs(),
              "sums_q": sums @ k.abs(), "sums_k": sums.T @ q.abs(),
              "all_q": k.abs().sum(0, keepdim=True) * scale + 0 * q,
              "all_k": (mask.double().T @ q.abs()) * scale, "all_v": mask.double().T @ grad.abs()}
    return r


def packed(q, k, v, q_len, k_len, causal, window, scale, grad=None, small=1.0):
    """Every sequence and head: {name: (value, bound)} in float64 on the CPU, in q's type's bounds.
    ``small``: what the type's smallest steps may cost an operand, in units of tiny; a kernel that
    multiplies its weights by 2^n before it rounds them has 2^-n."""
    u, tiny = U[q.dtype], TINY[q.dtype]
    h, g = q.shape[1], k.shape[1]
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    grad = None if grad is None else grad.detach().cpu().double()
    res = {"out": (torch.zeros_like(q), torch.zeros_like(q)),
           "lse": (torch.zeros(q.shape[:2]).double(), torch.zeros(q.shape[:2]).double())}
    if grad is not None:
        res |= {"q": (torch.zeros_like(q), torch.zeros_like(q)),
                "k": (torch.zeros_like(k), torch.zeros_like(k)),
                "v": (torch.zeros_like(v), torch.zeros_like(v))}
    tq = tk = 0
    f = 2.0**-20
    for nq, nk in zip(q_len, k_len):
        mask = seen(nq, nk, causal, window)
        a, b = slice(tq, tq + nq), slice(tk, tk + nk)
        for x in range(h):
            y = x // (h // g)
            r = one(q[a, x], k[b, y], v[b, y], mask, scale, None if grad is None else grad[a, x])
            size = float(r["size"])
            res["out"][0][a, x], res["lse"][0][a, x] = r["out"], r["lse"]
            res["out"][1][a, x] = (u + f * size) * r["abs_out"] + u * r["out"].abs() + \
                tiny * (1 + small * v[b, y].abs().sum(0))
            res["lse"][1][a, x] = f * size
            if grad is None:
                continue
            res["q"][0][a, x] = r["q"]
            res["q"][1][a, x] = u * (r["q"].abs() + r["abs_q"] + r["rough_q"]) + \
                f * size * (r["abs_q"] + r["sums_q"]) + tiny * (1 + small * r["all_q"])
            if nk:
                # rounded once over the group: its own rounding is added below
                res["k"][0][b, y] += r["k"]
                res["v"][0][b, y] += r["v"]
                res["k"][1][b, y] += u * (r["abs_k"] + r["rough_k"]) + \
                    f * size * (r["abs_k"] + r["sums_k"]) + tiny * (1 + small * r["all_k"])
                res["v"][1][b, y] += (u + f * size) * r["abs_v"] + tiny * (1 + small * r["all_v"])
        tq, tk = tq + nq, tk + nk
    if grad is not None:
        for n in ("k", "v"):
            res[n] = (res[n][0], res[n][1] + u * res[n][0].abs())
    return res


def check(name, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    inf = torch.isinf(value)
    assert torch.equal(got[inf], value[inf]), f"{name}: infinities"
    off = ((got - value).abs() / (SLACK * bound + 1e-300))[~inf]
    assert not torch.isnan(got).any(), f"{name}: NaN"
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"
