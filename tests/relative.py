"""The biased attention and layer norm in 64 bits on the CPU, with their gradients and how far an f32
computation that rounds to the operators' types may be from them. Plain formulas over whole matrices."""

import math

import torch

# The largest rounding error of a type, relative to the value: half a step.
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def attention(q, k, v, scale=0.125, cap=0.0, table=None, bucket=None, reach=0, slopes=None, window=0,
              span=None, q_first=0, dout=None):
    """q [nq][heads][64], k and v [nk][kv_heads][64]. A dict of o, lse, with dout dq, dk, dv, dtable, and
    for each x its bound's parts: x_sum, the sum of the terms' magnitudes that x is made of."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    (nq, heads, _), (nk, kv) = q.shape, k.shape[:2]
    each = heads // kv
    pos, j = q_first + torch.arange(nq), torch.arange(nk)
    t = j[None] - pos[:, None]
    ok = torch.ones(nq, nk, dtype=torch.bool)
    if span is not None:
        s = span.long().cpu()
        ok &= (j[None] >= s[:, :1]) & (j[None] < s[:, 1:])
    if window:
        ok &= t.abs() <= window
    out = {"o": torch.zeros_like(q), "lse": torch.empty(heads, nq, dtype=torch.float64)}
    out["o_sum"] = torch.zeros_like(q)
    most = 0.0
    if dout is not None:
        dout = dout.double().cpu()
        for x, y in (("dq", q), ("dk", k), ("dv", v)):
            out[x], out[x + "_sum"] = torch.zeros_like(y), torch.zeros_like(y)
        if table is not None:
            out["dtable"] = torch.zeros(table.shape, dtype=torch.float64)
            out["dtable_sum"] = torch.zeros(table.shape, dtype=torch.float64)
    if table is not None:
        which = bucket.long().cpu()[t.clamp(-reach, reach) + reach].clamp(0, table.shape[0] - 1)
    for h in range(heads):
        g = h // each
        a = scale * (q[:, h] @ k[:, g].T)
        slope = torch.ones_like(a)
        if cap:
            x = torch.tanh(a / cap)
            a, slope = cap * x, 1.0 - x * x
        if table is not None:
            a = a + table.double().cpu()[which, h]
        if slopes is not None:
            a = a - slopes.double().cpu()[h] * t.abs()
        a = torch.where(ok, a, -math.inf)
        top = a.amax(1, keepdim=True) if nk else torch.full((nq, 1), -math.inf, dtype=torch.float64)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(a - top)
        total = p.sum(1, keepdim=True)
        out["lse"][h] = (top + torch.log(total))[:, 0]
        p = torch.where(total > 0, p / torch.where(total > 0, total, 1.0), 0.0)
        # a masked pair takes no part, whatever v holds there
        vis = torch.where(ok.any(0)[:, None], v[:, g], 0.0)
        out["o"][:, h], out["o_sum"][:, h] = p @ vis, p @ vis.abs()
        seen = a[torch.isfinite(a)]
        most = max(most, float(seen.abs().max()) if seen.numel() else 0.0)
        if dout is None:
            continue
        d = dout[:, h]
        dp = torch.where(ok, d @ v[:, g].T, 0.0)
        big = torch.where(ok, d.abs() @ v[:, g].abs().T, 0.0)
        row = (d * out["o"][:, h]).sum(1, keepdim=True)
        ds = p * (dp - row)
        mag = p * (big + (d.abs() * out["o_sum"][:, h]).sum(1, keepdim=True))
        out["dv"][:, g] += p.T @ d
        out["dv_sum"][:, g] += p.T @ d.abs()
        if table is not None:
            out["dtable"][:, h].index_add_(0, which.flatten(), ds.flatten())
            out["dtable_sum"][:, h].index_add_(0, which.flatten(), mag.flatten())
        da = scale * slope * ds
        out["dq"][:, h] = da @ k[:, g]
        out["dk"][:, g] += da.T @ q[:, h]
        # `mag` bounds |dS| and stands for what rounding each factor of it costs
        out["dq_sum"][:, h] = scale * (mag @ k[:, g].abs())
        out["dk_sum"][:, g] += scale * (mag.T @ q[:, h].abs())
    out["most"] = most
    return out


def attention_bounds(ref, type, cap=0.0):
    """How far each output may be off, elementwise. A score is off by a few f32 roundings of its 64
    products and of its largest parts (the cap's tanh by some of its `cap`): 2^-20 (4 + most + cap)
    and with it the weight, relatively; weights and dS are rounded to the type before the products
    (u), sums are f32 (2^-18 of the terms' magnitudes for up to some thousands), and the result is
    rounded once. dS takes dO . o, whose o was rounded and came from rounded weights: 2 u of its terms."""
    u, w = U[type], 2.0 ** -20 * (4.0 + ref["most"] + cap) + 2.0 ** -18
    tiny = 2.0 ** -24 if type == "f16" else 1e-30  # (f16: results below its normal values)
    out = {"o": (u + w) * ref["o_sum"] + u * ref["o"].abs() + tiny,
           "lse": torch.full_like(ref["lse"], w)}
    for x in ("dq", "dk", "dv"):
        if x in ref:
            out[x] = ((u if x == "dv" else 3 * u) + 2 * w) * ref[x + "_sum"] + u * ref[x].abs() + tiny
    if "dtable" in ref:
        out["dtable"] = (2 * u + 2 * w) * ref["dtable_sum"] + 1e-30
    return out


def norm(x, gamma, beta, eps, dy=None):
    x, gamma = x.double().cpu(), gamma.double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    xh = (x - mean) * rstd
    out = {"y": xh * gamma + (0.0 if beta is None else beta.double().cpu()), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    out["xh"] = xh
    if dy is not None:
        dy = dy.double().cpu()
        g = dy * gamma
        out["dx"] = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out["dx_sum"] = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
        out["dgamma"], out["dgamma_sum"] = (dy * xh).sum(0), (dy * xh).abs().sum(0)
        out["dbeta"], out["dbeta_sum"] = dy.sum(0), dy.abs().sum(0)
    return out


def worst(got, want, bound):
    """The largest error in units of the bound (infinite where one is finite and the other is not, or
    they are different infinities)."""
    got, want = got.double().cpu(), want.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs() / bound)
    off = torch.where(torch.isfinite(want) | same, off, math.inf)
    off = torch.where(torch.isnan(off), math.inf, off)
    return float(off.max()) if off.numel() else 0.0
