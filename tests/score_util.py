"""64-bit definitions of the 8-bit products and the log-probability operators,
on the CPU and apart from the library."""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of f32


def quantize64(x):
    """(q int64, scale f32): both quotients rounded to f32, then halves to even."""
    x = x.detach().cpu().double()
    amax = x.abs().amax(1)
    bad = ~torch.isfinite(x).all(1)
    scale = (amax / 127).float()
    scale[bad] = math.nan
    ratio = (x / scale.double().unsqueeze(1)).float()
    q = torch.where((scale > 0).unsqueeze(1), ratio, torch.zeros_like(ratio))
    q = q.double().round().clamp(-127, 127)
    q[bad] = 0
    return q.long(), scale


def product(q, scale, wq, wscale, dtype):
    """f32(integer sum) * f32(scale * wscale), rounded to dtype: every rounding
    is part of the definition, so results are compared bit for bit."""
    acc = (q.double() @ wq.cpu().double().t()).float()  # exact below 2^53
    y = acc * (scale.cpu().unsqueeze(1) * wscale.cpu().unsqueeze(0))
    return y.to(dtype)


def logprobs64(logits, tokens, k):
    """The distribution of each row in 64 bits, and bounds of what f32 may be off.

    With d_i = x_i - M, p_i = e^d_i / Z, A1 = sum p|d| and A2 = sum p d^2: a term
    e^d is off by (1.25 |d| + 2) 2^-23 relative (the difference, its product with
    log2 e, the constant and 2 ulp of the exponential), a sum along at most L
    adds and rescalings by 2^-22 each; so log Z is off by
    z = 2^-23 (1.25 A1 + 4) + L 2^-22, and T/Z = sum p d by
    2^-23 (1.25 A2 + 4 A1) + L 2^-22 A1 + z A1."""
    x = logits.detach().cpu().double()
    T, V = x.shape
    L = max(8, -(-V // 32))  # no thread sums more than a warp's share of the row
    out = dict(logprobs=[], entropy=[], ids=[], top=[], tol_z=[], tol_h=[])
    for t in range(T):
        r = x[t]
        order = sorted(range(V), key=lambda i: (-r[i].item() if not math.isnan(r[i]) else math.inf,
                                                math.isnan(r[i]), i)) if V <= 4096 else None
        if order is None:
            key = torch.where(torch.isnan(r), -math.inf, r)
            order = torch.sort(key, descending=True, stable=True).indices[:k].tolist()
        ids = (order + [-1] * k)[:k]
        bad = bool(torch.isnan(r).any() or (r == math.inf).any())
        M = r.max()
        if bad:
            lp, H, z, h = torch.full_like(r, math.nan), math.nan, 0.0, 0.0
        elif M == -math.inf:
            lp, H, z, h = torch.full_like(r, -math.inf), 0.0, 0.0, 0.0
        else:
            d = r - M
            e = torch.exp(d)
            Z = e.sum()
            p, fin = e / Z, torch.where(torch.isinf(d), torch.zeros_like(d), d)
            lp = d - torch.log(Z)
            a1, a2 = (p * fin.abs()).sum().item(), (p * fin * fin).sum().item()
            H = (torch.log(Z) - (p * fin).sum()).item()
            z = 2.0 ** -23 * (1.25 * a1 + 4) + L * 2.0 ** -22
            h = z + 2.0 ** -23 * (1.25 * a2 + 4 * a1) + L * 2.0 ** -22 * a1 + z * a1
        g = []
        for tok in (tokens[t].tolist() if tokens is not None else []):
            g.append(0.0 if tok == -1 else math.nan if tok < 0 or tok >= V else lp[tok].item())
        out["logprobs"].append(g)
        out["entropy"].append(H)
        out["ids"].append(ids)
        out["top"].append([-math.inf if i < 0 and not bad else math.nan if bad else lp[i].item() for i in ids])
        out["tol_z"].append(z)
        out["tol_h"].append(h)
    return out


def check_logprobs(got, ref, what=""):
    """got: dict of tensors (logprobs, entropy, ids, top); ref: logprobs64's."""
    T = len(ref["entropy"])
    ids = got["ids"].cpu().tolist()
    for t in range(T):
        assert ids[t] == ref["ids"][t], (what, t, ids[t], ref["ids"][t])
        for name, tol in (("logprobs", ref["tol_z"][t]), ("top", ref["tol_z"][t])):
            for a, b in zip(got[name][t].tolist(), ref[name][t]):
                close(a, b, tol, (what, name, t))
        close(got["entropy"][t].item(), ref["entropy"][t], ref["tol_h"][t], (what, "entropy", t))


def close(a, b, tol, what):
    if math.isnan(b) or math.isinf(b):
        assert (math.isnan(a) and math.isnan(b)) or a == b, (what, a, b)
        return
    # the difference x - M, the subtraction of log Z and log itself round too
    assert abs(a - b) <= tol + 4 * EPS32 * (abs(b) + 1), (what, a, b, abs(a - b), tol)
