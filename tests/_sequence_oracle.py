"""Plain 64-bit implementations of the sequence operators (include/turboae_hip.h states their formulas) and the bounds of what the
library's 32-bit arithmetic may be off by.

Every bound counts roundings.  U = 2^-24 is half a step of fp32 relative to a value; a result of type t adds ``finfo(t).eps / 2``.  The
counts behind the constants: v_exp_f32 / v_log_f32 / v_rcp_f32 are good to one step (2 U), a product inside an exponent costs U times the
exponent, a sum of n terms at most n U of the sum of magnitudes.
"""
import torch

U = 2.0 ** -24


def rounding(dtype, value):
    """What storing `value` in this type may be off by: half a step, eps / 2 relative to it; below the smallest normal number (2^-14 in
    fp16) steps no longer shrink, so there it is eps / 2 of that number (2^-25 in fp16)."""
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs().clamp(min=f.tiny)


def silu(v):
    return v * torch.sigmoid(v)


def conv(x, weight, bias, state, lengths, act):
    """-> y, state, bound of y"""
    B, L, E = x.shape
    K = weight.shape[1]
    xs, w = x.double(), weight.double()
    y, new = torch.zeros(B, L, E, dtype=torch.float64), torch.zeros(B, K - 1, E, dtype=torch.float64)
    bound = torch.zeros_like(y)
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        seen = torch.cat([torch.zeros(K - 1, E, dtype=torch.float64) if state is None else state[b].double(), xs[b, :n]])
        pre = torch.zeros(n, E, dtype=torch.float64) + (0.0 if bias is None else bias.double())
        size = pre.abs()
        for k in range(K):
            pre = pre + w[:, k] * seen[k:k + n]
            size = size + (w[:, k] * seen[k:k + n]).abs()
        out = silu(pre) if act == "silu" else pre
        y[b, :n] = out
        # K + 1 roundings of the sum (a slope of silu is below 1.1); silu itself: 8 U, and |pre| U from its exponent
        bound[b, :n] = U * (1.1 * (K + 1) * size + (8 + pre.abs()) * out.abs()) + rounding(x.dtype, out) + 1e-30
        new[b] = seen[n:]
    return y, new, bound


def scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, lengths):
    """-> y, state, bound of y, bound of the state.  The same recurrence over magnitudes carries the bounds: a product of decays
    exp(-X) is off by X U a few times over (X below 87 where it is not 0), a step by 10 U (softplus), each position adds 4 roundings."""
    Bt, L, E = x.shape
    N = A.shape[1]
    h = torch.zeros(Bt, E, N, dtype=torch.float64) if state is None else state.double().clone()
    mag = h.abs()
    y, by = torch.zeros(Bt, L, E, dtype=torch.float64), torch.zeros(Bt, L, E, dtype=torch.float64)
    count = 4 * L + 1000
    for b in range(Bt):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for t in range(n):
            d = dt[b, t].double() + (0.0 if dt_bias is None else dt_bias.double())
            if softplus:
                d = torch.nn.functional.softplus(d, threshold=1e9)
            a = torch.exp(d[:, None] * A.double())
            u = (d * x[b, t].double())[:, None] * B[b, t].double()
            h[b], mag[b] = a * h[b] + u, a * mag[b] + u.abs()
            out = (h[b] * C[b, t].double()).sum(-1)
            size = (mag[b] * C[b, t].double().abs()).sum(-1)
            if D is not None:
                out, size = out + D.double() * x[b, t].double(), size + (D.double() * x[b, t].double()).abs()
            if z is not None:
                g = silu(z[b, t].double())
                out, size = out * g, size * g.abs() * (1 + (z[b, t].double().abs()) / count)
            y[b, t] = out
            by[b, t] = U * (count + N + 16) * size + rounding(x.dtype, out) + 1e-30
    return y, h, by, U * count * mag + 1e-30


def norm(v, weight, bias, center, eps):
    mean = v.mean(-1, keepdim=True) if center else torch.zeros_like(v[..., :1])
    rstd = 1.0 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    out = (v - mean) * rstd * weight.double()
    return (out if bias is None else out + bias.double()), rstd, v.abs().mean(-1, keepdim=True) if center else torch.zeros_like(mean)


def gate(g, act):
    return {"linear": lambda v: v, "tanh": torch.tanh, "sigmoid": torch.sigmoid, "silu": silu}[act](g)


def norm_residual(residual, block, g, scale, post_w, post_b, pre_w, pre_b, center, gate_act, alpha, eps, dtype):
    """-> r, normed, bound of r, bound of normed.  Sums of a row are taken in at most 32 + 10 steps of a tree (42 U); 64 U covers them with
    the products around them.  A gate is off by 8 U (tanh: 8 U of 1) and |g| U from its exponent."""
    r = residual.double()
    size = r.abs()
    if block is not None:
        p = block.double()
        err = torch.zeros_like(p)
        if post_w is not None:
            v = p
            p, rstd, mean = norm(v, post_w, post_b, center, eps)
            err = 64 * U * (rstd * post_w.double().abs() * (v.abs() + mean) + p.abs())
        f = torch.full_like(p, alpha)
        if scale is not None:
            f = f * scale.double()
        if g is not None:
            gv = gate(g.double(), gate_act)
            slack = (8 + g.double().abs()) * U * (gv.abs() + (1.0 if gate_act == "tanh" else 0.0))
            err = err * gv.abs() + p.abs() * slack
            p = p * gv
        r = r + f * p
        size = size + (f * p).abs()
        er = f.abs() * err + 8 * U * size
    else:
        er = torch.zeros_like(r)
    br = er + rounding(residual.dtype, r) + 1e-30
    if pre_w is None:
        return r, None, br, None
    n, rstd, mean = norm(r, pre_w, pre_b, center, eps)
    w = pre_w.double().abs()
    # an error of r moves the row's mean and deviation too: by at most its root mean square
    em = er + er.pow(2).mean(-1, keepdim=True).sqrt() * (1.0 + (r.abs() + mean) * rstd)
    return r, n, br, w * rstd * (em + 64 * U * (r.abs() + mean)) + 64 * U * n.abs() + rounding(dtype, n) + 1e-30


def quantize(x):
    """The definition's own 32-bit steps: 127 x, then a division; halves to even.  -> q (float64), scale (float32)"""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(most > 0, most, torch.ones_like(most)))
    return q.double(), (most / 127.0)[..., 0]


def int8_linear(x, weight, weight_scale, bias):
    """-> y, bound: the sum is exact, its conversion, the two scales, their product and the bias are 6 roundings"""
    q, s = quantize(x)
    y = (q @ weight.double().t()) * (s.double()[:, None] * weight_scale.double())
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, U * 6 * size + rounding(x.dtype, y) + 1e-30


def logprobs(logits, tokens, top):
    """-> logp, entropy, ids, top_logp, bound of a log probability of logit x, bound of the entropy.  Terms e^(x - m) are off by |x - m| U and
    two steps, of which what counts is |x - m| e^(x - m) < 0.4 of the largest; 64 of them are summed in a row before trees join them."""
    x = logits.double()
    V = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    none = torch.isnan(x).any(-1) | (m[..., 0] == float("inf"))
    empty = m[..., 0] == float("-inf")
    total = torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    lp = x - m - total                                          # not x - (m + total): next to the type's lowest value the sum would lose the total
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    safe = tokens.long().clamp(0, V - 1)
    logp = lp.gather(-1, safe[..., None])[..., 0]
    logp = torch.where(empty, torch.full_like(logp, float("-inf")), logp)
    nan = torch.full_like(logp, float("nan"))
    logp = torch.where(tokens < 0, torch.zeros_like(logp), logp)
    entropy = torch.where(empty, torch.zeros_like(entropy), entropy)
    logp = torch.where(none | (tokens >= V), nan, logp)
    entropy = torch.where(none, nan, entropy)
    order = torch.sort(torch.where(torch.isnan(x), torch.zeros_like(x), x), dim=-1, descending=True, stable=True).indices[..., :top]
    top_logp = torch.where(empty[..., None], torch.full_like(lp[..., :top], float("-inf")), lp.gather(-1, order))
    ids = torch.where(none[..., None], torch.full_like(order, -1), order)
    top_logp = torch.where(none[..., None], torch.full_like(top_logp, float("nan")), top_logp)
    scale = torch.where(torch.isfinite(m), m.abs(), torch.zeros_like(m)) + torch.nan_to_num(total.abs(), posinf=0.0)

    def bound(v):
        return U * (300 + 4 * torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)) + 4 * scale)

    return logp, entropy, ids, top_logp, bound, (U * (600 + 8 * scale[..., 0]) * (1 + torch.nan_to_num(entropy)))
