"""What is measured of the sequence operators (turboae_amd.sequence): their cases, their plain forms in elementary torch operations,
their definition in 64 bits, and what each has to read, write and compute.

The operators are one layer of a selective state-space sequence model and the reading of its answers: int8 products with per-token and
per-channel scales (the projections), the short causal convolution, the selective scan, the norms around the layer fused with its gate
and residual scale, and the log probabilities of given tokens.  Each has its form for prompts (or whole blocks of the code, the
framework's 500 blocks of 100 positions) and for single tokens.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda"


def listed():
    return [
        # one generated token for each of 64 sequences: the convolution's window of four, its last three inputs kept as state
        {"name": "conv_token", "op": "conv", "B": 64, "L": 1, "E": 4096, "K": 4, "dtype": "bf16", "state": True, "ragged": False},
        # four prompts of 2048 tokens; x is the left half of the input projection's output, so its rows are 2 E apart
        {"name": "conv_prompt", "op": "conv", "B": 4, "L": 2048, "E": 4096, "K": 4, "dtype": "bf16", "state": False, "ragged": False},
        # the same token's state update: bound by reading and writing the states
        {"name": "scan_token", "op": "scan", "B": 64, "L": 1, "E": 4096, "N": 16, "dtype": "bf16", "gate": True, "state": True, "ragged": False},
        # one long prompt: little to run side by side but the channels
        {"name": "scan_prompt", "op": "scan", "B": 1, "L": 4096, "E": 4096, "N": 16, "dtype": "bf16", "gate": True, "state": False, "ragged": False},
        # the framework's own batch: 500 blocks of at most 100 positions, twice its 100 units, in 32 bits, padded to the longest block
        {"name": "scan_blocks", "op": "scan", "B": 500, "L": 100, "E": 200, "N": 16, "dtype": "fp32", "gate": False, "state": False, "ragged": True},
        # 16 generated tokens: latency of one launch
        {"name": "norm_token", "op": "norm", "B": 16, "L": 1, "D": 2048, "dtype": "bf16", "residual": "bf16", "center": False, "gate": "token", "post": True, "pre": True},
        # four prompts of 2048 tokens, the residual stream kept in 32 bits
        {"name": "norm_prompt", "op": "norm", "B": 4, "L": 2048, "D": 4096, "dtype": "bf16", "residual": "fp32", "center": False, "gate": "token", "post": True, "pre": True},
        # the framework's batch at its 100 units: short rows, mean and deviation, one gate for each block
        {"name": "norm_blocks", "op": "norm", "B": 500, "L": 100, "D": 100, "dtype": "fp32", "residual": "fp32", "center": True, "gate": "sequence", "post": False, "pre": True},
        # four generated tokens through one projection: bound by reading the weights
        {"name": "int8_token", "op": "int8", "M": 4, "K": 4096, "N": 4096, "dtype": "bf16", "bias": False},
        # a prompt batch through the widest projection
        {"name": "int8_prompt", "op": "int8", "M": 8192, "K": 4096, "N": 8192, "dtype": "bf16", "bias": True},
        # the answers of one decoding step, with the alternatives a caller shows
        {"name": "logprobs_token", "op": "logprobs", "rows": 8, "V": 50001, "dtype": "fp32", "top": 20},
        # scoring given texts: 2048 positions over a large vocabulary
        {"name": "logprobs_prompt", "op": "logprobs", "rows": 2048, "V": 131072, "dtype": "bf16", "top": 8},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    while True:
        op = rng.choice(["conv", "scan", "scan", "norm", "int8", "int8", "logprobs"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        token = rng.random() < 0.3
        if op in ("conv", "scan"):
            c = {"op": op, "B": _log(rng, 1, 512), "L": 1 if token else _log(rng, 2, 8192), "E": _log(rng, 16, 8192)}
            if rng.random() < 0.5:
                c["E"] = max(16, c["E"] // 32 * 32)
            if op == "conv":
                c.update(K=rng.choice([2, 3, 4, 4, 5, 7]))
                cost, most = c["B"] * c["L"] * c["E"], 4 * 2048 * 4096
            else:
                c.update(N=rng.choice([1, 4, 8, 12, 16, 16, 32, 64]), gate=rng.random() < 0.6)
                cost, most = c["B"] * c["L"] * c["E"] * c["N"], 4096 * 4096 * 16
            c.update(dtype=dtype, state=token or rng.random() < 0.4, ragged=not token and rng.random() < 0.5)
        elif op == "norm":
            c = {"op": op, "B": _log(rng, 1, 512), "L": 1 if token else _log(rng, 2, 8192), "D": _log(rng, 32, 16384)}
            if rng.random() < 0.5:
                c["D"] = c["D"] // 32 * 32
            post, pre = rng.choice([(True, True), (True, False), (False, True)])
            c.update(dtype=dtype, residual=rng.choice([dtype, "fp32"]), center=rng.random() < 0.4, gate=rng.choice(["none", "token", "sequence"]), post=post, pre=pre)
            cost, most = c["B"] * c["L"] * c["D"], 4 * 2048 * 4096
        elif op == "int8":
            c = {"op": op, "M": _log(rng, 1, 32) if token else _log(rng, 33, 8192), "K": _log(rng, 32, 16384), "N": _log(rng, 32, 16384)}
            if rng.random() < 0.6:
                c["K"], c["N"] = c["K"] // 32 * 32, c["N"] // 32 * 32
            c.update(dtype=dtype, bias=rng.random() < 0.5)
            cost, most = c["M"] * c["K"] * c["N"], 8192 * 4096 * 8192
        else:
            c = {"op": op, "rows": _log(rng, 1, 32) if token else _log(rng, 33, 65536), "V": _log(rng, 2, 262144)}
            c.update(dtype=dtype, top=min(c["V"], rng.choice([0, 1, 5, 8, 20, 32])))
            cost, most = c["rows"] * c["V"] * SIZE[dtype] // 2, 2048 * 131072
        if cost <= most:
            return c


def _lengths(case, seed):
    """Lengths of a padded batch: every length from none to all of L as evenly as B allows, their order turned by the seed."""
    B, L = case["B"], case["L"]
    spread = [L - (i * 7919) % (L + 1) for i in range(B)]
    return [spread[(i + seed) % B] for i in range(B)]


def _valid(case):
    """Positions that are not padding."""
    return sum(_lengths(case, 0)) if case.get("ragged") else case["B"] * case["L"]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE)

    s = {"case": case}
    if case["op"] in ("conv", "scan"):
        B, L, E = case["B"], case["L"], case["E"]
        both = normal(B, L, 2 * E, dtype=dt)                      # the input projection's output: x and the gate z side by side
        s["x"] = both[:, :, :E]
        s["lengths"] = torch.tensor(_lengths(case, seed), dtype=torch.int32, device=DEVICE) if case["ragged"] else None
        if case["op"] == "conv":
            K = case["K"]
            s["weight"], s["bias"] = normal(E, K, std=K ** -0.5), normal(E, std=0.1)
            s["state"] = normal(B, K - 1, E, dtype=dt) if case["state"] else None
        else:
            N = case["N"]
            rank = -(-E // 16)
            low = normal(B, L, rank + 2 * N, dtype=dt)            # the second projection's output: low-rank steps, B and C
            s["Bm"], s["Cm"] = low[:, :, rank:rank + N], low[:, :, rank + N:]
            s["z"] = both[:, :, E:] if case["gate"] else None
            s["dt"] = normal(B, L, E, std=0.5, dtype=dt)
            s["A"] = -(torch.arange(1, N + 1, device=DEVICE, dtype=torch.float32) * torch.exp(normal(E, N, std=0.3)))
            step = torch.exp(uniform(E) * math.log(100.0) + math.log(1e-3))          # typical steps 0.001 .. 0.1
            s["dt_bias"] = step + torch.log(-torch.expm1(-step))                     # softplus(dt_bias) = step
            s["D"] = normal(E, std=0.5) + 1.0
            s["state"] = normal(B, E, N) if case["state"] else None
    elif case["op"] == "norm":
        B, L, D = case["B"], case["L"], case["D"]
        s["residual"] = normal(B, L, D, std=2.0, dtype=DTYPES[case["residual"]])
        s["block"] = normal(B, L, D, dtype=dt) + 0.25
        s["gate"] = {"none": None, "token": (B, L, D), "sequence": (B, 1, D)}[case["gate"]]
        s["gate"] = normal(*s["gate"], dtype=dt) if s["gate"] else None
        s["scale"] = normal(D, std=0.1) + 0.5
        s["post"] = normal(D, std=0.1) + 1.0 if case["post"] else None
        s["pre"] = normal(D, std=0.1) + 1.0 if case["pre"] else None
    elif case["op"] == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        outlier = 1.0 + 15.0 * (uniform(K) < 0.01).float()        # a few channels are far larger than the others, as activations have it
        s["x"] = (torch.randn(M, K, generator=g, device=DEVICE) * outlier).to(dt)
        rows = torch.zeros(N, -(-K // 64) * 64, dtype=torch.int8, device=DEVICE)     # rows on 64-byte boundaries, as a program lays its weights
        rows[:, :K] = torch.clamp(torch.round(torch.randn(N, K, generator=g, device=DEVICE) * 36.0), -127, 127).to(torch.int8)
        s["weight"] = rows[:, :K]
        s["weight_scale"] = (uniform(N) + 0.5) * (K ** -0.5 / 36.0)
        s["bias"] = normal(N) if case["bias"] else None
    else:
        R, V = case["rows"], case["V"]
        logits = normal(R, V, std=3.0)
        if V >= 64:                                               # tokens that a grammar forbids
            logits[:, torch.randint(0, V, (V // 64,), generator=g, device=DEVICE)] = -math.inf
        s["logits"] = logits.to(dt)
        s["tokens"] = torch.randint(0, V, (R,), generator=g, device=DEVICE)
    return s


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own_conv(s):
    from turboae_amd import sequence
    return sequence.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"], act="silu")


def _own_scan(s):
    from turboae_amd import sequence
    return sequence.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], lengths=s["lengths"])


def _own_norm(s):
    from turboae_amd import sequence
    residual, normed = sequence.norm_residual(s["residual"], s["block"], gate=s["gate"], scale=s["scale"], post_weight=s["post"], pre_weight=s["pre"],
                                              center=s["case"]["center"], eps=1e-5)
    return (residual,) if normed is None else (residual, normed)


def _own_int8(s):
    from turboae_amd import sequence
    return sequence.int8_linear(s["x"], s["weight"], s["weight_scale"], s["bias"])


def _own_logprobs(s):
    from turboae_amd import sequence
    logp, entropy, ids, top = sequence.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return (logp, entropy, ids, top) if s["case"]["top"] else (logp, entropy)


_own = {"conv": _own_conv, "scan": _own_scan, "norm": _own_norm, "int8": _own_int8, "logprobs": _own_logprobs}


# ------------------------------------------------------------------------------------------------ their plain forms, in 32 bits
def _plain_conv(s):
    x, w = s["x"], s["weight"]
    B, L, E = x.shape
    K = w.shape[1]
    before = s["state"] if s["state"] is not None else x.new_zeros(B, K - 1, E)
    padded = torch.cat([before, x], dim=1)
    y = (padded.unfold(1, K, 1).float() * w).sum(-1) + s["bias"]
    y = y * torch.sigmoid(y)
    if s["lengths"] is None:
        return y.to(x.dtype), padded[:, L:].contiguous()
    n = s["lengths"].long()[:, None]
    y = torch.where((torch.arange(L, device=x.device) < n)[:, :, None], y, 0.0)
    last = (n + torch.arange(K - 1, device=x.device))[:, :, None].expand(B, K - 1, E)
    return y.to(x.dtype), padded.gather(1, last)


def _plain_scan(s):
    x = s["x"].float()
    B, L, E = x.shape
    d = s["dt"].float() + s["dt_bias"]
    d = torch.where(d > 20.0, d, torch.log1p(torch.exp(d)))
    valid = None
    if s["lengths"] is not None:
        valid = (torch.arange(L, device=x.device) < s["lengths"][:, None])[:, :, None]
        d = torch.where(valid, d, 0.0)                            # a step of zero keeps the state
    a = torch.exp(d[..., None] * s["A"])
    h = (d * x)[..., None] * s["Bm"].float()[:, :, None, :]
    if s["state"] is not None:
        h[:, 0] += a[:, 0] * s["state"]
    reach = 1                                                     # every pass doubles how far back a position's sum reaches
    while reach < L:
        h = torch.cat([h[:, :reach], h[:, reach:] + a[:, reach:] * h[:, :-reach]], dim=1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], dim=1)
        reach *= 2
    y = (h * s["Cm"].float()[:, :, None, :]).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    return y.to(s["x"].dtype), h[:, -1].contiguous()


def _norm(v, weight, center, eps):
    if center:
        v = v - v.mean(-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight


def _plain_norm(s):
    center = s["case"]["center"]
    p = s["block"].float()
    if s["post"] is not None:
        p = _norm(p, s["post"], center, 1e-5)
    p = p * s["scale"]
    if s["gate"] is not None:
        p = p * torch.sigmoid(s["gate"].float())
    r = s["residual"].float() + p
    if s["pre"] is None:
        return (r.to(s["residual"].dtype),)
    return r.to(s["residual"].dtype), _norm(r, s["pre"], center, 1e-5).to(s["block"].dtype)


def _plain_int8(s):
    x = s["x"].float()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(most > 0, most, 1.0))
    y = (q @ s["weight"].float().t()) * ((most / 127.0) * s["weight_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    R, V = x.shape
    most = x.amax(-1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(-1, keepdim=True)
    lp = x - most - torch.log(total)
    logp = lp.gather(1, s["tokens"][:, None])[:, 0]
    entropy = -(torch.where(e > 0, lp, 0.0) * (e / total)).sum(-1)
    top = s["case"]["top"]
    if not top:
        return logp, entropy
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))    # whole numbers in the order of the values
    key = order * V + torch.arange(V - 1, -1, -1, device=x.device)                   # of equal values the lowest index first
    ids = V - 1 - torch.remainder(key.topk(top, -1).values, V)
    return logp, entropy, ids, lp.gather(1, ids)


_plain = {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm, "int8": _plain_int8, "logprobs": _plain_logprobs}


# ------------------------------------------------------------------------------------------------ their definitions, in 64 bits
def _exact_conv(s):
    x, w = s["x"].double(), s["weight"].double()
    B, L, E = x.shape
    K = w.shape[1]
    n = s["lengths"].tolist() if s["lengths"] is not None else [L] * B
    y = torch.zeros(B, L, E, dtype=torch.float64, device=x.device)
    state = torch.zeros(B, K - 1, E, dtype=torch.float64, device=x.device)
    for b in range(B):
        before = s["state"][b].double() if s["state"] is not None else state[b]
        seen = torch.cat([before, x[b, :n[b]]])
        out = s["bias"].double().expand(n[b], E).clone()
        for k in range(K):
            out += seen[k:k + n[b]] * w[:, k]
        y[b, :n[b]] = torch.nn.functional.silu(out)
        state[b] = seen[n[b]:]
    return y, state


def _exact_scan(s):
    x, A = s["x"].double(), s["A"].double()
    B, L, E = x.shape
    step = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=1e9)
    h = s["state"].double().clone() if s["state"] is not None else torch.zeros(B, E, A.shape[1], dtype=torch.float64, device=x.device)
    y = torch.zeros(B, L, E, dtype=torch.float64, device=x.device)
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=x.device)
    for t in range(L):
        d = step[:, t, :, None]
        new = torch.exp(d * A) * h + d * x[:, t, :, None] * s["Bm"][:, t].double()[:, None, :]
        on = (t < n)[:, None, None]
        h = torch.where(on, new, h)
        out = (h * s["Cm"][:, t].double()[:, None, :]).sum(-1) + s["D"].double() * x[:, t]
        if s["z"] is not None:
            out = out * torch.nn.functional.silu(s["z"][:, t].double())
        y[:, t] = torch.where(on[:, :, 0], out, 0.0)
    return y, h


def _exact_norm(s):
    center = s["case"]["center"]

    def norm(v, weight):
        mean = v.mean(-1, keepdim=True) if center else torch.zeros_like(v[..., :1])
        return (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + 1e-5) * weight.double()

    p = s["block"].double()
    p = norm(p, s["post"]) if s["post"] is not None else p
    g = 1.0 / (1.0 + torch.exp(-s["gate"].double())) if s["gate"] is not None else 1.0
    r = s["residual"].double() + s["scale"].double() * g * p
    return (r,) if s["pre"] is None else (r, norm(r, s["pre"]))


def _exact_int8(s):
    x = s["x"].double()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(most > 0, most, 1.0))
    y = torch.mm(q, s["weight"].double().t().contiguous()) * most / 127.0 * s["weight_scale"].double()
    return y + s["bias"].double() if s["bias"] is not None else y


def _exact_logprobs(s):
    top, got = s["case"]["top"], []
    for x, token in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = x.double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        got.append([lp.gather(1, token[:, None])[:, 0], torch.special.entr(torch.exp(lp)).sum(-1)])
        if top:
            values, ids = torch.sort(lp, dim=-1, descending=True, stable=True)
            got[-1] += [ids[:, :top], values[:, :top]]
    return tuple(torch.cat(v) for v in zip(*got))


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm, "int8": _exact_int8, "logprobs": _exact_logprobs}[case["op"]](s)


# ------------------------------------------------------------------------------------------------ what each cannot do without
def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "conv":
        B, L, E, K, n = case["B"], case["L"], case["E"], case["K"], _valid(case)
        states = B * (K - 1) * E * b * (2 if case["state"] else 1)
        return {"bytes": (n + B * L) * E * b + E * (K + 1) * 4 + states, "flops": (2 * K + 4) * n * E}
    if case["op"] == "scan":
        B, L, E, N, n = case["B"], case["L"], case["E"], case["N"], _valid(case)
        states = B * E * N * 4 * (2 if case["state"] else 1)
        reads = n * E * b * (3 if case["gate"] else 2) + 2 * n * N * b + E * (N + 2) * 4
        return {"bytes": reads + B * L * E * b + states, "flops": 7 * n * E * N + 12 * n * E}
    if case["op"] == "norm":
        n, D, r = case["B"] * case["L"], case["D"], SIZE[case["residual"]]
        gate = {"none": 0, "token": n, "sequence": case["B"]}[case["gate"]] * D * b
        return {"bytes": n * D * (b + 2 * r + (b if case["pre"] else 0)) + gate + D * 4 * (1 + case["post"] + case["pre"]), "flops": n * D * (4 + 4 * case["post"] + 4 * case["pre"])}
    if case["op"] == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * b + N * K + M * N * b + N * 4 * (1 + case["bias"]), "flops": 2 * M * K * N}
    R, V, top = case["rows"], case["V"], case["top"]
    return {"bytes": R * V * b + R * (8 + 8 + 12 * top), "flops": 5 * R * V}
