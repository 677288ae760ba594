"""The sequence operators (turboae_amd.sequence) against plain 64-bit implementations, at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

from tests import _sequence_oracle as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def inside(got, want, bound, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = (got - want).abs()[fine] - bound.expand_as(want)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0.0, (what, float(over.max()), float((got - want).abs()[fine].max()))


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def wide(t, dev, left=0, right=0):
    """The same values as a slice of a wider tensor whose other columns are NaN."""
    w = torch.full((*t.shape[:-1], left + t.shape[-1] + right), NAN, dtype=t.dtype, device=dev)
    w[..., left:left + t.shape[-1]] = t.to(dev)
    return w[..., left:left + t.shape[-1]]


# ---------------------------------------------------------------------------------------------------------------- causal_conv
CONV = [(dt, *shape) for dt in DT for shape in ((1, 1, 64, 4), (3, 1, 130, 4), (2, 5, 33, 3), (2, 16, 8, 8), (1, 17, 257, 2), (2, 100, 200, 5), (3, 47, 24, 1), (1, 33, 4096, 4))]


@pytest.mark.parametrize("dt,B,L,E,K", CONV)
@pytest.mark.parametrize("ragged", [False, True])
def test_causal_conv(gpu_device, dt, B, L, E, K, ragged):
    from turboae_amd import sequence
    g, t = gen(B * 7 + L * 3 + E + K), DT[dt]
    x, w, b = rnd(g, B, L, E, dtype=t), rnd(g, E, K), rnd(g, E)
    state = rnd(g, B, K - 1, E, dtype=t) if ragged else None
    lengths = torch.tensor([0, L, L // 2][:B] if B > 1 else [L // 2], dtype=torch.int32) if ragged else None
    act, bias = ("silu", b) if L % 2 else ("linear", None)
    y, s, bound = O.conv(x, w, bias, state, lengths, act)
    xd = wide(x, gpu_device, 0, E) if L % 3 else x.to(gpu_device)
    if ragged:
        for i in range(B):
            xd[i, int(lengths[i]):] = NAN                       # padding is not read
    got, new = sequence.causal_conv(xd, *on(gpu_device, w, bias, state, lengths), act=act)
    inside(got, y, bound, "y")
    assert torch.equal(new.cpu().double(), s)


def test_causal_conv_continues_from_its_state(gpu_device):
    """Whole = pieces = single tokens, with the state updated in place; results are the same to the bit."""
    from turboae_amd import sequence
    g = gen(1)
    x, w, b = on(gpu_device, rnd(g, 2, 50, 96, dtype=torch.bfloat16), rnd(g, 96, 4), rnd(g, 96))
    whole, last = sequence.causal_conv(x, w, b)
    state = torch.zeros(2, 3, 96, dtype=torch.bfloat16, device=gpu_device)
    parts = []
    for lo, hi in ((0, 1), (1, 3), (3, 20), (20, 21), (21, 50)):
        y, out = sequence.causal_conv(x[:, lo:hi], w, b, state=state, state_out=state)
        assert out is state
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, last)


# ---------------------------------------------------------------------------------------------------------------- selective_scan
def scan_case(seed, dt, B, L, E, N, gate, start, lengths):
    g, t = gen(seed), DT[dt]
    c = dict(x=rnd(g, B, L, E, dtype=t), dt=rnd(g, B, L, E, std=0.7, dtype=t), A=-(1 + torch.rand(E, N, generator=g) * N), B=rnd(g, B, L, N, dtype=t), C=rnd(g, B, L, N, dtype=t),
             D=rnd(g, E) if gate else None, z=rnd(g, B, L, E, std=2.0, dtype=t) if gate else None, dt_bias=rnd(g, E) - 2.0, softplus=True,
             state=rnd(g, B, E, N) if start else None, lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32))
    return c


def run_scan(c, dev, strided=True, **more):
    from turboae_amd import sequence
    E, N = c["A"].shape
    k = {n: (v.to(dev) if isinstance(v, torch.Tensor) else v) for n, v in c.items()}
    if strided:
        k["x"], k["B"], k["C"] = wide(c["x"], dev, 0, E), wide(c["B"], dev, 3, N), wide(c["C"], dev, 3 + N, 0)
        if c["z"] is not None:
            k["z"] = wide(c["z"], dev, E, 0)
    if c["lengths"] is not None:
        for i, n in enumerate(c["lengths"].tolist()):
            for name in ("x", "dt", "B", "C", "z"):
                if k[name] is not None:
                    k[name][i, max(n, 0):] = NAN
    return sequence.selective_scan(**k, **more)


SCAN = [("bf16", 2, 1, 96, 16, True, True, None), ("f32", 3, 1, 33, 5, False, True, None), ("f16", 1, 1, 4096, 16, True, False, None), ("f32", 2, 7, 20, 1, True, False, None),
        ("f32", 1, 32, 64, 16, False, False, None), ("bf16", 2, 33, 65, 16, True, True, None), ("f16", 3, 100, 40, 8, True, True, [100, 0, 61]),
        ("f32", 4, 65, 17, 12, False, True, [1, 64, 65, -3]), ("bf16", 2, 129, 31, 64, True, False, [129, 1000]), ("f32", 1, 300, 9, 33, True, True, None),
        ("f32", 1, 1000, 24, 16, True, True, None), ("bf16", 2, 515, 48, 4, True, True, [515, 130]), ("f32", 2, 700, 16, 16, False, True, [0, 257])]


@pytest.mark.parametrize("dt,B,L,E,N,gate,start,lengths", SCAN)
@pytest.mark.parametrize("strided", [False, True])
def test_selective_scan(gpu_device, dt, B, L, E, N, gate, start, lengths, strided):
    c = scan_case(L * 31 + E, dt, B, L, E, N, gate, start, lengths)
    y, h, by, bh = O.scan(**c)
    got, state = run_scan(c, gpu_device, strided)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


def test_selective_scan_without_softplus_and_with_extreme_steps(gpu_device):
    c = scan_case(5, "f32", 2, 40, 12, 16, True, True, None)
    c["softplus"], c["dt_bias"] = False, None
    c["dt"] = c["dt"].abs()
    c["dt"][0, ::3] = 0.0                                   # keeps the state
    c["dt"][1, ::5] = 200.0                                 # forgets all of it
    y, h, by, bh = O.scan(**c)
    got, state = run_scan(c, gpu_device)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")
    c = scan_case(6, "bf16", 1, 33, 12, 16, True, False, None)
    c["dt"][0, ::4], c["dt"][0, 1::4], c["z"][0, ::3], c["z"][0, 1::3] = 60.0, -60.0, -120.0, 300.0
    y, h, by, bh = O.scan(**c)
    got, state = run_scan(c, gpu_device)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


@pytest.mark.parametrize("E,L", [(24, 1000), (200, 150)])
def test_selective_scan_continues_from_its_state_in_place(gpu_device, E, L):
    from turboae_amd import sequence
    c = scan_case(7, "f32", 2, L, E, 16, True, True, None)
    y, h, by, bh = O.scan(**c)
    k = {n: (v.to(gpu_device) if isinstance(v, torch.Tensor) else v) for n, v in c.items()}
    state, parts = k.pop("state"), []
    for lo, hi in ((0, 1), (1, 2), (2, L // 2), (L // 2, L)):
        piece = {n: (v[:, lo:hi] if n in ("x", "dt", "B", "C", "z") else v) for n, v in k.items()}
        out, same = sequence.selective_scan(**piece, state=state, state_out=state)
        assert same is state
        parts.append(out)
    inside(torch.cat(parts, 1), y, by, "y")
    inside(state, h, bh, "state")


def test_selective_scan_is_the_same_every_time(gpu_device):
    c = scan_case(8, "bf16", 1, 2048, 64, 16, True, True, None)
    first = run_scan(c, gpu_device)
    for _ in range(3):
        again = run_scan(c, gpu_device)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---------------------------------------------------------------------------------------------------------------- norm_residual
NORM = [(dt, res, *shape) for dt, res in (("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32"))
        for shape in ((2, 3, 64), (1, 1, 1), (3, 2, 100), (2, 5, 33), (1, 2, 513), (2, 1, 1000), (1, 3, 2048), (1, 2, 4100), (1, 2, 8192), (1, 1, 16384), (1, 2, 32767))]


@pytest.mark.parametrize("dt,res,B,L,D", NORM)
@pytest.mark.parametrize("form", ["post pre token", "center post pre biases sequence tanh", "pre", "gate only silu", "linear gate pre", "no block"])
def test_norm_residual(gpu_device, dt, res, B, L, D, form):
    from turboae_amd import sequence
    g, t, r = gen(D + B), DT[dt], DT[res]
    words = form.split()
    residual, block = rnd(g, B, L, D, std=2.0, dtype=r), rnd(g, B, L, D, dtype=t) + 1.5
    gate = rnd(g, B, 1 if "sequence" in words else L, D, std=2.0, dtype=t) if any(w in words for w in ("token", "sequence", "gate")) else None
    act = next((w for w in words if w in ("tanh", "silu", "linear")), "sigmoid")
    post = (rnd(g, D, std=0.3) + 1.0) if "post" in words else None
    pre = (rnd(g, D, std=0.3) + 1.0) if "pre" in words or form == "no block" else None
    pb, qb = (rnd(g, D), rnd(g, D)) if "biases" in words else (None, None)
    scale = rnd(g, D) if "post" in words else None
    if form == "no block":
        block = None
    center, alpha = "center" in words, 0.5 if "sequence" in words else 1.0
    want = O.norm_residual(residual, block, gate, scale, post, pb, pre, qb, center, act, alpha, 1e-5, t)
    rd, bd, gd = residual.to(gpu_device), None if block is None else wide(block, gpu_device, 0, D), None if gate is None else wide(gate, gpu_device, D, 0)
    got, normed = sequence.norm_residual(rd, bd, gd, *on(gpu_device, scale, post, pb, pre, qb), center=center, gate_act=act, alpha=alpha, eps=1e-5, dtype=t if block is None else None)
    inside(got, want[0], want[2], "residual")
    if pre is None:
        assert normed is None
    else:
        assert normed.dtype == t
        inside(normed, want[1], want[3], "normed")
    if block is not None:                                   # in place, to the bit the same
        again, n2 = sequence.norm_residual(rd, bd, gd, *on(gpu_device, scale, post, pb, pre, qb), center=center, gate_act=act, alpha=alpha, eps=1e-5, residual_out=rd)
        assert again is rd and torch.equal(rd, got) and (normed is None or torch.equal(n2, normed))


def test_norm_residual_of_rows_without_variance(gpu_device):
    """Zero rows and constant rows stay finite; a row with NaN touches no other."""
    from turboae_amd import sequence
    x = torch.zeros(1, 4, 256)
    x[0, 1] = 1e4
    x[0, 2, 7] = NAN
    x[0, 3] = torch.arange(256.0)
    w = torch.ones(256)
    for center in (False, True):
        want = O.norm_residual(x[:, [0, 1, 3]], None, None, None, None, None, w, None, center, "sigmoid", 1.0, 1e-5, torch.float32)
        got = sequence.norm_residual(x.to(gpu_device), pre_weight=w.to(gpu_device), center=center)[1]
        inside(got[:, [0, 1, 3]], want[1], want[3], "normed")
        assert bool(torch.isnan(got[0, 2]).all())


# ---------------------------------------------------------------------------------------------------------------- int8
INT8 = [(dt, *shape) for dt in DT for shape in ((1, 16, 16), (1, 1, 1), (4, 256, 100), (3, 77, 5), (16, 1000, 33), (17, 64, 64), (33, 63, 130), (64, 129, 257), (100, 512, 200), (130, 4096, 72), (257, 300, 513), (1000, 200, 2050), (1030, 64, 4100), (3001, 130, 4100), (600, 1100, 700), (140, 4100, 70), (3330, 4100, 4099))]


def int8_case(g, t, M, K, N):
    x = rnd(g, M, K, dtype=t)
    x[:, ::37] = x[:, ::37] * 12
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    return x, w, torch.rand(N, generator=g) * 0.1, rnd(g, N)


def rows16(w, dev):
    step = -(-w.shape[1] // 16) * 16
    q = torch.full((w.shape[0], step), 77, dtype=torch.int8, device=dev)          # what stands behind a row does not matter
    q[:, :w.shape[1]] = w.to(dev)
    return q[:, :w.shape[1]]


@pytest.mark.parametrize("dt,M,K,N", INT8)
def test_int8_linear(gpu_device, dt, M, K, N):
    from turboae_amd import sequence
    g = gen(M * 3 + K + N)
    x, w, s, b = int8_case(g, DT[dt], M, K, N)
    if M > 2:
        x[1] = 0.0
    y, bound = O.int8_linear(x, w, s, b if N % 2 else None)
    got = sequence.int8_linear(wide(x, gpu_device, 1, 2) if K % 2 else x.to(gpu_device), rows16(w, gpu_device), s.to(gpu_device), b.to(gpu_device) if N % 2 else None)
    assert got.dtype == DT[dt]
    inside(got, y, bound, "y")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 16), (5, 100), (2, 4096), (4, 131)])
def test_quantize_int8(gpu_device, dt, R, K):
    """Equal to the definition's own steps; quotients half way between two whole numbers go to the even one."""
    from turboae_amd import sequence
    g = gen(R + K)
    x = rnd(g, R, K, dtype=DT[dt])
    x[0, 0] = 2.0
    x[0, 1:9] = torch.tensor([1.0, -1.0, 0.5, 1.5, 2.0 / 127, 3.0 / 127, -0.25, 0.0])[:max(0, min(8, K - 1))]
    if R > 2:
        x[1] = 0.0
        x[2, K // 2] = INF if K % 2 else NAN
    q, s = sequence.quantize_int8(x.to(gpu_device))
    wq, ws = O.quantize(x)
    rows = [i for i in range(R) if not (R > 2 and i == 2)]
    assert torch.equal(q.cpu().double()[rows], wq[rows]) and torch.equal(s.cpu()[rows], ws[rows])
    if R > 2:
        assert math.isnan(float(s[2])) and int(q[2].abs().sum()) == 0
    assert q.stride(0) % 64 == 0 and int(q.as_strided((R, q.stride(0)), (q.stride(0), 1))[:, K:].abs().sum()) == 0


@pytest.mark.parametrize("dt,size", [("f32", 1e-37), ("f32", 1e-40), ("f32", 3e38), ("bf16", 1e-37), ("bf16", 3e38), ("f16", 6e-8), ("f16", 6e4)])
def test_quantize_int8_of_tiny_and_huge_rows(gpu_device, dt, size):
    """Magnitudes whose reciprocal overflows, numbers below the normal ones, and the largest (where 127 x overflows 32 bits: as in 64)."""
    from turboae_amd import sequence
    x = (torch.linspace(-1.0, 1.0, 96)[None] * size).to(DT[dt])
    q, s = sequence.quantize_int8(x.to(gpu_device))
    wq, ws = O.quantize(x)
    if bool(torch.isfinite(x.float() * 127.0).all()):
        assert torch.equal(q.cpu().double(), wq) and torch.equal(s.cpu(), ws)
    else:
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu().double(), torch.round(x.double() * 127.0 / x.double().abs().max()))


def test_int8_rows_with_nan_spoil_only_themselves(gpu_device):
    from turboae_amd import sequence
    g = gen(3)
    x, w, s, b = int8_case(g, torch.float32, 40, 200, 48)
    y, bound = O.int8_linear(x, w, s, b)
    x[5, 3], x[7, 9] = NAN, -INF
    got = sequence.int8_linear(x.to(gpu_device), rows16(w, gpu_device), s.to(gpu_device), b.to(gpu_device))
    assert bool(torch.isnan(got[[5, 7]]).all())
    keep = [i for i in range(40) if i not in (5, 7)]
    inside(got[keep], y[keep], bound[keep], "y")


def test_int8_sums_stay_exact_at_the_largest_inputs(gpu_device):
    """131072 products of 127 * 127, all of one sign: 2.1e9 of 2^31."""
    from turboae_amd import sequence
    K = 131072
    x = torch.full((2, K), 3.0)
    x[1, ::2] = -3.0
    w = torch.full((3, K), 127, dtype=torch.int8)
    w[1] = -127
    w[2, ::2] = -127
    y, bound = O.int8_linear(x, w, torch.ones(3), None)
    inside(sequence.int8_linear(x.to(gpu_device), rows16(w, gpu_device), torch.ones(3, device=gpu_device)), y, bound, "y")


# ---------------------------------------------------------------------------------------------------------------- token_logprobs
LOGP = [(dt, *shape) for dt in DT for shape in ((7, 1, 1), (300, 2, 2), (65, 3, 0), (9, 56, 5), (5, 57, 32), (4, 64, 8), (3, 500, 20), (6, 2049, 32), (2, 5000, 8), (3, 32749, 4), (1, 50001, 20), (2, 131072, 8))]


def check_logprobs(logits, tokens, top, dev, given=None):
    from turboae_amd import sequence
    want = O.logprobs(logits, tokens, top)
    logp, entropy, ids, top_logp = sequence.token_logprobs(logits.to(dev) if given is None else given, tokens.to(dev), top=top)
    safe = tokens.long().clamp(0, logits.shape[-1] - 1)
    inside(logp, want[0], want[4](logits.double().gather(-1, safe[..., None]))[..., 0], "logp")
    inside(entropy, want[1], want[5], "entropy")
    if top == 0:
        assert ids is None and top_logp is None
        return
    assert torch.equal(ids.cpu(), want[2])
    inside(top_logp, want[3], want[4](logits.double().gather(-1, want[2].clamp(min=0))), "top_logp")


@pytest.mark.parametrize("dt,R,V,top", LOGP)
def test_token_logprobs(gpu_device, dt, R, V, top):
    g = gen(R + V)
    logits = rnd(g, R, V, std=3.0, dtype=DT[dt])               # 16-bit values repeat: equal ones in ascending order of their ids
    tokens = torch.randint(0, V, (R,), generator=g, dtype=torch.int32 if V % 2 else torch.int64)
    check_logprobs(logits, tokens, top, gpu_device, wide(logits, gpu_device, 3, 1) if R % 2 else None)


@pytest.mark.parametrize("V", [40, 700, 40000])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_token_logprobs_masks_and_bad_rows(gpu_device, dt, V):
    g = gen(V)
    x = rnd(g, 12, V, std=2.0, dtype=DT[dt])
    x[0] = -INF                                                # nothing left
    x[1] = -INF
    x[1, V - 2] = -5.0                                         # one token left
    x[2, 5:] = -INF                                            # fewer than `top` left
    x[3, 7] = NAN
    x[4, V - 1] = INF
    x[5] = 1.25                                                # all equal
    x[6] = torch.finfo(DT[dt]).min                             # the type's lowest value everywhere ...
    x[7, : V // 2] = torch.finfo(DT[dt]).min                   # ... and as a mask
    x[8, 0], x[8, 1:] = 0.0, -0.0                              # equal too
    x[9] = torch.arange(V).to(DT[dt])                          # the largest ones side by side
    tokens = torch.tensor([0, V - 2, V - 1, 1, 1, V - 1, 3, 0, 2, -1, -100, V], dtype=torch.int64)
    check_logprobs(x, tokens, 12, gpu_device)


def test_token_logprobs_of_adversarial_rows(gpu_device):
    """Rows whose largest values stand in one lane's, one part's or the last places."""
    V = 50000
    x = torch.zeros(5, V)
    x[0] = torch.arange(V, dtype=torch.float32) * 1e-3
    x[1] = -torch.arange(V, dtype=torch.float32) * 1e-3
    x[2, 4::512] = torch.arange(1, 1 + len(x[2, 4::512]), dtype=torch.float32)
    x[3, -40:] = 7.0
    x[4] = 300.0 * torch.sin(torch.arange(V, dtype=torch.float32))
    check_logprobs(x, torch.tensor([V - 1, 0, 4, V - 1, 17]), 32, gpu_device)


# ---------------------------------------------------------------------------------------------------------------- streams, graphs, devices
def test_operators_follow_the_current_stream_and_graphs_replay(gpu_device):
    """One decoding step captured on a side stream and replayed with other work between: every replay equals the eager call."""
    from turboae_amd import sequence
    g = gen(11)
    E, N, V, Bt = 128, 16, 5000, 4
    t = torch.bfloat16
    dev = gpu_device
    x = rnd(g, Bt, 1, E, dtype=t).to(dev)
    cw, cb, A, head = on(dev, rnd(g, E, 4), rnd(g, E), -torch.rand(E, N, generator=g) - 0.1, rnd(g, V, E, std=0.1))
    q, s = sequence.quantize_int8(head)
    w_norm = torch.ones(E, device=dev)
    tokens = torch.randint(0, V, (Bt,), generator=g).to(dev)
    bc = rnd(g, Bt, 1, 2 * N, dtype=t).to(dev)

    def step(conv_state, state):
        u, _ = sequence.causal_conv(x, cw, cb, state=conv_state, state_out=conv_state)
        y, _ = sequence.selective_scan(u, u, A, bc[..., :N], bc[..., N:], z=x, state=state, state_out=state)
        r, n = sequence.norm_residual(x, y, pre_weight=w_norm)
        logits = sequence.int8_linear(n[:, 0], q, s)
        return (r, *sequence.token_logprobs(logits, tokens, top=5))

    def fresh():
        return torch.zeros(Bt, 3, E, dtype=t, device=dev), torch.zeros(Bt, E, N, device=dev)

    eager_states, want = fresh(), []
    for i in range(4):
        x.copy_(rnd(gen(100 + i), Bt, 1, E, dtype=t))
        want.append([v.clone() for v in step(*eager_states)])
    states = fresh()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(*fresh())                                          # the library is loaded and warm before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(*states)
    torch.cuda.current_stream(dev).wait_stream(side)
    for v in states:
        v.zero_()
    for i in range(4):
        x.copy_(rnd(gen(100 + i), Bt, 1, E, dtype=t))
        graph.replay()
        step(*fresh())                                          # eager work between the replays
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
    assert torch.equal(states[0], eager_states[0]) and torch.equal(states[1], eager_states[1])


def test_refusals_name_what_is_wrong(gpu_device):
    from turboae_amd import sequence
    from turboae_amd._lib import TurboAEError
    dev = gpu_device
    x, w = torch.zeros(2, 4, 16, device=dev), torch.zeros(16, 4, device=dev)
    bad = [lambda: sequence.causal_conv(x[0], w), lambda: sequence.causal_conv(x, w[:8]), lambda: sequence.causal_conv(x, w.half()), lambda: sequence.causal_conv(x, w.t().contiguous().t()),
           lambda: sequence.causal_conv(x.transpose(1, 2), torch.zeros(4, 4, device=dev)), lambda: sequence.causal_conv(x, torch.zeros(16, 9, device=dev)),
           lambda: sequence.causal_conv(x, w, act="elu"), lambda: sequence.causal_conv(x, w, lengths=torch.zeros(2, dtype=torch.int64, device=dev)),
           lambda: sequence.causal_conv(x, w, state=torch.zeros(2, 3, 16)), lambda: sequence.causal_conv(x[:, :0], w), lambda: sequence.causal_conv(x.double(), w),
           lambda: sequence.causal_conv(x.clone().requires_grad_(), w)]
    A, bc = torch.zeros(16, 8, device=dev), torch.zeros(2, 4, 8, device=dev)
    buf = torch.zeros(2 * 16 * 8 + 8, device=dev)
    bad += [lambda: sequence.selective_scan(x, x[:, :2], A, bc, bc), lambda: sequence.selective_scan(x, x, torch.zeros(16, 65, device=dev), bc, bc),
            lambda: sequence.selective_scan(x, x, A, bc[..., :4], bc), lambda: sequence.selective_scan(x, x, A, bc, bc, z=x.half()), lambda: sequence.selective_scan(x, x, A, bc, bc, D=torch.zeros(15, device=dev)),
            lambda: sequence.selective_scan(x, x, A, bc, bc, state=buf[:256].view(2, 16, 8), state_out=buf[4:260].view(2, 16, 8)), lambda: sequence.selective_scan(x, x[0, 0], A, bc, bc)]
    ones = torch.ones(16, device=dev)
    bad += [lambda: sequence.norm_residual(x), lambda: sequence.norm_residual(x, x.half()[:, :3], pre_weight=ones), lambda: sequence.norm_residual(x.half(), x), lambda: sequence.norm_residual(x, x, gate=x[:1]),
            lambda: sequence.norm_residual(x, x, gate_act="elu"), lambda: sequence.norm_residual(x, x, post_weight=ones[:3]),
            lambda: sequence.norm_residual(x, x, residual_out=x[:, :1].expand(2, 4, 16)), lambda: sequence.norm_residual(x, pre_weight=ones, dtype=torch.int8)]
    q, s = sequence.quantize_int8(torch.ones(8, 20, device=dev))
    bad += [lambda: sequence.quantize_int8(x), lambda: sequence.int8_linear(torch.zeros(2, 21, device=dev), q, s), lambda: sequence.int8_linear(torch.zeros(2, 20, device=dev), q.contiguous(), s),
            lambda: sequence.int8_linear(torch.zeros(2, 20, device=dev), q.float(), s), lambda: sequence.int8_linear(torch.zeros(2, 20, device=dev), q, s[:4]),
            lambda: sequence.int8_linear(torch.zeros(2, 8, device=dev), torch.zeros(8, dtype=torch.int8, device=dev).view(1, 8), s[:1])]
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    lg = torch.zeros(4, 10, device=dev)
    bad += [lambda: sequence.token_logprobs(lg, t[:3]), lambda: sequence.token_logprobs(lg, t.float()), lambda: sequence.token_logprobs(lg, t, top=11), lambda: sequence.token_logprobs(lg, t, top=-1),
            lambda: sequence.token_logprobs(lg, t.cpu()), lambda: sequence.token_logprobs(lg.t(), torch.zeros(10, dtype=torch.int64, device=dev)), lambda: sequence.token_logprobs(lg.long(), t)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TurboAEError)):
            call()
            raise AssertionError(f"call {i} was not refused")
    with pytest.raises(TurboAEError, match="eps"):
        sequence.norm_residual(x, x, eps=0.0)
