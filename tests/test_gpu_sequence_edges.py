"""The sequence operators at the edges of what they take: every way in which a scan is cut, growing states, distances that pass 32 bits,
gates next to zero, outputs in every place that they may and may not have."""
import pytest
import torch

from tests import _sequence_oracle as O
from tests.test_gpu_sequence import DT, INF, NAN, gen, inside, on, rnd, run_scan, scan_case

pytestmark = pytest.mark.gpu

# batch, len, channels, states: few and many lanes for a channel, one and several pieces, by the time that the host expects of each
FORMS = [(5, 5, 19757, 1), (1, 421, 14432, 1), (5, 5, 19756, 5), (1, 700, 9011, 5), (5, 5, 19757, 9), (5, 5, 19756, 17), (5, 700, 1602, 5), (3, 5, 16885, 9), (1, 700, 4808, 9),
         (3, 5, 16885, 17), (3, 5, 16885, 33), (2, 700, 2193, 9), (2, 5, 12335, 17), (1, 700, 2566, 17), (1, 5, 12335, 33), (1, 500, 3512, 33), (3, 5, 16884, 1), (1, 421, 7701, 1),
         (3, 5, 16885, 5), (1, 500, 6582, 5), (2, 5, 12335, 5), (1, 421, 3512, 5), (2, 5, 12336, 9), (1, 500, 3512, 9), (1, 300, 1, 5), (1, 5, 12335, 9), (1, 421, 1874, 9), (1, 5, 12335, 17),
         (1, 421, 1874, 17), (1, 300, 4, 9), (1, 300, 3, 17), (1, 300, 1, 64), (5, 50, 19757, 9), (1, 2100, 4100, 9), (1, 2048, 4096, 9), (12, 12, 10543, 9), (1, 421, 1369, 9), (1, 421, 1602, 17),
         (1, 20, 4000, 3), (1, 20, 12335, 5), (2, 20, 12335, 9), (1, 20, 300, 9), (1, 20, 12335, 17), (1, 20, 300, 17), (1, 30, 3000, 33), (3, 7, 100, 64), (2, 12, 65, 4), (3, 2, 33, 16),
         (2, 24, 40, 64), (4, 9, 3, 2), (2, 3, 1, 1)]


@pytest.mark.parametrize("B,L,E,N", FORMS)
def test_selective_scan_in_every_form(gpu_device, B, L, E, N):
    dt = ("bf16", "f32", "f16")[(B + L + E + N) % 3]
    c = scan_case(B + L + E + N, dt, B, L, E, N, E % 3 != 0, L % 2 == 1, [L - 3 * i if i % 3 else L for i in range(B)])
    y, h, by, bh = O.scan(**c)
    got, state = run_scan(c, gpu_device, strided=E % 2 == 1)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


@pytest.mark.parametrize("E", [1, 24])
def test_selective_scan_of_growing_states(gpu_device, E):
    """A positive A: the factor across a piece of the positions passes the largest float.  A state of zero stays zero, and a tiny one grows
    to what it grows to step by step."""
    L, N = 300, 4
    c = scan_case(1, "f32", 1, L, E, N, False, False, None)
    c.update(A=torch.full((E, N), 0.5), dt=torch.full((1, L, E), 2.0), dt_bias=None, softplus=False)
    c["x"][:, :290] = 0.0                                       # nothing for 290 positions, growing by e for each
    y, h, by, bh = O.scan(**c)
    assert bool(torch.isfinite(h).all()) and float(h.abs().max()) > 0
    got, state = run_scan(c, gpu_device, False)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")
    c["dt"][:, :64], c["dt"][:, 64:128], c["dt"][:, 128:] = 0.0, 2.9, 0.0        # e^92.8 across one piece
    c["x"][:] = 0.0
    c["state"] = torch.full((1, E, N), 1e-37)
    y, h, by, bh = O.scan(**c)
    assert 1e3 < float(h.max()) < 1e4
    got, state = run_scan(c, gpu_device, False)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


def test_a_tanh_gate_keeps_its_digits_next_to_zero(gpu_device):
    """With a residual of zero r = tanh(gate), off by U of itself, not of 1.  From |g| = 1/4 on 1 - 2 s with s = 1 / (1 + w), w = e^2|g|: w is
    off by 3 U (exponent, exp), 1 + w by 3 U, s by 5 U; 2 s is 0.76 and the result 0.24 at 1/4, so 16 U and its own rounding, and less
    further out.  The series below: its first term and one rounding, 3 U.  20 U hold for both."""
    from turboae_amd import sequence
    size = torch.logspace(-30, 1, 500, base=2.0, dtype=torch.float32)
    g = torch.cat([size, -size, torch.tensor([0.0, 0.25, -0.25, 0.24999999, 30.0, -100.0])]).view(1, 1, -1)
    r, _ = sequence.norm_residual(torch.zeros_like(g).to(gpu_device), torch.ones_like(g).to(gpu_device), gate=g.to(gpu_device), gate_act="tanh")
    want = torch.tanh(g.double())
    inside(r, want, 20 * O.U * want.abs() + 1e-38, "tanh")


def far(dev, first, second, dtype):
    """Two rows of equal shape in one allocation, more than 2^31 elements apart: (2, ...) whose first stride passes 32 bits."""
    n = first.numel()
    gap = (1 << 31) + 64
    w = torch.empty(gap + n, dtype=dtype, device=dev)
    w[:n], w[gap:] = first.reshape(-1).to(dev), second.reshape(-1).to(dev)
    return w.as_strided((2, *first.shape), (gap, *first.contiguous().stride()))


def test_distances_that_pass_32_bits(gpu_device):
    from turboae_amd import sequence
    dev, t = gpu_device, torch.bfloat16
    g = gen(9)
    E, L, N, K, V = 72, 9, 16, 200, 3000
    x = rnd(g, 2, L, E, dtype=t)
    xd = far(dev, x[0], x[1], t)
    w, bias, pre = rnd(g, E, 4), rnd(g, E), 1 + rnd(g, E, std=0.1)
    y, s, bound = O.conv(x, w, bias, None, None, "silu")
    got, state = sequence.causal_conv(xd, *on(dev, w, bias))
    inside(got, y, bound, "conv")
    c = scan_case(2, "bf16", 2, L, E, N, True, True, None)
    c["x"] = x
    y, h, by, bh = O.scan(**c)
    k = {n: (v.to(dev) if isinstance(v, torch.Tensor) else v) for n, v in c.items()}
    k.update(x=xd)
    got, state = sequence.selective_scan(**k)
    inside(got, y, by, "scan")
    inside(state, h, bh, "state")
    one = {n: (v[:, :1] if n in ("dt", "B", "C", "z") else v) for n, v in c.items()}
    one["x"] = x[:, :1]
    y, h, by, bh = O.scan(**one)
    got, state = sequence.selective_scan(**{**{n: (v.to(dev) if isinstance(v, torch.Tensor) else v) for n, v in one.items()}, "x": xd[:, :1]})
    inside(got, y, by, "step")
    r, n, br, bn = O.norm_residual(x, x, None, None, None, None, pre, None, False, "sigmoid", 1.0, 1e-5, t)
    out = xd.clone(memory_format=torch.contiguous_format)
    got = sequence.norm_residual(xd, out, pre_weight=pre.to(dev), residual_out=xd)
    inside(got[0], r, br, "r")
    inside(got[1], n, bn, "normed")
    del xd, k, out, got
    rows = rnd(g, 2, K, dtype=t)
    q = torch.randint(-127, 128, (40, 208), generator=g, dtype=torch.int8)
    scale = torch.rand(40, generator=g)
    y, bound = O.int8_linear(rows, q[:, :K], scale, None)
    inside(sequence.int8_linear(far(dev, rows[0], rows[1], t), q.to(dev)[:, :K], scale.to(dev)), y, bound, "int8")
    lg = rnd(g, 2, V, dtype=t)
    tokens = torch.tensor([5, V - 1])
    want = O.logprobs(lg, tokens, 3)
    got = sequence.token_logprobs(far(dev, lg[0], lg[1], t), tokens.to(dev), top=3)
    inside(got[0], want[0], want[4](lg.double().gather(-1, tokens[:, None]))[:, 0], "logp")
    assert torch.equal(got[2].cpu(), want[2])


def test_outputs_lie_where_they_may_and_nowhere_else(gpu_device):
    from turboae_amd import sequence
    from turboae_amd._lib import TurboAEError
    dev, g = gpu_device, gen(4)
    x, w, ones = rnd(g, 2, 4, 16).to(dev), rnd(g, 16, 4).to(dev), torch.ones(16, device=dev)
    # rows of residual_out in another order of memory, and the block's own place
    want = sequence.norm_residual(x, x * 2, pre_weight=ones)
    out = torch.full((4, 2, 16), NAN, device=dev).transpose(0, 1)
    got = sequence.norm_residual(x, x * 2, pre_weight=ones, residual_out=out)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    buf = torch.zeros(2 * 4 * 16 + 16, device=dev)
    a, b = buf[:128].view(2, 4, 16), buf[16:].view(2, 4, 16)
    A, bc = -torch.ones(16, 8, device=dev), rnd(g, 2, 4, 8).to(dev)
    flat = rnd(g, 1, 4, 16).to(dev)
    bad = [lambda: sequence.norm_residual(a, x, residual_out=b), lambda: sequence.norm_residual(x, a, residual_out=b), lambda: sequence.norm_residual(x, x * 2, gate=x[:, :1], residual_out=x),
           lambda: sequence.norm_residual(x, x * 2, pre_weight=x[0, 0], residual_out=x), lambda: sequence.norm_residual(x, x * 2, residual_out=buf[:4 * 16 + 16].as_strided((2, 4, 16), (16, 16, 1))),
           lambda: sequence.causal_conv(flat, w, state_out=flat[:, 1:]),
           lambda: sequence.norm_residual(x, x * 2, pre_weight=ones, eps=1e-40), lambda: sequence.norm_residual(x, x * 2, pre_weight=ones, eps=-1.0)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TurboAEError)):
            call()
            raise AssertionError(i)
    both = rnd(g, 2 * 16 * 8).to(dev)
    with pytest.raises(ValueError, match="overlaps"):
        sequence.selective_scan(both[:128].view(2, 4, 16), x, A, bc, bc, state_out=both.view(2, 16, 8))


@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 6, 7, 9, 63, 66, 131, 257, 515, 1029, 2051, 4099, 8191, 20000, 16385, 32768, 32767, 32766, 32764])
@pytest.mark.parametrize("dt", DT)
def test_norms_of_any_width(gpu_device, dt, D):
    from turboae_amd import sequence
    g, t, dev = gen(D), DT[dt], gpu_device
    r, x, gate = rnd(g, 1, 3, D), rnd(g, 1, 3, D, dtype=t), rnd(g, 1, 3, D, dtype=t)
    post, pre = 1 + rnd(g, D, std=0.1), 1 + rnd(g, D, std=0.1)
    want = O.norm_residual(r, x, gate, None, post, None, pre, None, True, "sigmoid", 0.5, 1e-5, t)
    got = sequence.norm_residual(*on(dev, r, x), gate=gate.to(dev), post_weight=post.to(dev), pre_weight=pre.to(dev), center=True, alpha=0.5)
    inside(got[0], want[0], want[2], "r")
    inside(got[1], want[1], want[3], "normed")


def test_infinite_inputs_stay_in_their_channel(gpu_device):
    """An infinity in x is an infinity or NaN from its position on, in its own channel and sequence only."""
    from turboae_amd import sequence
    g, dev = gen(8), gpu_device
    x, dt, B, C = rnd(g, 2, 300, 16), rnd(g, 2, 300, 16), rnd(g, 2, 300, 16), rnd(g, 2, 300, 16)
    A = -torch.rand(16, 16, generator=g) - 0.1
    clean = sequence.selective_scan(*on(dev, x, dt, A, B, C))
    x[1, 100, 5] = INF
    y, h = sequence.selective_scan(*on(dev, x, dt, A, B, C))
    other = torch.ones(2, 300, 16, dtype=torch.bool)
    other[1, 100:, 5] = False
    assert torch.equal(y.cpu()[other], clean[0].cpu()[other])
    assert not bool(torch.isfinite(y[1, 100, 5])) and not bool(torch.isfinite(h[1, 5]).any())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("K", [1, 15, 64, 100, 511, 1000, 3001, 9000])
def test_int8_of_few_rows(gpu_device, dt, K):
    """1 to 17 rows, with one of zeros, one with a NaN and one with an infinity, which spoil only themselves; rows on any element."""
    from turboae_amd import sequence
    dev, t = gpu_device, DT[dt]
    for M in (1, 2, 3, 4, 5, 8, 9, 16, 17):
        for N in (1, 17, 40):
            g = gen(M * 1000 + K + N)
            x, w = rnd(g, M, K, dtype=t), torch.randint(-127, 128, (N, -(-K // 16) * 16), generator=g, dtype=torch.int8)
            s, b = torch.rand(N, generator=g), rnd(g, N)
            if M > 4:
                x[1], x[2, K // 2], x[4, K - 1] = 0.0, NAN, -INF
            keep = [i for i in range(M) if M <= 4 or i not in (2, 4)]
            y, bound = O.int8_linear(x[keep], w[:, :K], s, b)
            buf = torch.full((M, K + 3), NAN, dtype=t, device=dev)
            buf[:, 1:K + 1] = x.to(dev)
            got = sequence.int8_linear(buf[:, 1:K + 1], w.to(dev)[:, :K], s.to(dev), b.to(dev))
            inside(got[keep], y, bound, (M, N))
            assert len(keep) == M or bool(torch.isnan(got[[2, 4]]).all())
