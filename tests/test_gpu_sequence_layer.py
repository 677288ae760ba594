"""The sequence operators together: one layer of a selective state-space model from its residual to the log probabilities of its tokens, for a
padded batch of prompts and then token by token, eagerly and as replayed graphs.  Each operator's output is checked against the 64-bit
implementation on that operator's own inputs, so that a rounding on the way (8-bit whole numbers turn one into a step) widens no tolerance."""
import pytest
import torch

from tests import _sequence_oracle as O
from tests.test_gpu_sequence import DT, gen, inside, on, rnd

pytestmark = pytest.mark.gpu

B, L, D, E, N, R, V = 3, 70, 96, 192, 16, 12, 1000


class Layer:
    def __init__(self, dt, dev, seed=3):
        from turboae_amd import sequence
        g = gen(seed)
        self.t, self.dev = DT[dt], dev
        self.pre, self.post, self.last = on(dev, 1 + rnd(g, D, std=0.1), 1 + rnd(g, D, std=0.1), 1 + rnd(g, D, std=0.1))
        self.scale, self.dt_bias, self.skip = on(dev, 0.5 + torch.rand(D, generator=g), rnd(g, E) - 2.0, rnd(g, E))
        self.A = -(1 + torch.rand(E, N, generator=g) * N).to(dev)
        self.taps, self.taps_bias = on(dev, rnd(g, E, 4, std=0.5), rnd(g, E, std=0.1))
        self.linear = {n: sequence.quantize_int8(rnd(g, out, k, std=k ** -0.5).to(dev)) for n, (out, k) in
                       {"in": (2 * E, D), "x": (R + 2 * N, E), "dt": (E, R), "out": (D, E), "head": (V, D)}.items()}

    def states(self):
        return torch.zeros(B, 3, E, dtype=self.t, device=self.dev), torch.zeros(B, E, N, device=self.dev)

    def __call__(self, residual, tokens, conv, state, lengths=None, note=None):
        """residual (B, len, D); conv and state are updated in place.  `note` collects each operator's inputs and outputs."""
        from turboae_amd import sequence

        def call(op, *args, **kw):
            kept = None if note is None else ([v.clone() if isinstance(v, torch.Tensor) else v for v in args], {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
            out = getattr(sequence, op)(*args, **kw)
            if note is not None:
                note.append((op, *kept, [v.clone() if isinstance(v, torch.Tensor) else v for v in (out if isinstance(out, tuple) else (out,))]))
            return out

        n = call("norm_residual", residual, pre_weight=self.pre)[1]
        xz = call("int8_linear", n, *self.linear["in"])
        u, _ = call("causal_conv", xz[..., :E], self.taps, self.taps_bias, state=conv, lengths=lengths, state_out=conv)
        p = call("int8_linear", u, *self.linear["x"])
        dt = call("int8_linear", p[..., :R], *self.linear["dt"])
        y, _ = call("selective_scan", u, dt, self.A, p[..., R:R + N], p[..., R + N:], D=self.skip, z=xz[..., E:], dt_bias=self.dt_bias, state=state, lengths=lengths, state_out=state)
        o = call("int8_linear", y, *self.linear["out"])
        r, n = call("norm_residual", residual, o, scale=self.scale, post_weight=self.post, pre_weight=self.last)
        logits = call("int8_linear", n, *self.linear["head"])
        return (r, *call("token_logprobs", logits, tokens, top=5))


def cpu(v):
    return v.cpu() if isinstance(v, torch.Tensor) else v


def check(note):
    """Every operator of a run against the 64-bit one on the same inputs."""
    for op, args, kw, out in note:
        a, k, out = [cpu(v) for v in args], {n: cpu(v) for n, v in kw.items()}, [cpu(v) for v in out]
        if op == "norm_residual":
            r, n, br, bn = O.norm_residual(a[0], a[1] if len(a) > 1 else None, None, k.get("scale"), k.get("post_weight"), None, k["pre_weight"], None, False, "sigmoid", 1.0, 1e-5, a[0].dtype)
            if len(a) > 1:
                inside(out[0], r, br, op)
            inside(out[1], n, bn, op)
        elif op == "int8_linear":
            y, bound = O.int8_linear(a[0].reshape(-1, a[0].shape[-1]), a[1], a[2], None)
            inside(out[0].reshape(y.shape), y, bound, op)
        elif op == "causal_conv":
            y, s, bound = O.conv(a[0], a[1], a[2], k["state"], k["lengths"], "silu")
            inside(out[0], y, bound, op)
            assert torch.equal(out[1].double(), s)
        elif op == "selective_scan":
            y, h, by, bh = O.scan(*a, k["D"], k["z"], k["dt_bias"], True, k["state"], k["lengths"])
            inside(out[0], y, by, op)
            inside(out[1], h, bh, op)
        else:
            lg = a[0].reshape(-1, V)
            t = a[1].reshape(-1)
            want = O.logprobs(lg, t, 5)
            inside(out[0].reshape(-1), want[0], want[4](lg.double().gather(-1, t.clamp(min=0)[:, None]))[:, 0], "logp")
            inside(out[1].reshape(-1), want[1], want[5], "entropy")
            assert torch.equal(out[2].reshape(-1, 5), want[2])


def inputs(dt, dev, seed, n):
    g = gen(seed)
    return rnd(g, B, n, D, dtype=DT[dt]).to(dev), torch.randint(-1, V, (B, n), generator=g).to(dev)


@pytest.mark.parametrize("dt", DT)
def test_a_layer_on_padded_prompts_then_token_by_token(gpu_device, dt):
    layer = Layer(dt, gpu_device)
    conv, state = layer.states()
    lengths = torch.tensor([L, 0, 33], dtype=torch.int32, device=gpu_device)
    note = []
    layer(*inputs(dt, gpu_device, 20, L), conv, state, lengths=lengths, note=note)
    check(note)
    assert not bool(conv[1].any()) and not bool(state[1].any())                 # an empty sequence leaves its states as they were
    for i in range(3):
        note = []
        layer(*inputs(dt, gpu_device, 30 + i, 1), conv, state, note=note)
        check(note)


@pytest.mark.parametrize("dt", DT)
def test_a_prompt_in_two_calls_is_the_prompt_in_one(gpu_device, dt):
    """The states carry everything: conv's outputs are the same to the bit, the scan's are within the bounds of both ways of cutting it."""
    from turboae_amd import sequence
    layer = Layer(dt, gpu_device)
    x, _ = inputs(dt, gpu_device, 40, L)
    xz = sequence.int8_linear(x, *layer.linear["in"])
    at = 41
    conv, state = layer.states()
    whole, last = sequence.causal_conv(xz[..., :E], layer.taps, layer.taps_bias, state=conv)
    first, conv = sequence.causal_conv(xz[:, :at, :E], layer.taps, layer.taps_bias, state=conv)
    second, conv = sequence.causal_conv(xz[:, at:, :E], layer.taps, layer.taps_bias, state=conv)
    assert torch.equal(torch.cat([first, second], 1), whole) and torch.equal(conv, last)
    p = sequence.int8_linear(whole, *layer.linear["x"])
    step = sequence.int8_linear(p[..., :R], *layer.linear["dt"])

    def scan(a, b, h):
        return sequence.selective_scan(whole[:, a:b], step[:, a:b], layer.A, p[:, a:b, R:R + N], p[:, a:b, R + N:], D=layer.skip, z=xz[:, a:b, E:], dt_bias=layer.dt_bias, state=h)

    y, h, by, bh = O.scan(*(cpu(v) for v in (whole, step, layer.A, p[..., R:R + N], p[..., R + N:], layer.skip, xz[..., E:], layer.dt_bias)), True, None, None)
    y1, h1 = scan(0, at, None)
    y2, h2 = scan(at, L, h1)
    inside(torch.cat([y1, y2], 1), y, by, "y")
    inside(h2, h, bh, "state")


def test_prompt_and_step_replay_as_graphs(gpu_device):
    """Both captured once, each replay on new inputs equals the eager call to the bit, with eager work in between."""
    dt = "bf16"
    layer = Layer(dt, gpu_device)
    dev = gpu_device
    lengths = torch.tensor([L, 12, 33], dtype=torch.int32, device=dev)
    eager_states, want = layer.states(), []
    for i in range(3):
        want.append([v.clone() for v in layer(*inputs(dt, dev, 50 + i, L), *eager_states, lengths=lengths)])
        want.append([v.clone() for v in layer(*inputs(dt, dev, 60 + i, 1), *eager_states)])
    states = layer.states()
    prompt, step = inputs(dt, dev, 50, L), inputs(dt, dev, 60, 1)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graphs, got = [], []
    with torch.cuda.stream(side):
        layer(*prompt, *layer.states(), lengths=lengths)
        layer(*step, *layer.states())
        for static, n in ((prompt, lengths), (step, None)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got.append(layer(*static, *states, lengths=n))
            graphs.append(graph)
    torch.cuda.current_stream(dev).wait_stream(side)
    for v in states:
        v.zero_()
    for i in range(3):
        for j, (static, seed, n) in enumerate(((prompt, 50 + i, L), (step, 60 + i, 1))):
            for v, new in zip(static, inputs(dt, dev, seed, n)):
                v.copy_(new)
            graphs[j].replay()
            layer(*step, *layer.states())                       # eager work between the replays
            torch.cuda.synchronize()
            for a, b in zip(got[j], want[2 * i + j]):
                assert torch.equal(a, b), (i, j)
    for a, b in zip(states, eager_states):
        assert torch.equal(a, b)


def test_two_streams_at_once_change_nothing(gpu_device):
    dt = "f16"
    layer = Layer(dt, gpu_device)
    dev = gpu_device
    given = [inputs(dt, dev, 70 + i, L) for i in range(4)]
    want = []
    for i in range(4):
        s = layer.states()
        want.append([v.clone() for v in layer(*given[i], *s)] + list(s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [None] * 4
    states = [layer.states() for _ in range(4)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = [*layer(*given[i], *states[i]), *states[i]]
    torch.cuda.synchronize()
    for i in range(4):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b), i
