"""The sequence operators in the forms that only larger or rounder calls take.  Which form a case takes is counted without a GPU, beside these
lists (test_sequence_forms.py)."""
import pytest
import torch

from tests import _sequence_oracle as O
from tests.test_gpu_sequence import DT, INF, check_logprobs, gen, inside, int8_case, rnd, rows16, run_scan, scan_case, wide

pytestmark = pytest.mark.gpu

# one position: 1 or 4 sequences for each workgroup (the last of 4 not full), 1 to 64 lanes for a channel with 1 or 4 states each
STEPS = [("f32", 33, 16328, 1), ("bf16", 17, 16092, 2), ("f16", 17, 12240, 3), ("bf16", 9, 11931, 5), ("f32", 5, 8136, 13), ("bf16", 5, 6909, 17), ("f16", 5, 3428, 33), ("bf16", 66, 8232, 4),
         ("bf16", 17, 16376, 8), ("bf16", 66, 4096, 16), ("f32", 257, 2051, 12), ("f16", 5, 14112, 32), ("bf16", 6, 5472, 64),
         ("f32", 3, 40, 1), ("bf16", 3, 33, 2), ("f16", 4, 65, 3), ("f32", 3, 9, 9), ("bf16", 5, 70, 17), ("f16", 3, 33, 33), ("bf16", 3, 300, 4), ("f32", 4, 130, 8), ("bf16", 3, 257, 12),
         ("f16", 3, 64, 20), ("bf16", 4, 33, 40)]
# few positions, tiles and lanes that the other lists leave out
SHORT = [("bf16", 3, 2, 70, 2), ("f16", 2, 3, 40, 3), ("f32", 1, 2, 4, 4), ("bf16", 2, 2, 8221, 8), ("f32", 2, 2, 4395, 12), ("bf16", 100, 12, 130, 12), ("f16", 3, 12, 2048, 16), ("bf16", 220, 3, 131, 16),
         ("f32", 2, 2, 4, 20), ("bf16", 4, 9, 40, 20)]
LONG = [("bf16", 9, 15, 13176, 16), ("f32", 1, 2048, 4096, 16), ("bf16", 2, 15, 3, 17), ("f16", 1, 300, 4, 17), ("bf16", 2, 200, 4, 40), ("f32", 2, 2, 4, 12), ("bf16", 3, 7, 8, 17), ("f16", 1, 421, 1924, 17)]
SCANS = [(dt, B, 1, E, N) for dt, B, E, N in STEPS] + SHORT + LONG


@pytest.mark.parametrize("dt,B,L,E,N", SCANS)
@pytest.mark.parametrize("padded", [False, True])
def test_selective_scan_in_its_larger_forms(gpu_device, dt, B, L, E, N, padded):
    """padded: slices of wider tensors, lengths from none to all, gate and D, the state updated in place."""
    c = scan_case(B + L + E + N, dt, B, L, E, N, padded, True, [(7 * i) % (L + 1) if i % 3 else (L, 0)[i % 2] for i in range(B)] if padded else None)
    y, h, by, bh = O.scan(**c)
    c["state"] = c["state"].to(gpu_device)
    got, state = run_scan(c, gpu_device, strided=padded, state_out=c["state"] if padded else None)
    assert not padded or state is c["state"]
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


# 64 x 32 outputs for a workgroup, aligned rows of tiles, more 256 x 256 tiles than workgroups: all rows, or the first, the last and some between
INT8_LARGE = [("bf16", 128, 4096, 4096), ("f32", 100, 4100, 4090), ("f16", 100, 4100, 4090), ("bf16", 1000, 200, 2048), ("f16", 1000, 200, 2048), ("f32", 1000, 200, 2048), ("bf16", 3001, 130, 4096),
              ("bf16", 600, 1100, 704), ("f32", 600, 1100, 704), ("bf16", 4353, 4100, 4352), ("f16", 4353, 4100, 4344), ("f32", 4353, 4100, 4352), ("bf16", 4353, 4096, 4353)]


@pytest.mark.parametrize("dt,M,K,N", INT8_LARGE)
def test_int8_linear_in_its_larger_forms(gpu_device, dt, M, K, N):
    from turboae_amd import sequence
    x, w, s, b = int8_case(gen(M + K + N), DT[dt], M, K, N)
    rows = sorted({*range(0, M, max(1, M // 250)), *range(max(0, M - 20), M), *(r for r in range(256 - 2, M, 256)), *(r for r in range(256, M, 256))})
    y, bound = O.int8_linear(x[rows], w, s, b)
    got = sequence.int8_linear(x.to(gpu_device), rows16(w, gpu_device), s.to(gpu_device), b.to(gpu_device))
    assert got.shape == (M, N)
    inside(got[torch.tensor(rows, device=gpu_device)], y, bound, "y")
    # every output of every row: the sums of its columns against the sums of the oracle's products
    q, scale = O.quantize(x)
    whole = (q * scale.double()[:, None]).sum(0) @ w.double().t() * s.double() + M * b.double()
    size = ((q.abs() * scale.double()[:, None]).sum(0) @ w.double().abs().t()) * s.double() + M * b.double().abs()
    f = torch.finfo(DT[dt])
    inside(got.double().sum(0), whole, (6 * O.U + f.eps / 2) * size + M * f.eps / 2 * f.tiny, "columns")


# one workgroup of four waves for a row or a part of it, 32 or 64 elements for each lane
LOGP_LARGE = [("f32", 600, 7001, 0), ("bf16", 600, 7001, 8), ("f16", 300, 20000, 32), ("bf16", 600, 16000, 5), ("f32", 600, 16001, 32), ("bf16", 500, 20000, 8), ("f16", 5, (1 << 21) - 3, 20),
              ("bf16", 3, 300001, 32), ("bf16", 2100, 2040, 8), ("f32", 2100, 2045, 3)]


@pytest.mark.parametrize("dt,R,V,top", LOGP_LARGE)
@pytest.mark.parametrize("odd", [False, True])
def test_token_logprobs_in_its_larger_forms(gpu_device, dt, R, V, top, odd):
    g = gen(R + V)
    logits = rnd(g, R, V, std=3.0, dtype=DT[dt])
    tokens = torch.randint(0, V, (R,), generator=g)
    check_logprobs(logits, tokens, top, gpu_device, wide(logits, gpu_device, 3, 2) if odd else None)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [33, 56, 57, 60, 61, 63, 64, 65, 504, 505, 508, 511, 512, 513])
@pytest.mark.parametrize("left", [0, 1, 5])
def test_token_logprobs_of_short_rows_that_start_anywhere(gpu_device, dt, V, left):
    g = gen(V + left)
    logits = rnd(g, 130, V, std=3.0, dtype=DT[dt])
    tokens = torch.randint(0, V, (130,), generator=g)
    for top in (0, 1, min(V, 32)):
        check_logprobs(logits, tokens, top, gpu_device, wide(logits, gpu_device, left, 0))


# states that fill the lanes of every form, and states that do not
INFINITE = [("bf16", 1, 15, 3, 9), ("f32", 1, 15, 4, 9), ("f16", 1, 300, 3, 9), ("bf16", 1, 300, 4, 9), ("f32", 1, 15, 3, 17), ("bf16", 1, 15, 4, 17), ("f32", 1, 300, 3, 28), ("f16", 1, 300, 4, 17),
            ("bf16", 1, 15, 3, 33), ("f32", 1, 15, 4, 33), ("bf16", 1, 200, 7, 33), ("f16", 1, 200, 4, 33), ("f32", 1, 7, 3, 1), ("bf16", 1, 7, 4, 2), ("bf16", 1, 300, 3, 3), ("f32", 1, 300, 4, 1),
            ("f16", 1, 2, 3, 5), ("f32", 1, 2, 4, 5), ("bf16", 1, 300, 3, 7), ("f32", 1, 300, 4, 5), ("bf16", 1, 2, 3, 11), ("f32", 1, 2, 4, 9), ("f16", 1, 500, 1562, 9), ("bf16", 1, 421, 1788, 9),
            ("f32", 1, 7, 3, 28), ("bf16", 1, 7, 4, 17), ("f32", 1, 421, 1871, 17), ("bf16", 1, 421, 1852, 17), ("bf16", 9, 7, 14288, 9), ("f32", 9, 15, 13176, 14), ("f32", 1, 2048, 4096, 9), ("bf16", 1, 2048, 4096, 13),
            ("f32", 1, 2, 13260, 9), ("bf16", 1, 2, 3, 17), ("f16", 1, 2, 4, 3), ("f32", 1, 2, 4, 33), ("bf16", 1, 2, 8704, 5), ("f32", 1, 2, 9452, 12), ("bf16", 1, 2, 3, 20),
            ("f32", 3, 1, 33, 5), ("bf16", 3, 1, 70, 12), ("f32", 257, 1, 2051, 12),
            ("bf16", 1, 15, 3, 16), ("f32", 1, 15, 4, 16), ("f16", 1, 15, 3, 32), ("bf16", 1, 15, 4, 32), ("f32", 1, 15, 3, 64), ("f16", 1, 15, 4, 64), ("bf16", 1, 7, 3, 4), ("f32", 1, 7, 4, 4), ("bf16", 1, 7, 3, 8),
            ("f16", 1, 7, 4, 8), ("f32", 1, 7, 3, 16), ("bf16", 1, 7, 4, 16), ("bf16", 1, 7, 3, 32), ("f32", 1, 7, 4, 32), ("bf16", 6, 7, 2713, 4), ("f32", 1, 7, 3, 64), ("bf16", 9, 15, 13176, 16)]


@pytest.mark.parametrize("dt,B,L,E,N", INFINITE)
def test_infinities_come_out_as_the_formula_has_them(gpu_device, dt, B, L, E, N):
    """An infinite input, an infinite step and an infinite incoming state, each in a channel of its own, with everything positive: infinite
    from there on, no NaN, and other channels as they are.  Steps are small, so that no decay underflows to 0 (0 times infinity is NaN)."""
    c = scan_case(B + L + E + N, dt, B, L, E, N, True, True, None)
    for name in ("x", "B", "C", "D", "z", "state"):
        c[name] = c[name].abs() + 0.0625
    c["dt"] = c["dt"].clamp(-1.0, 1.0)
    c["dt_bias"] = torch.full((E,), -7.0)
    c["x"][0, L // 2, 0] = INF
    c["dt"][0, L // 2, 1] = INF
    c["state"][B - 1, E - 1, N - 1] = INF
    y, h, by, bh = O.scan(**c)
    assert not bool(torch.isnan(y).any()) and bool(torch.isinf(y[0, L // 2:, :2]).all()) and bool(torch.isinf(y[B - 1, :, E - 1]).all())
    got, state = run_scan(c, gpu_device, strided=False)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


@pytest.mark.parametrize("dt,B,L,E,N", [("f32", 2, 1, 40, 4), ("bf16", 33, 1, 16328, 1), ("f16", 3, 2, 9, 3), ("bf16", 2, 2, 4395, 12), ("f32", 2, 15, 6, 16), ("bf16", 2, 300, 8, 9), ("f16", 1, 300, 5, 4),
                                        ("f32", 9, 15, 13176, 16), ("f32", 1, 2048, 4096, 9)])
def test_an_absent_direct_term_adds_nothing_to_an_infinity(gpu_device, dt, B, L, E, N):
    """Without D an infinite x comes out of the states alone; a D of zeros makes NaN of it, as the formula does."""
    c = scan_case(B + L + E + N, dt, B, L, E, N, False, False, None)
    for name in ("x", "B", "C"):
        c[name] = c[name].abs() + 0.0625
    c["dt"], c["dt_bias"] = c["dt"].clamp(-1.0, 1.0), torch.full((E,), -7.0)
    c["x"][0, L // 2, 0] = INF
    for D in (None, torch.zeros(E)):
        c["D"] = D
        y, h, by, bh = O.scan(**c)
        assert bool(torch.isinf(y[0, L // 2, 0])) == (D is None)
        got, state = run_scan(c, gpu_device, strided=False)
        inside(got, y, by, "y")
        inside(state, h, bh, "state")


@pytest.mark.parametrize("dt,B,L,E,N", [("f32", 1, 300, 4, 9), ("bf16", 1, 700, 64, 16), ("f32", 1, 2048, 4096, 16), ("f32", 1, 300, 4, 64)])
def test_infinite_states_outlast_a_piece_of_the_positions(gpu_device, dt, B, L, E, N):
    """A position's factor is e^-5, that of the 64 and more positions of a piece 0 in 32 bits: an infinite state stays one all the same."""
    c = scan_case(B + L + E + N, dt, B, L, E, N, False, True, None)
    for name in ("x", "B", "C", "state"):
        c[name] = c[name].abs() + 0.0625
    c.update(A=torch.full((E, N), -5.0), dt=torch.ones_like(c["dt"]), dt_bias=None, softplus=False)
    c["state"][0, E // 2, N - 1] = INF
    y, h, by, bh = O.scan(**c)
    assert bool(torch.isinf(y[0, :, E // 2]).all()) and int(torch.isinf(h).sum()) == 1
    got, state = run_scan(c, gpu_device, strided=False)
    inside(got, y, by, "y")
    inside(state, h, bh, "state")


def test_leading_dimensions_that_do_not_fold_are_copied(gpu_device):
    """Rows that no single distance leads through, and last elements that are apart in three dimensions; in two they are refused."""
    from turboae_amd import sequence
    g, dev = gen(6), gpu_device
    x, w, s, b = int8_case(g, torch.bfloat16, 24, 48, 20)
    rows, q, s, b = x.view(4, 6, 48).to(dev), rows16(w, dev), s.to(dev), b.to(dev)
    logits, tokens = rnd(g, 4, 6, 300).to(dev), torch.randint(0, 300, (4, 6), generator=g).to(dev)
    for pick in (lambda v: v[:, 1:5], lambda v: v.transpose(0, 1), lambda v: v.mT.contiguous().mT):
        assert torch.equal(sequence.int8_linear(pick(rows), q, s, b), sequence.int8_linear(pick(rows).contiguous(), q, s, b))
        t = pick(tokens[..., None])[..., 0].contiguous()
        for a, e in zip(sequence.token_logprobs(pick(logits), t, top=4), sequence.token_logprobs(pick(logits).contiguous(), t, top=4)):
            assert torch.equal(a, e)
    for call in (lambda: sequence.int8_linear(rows[0].t().contiguous().t(), q, s, b), lambda: sequence.token_logprobs(logits[0].t().contiguous().t(), tokens[0])):
        with pytest.raises(ValueError, match="adjacent"):
            call()
