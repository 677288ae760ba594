"""What turboae_amd.sequence refuses before the library is called, seen without a GPU: tensors that say they are on one, so that a call
gets as far as it would there.  One that is let through fails on the missing device instead."""
import pytest
import torch
from torch.autograd import forward_ad

from tests import test_sequence_cpu as C
from turboae_amd import _lib, sequence


class OnDevice(torch.Tensor):
    is_cuda = True


def dev(t):
    return t.as_subclass(OnDevice)


def many(n, *shape, dtype=torch.float32):
    """A tensor of n equal parts without memory for them."""
    return dev(torch.zeros(1, *shape, dtype=dtype).expand(n, *shape))


PAST = (1 << 32) + 1                             # 1 in the library's 32-bit sizes


@pytest.mark.parametrize("call", [
    lambda n: sequence.causal_conv(many(n, 1, 1), dev(torch.zeros(1, 2))),
    lambda n: sequence.causal_conv(dev(torch.zeros(1, 1, 1).expand(1, n, 1)), dev(torch.zeros(1, 2))),
    lambda n: sequence.selective_scan(many(n, 1, 1), many(n, 1, 1), dev(-torch.ones(1, 1)), many(n, 1, 1), many(n, 1, 1)),
    lambda n: sequence.norm_residual(many(n, 1, 4), pre_weight=dev(torch.ones(4)), dtype=torch.float32),
    lambda n: sequence.quantize_int8(many(n, 4)),
    lambda n: sequence.int8_linear(many(n, 16), dev(torch.zeros(1, 16, dtype=torch.int8)), dev(torch.ones(1))),
    lambda n: sequence.int8_linear(dev(torch.zeros(1, 16)), dev(torch.zeros(1, 16, dtype=torch.int8).expand(n, 16)), dev(torch.ones(1).expand(n))),
    lambda n: sequence.token_logprobs(many(n, 1), dev(torch.zeros(1, dtype=torch.int32).expand(n))),
])
@pytest.mark.parametrize("n", [PAST, 1 << 31])
def test_sizes_past_32_bits_are_refused(call, n):
    """They would be cut to their low 32 bits on the way to the library, and most of the outputs left as they were allocated."""
    with pytest.raises(ValueError, match="2\\^31"):
        call(n)


def test_a_type_that_a_block_overrides_is_refused():
    """normed has the block's type; another one that is asked for beside it is not passed over."""
    r, b, w = dev(torch.zeros(1, 2, 4)), dev(torch.zeros(1, 2, 4, dtype=torch.bfloat16)), dev(torch.ones(4))
    with pytest.raises(ValueError, match="block"):
        sequence.norm_residual(r, b, pre_weight=w, dtype=torch.float32)


X, W, ONES = dev(torch.zeros(1, 2, 16)), dev(torch.zeros(16, 4)), dev(torch.ones(16))
A, BC = dev(-torch.ones(16, 8)), dev(torch.zeros(1, 2, 8))
Q, T = dev(torch.zeros(4, 16, dtype=torch.int8)), dev(torch.zeros(2, dtype=torch.int64))


def dual(t):
    return dev(forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("call", [
    lambda d: sequence.causal_conv(d(X), W), lambda d: sequence.causal_conv(X, W, d(ONES)), lambda d: sequence.causal_conv(X, W, state_out=d(dev(torch.zeros(1, 3, 16)))),
    lambda d: sequence.selective_scan(X, d(X), A, BC, BC), lambda d: sequence.selective_scan(X, X, A, BC, BC, z=d(X)), lambda d: sequence.selective_scan(X, X, d(A), BC, BC),
    lambda d: sequence.norm_residual(d(X), X), lambda d: sequence.norm_residual(X, X, gate=d(X)), lambda d: sequence.norm_residual(X, X, residual_out=d(dev(torch.zeros(1, 2, 16)))),
    lambda d: sequence.quantize_int8(d(X[0])), lambda d: sequence.int8_linear(d(X), Q, ONES[:4]), lambda d: sequence.int8_linear(X, Q, ONES[:4], bias=d(ONES[:4])),
    lambda d: sequence.token_logprobs(d(X[0]), T),
])
def test_forward_mode_tangents_are_refused(call):
    """A dual tensor does not require a gradient; without a refusal the call would return values whose tangents are gone."""
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(ValueError, match="tangent"):
            call(dual)


@pytest.mark.parametrize("call,shape", [
    (lambda out: sequence.causal_conv(X, W, state_out=out), (1, 3, 16)), (lambda out: sequence.causal_conv(X, W, state=out, state_out=out), (1, 3, 16)),
    (lambda out: sequence.selective_scan(X, X, A, BC, BC, state=out, state_out=out), (1, 16, 8)),
    (lambda out: sequence.norm_residual(X, X, residual_out=out), (1, 2, 16)), (lambda out: sequence.norm_residual(out, X, residual_out=out), (1, 2, 16)),
    (lambda out: sequence.norm_residual(X, pre_weight=ONES, residual_out=out), (1, 2, 16)),
])
def test_what_is_written_in_place_is_seen_by_autograd(monkeypatch, call, shape):
    """An older graph that has saved the tensor says so in its backward pass, as after any operation in place."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(sequence, "_raw_stream", lambda index: None)
    for name in ("tae_causal_conv", "tae_selective_scan", "tae_norm_residual"):
        monkeypatch.setattr(sequence._lib.load(), name, lambda *args: 0)
    out, w = dev(torch.ones(shape)), torch.ones(shape, requires_grad=True)
    saved = (w * out.as_subclass(torch.Tensor)).sum()
    call(out)
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()


def test_a_tensor_that_is_only_read_keeps_its_version(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(sequence, "_raw_stream", lambda index: None)
    monkeypatch.setattr(sequence._lib.load(), "tae_norm_residual", lambda *args: 0)
    r = dev(torch.ones(1, 2, 16))
    assert sequence.norm_residual(r, pre_weight=ONES)[0] is r and r._version == 0
    assert sequence.norm_residual(r, pre_weight=ONES, residual_out=r)[0] is r and r._version == 0
    sequence.norm_residual(r, r, pre_weight=ONES)
    assert r._version == 0


@pytest.mark.parametrize("make,entry", [(C.conv, "tae_causal_conv"), (C.scan, "tae_selective_scan"), (C.int8, "tae_int8_linear")])
def test_reserved_fields_have_to_be_zero(make, entry):
    C.refused(getattr(_lib.load(), entry), make(), "reserved", reserved=1)
