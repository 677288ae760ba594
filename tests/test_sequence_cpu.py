"""The sequence operators' C entry points refuse bad arguments before anything is launched (no GPU here: a call that got through would
return a HIP error instead), and the argument structures are the same on both sides of the binding."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

from turboae_amd import _lib, sequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20            # never read: every call below is refused

STRUCTS = {"tae_conv_args": _lib.TaeConvArgs, "tae_scan_args": _lib.TaeScanArgs, "tae_norm_args": _lib.TaeNormArgs, "tae_int8_args": _lib.TaeInt8Args,
           "tae_logprobs_args": _lib.TaeLogprobsArgs}


def refused(fn, args, match, **change):
    for k, v in change.items():
        setattr(args, k, v)
    rc = fn(C.byref(args), None)
    message = _lib.load().tae_last_error().decode()
    assert rc == -1 and match in message, (rc, message)


def build(cls, **values):
    a = cls()
    a.struct_size = C.sizeof(cls)
    for k, v in values.items():
        setattr(a, k, v)
    return a


def conv():
    return build(_lib.TaeConvArgs, batch=1, len=4, channels=8, taps=4, act=6, x_batch=32, x_row=8, x=PTR, weight=PTR, y=PTR)


def scan():
    return build(_lib.TaeScanArgs, batch=1, len=4000, channels=8, states=16, x=PTR, dt=PTR, a=PTR, b=PTR, c=PTR, y=PTR, state_out=PTR)


def norm():
    return build(_lib.TaeNormArgs, batch=1, len=4, dim=8, gate_act=5, eps=1e-5, alpha=1.0, residual=PTR, block=PTR, residual_out=2 * PTR)


def int8():
    return build(_lib.TaeInt8Args, rows=40, inputs=32, outputs=4, x_row=32, weight_row=32, x=PTR, weight=PTR, weight_scale=PTR, y=PTR)


def logprobs():
    return build(_lib.TaeLogprobsArgs, token_bytes=8, rows=2, vocab=100000, top=4, logits_row=100000, logits=PTR, tokens=PTR, logp=PTR, entropy=PTR, top_ids=PTR, top_logp=PTR)


@pytest.mark.parametrize("make,entry,match,change", [
    (conv, "tae_causal_conv", "struct_size", dict(struct_size=8)), (conv, "tae_causal_conv", "dtype", dict(dtype=3)), (conv, "tae_causal_conv", "batch", dict(batch=0)),
    (conv, "tae_causal_conv", ">= 1", dict(len=0)), (conv, "tae_causal_conv", "taps", dict(taps=9)), (conv, "tae_causal_conv", "taps", dict(taps=0)),
    (conv, "tae_causal_conv", "act", dict(act=0)), (conv, "tae_causal_conv", "NULL", dict(weight=None)),
    (scan, "tae_selective_scan", "struct_size", dict(struct_size=0)), (scan, "tae_selective_scan", "dtype", dict(dtype=-1)), (scan, "tae_selective_scan", "states", dict(states=65)),
    (scan, "tae_selective_scan", ">= 1", dict(channels=0)), (scan, "tae_selective_scan", "2^30", dict(len=(1 << 30) + 1)), (scan, "tae_selective_scan", "NULL", dict(state_out=None)),
    (scan, "tae_selective_scan", "workspace", dict()), (scan, "tae_selective_scan", "workspace", dict(workspace=PTR + 4, workspace_bytes=1 << 40)),
    (scan, "tae_selective_scan", "workspace", dict(workspace=PTR, workspace_bytes=16)),
    (norm, "tae_norm_residual", "struct_size", dict(struct_size=1)), (norm, "tae_norm_residual", "dtype", dict(dtype=7)), (norm, "tae_norm_residual", "residual", dict(residual_dtype=1)),
    (norm, "tae_norm_residual", "dim", dict(dim=32769)), (norm, "tae_norm_residual", "product", dict(batch=1 << 20, len=1 << 20)), (norm, "tae_norm_residual", "eps", dict(eps=0.0)),
    (norm, "tae_norm_residual", "eps", dict(eps=float("nan"))), (norm, "tae_norm_residual", "gate_act", dict(gate_act=3)), (norm, "tae_norm_residual", "NULL", dict(residual=None)),
    (norm, "tae_norm_residual", "needs residual_out", dict(residual_out=None)), (norm, "tae_norm_residual", "need a block", dict(block=None, gate=PTR)),
    (norm, "tae_norm_residual", "its weight", dict(pre_bias=PTR)), (norm, "tae_norm_residual", "come together", dict(normed=PTR)),
    (norm, "tae_norm_residual", "nothing to write", dict(block=None, residual_out=None)), (norm, "tae_norm_residual", "in-place", dict(residual_out=PTR, out_row=16)),
    (int8, "tae_int8_linear", "struct_size", dict(struct_size=1)), (int8, "tae_int8_linear", "dtype", dict(dtype=3)), (int8, "tae_int8_linear", "131072", dict(inputs=131073)),
    (int8, "tae_int8_linear", "rows", dict(rows=0)), (int8, "tae_int8_linear", "NULL", dict(y=None)), (int8, "tae_int8_linear", "16-byte", dict(weight=PTR + 8)),
    (int8, "tae_int8_linear", "16-byte", dict(weight_row=40)), (int8, "tae_int8_linear", "16-byte", dict(weight_row=16)), (int8, "tae_int8_linear", "workspace", dict()),
    (logprobs, "tae_token_logprobs", "struct_size", dict(struct_size=1)), (logprobs, "tae_token_logprobs", "dtype", dict(dtype=9)), (logprobs, "tae_token_logprobs", "vocab", dict(vocab=0)),
    (logprobs, "tae_token_logprobs", "2^21", dict(vocab=(1 << 21) + 1)), (logprobs, "tae_token_logprobs", "top", dict(top=33)), (logprobs, "tae_token_logprobs", "token_bytes", dict(token_bytes=2)),
    (logprobs, "tae_token_logprobs", "NULL", dict(tokens=None)), (logprobs, "tae_token_logprobs", "top needs", dict(top_ids=None)),
    (logprobs, "tae_token_logprobs", "aligned", dict(logits=PTR + 2)), (logprobs, "tae_token_logprobs", "workspace", dict()),
    (conv, "tae_causal_conv", "aligned", dict(dtype=1, x=PTR + 1)), (conv, "tae_causal_conv", "aligned", dict(weight=PTR + 2)), (conv, "tae_causal_conv", "aligned", dict(state_out=PTR + 2)),
    (scan, "tae_selective_scan", "aligned", dict(dtype=2, z=PTR + 1)), (scan, "tae_selective_scan", "aligned", dict(state_out=PTR + 2)), (scan, "tae_selective_scan", "aligned", dict(lengths=PTR + 1)),
    (norm, "tae_norm_residual", "aligned", dict(block=PTR + 2)), (norm, "tae_norm_residual", "aligned", dict(scale=PTR + 1)), (norm, "tae_norm_residual", "subnormal", dict(eps=1e-40)),
    (int8, "tae_int8_linear", "aligned", dict(x=PTR + 2, workspace=PTR, workspace_bytes=1 << 20)), (int8, "tae_int8_linear", "aligned", dict(bias=PTR + 2, workspace=PTR, workspace_bytes=1 << 20)),
    (logprobs, "tae_token_logprobs", "aligned", dict(top_ids=PTR + 4)), (logprobs, "tae_token_logprobs", "too many rows", dict(rows=(1 << 31) - 1, vocab=1 << 21, workspace=PTR, workspace_bytes=1 << 62)),
])
def test_bad_arguments_are_refused(make, entry, match, change):
    refused(getattr(_lib.load(), entry), make(), match, **change)


def test_quantize_refuses():
    q = _lib.load().tae_quantize_int8
    good = dict(dtype=0, x=PTR, x_row=32, rows=2, cols=32, q=PTR, q_row=32, scale=PTR)
    for match, change in (("dtype", dict(dtype=5)), ("NULL", dict(x=None)), ("NULL", dict(scale=None)), ("rows", dict(rows=0)), ("cols", dict(cols=0)), ("16-byte", dict(q_row=40)),
                          ("16-byte", dict(q_row=16)), ("16-byte", dict(q=PTR + 1))):
        a = {**good, **change}
        assert q(a["dtype"], a["x"], a["x_row"], a["rows"], a["cols"], a["q"], a["q_row"], a["scale"], None) == -1
        assert match in _lib.load().tae_last_error().decode()


def test_workspaces_are_sized_without_tensors():
    lib = _lib.load()
    a = int8()
    assert lib.tae_int8_linear_workspace(C.byref(a)) >= 40 * 32 + 160
    a.rows = 2
    assert lib.tae_int8_linear_workspace(C.byref(a)) == 0                        # few rows are quantised where they are used
    assert lib.tae_int8_linear_workspace(C.byref(build(_lib.TaeInt8Args, rows=0, inputs=4, outputs=4))) == 0
    assert lib.tae_selective_scan_workspace(C.byref(scan())) > 0
    one = scan()
    one.len = 1
    assert lib.tae_selective_scan_workspace(C.byref(one)) == 0
    assert lib.tae_token_logprobs_workspace(C.byref(logprobs())) >= 2 * 16
    for fn, cls in ((lib.tae_selective_scan_workspace, _lib.TaeScanArgs), (lib.tae_token_logprobs_workspace, _lib.TaeLogprobsArgs)):
        assert fn(C.byref(cls())) == 0 and fn(None) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(1, 2, 4)
    with pytest.raises(_lib.TurboAEError, match="no CPU fallback"):
        sequence.causal_conv(x, torch.zeros(4, 2))
    with pytest.raises(_lib.TurboAEError, match="no CPU fallback"):
        sequence.token_logprobs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64))


def test_argument_structures_match_the_header(tmp_path):
    """Field names and order from the header, sizes and offsets from a C compiler."""
    with open(os.path.join(ROOT, "include", "turboae_hip.h")) as fh:
        text = fh.read()
    for name, cls in STRUCTS.items():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [re.sub(r"[\s\*]", "", f) for line in body.split(";") if line.strip() for f in re.sub(r"^\s*(const\s+)?\w+", "", line).split(",")]
        assert fields == [f for f, _ in cls._fields_], name
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = "".join('printf("%%zu%s\\n", sizeof(%s)%s);' % (" %zu" * len(cls._fields_), n, "".join(", offsetof(%s, %s)" % (n, f) for f, _ in cls._fields_)) for n, cls in STRUCTS.items())
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "turboae_hip.h"\nint main(void) {%s return 0;}\n' % lines)
    exe = tmp_path / "s"
    subprocess.check_call([cc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60, check=True).stdout.splitlines()
    for line, cls in zip(out, STRUCTS.values()):
        assert [int(v) for v in line.split()] == [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
