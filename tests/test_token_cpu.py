"""CPU tier of the operators around the mixers: the oracle's gradients against differences, the C structs' layout, what
the C ABI and the Python entry points refuse, and the plans' workspaces."""

import ctypes
import math
import subprocess

import numpy as np
import pytest
import torch

import ssm_scan
from oracle import token_ref
from ssm_scan import _abi
from test_abi_cpu import HEADER


def test_struct_layouts(tmp_path):
    structs = {"ssm_rnorm_args": _abi.RnormArgs, "ssm_embed_args": _abi.EmbedArgs, "ssm_linear_args": _abi.LinearArgs,
               "ssm_sample_args": _abi.SampleArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines.append("return 0;}")
    (tmp_path / "l.c").write_text("\n".join(lines))
    subprocess.run(["gcc", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        cname, field, val = line.split()
        assert (ctypes.sizeof(structs[cname]) if field == "size" else getattr(structs[cname], field).offset) == int(val), line


# ---------------------------------------------------------------- the oracle
def differences(f, x, d, h=1e-6):
    """The directional derivative of f at x along d."""
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


def test_oracle_norm_gradients():
    g = torch.Generator().manual_seed(0)
    s, w, dy, ds, d, dw = (torch.randn(*sh, generator=g, dtype=torch.float64) for sh in ((3, 7), (7,), (3, 7), (3, 7), (3, 7), (7,)))
    _, grad, gw, _ = token_ref.norm(s, w, dy=dy, ds=ds)
    want = differences(lambda t: (token_ref.norm(t, w) * dy).sum() + (t * ds).sum(), s, d)
    assert abs(want - (grad * d).sum()) < 1e-7
    assert abs(differences(lambda t: (token_ref.norm(s, t) * dy).sum(), w, dw) - (gw * dw).sum()) < 1e-7


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_oracle_linear_gradients(act):
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*sh, generator=g, dtype=torch.float64) for sh in ((4, 5), (3, 5), (3,), (4, 3), (4, 3)))
    res = token_ref.linear(x, w, b, act, r, dy)
    want = (torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu if act else lambda t: t)(x @ w.t() + b) + r
    assert torch.allclose(res["y"], want, atol=1e-12)
    for name, t, grad in (("x", x, res["dx"]), ("w", w, res["dw"]), ("b", b, res["dbias"]), ("r", r, res["dresidual"])):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        ops = dict(x=x, w=w, b=b, r=r)

        def f(v):
            o = dict(ops, **{name: v})
            return (token_ref.linear(o["x"], o["w"], o["b"], act, o["r"])["y"] * dy).sum()
        assert abs(differences(f, t, d) - (grad * d).sum()) < 1e-7, name


def test_oracle_embedding():
    w = torch.randn(5, 3, dtype=torch.float64)
    tok = torch.tensor([[0, 4], [-1, 5], [4, 4]])
    dout = torch.randn(3, 2, 3, dtype=torch.float64)
    out, dw, _ = token_ref.embedding(tok, w, 2.0, dout)
    leaf = w.clone().requires_grad_()
    there = ((tok >= 0) & (tok < 5)).reshape(-1, 1)
    ref = 2.0 * leaf[tok.clamp(0, 4).reshape(-1)] * there
    assert torch.equal(out, ref.detach())
    assert torch.allclose(dw, torch.autograd.grad(ref, leaf, dout.reshape(6, 3))[0])


def test_oracle_sample_by_hand():
    logits = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]], dtype=torch.float64))

    def at(u, **kw):
        t, lp = token_ref.sample(logits, torch.tensor([u], dtype=torch.float64), **kw)
        return t[0], lp[0]

    assert [at(u)[0] for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [at(u, top_k=2)[0] for u in (0.0, 0.57, 0.58, 0.99)] == [1, 1, 3, 3]     # 4 : 3
    assert [at(u, top_p=0.65)[0] for u in (0.0, 0.57, 0.58)] == [1, 1, 3]
    assert [at(u, top_p=0.75)[0] for u in (0.43, 0.45, 0.66, 0.67)] == [1, 2, 2, 3]  # 4 : 2 : 3
    assert [at(u, min_p=0.6)[0] for u in (0.5, 0.6)] == [1, 3]
    assert at(0.9, temperature=0.0) == (1, 0.0)
    assert math.isclose(at(0.0, top_k=2)[1], math.log(4 / 7))
    assert token_ref.sample(torch.full((1, 3), -math.inf), torch.zeros(1))[0][0] == -1


# ---------------------------------------------------------------- what is refused
def rnorm(**kw):
    a = _abi.RnormArgs(rows=4, dim=8, dtype=_abi.BF16, res_dtype=_abi.BF16, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def embed(**kw):
    a = _abi.EmbedArgs(n=4, vocab=10, dim=8, dtype=_abi.F32, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def linear(**kw):
    t = _abi.Tensor(256, (ctypes.c_int64 * 3)(8, 1, 0))
    a = _abi.LinearArgs(m=4, n=8, k=8, dtype=_abi.BF16, x=t, weight=t)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def sample(**kw):
    a = _abi.SampleArgs(rows=4, vocab=10, dtype=_abi.F32, temperature=1.0, top_p=1.0, min_p=0.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("make,check,bad", [
    (rnorm, "ssm_rnorm_check", [dict(rows=0), dict(dim=0), dict(dim=16385), dict(dtype=_abi.F64), dict(res_dtype=_abi.F16), dict(eps=-1.0),
                                dict(eps=math.nan), dict(rows=1 << 40)]),
    (embed, "ssm_embed_check", [dict(n=0), dict(vocab=0), dict(dim=0), dict(dtype=_abi.F64), dict(scale=math.inf), dict(vocab=(1 << 27) + 1),
                                dict(n=1 << 40), dict(dim=1 << 24)]),
    (linear, "ssm_linear_check", [dict(m=0), dict(n=0), dict(k=0), dict(dtype=_abi.F32), dict(activation=3), dict(activation=-1),
                                  dict(m=(1 << 24) + 1), dict(m=1 << 20, n=1 << 15), dict(in8=1), dict(x=_abi.Tensor()),
                                  dict(weight=_abi.Tensor(256, (ctypes.c_int64 * 3)(8, 2, 0)))]),
    (sample, "ssm_sample_check", [dict(rows=0), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(dtype=_abi.F64), dict(temperature=-1.0),
                                  dict(temperature=math.nan), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=-0.1), dict(rows=1 << 31)]),
])
def test_checks(make, check, bad):
    fn = getattr(_abi.lib(), check)
    assert fn(ctypes.byref(make())) == _abi.OK
    assert fn(None) == _abi.EINVAL
    for kw in bad:
        assert fn(ctypes.byref(make(**kw))) == _abi.EINVAL, kw
        assert _abi.lib().ssm_last_error()


def test_launches_without_operands_or_workspace():
    """Refused before anything reaches the device."""
    lib = _abi.lib()
    t = _abi.Tensor(256, (ctypes.c_int64 * 3)(8, 1, 0))
    assert lib.ssm_rnorm_fwd(ctypes.byref(rnorm()), None) == _abi.EINVAL
    assert lib.ssm_rnorm_fwd(ctypes.byref(rnorm(x=t, q=t)), None) == _abi.EINVAL                      # no scale
    assert lib.ssm_rnorm_fwd(ctypes.byref(rnorm(x=t, residual=t, weight=256, out=t)), None) == _abi.EINVAL   # no sum
    assert lib.ssm_rnorm_bwd(ctypes.byref(rnorm(sum=t, dout=t, dx=t, weight=256, dweight=256)), None) == _abi.ESPACE
    assert lib.ssm_embed_fwd(ctypes.byref(embed()), None) == _abi.EINVAL
    assert lib.ssm_embed_bwd(ctypes.byref(embed(tokens=256, dout=t, dweight=256)), None) == _abi.ESPACE
    assert lib.ssm_embed_bwd(ctypes.byref(embed(tokens=256, dout=t, dweight=256, n=1 << 27)), None) == _abi.EINVAL
    assert lib.ssm_linear_fwd(ctypes.byref(linear()), None) == _abi.EINVAL
    assert lib.ssm_linear_fwd(ctypes.byref(linear(m=100, n=4096, k=4096, out=t)), None) == _abi.ESPACE   # splits of k
    assert lib.ssm_linear_bwd(ctypes.byref(linear(dout=t, activation=1)), None) == _abi.EINVAL          # no z
    assert lib.ssm_linear_bwd(ctypes.byref(linear(in8=1, x_scale=256, weight_scale=256, dout=t)), None) == _abi.EINVAL
    assert lib.ssm_sample(ctypes.byref(sample(logits=t)), None) == _abi.EINVAL
    assert lib.ssm_sample(ctypes.byref(sample(logits=t, u=256, token=256, logprob=256, vocab=100000)), None) == _abi.ESPACE


def test_workspaces():
    lib = _abi.lib()
    assert lib.ssm_rnorm_workspace_bytes(ctypes.byref(rnorm())) == 0
    assert lib.ssm_rnorm_workspace_bytes(ctypes.byref(rnorm(dweight=256))) >= 4 * 8 * 4
    assert lib.ssm_embed_workspace_bytes(ctypes.byref(embed(n=1))) > 0
    big = lib.ssm_embed_workspace_bytes(ctypes.byref(embed(n=1 << 20, vocab=1 << 17, dim=1024)))
    assert big < (1 << 20) * 1024 * 4      # below one gradient row a token: sums of whole pieces alone
    assert lib.ssm_sample_workspace_bytes(ctypes.byref(sample())) == 0
    assert lib.ssm_sample_workspace_bytes(ctypes.byref(sample(vocab=1 << 24, rows=3, top_k=5))) > 0
    aligned = linear(m=512, n=512, k=512)
    assert lib.ssm_linear_workspace_bytes(ctypes.byref(aligned)) >= 0
    odd = linear(m=512, n=512, k=511)      # rows that are copied
    assert lib.ssm_linear_workspace_bytes(ctypes.byref(odd)) >= 2 * 512 * 512 * 2


def test_there_is_no_cpu_path():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for call in (lambda: ssm_scan.add_rms_norm(x, x, w), lambda: ssm_scan.rms_norm_8bit(x, w), lambda: ssm_scan.quantize_rows(x),
                 lambda: ssm_scan.embedding(torch.zeros(2, dtype=torch.long), x), lambda: ssm_scan.linear_act(x.bfloat16(), x.bfloat16()),
                 lambda: ssm_scan.linear_8bit(x.to(torch.float8_e4m3fn), w[:2], x.to(torch.float8_e4m3fn), w[:2]),
                 lambda: ssm_scan.sample(x, w[:2])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_embedding_layers_on_the_cpu_stay_torchs():
    from ssm_scan import linear as lin
    layer = torch.nn.Embedding(5000, 4)
    idx = torch.randint(0, 5000, (7,))
    out = lin.embedding(layer, idx)
    assert torch.equal(out, layer(idx)) and torch.autograd.grad(out.sum(), layer.weight)[0].shape == (5000, 4)


def test_perf_cases_agree_with_the_oracle():
    """The definition of the draw, as the measured cases state it, on the CPU."""
    r = np.random.default_rng(0)
    logits = torch.from_numpy(r.normal(size=(20, 50)))
    u = torch.from_numpy(r.random(20))
    t, lp = token_ref.sample(logits, u, temperature=0.8, top_k=10, top_p=0.9)
    for b in range(20):
        w = torch.softmax(logits[b] / 0.8, 0)
        order = torch.argsort(w, descending=True)[:10]
        keep = order[: int((torch.cumsum(w[order], 0) < 0.9 * w[order].sum()).sum()) + 1].sort().values
        c = torch.cumsum(w[keep], 0)
        at = int((c <= u[b] * c[-1]).sum())
        assert t[b] == keep[at] and math.isclose(lp[b], float(torch.log(w[keep[at]] / c[-1])), rel_tol=1e-9)
