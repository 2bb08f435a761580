"""CPU tier of the gated delta rule and the grouped norm: the float64 oracles' hand-written gradients
against differences and autograd, the argument structs' layout, and every refusal of the C ABI and of
the Python entry points (which are made before anything is launched)."""

import ctypes
import os
import subprocess

import pytest
import torch

from oracle import delta_ref
import ssm_scan
from ssm_scan import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def inputs(B=2, L=9, Hk=2, H=4, Dk=5, Dv=3, seed=0):
    r = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=r, dtype=torch.float64)

    return dict(q=rn(B, L, Hk, Dk), k=rn(B, L, Hk, Dk), v=rn(B, L, H, Dv), g=-rn(B, L, H).abs(),
                beta=torch.sigmoid(rn(B, L, H)), h0=rn(B, H, Dk, Dv)), rn(B, L, H, Dv), rn(B, H, Dk, Dv)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_delta_oracle_gradient_matches_differences(qk_norm):
    """Central differences with step 1e-5 are off by about 1e-10 (curvature) + 1e-11 (float64 noise) of
    the loss's terms: 1e-7 of the gradient's size is allowed."""
    args, do, dl = inputs()
    _, _, grads = delta_ref.delta(**args, qk_norm=qk_norm, dout=do, dlast=dl)

    def loss(a):
        o, last = delta_ref.delta(**a, qk_norm=qk_norm)
        return ((o * do).sum() + (last * dl).sum()).item()

    r = torch.Generator().manual_seed(5)
    for name, t in args.items():
        d = torch.randn(t.shape, generator=r, dtype=torch.float64)
        e = 1e-5
        diff = (loss({**args, name: t + e * d}) - loss({**args, name: t - e * d})) / (2 * e)
        want = (grads[name] * d).sum().item()
        assert abs(diff - want) < 1e-7 * grads[name].norm().item() * d.norm().item(), name


@pytest.mark.parametrize("mode", ["gate", "silu", None])
@pytest.mark.parametrize("center", [False, True])
def test_group_norm_oracle_gradient_matches_autograd(mode, center):
    r = torch.Generator().manual_seed(1)
    x, gate, dy = (torch.randn(7, 12, generator=r, dtype=torch.float64) for _ in range(3))
    w, b = (torch.randn(12, generator=r, dtype=torch.float64) for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, b, gate)]
    xg = x.unflatten(-1, (3, 4))
    xg = xg - xg.mean(-1, keepdim=True) if center else xg
    z = (xg / (xg.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()).flatten(-2) * w + b
    y = z * torch.nn.functional.silu(gate) if mode == "gate" else torch.nn.functional.silu(z) if mode else z
    want = torch.autograd.grad(y, leaves, dy, allow_unused=True)
    got_y, got = delta_ref.group_norm(x, 3, w, b, gate if mode == "gate" else None, "silu" if mode == "silu" else None,
                                      center, dout=dy)
    torch.testing.assert_close(got_y, y.detach(), rtol=1e-12, atol=1e-12)
    for n, d in zip(("x", "weight", "bias", "gate"), want):
        if d is not None:
            torch.testing.assert_close(got[n], d, rtol=1e-11, atol=1e-11)


def test_ctypes_layout_matches_c_header(tmp_path):
    structs = {"ssm_delta_args": _abi.DeltaArgs, "ssm_delta_step_args": _abi.DeltaStepArgs, "ssm_gnorm_args": _abi.GnormArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT}/include/ssm_scan.h"', "int main(void){"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    for line in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, field, val = line.split()
        py = structs[cname]
        assert (ctypes.sizeof(py) if field == "size" else getattr(py, field).offset) == int(val), line


def delta_args(step=False, **kw):
    a = _abi.DeltaStepArgs() if step else _abi.DeltaArgs()
    vals = dict(batch=2, key_heads=2, heads=4, key_dim=64, value_dim=64, dtype=_abi.BF16, scale=0.125)
    vals.update(kw)
    drop = vals.pop("drop", ())
    if not step:
        vals.setdefault("seqlen", 100)
    for n, v in vals.items():
        setattr(a, n, v)
    t = torch.zeros(1)
    for n in ("q", "k", "v", "g", "beta", "out"):
        if n not in drop:
            setattr(a, n, _abi.Tensor(t.data_ptr(), (ctypes.c_int64 * 3)(1, 1, 1)))
    if step and "h" not in drop:
        a.h = t.data_ptr()
    a._keep = t
    return a


REFUSED = [dict(dtype=_abi.F64), dict(dtype=9), dict(batch=0), dict(heads=0), dict(key_heads=0), dict(key_dim=0), dict(value_dim=0),
           dict(key_dim=129), dict(heads=3), dict(scale=float("inf")), dict(scale=float("nan")), dict(batch=1 << 31, heads=1 << 20),
           dict(drop=("q",)), dict(drop=("k",)), dict(drop=("v",)), dict(drop=("g",)), dict(drop=("beta",))]


@pytest.mark.parametrize("kw", REFUSED + [dict(seqlen=0), dict(seqlen=1 << 32), dict(batch=1 << 20, seqlen=1 << 20)])
def test_delta_refusals(kw):
    a = delta_args(**kw)
    with pytest.raises(ValueError):
        _abi.check(_abi.lib().ssm_delta_check(ctypes.byref(a)), "ssm_delta")
    assert _abi.lib().ssm_delta_saved_bytes(ctypes.byref(a)) == -1
    assert _abi.lib().ssm_delta_fwd_workspace_bytes(ctypes.byref(a)) == -1
    assert _abi.lib().ssm_delta_bwd_workspace_bytes(ctypes.byref(a)) == -1


@pytest.mark.parametrize("kw", REFUSED + [dict(drop=("h",)), dict(drop=("out",))])
def test_delta_step_refusals(kw):
    with pytest.raises(ValueError):
        _abi.check(_abi.lib().ssm_delta_step_check(ctypes.byref(delta_args(step=True, **kw))), "ssm_delta_step")


def test_delta_launches_refuse_before_the_device():
    """Missing outputs, a missing or small workspace and a missing saved buffer are host errors."""
    lib, a = _abi.lib(), delta_args()
    assert lib.ssm_delta_check(ctypes.byref(a)) == 0
    assert lib.ssm_delta_fwd(ctypes.byref(a), None) == _abi.ESPACE
    a.workspace, a.workspace_bytes = a.q.data, lib.ssm_delta_fwd_workspace_bytes(ctypes.byref(a)) - 1
    assert lib.ssm_delta_fwd(ctypes.byref(a), None) == _abi.ESPACE
    assert lib.ssm_delta_bwd(ctypes.byref(a), None) == _abi.EINVAL and b"saved" in lib.ssm_last_error()
    a.saved = a.q.data
    for n in ("dout", "dq", "dk", "dv", "dg", "dbeta"):
        assert lib.ssm_delta_bwd(ctypes.byref(a), None) == _abi.EINVAL and n.encode() in lib.ssm_last_error()
        setattr(a, n, a.q)
    assert lib.ssm_delta_bwd(ctypes.byref(a), None) == _abi.ESPACE
    a = delta_args(drop=("out",))
    assert lib.ssm_delta_fwd(ctypes.byref(a), None) == _abi.EINVAL and b"out" in lib.ssm_last_error()


def gnorm_args(**kw):
    a = _abi.GnormArgs()
    vals = dict(rows=10, groups=4, group_size=32, dtype=_abi.F32, eps=1e-5)
    vals.update(kw)
    drop, stride = vals.pop("drop", ()), vals.pop("stride", 1)
    for n, v in vals.items():
        setattr(a, n, v)
    t = torch.zeros(1)
    for n in ("x", "gate", "out", "dout", "dx", "dgate"):
        if n not in drop:
            setattr(a, n, _abi.Tensor(t.data_ptr(), (ctypes.c_int64 * 3)(128, stride, 0)))
    a._keep = t
    return a


@pytest.mark.parametrize("kw", [dict(rows=0), dict(groups=0), dict(group_size=0), dict(group_size=1025), dict(dtype=_abi.F64),
                                dict(activation=3), dict(activation=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(drop=("x",)),
                                dict(activation=2, drop=("gate",)), dict(stride=2), dict(rows=1 << 31),
                                dict(rows=1 << 30, groups=2)])
def test_group_norm_refusals(kw):
    a = gnorm_args(**kw)
    with pytest.raises(ValueError):
        _abi.check(_abi.lib().ssm_gnorm_check(ctypes.byref(a)), "ssm_gnorm")
    assert _abi.lib().ssm_gnorm_workspace_bytes(ctypes.byref(a)) == -1


def test_group_norm_launches_refuse_before_the_device():
    lib = _abi.lib()
    assert lib.ssm_gnorm_fwd(ctypes.byref(gnorm_args(drop=("out",))), None) == _abi.EINVAL
    for n in ("dout", "dx", "dgate"):
        assert lib.ssm_gnorm_bwd(ctypes.byref(gnorm_args(activation=2, drop=(n,))), None) == _abi.EINVAL
    a = gnorm_args(activation=2)
    a.dweight = a.x.data
    assert lib.ssm_gnorm_bwd(ctypes.byref(a), None) == _abi.ESPACE


def test_python_entry_points_need_gpu_tensors():
    a, _, _ = inputs()
    a = {n: t.float() for n, t in a.items()}
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_rule(**a)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_step(a["h0"], *(a[n][:, 0] for n in ("q", "k", "v", "g", "beta")))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.group_norm(torch.zeros(3, 8), 2)
    with pytest.raises(ValueError, match="activation"):
        ssm_scan.group_norm(torch.zeros(3, 8), 2, activation="relu")
    with pytest.raises(ValueError, match="exclude"):
        ssm_scan.group_norm(torch.zeros(3, 8), 2, gate=torch.zeros(3, 8), activation="silu")
