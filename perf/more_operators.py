"""What a language model does around its sequence mixers, as it is measured: the token embedding with its gradient,
the norm that takes the residual's addition along (with an 8-bit form), the linear layer with its epilogue (16 and
8 bits), and the draw of the next token.

listed() and draw() give cases, prepare() what a program holds before the call, run() one pass: with `own` through
ssm_scan's entry points, without it in elementary torch operations.  exact() gives the same outputs from the
definitions in float64, with the gradients written out by hand.

  embedding     out_i = scale weight[token_i]  (a zero row where token_i < 0: padding)
                dweight_v = scale sum over i with token_i = v of dout_i
  norm          s = x + residual, rounded to the residual's type;  y = s / sqrt(mean(s^2) + eps) weight
                8 bits: scale = max |y| / 448 per row (1 for a row of zeros), q = y / scale in e4m3
  linear        y = act(x W^T + bias) + residual;  8 bits: x = q scale and W = q scale per row
  sample        w_i = exp((l_i - max l) / T); kept are, in descending order of l (ties: the lower index first), the
                first top_k, of those the shortest prefix that holds top_p of their mass, of those all with w_i >= min_p;
                the token is the first kept index at which the running sum of kept w passes u times their sum
                (T = 0: the first of the order), and log(w / sum of kept w) its log probability
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
TOP8 = 448.0   # the largest e4m3 value


def listed():
    return [
        # the byte LM's training batch (B16 L512, d_model 256) in its own type
        dict(name="embed lm train", op="embed", train=True, n=8192, V=256, D=256, dtype="fp32", pad=False),
        # a subword vocabulary with an odd number of rows, padded batch, frequent tokens first: the gradient is dense
        dict(name="embed 50k train", op="embed", train=True, n=16384, V=50001, D=1024, dtype="bf16", pad=True),
        # a decode step of 64 streams: the norm in front of an 8-bit projection
        dict(name="norm8 decode", op="norm", mode="8bit", R=64, D=4096, dtype="bf16", wide=False, add=True),
        # every block of a larger layer's training batch
        dict(name="norm train 16k", op="norm", mode="train", R=16384, D=2048, dtype="bf16", wide=False, add=True),
        # the byte LM's training batch
        dict(name="norm train lm", op="norm", mode="train", R=8192, D=256, dtype="fp32", wide=False, add=True),
        # a token of one stream through an input projection
        dict(name="linear b1", op="linear", train=False, bits=16, M=1, N=4096, K=1024, dtype="bf16", act=None, bias=False,
             residual=False),
        # a token of 64 streams through 8-bit weights
        dict(name="linear8 b64", op="linear", train=False, bits=8, M=64, N=8192, K=4096, dtype="bf16", act="silu", bias=True,
             residual=False),
        # odd sizes in every dimension, everything on
        dict(name="linear odd train", op="linear", train=True, bits=16, M=1000, N=777, K=520, dtype="fp16", act="gelu", bias=True,
             residual=True),
        # the largest: a training batch through an expanding projection with its activation
        dict(name="linear train 8k", op="linear", train=True, bits=16, M=8192, N=8192, K=2048, dtype="bf16", act="silu", bias=True,
             residual=False),
        # a prompt through an 8-bit output projection, added to the residual stream
        dict(name="linear8 prefill", op="linear", train=False, bits=8, M=4096, N=4096, K=8192, dtype="bf16", act=None, bias=False,
             residual=True),
        # the byte LM's next token
        dict(name="sample b1", op="sample", B=1, V=256, dtype="fp32", rows=False, T=0.8, top_k=40, top_p=0.0, min_p=0.0),
        # a serving batch whose requests each have settings of their own
        dict(name="sample b64 128k", op="sample", B=64, V=131072, dtype="bf16", rows=True, T=0.0, top_k=0, top_p=0.0, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["embed", "norm", "linear", "linear", "sample"])
    if op == "embed":
        V, D = _log(rng, 30, 130000), rng.choice([64, 100, 256, 512, 1000, 1024, 2048])
        while V * D > 50001 * 1024:
            D //= 2
        return dict(op=op, train=rng.random() < 0.7, n=_log(rng, 1, 20000), V=V, D=D,
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), pad=rng.random() < 0.5)
    if op == "norm":
        D = rng.choice([64, 100, 256, 500, 768, 1024, 2048, 4096, 5120, 8192])
        mode = rng.choice(["train", "train", "infer", "8bit"])
        return dict(op=op, mode=mode, R=_log(rng, 1, min(20000, 16384 * 2048 // D)), D=D,
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), wide=rng.random() < 0.3, add=mode != "8bit" or rng.random() < 0.5)
    if op == "linear":
        bits, train = (8, False) if rng.random() < 0.4 else (16, rng.random() < 0.5)
        N, K = rng.choice([48, 200, 256, 515, 1000, 1024, 2048, 4096, 8192]), rng.choice([40, 256, 333, 512, 1000, 1024, 2048, 4096, 8192])
        return dict(op=op, train=train, bits=bits, M=_log(rng, 1, max(1, min(8192, (1 << 36) // (N * K)))), N=N, K=K,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), act=rng.choice([None, "silu", "gelu"]), bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    rows = rng.random() < 0.5
    V = _log(rng, 30, 131072)
    return dict(op=op, B=_log(rng, 1, max(1, min(256, (1 << 23) // V))), V=V, dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=rows,
                T=0.0 if rows else rng.choice([0.0, 0.6, 1.0, 1.3]), top_k=0 if rows else rng.choice([0, 1, 20, 1000]),
                top_p=0.0 if rows else rng.choice([0.0, 0.5, 0.95]), min_p=0.0 if rows else rng.choice([0.0, 0.05]))


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    def rand(*s):
        return torch.rand(*s, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] == "embed":
        n, V, D = case["n"], case["V"], case["D"]
        # text: the r-th most frequent token comes about 1/r as often as the first; ranks lie anywhere in the vocabulary
        rank = torch.exp(rand(n) * math.log(V + 1)).long().sub_(1).clamp_(0, V - 1)
        s["tokens"] = torch.randperm(V, generator=g, device="cuda")[rank]
        if case["pad"]:
            s["tokens"][rand(n) < 0.05] = -1
        s["weight"], s["scale"] = (0.02 * randn(V, D)).to(dt), math.sqrt(D)
        if case["train"]:
            s["weight"].requires_grad_()
            s["dout"] = randn(n, D).to(dt)
    elif case["op"] == "norm":
        R, D = case["R"], case["D"]
        s.update(x=randn(R, D).to(dt), weight=1 + 0.2 * randn(D),
                 residual=(2 * randn(R, D)).to(torch.float32 if case["wide"] else dt) if case["add"] else None)
        if case["mode"] == "train":
            s["dy"], s["ds"] = randn(R, D).to(dt), randn(R, D).to(s["residual"].dtype)
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_()
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x, w = randn(M, K), randn(N, K) / math.sqrt(K)
        if case["bits"] == 8:
            (s["x"], s["xs"]), (s["w"], s["ws"]) = _rows8(x), _rows8(w)
        else:
            s["x"], s["w"] = x.to(dt), w.to(dt)
        s["bias"] = (0.5 * randn(N)).to(dt) if case["bias"] else None
        s["residual"] = randn(M, N).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(M, N).to(dt)
            for name in ("x", "w", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_()
    else:
        B, V = case["B"], case["V"]
        # a few likely tokens over a broad floor, and some that a grammar forbids
        logits = 2.0 * randn(B, V) + 3.0 * rand(B, V).pow(20)
        logits[rand(B, V) < 0.02] = -math.inf
        logits[:, 0] = 0.0
        s.update(logits=logits.to(dt), u=rand(B))
        if case["rows"]:
            def choose(values, dtype):
                return torch.tensor(values, dtype=dtype, device="cuda")[torch.randint(len(values), (B,), generator=g, device="cuda")]
            s.update(T=choose([0.0, 0.5, 0.7, 1.0, 1.3], torch.float32), top_k=choose([0, 1, 40, 200, 5000], torch.int64),
                     top_p=choose([1.0, 0.5, 0.9, 0.99], torch.float32), min_p=choose([0.0, 0.0, 0.02], torch.float32))
        else:
            s.update(T=case["T"], top_k=case["top_k"] or None, top_p=case["top_p"] or None, min_p=case["min_p"] or None)
    return s


# ---------------------------------------------------------------- plain form
def _rows8(y):
    amax = y.abs().amax(-1)
    scale = torch.where(amax > 0, amax / TOP8, torch.ones_like(amax))
    return (y / scale[..., None]).to(torch.float8_e4m3fn), scale


def _act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) if act == "gelu" else z


def _grads(outs, douts, leaves):
    return torch.autograd.grad(outs, leaves, douts)


def _plain_embed(s, case):
    tokens, w = s["tokens"], s["weight"].detach()
    there = (tokens >= 0)[:, None]
    at = tokens.clamp(min=0)
    res = {"out": (w[at].float() * s["scale"] * there).to(w.dtype)}
    if case["train"]:
        d = torch.zeros(w.shape, device=w.device).index_add_(0, at, s["dout"].float() * s["scale"] * there)
        res["dweight"] = d.to(w.dtype)
    return res


def _plain_norm(s, case):
    train = case["mode"] == "train"
    x, w = s["x"].detach(), s["weight"].detach()
    t = x.float() + s["residual"].detach().float() if case["add"] else x.float()
    stored = t.to(s["residual"].dtype if case["add"] else x.dtype)
    t, w = stored.float().requires_grad_(train), w.clone().requires_grad_(train)
    y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w
    res = {"s": stored} if case["add"] else {}
    if case["mode"] == "8bit":
        res["q"], res["scale"] = _rows8(y)
        return res
    res["y"] = y.detach().to(x.dtype)
    if train:
        dt, dw = _grads([y], [s["dy"].float()], [t, w])
        dt = dt + s["ds"].float()
        res.update(dx=dt.to(x.dtype), dresidual=dt.to(stored.dtype), dweight=dw)
    return res


def _plain_linear(s, case):
    names = [n for n in ("x", "w", "bias", "residual") if s[n] is not None]
    f = {n: s[n].detach().float().requires_grad_(case["train"]) for n in names}
    z = f["x"] @ f["w"].t()
    if case["bits"] == 8:
        z = z * s["xs"][:, None] * s["ws"]
    if "bias" in f:
        z = z + f["bias"]
    y = _act(z, case["act"])
    if "residual" in f:
        y = y + f["residual"]
    res = {"y": y.detach().to(DTYPES[case["dtype"]])}
    if case["train"]:
        grads = _grads([y], [s["dy"].float()], [f[n] for n in names])
        res.update({"d" + n: d.to(s[n].dtype) for n, d in zip(names, grads)})
    return res


def _setting(v, off, B):
    """A setting per row, in float64."""
    if isinstance(v, torch.Tensor):
        return v.double()[:, None]
    return torch.full((B, 1), off if v is None else float(v), dtype=torch.float64, device="cuda")


def _plain_sample(s):
    logits, u = s["logits"].double(), s["u"].double()[:, None]
    B, V = logits.shape
    T, k, p, m = (_setting(s[n], off, B) for n, off in (("T", 1.0), ("top_k", 0.0), ("top_p", 1.0), ("min_p", 0.0)))
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    greedy = T == 0
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(greedy, torch.ones_like(T), T))
    place = torch.arange(V, device=logits.device)
    keep = (place < torch.where(k > 0, k, torch.full_like(k, V))) & (place < torch.where(greedy, 1, V))
    mass = torch.cumsum(w * keep, -1)
    before = torch.cat([mass.new_zeros(B, 1), mass[:, :-1]], 1)
    keep &= ((p >= 1) | (before < p * mass[:, -1:])) & (w >= m)
    kept = torch.zeros_like(w).scatter_(1, order.indices, w * keep)   # by index again
    run_sum = torch.cumsum(kept, -1)
    total = run_sum[:, -1:]
    token = (run_sum <= u * total).sum(-1, keepdim=True).clamp(max=V - 1)
    return {"token": token[:, 0], "logprob": torch.log(kept.gather(1, token) / total)[:, 0].float()}


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "embed":
        return _plain_embed(s, case)
    if case["op"] == "norm":
        return _plain_norm(s, case)
    return _plain_linear(s, case) if case["op"] == "linear" else _plain_sample(s)


# ---------------------------------------------------------------- the framework's calls
def _run_own(s, case):
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-ssm-benchmark_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ssm_scan
    op = case["op"]
    if op == "sample":
        token, logprob = ssm_scan.sample(s["logits"], s["u"], temperature=s["T"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "logprob": logprob}
    if op == "embed":
        out = ssm_scan.embedding(s["tokens"], s["weight"], scale=s["scale"])
        if not case["train"]:
            return {"out": out}
        return {"out": out.detach(), "dweight": _grads([out], [s["dout"]], [s["weight"]])[0]}
    if op == "norm":
        if case["mode"] == "8bit":
            r = ssm_scan.rms_norm_8bit(s["x"], s["weight"], residual=s["residual"], eps=EPS)
            return dict(zip(("q", "scale", "s"), r))
        y, t = ssm_scan.add_rms_norm(s["x"], s["residual"], s["weight"], eps=EPS)
        if case["mode"] == "infer":
            return {"y": y, "s": t}
        dx, dr, dw = _grads([y, t], [s["dy"], s["ds"]], [s["x"], s["residual"], s["weight"]])
        return {"y": y.detach(), "s": t.detach(), "dx": dx, "dresidual": dr, "dweight": dw}
    if case["bits"] == 8:
        return {"y": ssm_scan.linear_8bit(s["x"], s["xs"], s["w"], s["ws"], bias=s["bias"], activation=case["act"],
                                          residual=s["residual"], dtype=DTYPES[case["dtype"]])}
    y = ssm_scan.linear_act(s["x"], s["w"], bias=s["bias"], activation=case["act"], residual=s["residual"])
    if not case["train"]:
        return {"y": y}
    names = [n for n in ("x", "w", "bias", "residual") if s[n] is not None]
    res = {"y": y.detach()}
    res.update({"d" + n: d for n, d in zip(names, _grads([y], [s["dy"]], [s[n] for n in names]))})
    return res


# ---------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "embed":
        n, V, D = case["n"], case["V"], case["D"]
        moved, fl = 8 * n + min(n, V) * D * e + n * D * e, n * D
        if case["train"]:   # dout in, the whole gradient out
            moved, fl = moved + n * D * e + V * D * e, fl + 2 * n * D
        return {"bytes": moved, "flops": fl}
    if case["op"] == "norm":
        n, D = case["R"] * case["D"], case["D"]
        es = 4 if case["wide"] else e
        moved = n * e + (2 * n * es if case["add"] else 0) + 4 * D
        if case["mode"] == "8bit":
            return {"bytes": moved + n + 4 * case["R"], "flops": 8 * n}
        moved, fl = moved + n * e, 6 * n
        if case["mode"] == "train":   # dy and ds in; the input's and the residual's gradient (one where their types agree) and the weight's out
            moved, fl = moved + n * e + n * es + n * es + (n * e if es != e else 0) + 4 * D, fl + 12 * n
        return {"bytes": moved, "flops": fl}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        ei = case["bits"] // 8
        moved = (M * K + N * K) * ei + M * N * 2 * (1 + case["residual"]) + (2 * N if case["bias"] else 0)
        moved += 4 * (M + N) if case["bits"] == 8 else 0
        fl = 2 * M * N * K
        if case["train"]:   # dy in; dx, dw and the others' out
            moved, fl = moved + M * N * 2 + (M * K + N * K) * 2 + (2 * N if case["bias"] else 0), 3 * fl
        return {"bytes": moved, "flops": fl}
    return {"bytes": case["B"] * case["V"] * e + 16 * case["B"], "flops": 10 * case["B"] * case["V"]}


# ---------------------------------------------------------------- float64, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    types = {n: t.dtype for n, t in s.items() if isinstance(t, torch.Tensor)}
    s = {n: t.detach().double() if isinstance(t, torch.Tensor) and n != "tokens" else t for n, t in s.items()}
    if case["op"] == "embed":
        return _exact_embed(s, case)
    return _exact_norm(s, case, types) if case["op"] == "norm" else _exact_linear(s, case)


def _exact_embed(s, case):
    tokens, w = s["tokens"], s["weight"]
    rows = torch.cat([w, w.new_zeros(1, w.shape[1])])   # the last row is padding's
    res = {"out": s["scale"] * rows[tokens]}
    if case["train"]:
        order = torch.argsort(tokens)
        d = torch.zeros_like(rows)
        for part in order.split(2048):   # equal tokens lie together
            t, count = torch.unique_consecutive(tokens[part], return_counts=True)
            ends = torch.cumsum(s["dout"][part], 0)[torch.cumsum(count, 0) - 1]
            d[t] += torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1]))
        res["dweight"] = s["scale"] * d[:-1]
    return res


def _exact_norm(s, case, types):
    x, w = s["x"], s["weight"]
    total = x + s["residual"] if case["add"] else x
    t = total.to(types["residual" if case["add"] else "x"]).double()   # y is of the stored sum
    r = (t.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    y = t * r * w
    res = {"s": total} if case["add"] else {}
    if case["mode"] == "8bit":
        scale = y.abs().amax(-1) / TOP8
        scale[scale == 0] = 1.0
        res.update(scale=scale, q=(y / scale[:, None]).float().to(torch.float8_e4m3fn).double())
        return res
    res["y"] = y
    if case["mode"] == "train":
        h = s["dy"] * w
        d = s["ds"] + r * (h - t * r * r * (h * t).mean(-1, keepdim=True))
        res.update(dx=d, dresidual=d, dweight=(s["dy"] * t * r).sum(0))
    return res


def _exact_linear(s, case):
    x, w = s["x"], s["w"]
    if case["bits"] == 8:
        x, w = x * s["xs"][:, None], w * s["ws"][:, None]
    z = torch.mm(x, w.t())
    if case["bias"]:
        z += s["bias"]
    if case["act"] == "silu":
        gate = torch.special.expit(z)
        y, slope = z * gate, gate * (1 + z * (1 - gate))
    elif case["act"] == "gelu":
        gate = torch.special.ndtr(z)
        y, slope = z * gate, gate + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    res = {"y": y + s["residual"] if case["residual"] else y}
    if case["train"]:
        dz = s["dy"] * slope
        res.update(dx=torch.mm(dz, w), dw=torch.mm(dz.t().contiguous(), x))
        if case["bias"]:
            res["dbias"] = dz.sum(0)
        if case["residual"]:
            res["dresidual"] = s["dy"]
    return res


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()

    def setting(name, row, off):
        v = s[name]
        return off if v is None else float(v[row]) if isinstance(v, torch.Tensor) else float(v)

    tokens, logprobs = [], []
    for b in range(len(logits)):
        T, k, p, m = (setting(n, b, off) for n, off in (("T", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        order = np.lexsort((np.arange(logits.shape[1]), -logits[b]))
        order = order[:1] if T == 0 else order[:int(k)] if k else order
        w = np.exp((logits[b][order] - logits[b][order[0]]) / (T or 1.0))
        if p < 1:
            reach = int(np.argmax(np.cumsum(w) >= p * w.sum())) + 1
            order, w = order[:reach], w[:reach]
        order, w = order[w >= m], w[w >= m]
        back = np.argsort(order)
        order, w = order[back], w[back]
        at = min(int(np.searchsorted(np.cumsum(w), u[b] * w.sum(), side="right")), len(w) - 1)
        tokens.append(int(order[at]))
        logprobs.append(math.log(w[at] / w.sum()))
    return {"token": torch.tensor(tokens), "logprob": torch.tensor(logprobs, dtype=torch.float64)}
