"""The operators of dpvo_amd.blocks as they are measured: gated feed-forward blocks and the norms around them, in a plain form (elementary torch
operations in 32 bits, rounded once at the end) and, where `own` is true, as calls of the framework.

A case's "op" is
  "ff"     y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd                                     blocks.gated_feed_forward
  "block"  y = x + sigmoid(x Wg^T + bg) * (relu(x W1^T + b1) W2^T + b2)                          blocks.gated_residual (the update operator's)
  "norm"   s = x + scale * act(gate) * post(f);  h = norm(s)                                    blocks.residual_norm
and with "train" a pass returns the outputs and the gradients of every input and parameter.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token through a feed-forward block: latency, the weights' bytes
        {"name": "ff_token", "op": "ff", "dtype": "bf16", "M": 1, "K": 1024, "F": 4096, "act": "silu", "bias": False, "train": False},
        # a short ragged batch with biases
        {"name": "ff_ragged", "op": "ff", "dtype": "f16", "M": 333, "K": 768, "F": 2048, "act": "gelu", "bias": True, "train": False},
        # a training step's ordinary block
        {"name": "ff_train", "op": "ff", "dtype": "bf16", "M": 4096, "K": 1024, "F": 4096, "act": "silu", "bias": False, "train": True},
        # the largest training step
        {"name": "ff_train_large", "op": "ff", "dtype": "bf16", "M": 8192, "K": 4096, "F": 8192, "act": "silu", "bias": False, "train": True},
        # odd sizes in 32 bits: the 882 correlation features of an edge, an odd hidden width
        {"name": "ff_train_odd_f32", "op": "ff", "dtype": "f32", "M": 1237, "K": 882, "F": 385, "act": "gelu_tanh", "bias": True, "train": True},
        # the update operator's gated block on one frame's patches
        {"name": "block_patches", "op": "block", "dtype": "f16", "M": 96, "K": 384, "bias": True, "train": False},
        # ... on the steady state's edges (45 312 of them)
        {"name": "block_edges", "op": "block", "dtype": "f16", "M": 45312, "K": 384, "bias": True, "train": False},
        # ... trained on them
        {"name": "block_edges_train", "op": "block", "dtype": "f16", "M": 45312, "K": 384, "bias": True, "train": True},
        # ... in 32 bits, on a window's edges (served only: where 32 bits leave the sign of a ReLU's input open, its derivative is either 0 or 1)
        {"name": "block_f32", "op": "block", "dtype": "f32", "M": 9216, "K": 384, "bias": True, "train": False},
        # one token's norms and residual
        {"name": "norm_token", "op": "norm", "dtype": "bf16", "stream": "bf16", "M": 1, "K": 1024, "groups": 1, "gate": "identity", "kind": "rms", "post": "rms",
         "scale": 1.0, "train": False},
        # the tail of one gated block and the LayerNorm before the next, on the edges: 32-bit hidden state, 16-bit branch
        {"name": "norm_edges", "op": "norm", "dtype": "f16", "stream": "f32", "M": 45312, "K": 384, "groups": 45312, "gate": "sigmoid", "kind": "layer", "post": "none",
         "scale": 1.0, "train": False},
        # a wide block's training step, gated for each of four sequences
        {"name": "norm_train_wide", "op": "norm", "dtype": "bf16", "stream": "bf16", "M": 8192, "K": 4096, "groups": 4, "gate": "identity", "kind": "rms", "post": "rms",
         "scale": 0.5, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """a width: mostly a multiple of 64, as models have them, sometimes any number"""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["ff", "ff", "block", "norm"])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    train = rng.random() < 0.5
    if op == "norm":
        K = _size(rng, 64, 8192)
        M = _log(rng, 1, max(2, min(45312, 33554432 // K)))
        groups = rng.choice([1, M, M, 4])
        M = max(8, M // 4 * 4) if groups == 4 else M
        return {"op": op, "dtype": dtype, "stream": rng.choice([dtype, dtype, "f32"]), "M": M, "K": K, "groups": groups, "gate": rng.choice(["identity", "sigmoid"]),
                "kind": rng.choice(["layer", "rms"]), "post": rng.choice(["none", "layer", "rms"]), "scale": rng.choice([1.0, 0.5]), "train": train}
    most = 2.0e10 if dtype == "f32" else 2.0e11          # M * K * F: a 32-bit product runs at a sixteenth of the rate
    if op == "block":
        K = _size(rng, 64, 1024)
        M = _log(rng, 1, min(45312, most / (K * K)))
        return {"op": op, "dtype": dtype, "M": M, "K": K, "bias": rng.random() < 0.7, "train": train and dtype != "f32"}
    K, F = _size(rng, 64, 4096), _size(rng, 64, 8192)
    M = _log(rng, 1, min(16384, most / (K * F)))
    return {"op": op, "dtype": dtype, "M": M, "K": K, "F": F, "act": rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid"] + ([] if dtype == "f32" and train else ["relu"])), "bias": rng.random() < 0.3,
            "train": train}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, M, K = TYPES[case["dtype"]], case["M"], case["K"]
    train = case["train"]

    def normal(*shape, dtype=dt, scale=1.0, mean=0.0, leaf=True):
        t = (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)
        return t.requires_grad_(train and leaf)

    def layer(n, k):                                      # a Linear's usual initial values
        w = ((torch.rand(n, k, generator=g, device="cuda") * 2 - 1) / math.sqrt(k)).to(dt).requires_grad_(train)
        b = ((torch.rand(n, generator=g, device="cuda") * 2 - 1) / math.sqrt(k)).to(dt).requires_grad_(train) if case["bias"] else None
        return w, b

    s = {"case": case}
    if case["op"] == "ff":
        s["x"] = normal(M, K)
        s["wg"], s["bg"] = layer(case["F"], K)
        s["wu"], s["bu"] = layer(case["F"], K)
        s["wd"], s["bd"] = layer(K, case["F"])
        s["leaves"] = ["x", "wg", "wu", "wd"] + (["bg", "bu", "bd"] if case["bias"] else [])
        s["dy"] = normal(M, K, scale=0.1, leaf=False) if train else None
    elif case["op"] == "block":
        s["x"] = normal(M, K)
        for n in ("g", "1", "2"):
            s["w" + n], s["b" + n] = layer(K, K)
        s["leaves"] = ["x", "wg", "w1", "w2"] + (["bg", "b1", "b2"] if case["bias"] else [])
        s["dy"] = normal(M, K, scale=0.1, leaf=False) if train else None
    else:
        st = TYPES[case["stream"]]
        s["x"] = normal(M, K, dtype=st, scale=2.0, mean=0.25)
        s["f"] = normal(M, K)
        s["gate"] = normal(*([K] if case["groups"] == 1 else [case["groups"], 1, K] if case["groups"] < M else [M, K]))
        s["w"] = normal(K, dtype=st, scale=0.1, mean=1.0)
        s["b"] = normal(K, dtype=st, scale=0.1) if case["kind"] == "layer" else None
        s["pw"] = normal(K, dtype=st, scale=0.1, mean=1.0) if case["post"] != "none" else None
        s["pb"] = normal(K, dtype=st, scale=0.1) if case["post"] == "layer" else None
        if 1 < case["groups"] < M:                        # sequences of equal length, one gate each
            for n in ("x", "f"):
                s[n] = s[n].detach().view(case["groups"], M // case["groups"], K).requires_grad_(train)
        s["leaves"] = [n for n in ("x", "f", "gate", "w", "b", "pw", "pb") if s[n] is not None]
        s["ds"] = normal(*s["x"].shape, dtype=st, scale=0.1, leaf=False) if train else None
        s["dh"] = normal(*s["x"].shape, scale=0.1, leaf=False) if train else None
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _act(name, z):
    if name == "identity":
        return z
    if name == "relu":
        return z * (z > 0)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))


def _proj(x, w, b):
    y = x @ w.t()
    return y if b is None else y + b


def _norm(x, kind, w, b):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-3) * w
    return y if b is None else y + b


def _plain(s):
    c = s["case"]
    v = {k: t.float() if torch.is_tensor(t) else t for k, t in s.items() if k not in ("case", "leaves")}
    if c["op"] == "ff":
        h = _act(c["act"], _proj(v["x"], v["wg"], v["bg"])) * _proj(v["x"], v["wu"], v["bu"])
        return [_proj(h, v["wd"], v["bd"]).to(s["x"].dtype)]
    if c["op"] == "block":
        t = _act("relu", _proj(v["x"], v["w1"], v["b1"]))
        return [(v["x"] + _act("sigmoid", _proj(v["x"], v["wg"], v["bg"])) * _proj(t, v["w2"], v["b2"])).to(s["x"].dtype)]
    f = v["f"] if c["post"] == "none" else _norm(v["f"], c["post"], v["pw"], v["pb"])
    y = v["x"] + c["scale"] * _act(c["gate"], v["gate"]) * f
    return [y.to(s["x"].dtype), _norm(y, c["kind"], v["w"], v["b"]).to(s["f"].dtype)]


def _framework(s):
    from dpvo_amd import blocks
    c = s["case"]
    if c["op"] == "ff":
        return [blocks.gated_feed_forward(s["x"], s["wg"], s["wu"], s["wd"], s["bg"], s["bu"], s["bd"], activation=c["act"])]
    if c["op"] == "block":
        return [blocks.gated_residual(s["x"], s["wg"], s["bg"], s["w1"], s["b1"], s["w2"], s["b2"])]
    return list(blocks.residual_norm(s["x"], s["f"], s["w"], s["b"], norm=c["kind"], eps=1e-3, gate=s["gate"], gate_activation=c["gate"], scale=c["scale"],
                                     post_norm=None if c["post"] == "none" else c["post"], post_weight=s["pw"], post_bias=s["pb"], out_dtype=s["f"].dtype))


def run(s):
    if not s["case"]["train"]:
        with torch.no_grad():
            return _framework(s) if own else _plain(s)
    outs = _framework(s) if own else _plain(s)
    up = [s["dy"]] if s["case"]["op"] != "norm" else [s["ds"], s["dh"]]
    grads = torch.autograd.grad(outs, [s[n] for n in s["leaves"]], up)
    return [o.detach() for o in outs] + list(grads)


def work(case):
    M, K, n = case["M"], case["K"], BYTES[case["dtype"]]
    if case["op"] == "norm":
        m = BYTES[case["stream"]]
        G = case["groups"]
        fwd = M * K * (m + n) + G * K * n + M * K * (m + n)                    # x, f, gate in; s, h out
        bwd = M * K * (m + n) + M * K * (m + n) + G * K * n                    # ds, dh in; dx, df, dgate out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": M * K * (20 + (40 if case["train"] else 0))}
    F = case["F"] if case["op"] == "ff" else K
    weights = 3 * K * F * n
    flops = 6 * M * K * F
    if case["train"]:
        return {"bytes": 2 * weights + 4 * M * K * n, "flops": 3 * flops}     # x, dy in, y, dx out; weights in, their gradients out
    return {"bytes": weights + 2 * M * K * n, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def _act64(name, z):
    """value and derivative"""
    one = torch.ones_like(z)
    if name == "identity":
        return z, one
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name in ("sigmoid", "silu"):
        p = torch.sigmoid(z)
        return (p, p * (1 - p)) if name == "sigmoid" else (z * p, p + z * p * (1 - p))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return z * (1 + t) / 2, (1 + t) / 2 + z * (1 - t * t) / 2 * k * (1 + 3 * 0.044715 * z * z)


def _norm64(x, kind):
    """the normalised rows and their rows' factor"""
    if kind == "layer":
        r = (x.var(-1, unbiased=False, keepdim=True) + 1e-3).rsqrt()
        return (x - x.mean(-1, keepdim=True)) * r, r
    r = (x.pow(2).mean(-1, keepdim=True) + 1e-3).rsqrt()
    return x * r, r


def _norm64_back(d, xh, r, kind):
    d = d - xh * (d * xh).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0)
    return d * r


def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double() if torch.is_tensor(t) else t for k, t in s.items() if k not in ("case", "leaves")}
    train = case["train"]
    b0 = lambda b: 0 if b is None else b  # noqa: E731
    if case["op"] == "ff":
        x = v["x"]
        g, u = x.mm(v["wg"].T) + b0(v["bg"]), x.mm(v["wu"].T) + b0(v["bu"])
        a, da = _act64(case["act"], g)
        h = a * u
        out = [h.mm(v["wd"].T) + b0(v["bd"])]
        if train:
            dy = v["dy"]
            dh = dy.mm(v["wd"])
            dg, du = dh * u * da, dh * a
            d = {"x": dg.mm(v["wg"]) + du.mm(v["wu"]), "wg": dg.T.mm(x), "wu": du.T.mm(x), "wd": dy.T.mm(h), "bg": dg.sum(0), "bu": du.sum(0), "bd": dy.sum(0)}
    elif case["op"] == "block":
        x = v["x"]
        p = x.mm(v["w1"].T) + b0(v["b1"])
        t, dt = _act64("relu", p)
        a, da = _act64("sigmoid", x.mm(v["wg"].T) + b0(v["bg"]))
        r = t.mm(v["w2"].T) + b0(v["b2"])
        out = [x + a * r]
        if train:
            dy = v["dy"]
            dg, dr = dy * r * da, dy * a
            dp = dr.mm(v["w2"]) * dt
            d = {"x": dy + dg.mm(v["wg"]) + dp.mm(v["w1"]), "wg": dg.T.mm(x), "w1": dp.T.mm(x), "w2": dr.T.mm(t), "bg": dg.sum(0), "b1": dp.sum(0), "b2": dr.sum(0)}
    else:
        shape = s["x"].shape
        fh, fr = (v["f"], None) if case["post"] == "none" else _norm64(v["f"], case["post"])
        f = fh if fr is None else fh * v["pw"] + b0(v["pb"])
        a, da = _act64(case["gate"], v["gate"])
        y = v["x"] + case["scale"] * a * f
        yh, r = _norm64(y, case["kind"])
        out = [y, yh * v["w"] + b0(v["b"])]
        if train:
            rows = lambda t: t.reshape(-1, shape[-1])  # noqa: E731
            dy = v["ds"] + _norm64_back(v["dh"] * v["w"], yh, r, case["kind"])
            q = case["scale"] * dy
            df = q * a
            dgate = q * f * da
            dgate = dgate.sum_to_size(v["gate"].shape) if case["groups"] < case["M"] or case["M"] == 1 else dgate
            d = {"x": dy, "gate": dgate.reshape(v["gate"].shape), "w": rows(v["dh"] * yh).sum(0), "b": rows(v["dh"]).sum(0),
                 "pw": rows(df * fh).sum(0), "pb": rows(df).sum(0), "f": df if fr is None else _norm64_back(df * v["pw"], fh, fr, case["post"])}
    return out + ([d[n] for n in s["leaves"]] if train else [])
