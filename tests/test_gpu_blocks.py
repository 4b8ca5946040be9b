"""The gated feed-forward blocks and norms of dpvo_amd.blocks against the formulas in 64 bits.

Every tolerance is an error bound that is carried along with the 64-bit value (class V): a product of n terms adds n 2^-24 of the sum of the
terms' magnitudes (f32 accumulation in any order), a rounding to fewer bits adds half a step of the type, an elementary f32 function a few
2^-24 of its size.  A result has to lie within its bound at EVERY element."""
import math

import pytest
import torch

from dpvo_amd import _lib as L
from dpvo_amd import blocks

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {t: torch.finfo(t).eps / 2 for t in (F16, BF16, F32)}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}      # half the smallest step
U = 2.0 ** -24


class V:
    """a 64-bit value and the bound of its error"""

    def __init__(self, v, e=None):
        self.v = v
        self.e = torch.zeros_like(v) if e is None else e

    def top(self):
        return self.v.abs() + self.e

    def f32(self, n=1):
        """n f32 operations that each err by half a step of about this size"""
        return V(self.v, self.e + n * U * self.top())

    def to(self, t):
        return V(self.v, self.e + HALF[t] * self.top() + TINY[t])

    def __add__(self, o):
        return V(self.v + o.v, self.e + o.e).f32()

    def __mul__(self, o):
        return V(self.v * o.v, self.e * o.top() + o.e * self.v.abs()).f32()

    def mm(self, o):
        n = self.v.shape[-1] + 2
        mag = self.top() @ o.top()
        return V(self.v @ o.v, self.e @ o.v.abs() + self.v.abs() @ o.e + self.e @ o.e + n * U * mag)

    def t(self):
        return V(self.v.t(), self.e.t())

    def sum0(self):
        n = self.v.shape[0] + 2
        return V(self.v.sum(0), self.e.sum(0) + n * U * self.top().sum(0))


def rows_f(x):
    return V(x.detach().double().cpu())


def act(name, z):
    """(value, derivative) with the bounds of both.  Each function and its derivative has a slope of at most 1.2; the hardware exponential
    is good to |z| 2^-23 + 2^-22 relative, what it makes is at most about |z| + 1."""
    v = z.v
    if name == "identity":
        return V(v, z.e), V(torch.ones_like(v))
    if name == "relu":
        near = v.abs() <= z.e
        return V(v.clamp(min=0), z.e), V((v > 0).double(), near.double())
    if name in ("sigmoid", "silu"):
        s = torch.sigmoid(v)
        y, d = (s, s * (1 - s)) if name == "sigmoid" else (v * s, s + v * s * (1 - s))
    elif name == "gelu":
        c = 0.5 * torch.erfc(-v / math.sqrt(2))
        y, d = v * c, c + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    else:
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v ** 3))
        y, d = v * (1 + t) / 2, (1 + t) / 2 + v * (1 - t * t) / 2 * k * (1 + 3 * 0.044715 * v * v)
    own = 16 * U * (v.abs() + 1)
    return V(y, 1.2 * z.e + own), V(d, 1.2 * z.e + own)


def proj(x, w, b=None):
    y = x.mm(w.t())
    return y if b is None else y + b


def within(got, want, t, what):
    want = want.to(t)
    g = got.detach().double().cpu().reshape(want.v.shape)
    assert got.dtype == t, (what, got.dtype)
    bad = ~((g - want.v).abs() <= want.e)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound; worst error "
                           f"{float((g - want.v).abs()[bad].max()):.3e} against {float(want.e[bad].max()):.3e}")


def make(g, *shape, t=F32, scale=1.0, mean=0.0, grad=True):
    x = (torch.randn(*shape, generator=g) * scale + mean).to(t).cuda()
    return x.requires_grad_(grad)


def layer(g, n, k, t, bias=True, grad=True):
    s = 1 / math.sqrt(max(k, 1))
    return make(g, n, k, t=t, scale=s, grad=grad), make(g, n, t=t, scale=s, grad=grad) if bias else None


TYPES = [F16, BF16, F32]
# (M, K, N): single elements, single tokens, below / at / above a tile and a block of the sum, odd everything
SIZES = [(1, 1, 1), (1, 384, 384), (2, 7, 5), (3, 65, 130), (16, 64, 128), (33, 33, 31), (96, 384, 385), (128, 128, 128), (129, 63, 257),
         (300, 882, 100), (640, 200, 72)]


# ------------------------------------------------------------------------------------------------------------------ linear
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(dev, t, M, K, N):
    g = torch.Generator().manual_seed(M * 131 + K * 7 + N)
    for a, bias in (("identity", True), ("relu", True), ("gelu", False)):
        x = make(g, M, K, t=t)
        w, b = layer(g, N, K, t, bias)
        dy = make(g, M, N, t=t, grad=False)
        y = blocks.linear(x, w, b, a)
        with torch.no_grad():
            assert torch.equal(y, blocks.linear(x, w, b, a))          # serving and training make the same bits
        X, W, D = rows_f(x), rows_f(w), rows_f(dy)
        z = proj(X, W, rows_f(b) if bias else None)
        v, d = act(a, z)
        within(y, v, t, f"y {a}")
        grads = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy)
        dz = D if a == "identity" else (D * d).to(t)
        within(grads[0], dz.mm(W), t, f"dx {a}")
        within(grads[1], dz.t().mm(X), t, f"dw {a}")
        if bias:
            within(grads[2], dz.sum0(), t, f"db {a}")


# ------------------------------------------------------------------------------------------------------------------ gated linear
def gated_reference(x, wg, wu, bg, bu, a, v=None, res=None):
    g = proj(x, wg, bg)
    u = proj(x if v is None else v, wu, bu)
    y, d = act(a, g)
    out = y * u
    return (out if res is None else out + res), g, u, y, d


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("other", [False, True])
def test_gated_linear(dev, t, M, K, N, other):
    g = torch.Generator().manual_seed(M * 17 + K * 3 + N + other)
    a = ["silu", "gelu", "sigmoid", "gelu_tanh", "relu", "identity"][(M + K + N) % 6]
    x = make(g, M, K, t=t)
    Kv = K // 2 + 3 if other else K
    v = make(g, M, Kv, t=t) if other else None
    res = make(g, M, N, t=t) if other else None
    bias = (M + N) % 2 == 0
    wg, bg = layer(g, N, K, t, bias)
    wu, bu = layer(g, N, Kv, t, bias)
    dy = make(g, M, N, t=t, grad=False)
    y = blocks.gated_linear(x, wg, wu, bg, bu, a, up_input=v, residual=res)
    with torch.no_grad():
        assert torch.equal(y, blocks.gated_linear(x, wg, wu, bg, bu, a, up_input=v, residual=res))
    f = lambda q: None if q is None else rows_f(q)  # noqa: E731
    out, G, Uu, ya, da = gated_reference(f(x), f(wg), f(wu), f(bg), f(bu), a, f(v), f(res))
    within(y, out, t, f"y {a}")
    leaves = [x, wg, wu] + ([bg, bu] if bias else []) + ([v, res] if other else [])
    grads = list(torch.autograd.grad(y, leaves, dy))
    D = rows_f(dy)
    dg, du = (D * Uu * da).to(t), (D * ya).to(t)
    dx = dg.mm(f(wg))
    if other:
        within(grads[-2], du.mm(f(wu)), t, "dv")
        assert torch.equal(grads[-1], dy)
    else:
        dx = dx + du.mm(f(wu))
    within(grads[0], dx, t, "dx")
    within(grads[1], dg.t().mm(f(x)), t, "dwg")
    within(grads[2], du.t().mm(f(v if other else x)), t, "dwu")
    if bias:
        within(grads[3], dg.sum0(), t, "dbg")
        within(grads[4], du.sum0(), t, "dbu")


# ------------------------------------------------------------------------------------------------------------------ feed-forward
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,F,N,a,bias", [(1, 64, 256, 64, "silu", False), (5, 33, 70, 21, "gelu", True), (130, 96, 200, 96, "gelu_tanh", True),
                                            (257, 384, 64, 384, "sigmoid", False), (64, 100, 384, 100, "relu", True), (1500, 64, 64, 64, "silu", True)])
def test_feed_forward(dev, t, M, K, F, N, a, bias):
    g = torch.Generator().manual_seed(M + K + F)
    x = make(g, M, K, t=t)
    wg, bg = layer(g, F, K, t, bias)
    wu, bu = layer(g, F, K, t, bias)
    wd, bd = layer(g, N, F, t, bias)
    dy = make(g, M, N, t=t, grad=False)
    y = blocks.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, a)
    with torch.no_grad():
        assert torch.equal(y, blocks.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, a))
    f = lambda q: None if q is None else rows_f(q)  # noqa: E731
    h, G, Uu, ya, da = gated_reference(f(x), f(wg), f(wu), f(bg), f(bu), a)
    h = h.to(t)
    within(y, proj(h, f(wd), f(bd)), t, "y")
    leaves = [x, wg, wu, wd] + ([bg, bu, bd] if bias else [])
    grads = torch.autograd.grad(y, leaves, dy)
    D = rows_f(dy)
    dh = D.mm(f(wd))
    dg, du = (dh * Uu * da).to(t), (dh * ya).to(t)
    want = [dg.mm(f(wg)) + du.mm(f(wu)), dg.t().mm(f(x)), du.t().mm(f(x)), D.t().mm(h)] + ([dg.sum0(), du.sum0(), D.sum0()] if bias else [])
    for name, got, w in zip(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), grads, want):
        within(got, w, t, name)


# ------------------------------------------------------------------------------------------------------------------ gated residual
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,D,H", [(1, 384, 384), (96, 384, 384), (77, 45, 90), (700, 64, 64)])
def test_gated_residual(dev, t, M, D, H):
    g = torch.Generator().manual_seed(M + D)
    x = make(g, 1, M, D, t=t)
    wg, bg = layer(g, D, D, t)
    w1, b1 = layer(g, H, D, t)
    w2, b2 = layer(g, D, H, t)
    dy = make(g, 1, M, D, t=t, grad=False)
    y = blocks.gated_residual(x, wg, bg, w1, b1, w2, b2)
    assert y.shape == x.shape
    with torch.no_grad():
        assert torch.equal(y, blocks.gated_residual(x, wg, bg, w1, b1, w2, b2))
    f = rows_f
    X = f(x[0])
    p = proj(X, f(w1), f(b1))
    r, dr_ = act("relu", p)
    h = r.to(t)
    out, G, R, ya, da = gated_reference(X, f(wg), f(w2), f(bg), f(b2), "sigmoid", h, X)
    within(y, out, t, "y")
    grads = torch.autograd.grad(y, [x, wg, bg, w1, b1, w2, b2], dy)
    Dy = f(dy[0])
    dg, dr = (Dy * R * da).to(t), (Dy * ya).to(t)
    dp = (dr.mm(f(w2)) * dr_).to(t)
    want = [dg.mm(f(wg)) + dp.mm(f(w1)) + Dy, dg.t().mm(X), dg.sum0(), dp.t().mm(X), dp.sum0(), dr.t().mm(h), dr.sum0()]
    for name, got, w in zip(("dx", "dwg", "dbg", "dw1", "db1", "dw2", "db2"), grads, want):
        within(got, w, t, name)


# ------------------------------------------------------------------------------------------------------------------ norms
def row_mean(z):
    n = z.v.shape[-1]
    return V(z.v.mean(-1, keepdim=True), (z.e.sum(-1, keepdim=True) + (n + 2) * U * z.top().sum(-1, keepdim=True)) / n)


def normalise(z, kind, eps):
    if kind == "layer":
        z = z + row_mean(z) * V(torch.full_like(z.v[..., :1], -1.0))
    q = row_mean(z * z)
    s = q.v + eps
    r = V(s.rsqrt(), 0.5 * q.e * (s - q.e).clamp(min=eps) ** -1.5).f32(4)
    return z * r, r


def norm_back(d, xh, r, kind):
    o = d + xh * row_mean(d * xh) * V(torch.full_like(r.v, -1.0))
    if kind == "layer":
        o = o + row_mean(d) * V(torch.full_like(r.v, -1.0))
    return o * r


NORM_SIZES = [(1, 1), (3, 2), (5, 7), (1, 1024), (33, 64), (17, 129), (40, 384), (1030, 384), (9, 385), (6, 513), (65, 1000), (4, 1536), (3, 2048), (7, 2056),
              (5, 4096), (3, 4100), (3, 8192), (2, 8193), (2, 16384)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("tx,th", [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)], ids=str)
@pytest.mark.parametrize("M,D", NORM_SIZES)
def test_norm(dev, kind, tx, th, M, D):
    g = torch.Generator().manual_seed(M * 3 + D)
    x = make(g, M, D, t=tx, scale=1.5, mean=0.5)
    w = make(g, D, t=tx, scale=0.2, mean=1.0)
    b = make(g, D, t=tx) if D % 2 == 0 else None
    dh = make(g, M, D, t=th, grad=False)
    h = blocks.norm(x, w, b, kind, eps=1e-3, out_dtype=th)
    xh, r = normalise(rows_f(x), kind, 1e-3)
    o = xh * rows_f(w)
    within(h, o if b is None else o + rows_f(b), th, "h")
    leaves = [x, w] + ([b] if b is not None else [])
    grads = torch.autograd.grad(h, leaves, dh)
    Dh = rows_f(dh)
    within(grads[0], norm_back(Dh * rows_f(w), xh, r, kind), tx, "dx")
    within(grads[1], (Dh * xh).sum0(), tx, "dw")
    if b is not None:
        within(grads[2], Dh.sum0(), tx, "db")


def residual_norm_case(g, tx, tb, lead, D, kind, post, gate, gate_act, scale, use):
    x = make(g, *lead, D, t=tx, scale=1.5, mean=0.25)
    f = make(g, *lead, D, t=tb, scale=1.2, mean=-0.2)
    ga = None if gate is None else make(g, *gate, D, t=tb)
    w = make(g, D, t=tx, scale=0.2, mean=1.0) if kind else None
    b = make(g, D, t=tx, scale=0.2) if kind == "layer" else None
    pw = make(g, D, t=tx, scale=0.2, mean=1.0) if post else None
    pb = make(g, D, t=tx, scale=0.2) if post == "layer" else None
    s, h = blocks.residual_norm(x, f, w, b, norm=kind, eps=1e-3, gate=ga, gate_activation=gate_act, scale=scale, post_norm=post, post_weight=pw,
                                post_bias=pb, post_eps=1e-2)
    assert s.shape == x.shape and (h is None) == (kind is None)
    with torch.no_grad():
        s2, h2 = blocks.residual_norm(x, f, w, b, norm=kind, eps=1e-3, gate=ga, gate_activation=gate_act, scale=scale, post_norm=post,
                                      post_weight=pw, post_bias=pb, post_eps=1e-2)
        assert torch.equal(s, s2) and (h is None or torch.equal(h, h2))
    M = x.numel() // D
    R = lambda q: V(q.detach().double().cpu().reshape(-1, D))  # noqa: E731
    P, fr = (R(f), None) if post is None else normalise(R(f), post, 1e-2)
    fh = P
    if post:
        P = P * R(pw)
        P = P if pb is None else P + R(pb)
    if ga is None:
        A, dA = V(torch.ones(M, D, dtype=torch.float64)), None
        inc = P
    else:
        full = V(ga.detach().double().cpu().expand(*lead, D).reshape(M, D)) if ga.dim() == len(lead) + 1 else V(ga.detach().double().cpu().expand(M, D))
        A, dA = act(gate_act, full)
        inc = A * P
    c = V(torch.full((1, 1), float(scale), dtype=torch.float64))
    S = R(x) + inc * c
    within(s, S, tx, "s")
    outs, ups = [], []
    DY = None
    if use != "h":
        ds = make(g, *lead, D, t=tx, grad=False)
        outs.append(s)
        ups.append(ds)
        DY = R(ds)
    leaves = [("x", x, tx), ("f", f, tb)]
    want = {}
    if kind:
        sh, r = normalise(S, kind, 1e-3)
        o = sh * R(w)
        within(h, o if b is None else o + R(b), tb, "h")
        leaves.append(("w", w, tx))
        if b is not None:
            leaves.append(("b", b, tx))
        Z = V(torch.zeros(M, D, dtype=torch.float64))
        if use != "s":
            dh = make(g, *lead, D, t=tb, grad=False)
            outs.append(h)
            ups.append(dh)
            Dh = R(dh)
            back = norm_back(Dh * R(w), sh, r, kind)
            DY = back if DY is None else DY + back
        else:
            Dh = Z
        want["w"], want["b"] = (Dh * sh).sum0(), Dh.sum0()
    want["x"] = DY
    q = DY * c
    dp = q * A
    if ga is not None:
        dga = q * P * dA
        n = ga.numel() // D
        k = M // n
        want["gate"] = dga if n == M else V(dga.v.reshape(n, k, D).sum(1), (dga.e.reshape(n, k, D) + (k + 2) * U * dga.top().reshape(n, k, D)).sum(1))
        leaves.append(("gate", ga, tb))
    want["f"] = dp
    if post:
        want["pw"], want["pb"] = (dp * fh).sum0(), dp.sum0()
        want["f"] = norm_back(dp * R(pw), fh, fr, post)
        leaves.append(("pw", pw, tx))
        if pb is not None:
            leaves.append(("pb", pb, tx))
    grads = torch.autograd.grad(outs, [t for _, t, _ in leaves], ups)
    for (name, leaf, t), got in zip(leaves, grads):
        assert got.shape == leaf.shape
        within(got, want[name], t, f"d{name}")


@pytest.mark.parametrize("tx,tb", [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)], ids=str)
@pytest.mark.parametrize("lead,D,kind,post,gate,gate_act,scale,use", [
    ((1,), 1, "layer", None, None, "identity", 1.0, "sh"),
    ((1,), 1024, "rms", "rms", (), "identity", 1.0, "sh"),
    ((40,), 384, "layer", None, (40,), "sigmoid", 1.0, "sh"),
    ((2, 20), 384, "layer", "layer", (2, 20), "silu", 0.5, "sh"),
    ((3, 70), 129, "rms", "rms", (3, 1), "identity", 0.5, "sh"),
    ((600, 2), 65, "rms", None, (600, 1), "sigmoid", 2.0, "sh"),
    ((5, 4, 3), 520, "layer", "rms", (5, 1, 1), "silu", -1.0, "sh"),
    ((130,), 100, None, "layer", (1,), "relu", 1.0, "sh"),
    ((66,), 1100, "rms", "layer", (66,), "sigmoid", 1.0, "h"),
    ((66,), 40, "rms", "layer", (), "sigmoid", 1.0, "s"),
    ((9,), 4097, "layer", "rms", (1,), "sigmoid", 1.0, "sh"),
    ((4,), 8000, "rms", "layer", (4,), "sigmoid", 1.0, "sh"),
    ((3,), 16383, "layer", "layer", (3,), "identity", 1.0, "sh"),
    # lanes without a column (D is no multiple of a row's lanes) beside a gate that is not 0 there: their mean must not reach the branch's sums
    ((5,), 671, "layer", "layer", (5,), "sigmoid", 1.0, "sh"),
    ((9,), 384, "layer", "layer", (), "sigmoid", 1.0, "sh"),
    ((6,), 2560, "layer", "layer", (6,), "sigmoid", 0.5, "sh"),
    ((3,), 10000, "layer", "layer", (3,), "sigmoid", 1.0, "h"),
])
def test_residual_norm(dev, tx, tb, lead, D, kind, post, gate, gate_act, scale, use):
    g = torch.Generator().manual_seed(D + len(lead))
    residual_norm_case(g, tx, tb, lead, D, kind, post, gate, gate_act, scale, use)


# ------------------------------------------------------------------------------------------------------------------ together, as the model has them
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_update_gru(dev, t):
    """Update.gru (LayerNorm, gated residual block, twice) and its gradients, through the model's own module, against the carried bounds"""
    from dpvo_amd import net as N
    torch.manual_seed(3)
    gru = N.Update(3).gru.to(dev)
    with torch.no_grad():
        for p in gru.parameters():
            if p.dim() == 1:
                p.add_(0.05 * torch.randn_like(p))
    g = torch.Generator().manual_seed(8)
    x = make(g, 1, 150, 384, t=t)
    dy = make(g, 1, 150, 384, t=t, grad=False)
    y = gru(x)
    grads = torch.autograd.grad(y, [x, *gru.parameters()], dy)
    names = ["x"] + [n for n, _ in gru.named_parameters()]
    par = {n: p for n, p in gru.named_parameters()}
    op = lambda n: V(par[n].detach().to(t).double().cpu())  # noqa: E731
    full = lambda n: rows_f(par[n])  # noqa: E731
    z, kept = rows_f(x[0]), []
    for i in (0, 2):
        xh, r = normalise(z, "layer", 1e-3)
        h = (xh * full(f"{i}.weight") + full(f"{i}.bias")).to(t)
        q = f"{i + 1}."
        a, d1 = act("relu", proj(h, op(q + "res.0.weight"), op(q + "res.0.bias")))
        a = a.to(t)
        out, G, R, ya, da = gated_reference(h, op(q + "gate.0.weight"), op(q + "res.2.weight"), op(q + "gate.0.bias"), op(q + "res.2.bias"), "sigmoid", a, h)
        kept.append((xh, r, h, a, d1, R, ya, da))
        z = out.to(t)
    within(y, z, t, "y")
    want, D = {}, rows_f(dy[0])
    for i in (2, 0):
        xh, r, h, a, d1, R, ya, da = kept[i // 2]
        q = f"{i + 1}."
        dg, dr = (D * R * da).to(t), (D * ya).to(t)
        dp = (dr.mm(op(q + "res.2.weight")) * d1).to(t)
        for n, u, v in (("gate.0", dg, h), ("res.0", dp, h), ("res.2", dr, a)):
            want[q + n + ".weight"], want[q + n + ".bias"] = u.t().mm(v).to(t), u.sum0().to(t)
        D = (dg.mm(op(q + "gate.0.weight")) + dp.mm(op(q + "res.0.weight")) + D).to(t)
        want[f"{i}.weight"], want[f"{i}.bias"] = (D * xh).sum0(), D.sum0()
        D = norm_back(D * full(f"{i}.weight"), xh, r, "layer").to(t)
    want["x"] = D
    for n, got in zip(names, grads):
        within(got, want[n], got.dtype, n)


def test_gru_is_the_stage_of_the_tracker(dev):
    """the same stage in Update.forward's comparator pieces (launch by launch, f16 operands, f32 state) and here in f16: each is within the
    roundings of its f16 operands of the other"""
    from dpvo_amd import net as N
    torch.manual_seed(4)
    upd = N.Update(3).to(dev)
    x = torch.randn(1, 200, 384, generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        y = upd.gru(x)
        P = upd.pack()
        z = x[0].clone()
        h1 = torch.empty(200, 384, dtype=F16, device=dev)
        fg = torch.empty(200, 768, dtype=F16, device=dev)
        for name in ("g0", "g1"):
            gm, b, Wrg, brg, W2, b2 = P[name]
            N.layernorm(z, gm, b, y_f32=z, y_f16=h1)
            N.linear(h1, Wrg, brg, out=fg, epilogue=N.EPI_RELU_SIG, n_split=384)
            N.linear(fg[:, :384], W2, b2, out=z, epilogue=N.EPI_GATED, gate=fg[:, 384:])
    # roundings per block: operand h, weights, the hidden layer, the gate, twice over; each half a step (2^-11) of values of a few units
    assert float((y[0] - z).abs().max()) < 16 * 2.0 ** -11 * float(z.abs().max())
