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


def on_gpu(x):
    """the same on the GPU, for sizes where the CPU's 64-bit products would take long"""
    return V(x.detach().double())


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
    g = got.detach().double().to(want.v.device).reshape(want.v.shape)
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
         (300, 882, 100), (640, 200, 72), (70, 385, 882), (100, 2500, 64), (1300, 90, 330), (1100, 600, 300), (2900, 100, 900)]


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
    # widths that end inside a lane's piece, of every number of lanes
    ((70,), 5, "layer", "layer", (70,), "sigmoid", 1.0, "sh"),
    ((70,), 253, "layer", "rms", (1,), "silu", 1.0, "sh"),
    ((37,), 1003, "layer", "layer", (37,), "sigmoid", 1.0, "sh"),
    ((21,), 1999, "rms", "layer", (1,), "sigmoid", 1.0, "sh"),
    ((11,), 3001, "layer", "layer", (11,), "sigmoid", 1.0, "sh"),
    # rows over a whole workgroup: many groups, parts of a group, one of the two results alone, no gate, no norm
    ((140, 2), 4099, "layer", "layer", (140, 1), "sigmoid", 0.5, "sh"),
    ((3, 100), 4104, "rms", "rms", (3, 1), "identity", 1.0, "sh"),
    ((300,), 4097, "layer", "layer", (), "sigmoid", 1.0, "s"),
    ((150,), 5000, "layer", None, None, "identity", 1.0, "h"),
    ((20,), 8193, None, "layer", (1,), "relu", 1.0, "sh"),
    ((30,), 4200, "layer", "layer", (1,), "sigmoid", 1.0, "sh"),
    ((5,), 12001, "rms", "layer", (5,), "silu", 1.0, "sh"),
])
def test_residual_norm(dev, tx, tb, lead, D, kind, post, gate, gate_act, scale, use):
    g = torch.Generator().manual_seed(D + len(lead))
    residual_norm_case(g, tx, tb, lead, D, kind, post, gate, gate_act, scale, use)


# ------------------------------------------------------------------------------------------------------------------ large tiles and long sums
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,F,N", [(5013, 2311, 2317, 2305), (4100, 1030, 2310, 1030), (20011, 200, 136, 72), (45312, 384, 384, 384), (2000, 1500, 700, 300)])
def test_feed_forward_large(dev, t, M, K, F, N):
    """sizes that reach the 256- and 128-wide tiles of every product, sums in parts, and tiles that hang over in both directions"""
    g = torch.Generator().manual_seed(M)
    x = make(g, M, K, t=t)
    wg, bg = layer(g, F, K, t)
    wu, bu = layer(g, F, K, t)
    wd, bd = layer(g, N, F, t)
    dy = make(g, M, N, t=t, grad=False)
    f = on_gpu
    h, G, Uu, ya, da = gated_reference(f(x), f(wg), f(wu), f(bg), f(bu), "silu")
    h = h.to(t)
    y = blocks.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, "silu")
    within(y, proj(h, f(wd), f(bd)), t, "y")
    grads = torch.autograd.grad(y, [x, wg, wu, wd, bg, bu, bd], dy)
    D = f(dy)
    dh = D.mm(f(wd))
    dg, du = (dh * Uu * da).to(t), (dh * ya).to(t)
    want = [dg.mm(f(wg)) + du.mm(f(wu)), dg.t().mm(f(x)), du.t().mm(f(x)), D.t().mm(h), dg.sum0(), du.sum0(), D.sum0()]
    for name, got, w in zip(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), grads, want):
        within(got, w, t, name)
    again = torch.autograd.grad(blocks.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, "silu"), [x, wg, wu, wd, bg, bu, bd], dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))       # no order of sums changes from run to run


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(5013, 2311, 2317), (9000, 384, 390)])
def test_gated_linear_large_two_inputs(dev, t, M, K, N):
    g = torch.Generator().manual_seed(M + 1)
    x, v, res = make(g, M, K, t=t), make(g, M, K + 5, t=t), make(g, M, N, t=t)
    wg, bg = layer(g, N, K, t)
    wu, bu = layer(g, N, K + 5, t)
    dy = make(g, M, N, t=t, grad=False)
    f = on_gpu
    y = blocks.gated_linear(x, wg, wu, bg, bu, "sigmoid", up_input=v, residual=res)
    out, G, Uu, ya, da = gated_reference(f(x), f(wg), f(wu), f(bg), f(bu), "sigmoid", f(v), f(res))
    within(y, out, t, "y")
    grads = torch.autograd.grad(y, [x, v, wg, wu, bg, bu], dy)
    D = f(dy)
    dg, du = (D * Uu * da).to(t), (D * ya).to(t)
    want = [dg.mm(f(wg)), du.mm(f(wu)), dg.t().mm(f(x)), du.t().mm(f(v)), dg.sum0(), du.sum0()]
    for name, got, w in zip(("dx", "dv", "dwg", "dwu", "dbg", "dbu"), grads, want):
        within(got, w, t, name)


# ------------------------------------------------------------------------------------------------------------------ layouts
def odd_place(x, ld=None, shift=1):
    """the same values at an address `shift` elements behind an allocation's, with rows `ld` apart"""
    M, K = x.shape
    ld = ld or K
    buf = torch.full((shift + M * ld + 7,), float("nan"), dtype=x.dtype, device=x.device)
    v = buf[shift:shift + M * ld].view(M, ld)[:, :K]
    v.copy_(x)
    return v


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(5, 33, 17), (70, 129, 65), (300, 384, 200), (1100, 250, 390)])
@pytest.mark.parametrize("pad", [0, 3])
def test_unaligned_rows(dev, t, M, K, N, pad):
    """rows that start at any element, with NaN between and behind them: nothing outside a row may be used"""
    g = torch.Generator().manual_seed(M + pad)
    x, wg, wu = make(g, M, K, t=t, grad=False), make(g, N, K, t=t, scale=0.1, grad=False), make(g, N, K, t=t, scale=0.1, grad=False)
    b, res, dy = make(g, N, t=t, grad=False), make(g, M, N, t=t, grad=False), make(g, M, N, t=t, grad=False)
    for a in ("silu", "identity"):
        want = [p.clone().requires_grad_() for p in (x, wg, wu, b, res)]
        y0 = blocks.gated_linear(want[0], want[1], want[2], want[3], want[3], a, residual=want[4])
        g0 = torch.autograd.grad(y0, want, dy)
        got = [odd_place(p, p.shape[1] + pad).requires_grad_() for p in (x, wg, wu)] + [odd_place(b[None])[0].requires_grad_(),
                                                                                      odd_place(res, N + pad).requires_grad_()]
        y1 = blocks.gated_linear(got[0], got[1], got[2], got[3], got[3], a, residual=got[4])
        g1 = torch.autograd.grad(y1, got, odd_place(dy, N + pad))
        assert torch.equal(y0, y1)
        assert all(torch.equal(p, q) for p, q in zip(g0, g1))
    for p, q in ((x, odd_place(x, K + pad)), (x.t().contiguous().t(), x.t().contiguous().t())):
        assert torch.equal(blocks.linear(x, wg, b), blocks.linear(q, odd_place(wg, K + pad), b))
    w = make(g, K, t=t, grad=False)
    assert torch.equal(blocks.norm(x, w), blocks.norm(odd_place(x, K + pad), odd_place(w[None])[0]))
    s0 = blocks.residual_norm(x, x, w, gate=w, post_norm="rms", post_weight=w)
    s1 = blocks.residual_norm(odd_place(x, K + pad), odd_place(x, K + pad, 3), odd_place(w[None])[0], gate=odd_place(w[None])[0], post_norm="rms", post_weight=w)
    assert all(torch.equal(p, q) for p, q in zip(s0, s1))


def test_layouts_are_accepted(dev):
    """any strides, leading shapes and broadcast gradients give what contiguous rows give"""
    g = torch.Generator().manual_seed(0)
    x = make(g, 6, 5, 24, grad=False)
    w, wu = make(g, 10, 24, scale=0.2, grad=False), make(g, 10, 24, scale=0.2, grad=False)
    flat = blocks.gated_linear(x.reshape(30, 24), w, wu)
    assert torch.equal(blocks.gated_linear(x, w, wu).reshape(30, 10), flat)
    assert torch.equal(blocks.gated_linear(x.transpose(0, 1), w, wu), blocks.gated_linear(x.transpose(0, 1).contiguous(), w, wu))
    assert torch.equal(blocks.gated_linear(x, w.t().contiguous().t(), wu).reshape(30, 10), flat)
    assert torch.equal(blocks.gated_linear(x[0, 0], w, wu), flat[0])              # a vector
    assert torch.equal(blocks.gated_linear(x[:1, :1].expand(3, 4, 24), w, wu), flat[:1, None].expand(1, 12, 10).reshape(3, 4, 10))
    p = x.clone().requires_grad_()
    a, = torch.autograd.grad(blocks.gated_linear(p, w, wu).sum(), p)              # the gradient that arrives is an expanded scalar
    b, = torch.autograd.grad(blocks.gated_linear(p, w, wu), p, torch.ones(6, 5, 10, device=dev))
    assert torch.equal(a, b)
    a, = torch.autograd.grad(blocks.norm(p).sum(), p)
    b, = torch.autograd.grad(blocks.norm(p), p, torch.ones_like(x))
    assert torch.equal(a, b)
    same = [w.clone().requires_grad_()]                                           # one leaf in two places
    got, = torch.autograd.grad(blocks.gated_linear(x, same[0], same[0]).sum(), same)
    two = [w.clone().requires_grad_(), w.clone().requires_grad_()]
    ga, gb = torch.autograd.grad(blocks.gated_linear(x, *two).sum(), two)
    assert torch.equal(got, ga + gb)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_no_rows(dev, t):
    x = torch.zeros(0, 3, 40, dtype=t, device=dev, requires_grad=True)
    w, b = torch.ones(24, 40, dtype=t, device=dev, requires_grad=True), torch.ones(24, dtype=t, device=dev, requires_grad=True)
    wd = torch.ones(40, 24, dtype=t, device=dev, requires_grad=True)
    for y, leaves in ((blocks.linear(x, w, b, "relu"), [x, w, b]), (blocks.gated_linear(x, w, w, b, b), [x, w, b]),
                      (blocks.gated_feed_forward(x, w, w, wd, b, b), [x, w, b, wd]), (blocks.norm(x, wd[:, 0], wd[:, 1]), [x, wd])):
        assert y.shape[:2] == (0, 3)
        for p, q in zip(leaves, torch.autograd.grad(y, leaves, torch.zeros_like(y))):
            assert q.shape == p.shape and not q.any()
    gate = torch.ones(0, 1, 40, dtype=t, device=dev, requires_grad=True)
    row = torch.ones(40, dtype=t, device=dev, requires_grad=True)
    for ga in (gate, row):
        s, h = blocks.residual_norm(x, x, row, gate=ga)
        assert s.shape == h.shape == x.shape
        for p, q in zip((x, row, ga), torch.autograd.grad([s, h], [x, row, ga], [torch.zeros_like(s), torch.zeros_like(h)], allow_unused=True)):
            assert q.shape == p.shape and not q.any()


def test_some_gradients(dev):
    """whatever subset of the leaves asks for a gradient, each gets what it gets when all ask"""
    g = torch.Generator().manual_seed(2)
    base = dict(x=make(g, 70, 48), wg=make(g, 36, 48), wu=make(g, 36, 48), wd=make(g, 48, 36), bg=make(g, 36), bu=make(g, 36), bd=make(g, 48))
    run = {"ff": (lambda d: [blocks.gated_feed_forward(d["x"], d["wg"], d["wu"], d["wd"], d["bg"], d["bu"], d["bd"])], list(base)),
           "block": (lambda d: [blocks.gated_residual(d["x"], d["sq"], d["bd"], d["wg"], d["bg"], d["wd"], d["bd"])], ["x", "wg", "wd", "bg", "sq"]),
           "linear": (lambda d: [blocks.linear(d["x"], d["wg"], d["bg"], "silu")], ["x", "wg", "bg"]),
           "two": (lambda d: [blocks.gated_linear(d["x"], d["wg"], d["sq"][:36, :36].contiguous(), d["bg"], d["bu"], up_input=d["v"], residual=d["v"])],
                   ["x", "wg", "sq", "bg", "bu", "v"]),
           "norm": (lambda d: list(blocks.residual_norm(d["x"], d["f"], d["n"], d["bd"], gate=d["gate"], gate_activation="sigmoid", post_norm="layer",
                                                        post_weight=d["pn"], post_bias=d["pb"])), ["x", "f", "n", "bd", "gate", "pn", "pb"])}
    base.update(sq=make(g, 48, 48), v=make(g, 70, 36), f=make(g, 70, 48), n=make(g, 48), gate=make(g, 48), pn=make(g, 48), pb=make(g, 48))
    for name, (f, leaves) in run.items():
        outs = f(base)
        ups = [torch.randn(o.shape, generator=g).cuda() for o in outs]
        full = dict(zip(leaves, torch.autograd.grad(outs, [base[k] for k in leaves], ups)))
        for n in range(len(leaves)):
            for some in ([leaves[n]], leaves[:n] + leaves[n + 1:]):
                d = {k: v.detach().requires_grad_(k in some) for k, v in base.items()}
                for k, got in zip(some, torch.autograd.grad(f(d), [d[k] for k in some], ups)):
                    assert torch.equal(got, full[k]), (name, some, k)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_infinities_and_nan_stay_in_their_rows(dev, t):
    g = torch.Generator().manual_seed(5)
    for M, K, N in ((3, 70, 40), (100, 70, 40), (300, 200, 150)):
        x, w, wu = make(g, M, K, t=t, grad=False), make(g, N, K, t=t, scale=0.1, grad=False), make(g, N, K, t=t, scale=0.1, grad=False)
        y = blocks.gated_linear(x, w, wu)
        bad = x.clone()
        bad[1, 5], bad[2, 7] = float("nan"), float("inf")
        z = blocks.gated_linear(bad, w, wu)
        keep = [i for i in range(M) if i not in (1, 2)]
        assert torch.equal(z[keep], y[keep]) and z[1].isnan().all() and not z[2].isfinite().all()
        wb = w.clone()
        wb[4, 3] = float("nan")                                       # one output column
        z = blocks.gated_linear(x, wb, wu)
        cols = [i for i in range(N) if i != 4]
        assert torch.equal(z[:, cols], y[:, cols]) and z[:, 4].isnan().all()
        n0, n1 = blocks.norm(x), blocks.norm(bad)
        assert torch.equal(n1[keep], n0[keep]) and n1[1].isnan().all()
        p, q = x.clone().requires_grad_(), w.clone().requires_grad_()
        dy = make(g, M, N, t=t, grad=False)
        d0 = torch.autograd.grad(blocks.gated_linear(p, q, wu), [p, q], dy)
        db = dy.clone()
        db[1, 6] = float("nan")
        d1 = torch.autograd.grad(blocks.gated_linear(p, q, wu), [p, q], db)
        assert torch.equal(d1[0][keep], d0[0][keep]) and d1[0][1].isnan().all()
        cols = [i for i in range(N) if i != 6]
        assert torch.equal(d1[1][cols], d0[1][cols]) and d1[1][6].isnan().all()


def test_many_elements(dev):
    """offsets that pass 32 bits: 36 million rows of 64 in 16 bits (2.3e9 elements), first and last rows against a small call"""
    M, K, N = 36_000_000, 8, 64
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(M, K, generator=g, device=dev).half()
    w, wu = torch.randn(N, K, generator=g, device=dev).half(), torch.randn(N, K, generator=g, device=dev).half()
    y = blocks.gated_linear(x, w, wu)
    for a, b in ((0, 5000), (M // 2 - 77, M // 2 + 4001), (M - 5000, M)):
        assert torch.equal(y[a:b], blocks.gated_linear(x[a:b], w, wu))
    s, h = blocks.residual_norm(y, y, norm="rms")
    for a, b in ((0, 50), (M - 50, M)):
        s1, h1 = blocks.residual_norm(y[a:b], y[a:b], norm="rms")
        assert torch.equal(s[a:b], s1) and torch.equal(h[a:b], h1)
    del s, h
    # a weight's gradient over all of them: 1 in the rows that count, 0 elsewhere
    p = w.clone().requires_grad_()
    dy = torch.zeros_like(y)
    dy[-3:] = 1
    got, = torch.autograd.grad(blocks.linear(x, p), p, dy)
    torch.testing.assert_close(got.float(), x[-3:].float().sum(0).expand(N, K), rtol=2.0 ** -11, atol=1e-6)


# ------------------------------------------------------------------------------------------------------------------ streams and graphs
def block_step(d):
    """norm -> gated feed-forward -> (gate, residual) -> norm -> gated residual block, and all gradients"""
    h = blocks.norm(d["x"], d["n1"], d["b1"])
    f = blocks.gated_feed_forward(h, d["wg"], d["wu"], d["wd"], d["bg"], d["bg"], d["n1"])
    s, h = blocks.residual_norm(d["x"], f, d["n2"], norm="rms", gate=d["gate"], gate_activation="sigmoid", scale=0.5, post_norm="layer", post_weight=d["n1"],
                                post_bias=d["b1"])
    y = blocks.gated_residual(h, d["sq"], d["b1"], d["wg"], d["bg"], d["wd"], d["b1"])
    return [s, y, *torch.autograd.grad([s, y], list(d.values()), [torch.ones_like(s), torch.full_like(y, 0.5)])]


def block_leaves(t, M=200, D=96, F=160, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {"x": make(g, M, D, t=t), "n1": make(g, D, t=t, scale=0.2, mean=1.0), "b1": make(g, D, t=t, scale=0.2), "wg": make(g, F, D, t=t, scale=0.1),
            "wu": make(g, F, D, t=t, scale=0.1), "wd": make(g, D, F, t=t, scale=0.1), "bg": make(g, F, t=t, scale=0.2), "n2": make(g, D, t=t, scale=0.2, mean=1.0),
            "gate": make(g, D, t=t), "sq": make(g, D, D, t=t, scale=0.1)}


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_the_run_of_them_on_two_streams(dev, t):
    """two runs at once on two streams give what each gives alone"""
    a, b = block_leaves(t), block_leaves(t, M=333, seed=1)
    want = [block_step(a), block_step(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, d in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                got.append(block_step(d))
        torch.cuda.synchronize()
        for w, q in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(w, q))


def test_two_threads(dev):
    """steps from two host threads at once, each on its own stream: nothing is shared between calls"""
    import threading
    leaves = [block_leaves(t, M=120, D=384, F=700) for t in (F16, F32)]
    want = [block_step(d) for d in leaves]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got[i].append(block_step(leaves[i]))
            s.synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == 10 and all(torch.equal(x, y) for step in got[i] for x, y in zip(step, want[i]))


def test_captured_graphs(dev):
    """two graphs of forward passes (with and without sums in parts) and one of a whole step, replayed in turn with eager calls between: every replay
    equals the eager result on the inputs of the moment"""
    leaves = {k: v.detach() for k, v in block_leaves(F16, M=200, D=384, F=2048).items()}

    def forward(d):
        h = blocks.norm(d["x"], d["n1"], d["b1"])
        f = blocks.gated_feed_forward(h, d["wg"], d["wu"], d["wd"], d["bg"], d["bg"], d["n1"])
        return list(blocks.residual_norm(d["x"], f, d["n2"], norm="rms", gate=d["gate"]))

    def step(d):
        return block_step({k: v.detach().requires_grad_() for k, v in d.items()})

    wide = {"x": torch.randn(64, 4096, device=dev).half()}
    wider = {"x": torch.randn(64, 5001, device=dev)}

    def wide_step(d):
        x = d["x"].detach().requires_grad_()
        w, b = (torch.ones_like(x[0]).detach().requires_grad_() for _ in range(2))
        s, h = blocks.residual_norm(x, x * 0.5, w, b, gate=w, post_norm="layer", post_weight=w, post_bias=b)
        return [h, *torch.autograd.grad([s, h], [x, w, b], [torch.ones_like(s), torch.ones_like(h)])]

    jobs = []
    for f, d in ((forward, leaves), (step, leaves), (forward, {**leaves, "x": leaves["x"][:50].clone()}), (wide_step, wide), (wide_step, wider)):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f(d)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(d)
        jobs.append((f, d, graph, out))
    for k in range(4):
        for f, d, graph, out in jobs:
            d["x"].copy_(torch.randn(d["x"].shape, generator=torch.Generator().manual_seed(k)).half())
            graph.replay()
            want = f(d)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want)), (f.__name__, k)


def test_second_order_is_refused(dev):
    x = torch.randn(4, 8, device=dev, requires_grad=True)
    w = torch.randn(8, 8, device=dev, requires_grad=True)
    g, = torch.autograd.grad(blocks.linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), w)


def test_gradients_against_differences(dev):
    """the gradients of a whole run in f32 against central differences of the plain formula in 64 bits along random directions"""
    d = block_leaves(F32, M=20, D=24, F=32)
    grads = block_step(d)[2:]
    g = torch.Generator().manual_seed(9)
    val = {k: v.detach().double().cpu() for k, v in d.items()}
    dirs = {k: torch.randn(v.shape, generator=g, dtype=torch.float64) for k, v in val.items()}

    def loss(v):
        ln = lambda x, w, b: torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-3)  # noqa: E731
        rms = lambda x, w: x * (x.pow(2).mean(-1, keepdim=True) + 1e-3).rsqrt() * w  # noqa: E731
        lin = torch.nn.functional.linear
        h = ln(v["x"], v["n1"], v["b1"])
        f = lin(torch.nn.functional.silu(lin(h, v["wg"], v["bg"])) * lin(h, v["wu"], v["bg"]), v["wd"], v["n1"])
        s = v["x"] + 0.5 * torch.sigmoid(v["gate"]) * ln(f, v["n1"], v["b1"])
        h = rms(s, v["n2"])
        y = h + torch.sigmoid(lin(h, v["sq"], v["b1"])) * lin(torch.relu(lin(h, v["wg"], v["bg"])), v["wd"], v["b1"])
        return s.sum() + 0.5 * y.sum()

    e = 1e-5
    for k, got in zip(d, grads):
        up, dn = dict(val), dict(val)
        up[k], dn[k] = val[k] + e * dirs[k], val[k] - e * dirs[k]
        want = float(loss(up) - loss(dn)) / (2 * e)
        have = float((got.double().cpu() * dirs[k]).sum())
        # f32 sums of some hundred terms, and e^2 of the difference
        assert abs(have - want) < 2e-4 * float((got.double().cpu().abs() * dirs[k].abs()).sum()) + 1e-6, (k, have, want)


def test_the_bounds_see_a_mistake():
    """the oracle with a sign, a factor or a dropped term is outside the bounds by which the kernels are held (nothing runs on the GPU here)"""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(40, 64, generator=g).half(), (torch.randn(30, 64, generator=g) / 8).half()
    z = proj(rows_f(x), rows_f(w))
    v, d = act("silu", z)
    for wrong in (v.v * 1.002, v.v + 2e-3, torch.relu(z.v), v.v.roll(1, 0)):
        with pytest.raises(AssertionError):
            within(wrong.half(), v, F16, "planted")
    within(v.v.half(), v, F16, "right")
    xh, r = normalise(rows_f(x), "layer", 1e-3)
    for wrong in (normalise(rows_f(x), "rms", 1e-3)[0].v, normalise(rows_f(x), "layer", 1e-2)[0].v):
        with pytest.raises(AssertionError):
            within(wrong.half(), xh, F16, "planted")


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


@pytest.mark.parametrize("D", [1, 20])
def test_pending_signs(dev, D):
    """inputs that are negated views, and the gradient that a complex conjugate sends back: a negated view too, with rows where D is 1"""
    g = torch.Generator().manual_seed(11)
    neg = lambda t: torch._neg_view(-t)  # noqa: E731
    x, n, e, f, r = make(g, 9, D, grad=False), make(g, D, grad=False), make(g, D, grad=False), make(g, 9, D, grad=False), make(g, 9, 12, grad=False)
    w, wu, b, wd, sq = (make(g, *s, grad=False) for s in ((12, D), (12, D), (12,), (D, 12), (D, D)))
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    runs = [(lambda x, sq, e: blocks.linear(x, sq, e, "silu"), (x, sq, e)),
            (lambda x, w, c, b, r: blocks.gated_linear(x, w, c, b, b, residual=r), (x, w, wu, b, r)),
            (lambda x, w, c, d, b, e: blocks.gated_feed_forward(x, w, c, d, b, b, e), (x, w, wu, wd, b, e)),
            (lambda x, sq, e, w, b, d: blocks.gated_residual(x, sq, e, w, b, d, e), (x, sq, e, w, b, wd)),
            (lambda x, n, e: blocks.norm(x, n, e, "rms"), (x, n, e)),
            (lambda x, f, n, e: blocks.residual_norm(x, f, n, e, gate=n, post_norm="rms", post_weight=e)[1], (x, f, n, e))]
    for k, (run, args) in enumerate(runs):
        want = [t.clone().requires_grad_() for t in args]
        got = [neg(t).requires_grad_() for t in args]
        y0, y1 = run(*want), run(*got)
        assert torch.equal(y0, y1), k
        dy = torch.randn(y0.shape, generator=g).cuda()
        for p, q in zip(torch.autograd.grad(y0, want, dy), torch.autograd.grad(y1, got, neg(dy))):
            assert torch.equal(p, q), k
        # the imaginary part of a conjugate is minus the values
        p, = torch.autograd.grad((run(*want) * dy).sum(), want[:1])
        q, = torch.autograd.grad((torch.complex(dy, run(*want)).conj().imag * -dy).sum(), want[:1])
        assert torch.equal(p, q), k


def test_update_forward_after_training_the_stage(dev):
    """Update.forward uses the parameters of the moment while `gru` is trained (f16, by a fused step)"""
    from dpvo_amd import net as N
    from tests import helpers as H
    torch.manual_seed(6)
    upd = N.Update(3).to(dev)
    ii, jj, kk, _ = H.small_graph(14, 8)
    E = ii.numel()
    ii, jj, kk = ii.to(dev), jj.to(dev), kk.to(dev)
    g = torch.Generator().manual_seed(0)
    net, inp, corr = (torch.randn(1, E, n, generator=g).cuda() * s for n, s in ((384, 1.0), (384, 0.5), (882, 0.5)))
    call = lambda u: u(net, inp.half(), corr.half(), None, ii, jj, kk)  # noqa: E731

    def fresh():
        u = N.Update(3).to(dev)
        u.load_state_dict(upd.state_dict())
        return u
    first = call(upd)
    opt = torch.optim.AdamW(upd.gru.parameters(), lr=0.05, fused=True)
    for _ in range(2):
        upd.gru(net.half()).float().square().mean().backward()
        call(upd)
        opt.step()
        now, want = call(upd), call(fresh())
        assert torch.equal(now[0], want[0]) and torch.equal(now[1][0], want[1][0]) and torch.equal(now[1][1], want[1][1])
    assert not torch.equal(now[0], first[0])
    upd.pack()
    P = upd.operands()
    assert upd.operands() is P and torch.equal(call(upd)[0], now[0])


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,D,H", [(3, 70, 40), (100, 70, 40), (300, 200, 150), (5000, 384, 385)])
def test_nan_shows_in_gradients_of_the_gated_residual(dev, t, M, D, H):
    """a NaN in a row, or in a hidden bias, reaches the gradients that it makes unknown -- the ReLU's mask does not turn it into a 0 -- and no others"""
    g = torch.Generator().manual_seed(M)
    x = make(g, M, D, t=t)
    wg, bg = layer(g, D, D, t)
    w1, b1 = layer(g, H, D, t)
    w2, b2 = layer(g, D, H, t)
    dy = make(g, M, D, t=t, grad=False)
    leaves = [x, wg, bg, w1, b1, w2, b2]
    d0 = torch.autograd.grad(blocks.gated_residual(*leaves), leaves, dy)
    with torch.no_grad():
        bad = [p.clone() for p in leaves]
        bad[0][1, 5] = float("nan")
    bad = [p.requires_grad_() for p in bad]
    y = blocks.gated_residual(*bad)
    d1 = torch.autograd.grad(y, bad, dy)
    keep = [i for i in range(M) if i != 1]
    assert y[1].isnan().all() and y[keep].isfinite().all()
    assert d1[0][1].isnan().all() and torch.equal(d1[0][keep], d0[0][keep])
    for got in d1[1:]:                                                          # every weight and bias sums over the bad row
        assert got.isnan().all()
    with torch.no_grad():
        bad = [p.clone() for p in leaves]
        bad[4][7] = float("nan")                                                # one hidden feature: of no row's gate, of every row's product
    bad = [p.requires_grad_() for p in bad]
    d1 = torch.autograd.grad(blocks.gated_residual(*bad), bad, dy)
    rows = [i for i in range(H) if i != 7]
    # the hidden layer's gradient is known but for that feature, where the formula has a NaN's derivative times a number
    assert torch.equal(d1[4][rows], d0[4][rows]) and torch.equal(d1[3][rows], d0[3][rows])
    assert torch.equal(d1[5][:, rows], d0[5][:, rows]) and d1[5][:, 7].isnan().all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(3, 20, 7), (200, 72, 90), (3000, 200, 130)])
def test_nan_passes_the_relus_derivative(dev, t, M, K, N):
    """relu of a NaN sum: the gradient that arrives goes on (as by a mask of `<= 0`), so that its bias and weights do not look clean"""
    g = torch.Generator().manual_seed(M)
    x, dy = make(g, M, K, t=t, grad=False), make(g, M, N, t=t, grad=False)
    w, b = layer(g, N, K, t)
    wu, _ = layer(g, N, K, t, False)
    with torch.no_grad():
        b[2] = float("nan")
    db, = torch.autograd.grad(blocks.linear(x, w, b, "relu"), b, dy)
    within(db[2:3], rows_f(dy[:, 2:3]).sum0(), t, "db")
    dw, db = torch.autograd.grad(blocks.gated_linear(x, w, wu, b, activation="relu"), (w, b), dy)
    U_ = proj(rows_f(x), rows_f(wu))
    d = rows_f(dy[:, 2:3]) * V(U_.v[:, 2:3], U_.e[:, 2:3])
    within(db[2:3], d.to(t).sum0(), t, "db gated")
    within(dw[2:3], d.to(t).t().mm(rows_f(x)), t, "dw gated")
    h, gate = make(g, M, N, t=t, grad=False), make(g, M, N, t=t, grad=False)
    gate[1, 3] = float("nan")
    gate.requires_grad_()
    s, _ = blocks.residual_norm(torch.zeros_like(h), h, norm=None, gate=gate, gate_activation="relu")
    got, = torch.autograd.grad(s, gate, dy)
    want = dy * h * (gate.detach() <= 0).logical_not()
    assert s[1, 3].isnan() and torch.equal(got, want)


@pytest.mark.parametrize("t", [BF16, F32], ids=str)
@pytest.mark.parametrize("a", list(blocks.ACTIVATIONS))
def test_derivatives_at_large_sums(dev, t, a):
    """sums of 1 to 2^120, of either sign, one to a row: far from 0 every derivative is 0 or 1 (the identity's: 1; the sigmoid's: 0)"""
    z = torch.tensor([s * 2.0 ** e for e in range(0, 121) for s in (1, -1)])[:, None].to(t).cuda()
    one = torch.ones(1, 1, dtype=t, device=dev)
    x = z.clone().requires_grad_()
    u = torch.ones_like(z).requires_grad_()
    Z = rows_f(z)
    v, d = act(a, Z)
    # (values of the 64-bit form where its own powers overflow: x^3 does not before 2^341)
    y = blocks.linear(x, one, None, a)
    within(y, v, t, "y")
    got, = torch.autograd.grad(y, x, torch.ones_like(y))
    # |z| >= 2^20: `act`'s bound of the derivative grows with |z|, the derivative does not
    far = (Z.v.abs() >= 2.0 ** 20).flatten()
    within(got[~far], V(d.v[~far], d.e[~far]), t, "dx")
    assert torch.equal(got[far].double().cpu(), d.v[far]), got[far].flatten()
    gx, gu = torch.autograd.grad(blocks.gated_linear(x, one, one, activation=a, up_input=u), (x, u), torch.ones_like(y))
    assert torch.equal(gx, got) and torch.equal(gu, y)


@pytest.mark.parametrize("tb", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("a,D", [("sigmoid", 384), ("silu", 384), ("sigmoid", 385), ("silu", 4000), ("sigmoid", 4104), ("silu", 5001)])
def test_gates_of_a_f32_stream_are_f32(dev, tb, a, D):
    """act(gate) where it is itself the f32 result (0 + gate * 1), and where it is a f32 gradient (of post_bias, over one row): 1 / (1 + e) from an
    exponential within a unit in the last place (2 U of e / (1 + e)), a sum and a division (U each), and silu's or the gradient's product (U): 5 U"""
    gate = torch.linspace(-20, 20, D).to(tb).cuda()
    v = act(a, rows_f(gate))[0].v
    x, one = torch.zeros(1, D, device=dev), torch.ones(1, D, dtype=tb, device=dev)
    s, _ = blocks.residual_norm(x, one, norm=None, gate=gate, gate_activation=a)
    within(s[0], V(v, 5 * U * v.abs()), F32, "s")
    pw, pb = torch.ones(D, device=dev), torch.zeros(D, device=dev, requires_grad=True)
    s, _ = blocks.residual_norm(x, one, norm=None, gate=gate, gate_activation=a, post_norm="rms", post_weight=pw, post_bias=pb)
    got, = torch.autograd.grad(s, pb, torch.ones_like(s))
    within(got, V(v, 5 * U * v.abs()), F32, "d post_bias")


def test_operand_images_on_another_stream(dev):
    """images that one stream has yet to write are used by a call on another only behind that, and last until that call is done"""
    from dpvo_amd import net as N
    from tests import helpers as H
    torch.manual_seed(7)
    upd = N.Update(3).to(dev)
    ii, jj, kk, _ = H.small_graph(14, 8)
    E = ii.numel()
    ii, jj, kk = ii.to(dev), jj.to(dev), kk.to(dev)
    g = torch.Generator().manual_seed(0)
    net, inp, corr = (torch.randn(1, E, n, generator=g).cuda() * s for n, s in ((384, 1.0), (384, 0.5), (882, 0.5)))
    call = lambda: upd(net, inp.half(), corr.half(), None, ii, jj, kk)[0]  # noqa: E731
    want = call()
    busy = torch.randn(8192, 8192, device=dev)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        assert torch.equal(call(), want)                                        # (plan and workspaces of this stream)
    torch.cuda.synchronize()
    for _ in range(3):
        y = busy
        for _ in range(6):
            y = y @ busy * 1e-4                                                 # some tens of milliseconds in front of the images
        upd.pack()
        kept = [torch.full_like(t, float("nan")) for t in upd._packed["_fw"]]   # (behind them: over memory that the last images left)
        with torch.cuda.stream(other):
            got = call()
            upd.pack()                                                          # the images of the call are dropped while it runs
            more = [torch.full_like(t, float("nan")) for t in upd._packed["_fw"]]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del kept, more
