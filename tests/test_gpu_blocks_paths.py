"""Every path that dpvo_amd.blocks chooses between, by sizes listed for it: each form, epilogue, tile and cut of the products, and the norms' loops
over several rows of a workgroup.  tests/test_blocks.py evaluates the library's own rules (dpvo_amd/csrc/blocks_plan.h) over a grid of sizes and sees
that the lists below reach whatever the rules return there.

Products are held to equality: inputs are whole numbers whose products and sums stay below 2^24, so that f32 sums are exact in any order, and a result
is the exact number rounded once -- a block of the sum left out, counted twice or taken from elsewhere shows at once.  Norms, activations and their
derivatives are held to the bounds that test_gpu_blocks.py carries along."""
import pytest
import torch

from dpvo_amd import blocks
from tests.test_gpu_blocks import BF16, F16, F32, TYPES, U, V, act, norm_back, normalise, on_gpu, proj, within

pytestmark = pytest.mark.gpu

# y [M,N] from x [M,K]: few rows by 4 and 16 waves and in groups of 64, tiles of 64 by four and two waves, of 128 and 256, parts of both
FORWARD = [(13, 200, 130), (7, 1030, 75), (70, 386, 200), (64, 2050, 33), (333, 517, 705), (333, 768, 2048), (517, 200, 5013), (1030, 705, 2050), (2050, 201, 3001),
           (100, 4200, 90), (100, 4201, 91), (705, 3000, 2050), (2055, 2600, 1027), (1540, 1030, 5013), (1301, 1091, 5121), (4096, 1024, 4096), (260, 1030, 9001)]
# dx [M,N] from a [M,K]
INPUT_GRADIENTS = [(13, 200, 130), (333, 517, 705), (517, 200, 5013), (2050, 201, 3001), (100, 4200, 90), (70, 1091, 1301), (705, 3000, 2050), (2055, 2600, 1027),
                   (1540, 1030, 5013), (4100, 1091, 2050), (4096, 1024, 4096)]
# dw [N,K] over M rows, one product after the other
WEIGHT_GRADIENTS = [(13, [(130, 200)]), (333, [(2048, 768), (2048, 768), (768, 2048)]), (517, [(5013, 200)]), (201, [(2050, 3001)]), (4201, [(100, 90), (35, 70)]),
                    (1301, [(90, 33), (33, 90), (7, 5), (1, 1)]), (20011, [(705, 386), (386, 705)]), (20011, [(386, 386)]), (1091, [(2050, 2050), (2050, 2050), (700, 2050)]),
                    (4096, [(4096, 1024), (4096, 1024), (1024, 4096)])]


def whole(g, *shape, t, top=1):
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(t)


def gen(*a):
    return torch.Generator(device="cuda").manual_seed(sum(x * 7 ** i for i, x in enumerate(a)) % 2 ** 31)


def exactly(got, want, t, what):
    """want: whole numbers in 64 bits"""
    assert float(want.abs().max()) < 2.0 ** 24 and got.dtype == t, what
    bad = got != want.to(t)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} differ, the first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", FORWARD)
def test_forward_products(dev, t, M, K, N):
    g = gen(M, K, N)
    x, v, w, wu = whole(g, M, K, t=t), whole(g, M, K + 2, t=t), whole(g, N, K, t=t), whole(g, N, K, t=t)
    wv, b, bu, res = whole(g, N, K + 2, t=t), whole(g, N, t=t, top=5), whole(g, N, t=t, top=5), whole(g, M, N, t=t, top=9)
    d = [p.double() for p in (x, v, w, wu, wv, b, bu, res)]
    G, S, R = d[0] @ d[2].t() + d[5], d[0] @ d[3].t() + d[6], d[1] @ d[4].t() + d[6]
    exactly(blocks.linear(x, w, b), G, t, "linear")
    exactly(blocks.linear(x, w), G - d[5], t, "linear without a bias")
    exactly(blocks.linear(x, w, b, "relu"), G.clamp(min=0), t, "linear relu")
    exactly(blocks.gated_linear(x, w, wu, b, bu, "identity"), G * S, t, "gated, one input")
    exactly(blocks.gated_linear(x, w, wu, b, bu, "relu", residual=res), G.clamp(min=0) * S + d[7], t, "gated, one input, residual")
    exactly(blocks.gated_linear(x, w, wv, b, bu, "relu", up_input=v, residual=res), G.clamp(min=0) * R + d[7], t, "gated, two inputs")
    for got, want in zip(blocks._forward(x, w, b, 1, save=True), (G.clamp(min=0), G)):
        exactly(got, want, got.dtype, "linear, saved")
    for got, want in zip(blocks._forward(x, w, b, 0, None, wu, bu, None, True), (G * S, G, S)):
        exactly(got, want, got.dtype, "one input, saved")
    for got, want in zip(blocks._forward(x, w, b, 0, v, wv, bu, None, True), (G * R, G, R)):
        exactly(got, want, got.dtype, "two inputs, saved")
    x, w, wu = x * 0.25, w * 0.5, wu * 0.5
    f = on_gpu
    z, up = proj(f(x), f(w), f(b)), proj(f(x), f(wu), f(bu))
    for a in ("sigmoid", "silu", "gelu", "gelu_tanh"):
        ya = act(a, z)[0]
        within(blocks.linear(x, w, b, a), ya, t, a)
        within(blocks.gated_linear(x, w, wu, b, bu, a), ya * up, t, f"gated {a}")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", INPUT_GRADIENTS)
def test_input_gradient_products(dev, t, M, K, N):
    g = gen(M, K, N, 1)
    a, b, a2, b2 = whole(g, M, K, t=t), whole(g, K, N, t=t), whole(g, M, K + 5, t=t), whole(g, K + 5, N, t=t)
    add, gate, up = whole(g, M, N, t=t, top=9), whole(g, M, N, t=F32, top=9), whole(g, M, N, t=F32, top=9)
    C = a.double() @ b.double()
    C2 = C + a2.double() @ b2.double()
    exactly(blocks._dx([(a, b)])[0], C, t, "one")
    exactly(blocks._dx([(a, b), (a2, b2)])[0], C2, t, "two")
    exactly(blocks._dx([(a, b), (a2, b2)], addend=add)[0], C2 + add.double(), t, "two and an addend")
    for act_code, y, slope in ((0, gate, torch.ones_like(gate)), (1, gate.clamp(min=0), (gate > 0).float())):
        dg, du = blocks._dx([(a, b)], gate=gate, up=up, act=act_code)
        exactly(dg, C * up.double() * slope.double(), t, "through a gate")
        exactly(du, C * y.double(), t, "through a product")
        exactly(blocks._dx([(a, b)], gate=gate, act=act_code)[0], C * slope.double(), t, "through an activation")
    m = gate.to(t)
    exactly(blocks._dx([(a, b)], mask=m)[0], torch.where(m > 0, C, 0.0), t, "masked")
    exactly(blocks._dx([(a, b), (a2, b2)], mask=m)[0], torch.where(m > 0, C2, 0.0), t, "two, masked")
    gate = gate / 4
    for name in ("sigmoid", "silu", "gelu", "gelu_tanh"):
        ya, da = act(name, V(gate.double()))
        dg, du = blocks._dx([(a, b)], gate=gate, up=up, act=blocks.ACTIVATIONS[name])
        within(dg, V(C) * V(up.double()) * da, t, f"through a gate, {name}")
        within(du, V(C) * ya, t, f"through a product, {name}")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,sizes", WEIGHT_GRADIENTS)
def test_weight_gradient_products(dev, t, M, sizes):
    g = gen(M, len(sizes), sizes[0][0], 2)
    for db in (True, False):
        jobs = [(whole(g, M, N, t=t), whole(g, M, K, t=t), True, db and i != 1) for i, (N, K) in enumerate(sizes)]
        for i, ((a, b, _, want_b), (dw, got_b)) in enumerate(zip(jobs, blocks._dw(jobs))):
            exactly(dw, a.double().t() @ b.double(), t, f"dw {i}")
            assert (got_b is not None) == want_b
            if want_b:
                exactly(got_b, a.double().sum(0), t, f"db {i}")


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("M,K,N", [(1540, 1030, 5013), (4096, 1024, 4096), (260, 1030, 9001)])
def test_gated_linear_of_the_largest_tile(dev, t, M, K, N):
    """one input, both sums saved, and every gradient, where the product of the two runs on 256-wide tiles"""
    g = gen(M, K, N, 3)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device=dev) * scale).to(t).requires_grad_()  # noqa: E731
    x, w, wu, b, bu = r(M, K), r(N, K, scale=K ** -0.5), r(N, K, scale=K ** -0.5), r(N), r(N)
    dy = r(M, N).detach()
    y = blocks.gated_linear(x, w, wu, b, bu, "silu")
    f = on_gpu
    G, S = proj(f(x), f(w), f(b)), proj(f(x), f(wu), f(bu))
    ya, da = act("silu", G)
    within(y, ya * S, t, "y")
    with torch.no_grad():
        assert torch.equal(y, blocks.gated_linear(x, w, wu, b, bu, "silu"))
    grads = torch.autograd.grad(y, [x, w, wu, b, bu], dy)
    dg, du = (f(dy) * S * da).to(t), (f(dy) * ya).to(t)
    want = [dg.mm(f(w)) + du.mm(f(wu)), dg.t().mm(f(x)), du.t().mm(f(x)), dg.sum0(), du.sum0()]
    for name, got, q in zip(("dx", "dw", "dwu", "db", "dbu"), grads, want):
        within(got, q, t, name)


# ------------------------------------------------------------------------------------------------------------------ norms
# leading sizes, D, the gate's leading sizes (None: no gate): several rounds of rows in a workgroup, forward and backward, for every number of lanes
# with whole and ragged rows; parts of a group of several rounds; several groups in a workgroup, the last workgroup short of some
NORMS = [
    ((40000,), 100, (1,)), ((140000,), 104, (1,)), ((20011,), 201, (1,)), ((70003,), 200, (1,)), ((9001,), 385, (1,)), ((33003,), 384, (1,)),
    ((5001,), 1001, (1,)), ((8300,), 520, (1,)), ((2501,), 2001, (1,)), ((8200,), 1032, (1,)), ((2101,), 3001, (1,)), ((8201,), 2056, (1,)),
    ((700,), 4104, (1,)), ((8200,), 4104, None), ((400,), 4097, (1,)), ((8193,), 5001, None), ((300,), 9000, (1,)), ((400,), 8193, (1,)),
    ((5001,), 1001, (5001,)), ((33003,), 384, None), ((700,), 4104, (700,)),
    ((4, 2501), 385, (4, 1)), ((3, 7001), 104, (3, 1)), ((5, 601), 2056, (5, 1)), ((7, 333), 1001, (7, 1)), ((3, 201), 4104, (3, 1)), ((3, 150), 5001, (3, 1)),
    ((1500, 3), 65, (1500, 1)), ((1501, 3), 200, (1501, 1)), ((2500, 5), 385, (2500, 1)), ((1025, 17), 104, (1025, 1)), ((4100, 2), 520, (4100, 1)), ((2100, 2), 1001, (2100, 1)),
    ((1501, 2), 2000, (1501, 1)), ((1100, 3), 1601, (1100, 1)), ((700, 2), 3001, (700, 1)), ((1030, 2), 2056, (1030, 1)), ((600, 2), 4104, (600, 1)), ((300, 2), 4097, (300, 1)),
    ((301, 2), 9000, (301, 1)), ((5000, 9), 201, (5000, 1)), ((1501, 3), 384, (1501, 1)), ((3, 5001), 384, (3, 1)),
]
# ... of a bare branch (the 1024-lane form of 16-bit rows holds four sums)
NORMS_PLAIN = [((301, 2), 4104, (301, 1)), ((3, 301), 8000, (3, 1)), ((800,), 4104, (1,)), ((300, 4), 64, (300, 1))]
NORM_ALONE = [(20011, 100), (9001, 200), (5001, 384), (5001, 1000), (2501, 2000), (1301, 4096), (700, 8192), (300, 8192), (300, 8193)]
NORM_TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)]


def sum_rows(z, k):
    """over groups of k rows: a lane's rounds, the row slots (16), the workgroups' parts in 16 shares of at most 256, the shares: that many additions
    of f32 after one another at most"""
    M, D = z.v.shape
    n = 300 + k // 1000
    s = lambda q: q.reshape(M // k, k, D).sum(1)  # noqa: E731
    return V(s(z.v), s(z.e) + n * U * s(z.top()))


@pytest.mark.parametrize("tx,tb", NORM_TYPES, ids=str)
@pytest.mark.parametrize("lead,D,gate", NORMS + NORMS_PLAIN)
def test_norm_rows(dev, tx, tb, lead, D, gate):
    g = gen(D, *lead)
    kind, post = ("layer", "rms") if (lead[0] + D) % 2 else ("rms", "layer")
    post = None if (lead, D, gate) in NORMS_PLAIN else post
    r = lambda *s, t, scale=1.0, mean=0.0: (torch.randn(*s, generator=g, device=dev) * scale + mean).to(t).requires_grad_()  # noqa: E731
    x, f = r(*lead, D, t=tx, scale=1.5, mean=0.25), r(*lead, D, t=tb, scale=1.2, mean=-0.2)
    ga = None if gate is None else r(*gate, D, t=tb)
    tp = tx if lead[0] < 100000 else F32                                        # (sums of 140 000 pass what f16 holds)
    w, b, pw, pb = r(D, t=tp, scale=0.2, mean=1.0), r(D, t=tp, scale=0.2), r(D, t=tp, scale=0.2, mean=1.0), r(D, t=tp, scale=0.2)
    ds, dh = r(*lead, D, t=tx, mean=0.5).detach(), r(*lead, D, t=tb, mean=0.5).detach()
    s, h = blocks.residual_norm(x, f, w, b, norm=kind, eps=1e-3, gate=ga, gate_activation="sigmoid", scale=0.5, post_norm=post,
                                post_weight=pw if post else None, post_bias=pb if post else None)
    M = x.numel() // D
    R = lambda q: V(q.detach().double().reshape(-1, D))  # noqa: E731
    par = lambda q: V(q.detach().double())  # noqa: E731
    if post:
        fh, fr = normalise(R(f), post, 1e-3)
        P = fh * par(pw) + par(pb)
    else:
        P = R(f)
    c = V(torch.full((1, 1), 0.5, dtype=torch.float64, device=dev))
    if ga is not None:
        A, dA = act("sigmoid", V(ga.detach().double().expand(*lead, D).reshape(M, D)))
        inc = A * P
    else:
        inc = P
    S = R(x) + inc * c
    within(s, S, tx, "s")
    sh, sr = normalise(S, kind, 1e-3)
    within(h, sh * par(w) + par(b), tb, "h")
    leaves = {"x": x, "f": f, "w": w, "b": b, **({"pw": pw, "pb": pb} if post else {}), **({} if ga is None else {"gate": ga})}
    grads = dict(zip(leaves, torch.autograd.grad([s, h], list(leaves.values()), [ds, dh])))
    Dh = R(dh)
    DY = norm_back(Dh * par(w), sh, sr, kind) + R(ds)
    within(grads["x"], DY, tx, "dx")
    q = DY * c
    if ga is not None:
        dga, k = q * P * dA, M // (ga.numel() // D)
        within(grads["gate"], dga if k == 1 else sum_rows(dga, k), tb, "dgate")
        q = q * A
    within(grads["f"], norm_back(q * par(pw), fh, fr, post) if post else q, tb, "df")
    for name, want in [("w", Dh * sh), ("b", Dh)] + ([("pw", q * fh), ("pb", q)] if post else []):
        within(grads[name], sum_rows(want, M), tp, name)


@pytest.mark.parametrize("tx,th", NORM_TYPES, ids=str)
@pytest.mark.parametrize("M,D", NORM_ALONE)
def test_norm_alone_rows(dev, tx, th, M, D):
    """`norm` with two sums (the 1024-lane form up to 8192 in 16 bits among them)"""
    g = gen(M, D, 4)
    kind = "rms" if (M + D) % 2 else "layer"
    x, dh = (torch.randn(M, D, generator=g, device=dev) * 1.5 + 0.5).to(tx).requires_grad_(), (torch.randn(M, D, generator=g, device=dev) + 0.5).to(th)
    w, b = ((torch.randn(D, generator=g, device=dev) * 0.2 + 1.0).to(tx).requires_grad_() for _ in range(2))
    h = blocks.norm(x, w, b, kind, eps=1e-3, out_dtype=th)
    R = lambda q: V(q.detach().double())  # noqa: E731
    xh, r = normalise(R(x), kind, 1e-3)
    within(h, xh * R(w) + R(b), th, "h")
    dx, dw, db = torch.autograd.grad(h, [x, w, b], dh)
    within(dx, norm_back(R(dh) * R(w), xh, r, kind), tx, "dx")
    within(dw, sum_rows(R(dh) * xh, M), tx, "dw")
    within(db, sum_rows(R(dh), M), tx, "db")


@pytest.mark.parametrize("tb", [F16, BF16], ids=str)
@pytest.mark.parametrize("lead,D,gate", [((5,), 7, (5,)), ((300,), 384, (1,)), ((40, 3), 385, (40, 1)), ((9,), 2056, None), ((30,), 3001, (30,)), ((20,), 4104, (1,)), ((11,), 9001, (11,))])
def test_f32_rows_behind_a_16_bit_branch(dev, tb, lead, D, gate):
    """x, s and h in f32, branch and gate in 16 bits (`out_dtype` x's): h's gradient arrives in f32"""
    g = gen(D, *lead, 5)
    r = lambda *s, t, mean=0.0: (torch.randn(*s, generator=g, device=dev) + mean).to(t).requires_grad_()  # noqa: E731
    x, f, w, b = r(*lead, D, t=F32), r(*lead, D, t=tb), r(D, t=F32, mean=1.0), r(D, t=F32)
    ga = None if gate is None else r(*gate, D, t=tb)
    ds, dh = r(*lead, D, t=F32).detach(), r(*lead, D, t=F32).detach()
    s, h = blocks.residual_norm(x, f, w, b, gate=ga, gate_activation="silu", out_dtype=F32)
    M = x.numel() // D
    R = lambda q: V(q.detach().double().reshape(-1, D))  # noqa: E731
    par = lambda q: V(q.detach().double())  # noqa: E731
    A, dA = (V(torch.ones(M, D, dtype=torch.float64, device=dev)), None) if ga is None else act("silu", V(ga.detach().double().expand(*lead, D).reshape(M, D)))
    S = R(x) + R(f) * A
    within(s, S, F32, "s")
    sh, sr = normalise(S, "layer", 1e-3)
    within(h, sh * par(w) + par(b), F32, "h")
    leaves = {"x": x, "f": f, "w": w, "b": b, **({} if ga is None else {"gate": ga})}
    grads = dict(zip(leaves, torch.autograd.grad([s, h], list(leaves.values()), [ds, dh])))
    DY = norm_back(R(dh) * par(w), sh, sr, "layer") + R(ds)
    within(grads["x"], DY, F32, "dx")
    within(grads["f"], DY * A, tb, "df")
    within(grads["w"], sum_rows(R(dh) * sh, M), F32, "dw")
    within(grads["b"], sum_rows(R(dh), M), F32, "db")
    if ga is not None:
        dga, k = DY * R(f) * dA, M // (ga.numel() // D)
        within(grads["gate"], dga if k == 1 else sum_rows(dga, k), tb, "dgate")
