"""dpvo_amd.blocks on the host: what each operator refuses, the C entries' argument checks, and the ctypes mirrors of their structs.  (No GPU.)"""
import ctypes
import os
import subprocess

import pytest
import torch

from dpvo_amd import _lib as L
from dpvo_amd import blocks

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
z = torch.zeros
H, D = torch.float16, torch.float64


@pytest.mark.parametrize("call,why", [
    (lambda: blocks.linear(z(3, 4), z(5, 3)), "its input has 4 features"),
    (lambda: blocks.linear(z(3, 4), z(5, 4, 1)), "its input has 4 features"),
    (lambda: blocks.linear(z(()), z(5, 4)), "no feature dimension"),
    (lambda: blocks.linear(z(3, 0), z(5, 0)), "no features"),
    (lambda: blocks.linear(z(3, 4), z(0, 4)), "no features"),
    (lambda: blocks.linear(z(3, 4), z(5, 4), z(4)), "bias of weight"),
    (lambda: blocks.linear(z(3, 4), z(5, 4, dtype=H)), "must have the input's dtype"),
    (lambda: blocks.linear(z(3, 4), z(5, 4), z(5, dtype=H)), "must have the input's dtype"),
    (lambda: blocks.linear(z(3, 4, dtype=D), z(5, 4, dtype=D)), "unsupported dtype"),
    (lambda: blocks.linear(z(3, 4, dtype=torch.int32), z(5, 4, dtype=torch.int32)), "unsupported dtype"),
    (lambda: blocks.linear(z(3, 4), z(5, 4), activation="tanh"), "activation is 'tanh'"),
    (lambda: blocks.linear(z(3, 4), z(5, 4), activation=None), "activation is None"),
    (lambda: blocks.linear(z(3, 4), z(5, 4, device="meta")), "tensors on cpu and meta"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(6, 4)), "w_gate makes 5 features, w_up 6"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), up_input=z(2, 4)), "up_input"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), up_input=z(1, 3, 4)), "up_input"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), up_input=z(3, 7)), "its input has 7 features"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), up_input=z(3, 4, dtype=H)), "up_input"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), residual=z(3, 4)), "residual"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), residual=z(5)), "residual"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), residual=z(3, 5, dtype=H)), "residual"),
    (lambda: blocks.gated_feed_forward(z(3, 4), z(5, 4), z(5, 4), z(4, 6)), "its input has 5 features"),
    (lambda: blocks.gated_feed_forward(z(3, 4), z(5, 4), z(5, 4), z(4, 5), b_down=z(5)), "bias of w_down"),
    (lambda: blocks.gated_residual(z(3, 4), z(5, 4), None, z(6, 4), None, z(4, 6), None), "must make x's 4 features"),
    (lambda: blocks.gated_residual(z(3, 4), z(4, 4), None, z(6, 4), None, z(5, 6), None), "must make x's 4 features"),
    (lambda: blocks.gated_residual(z(3, 4), z(4, 4), None, z(6, 4), None, z(4, 5), None), "its input has 6 features"),
    (lambda: blocks.norm(z(3, 4), z(5)), "weight is (5,)"),
    (lambda: blocks.norm(z(3, 4), z(4), z(4, dtype=H)), "all of one dtype"),
    (lambda: blocks.norm(z(3, 4), z(4, dtype=D)), "parameters are"),
    (lambda: blocks.norm(z(3, 0)), "rows of 0 elements"),
    (lambda: blocks.norm(z(1, 16385)), "rows of 16385 elements"),
    (lambda: blocks.norm(z(3, 4), kind="batch"), "kind is 'batch'"),
    (lambda: blocks.norm(z(3, 4), kind=None), "kind is None"),
    (lambda: blocks.norm(z(3, 4, dtype=H), out_dtype=torch.float32), "out_dtype"),
    (lambda: blocks.norm(z(3, 4), out_dtype=D), "out_dtype"),
    (lambda: blocks.residual_norm(z(3, 4), z(2, 4)), "branch"),
    (lambda: blocks.residual_norm(z(3, 4, dtype=H), z(3, 4)), "branch"),
    (lambda: blocks.residual_norm(z(3, 4, dtype=H), z(3, 4, dtype=torch.bfloat16)), "branch"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), gate=z(2, 4)), "gate (2, 4) must be shaped"),
    (lambda: blocks.residual_norm(z(2, 3, 4), z(2, 3, 4), gate=z(3, 4)), "must be shaped"),
    (lambda: blocks.residual_norm(z(2, 3, 4), z(2, 3, 4), gate=z(1, 3, 4)), "must be shaped"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), gate=z(3, 1)), "does not go with x"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), gate=z(1, 3, 4)), "does not go with x"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), gate=z(3, 4, dtype=H)), "gate is torch.float16"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), gate=z(4), gate_activation="gelu"), "gate_activation is 'gelu'"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), z(4), norm=None), "without a norm"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), post_weight=z(4)), "without a post_norm"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4), z(4), post_norm="rms", post_weight=z(4, dtype=H)), "all of one dtype"),
    (lambda: blocks.residual_norm(z(3, 4), z(3, 4, dtype=H), out_dtype=torch.bfloat16), "out_dtype"),
    # right in every other respect: there is no CPU path
    (lambda: blocks.linear(z(3, 4), z(5, 4), z(5)), "run on the GPU only"),
    (lambda: blocks.gated_linear(z(3, 4), z(5, 4), z(5, 4), residual=z(3, 5)), "run on the GPU only"),
    (lambda: blocks.gated_feed_forward(z(3, 4), z(5, 4), z(5, 4), z(4, 5)), "run on the GPU only"),
    (lambda: blocks.gated_residual(z(3, 4), z(4, 4), None, z(6, 4), z(6), z(4, 6), None), "run on the GPU only"),
    (lambda: blocks.norm(z(3, 4), z(4), z(4)), "run on the GPU only"),
    (lambda: blocks.residual_norm(z(2, 3, 4), z(2, 3, 4), z(4), gate=z(2, 1, 4)), "run on the GPU only"),
])
def test_refusals(call, why):
    with pytest.raises(L.DPVOHipError, match=None) as e:
        call()
    assert why in str(e.value), str(e.value)


def test_rows_and_gate_rows():
    """the leading dimension that a view is handed on with, and how many gate rows a shape stands for"""
    t = z(6, 5, 8)
    assert blocks._rows(t)[1] == 8 and blocks._rows(t)[0].shape == (30, 8)
    v = z(10, 12)[:, :8]
    assert blocks._rows(v)[1] == 12 and blocks._rows(v)[0].data_ptr() == v.data_ptr()
    assert blocks._rows(z(8, 10).t())[1] == 8                                  # elements apart: copied
    assert blocks._rows(z(1, 8).expand(4, 8))[1] == 8                          # rows on top of each other: copied
    assert blocks._rows(z(8))[0].shape == (1, 8)
    assert blocks._rows(z(0, 3, 8))[0].shape == (0, 8)
    big = torch.empty(2, 5_000_000, dtype=H)[:, :8]
    assert blocks._rows(big)[1] == 8                                           # too far apart for 32-bit offsets in a tile: copied
    g = lambda x, s: blocks._gate_rows("t", z(*x), z(*s))  # noqa: E731
    assert g((2, 3, 4), (4,)) == g((2, 3, 4), (1, 4)) == g((2, 3, 4), (1, 1, 4)) == 1
    assert g((2, 3, 4), (2, 1, 4)) == 2 and g((2, 3, 4), (2, 3, 4)) == 6 and g((1, 3, 4), (3, 4)) == 3 and g((0, 4), (0, 4)) == 0


def test_entries_check_their_arguments():
    """error codes before anything touches the device"""
    lib, null, INVALID, UNSUPPORTED, WORKSPACE = L.lib(), None, -1, -2, -3
    one = ctypes.addressof(ctypes.c_int64(0))                                   # an address that no accepted call reads
    p = L.GatedLinear()
    assert lib.dpvo_gated_linear(null, null, 0, null) == INVALID and lib.dpvo_gated_linear_workspace_bytes(null) == 0
    assert lib.dpvo_gated_linear(ctypes.byref(p), null, 0, null) == 0           # no rows: nothing to do
    ok = dict(x=one, w_gate=one, y=one, ldx=64, ldwg=64, ldy=32, M=70, N=32, K=64, dtype=0)

    def call(**kw):
        q = L.GatedLinear()
        for k, v in {**ok, **kw}.items():
            setattr(q, k, v)
        return lib.dpvo_gated_linear(ctypes.byref(q), null, 0, null)
    for bad in (dict(M=-1), dict(N=-1), dict(K=-1), dict(Kv=-1), dict(dtype=3), dict(activation=6), dict(activation=-1), dict(x=None), dict(y=None),
                dict(w_gate=None), dict(ldx=63), dict(ldwg=63), dict(ldy=31), dict(residual=one, ldr=31), dict(w_up=one, Kv=8, ldv=8, ldwu=8, v=None),
                dict(w_up=one, v=one, Kv=8, ldv=7, ldwu=8), dict(w_up=one, v=one, Kv=8, ldv=8, ldwu=7), dict(ldx=2 ** 31)):
        assert call(**bad) == INVALID, bad
    q = L.GatedLinear()
    for k, v in {**ok, "M": 100, "N": 64, "K": 64 * 64, "ldx": 64 * 64, "ldwg": 64 * 64, "ldy": 64}.items():
        setattr(q, k, v)
    assert lib.dpvo_gated_linear_workspace_bytes(ctypes.byref(q)) > 0 and lib.dpvo_gated_linear(ctypes.byref(q), null, 0, null) == WORKSPACE
    assert lib.dpvo_gated_linear_dact(null, 4, null, null, null, null, 4, 0, 0, 3, 4, null) == INVALID
    assert lib.dpvo_gated_linear_dact(null, 4, null, null, null, null, 4, 0, 0, 0, 4, null) == 0
    assert lib.dpvo_gated_linear_dact(one, 4, one, one, one, null, 4, 0, 3, 3, 4, null) == INVALID
    assert lib.dpvo_gated_linear_dact(one, 3, one, null, one, null, 4, 0, 3, 3, 4, null) == INVALID

    def dx(**kw):
        q = L.GatedLinearDx()
        q.a[0] = q.b[0] = q.dx = one
        q.lda[0], q.ldb[0], q.K[0], q.lddx, q.M, q.N = 64, 32, 64, 32, 70, 32
        for k, v in kw.items():
            if isinstance(v, tuple):
                getattr(q, k)[v[0]] = v[1]
            else:
                setattr(q, k, v)
        return q, lib.dpvo_gated_linear_dx(ctypes.byref(q), null, 0, null)
    assert lib.dpvo_gated_linear_dx(null, null, 0, null) == INVALID and lib.dpvo_gated_linear_dx_workspace_bytes(null) == 0
    for bad in (dict(M=-1), dict(N=-2), dict(K=(0, -1)), dict(dtype=7), dict(activation=9), dict(a=(0, None)), dict(b=(0, None)), dict(dx=None), dict(lda=(0, 63)),
                dict(ldb=(0, 31)), dict(lddx=31), dict(addend=one, ldadd=3), dict(mask=one, ldmask=3), dict(gate=one, mask=one, ldmask=32), dict(up=one),
                dict(gate=one, up=one)):
        assert dx(**bad)[1] == INVALID, bad
    assert dx(gate=one, addend=one, ldadd=32)[1] == UNSUPPORTED
    q, rc = dx(M=64, N=64, K=(0, 64 * 64), lda=(0, 64 * 64), ldb=(0, 64), lddx=64)
    assert rc == WORKSPACE and lib.dpvo_gated_linear_dx_workspace_bytes(ctypes.byref(q)) >= 2 * 64 * 64 * 4

    def dw(**kw):
        q = L.GatedLinearDw()
        q.a[0] = q.b[0] = q.dw[0] = one
        q.lda[0], q.ldb[0], q.N[0], q.K[0], q.M, q.n = 32, 64, 32, 64, 70, 1
        for k, v in kw.items():
            if isinstance(v, tuple):
                getattr(q, k)[v[0]] = v[1]
            else:
                setattr(q, k, v)
        return lib.dpvo_gated_linear_dw(ctypes.byref(q), null, 0, null)
    for bad in (dict(M=-1), dict(n=5), dict(n=-1), dict(dtype=3), dict(N=(0, -1)), dict(K=(0, -1)), dict(a=(0, None)), dict(b=(0, None)), dict(dw=(0, None)),
                dict(lda=(0, 31)), dict(ldb=(0, 63))):
        assert dw(**bad) == INVALID, bad
    assert dw(n=0) == 0 and dw(M=45312) == WORKSPACE

    def rn(back=False, **kw):
        q = L.ResidualNorm()
        q.x = q.f = q.s = q.h = one
        q.ldx = q.ldf = q.D = 32
        q.M, q.groups, q.x_dtype, q.f_dtype, q.h_dtype, q.w_dtype, q.norm, q.scale = 5, 5, 1, 1, 1, 1, 1, 1.0
        for k, v in kw.items():
            setattr(q, k, v)
        return lib.dpvo_residual_norm_backward(ctypes.byref(q), null, 0, null) if back else lib.dpvo_residual_norm(ctypes.byref(q), null)
    assert lib.dpvo_residual_norm(null, null) == INVALID and lib.dpvo_residual_norm_backward(null, null, 0, null) == INVALID
    for bad in (dict(M=-1), dict(D=0), dict(x_dtype=3), dict(f_dtype=-1), dict(w_dtype=9), dict(norm=3), dict(post=-1), dict(gate_activation=7), dict(x=None),
                dict(gate=one, ldgate=32, groups=0), dict(gate=one, ldgate=32, groups=2), dict(gate=one, ldgate=31), dict(ldx=31), dict(ldf=31), dict(h=None),
                dict(norm=0, s=None), dict(gate=one, ldgate=32, f=None)):
        assert rn(**bad) == INVALID, bad
    for bad in (dict(x_dtype=0), dict(h_dtype=2), dict(D=16385, ldx=16385, ldf=16385), dict(gate_activation=4), dict(M=2 ** 31)):
        assert rn(**bad) == UNSUPPORTED, bad
    assert rn(M=0) == 0
    for bad in (dict(ds=one, ldds=3), dict(dh=one, lddh=3), dict(dgate=one), dict(f=None, df=one), dict(dpw=one)):
        assert rn(True, **bad) == INVALID, bad
    assert rn(True, dh=one, lddh=32, dw=one) == WORKSPACE
    assert rn(True, M=0) == 0
    # a size without a workspace behind it
    big = 1 << 40
    q = L.GatedLinear(**{**ok, "M": 100, "N": 64, "K": 64 * 64, "ldx": 64 * 64, "ldwg": 64 * 64, "ldy": 64})
    assert lib.dpvo_gated_linear(ctypes.byref(q), null, big, null) == WORKSPACE
    q, _ = dx(M=64, N=64, K=(0, 64 * 64), lda=(0, 64 * 64), ldb=(0, 64), lddx=64)
    assert lib.dpvo_gated_linear_dx(ctypes.byref(q), null, big, null) == WORKSPACE
    q = L.GatedLinearDw((one,), (one,), (one,), (), (32,), (64,), (32,), (64,), 45312, 1, 0)
    assert lib.dpvo_gated_linear_dw_workspace_bytes(ctypes.byref(q)) > 0 and lib.dpvo_gated_linear_dw(ctypes.byref(q), null, big, null) == WORKSPACE
    for D in (32, 5000):
        q = L.ResidualNorm(x=one, dh=one, dw=one, ldx=D, lddh=D, D=D, M=5, x_dtype=1, f_dtype=1, h_dtype=1, w_dtype=1, norm=1)
        assert lib.dpvo_residual_norm_backward_workspace_bytes(ctypes.byref(q)) > 0 and lib.dpvo_residual_norm_backward(ctypes.byref(q), null, big, null) == WORKSPACE


def test_structs_match_the_header(tmp_path):
    probes = {"dpvo_gated_linear_t": L.GatedLinear, "dpvo_gated_linear_dx_t": L.GatedLinearDx, "dpvo_gated_linear_dw_t": L.GatedLinearDw,
              "dpvo_residual_norm_t": L.ResidualNorm}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dpvo_hip.h"', 'int main(void) {']
    for c, cls in probes.items():
        lines.append(f'  printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "probe")])
    out = dict(l.split() for l in subprocess.check_output([str(tmp_path / "probe")], text=True).splitlines())
    for c, cls in probes.items():
        assert int(out[c]) == ctypes.sizeof(cls), c
        for f, _ in cls._fields_:
            assert int(out[f"{c}.{f}"]) == getattr(cls, f).offset, (c, f)
    hdr = open(os.path.join(ROOT, "include", "dpvo_hip.h")).read()
    import re
    codes = {k: int(v) for k, v in re.findall(r"#define DPVO_((?:ACT|NORM)_[A-Z_]+|F16|F32|BF16) (\d+)", hdr)}
    assert {k: codes["ACT_" + k.upper()] for k in blocks.ACTIVATIONS} == blocks.ACTIVATIONS
    assert {"layer": codes["NORM_LAYER"], "rms": codes["NORM_RMS"], None: codes["NORM_NONE"]} == blocks.NORMS
    assert (codes["F16"], codes["F32"], codes["BF16"]) == (L.F16, L.F32, L.BF16)


def test_state_dict_keys_stay():
    """the stage that became callable keeps its names in a checkpoint"""
    from dpvo_amd import net as N
    keys = list(N.Update(3).gru.state_dict())
    assert keys == ["0.weight", "0.bias"] + [f"1.{k}.{w}" for k in ("gate.0", "res.0", "res.2") for w in ("weight", "bias")] + ["2.weight", "2.bias"] + \
        [f"3.{k}.{w}" for k in ("gate.0", "res.0", "res.2") for w in ("weight", "bias")]


# ------------------------------------------------------------------------------------------------------------------ what torch records elsewhere
# every operator with tensors t(name, shape) in the place of its inputs: `make(f)` is one call with f around the named one
CALLS = [
    ("linear", lambda t: blocks.linear(t("x", 3, 4), t("w", 5, 4), t("b", 5))),
    ("gated_linear", lambda t: blocks.gated_linear(t("x", 3, 4), t("w", 5, 4), t("wu", 5, 4), t("b", 5), t("bu", 5), up_input=t("v", 3, 4), residual=t("r", 3, 5))),
    ("gated_feed_forward", lambda t: blocks.gated_feed_forward(t("x", 3, 4), t("w", 5, 4), t("wu", 5, 4), t("wd", 4, 5), t("b", 5), t("bu", 5), t("bd", 4))),
    ("gated_residual", lambda t: blocks.gated_residual(t("x", 3, 4), t("w", 4, 4), t("b", 4), t("w1", 6, 4), t("b1", 6), t("w2", 4, 6), t("b2", 4))),
    ("norm", lambda t: blocks.norm(t("x", 3, 4), t("w", 4), t("b", 4))),
    ("residual_norm", lambda t: blocks.residual_norm(t("x", 3, 4), t("f", 3, 4), t("w", 4), t("b", 4), gate=t("gate", 4), post_norm="layer",
                                                     post_weight=t("pw", 4), post_bias=t("pb", 4))),
]


def names_of(call):
    names = []

    def t(name, *shape):
        names.append(name)
        return z(*shape)
    with pytest.raises(L.DPVOHipError, match="run on the GPU only"):
        call(t)
    return names


@pytest.mark.parametrize("what,call", CALLS, ids=[c[0] for c in CALLS])
def test_forward_mode_is_refused(what, call):
    """a dual tensor in any place: its tangent would be dropped"""
    from torch.autograd import forward_ad as fw
    for grad in (False, True):
        for name in names_of(call):
            with fw.dual_level(), pytest.raises(L.DPVOHipError, match="forward-mode"):
                call(lambda n, *s: fw.make_dual(z(*s, requires_grad=grad), torch.ones(*s)) if n == name else z(*s))
    with fw.dual_level(), pytest.raises(L.DPVOHipError, match="run on the GPU only"):
        call(lambda n, *s: z(*s))                                               # a level alone is no dual tensor


@pytest.mark.parametrize("f,n", [(blocks._Linear, 1), (blocks._GatedLinear, 1), (blocks._FeedForward, 1), (blocks._GatedResidual, 1), (blocks._ResidualNorm, 2)])
def test_forward_mode_of_a_backward_is_refused(f, n):
    """... and as the gradient that arrives"""
    from torch.autograd import forward_ad as fw
    with fw.dual_level(), torch.no_grad(), pytest.raises(L.DPVOHipError, match="forward-mode"):
        f.backward.__wrapped__(None, *[fw.make_dual(z(3, 4), torch.ones(3, 4)) for _ in range(n)])


@pytest.mark.parametrize("what,call", CALLS, ids=[c[0] for c in CALLS])
def test_traces_are_refused(what, call):
    """torch.jit.trace and make_fx would record the outputs' allocation and nothing that fills it"""
    from torch.fx.experimental.proxy_tensor import make_fx
    f = lambda x: call(lambda n, *s: x if n == "x" else z(*s))  # noqa: E731
    with torch.no_grad():
        with pytest.raises(L.DPVOHipError, match="jit.trace"):
            torch.jit.trace(f, z(3, 4))
        for mode in ("real", "fake", "symbolic"):
            with pytest.raises(L.DPVOHipError, match="make_fx"):
                make_fx(f, tracing_mode=mode)(z(3, 4))


class Elsewhere(torch.Tensor):
    """a tensor without memory: its values are another tensor's"""
    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


@pytest.mark.parametrize("what,call", CALLS, ids=[c[0] for c in CALLS])
def test_tensors_without_memory_are_refused(what, call):
    """an address of 0 would stand for a parameter that is not there"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    for name in names_of(call):
        with pytest.raises(L.DPVOHipError, match="a Elsewhere, whose values"):
            call(lambda n, *s: Elsewhere(z(*s)) if n == name else z(*s))
    with FakeTensorMode(), pytest.raises(L.DPVOHipError, match="FakeTensor"):
        call(lambda n, *s: z(*s))

    class Named(torch.Tensor):                                                  # a subclass in name only is an ordinary tensor
        pass
    with pytest.raises(L.DPVOHipError, match="run on the GPU only"):
        call(lambda n, *s: z(*s).as_subclass(Named) if n in "xw" else torch.nn.Parameter(z(*s)))


def test_pending_signs_are_resolved():
    """a negated view: its memory holds the values with the other sign"""
    for shape in ((4, 6), (2, 3, 6), (1, 6), (6,), (4, 1), (2, 3, 1), (1,)):
        x = torch.randn(*shape)
        for neg in (torch._neg_view(x), torch.complex(x, x).conj().imag):
            assert neg.is_neg()
            for t in (neg, neg[..., ::2], neg[..., :5]):
                r, ld = blocks._rows(t)
                assert not r.is_neg() and ld >= r.shape[1] and torch.equal(r, t.reshape(-1, t.shape[-1]))
                if t.dim() == 1:
                    r = blocks._vector(t)
                    assert not r.is_neg() and torch.equal(r, t)


# ------------------------------------------------------------------------------------------------------------------ the model's modules
def plain_blocks(monkeypatch):
    """the two operators that the model's stage calls, in torch on the host: what surrounds them is tested here"""
    F = torch.nn.functional
    monkeypatch.setattr(blocks, "norm", lambda x, w, b, kind, eps: F.layer_norm(x, x.shape[-1:], w, b, eps))
    monkeypatch.setattr(blocks, "gated_residual", lambda x, wg, bg, w1, b1, w2, b2: x + torch.sigmoid(F.linear(x, wg, bg)) * F.linear(F.relu(F.linear(x, w1, b1)), w2, b2))


class Adapter(torch.nn.Linear):
    def forward(self, x):
        return super().forward(x) + 1


def hooked(register):
    def change(gru):
        getattr(gru[1].res[2], register)(lambda *a: None)
    return change


def replaced(path, module):
    def change(gru):
        *up, last = path.split(".")
        setattr(gru.get_submodule(".".join(up)) if up else gru, last, module)
    return change


@pytest.mark.parametrize("change", [
    hooked("register_forward_hook"), hooked("register_forward_pre_hook"), hooked("register_full_backward_hook"), hooked("register_full_backward_pre_hook"),
    lambda gru: gru[3].gate.register_forward_hook(lambda *a: None), lambda gru: gru[1].gate[1].register_forward_hook(lambda *a: None),
    lambda gru: gru[2].register_forward_hook(lambda *a: None), lambda gru: torch.nn.utils.weight_norm(gru[1].res[0]),
    replaced("1.gate.0", Adapter(384, 384)), replaced("1.res.2", torch.nn.Identity()), replaced("1.gate.1", torch.nn.Tanh()), replaced("3.res.1", torch.nn.GELU()),
    replaced("1.res", torch.nn.Sequential(torch.nn.Linear(384, 384), torch.nn.ReLU(), torch.nn.Dropout(), torch.nn.Linear(384, 384))),
    replaced("0", type("Norm", (torch.nn.LayerNorm,), {"forward": lambda self, x: x})(384)), replaced("0", torch.nn.LayerNorm((2, 384), elementwise_affine=False)),
    lambda gru: setattr(gru[1].res[0], "forward", lambda x: x),
])
def test_children_that_would_do_something_else_are_refused(change, monkeypatch):
    """the stage reads its children's parameters and does not call them"""
    from dpvo_amd import net as N
    plain_blocks(monkeypatch)
    gru = N.Update(3).gru
    gru(z(2, 384))
    change(gru)
    with pytest.raises(L.DPVOHipError):
        gru(z(2, 384))


def test_children_that_are_read(monkeypatch):
    """no bias, a parametrized weight, a subclass with the same forward, hooks on the block itself: what a call of them would give"""
    from dpvo_amd import net as N
    plain_blocks(monkeypatch)
    torch.manual_seed(0)
    gru, x, seen = N.Update(3).gru, torch.randn(5, 384), []
    gru[1].gate[0] = torch.nn.Linear(384, 384, bias=False)
    gru[1].res[0] = type("Same", (torch.nn.Linear,), {})(384, 384)
    torch.nn.utils.parametrizations.weight_norm(gru[3].res[0])
    gru[3].register_forward_hook(lambda m, a, y: seen.append(y))
    y = gru(x)
    h = gru[0](x)
    h = gru[2](h + gru[1].gate(h) * gru[1].res(h))
    torch.testing.assert_close(y, h + gru[3].gate(h) * gru[3].res(h))
    assert len(seen) == 1 and seen[0] is y
    g, = torch.autograd.grad(y.sum(), [gru[3].res[0].parametrizations.weight.original1])
    assert g.abs().sum() > 0


def test_the_trackers_images_follow_training(monkeypatch):
    """whatever changes the stage's parameters by way of its modules, the next call of the update operator has images of the new ones"""
    from dpvo_amd import net as N
    plain_blocks(monkeypatch)
    torch.manual_seed(1)
    network = N.VONet()
    upd = network.update

    def right():
        fresh = N.Update(3)
        fresh.load_state_dict(upd.state_dict(), assign=True)
        P, want = upd.operands(), fresh.pack()
        return all(torch.equal(a, b) for k in ("g0", "g1", "c1", "norm") for a, b in zip(P[k], want[k]))
    upd.pack()
    P = upd.operands()
    assert upd.operands() is P and right()
    with torch.no_grad():
        upd.gru(z(1, 3, 384))
    assert upd.operands() is P                                                  # nothing recorded: the images stay
    opt = torch.optim.AdamW(upd.gru.parameters(), lr=0.1, fused=True)           # (leaves no mark on the parameters)
    for use in ((), ("forward",), ("forward", "backward"), ("forward", "backward", "step")):    # after which of them the tracker runs too
        y = upd.gru(torch.randn(1, 3, 384))
        assert "forward" not in use or right()
        y.square().sum().backward()
        assert "backward" not in use or right()
        opt.step()
        assert right()
    upd.pack()
    P = upd.operands()
    assert upd.operands() is P                                                  # training is over
    for part in (upd.gru[1], upd.gru[3], upd.gru):                              # a part alone
        part(torch.randn(1, 3, 384)).square().sum().backward()
        assert right()
        for p in part.parameters():
            p.data.add_(0.01)
        assert right()
        upd.pack()
    for n, p in upd.gru.named_parameters():                                     # the norms alone
        p.requires_grad_(n.split(".")[0] in "02")
    upd.gru(torch.randn(1, 3, 384)).sum().backward()
    upd.gru[0].weight.data.add_(0.01)
    assert right()
    upd.pack()
    for m in (network, upd, upd.gru, upd.gru[3]):                               # loads, casts
        state = {k: torch.randn_like(v) if v.is_floating_point() else v for k, v in m.state_dict().items()}
        for assign in (False, True):
            P = upd.operands()
            m.load_state_dict({k: v + assign for k, v in state.items()}, assign=assign)
            assert upd.operands() is not P and right()
            P = upd.operands()
            assert upd.operands() is P
        m.half()
        assert upd.operands() is not P and right()
        m.float()
        assert right() and upd.operands() is upd.operands()


# ------------------------------------------------------------------------------------------------------------------ what the GPU tests reach
PATHS = r"""
#include <stdio.h>
#include <string.h>
#include <set>
#include <string>
#include "blocks_plan.h"
using namespace blk;
static std::string key(int form, int epi, int dtype, Plan c) {
  static const char *forms[] = {"nt", "nn", "tn"}, *epis[] = {"lin", "gate", "gate2", "dact"}, *kinds[] = {"tile", "big", "small", "tiny", "few"};
  return std::string(dtype == DPVO_F32 ? "f32 " : "16 ") + forms[form] + " " + epis[epi] + " " + kinds[c.kind] + (c.splits > 1 ? " parts" : "");
}
// y [M,N] from x [M,K]; inputs: 0 without a second product, 1 and 2; plain: no activation, nothing saved
static std::string forward(int dtype, int inputs, bool plain, int64_t M, int64_t K, int64_t N) {
  char x[2];
  float save;
  dpvo_gated_linear_t p = {};
  p.x = x, p.v = inputs == 2 ? x + 1 : x, p.w_gate = x, p.w_up = inputs ? x : nullptr, p.save_gate = plain ? nullptr : &save;
  p.ldx = p.ldwg = p.ldv = p.ldwu = p.K = K, p.Kv = inputs ? K : 0, p.ldy = p.N = N, p.M = M, p.dtype = dtype, p.activation = !plain;
  const int e = linear_epi(&p);
  if (!linear_few(&p, e)) return key(F_NT, e, dtype, linear_plan(&p, e));
  return key(F_NT, e, dtype, Plan{T_FEW, 1}) + (M > 16 ? " 64 rows" : K > (dtype == DPVO_F32 ? 512 : 1024) ? " 16 waves" : " 4 waves");
}
static std::string dx(int dtype, bool through, int64_t M, int64_t N, int64_t nb) { return key(F_NN, through ? E_DACT : E_LIN, dtype, dx_plan(M, N, nb, dtype, !through)); }
int main() {
  std::set<std::string> all;
  const int64_t size[] = {1, 7, 16, 17, 33, 64, 100, 200, 300, 500, 700, 1000, 1500, 2000, 4100, 6000, 9000, 20000, 45000}, sum[] = {7, 64, 200, 384, 500, 700, 1024, 1100, 2100, 4200, 9000};
  for (int t = 0; t < 3; ++t)
    for (int64_t M : size)
      for (int64_t N : size)
        for (int64_t K : sum) {
          all.insert(forward(t, 0, true, M, K, N));
          for (int i = 0; i < 3; ++i) all.insert(forward(t, i, false, M, K, N));
          const int64_t nb = ceil_div(K, block_k(t));
          all.insert(dx(t, false, M, N, nb)), all.insert(dx(t, false, M, N, 2 * nb)), all.insert(dx(t, true, M, N, nb));
          for (int n = 1; n <= MAXP; ++n)
            for (int sides = 0; sides < 2; ++sides) {
              dpvo_gated_linear_dw_t p = {};
              p.n = n, p.M = sides ? K * 5 : M, p.dtype = t;
              for (int i = 0; i < n; ++i) p.N[i] = N, p.K[i] = sides ? M : K;
              all.insert(key(F_TN, E_LIN, t, dw_plan(&p)));
            }
        }
  for (auto& k : all) printf("all %s\n", k.c_str());
  char op[16];
  while (scanf("%15s", op) == 1) {
    long a[32];
    int n;
    if (scanf("%d", &n) != 1 || n > 32) return 1;
    for (int i = 0; i < n; ++i)
      if (scanf("%ld", a + i) != 1) return 1;
    for (int t = 0; t < 3; ++t) {
      const int64_t bk = block_k(t);
      if (!strcmp(op, "forward")) {
        printf("hit %s\n", forward(t, 0, true, a[0], a[1], a[2]).c_str());
        for (int i = 0; i < 3; ++i) printf("hit %s\n", forward(t, i, false, a[0], a[1], a[2]).c_str());
      } else if (!strcmp(op, "dx")) {
        for (int two = 0; two < 2; ++two)
          for (int e = 0; e < 2; ++e) printf("hit %s\n", dx(t, e, a[0], a[2], ceil_div(a[1], bk) + two * ceil_div(a[1] + 5, bk)).c_str());
      } else if (!strcmp(op, "dw")) {
        dpvo_gated_linear_dw_t p = {};
        p.M = a[0], p.n = (n - 1) / 2, p.dtype = t;
        for (int i = 0; i < p.n; ++i) p.N[i] = a[1 + 2 * i], p.K[i] = a[2 + 2 * i];
        printf("hit %s\n", key(F_TN, E_LIN, t, dw_plan(&p)).c_str());
      } else {                                            // norm: rows, D, gate rows (0: no gate), a branch (1: behind a norm with parameters)
        dpvo_residual_norm_t p = {};
        char x;
        p.M = a[0], p.D = (int)a[1], p.groups = a[2], p.gate = a[2] ? &x : nullptr, p.f = a[3] ? &x : nullptr, p.x_dtype = t, p.dw = p.db = &x;
        if (a[3]) p.dgate = p.gate ? &x : nullptr;
        if (a[3] == 1) p.dpw = p.dpb = &x;
        const NormPlan c = norm_plan(p);
        const int fs = norm_shape(p, false, 0);
        printf("norm %d %d %ld %ld %ld %ld %ld %ld %d %d %ld\n", t, c.sh, (long)c.groups, (long)c.rpg, (long)c.gpb, (long)c.bpg, (long)c.blocks, (long)norm_slots(c.sh), c.shared, fs,
               (long)norm_slots(fs));
      }
    }
  }
}
"""


@pytest.fixture(scope="module")
def paths(tmp_path_factory):
    """the library's rules, by themselves: what they return over a grid of sizes, and for the sizes that the GPU tests list"""
    from tests import test_gpu_blocks_paths as G
    d = tmp_path_factory.mktemp("paths")
    (d / "paths.cpp").write_text(PATHS)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "dpvo_amd", "csrc"), "-I", os.path.join(ROOT, "include"), str(d / "paths.cpp"), "-o", str(d / "paths")])
    cases = [("forward", *c) for c in G.FORWARD] + [("dx", *c) for c in G.INPUT_GRADIENTS] + [("dw", M, *(n for s in sizes for n in s)) for M, sizes in G.WEIGHT_GRADIENTS]
    for lead, D, gate in G.NORMS + G.NORMS_PLAIN:
        rows, groups = 1, 1
        for n in lead:
            rows *= n
        for n in gate or (0,):
            groups *= n
        cases.append(("norm", rows, D, groups, 1 if (lead, D, gate) in G.NORMS else 2))
    cases += [("norm", M, D, 0, 0) for M, D in G.NORM_ALONE]
    text = "\n".join(" ".join(map(str, (c[0], len(c) - 1, *c[1:]))) for c in cases)
    out = subprocess.run([str(d / "paths")], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
    kept = {k: [l[len(k) + 1:] for l in out if l.startswith(k + " ")] for k in ("all", "hit", "norm")}
    assert sum(map(len, kept.values())) == len(out)
    return kept


def test_the_gpu_tests_reach_every_product(paths):
    every, reached = set(paths["all"]), set(paths["hit"])
    assert len(every) > 60 and not every - reached, sorted(every - reached)
    assert not reached - every, sorted(reached - every)                          # (the grid is wide enough)


def test_no_product_is_built_that_nothing_reaches(paths):
    """the tile kernels in the library, by form, epilogue and tile, as many of each as there are types that choose it"""
    import collections
    import re
    import shutil
    if not shutil.which("nm"):
        pytest.skip("no nm")
    names = {"nt": 0, "nn": 1, "tn": 2}, {"lin": 0, "gate": 1, "gate2": 2, "dact": 3}, {"tile": 0, "big": 1, "small": 2, "tiny": 3}
    want = collections.Counter()
    for k in {tuple(k.split()[:4]) for k in paths["all"]}:
        if k[3] in names[2]:
            want[tuple(n[x] for n, x in zip(names, k[1:]))] += 1 if k[0] == "f32" else 2
    out = subprocess.check_output(["nm", "-C", L.LIB_PATH], text=True)
    have = collections.Counter(tuple(map(int, m)) for m in re.findall(r" [dD] void blk::\(anonymous namespace\)::gemm_kernel<(\d), (\d), (\d)>\(", out))
    assert have == want


def test_the_gpu_tests_reach_the_loops_of_the_norms(paths):
    """backward: for every number of lanes a workgroup with several rounds of rows, with several groups, and the last of them short; with parts of a
    group of several rounds; forward: workgroups that go round.  (Shapes: blocks_plan.h's NORM_SHAPES, 12 the 1024 lanes, 13 the wide rows)"""
    rounds, groups, short, parts, forward = set(), set(), set(), set(), set()
    for l in paths["norm"]:
        t, sh, n, rpg, gpb, bpg, blocks_, slots, shared, fsh, fslots = map(int, l.split())
        if -(-rpg // slots) >= 2 * bpg:
            rounds.add(sh)
        if gpb > 1:
            groups.add(sh)
            if n % gpb:
                short.add(sh)
        if shared and bpg > 1 and -(-rpg // slots) >= 2 * bpg:
            parts.add(sh)
        rows, D = n * rpg, None
        most = {13: 8192}.get(fsh, 2048 if 6 <= fsh <= 11 else 8192)
        if rows > most * fslots:
            forward.add(fsh)
    every = set(range(14))
    assert rounds == every, every - rounds
    assert forward == every - {12}, every - forward                              # (the 1024 lanes go backward only)
    assert groups == every, every - groups
    assert len(short) >= 8 and 13 in short and 12 in short, short
    assert len(parts) >= 8 and {2, 8, 12, 13} <= parts, parts


def test_the_gpu_tests_bounds_see_a_mistake():
    """the oracle with mistakes planted, on the host: bounds, exact products, sums over rows"""
    from tests import test_gpu_blocks as B, test_gpu_blocks_paths as G
    B.test_the_bounds_see_a_mistake()
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(-1, 2, (3000, n), generator=g).double() for n in (40, 30))
    right = a.t() @ b
    for t in (torch.float16, torch.bfloat16, torch.float32):
        G.exactly(right.to(t), right, t, "right")
        for rows in (slice(0, 2999), slice(64, 3000), slice(0, 2936)):           # one row, a first or a last block of the sum left out
            with pytest.raises(AssertionError):
                G.exactly((a[rows].t() @ b[rows]).to(t), right, t, "planted")
    q = B.V(torch.randn(3000, 20, generator=g, dtype=torch.float64) + 0.5)
    want = G.sum_rows(q, 3000)
    B.within(q.v.float().sum(0, keepdim=True), want, torch.float32, "right")
    for wrong in (q.v[:2999], q.v[64:], q.v[::2] * 2):
        with pytest.raises(AssertionError):
            B.within(wrong.float().sum(0, keepdim=True), want, torch.float32, "planted")


@pytest.mark.parametrize("t,most", [(H, 4194303), (torch.bfloat16, 4194303), (torch.float32, 2097151)], ids=str)
def test_rows_that_are_too_long_are_refused_before_any_launch(t, most):
    e = lambda *s: torch.empty(*s, dtype=t)  # noqa: E731
    long, too = e(1, most), e(1, most + 1)
    with pytest.raises(L.DPVOHipError, match="run on the GPU only"):
        blocks.linear(long, long)
    with pytest.raises(L.DPVOHipError, match="rows of at most"):
        blocks.linear(too, too)
    with pytest.raises(L.DPVOHipError, match="rows of at most"):
        blocks.gated_linear(e(1, 4), e(1, 4), too, up_input=too)
    with pytest.raises(L.DPVOHipError, match="rows of at most"):
        blocks.gated_feed_forward(e(1, 4), e(most + 1, 4), e(most + 1, 4), e(2, most + 1))
    # as many outputs: a gradient's rows, so only where one will be asked for
    x, w = e(1, 2), e(most + 1, 2)
    with pytest.raises(L.DPVOHipError, match="run on the GPU only"):
        blocks.linear(x, w)
    for leaf in (x, w):
        leaf.requires_grad_()
        with pytest.raises(L.DPVOHipError, match="rows of at most"):
            blocks.linear(x, w)
        with torch.no_grad(), pytest.raises(L.DPVOHipError, match="run on the GPU only"):
            blocks.linear(x, w)
        leaf.requires_grad_(False)


def test_a_packed_network_can_be_copied():
    """an average of the weights, or a checkpoint of the whole module, taken while the tracker's images are there"""
    import copy
    import io
    from dpvo_amd import net as N
    network = N.VONet()
    P = network.update.pack()
    twin = copy.deepcopy(network)
    buf = io.BytesIO()
    torch.save(network, buf)
    assert network.update.operands() is P
    with torch.no_grad():
        twin.update.gru[1].res[2].weight.add_(1)
    a, b = P["g0"][4], twin.update.operands()["g0"][4]
    assert torch.equal(b, twin.update.gru[1].res[2].weight.half()) and not torch.equal(a, b) and network.update.operands() is P
    assert all(torch.equal(p, q) for p, q in zip(twin.state_dict().values(), network.state_dict().values()) if p.shape != (384, 384))
