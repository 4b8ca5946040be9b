"""Gated feed-forward blocks and the norms around them, with their gradients: the update operator's gated residual block and its LayerNorms
(dpvo/blocks.py:15-24, dpvo/net.py:44-59) as differentiable operators of any width, and their relatives.

    linear(x, w, b, activation)                y = act(x w^T + b)
    gated_linear(x, wg, wu, ...)               y = act(x wg^T + bg) * (v wu^T + bu) [+ residual]         (v = x, or another input)
    gated_feed_forward(x, wg, wu, wd, ...)     y = (act(x wg^T + bg) * (x wu^T + bu)) wd^T + bd
    gated_residual(x, wg, bg, w1, b1, w2, b2)  y = x + sigmoid(x wg^T + bg) * (relu(x w1^T + b1) w2^T + b2)
    norm(x, w, b)                              LayerNorm or RMSNorm before a block
    residual_norm(x, f, w, b, gate=...)        s = x + scale * act(gate) * post(f);  h = norm(s)          after a block and before the next

Operands are float16, bfloat16 or float32 CUDA tensors of one type (`residual_norm`: the stream x may be float32 beside a 16-bit branch);
products run on the matrix cores, sums, statistics and activations are float32.  What enters a second matrix product is rounded to the operands'
type, as the matrix cores take it: the hidden product act(..) * (..), and in the backward pass the gradients of the sums (which the activations'
derivatives read in float32, as saved).  So a 16-bit block's results are a step or two of its type's rounding away from the formula's, and its
gradients need the loss scaled as those of any 16-bit operands.  Everything runs on the current stream of the tensors' device.
Gradients of first order are provided, in reverse mode; results and gradients do not vary from run to run.  Autocast is not consulted.  Dual tensors,
torch.jit.trace, make_fx and tensors without memory of their own are refused.  A backward pass that is captured into a graph follows PyTorch's rule:
no eager graph of the same leaves may be alive."""
import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

ACTIVATIONS = {"identity": 0, "relu": 1, "sigmoid": 2, "silu": 3, "gelu": 4, "gelu_tanh": 5}
GATE_ACTIVATIONS = {k: ACTIVATIONS[k] for k in ("identity", "relu", "sigmoid", "silu")}
NORMS = {None: 0, "layer": 1, "rms": 2}
MAX_NORM_WIDTH = 16384
_DTYPES = {torch.float16: L.F16, torch.float32: L.F32, torch.bfloat16: L.BF16}
_MAX_LD = {2: (2 ** 31 - 1) // 512, 4: (2 ** 31 - 1) // 1024}      # rows are addressed with 32 bits within a tile


# ------------------------------------------------------------------------------------------------------------------ checks
def _fail(what, why):
    raise L.DPVOHipError(f"{what}: {why}")


def _code(table, key, what, arg):
    try:
        return table[key]
    except (KeyError, TypeError):
        _fail(what, f"{arg} is {key!r}, not one of {', '.join(map(repr, table))}")


_is_tracing, _modes, _PROXY = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._TorchDispatchModeKey.PROXY
_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}


def _check_recording(what, tensors):
    """the kernels read and write memory behind torch's back: what would record a call sees nothing of it"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _fail(what, "forward-mode derivatives are not provided, and an input is a dual tensor")
    if _is_tracing() or (_modes() and torch._C._get_dispatch_mode(_PROXY) is not None):
        _fail(what, "a call under torch.jit.trace or make_fx: what the kernels write is not recorded, a trace would return memory as it was")


def _check_type(what, t):
    if type(t).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__:
        _fail(what, f"a {type(t).__name__}, whose values do not lie in memory of its own")


def _check_gradients(what, *tensors):
    """those that arrive"""
    if forward_ad._current_level >= 0 or _is_tracing() or _modes():
        _check_recording(what, tensors)
    for t in tensors:
        if type(t) not in _PLAIN:
            _check_type(what, t)


def _check(what, x, *others):
    """tensors whose values lie in their memory, a call that nothing else records, one device, a dtype that the kernels know"""
    if forward_ad._current_level >= 0 or _is_tracing() or _modes():
        _check_recording(what, (x, *others))
    if type(x) not in _PLAIN:
        _check_type(what, x)
    i = x.get_device()
    for t in others:
        if t is not None:
            if type(t) not in _PLAIN:
                _check_type(what, t)
            if t.get_device() != i or (i < 0 and t.device != x.device):
                _fail(what, f"tensors on {x.device} and {t.device}")
    if x.dtype not in _DTYPES:
        _fail(what, f"unsupported dtype {x.dtype} (float16, bfloat16, float32)")


def _check_layer(what, x, K, w, b, name):
    if w.dim() != 2 or w.shape[1] != K:
        _fail(what, f"{name} is {tuple(w.shape)}, its input has {K} features")
    if 0 in w.shape:
        _fail(what, f"{name} is {tuple(w.shape)}: no features")
    if w.dtype != x.dtype or (b is not None and b.dtype != x.dtype):
        _fail(what, f"{name} and its bias must have the input's dtype {x.dtype}")
    most = _MAX_LD[x.element_size()]
    if K > most or (w.shape[0] > most and _wants_grad(x, w, b)):           # (forward alone, outputs are addressed with 64 bits)
        _fail(what, f"{name} is {tuple(w.shape)}: rows of at most {most} elements, and in the backward pass outputs too")
    if b is not None and tuple(b.shape) != (w.shape[0],):
        _fail(what, f"the bias of {name} is {tuple(b.shape)}, not ({w.shape[0]},)")


def _features(what, x):
    if x.dim() < 1:
        _fail(what, "the input has no feature dimension")
    return x.shape[-1]


# ------------------------------------------------------------------------------------------------------------------ launches
def _rows(t):
    """[..., K] as rows whose elements are contiguous: (tensor [M,K], leading dimension); a copy only where no such view exists, or where the sign
    is pending (the gradient that comes back through a complex conjugate's imaginary part is a negated view; one of a single feature has rows)"""
    if t.is_neg():
        t = t.resolve_neg()
    if t.is_contiguous():
        K = t.shape[-1]
        return t if t.dim() == 2 else t.view(-1 if K else t.numel(), K), K
    K = t.shape[-1]
    if t.dim() != 2:
        M = 1
        for n in t.shape[:-1]:
            M *= n
        t = t.reshape(M, K)
    if t.shape[0] <= 1 and (K <= 1 or t.stride(1) == 1):
        return t, K
    ld = t.stride(0)
    if (K > 1 and t.stride(1) != 1) or ld < K or ld > _MAX_LD[t.element_size()]:
        t = t.contiguous()
        ld = K
    return t, ld


def _vector(t):
    if t is None:
        return t
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.stride(0) == 1 or t.shape[0] <= 1 else t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


class _Here:
    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_HERE = _Here()
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _on(x):
    """context: the current device is x's"""
    return _HERE if x.get_device() == _current_device() else torch.cuda.device(x.device)


def _stream(x):
    return _raw_stream(x.get_device())


def _scratch(nbytes, device):
    """of the current stream, and of a captured graph's own pool: never shared between graphs"""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(x, wg, bg, act, v=None, wu=None, bu=None, residual=None, save=False):
    """x, v, residual: rows.  -> y [M,N], and with `save` the two float32 sums"""
    x, ldx = _rows(x)
    wg, ldwg = _rows(wg)
    M, N = x.shape[0], wg.shape[0]
    ldv = ldwu = ldr = Kv = 0
    if wu is not None:
        if v is None:
            v, ldv = x, ldx
        else:
            v, ldv = _rows(v)
        wu, ldwu = _rows(wu)
        Kv = wu.shape[1]
    if residual is not None:
        residual, ldr = _rows(residual)
    bg, bu = _vector(bg), _vector(bu)
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    sg = torch.empty(M, N, dtype=torch.float32, device=x.device) if save else None
    su = torch.empty(M, N, dtype=torch.float32, device=x.device) if save and wu is not None else None
    p = L.GatedLinear(_p(x), _p(v) if wu is not None else None, _p(wg), _p(wu), _p(bg), _p(bu), _p(residual), _p(y), _p(sg), _p(su), ldx, ldv,
                      ldwg, ldwu, ldr, N, M, N, x.shape[1], Kv, _DTYPES[x.dtype], act)
    lib, n, ws = L.lib(), 0, None
    if act == 0 and wu is None and M > 16:                       # (few rows: never in parts)
        n = lib.dpvo_gated_linear_workspace_bytes(ctypes.byref(p))
        ws = _scratch(n, x.device)
    rc = lib.dpvo_gated_linear(ctypes.byref(p), _p(ws), n, _stream(x))
    if rc:
        L.check(rc, "dpvo_gated_linear")
    return y, sg, su


def _dact(dy, gate, up, act):
    dy, ld = _rows(dy)
    M, N = dy.shape
    dg = torch.empty(M, N, dtype=dy.dtype, device=dy.device)
    du = torch.empty_like(dg) if up is not None else None
    L.check(L.lib().dpvo_gated_linear_dact(_p(dy), ld, _p(gate), _p(up), _p(dg), _p(du), N, _DTYPES[dy.dtype], act, M, N, _stream(dy)),
            "dpvo_gated_linear_dact")
    return dg, du


def _dx(pairs, addend=None, gate=None, up=None, mask=None, act=0):
    """sum of a . w over `pairs` (one or two); -> dx, and with `up` the second gradient"""
    a0, lda0 = _rows(pairs[0][0])
    w0, ldw0 = _rows(pairs[0][1])
    a1 = w1 = None
    lda1 = ldw1 = K1 = ldadd = ldmask = 0
    if len(pairs) == 2:
        a1, lda1 = _rows(pairs[1][0])
        w1, ldw1 = _rows(pairs[1][1])
        K1 = a1.shape[1]
    M, K0 = a0.shape
    N = w0.shape[1]
    dx = torch.empty(M, N, dtype=a0.dtype, device=a0.device)
    dx2 = torch.empty_like(dx) if up is not None else None
    if addend is not None:
        addend, ldadd = _rows(addend)
    if mask is not None:
        mask, ldmask = _rows(mask)
    p = L.GatedLinearDx((a0.data_ptr(), _p(a1)), (w0.data_ptr(), _p(w1)), _p(addend), _p(mask), _p(gate), _p(up), dx.data_ptr(), _p(dx2), (lda0, lda1),
                        (ldw0, ldw1), (K0, K1), ldadd, ldmask, N, M, N, _DTYPES[a0.dtype], act)
    lib = L.lib()
    n = lib.dpvo_gated_linear_dx_workspace_bytes(ctypes.byref(p))
    ws = _scratch(n, a0.device)
    rc = lib.dpvo_gated_linear_dx(ctypes.byref(p), _p(ws), n, _stream(a0))
    if rc:
        L.check(rc, "dpvo_gated_linear_dx")
    return dx, dx2


def _dw(jobs):
    """jobs: (gradient of the sums [M,N], input [M,K], want dw, want db) -> [(dw, db), ...]"""
    pa, pb, pdw, pdb, la, lb, ns, ks = [], [], [], [], [], [], [], []
    keep, out = [], []
    for a, b, want_w, want_b in jobs:
        if not (want_w or want_b):
            out.append((None, None))
            continue
        a, lda = _rows(a)
        b, ldb = _rows(b)
        N, K = a.shape[1], b.shape[1]
        dw = torch.empty(N, K, dtype=a.dtype, device=a.device)               # (db is made beside it)
        db = torch.empty(N, dtype=a.dtype, device=a.device) if want_b else None
        keep += (a, b, dw)
        out.append((dw if want_w else None, db))
        pa.append(a.data_ptr())
        pb.append(b.data_ptr())
        pdw.append(dw.data_ptr())
        pdb.append(_p(db))
        la.append(lda)
        lb.append(ldb)
        ns.append(N)
        ks.append(K)
    if keep:
        a = keep[0]
        p = L.GatedLinearDw(*map(tuple, (pa, pb, pdw, pdb, la, lb, ns, ks)), a.shape[0], len(pa), _DTYPES[a.dtype])
        lib = L.lib()
        n = lib.dpvo_gated_linear_dw_workspace_bytes(ctypes.byref(p))
        ws = _scratch(n, a.device)
        rc = lib.dpvo_gated_linear_dw(ctypes.byref(p), _p(ws), n, _stream(a))
        if rc:
            L.check(rc, "dpvo_gated_linear_dw")
    return out


def _like(y, x, n):
    """rows y [M, n] in the leading shape of x"""
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------------------------ linear
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, act):
        with _on(x):
            y, pre, _ = _forward(x, w, b, act, save=act != 0)
        ctx.save_for_backward(x, w, pre)
        ctx.act = act
        return _like(y, x, w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_gradients("linear", dy)
        x, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        with _on(x):
            dy = _rows(dy)[0]
            d = dy if ctx.act == 0 else _dact(dy, pre, None, ctx.act)[0]
            dx = _dx([(d, w)])[0].view(x.shape) if need[0] else None
            (dw, db), = _dw([(d, x, need[1], need[2])])
        return dx, dw, db, None


def linear(x, weight, bias=None, activation="identity"):
    """act(x weight^T + bias): x [..., K], weight [N, K], bias [N] -> [..., N]"""
    what = "linear"
    _check(what, x, weight, bias)
    K = _features(what, x)
    act = _code(ACTIVATIONS, activation, what, "activation")
    _check_layer(what, x, K, weight, bias, "weight")
    L.require_cuda(x)
    if _wants_grad(x, weight, bias):
        return _Linear.apply(x, weight, bias, act)
    with _on(x):
        return _like(_forward(x, weight, bias, act)[0], x, weight.shape[0])


# ------------------------------------------------------------------------------------------------------------------ gated linear
class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, v, residual, act):
        with _on(x):
            y, g, u = _forward(x, wg, bg, act, v, wu, bu, residual, save=True)
        ctx.save_for_backward(x, v, wg, wu, g, u)
        ctx.act = act
        return _like(y, x, wg.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_gradients("gated_linear", dy)
        x, v, wg, wu, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dv = dwg = dwu = dbg = dbu = None
        with _on(x):
            if any(need[:6]):
                dg, du = _dact(dy, g, u, ctx.act)
                if v is None:
                    if need[0]:
                        dx = _dx([(dg, wg), (du, wu)])[0].view(x.shape)
                else:
                    if need[0]:
                        dx = _dx([(dg, wg)])[0].view(x.shape)
                    if need[5]:
                        dv = _dx([(du, wu)])[0].view(v.shape)
                (dwg, dbg), (dwu, dbu) = _dw([(dg, x, need[1], need[3]), (du, x if v is None else v, need[2], need[4])])
        return dx, dwg, dwu, dbg, dbu, dv, dy if need[6] else None, None


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu", up_input=None, residual=None):
    """act(x w_gate^T + b_gate) * (v w_up^T + b_up) [+ residual] with both projections, the activation and the product in one kernel;
    v is x, or `up_input` [..., Kv].  x [..., K], w_gate [N, K], w_up [N, Kv], residual [..., N] -> [..., N]"""
    what = "gated_linear"
    _check(what, x, w_gate, w_up, b_gate, b_up, up_input, residual)
    K = _features(what, x)
    act = _code(ACTIVATIONS, activation, what, "activation")
    _check_layer(what, x, K, w_gate, b_gate, "w_gate")
    if up_input is not None and (up_input.dtype != x.dtype or up_input.shape[:-1] != x.shape[:-1] or up_input.dim() != x.dim()):
        _fail(what, f"up_input {tuple(up_input.shape)} {up_input.dtype} does not go with x {tuple(x.shape)} {x.dtype}")
    _check_layer(what, x, K if up_input is None else up_input.shape[-1], w_up, b_up, "w_up")
    if w_up.shape[0] != w_gate.shape[0]:
        _fail(what, f"w_gate makes {w_gate.shape[0]} features, w_up {w_up.shape[0]}")
    if residual is not None and (residual.dtype != x.dtype or tuple(residual.shape) != (*x.shape[:-1], w_gate.shape[0])):
        _fail(what, f"residual {tuple(residual.shape)} {residual.dtype} is not {(*x.shape[:-1], w_gate.shape[0])} {x.dtype}")
    L.require_cuda(x)
    if _wants_grad(x, w_gate, w_up, b_gate, b_up, up_input, residual):
        return _GatedLinear.apply(x, w_gate, w_up, b_gate, b_up, up_input, residual, act)
    with _on(x):
        return _like(_forward(x, w_gate, b_gate, act, up_input, w_up, b_up, residual)[0], x, w_gate.shape[0])


# ------------------------------------------------------------------------------------------------------------------ feed-forward block
class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, bg, bu, bd, act):
        with _on(x):
            h, g, u = _forward(x, wg, bg, act, None, wu, bu, save=True)
            y = _forward(h, wd, bd, 0)[0]
        ctx.save_for_backward(x, wg, wu, wd, h, g, u)
        ctx.act = act
        return _like(y, x, wd.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_gradients("gated_feed_forward", dy)
        x, wg, wu, wd, h, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dwg = dwu = dbg = dbu = None
        with _on(x):
            dy = _rows(dy)[0]
            jobs = [(dy, h, need[3], need[6])]
            if any(need[i] for i in (0, 1, 2, 4, 5)):
                dg, du = _dx([(dy, wd)], gate=g, up=u, act=ctx.act)
                if need[0]:
                    dx = _dx([(dg, wg), (du, wu)])[0].view(x.shape)
                jobs += [(dg, x, need[1], need[4]), (du, x, need[2], need[5])]
            out = _dw(jobs)
            (dwd, dbd) = out[0]
            if len(out) > 1:
                (dwg, dbg), (dwu, dbu) = out[1:]
        return dx, dwg, dwu, dwd, dbg, dbu, dbd, None


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down: x [..., K], w_gate, w_up [F, K], w_down [N, F] -> [..., N].
    The product is rounded to x's dtype between the two kernels, as the second one's operand."""
    what = "gated_feed_forward"
    _check(what, x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    K = _features(what, x)
    act = _code(ACTIVATIONS, activation, what, "activation")
    _check_layer(what, x, K, w_gate, b_gate, "w_gate")
    _check_layer(what, x, K, w_up, b_up, "w_up")
    if w_up.shape[0] != w_gate.shape[0]:
        _fail(what, f"w_gate makes {w_gate.shape[0]} features, w_up {w_up.shape[0]}")
    _check_layer(what, x, w_gate.shape[0], w_down, b_down, "w_down")
    L.require_cuda(x)
    if _wants_grad(x, w_gate, w_up, w_down, b_gate, b_up, b_down):
        return _FeedForward.apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)
    with _on(x):
        h = _forward(x, w_gate, b_gate, act, None, w_up, b_up)[0]
        return _like(_forward(h, w_down, b_down, 0)[0], x, w_down.shape[0])


# ------------------------------------------------------------------------------------------------------------------ gated residual block
_RELU, _SIGMOID = ACTIVATIONS["relu"], ACTIVATIONS["sigmoid"]


class _GatedResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, bg, w1, b1, w2, b2):
        with _on(x):
            t = _forward(x, w1, b1, _RELU)[0]
            y, g, r = _forward(x, wg, bg, _SIGMOID, t, w2, b2, residual=x, save=True)
        ctx.save_for_backward(x, wg, w1, w2, t, g, r)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_gradients("gated_residual", dy)
        x, wg, w1, w2, t, g, r = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dwg = dbg = dw1 = db1 = dw2 = db2 = None
        with _on(x):
            dy = _rows(dy)[0]
            dg, dr = _dact(dy, g, r, _SIGMOID)
            # the ReLU's derivative is 0 where its output (as rounded: an f16 sum up to 2^-25 has become 0) is: the gradient of its input is masked in
            # the product's epilogue, and a NaN passes
            dp = _dx([(dr, w2)], mask=t)[0] if need[0] or need[3] or need[4] else None
            if need[0]:
                dx = _dx([(dg, wg), (dp, w1)], addend=dy)[0].view(x.shape)
            jobs = [(dg, x, need[1], need[2]), (dr, t, need[5], need[6])]
            if dp is not None:
                jobs.append((dp, x, need[3], need[4]))
            out = _dw(jobs)
            (dwg, dbg), (dw2, db2) = out[:2]
            if dp is not None:
                dw1, db1 = out[2]
        return dx, dwg, dbg, dw1, db1, dw2, db2


def gated_residual(x, w_gate, b_gate, w_in, b_in, w_out, b_out):
    """x + sigmoid(x w_gate^T + b_gate) * (relu(x w_in^T + b_in) w_out^T + b_out)  (GatedResidual.forward, dpvo/blocks.py:15-24):
    x [..., D], w_gate [D, D], w_in [H, D], w_out [D, H], biases or None -> [..., D]"""
    what = "gated_residual"
    _check(what, x, w_gate, b_gate, w_in, b_in, w_out, b_out)
    D = _features(what, x)
    _check_layer(what, x, D, w_gate, b_gate, "w_gate")
    _check_layer(what, x, D, w_in, b_in, "w_in")
    _check_layer(what, x, w_in.shape[0], w_out, b_out, "w_out")
    if w_gate.shape[0] != D or w_out.shape[0] != D:
        _fail(what, f"w_gate and w_out must make x's {D} features: {w_gate.shape[0]}, {w_out.shape[0]}")
    L.require_cuda(x)
    if _wants_grad(x, w_gate, b_gate, w_in, b_in, w_out, b_out):
        return _GatedResidual.apply(x, w_gate, b_gate, w_in, b_in, w_out, b_out)
    with _on(x):
        t = _forward(x, w_in, b_in, _RELU)[0]
        return _like(_forward(x, w_gate, b_gate, _SIGMOID, t, w_out, b_out, residual=x)[0], x, D)


# ------------------------------------------------------------------------------------------------------------------ norms
def _norm_struct(x, f, gate, w, b, pw, pb, cfg, s, h, ds, dh, grads):
    """the C struct and what must stay alive (positional: assigning its fields one by one takes longer than the launch)"""
    norm_k, post_k, gate_act, scale, eps, post_eps, h_dtype, groups = cfg
    x, ldx = _rows(x)
    ldf = ldg = ldds = lddh = 0
    if f is not None:
        f, ldf = _rows(f)
    if gate is not None:
        gate, ldg = _rows(gate)
    if ds is not None:
        ds, ldds = _rows(ds)
    if dh is not None:
        dh, lddh = _rows(dh)
    w, b, pw, pb = _vector(w), _vector(b), _vector(pw), _vector(pb)
    hd = _DTYPES[h_dtype]
    par = w if w is not None else b if b is not None else pw if pw is not None else pb
    M, D = x.shape
    p = L.ResidualNorm(x.data_ptr(), _p(f), _p(gate), _p(w), _p(b), _p(pw), _p(pb), _p(s), _p(h), _p(ds), _p(dh),
                       *(grads if grads is _NO_GRADS else map(_p, grads)), ldx, ldf, ldg,
                       ldds, lddh, M, groups, D, _DTYPES[x.dtype], hd if f is None else _DTYPES[f.dtype], hd,
                       L.F32 if par is None else _DTYPES[par.dtype], norm_k, post_k, gate_act, scale, eps, post_eps)
    return p, (x, f, gate, w, b, pw, pb, ds, dh)


_NO_GRADS = (None,) * 7


def _new(x, dtype):
    """contiguous, of x's shape"""
    if dtype == x.dtype and x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def _norm_forward(x, f, gate, w, b, pw, pb, cfg):
    """-> s (None without a branch), h (None without a norm)"""
    with _on(x):
        s = _new(x, x.dtype) if f is not None else None
        h = _new(x, cfg[6]) if cfg[0] else None
        p, keep = _norm_struct(x, f, gate, w, b, pw, pb, cfg, s, h, None, None, _NO_GRADS)
        rc = L.lib().dpvo_residual_norm(ctypes.byref(p), _stream(x))
    if rc:
        L.check(rc, "dpvo_residual_norm")
    return s, h


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, w, b, pw, pb, cfg):
        s, h = _norm_forward(x, f, gate, w, b, pw, pb, cfg)
        ctx.save_for_backward(x, f, gate, w, b, pw, pb)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, dh):
        _check_gradients("residual_norm", ds, dh)
        x, f, gate, w, b, pw, pb = ctx.saved_tensors
        grads = [None] * 7
        if ds is None and dh is None:
            return (*grads, None)
        with _on(x):
            make = torch.empty if x.numel() else torch.zeros
            for i, t in enumerate((x, f, gate, w, b, pw, pb)):
                if t is not None and ctx.needs_input_grad[i]:
                    grads[i] = make(t.shape, dtype=t.dtype, device=t.device)
            if x.numel():
                p, keep = _norm_struct(x, f, gate, w, b, pw, pb, ctx.cfg, None, None, ds, dh, grads)
                lib = L.lib()
                n = lib.dpvo_residual_norm_backward_workspace_bytes(ctypes.byref(p))
                ws = _scratch(n, x.device)
                L.check(lib.dpvo_residual_norm_backward(ctypes.byref(p), _p(ws), n, _stream(x)), "dpvo_residual_norm_backward")
        return (*grads, None)


def _gate_rows(what, x, gate):
    """how many rows of `gate` there are: it is shaped like x, or with ones (or nothing) in the place of x's last leading dimensions"""
    if gate.dim() == 1 and gate.shape[0] == x.shape[-1]:
        return 1
    lead = [1] * (x.dim() - gate.dim()) + list(gate.shape[:-1])
    if gate.dim() > x.dim() or gate.dim() < 1 or gate.shape[-1] != x.shape[-1]:
        _fail(what, f"gate {tuple(gate.shape)} does not go with x {tuple(x.shape)}")
    k, rows = 0, 1
    while k < len(lead) and lead[k] == x.shape[k]:
        rows *= lead[k]
        k += 1
    if any(n != 1 for n in lead[k:]):
        _fail(what, f"gate {tuple(gate.shape)} must be shaped like x {tuple(x.shape)} up to some dimension, and 1 (or nothing) from there")
    return rows


def _check_params(what, D, params):
    dtype = None
    for name, t in params:
        if t is None:
            continue
        if tuple(t.shape) != (D,):
            _fail(what, f"{name} is {tuple(t.shape)}, not ({D},)")
        if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
            _fail(what, f"{name} is {t.dtype}: parameters are float16, bfloat16 or float32, all of one dtype")
        dtype = t.dtype


def _check_width(what, x):
    D = _features(what, x)
    if not 1 <= D <= MAX_NORM_WIDTH:
        _fail(what, f"rows of {D} elements (1 to {MAX_NORM_WIDTH})")
    return D


def _h_dtype(what, x, other, out_dtype):
    h = other if out_dtype is None else out_dtype
    if h not in (x.dtype, other):
        _fail(what, f"out_dtype {h} is neither {x.dtype} nor {other}")
    return h


def norm(x, weight=None, bias=None, kind="layer", eps=1e-3, out_dtype=None):
    """(x - mean) / sqrt(var + eps) * weight + bias ("layer") or x / sqrt(mean(x^2) + eps) * weight + bias ("rms") over the last dimension.
    out_dtype: x's, or a 16-bit type for a float32 x."""
    what = "norm"
    _check(what, x, weight, bias)
    D = _check_width(what, x)
    if kind is None:
        _fail(what, "kind is None, not 'layer' or 'rms'")
    code = _code(NORMS, kind, what, "kind")
    _check_params(what, D, (("weight", weight), ("bias", bias)))
    h = x.dtype if out_dtype is None else out_dtype
    if h != x.dtype and (x.dtype != torch.float32 or h not in _DTYPES):
        _fail(what, f"out_dtype {h} for {x.dtype} rows")
    cfg = (code, 0, 0, 1.0, float(eps), 0.0, h, 1)
    L.require_cuda(x)
    if _wants_grad(x, weight, bias):
        return _ResidualNorm.apply(x, None, None, weight, bias, None, None, cfg)[1]
    return _norm_forward(x, None, None, weight, bias, None, None, cfg)[1]


def residual_norm(x, branch, weight=None, bias=None, *, norm="layer", eps=1e-3, gate=None, gate_activation="identity", scale=1.0,
                  post_norm=None, post_weight=None, post_bias=None, post_eps=None, out_dtype=None):
    """s = x + scale * act(gate) * post_norm(branch) and h = norm(s), in one pass: what follows a block and precedes the next.

    x, branch [..., D]: of one dtype, or x float32 beside a 16-bit branch.  gate (branch's dtype): shaped like x, or with ones (or nothing) in
    the place of x's last leading dimensions -- [B, 1, D] gates each of B sequences, [D] everything; gate_activation: "identity", "relu",
    "sigmoid" or "silu".  norm, post_norm: "layer", "rms" or None.
    -> (s in x's dtype, h in out_dtype: branch's or x's; None if norm is None).  The norm reads s before it is rounded."""
    what = "residual_norm"
    _check(what, x, branch, gate, weight, bias, post_weight, post_bias)
    D = _check_width(what, x)
    if branch.shape != x.shape or branch.dtype not in _DTYPES or (branch.dtype != x.dtype and x.dtype != torch.float32):
        _fail(what, f"branch {tuple(branch.shape)} {branch.dtype} does not go with x {tuple(x.shape)} {x.dtype}")
    rows = 1
    if gate is not None:
        if gate.dtype != branch.dtype:
            _fail(what, f"gate is {gate.dtype}, branch {branch.dtype}")
        rows = _gate_rows(what, x, gate)
    cfg = (_code(NORMS, norm, what, "norm"), _code(NORMS, post_norm, what, "post_norm"), _code(GATE_ACTIVATIONS, gate_activation, what, "gate_activation"),
           float(scale), float(eps), float(eps if post_eps is None else post_eps), _h_dtype(what, x, branch.dtype, out_dtype), rows)
    if norm is None and (weight is not None or bias is not None):
        _fail(what, "weight or bias without a norm")
    if post_norm is None and (post_weight is not None or post_bias is not None):
        _fail(what, "post_weight or post_bias without a post_norm")
    _check_params(what, D, (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias)))
    L.require_cuda(x)
    if _wants_grad(x, branch, gate, weight, bias, post_weight, post_bias):
        return _ResidualNorm.apply(x, branch, gate, weight, bias, post_weight, post_bias, cfg)
    return _norm_forward(x, branch, gate, weight, bias, post_weight, post_bias, cfg)
