"""Operators of a sequence block on the HIP path: layer norm, linear with a fused epilogue, gated linear recurrence.

They stand next to the BatchNorm, Linear and Conv1d ops of the model programs for modules that treat every time step of a
window as a row: a module built from them trains through `vae_amd.train.train` (autograd path) with `vae_amd.optim.Adam`.
Each is one launch forward, or two or three where sums are split or ragged rows laid out anew, and differentiable once.
Tensors are fp32, bf16 or fp16 on an MI355X; sums, statistics and states are fp32 (include/vae_amd.h, vae_layer_norm_* /
vae_dense_* / vae_gated_scan_*).  Calls run on the current stream of the tensors' device, allocate through torch's allocator
and can be captured in a graph.  Forward-mode duals, and calls under torch.jit.trace or make_fx, are refused.  Before a backward
pass is captured, drop the eager graphs (losses, outputs) of the same leaves: torch ties a leaf's gradient node to the stream of
the first graph that it was in and would wait for that stream inside the capture, which ends the process.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

_TYPES = {torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}
_ACTS = {"none": L.ACT_NONE, "leaky": L.ACT_LEAKY, "sigmoid": L.ACT_SIGMOID, "gelu": L.ACT_GELU, "silu": L.ACT_SILU}


def _begin(what, x):
    """Checks of the first tensor: (device, VAE_T_* of its type)."""
    device = x.device
    if device.index not in L._device_ok:
        L.require_device(x)
    code = _TYPES.get(x.dtype)
    if code is None:
        raise L.VaeAmdError(f"{what}: fp32, bf16 or fp16 tensors (got {x.dtype})")
    return device, code


def _same(what, t, name, shape, dtypes, device):
    if t.shape == shape and t.dtype in dtypes and t.device == device:
        return
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype not in dtypes:
        raise L.VaeAmdError(f"{what}: {name} is {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    raise L.VaeAmdError(f"{what}: {name} is on {t.device}, the input on {device}")


_raw_stream = torch._C._cuda_getCurrentRawStream  # (torch.cuda.current_stream() takes 15 us on the autograd thread)


def _call(fn, name, device, *args):
    """fn(*args, stream) on the current stream of `device`, whichever device is the current one."""
    i = device.index
    if torch.cuda.current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc != 0:
        L.check(rc, name)


def _p(t):
    return t.data_ptr() if t is not None else None


def _rows(t, cols):
    """t as rows of `cols` contiguous elements at one stride: (tensor that owns the memory, rows, stride); copies where the
    strides are others."""
    rows = t.numel() // cols
    if t.is_contiguous():
        return t, rows, cols
    if t.stride(-1) == 1:
        ld, n = 0, 1
        for size, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
            if size == 1:  # (the last step of every window, say)
                continue
            if n == 1:
                ld = stride
            elif stride != ld * n:
                ld = 0
                break
            n *= size
        if ld >= cols:
            return t, rows, ld
    return t.contiguous(), rows, cols


def _once(backward):
    """once_differentiable, at the price of one question where no second derivative is asked for (2 of 109 us a pass otherwise)."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        if forward_ad._current_level >= 0 and any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
            raise L.VaeAmdError("vae_amd.layers: no forward-mode derivative of a backward pass")
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


_is_tracing, _modes, _PROXY = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._TorchDispatchModeKey.PROXY


def _through_function(what, *ts):
    """Does the call go through its autograd function: where a gradient is asked for, and where forward-mode duals may be about (the
    function refuses them).  The kernels write through pointers: of a bare call torch sees the empty result alone, so a dual would lose
    its tangent and a trace keep the allocation.  Tracing is refused with gradients too: a replay skips the checks of types and sizes."""
    if _is_tracing() or (_modes() and torch._C._get_dispatch_mode(_PROXY) is not None):
        raise L.VaeAmdError(f"{what}: torch.jit.trace and make_fx cannot record this call")
    return forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts))


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_forward(x, weight, bias, eps, device, code, save):
    C = x.shape[-1]
    xr, rows, ld = _rows(x, C)
    y = torch.empty_like(xr, memory_format=torch.contiguous_format)
    w = weight if weight is not None else bias
    wtype = _TYPES[w.dtype] if w is not None else L.T_F32
    stat = mean = rstd = None
    if save:
        stat = xr.new_empty((2, rows), dtype=torch.float32)
        mean = stat.data_ptr()
        rstd = mean + 4 * rows
    if rows:
        _call(L.lib().vae_layer_norm_forward, "vae_layer_norm_forward", device, xr.data_ptr(), ld, _p(weight), _p(bias), y.data_ptr(),
              C, mean, rstd, rows, C, eps, code, wtype)
    return y, xr, rows, ld, stat, wtype


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, device, code):
        y, xr, rows, ld, stat, wtype = _norm_forward(x, weight, bias, eps, device, code, True)
        ctx.save_for_backward(xr, weight, bias, stat)
        ctx.geom = rows, x.shape[-1], ld, device, code, wtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        xr, weight, bias, stat = ctx.saved_tensors
        rows, C, ldx, device, code, wtype = ctx.geom
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty_like(xr, memory_format=torch.contiguous_format) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        dy, _, lddy = _rows(dy, C)
        lib = L.lib()
        ws = xr.new_empty(lib.vae_layer_norm_workspace_floats(rows, C), dtype=torch.float32) if need_w or need_b else None
        sp = stat.data_ptr()
        _call(lib.vae_layer_norm_backward, "vae_layer_norm_backward", device, dy.data_ptr(), lddy, xr.data_ptr(), ldx, _p(weight),
              sp, sp + 4 * rows, _p(dx), C, _p(dw), _p(db), _p(ws), rows, C, code, wtype)
        return dx, dw, db, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, with the biased variance.

    x (..., C); weight, bias (C) or None, fp32 or of x's type (both of one type).  Rows may lie at any stride.  The gradients of
    weight and bias are sums over all rows in fp32, added in a fixed order."""
    device, code = _begin("layer_norm", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: input of shape {tuple(x.shape)}")
    shape, kinds = x.shape[-1:], (torch.float32, x.dtype)
    if weight is not None:
        _same("layer_norm", weight, "weight", shape, kinds, device)
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if bias is not None:
        _same("layer_norm", bias, "bias", shape, kinds if weight is None else (weight.dtype,), device)
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if _through_function("layer_norm", x, weight, bias):
        return _NormFn.apply(x, weight, bias, float(eps), device, code)
    return _norm_forward(x, weight, bias, float(eps), device, code, False)[0]


# ---------------------------------------------------------------------------------------------------- linear
def _linear_forward(x, weight, bias, act, slope, residual, device, code, save):
    N, K = weight.shape
    xr, M, ldx = _rows(x, K)
    wr, _, ldw = _rows(weight, K)
    y = xr.new_empty(x.shape[:-1] + (N,))
    aux = None
    if M:
        rr, ldr = None, 0
        if residual is not None:
            rr, _, ldr = _rows(residual, N)
        lib = L.lib()
        if save and act != L.ACT_NONE:
            aux = xr.new_empty(lib.vae_dense_aux_bytes(M, N, act, code), dtype=torch.uint8)
        ws = None
        if M > 1:  # (a served model's one token skips the question)
            n = lib.vae_dense_forward_workspace_floats(M, N, K, code)
            ws = xr.new_empty(n, dtype=torch.float32) if n else None
        _call(lib.vae_dense_forward, "vae_dense_forward", device, xr.data_ptr(), ldx, wr.data_ptr(), ldw, _p(bias), _p(rr), ldr,
              y.data_ptr(), N, _p(aux), _p(ws), M, N, K, act, slope, code)
    return y, xr, wr, aux, (M, N, K, ldx, ldw, act, slope, device, code)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, slope, device, code):
        y, xr, wr, aux, ctx.geom = _linear_forward(x, weight, bias, act, slope, residual, device, code, True)
        ctx.save_for_backward(xr, wr, aux)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        xr, wr, aux = ctx.saved_tensors
        M, N, K, ldx, ldw, act, slope, device, code = ctx.geom
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        like = torch.empty_like if M else torch.zeros_like
        dx = like(xr, memory_format=torch.contiguous_format) if need_x else None
        dw = like(wr, memory_format=torch.contiguous_format) if need_w else None
        db = (xr.new_empty if M else xr.new_zeros)((N,)) if need_b else None
        if M and (need_x or need_w or need_b):
            dyr, _, lddy = _rows(dy, N)
            lib = L.lib()
            ws = xr.new_empty(lib.vae_dense_workspace_floats(M, N, K, act, code), dtype=torch.float32)
            _call(lib.vae_dense_backward, "vae_dense_backward", device, dyr.data_ptr(), lddy, xr.data_ptr(), ldx, wr.data_ptr(),
                  ldw, _p(aux), _p(dx), _p(dw), _p(db), ws.data_ptr(), M, N, K, act, slope, code)
        return dx, dw, db, dy if need_r else None, None, None, None, None


def linear(x, weight, bias=None, act="none", slope=0.0, residual=None):
    """act(x @ weight.T + bias) + residual in one product, everything behind it in the product's epilogue.

    x (..., K), weight (N, K), bias (N) or None, residual (..., N) or None, all of one type (fp32, bf16, fp16).  act: "none", "leaky"
    (negative side times `slope`; 0: ReLU), "sigmoid", "gelu" (the error function's), "silu".  One row runs as well as many:
    a served model's single tokens take a form of their own."""
    device, code = _begin("linear", x)
    if act not in _ACTS:
        raise ValueError(f"linear: activation {act!r}, expected one of {', '.join(_ACTS)}")
    shape = weight.shape
    if len(shape) != 2 or x.dim() < 1 or x.shape[-1] != shape[1] or shape[0] < 1 or shape[1] < 1:
        raise ValueError(f"linear: input of shape {tuple(x.shape)} with a weight of shape {tuple(shape)}")
    kinds = (x.dtype,)
    _same("linear", weight, "weight", shape, kinds, device)
    if bias is not None:
        _same("linear", bias, "bias", shape[:1], kinds, device)
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if residual is not None:
        _same("linear", residual, "residual", x.shape[:-1] + shape[:1], kinds, device)
    if _through_function("linear", x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, residual, _ACTS[act], float(slope), device, code)
    return _linear_forward(x, weight, bias, _ACTS[act], float(slope), residual, device, code, False)[0]


# ------------------------------------------------------------------------------------------------ gated scan
def _steps(t):
    """t (B, T, D) with contiguous features, as (tensor that owns the memory, sequence stride, step stride)."""
    if t.stride(2) != 1 and t.shape[2] > 1:
        t = t.contiguous()
    return t, t.stride(0), t.stride(1)


def _scan_forward(x, gate, h0, lengths, device, code, save):
    B, T, D = x.shape
    xs, xb, xt = _steps(x)
    gs, gb, gt = _steps(gate)
    y = torch.empty_like(xs, memory_format=torch.contiguous_format)
    hl = xs.new_empty((B, D), dtype=torch.float32)
    kept = None
    lib = L.lib()
    n = lib.vae_gated_scan_workspace_floats(B, T, D, code)
    ws = xs.new_empty(n, dtype=torch.float32) if n else None
    if save:
        n = lib.vae_gated_scan_kept_floats(B, T, D)
        kept = xs.new_empty(n, dtype=torch.float32) if n else None
    _call(lib.vae_gated_scan_forward, "vae_gated_scan_forward", device, xs.data_ptr(), xb, xt, gs.data_ptr(), gb, gt, _p(h0),
          _p(lengths), y.data_ptr(), hl.data_ptr(), _p(kept), _p(ws), B, T, D, code)
    return y, hl, xs, gs, kept


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths, device, code):
        y, hl, xs, gs, kept = _scan_forward(x, gate, h0, lengths, device, code, True)
        ctx.save_for_backward(xs, gs, h0, lengths, kept)
        ctx.device, ctx.code = device, code
        ctx.set_materialize_grads(False)
        return y, hl

    @staticmethod
    @_once
    def backward(ctx, dy, dhl):
        xs, gs, h0, lengths, kept = ctx.saved_tensors
        B, T, D = xs.shape
        need_x, need_g, need_h = ctx.needs_input_grad[:3]
        if dy is None and dhl is None:
            return (None,) * 6
        dx = torch.empty_like(xs, memory_format=torch.contiguous_format) if need_x else None
        dg = torch.empty_like(xs, memory_format=torch.contiguous_format) if need_g else None
        dh0 = torch.empty_like(h0) if need_h else None
        db = dt = 0
        if dy is not None:
            dy, db, dt = _steps(dy)
        if dhl is not None:
            dhl = dhl.contiguous()
        lib, code = L.lib(), ctx.code
        n = lib.vae_gated_scan_workspace_floats(B, T, D, code)
        ws = xs.new_empty(n, dtype=torch.float32) if n else None
        _call(lib.vae_gated_scan_backward, "vae_gated_scan_backward", ctx.device, _p(dy), db, dt, _p(dhl), xs.data_ptr(), xs.stride(0),
              xs.stride(1), gs.data_ptr(), gs.stride(0), gs.stride(1), _p(h0), _p(lengths), _p(kept), _p(dx), _p(dg), _p(dh0),
              _p(ws), B, T, D, code)
        return dx, dg, dh0, None, None, None


def gated_scan(x, gate, h0=None, lengths=None):
    """h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t over the steps of (B, T, D) windows, every feature by itself.

    Returns (y, h_last): y (B, T, D) holds h_t in x's type, h_last (B, D) the fp32 state behind the last step.  h0 (B, D), fp32: the
    state before the first step (None: zeros); one step with h0 is how a served model advances.  lengths (B), int32 or int64 on
    the same device: steps at and behind a sequence's length are padding, whatever they hold; y is 0 there, the state stays.
    x and gate may be strided views with contiguous features (the halves of one projection)."""
    device, code = _begin("gated_scan", x)
    if x.dim() != 3:
        raise ValueError(f"gated_scan: input of shape {tuple(x.shape)}, expected (batch, steps, features)")
    B, T, D = x.shape
    _same("gated_scan", gate, "gate", x.shape, (x.dtype,), device)
    if h0 is not None:
        _same("gated_scan", h0, "h0", (B, D), (torch.float32,), device)
        if not h0.is_contiguous():
            h0 = h0.contiguous()
    if lengths is not None:
        _same("gated_scan", lengths, "lengths", (B,), (torch.int32, torch.int64), device)
        if lengths.dtype != torch.int32 or not lengths.is_contiguous():
            lengths = lengths.clamp(0, T).to(torch.int32).contiguous()
    if B == 0 or T == 0 or D == 0:  # no step: the state stays
        h = h0 if h0 is not None else torch.zeros(B, D, device=device)
        return x * gate, h.clone()
    if _through_function("gated_scan", x, gate, h0):
        return _ScanFn.apply(x, gate, h0, lengths, device, code)
    return _scan_forward(x, gate, h0, lengths, device, code, False)[:2]
