"""Operators of a trainable policy on torch tensors, as hand-written HIP kernels of libg1env.so (include/g1nn.h):

    y = rms_norm(x, weight)                                 root-mean-square norm of rows
    y, h = rms_norm(x, weight, residual=r)                  of the stream h = x + r
    q, scale, h = rms_norm_q8(x, weight, residual=r)        its rows in 8 bits, for a policy that acts
    y = gated_linear(x, w_gate, w_up, b_gate, b_up)         act(x w_gate^T + b_gate) * (x w_up^T + b_up)
    y = gated_linear_q8(q, scale, qg, sg, qu, su, ...)      the same on 8-bit rows and weights
    norm = clip_grad_norm(grads, max_norm)                  global norm, and clipping, of many tensors

rms_norm and gated_linear have gradients (torch.autograd). Tensors are float32 or bfloat16 on one GPU, all of one
type in a call; rows have contiguous elements, and a two-dimensional input may have any row stride. Work goes to torch's
current stream, outputs and workspaces come from torch's allocator, and nothing waits for the GPU. An argument that a
kernel does not take raises ValueError, a failed launch RuntimeError; there is no fallback path.
"""
import array
import ctypes

import torch

from g1env import lib

_c = ctypes
_vp, _i, _l, _f = _c.c_void_p, _c.c_int, _c.c_long, _c.c_float

# name -> (restype, argtypes), one for every symbol of include/g1nn.h
SIGNATURES = {
    "g1_nn_rms_norm": (_i, [_i, _l, _i, _vp, _l, _vp, _l, _vp, _f, _vp, _vp, _vp, _vp]),
    "g1_nn_rms_norm_q8": (_i, [_i, _l, _i, _vp, _l, _vp, _l, _vp, _f, _vp, _vp, _vp, _vp]),
    "g1_nn_rms_norm_backward": (_i, [_i, _l, _i] + [_vp, _l] * 3 + [_vp] * 6),
    "g1_nn_rms_norm_backward_workspace": (_l, [_i, _l, _i]),
    "g1_nn_gated": (_i, [_i, _l, _i, _i] + [_vp, _l] * 3 + [_vp, _vp, _i, _vp, _vp]),
    "g1_nn_gated_backward": (_i, [_i, _l, _i, _i] + [_vp, _l] * 3 + [_vp, _vp, _i, _vp, _l] + [_vp] * 7),
    "g1_nn_gated_backward_workspace": (_l, [_i, _l, _i, _i]),
    "g1_nn_gated_q8": (_i, [_i, _l, _i, _i, _vp, _l] + [_vp] * 7 + [_i, _vp, _vp]),
    "g1_nn_clip": (_i, [_i] + [_vp] * 5 + [_f, _vp, _vp, _vp]),
    "g1_nn_clip_workspace": (_l, [_i]),
}
for _name, (_res, _args) in SIGNATURES.items():
    getattr(lib, _name).restype, getattr(lib, _name).argtypes = _res, _args

ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2, "elu": 3}
_TYPE = {torch.float32: 0, torch.bfloat16: 1}


_TYPE_OF = _TYPE.get
_stream_of = torch._C._cuda_getCurrentRawStream   # torch.cuda.current_stream(i).cuda_stream, a twentieth of its time
_device_now = torch._C._cuda_getDevice


def _run(index, fn, *args):
    """Run an entry point on the current stream of device `index`."""
    if index == _device_now():
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream_of(index))
    if rc == -1:
        raise ValueError("refused by libg1env.so (the reason is on stderr)")
    if rc:
        raise RuntimeError("a kernel launch failed (the reason is on stderr)")


def _want(t, name, index, dtype, shape=None):
    """Check a tensor's place, type and shape."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} is not a tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _first(x, name="x"):
    """The type code of the tensor that the others have to go with."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} is not a tensor on a GPU")
    code = _TYPE_OF(x.dtype)
    if code is None:
        raise ValueError(f"{name} is {x.dtype}: float32 and bfloat16 are supported")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} has no row elements")
    return code


def _vector(t, name, index, dtype, shape):
    """Address of a contiguous vector, or None."""
    if t is None:
        return None
    _want(t, name, index, dtype, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _stride(t, name):
    """Elements from row to row of t seen as rows of its last dimension."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.dim() == 2:
        rows, cols = t.stride()
        if cols == 1 or t.shape[1] == 1:
            return rows
    raise ValueError(f"{name}: rows must be contiguous, and evenly spaced")


def _even(t):
    """t itself where its rows can be read as they lie, else a contiguous copy (gradients come in any layout)."""
    return t if t.is_contiguous() or (t.dim() == 2 and t.stride(1) == 1) else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _once():
    """In a backward pass: gradients are enabled there only where a graph of it is asked for."""
    if torch.is_grad_enabled():
        raise RuntimeError("the gradients of g1nn's operators cannot be differentiated again (create_graph)")


# ------------------------------------------------------------------------------------ norm
def _norm_args(x, weight, residual):
    code = _first(x)
    index, dtype, shape = x.get_device(), x.dtype, x.shape
    K = shape[-1]
    w = _vector(weight, "weight", index, dtype, (K,))
    if w is None:
        raise ValueError("weight is not a tensor")
    xs, r, rs = _stride(x, "x"), None, 0
    if residual is not None:
        _want(residual, "residual", index, dtype, shape)
        r, rs = residual.data_ptr(), _stride(residual, "residual")
    return index, (code, x.numel() // K, K, x.data_ptr(), xs, r, rs, w)


def _like(x):
    """A new contiguous tensor of x's shape and type."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _norm_forward(x, weight, residual, eps, keep):
    index, args = _norm_args(x, weight, residual)
    y = _like(x)
    h = _like(x) if residual is not None else None
    rstd = x.new_empty(args[1], dtype=torch.float32) if keep else None
    _run(index, lib.g1_nn_rms_norm, *args, eps, y.data_ptr(), _ptr(h), _ptr(rstd))
    return y, h, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, h, rstd = _norm_forward(x, weight, residual, eps, True)
        ctx.save_for_backward(x if h is None else h, rstd, weight)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        _once()
        h, rstd, weight = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:
            return dh if need_x else None, None, dh if need_r else None, None
        K = h.shape[-1]
        M = h.numel() // K
        code = _TYPE[h.dtype]
        dy = _even(dy)
        dh = None if dh is None else _even(dh)
        dx = _like(h)
        dw = ws = None
        if need_w:
            dw = torch.empty_like(weight)
            ws = h.new_empty(lib.g1_nn_rms_norm_backward_workspace(code, M, K), dtype=torch.uint8)
        _run(h.get_device(), lib.g1_nn_rms_norm_backward, code, M, K, dy.data_ptr(), _stride(dy, "dy"), _ptr(dh),
             0 if dh is None else _stride(dh, "dh"), h.data_ptr(), _stride(h, "h"), rstd.data_ptr(),
             weight.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(ws))
        return dx if need_x else None, dw, dx if need_r else None, None


def rms_norm(x, weight, eps=1e-6, residual=None):
    """Rows of x (with a residual: of the stream h = x + residual) divided by the root of their mean square, times
    weight [K]. Returns y, or (y, h) with a residual. The statistics are taken in 32 bits of the sum before it is
    rounded to h's type. Differentiable in x, weight and residual; K <= 32768."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, weight, residual, eps)
    y, h, _ = _norm_forward(x, weight, residual, eps, False)
    return y if residual is None else (y, h)


def rms_norm_q8(x, weight, eps=1e-6, residual=None):
    """rms_norm with its rows in 8 bits: (q int8, scale float32 per row), and h with a residual; q * scale stands for
    the normed row, with its largest value at 127. A row of zeros has scale 0; a row with an infinity or a NaN has q = 0
    and a scale of NaN. No gradients."""
    index, args = _norm_args(x, weight, residual)
    q = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    h = _like(x) if residual is not None else None
    _run(index, lib.g1_nn_rms_norm_q8, *args, eps, q.data_ptr(), scale.data_ptr(), _ptr(h))
    return (q, scale) if h is None else (q, scale, h)


# ------------------------------------------------------------------------------------ gated block
def _act(name):
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return code


def _gated_args(x, w_gate, w_up, b_gate, b_up, activation):
    code = _first(x)
    index, dt, K = x.get_device(), x.dtype, x.shape[-1]
    _want(w_gate, "w_gate", index, dt)
    shape = w_gate.shape
    if len(shape) != 2 or shape[0] < 1 or shape[1] != K:
        raise ValueError(f"w_gate has shape {tuple(shape)}, not (F, {K})")
    _want(w_up, "w_up", index, dt, shape)
    F = shape[0]
    return index, (code, x.numel() // K, K, F, x.data_ptr(), _stride(x, "x"), w_gate.data_ptr(),
                   _stride(w_gate, "w_gate"), w_up.data_ptr(), _stride(w_up, "w_up"),
                   _vector(b_gate, "b_gate", index, dt, (F,)), _vector(b_up, "b_up", index, dt, (F,)), _act(activation))


def _gated_forward(x, w_gate, w_up, b_gate, b_up, activation):
    index, args = _gated_args(x, w_gate, w_up, b_gate, b_up, activation)
    y = x.new_empty(x.shape[:-1] + (args[3],))
    _run(index, lib.g1_nn_gated, *args, y.data_ptr())
    return y


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        return _gated_forward(x, w_gate, w_up, b_gate, b_up, activation)

    @staticmethod
    def backward(ctx, dy):
        _once()
        tensors = ctx.saved_tensors
        index, args = _gated_args(*tensors, ctx.activation)
        dy = _even(dy)
        grads = [_like(t) if need else None for t, need in zip(tensors, ctx.needs_input_grad)]
        ws = dy.new_empty(lib.g1_nn_gated_backward_workspace(*args[:4]), dtype=torch.uint8)
        _run(index, lib.g1_nn_gated_backward, *args, dy.data_ptr(), _stride(dy, "dy"), *[_ptr(g) for g in grads],
             ws.data_ptr())
        return (*grads, None)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """activation(x w_gate^T + b_gate) * (x w_up^T + b_up) for rows x [..., K] and weights [F, K]. Both projections,
    the activation ("silu", "gelu" in its tanh form, "sigmoid" or "elu") and the product are one kernel. Differentiable
    in all tensors; the gradients compute the projections again, so no [.., F] values are kept for them."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
                                    (b_gate is not None and b_gate.requires_grad) or
                                    (b_up is not None and b_up.requires_grad)):
        return _Gated.apply(x, w_gate, w_up, b_gate, b_up, activation)
    return _gated_forward(x, w_gate, w_up, b_gate, b_up, activation)


def quantize_rows(w):
    """(q int8, scale float32 [rows]) of a weight matrix [F, K], once, for gated_linear_q8: the largest value of each
    row at 127."""
    w = w.detach().float()
    a = w.abs().amax(-1)
    inv = torch.where(a > 0, torch.full_like(a, 127.0) / a, torch.zeros_like(a))
    return torch.round(w * inv[:, None]).to(torch.int8), a / 127.0


def gated_linear_q8(q, scale, w_gate_q, s_gate, w_up_q, s_up, b_gate=None, b_up=None, activation="silu",
                    dtype=torch.float32):
    """The gated block on 8-bit rows q [..., K] with a scale each (rms_norm_q8) and 8-bit weights [F, K] with a scale
    per output (quantize_rows); float32 biases; y [..., F] in dtype. The products are summed as whole numbers. No
    gradients."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype is not torch.int8 or q.dim() < 1 or q.shape[-1] < 1:
        raise ValueError("q is not an int8 tensor of rows on a GPU")
    code = _TYPE_OF(dtype)
    if code is None:
        raise ValueError(f"{dtype}: float32 and bfloat16 are supported")
    index, rows, f32 = q.get_device(), q.shape, torch.float32
    K = rows[-1]
    _want(w_gate_q, "w_gate_q", index, torch.int8)
    shape = w_gate_q.shape
    if len(shape) != 2 or shape[0] < 1 or shape[1] != K:
        raise ValueError(f"w_gate_q has shape {tuple(shape)}, not (F, {K})")
    F = shape[0]
    for t, name in ((scale, "scale"), (s_gate, "s_gate"), (s_up, "s_up")):
        if t is None:
            raise ValueError(f"{name} is not a tensor")
    args = (code, q.numel() // K, K, F, q.data_ptr(), _stride(q, "q"), _vector(scale, "scale", index, f32, rows[:-1]),
            _vector(w_gate_q, "w_gate_q", index, torch.int8, shape), _vector(s_gate, "s_gate", index, f32, (F,)),
            _vector(w_up_q, "w_up_q", index, torch.int8, shape), _vector(s_up, "s_up", index, f32, (F,)),
            _vector(b_gate, "b_gate", index, f32, (F,)), _vector(b_up, "b_up", index, f32, (F,)), _act(activation))
    if None in args[6:11]:
        raise ValueError("w_up_q is not a tensor")
    y = q.new_empty(rows[:-1] + (F,), dtype=dtype)
    _run(index, lib.g1_nn_gated_q8, *args, y.data_ptr())
    return y


# ------------------------------------------------------------------------------------ clipping
def _table(kind, values):
    """A C array of whole numbers, which lives as long as what is returned: (array, address)."""
    t = array.array(kind, values)
    return t, t.buffer_info()[0]


def _tensors(ts, what, index):
    codes = [_TYPE_OF(t.dtype) for t in ts]
    for t, code in zip(ts, codes):
        if t.get_device() != index or code is None or not t.is_contiguous():
            raise ValueError(f"{what} on {t.device}, {t.dtype}{'' if t.is_contiguous() else ', not contiguous'}: contiguous "
                             f"float32 and bfloat16 tensors on one GPU are supported")
    return _table("q", [t.data_ptr() for t in ts]), _table("i", codes)


def clip_grad_norm(grads, max_norm, out=None):
    """The Euclidean norm of all gradients together (a float32 tensor without dimensions, on the GPU), and the
    gradients times min(1, max_norm / (norm + 1e-6)): in place, or into the tensors `out` of the same shapes (float32
    or bfloat16, so 16-bit gradients can be clipped into 32-bit ones). The tensors are contiguous. The squares are summed
    in 64 bits in an order that does not change. A norm that is infinite or NaN makes the factor 0 or NaN."""
    grads = list(grads)
    if not grads:
        raise ValueError("no gradients")
    index = grads[0].get_device()
    if index < 0:
        raise ValueError("the gradients are not on a GPU")
    (pin, pin_at), (tin, tin_at) = _tensors(grads, "a gradient", index)
    pout_at, tout_at = pin_at, tin_at
    if out is not None:
        out = list(out)
        if [t.shape for t in out] != [t.shape for t in grads]:
            raise ValueError("the outputs have other shapes than the gradients")
        (pout, pout_at), (tout, tout_at) = _tensors(out, "an output", index)
    n = len(grads)
    sizes, sizes_at = _table("q", [t.numel() for t in grads])
    # the norm, and behind it the workspace
    both = grads[0].new_empty(4 + lib.g1_nn_clip_workspace(n) // 4, dtype=torch.float32)
    _run(index, lib.g1_nn_clip, n, pin_at, tin_at, pout_at, tout_at, sizes_at, max_norm, both.data_ptr(),
         both.data_ptr() + 16)
    return both[0]


def clip_grad_norm_(parameters, max_norm):
    """clip_grad_norm, in place, of the gradients of those parameters that have one. Without any, a norm of 0."""
    parameters = list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    return clip_grad_norm(grads, max_norm)
