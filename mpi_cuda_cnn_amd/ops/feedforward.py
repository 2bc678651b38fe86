"""Feed-forward, 8-bit and distillation operators on torch tensors.

Like the rest of ``ops`` they launch on the current stream of the tensors'
device, allocate their outputs and scratch from torch's caching allocator (so
they may run on any stream, on any device and inside a captured graph) and
have no CPU fallback.  They compute no autograd graph: a backward pass is a
function of its own.

Rows may be strided views.  The kernels read rows in 16-byte pieces: tensors
whose rows are not whole pieces, or not aligned to them, are copied into padded
rows first, in one launch a call; products of up to 32 rows take them as they are, unless only these rows need a copy and
the weights are large.
"""

from __future__ import annotations

import torch

from .. import _C

_K = _C.kernels
# the current stream's handle without the Stream object that torch.cuda.current_stream() builds (1.8 us of a call's 10)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_GATE = {"none": _K.GATE_NONE, "relu": _K.GATE_RELU, "tanh": _K.GATE_TANH, "silu": _K.GATE_SILU,
         "gelu": _K.GATE_GELU}
_SPLIT_ROWS, _SPLIT_BYTES, _SPLIT_OUTPUTS = _K.SPLIT_ROWS, _K.SPLIT_BYTES, _K.SPLIT_OUTPUTS
_ACT = {"none": _K.ACT_NONE, "relu": _K.ACT_RELU, "tanh": _K.ACT_TANH}


def _fail(what):
    raise RuntimeError("mpi_cuda_cnn_amd.ops: " + what)


def _matrix(t, name, dtype, rows=-1, cols=-1):
    """(rows, columns) of t, a 2-D tensor of dtype (one or a tuple), with the numbers of them that are given."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        _fail(f"{name} must be a 2-D tensor")
    if t.dtype is not dtype and not (isinstance(dtype, tuple) and t.dtype in dtype):
        _fail(f"{name} has dtype {t.dtype}, expected {dtype}")
    r, c = t.shape
    if (rows >= 0 and r != rows) or (cols >= 0 and c != cols):
        _fail(f"{name} has shape {(r, c)}, expected {(rows if rows >= 0 else 'any', cols if cols >= 0 else 'any')}")
    return r, c


def _vector(t, name, n, dtype=torch.float32):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.shape[0] != n:
        _fail(f"{name} must be a vector of {n}")
    if t.dtype is not dtype:
        _fail(f"{name} has dtype {t.dtype}, expected {dtype}")


def _device(first, *more):
    """The one GPU that all tensors (None: not given) are on."""
    index = first.get_device()  # (-1 on the CPU; an eighth of the time of comparing device objects)
    if index < 0 or not first.is_cuda:
        _fail("tensors must be on the GPU (no CPU fallback)")
    for t in more:
        if t is not None and t.get_device() != index:
            _fail(f"tensors on different devices ({first.device} and {t.device})")
    return first.device


# Where up to 32 rows alone are not whole pieces they are copied for weights of so many bytes an output column or in all,
# as the kernel that takes rows of any alignment reads the weights as such rows too (us, with a copy / without):
# 1 x 4096 x 8192 27.9 / 36.7, 32 x 4096 x 8192 37 / 56, 1 x 4096 x 512 13.0 / 18.2, int8 1 x 16384 x 64 13.6 / 19.5;
# below it the launch costs more: 1 x 2048 x 2048 12.0 / 10.6, 32 x 512 x 8192 11.8 / 7.9, int8 1 x 8192 x 512 13.0 / 11.0
_COPY_COLUMN, _COPY_WEIGHTS = 1 << 14, 1 << 25


def _pieces(dev, n, x, *weights):
    """((t or a copy, row pitch) of x and the weights, any): rows of whole, aligned 16-byte pieces of n elements, zeros
    behind the last column.  All copies that a call needs are made by one kernel; none for few rows of x (any is then
    True) where a copy would cost more than the product."""
    ts, part = [], []  # (ts: until the kernel is launched, a tensor made here must not go back to the allocator before)
    for t in (x, *weights):
        rows, cols = t.shape
        ld, unit = t.stride()
        if unit != 1 and cols > 1:
            t = t.contiguous()
            ld = cols
        elif rows <= 1:
            ld = cols
        if not (cols % n == 0 and cols <= ld < 1 << 22 and ld % n == 0 and t.data_ptr() % 16 == 0):
            part.append(len(ts))
        ts.append((t, ld))
    if part and x.shape[0] <= _K.ANY_ROWS:
        column = cols * len(weights) * t.element_size()
        if part != [0] or (column < _COPY_COLUMN and column * rows < _COPY_WEIGHTS):
            ts.append(True)
            return ts
    out, todo = ts[:], []
    for i in part:
        t, ld = ts[i]
        rows, cols = t.shape
        pitch = (cols + n - 1) // n * n
        copy = torch.empty(rows, pitch, dtype=t.dtype, device=dev)
        size = t.element_size()
        todo.append((t.data_ptr(), copy.data_ptr(), ld * size, pitch * size, rows, cols * size))
        out[i] = (copy, pitch)
    if todo:
        _run(dev, _K.pad_rows, todo)
    out.append(False)
    return out


def _work(dev, nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _run(dev, fn, *args):
    """fn(*args, stream) with dev as the current device (a kernel's launch goes to the current one)."""
    index = dev.index
    if index == _current():
        fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            fn(*args, _raw_stream(index))


def _gate_kind(act):
    kind = _GATE.get(act)
    if kind is None:
        _fail(f"unknown activation {act!r} (one of {', '.join(_GATE)})")
    return kind


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, act: str = "silu", save: bool = False):
    """h = act(x @ w_gate.T) * (x @ w_up.T): both projections of a gated feed-forward block, the activation and the
    product in one kernel.

    x [M, D], w_gate, w_up [F, D], bf16, D < 4194304; act: none, relu, tanh, silu or gelu (the erf form).  Sums, activation and
    product are fp32, h [M, F] is rounded once to bf16.  With save=True returns (h, gate, up), the two projections
    rounded to bf16, which gated_linear_bwd takes."""
    kind = _gate_kind(act)
    M, D = _matrix(x, "x", torch.bfloat16)
    F, _ = _matrix(w_gate, "w_gate", torch.bfloat16, -1, D)
    _matrix(w_up, "w_up", torch.bfloat16, F, D)
    if D == 0 or F == 0:
        _fail("gated_linear: empty weights")
    dev = _device(x, w_gate, w_up)
    h = torch.empty(M, F, dtype=torch.bfloat16, device=dev)
    gate, up = (torch.empty_like(h), torch.empty_like(h)) if save else (None, None)
    if M:
        if (D % 8 == 0 and x.is_contiguous() and w_gate.is_contiguous() and w_up.is_contiguous()
                and not (x.data_ptr() | w_gate.data_ptr() | w_up.data_ptr()) & 15):  # the usual case, in less time
            xa, ldx, wg, wu, ldw, any_ = x, D, w_gate, w_up, D, False
        else:
            (xa, ldx), (wg, ldw), (wu, ldu), any_ = _pieces(dev, 8, x, w_gate, w_up)
            if ldu != ldw:  # both weights are read with one pitch
                wg, wu, ldw = wg.contiguous(), wu.contiguous(), wg.shape[1]
        few = M > _SPLIT_ROWS and 2 * D >= _SPLIT_BYTES and M * F <= _SPLIT_OUTPUTS and not any_  # (others are never split)
        work = _work(dev, _K.gated_forward_bytes(M, D, F)) if few else None
        _run(dev, _K.gated_forward, M, D, F, kind, xa.data_ptr(), ldx, wg.data_ptr(), wu.data_ptr(), ldw, h.data_ptr(),
             gate.data_ptr() if save else 0, up.data_ptr() if save else 0, any_, work.data_ptr() if work is not None else 0)
    return (h, gate, up) if save else h


def linear_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              b: torch.Tensor | None = None, act: str = "none", out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y = act((x @ w.T) * x_scale[:, None] * w_scale + b) on 8-bit integers.

    x [M, K] int8 with a scale per row (token) x_scale [M], w [N, K] int8 with a scale per row (output channel)
    w_scale [N], b [N] or None, all three fp32; act: none, relu or tanh.  The integer sum is exact in 32 bits
    (K <= 131071), scaling, bias and activation are fp32, y [M, N] is rounded once to out_dtype (bf16 or fp32)."""
    if act not in _ACT:
        _fail(f"unknown activation {act!r} (one of {', '.join(_ACT)})")
    if out_dtype not in (torch.bfloat16, torch.float32):
        _fail(f"linear_i8: unsupported out_dtype {out_dtype} (bf16 / fp32)")
    M, K = _matrix(x, "x", torch.int8)
    N, _ = _matrix(w, "w", torch.int8, -1, K)
    if K == 0 or N == 0:
        _fail("linear_i8: empty weights")
    if K > _K.LINEAR_I8_MAX_K:
        _fail(f"linear_i8: K = {K} is over {_K.LINEAR_I8_MAX_K}, the most that 32-bit sums hold exactly")
    _vector(x_scale, "x_scale", M)
    _vector(w_scale, "w_scale", N)
    if b is not None:
        _vector(b, "b", N)
    dev = _device(x, x_scale, w, w_scale, b)
    y = torch.empty(M, N, dtype=out_dtype, device=dev)
    if M:
        if K % 16 == 0 and x.is_contiguous() and w.is_contiguous() and not (x.data_ptr() | w.data_ptr()) & 15:
            xa, ldx, wa, ldw, any_ = x, K, w, K, False  # the usual case, in less time
        else:
            (xa, ldx), (wa, ldw), any_ = _pieces(dev, 16, x, w)
        sx, sw = x_scale.contiguous(), w_scale.contiguous()
        bias = b.contiguous() if b is not None else None
        few = M > _SPLIT_ROWS and K >= _SPLIT_BYTES and M * N <= _SPLIT_OUTPUTS and not any_
        work = _work(dev, _K.linear_i8_bytes(M, N, K)) if few else None
        _run(dev, _K.linear_i8, M, N, K, _ACT[act], xa.data_ptr(), ldx, sx.data_ptr(), wa.data_ptr(), ldw, sw.data_ptr(),
             bias.data_ptr() if bias is not None else 0, y.data_ptr(), out_dtype == torch.float32, any_,
             work.data_ptr() if work is not None else 0)
    return y


def _strided(t):
    """(t or a copy, row pitch): unit stride along the columns."""
    if t.is_contiguous():
        return t, t.shape[1]
    rows, cols = t.shape
    ld, unit = t.stride()
    if (cols > 1 and unit != 1) or (rows > 1 and ld < cols):
        t = t.contiguous()
        ld = cols
    return t, ld if rows > 1 else cols


def gated_linear_bwd(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, gate: torch.Tensor,
                     up: torch.Tensor, act: str = "silu"):
    """(dx [M, D], dw_gate [F, D], dw_up [F, D]), bf16, of gated_linear from dh [M, F] and the (gate, up) that it saved;
    M <= 4000000, F <= 1048576.

    The gradients of the two projections are rounded to bf16, the matrix unit's operand type; sums are fp32 in a fixed
    order (the same call gives the same bits)."""
    kind = _gate_kind(act)
    M, D = _matrix(x, "x", torch.bfloat16)
    F, _ = _matrix(w_gate, "w_gate", torch.bfloat16, -1, D)
    _matrix(w_up, "w_up", torch.bfloat16, F, D)
    for t, name in ((dh, "dh"), (gate, "gate"), (up, "up")):
        _matrix(t, name, torch.bfloat16, M, F)
    if D == 0 or F == 0:
        _fail("gated_linear_bwd: empty weights")
    dev = _device(x, w_gate, w_up, dh, gate, up)
    dx = torch.empty(M, D, dtype=torch.bfloat16, device=dev)
    if M == 0:
        return dx, torch.zeros_like(w_gate, memory_format=torch.contiguous_format), torch.zeros_like(
            w_up, memory_format=torch.contiguous_format)
    dw = torch.empty(2, F, D, dtype=torch.bfloat16, device=dev)
    work = torch.empty(_K.gated_backward_bytes(M, D, F), dtype=torch.uint8, device=dev)
    dh, gate, up = dh.contiguous(), gate.contiguous(), up.contiguous()
    xa, ldx = _strided(x)
    wg, ldw = _strided(w_gate)
    wu, ldu = _strided(w_up)
    if ldu != ldw:
        wg, wu, ldw = wg.contiguous(), wu.contiguous(), D
    _run(dev, _K.gated_backward, M, D, F, kind, dh.data_ptr(), gate.data_ptr(), up.data_ptr(), xa.data_ptr(), ldx,
         wg.data_ptr(), wu.data_ptr(), ldw, dx.data_ptr(), dw.data_ptr(), work.data_ptr())
    return (dx, *dw.unbind())


def rmsnorm_i8(x: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """(q, scale, s): s = x + residual, y = s * w / sqrt(mean(s**2) + eps) quantised per row to 8 bits.

    x, residual [M, D], w [D], all bf16 or all fp32, D <= 32768.  scale [M] fp32 = max|y| / 127 and q [M, D] int8 =
    y / scale rounded to nearest even: linear_i8's x and x_scale.  s [M, D] in x's type, from which the norm is NOT
    taken again (it is of the unrounded sum); without a residual s is x.  A row of zeros has scale 0; a row that holds
    a value that is not finite, or overflows fp32 in its sum of squares or in s * w (with eps = 0: or underflows the
    sum), has scale NaN and q = 0, so what is computed from it is NaN.  Inference only: an 8-bit output has no gradient."""
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bfloat16, torch.float32):
        _fail("x must be a bf16 or fp32 tensor")
    M, D = _matrix(x, "x", x.dtype)
    if D == 0 or D > _K.RMSNORM_I8_MAX_D:
        _fail(f"rmsnorm_i8: rows of 1 to {_K.RMSNORM_I8_MAX_D} values, got {D}")
    _vector(w, "w", D, x.dtype)
    if residual is not None:
        _matrix(residual, "residual", x.dtype, M, D)
    if not 0 <= eps < 1e38:
        _fail(f"rmsnorm_i8: eps = {eps} must be finite and not negative")
    dev = _device(x, w, residual)
    q = torch.empty(M, D, dtype=torch.int8, device=dev)
    scale = torch.empty(M, dtype=torch.float32, device=dev)
    s = x if residual is None else torch.empty(M, D, dtype=x.dtype, device=dev)
    if M:
        xa, ldx = _strided(x)
        ra, ldr = _strided(residual) if residual is not None else (None, 0)
        wa = w.contiguous()
        _run(dev, _K.rmsnorm_i8, M, D, x.dtype == torch.float32, xa.data_ptr(), ldx, ra.data_ptr() if ra is not None else 0,
             ldr, wa.data_ptr(), eps, s.data_ptr() if ra is not None else 0, q.data_ptr(), scale.data_ptr())
    return q, scale, s


def distill_kl(logits: torch.Tensor, t_logits: torch.Tensor, t_index: torch.Tensor, temperature: float = 1.0,
               scale: float = 1.0, grad: bool = True, grad_dtype: torch.dtype | None = None):
    """(dlogits, loss): distillation from a teacher's top logits, forward and backward in one call.

    logits [M, N] (the student's, bf16 or fp32); row m of t_logits [M, K] (bf16 or fp32) holds the teacher's logits of
    the classes t_index [M, K] (int32 or int64), K <= 1024, in any order.  An entry whose class is not in [0, N) (say
    -1) or whose logit is -inf is not there; classes that occur twice add up.  With T = temperature
    (1e-6 to 1e6), q = softmax(t_logits[m] / T) over the entries that are there and p = softmax(logits[m] / T):

        loss[m]    = T**2 * sum_k q_k (log q_k - log p[t_index[m, k]])            fp32 [M]
        dlogits[m] = scale * T * (p - q scattered to its classes)                 [M, N]

    The loss is a difference of fp32 logarithms: it is off by up to some 2**-18 * T**2, which matters where the entries
    are nearly all of the classes, as the loss does not grow with T then (1000 of 1000 classes, loss 6.5: 8e-3 at T =
    100, 1 at T = 1000).  The gradient is off by some 2**-20 * scale * T * (p + q).

    A row without entries has loss 0 and gradient 0.  dlogits is the gradient of scale * loss.sum(), in grad_dtype
    (default: the logits' type; fp32 logits have fp32 gradients); None with grad=False."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.bfloat16, torch.float32):
        _fail("logits must be a bf16 or fp32 tensor")
    M, N = _matrix(logits, "logits", logits.dtype)
    if N == 0:
        _fail("distill_kl: no classes")
    _, K = _matrix(t_logits, "t_logits", (torch.bfloat16, torch.float32), M)
    _matrix(t_index, "t_index", (torch.int32, torch.int64), M, K)
    if K > _K.DISTILL_MAX_K:
        _fail(f"distill_kl: at most {_K.DISTILL_MAX_K} entries per row, got {K}")
    if not (1e-6 <= temperature <= 1e6):
        _fail(f"distill_kl: temperature = {temperature} must lie between 1e-6 and 1e6")
    out = logits.dtype if grad_dtype is None else grad_dtype
    if out not in (torch.float32, logits.dtype):
        _fail(f"distill_kl: unsupported grad_dtype {out} (fp32 or the logits' type)")
    dev = _device(logits, t_logits, t_index)
    dz = torch.empty(M, N, dtype=out, device=dev) if grad else None
    loss = torch.empty(M, dtype=torch.float32, device=dev)
    if M:
        f32 = logits.dtype == torch.float32
        za, ldz = _strided(logits)
        tl, ti = t_logits.contiguous(), t_index.contiguous()
        work = _work(dev, _K.distill_bytes(M, N, f32))
        _run(dev, _K.distill_kl, M, N, K, za.data_ptr(), ldz, f32, tl.data_ptr(), tl.dtype == torch.float32, ti.data_ptr(),
             ti.dtype == torch.int64, temperature, scale, dz.data_ptr() if grad else 0, out == torch.float32,
             loss.data_ptr(), work.data_ptr() if work is not None else 0)
    return dz, loss


__all__ = ["gated_linear", "gated_linear_bwd", "linear_i8", "rmsnorm_i8", "distill_kl"]
