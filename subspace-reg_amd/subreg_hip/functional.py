"""torch.autograd.Function stubs over the C ABI (the reference's "nn.Module + autograd" seam).

Every op launches a hand-written gfx950 kernel on torch's current stream; torch only owns the
memory and records the graph.  Reference call sites are named on each class.
"""
import ctypes as C

import torch

from . import _lib


def _f32c(t):
    assert t.is_cuda, "subreg_hip ops need CUDA (HIP) tensors - there is no CPU fallback"
    assert t.dtype == torch.float32
    return t.contiguous()


class LinearFn(torch.autograd.Function):
    """nn.Linear(640, n_cls, bias) - models/resnet_language.py:138-140,187."""

    @staticmethod
    def forward(ctx, feat, weight, bias):
        lib = _lib.load()
        feat, weight = _f32c(feat), _f32c(weight)
        bias_c = _f32c(bias) if bias is not None else None
        B, D = feat.shape
        N = weight.shape[0]
        logits = torch.empty(B, N, dtype=torch.float32, device=feat.device)
        _lib.check(lib.subreg_linear_fwd(_lib.ptr(feat), _lib.ptr(weight), _lib.ptr(bias_c), _lib.ptr(logits), B, N, D,
                                         _lib.stream_ptr()), "linear_fwd")
        ctx.save_for_backward(feat, weight)
        ctx.has_bias = bias is not None
        return logits

    @staticmethod
    def backward(ctx, dlogits):
        lib = _lib.load()
        feat, weight = ctx.saved_tensors
        dlogits = _f32c(dlogits)
        B, D = feat.shape
        N = weight.shape[0]
        need_f, need_w, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        dfeat = torch.empty_like(feat) if need_f else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty(N, dtype=torch.float32, device=feat.device) if need_b else None
        _lib.check(lib.subreg_linear_bwd(_lib.ptr(dlogits), _lib.ptr(feat), _lib.ptr(weight), _lib.ptr(dw), _lib.ptr(db),
                                         _lib.ptr(dfeat), B, N, D, _lib.stream_ptr()), "linear_bwd")
        return dfeat, dw, db


class SubspaceProjectFn(torch.autograd.Function):
    """P = w Q^T Q, Q rows = orthonormal basis of span(W_base) - LangPuller.get_projected_weight, :92-97.
    The projector is symmetric, so the backward is the same projection applied to grad_output."""

    @staticmethod
    def forward(ctx, w, q):
        lib = _lib.load()
        w, q = _f32c(w), _f32c(q)
        k, D = w.shape
        p = torch.empty_like(w)
        _lib.check(lib.subreg_subspace_project(_lib.ptr(w), _lib.ptr(q), _lib.ptr(p), k, q.shape[0], D,
                                               _lib.stream_ptr()), "subspace_project")
        ctx.save_for_backward(q)
        return p

    @staticmethod
    def backward(ctx, g):
        lib = _lib.load()
        (q,) = ctx.saved_tensors
        g = _f32c(g)
        out = torch.empty_like(g)
        _lib.check(lib.subreg_subspace_project(_lib.ptr(g), _lib.ptr(q), _lib.ptr(out), g.shape[0], q.shape[0], g.shape[1],
                                               _lib.stream_ptr()), "subspace_project(bwd)")
        return out, None


def subspace_basis(base_weight):
    """Orthonormal basis rows [n_base, D] of span(base_weight rows) (replaces torch.qr, :93-94)."""
    lib = _lib.load()
    wb = _f32c(base_weight.detach())
    nb, D = wb.shape
    q = torch.empty_like(wb)
    scratch = torch.empty(nb * D, dtype=torch.float64, device=wb.device)
    info = torch.zeros(1, dtype=torch.int32, device=wb.device)
    _lib.check(lib.subreg_subspace_basis(_lib.ptr(wb), _lib.ptr(q), _lib.ptr(scratch), nb, D, _lib.ptr(info),
                                         _lib.stream_ptr()), "subspace_basis")
    return q, info


class CrossEntropyFn(torch.autograd.Function):
    """nn.CrossEntropyLoss() with mean reduction (train_supervised.py:138, language_eval.py:252); `counters` (optional
    int32[2] tensor) receives the batch's top-1 / top-5 hit counts in the same launch."""

    @staticmethod
    def forward(ctx, logits, target, counters=None, topk=5):
        lib = _lib.load()
        z = _f32c(logits)
        t = target.to(torch.int64).contiguous()
        B, N = z.shape
        rowloss = torch.empty(B, dtype=torch.float32, device=z.device)
        loss = torch.empty(1, dtype=torch.float32, device=z.device)
        dz = torch.empty_like(z)
        _lib.check(lib.subreg_softmax_ce(_lib.ptr(z), _lib.ptr(t), B, N, int(topk), _lib.ptr(rowloss), _lib.ptr(loss), _lib.ptr(dz),
                                         _lib.ptr(counters), _lib.stream_ptr()), "softmax_ce")
        ctx.save_for_backward(dz)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        (dz,) = ctx.saved_tensors
        return dz * g, None, None, None


def cross_entropy(logits, target, counters=None, topk=5):
    return CrossEntropyFn.apply(logits, target, counters, topk)


class SemanticTargetFn(torch.autograd.Function):
    """softmax(E_novel E_base^T / temp [diag := -9999]) @ W_base - LangPuller.forward, :75-83 (gradient to W_base)."""

    @staticmethod
    def forward(ctx, base_weight, novel_embeds, base_embeds, temp, mask):
        lib = _lib.load()
        wb, en, eb = _f32c(base_weight), _f32c(novel_embeds), _f32c(base_embeds)
        assert en.shape[1] == eb.shape[1] and eb.shape[0] == wb.shape[0]
        probs = torch.empty(en.shape[0], eb.shape[0], dtype=torch.float32, device=wb.device)
        out = torch.empty(en.shape[0], wb.shape[1], dtype=torch.float32, device=wb.device)
        _lib.check(lib.subreg_semantic_target(_lib.ptr(en), _lib.ptr(eb), _lib.ptr(wb), en.shape[0], eb.shape[0], en.shape[1],
                                              wb.shape[1], float(temp), int(bool(mask)), _lib.ptr(probs), _lib.ptr(out),
                                              _lib.stream_ptr()), "semantic_target")
        ctx.save_for_backward(probs)
        ctx.shape = tuple(wb.shape)
        return out

    @staticmethod
    def backward(ctx, g):
        (probs,) = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            return None, None, None, None, None
        lib = _lib.load()
        g = _f32c(g)
        gw = torch.empty(ctx.shape, dtype=torch.float32, device=g.device)
        _lib.check(lib.subreg_semantic_target_bwd(_lib.ptr(probs), _lib.ptr(g), probs.shape[0], probs.shape[1], ctx.shape[1],
                                                  _lib.ptr(gw), _lib.stream_ptr()), "semantic_target(bwd)")
        return gw, None, None, None, None


class SqDiffFn(torch.autograd.Function):
    """pull * ||inspired - weights||_F^2 - LangPuller.loss1, :89-90 (gradient to both arguments)."""

    @staticmethod
    def forward(ctx, inspired, weights, pull):
        lib = _lib.load()
        a, b = _f32c(inspired), _f32c(weights)
        assert a.shape == b.shape
        loss = torch.empty(1, dtype=torch.float32, device=a.device)
        _lib.check(lib.subreg_sqdiff(_lib.ptr(a), _lib.ptr(b), a.numel(), float(pull), _lib.ptr(loss), None, 0.0, None,
                                     None, _lib.stream_ptr()), "sqdiff")
        ctx.save_for_backward(a, b)
        ctx.pull = float(pull)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        lib = _lib.load()
        a, b = ctx.saved_tensors
        g = _f32c(g.reshape(1))
        ga = torch.empty_like(a) if ctx.needs_input_grad[0] else None
        gb = torch.empty_like(b) if ctx.needs_input_grad[1] else None
        _lib.check(lib.subreg_sqdiff(_lib.ptr(a), _lib.ptr(b), a.numel(), 0.0, None, _lib.ptr(g), 2.0 * ctx.pull,
                                     _lib.ptr(ga), _lib.ptr(gb), _lib.stream_ptr()), "sqdiff(bwd)")
        return ga, gb, None


class FrobFn(torch.autograd.Function):
    """lmbd * ||rows - anchor||_F, NOT squared, zero sub-gradient at 0 - ResNet.regloss/reglossnovel, :229-240."""

    @staticmethod
    def forward(ctx, rows, anchor, lmbd):
        lib = _lib.load()
        a, b = _f32c(rows), _f32c(anchor)
        assert a.shape == b.shape
        loss = torch.empty(1, dtype=torch.float32, device=a.device)
        _lib.check(lib.subreg_frob(_lib.ptr(a), _lib.ptr(b), a.numel(), float(lmbd), _lib.ptr(loss), None, None,
                                   _lib.stream_ptr()), "frob")
        ctx.save_for_backward(a, b)
        ctx.lmbd = float(lmbd)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        lib = _lib.load()
        a, b = ctx.saved_tensors
        g = _f32c(g.reshape(1))
        ga = torch.empty_like(a)
        _lib.check(lib.subreg_frob(_lib.ptr(a), _lib.ptr(b), a.numel(), ctx.lmbd, None, _lib.ptr(g), _lib.ptr(ga),
                                   _lib.stream_ptr()), "frob(bwd)")
        return ga, None, None


# ---------------------------------------------------------------- teacher / student operators
# The answers of a frozen teacher (its head in 8 bits, the largest logits of each row) and the loss of a student trained on them
# (the reference keeps such losses in distill/).  fp32, bf16 and fp16; rows may be strided; any leading dimensions.
_FLOAT_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _float_code(t, name):
    code = _FLOAT_CODE.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return code


def _on_device(**tensors):
    """The one device all tensors (None: absent) live on."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("%s is on %s, the other tensors are on %s" % (name, t.device, dev))
    if dev.type != "cuda":
        raise RuntimeError("subreg_hip ops need CUDA (HIP) tensors - there is no CPU fallback (got %s)" % dev)
    return dev


def _rows(t, name):
    """t as rows: [n, last] with a contiguous last dimension (a copy only where the strides ask for one)."""
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError("%s needs a last dimension of at least one element, got shape %s" % (name, tuple(t.shape)))
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[0] >= 2 ** 22 or t.shape[1] > 2 ** 30:
        raise ValueError("%s: %d rows of %d; a call takes up to 2^22 - 1 rows of up to 2^30" % (name, t.shape[0], t.shape[1]))
    return _row_major(t)


def _row_major(t):
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _launch(dev, fn, what, *args):
    """fn(*args, stream) on the current stream of `dev`, with `dev` as the current device."""
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _launch(dev, fn, what, *args)
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _lib.check(rc, what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def quantize_rows(x):
    """8-bit codes of each row and their scale: x ~ codes * scale[..., None].

    a = max(max |row|, 2^-100); scale = a / 127; codes = round_half_even(x * (127 / a)), every operation in fp32, so the codes are
    reproducible bit for bit.  A row with a NaN or an infinity: scale NaN, codes 0.  Returns (codes int8 [..., K], scale fp32 [...]);
    the codes' rows start at multiples of 16 bytes, the layout linear_int8 reads fastest.  No gradient."""
    code = _float_code(x, "x")
    rows = _rows(x.detach(), "x")
    dev = _on_device(x=x)
    n, dim = rows.shape
    pitch = (dim + 15) // 16 * 16
    codes = torch.empty(n, pitch, dtype=torch.int8, device=dev)
    scale = torch.empty(n, dtype=torch.float32, device=dev)
    if n:
        _launch(dev, _lib.load().subreg_quantize_rows, "quantize_rows", rows.data_ptr(), rows.stride(0), code, n, dim,
                codes.data_ptr(), pitch, scale.data_ptr())
    return codes[:, :dim].view(x.shape), scale.view(x.shape[:-1])


def _readable16(t):
    """Whether every row of int8 rows may be read up to the next multiple of 16 columns (which aligned rows are)."""
    if t.data_ptr() % 16 or t.stride(0) % 16 or t.shape[1] % 16 == 0:
        return True
    end = t.storage_offset() + (t.shape[0] - 1) * t.stride(0) + (t.shape[1] + 15) // 16 * 16
    return end <= t.untyped_storage().nbytes()


def linear_int8(x, weight, weight_scale, bias=None, x_scale=None, out_dtype=None):
    """nn.Linear with 8-bit integer operands: y = (codes(x) @ weight^T) * x_scale[..., None] * weight_scale (+ bias).

    weight int8 [N, K], weight_scale fp32 [N] (quantize_rows of the fp32 weight, once), bias fp32 [N] or None.
    x: float [..., K] - each row ("token") is quantised within the call as quantize_rows does - or int8 codes with x_scale fp32
    [...].  The integer sums are exact; y is rounded once, to out_dtype (default: x's type, fp32 for codes).
    For frozen heads: there is no gradient, an x that requires one is refused while autograd records."""
    if weight.dtype != torch.int8 or weight.dim() != 2 or weight.shape[0] < 1:
        raise ValueError("weight must be int8 [N, K], got %s %s" % (weight.dtype, tuple(weight.shape)))
    n, dim = weight.shape
    if x.dim() < 1 or x.shape[-1] != dim:
        raise ValueError("x %s does not fit weight %s" % (tuple(x.shape), tuple(weight.shape)))
    if dim > _lib.I8_MAX_DIM:
        raise ValueError("K = %d: 32-bit sums are exact up to K = %d" % (dim, _lib.I8_MAX_DIM))
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,):
        raise ValueError("weight_scale must be float32 [%d]" % n)
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,)):
        raise ValueError("bias must be float32 [%d]" % n)
    if x.dtype == torch.int8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1]:
            raise ValueError("int8 x needs x_scale, float32 %s" % (tuple(x.shape[:-1]),))
        code = _lib.I8
    else:
        if x_scale is not None:
            raise ValueError("x_scale belongs to int8 x; a float x is quantised here")
        code = _float_code(x, "x")
    if torch.is_grad_enabled() and (x.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("linear_int8 has no gradient: call it under torch.no_grad() or on detached tensors")
    out_dtype = out_dtype or (torch.float32 if code == _lib.I8 else x.dtype)
    if out_dtype not in _FLOAT_CODE:
        raise TypeError("out_dtype must be float32, bfloat16 or float16, got %s" % out_dtype)
    rows, w = _rows(x, "x"), _rows(weight, "weight")
    dev = _on_device(x=x, weight=weight, weight_scale=weight_scale, bias=bias, x_scale=x_scale)
    if not _readable16(w):
        w = torch.nn.functional.pad(w, (0, -dim % 16))[:, :dim]
    m = rows.shape[0]
    y = torch.empty(x.shape[:-1] + (n,), dtype=out_dtype, device=dev)
    if m:
        lib = _lib.load()
        nbytes = lib.subreg_linear_int8_ws_bytes(m, dim, n, code, w.data_ptr(), w.stride(0))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        xs = None if x_scale is None else x_scale.reshape(-1).contiguous()
        ws_, b_ = weight_scale.contiguous(), None if bias is None else bias.contiguous()
        _launch(dev, lib.subreg_linear_int8, "linear_int8", rows.data_ptr(), rows.stride(0), code, _ptr(xs), w.data_ptr(), w.stride(0),
                ws_.data_ptr(), _ptr(b_), y.data_ptr(), _FLOAT_CODE[out_dtype], m, dim, n, ws.data_ptr(), nbytes)
    return y


def top_logits(logits, k):
    """The k largest logits of each row, largest first, equal ones by the lower index: (values [..., k], indices int64 [..., k]).

    k <= 256.  A NaN counts as larger than every number, so that it shows.  What a teacher's answer is kept as.  No gradient."""
    code = _float_code(logits, "logits")
    rows = _rows(logits.detach(), "logits")
    n, vocab = rows.shape
    k = int(k)
    if not 1 <= k <= min(vocab, _lib.TOP_MAX):
        raise ValueError("k = %d: 1 ... min(%d, %d) are served" % (k, vocab, _lib.TOP_MAX))
    dev = _on_device(logits=logits)
    shape = logits.shape[:-1] + (k,)
    values = torch.empty(shape, dtype=logits.dtype, device=dev)
    indices = torch.empty(shape, dtype=torch.int64, device=dev)
    if n:
        _launch(dev, _lib.load().subreg_top_logits, "top_logits", rows.data_ptr(), rows.stride(0), code, n, vocab, k, values.data_ptr(),
                indices.data_ptr())
    return values, indices


_REDUCTION = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}


def _distill_desc(z, tv, ti, target, temperature, kd_weight, ce_weight, ignore_index, reduction, ws):
    return _lib.DistillDesc(z.data_ptr(), tv.data_ptr(), ti.data_ptr(), _ptr(target), z.stride(0), tv.stride(0), ti.stride(0),
                            _FLOAT_CODE[z.dtype], _FLOAT_CODE[tv.dtype], z.shape[0], z.shape[1], tv.shape[1],
                            temperature, kd_weight, ce_weight, ignore_index, reduction, 0, None, 0, None, None, ws.data_ptr(), ws.numel())


def _kinds(z, tv, ti, target):
    """What the kernel's bounds rest on."""
    dev = z.device
    return (z.shape, tv.shape, z.dtype, tv.dtype, dev, tv.device == dev and ti.device == dev and ti.shape == tv.shape,
            ti.dtype, target is not None and (target.shape, target.dtype, target.device == dev))


class DistillLossFn(torch.autograd.Function):
    """The loss, and in the same pass over the logits its gradient for an upstream factor of 1 (as CrossEntropyFn does).  The backward
    hands that gradient on where the factor is 1; elsewhere it is computed again with the factor, in fp32 and rounded once - a
    gradient scaled after it was rounded would lose what a loss scale is there to keep (fp16)."""

    @staticmethod
    def forward(ctx, z, tv, ti, target, need_grad, shape, *args):
        lib, dev = _lib.load(), z.device
        ws = torch.empty(lib.subreg_distill_ws_bytes(z.shape[0]), dtype=torch.uint8, device=dev)
        d = _distill_desc(z, tv, ti, target, *args, ws)
        loss = torch.empty(shape, dtype=torch.float32, device=dev)
        d.loss = loss.data_ptr()
        if need_grad:
            dz = torch.empty(z.shape, dtype=z.dtype, device=dev)
            d.dlogits = dz.data_ptr()
            ctx.save_for_backward(z, tv, ti, target)
            ctx.dz, ctx.ws, ctx.desc = dz, ws, d
            ctx.kinds = _kinds(z, tv, ti, target)
        _launch(dev, lib.subreg_distill_loss, "distill_loss", C.byref(d))
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        d, dz = ctx.desc, ctx.dz
        # Under saved-tensor hooks (checkpointing, offloading) these are other tensors than the forward's, which may be gone, and a
        # hook may have laid them out anew.
        saved = z, tv, ti, target = ctx.saved_tensors
        if _kinds(*saved) != ctx.kinds:
            raise RuntimeError("distill_loss: a saved tensor was unpacked with another shape, type or device")
        z, tv, ti, target = _row_major(z), _row_major(tv), _row_major(ti), target if target is None else target.contiguous()
        d.logits, d.top_values, d.top_indices, d.target = z.data_ptr(), tv.data_ptr(), ti.data_ptr(), _ptr(target)
        d.logits_stride, d.values_stride, d.indices_stride = z.stride(0), tv.stride(0), ti.stride(0)
        g = g.reshape(-1)
        d.grad_scale, d.grad_scale_stride = g.data_ptr(), g.stride(0) if g.numel() > 1 else 0
        d.loss = None
        if dz is None:                                   # a second backward over a retained graph: the first took the buffer
            d.flags, dz = _lib.DISTILL_COUNTED, torch.empty(z.shape, dtype=z.dtype, device=z.device)
            d.dlogits = dz.data_ptr()
        else:
            d.flags, ctx.dz = _lib.DISTILL_COUNTED | _lib.DISTILL_SKIP_UNIT, None
        _launch(z.device, _lib.load().subreg_distill_loss, "distill_loss(bwd)", C.byref(d))
        return dz, None, None, None, None, None, None, None, None, None, None


def distill_loss(logits, top_values, top_indices, target=None, temperature=1.0, kd_weight=1.0, ce_weight=0.0, ignore_index=-100,
                 reduction="mean"):
    """Loss of a student on a teacher's kept logits, with the labels' cross entropy in the same pass.

    logits [..., V] of the student; top_values [..., k], top_indices int64 [..., k] (top_logits of the teacher's; an index < 0 or a
    value of -inf drops the entry, an index may repeat); target int64 [...] or None.  Per row
        kd_weight T^2 KL(softmax(top_values / T) || softmax(logits / T)) + ce_weight CE(logits, target)
    with the teacher's softmax over the row's kept entries.  A row without kept entries has no first term, one whose target is
    ignore_index no second; a row with neither is not read, its gradient is 0.  reduction "mean": each term over the rows that have it
    (no such row: 0); "sum"; "none": [...].  Gradient for the logits only, in their type;
    inside a captured graph take it with torch.autograd.grad (as train.GraphedStep does), not with backward().  An index >= V, or a target outside
    [0, V), makes its row's loss and gradient NaN.  temperature: 1e-30 ... 1e15, with kd_weight * temperature ** 2 up to 1e30."""
    _float_code(logits, "logits")
    _float_code(top_values, "top_values")
    lead = logits.shape[:-1]
    if top_indices.dtype not in (torch.int64, torch.int32) or (target is not None and target.dtype not in (torch.int64, torch.int32)):
        raise TypeError("top_indices and target must be int64 or int32")
    if top_values.shape != top_indices.shape or top_values.shape[:-1] != lead or top_values.dim() != logits.dim():
        raise ValueError("top_values %s and top_indices %s do not fit logits %s"
                         % (tuple(top_values.shape), tuple(top_indices.shape), tuple(logits.shape)))
    if target is not None and target.shape != lead:
        raise ValueError("target %s does not fit logits %s" % (tuple(target.shape), tuple(logits.shape)))
    if reduction not in _REDUCTION:
        raise ValueError("reduction must be 'none', 'sum' or 'mean', got %r" % (reduction,))
    temperature, kd_weight, ce_weight = float(temperature), float(kd_weight), float(ce_weight)
    if not 1e-30 <= temperature <= 1e15:
        raise ValueError("temperature must lie in 1e-30 ... 1e15, got %r" % temperature)
    if not abs(kd_weight) * temperature * max(temperature, 1.0) <= 1e30 or not abs(ce_weight) <= 1e30:
        raise ValueError("kd_weight * temperature ** 2 and ce_weight must be numbers up to 1e30")
    z, tv, ti = _rows(logits, "logits"), _rows(top_values.detach(), "top_values"), _rows(top_indices, "top_indices").to(torch.int64)
    if tv.shape[1] > _lib.TOP_MAX:
        raise ValueError("%d entries a row: at most %d are served" % (tv.shape[1], _lib.TOP_MAX))
    _on_device(logits=logits, top_values=top_values, top_indices=top_indices, target=target)
    shape = lead if reduction == "none" else ()
    if z.shape[0] == 0:
        empty = z.float().sum(1)
        return empty.reshape(lead) if reduction == "none" else empty.sum()
    y = None if target is None or ce_weight == 0.0 else target.reshape(-1).to(torch.int64).contiguous()
    need = torch.is_grad_enabled() and z.requires_grad
    return DistillLossFn.apply(z, tv, ti, y, need, shape, temperature, kd_weight, ce_weight, int(ignore_index), _REDUCTION[reduction])
