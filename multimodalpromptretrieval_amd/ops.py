"""Tensor operators for tuning and serving readers of T5's kind on the device.

The framework's trainer (``train.py``) runs the reference's own step: fp32, teacher forcing, cross
entropy.  ``T5VisionModel`` trains by that loss alone: its logits carry no gradient (``sequence_logps``
scores answers with them, as a reference model).  These operators are for a reader that a user
writes in torch next to it, to tune it on chosen and rejected answers, in bf16, on longer
prompts; each is a differentiable torch function over hand-written kernels of libmpr.so:

* ``embed`` — scaled embedding lookup; its gradient sums the positions of each token, sorted on the
  device (``train.EmbedFn`` groups them on the host);
* ``cross_attention`` — attention to an encoder's states of another length, with key / value heads
  that query heads share, forward and backward, and its form for single tokens;
* ``sequence_logps`` / ``preference_loss`` — log-probabilities of label sequences, and the loss of
  paired answers over them, with the gradient of the logits;
* ``grad_norm`` / ``clip_grads_`` — the global L2 norm of many gradients, and their clipping
  (``T5VisionModel.clip_grad_norm_`` clips a model's).

Conventions.  Floating tensors are float32, bfloat16 or float16; sums and statistics are 32 bits or
wider, and a result is rounded once to its type (bf16 attention also rounds the probabilities
between its two products).  Work goes to the current stream of the tensors' device, which need not
be the current device.  Workspaces come from torch's caching allocator in every call, so calls on
several streams and captured graphs share nothing; nothing waits for the GPU, so device tensors may
be captured into a graph (token ids and labels on the host are uploaded: not inside a capture).
Results are the same bits on every run.  What a call cannot take is refused with ``ValueError`` /
``TypeError`` before anything is launched.  The gradients themselves are not differentiable again;
forward-mode derivatives and ``torch.jit.trace`` are refused (``NotImplementedError``).

Capturing a backward pass: torch ties a leaf's gradient accumulation to the stream of the first
graph that reached it, so drop every loss of the same leaves that ran eagerly (``del loss``) before
capturing, as torch asks for any captured backward.
"""
from __future__ import annotations

import ctypes
import math
from array import array
from functools import lru_cache
from operator import attrgetter, index

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_IDS = {torch.int32: 0, torch.int64: 1}


# ---- arguments -----------------------------------------------------------------------------------
def _floating(t, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, got {type(t).__name__}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: float32, bfloat16 or float16 is needed, got {t.dtype}")
    return code


def _on_gpu(t, name: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{name}: libmpr runs on a GPU, the tensor is on {t.device}")


def _same(a, b, what: str) -> None:
    if a.device != b.device:
        raise ValueError(f"{what}: tensors on {a.device} and {b.device}")
    if a.dtype != b.dtype:
        raise TypeError(f"{what}: {a.dtype} and {b.dtype}")


def _eager(what: str, tensors) -> None:
    """Refuses what a call would otherwise lose without a word: the tangents of forward-mode
    derivatives (no operator has a formula for them), and in a trace the kernels themselves."""
    if torch._C._get_tracing_state() is not None:
        raise NotImplementedError(f"{what}: torch.jit.trace cannot record libmpr's kernels")
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: no forward-mode derivative")


def _rows(t):
    """The tensor with its last dimension contiguous."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _matrix(t):
    """A matrix whose rows are contiguous and do not overlap."""
    if t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _tokens(t, device, name: str, below: int, lowest: int):
    """Token ids as a contiguous device tensor; ids on the host are checked and uploaded."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _IDS:
        raise TypeError(f"{name}: an int32 or int64 tensor is needed, got "
                        f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.is_cuda and t.device == device:
        return t if t.is_contiguous() else t.contiguous()
    if t.device.type == "cpu":
        if t.numel() and (int(t.max()) >= below or int(t.min()) < lowest):
            raise IndexError(f"{name}: values from {int(t.min())} to {int(t.max())}, "
                             f"needed in [{lowest}, {below})")
    elif t.device != device:
        raise ValueError(f"{name}: on {t.device}, needed on {device} (or the host)")
    if device.type != "cuda":
        raise ValueError(f"{name}: libmpr runs on a GPU, the operands are on {device}")
    with torch.cuda.device(device):
        return _lib.to_device_async(t, device).contiguous()


@lru_cache(maxsize=4096)
def _i64(*vals):
    """The sizes or strides as a C array (read only: shared between calls)."""
    return (ctypes.c_int64 * len(vals))(*vals)


def _call(device, name: str, *args) -> None:
    """The library call on the current stream of `device`."""
    i = device.index
    if torch._C._cuda_getDevice() == i:
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(i))


def _ptr(t):
    return None if t is None else t.data_ptr()


@lru_cache(maxsize=4096)
def _bytes(name: str, *sizes) -> int:
    """The size that a workspace entry answers for these sizes."""
    n = ctypes.c_int64()
    _lib.call(name, *sizes, ctypes.byref(n))
    return n.value


def _workspace(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _first_order(backward):
    """``once_differentiable``, entered only where the gradient is asked for with a graph."""
    once = once_differentiable(backward)

    def wrapper(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return wrapper


# ---- embedding -----------------------------------------------------------------------------------
def _embed_fwd(weight, ids, scale):
    w = _matrix(weight)
    V, d = w.shape
    out = torch.empty((*ids.shape, d), dtype=w.dtype, device=w.device)
    _call(w.device, "mpr_embed_lookup", _ptr(w), _DTYPES[w.dtype], V, w.stride(0),
          _ptr(ids), _IDS[ids.dtype], ids.numel(), d, scale, _ptr(out))
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.table = (weight.shape, weight.dtype)
        ctx.args = (scale, padding_idx)
        return _embed_fwd(weight, ids, scale)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        (ids,), ((V, d), dtype), (scale, pad) = ctx.saved_tensors, ctx.table, ctx.args
        n, code = ids.numel(), _DTYPES[dtype]
        dout = _matrix(dout if dout.dim() == 2 else dout.reshape(n, d))
        dw = torch.empty((V, d), dtype=dtype, device=dout.device)
        nbytes = _bytes("mpr_embed_grad_workspace", code, n, V, d)
        ws = _workspace(nbytes, dout.device)
        _call(dout.device, "mpr_embed_grad", _ptr(dout), code, dout.stride(0),
              _ptr(ids), _IDS[ids.dtype], n, V, d, scale, pad, _ptr(dw), _ptr(ws),
              nbytes)
        return dw, None, None, None


def embed(weight, ids, scale: float = 1.0, padding_idx: int = None):
    """``scale * weight[ids]``: ``weight`` [V, d] -> [*ids.shape, d] in the weight's type.

    The gradient ``dweight[v] = scale * sum of dout over the positions with ids == v`` is dense, and
    zero for ``padding_idx`` (counted from the end if negative).  ``ids``: int32 or int64, on the
    weight's device or the host (there checked against the table).  An id outside the table that
    lies on the device cannot be refused without waiting for the GPU: it gives a row of NaN and no
    gradient."""
    _floating(weight, "embed weight")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"embed: a table [V, d] is needed, got {tuple(weight.shape)}")
    V = weight.shape[0]
    pad = -1
    if padding_idx is not None:
        padding_idx = index(padding_idx)
        if not -V <= padding_idx < V:
            raise ValueError(f"embed: padding_idx {padding_idx} in a table of {V} rows")
        pad = padding_idx % V
    scale = float(scale)
    _eager("embed", (weight,))
    ids = _tokens(ids, weight.device, "embed ids", V, 0)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embed.apply(weight, ids, scale, pad)
    return _embed_fwd(weight, ids, scale)


# ---- cross attention -----------------------------------------------------------------------------
_MOST_SCALE = 2.0 ** 120  # times log2(e), it is still a float32
_FEW_ROWS = 8  # rows of a key head that the single-token kernel takes, in any type


def _heads(t):
    """The tensor with the elements of a head adjacent and every head at a multiple of 4 bytes."""
    b, l, h, d = t.stride()
    if d == 1 and (t.dtype == torch.float32 or
                   not ((b | l | h) & 1 or t.data_ptr() & 3)):
        return t
    # (a copy made by clone or contiguous may keep an odd stride of a dimension of size 1)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


@lru_cache(maxsize=4096)
def _xattn_plan(code, q_shape, k_shape, q_st, k_st, v_st, keep_st, dout_st):
    """(dims, strides as the library takes them, workspace bytes of a forward and of a backward)."""
    B, Lq, H, D = q_shape
    dims = _i64(B, H, k_shape[2], Lq, k_shape[1], D)
    strides = _i64(*q_st[:3], *k_st[:3], *v_st[:3], keep_st, *dout_st[:3])
    fwd, bwd = ctypes.c_int64(), ctypes.c_int64()
    _lib.call("mpr_xattn_workspace", dims, code, ctypes.byref(fwd), ctypes.byref(bwd))
    return dims, strides, fwd.value, bwd.value


def _xattn_fwd(q, k, v, keep, scale, for_grad):
    """(out, what rounding took off it (bf16), the rows' statistic), the latter two for_grad."""
    code, shape = _DTYPES[q.dtype], q.shape
    dims, strides, nbytes, _ = _xattn_plan(
        code, shape, k.shape, q.stride(), k.stride(), v.stride(),
        0 if keep is None else keep.stride(0), (0, 0, 0))
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    rest = lse = None
    if for_grad:
        lse = torch.empty((shape[0], shape[2], shape[1]), dtype=torch.float32, device=q.device)
        rest = torch.empty_like(out) if code == 1 else None
    ws = _workspace(nbytes, q.device)
    _call(q.device, "mpr_xattn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(keep), code,
          dims, strides, scale, out.data_ptr(), _ptr(rest), _ptr(lse), _ptr(ws), nbytes)
    return out, rest, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, keep, scale):
        q, k, v = _heads(q), _heads(k), _heads(v)
        out, rest, lse = _xattn_fwd(q, k, v, keep, scale, True)
        ctx.save_for_backward(q, k, v, keep, out, rest, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        q, k, v, keep, out, rest, lse = ctx.saved_tensors
        dout = _heads(dout)
        code = _DTYPES[q.dtype]
        dims, strides, _, nbytes = _xattn_plan(
            code, q.shape, k.shape, q.stride(), k.stride(), v.stride(),
            0 if keep is None else keep.stride(0), dout.stride())
        need_q, need_k, need_v = ctx.needs_input_grad[:3]

        def like(t, wanted):
            return torch.empty(t.shape, dtype=t.dtype, device=t.device) if wanted else None
        dq = like(q, need_q)
        dk = like(k, need_k or need_v)
        dv = like(v, need_k or need_v)
        ws = _workspace(nbytes, q.device)
        _call(q.device, "mpr_xattn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(keep), code,
              dims, strides, ctx.scale, out.data_ptr(), _ptr(rest), lse.data_ptr(),
              dout.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), nbytes)
        return dq, dk if need_k else None, dv if need_v else None, None, None


def cross_attention(q, k, v, key_mask=None, scale: float = 1.0):
    """``softmax(scale q k^T) v`` of queries ``q`` [B, Lq, H, D] over an encoder's ``k``, ``v``
    [B, Lk, Hkv, D] -> [B, Lq, H, D].

    H is a multiple of Hkv: query head h reads key head ``h // (H // Hkv)``, and the gradients of a
    key head sum its query heads'.  D is a multiple of 8 up to 128.  ``scale`` 1 is T5's.
    ``key_mask`` [B, Lk] (or [1, Lk]): the keys that are not 0 / False are attended to; what a
    masked key holds (NaN, infinities) touches nothing and its gradient is 0, and a row whose keys
    are all masked, or Lk = 0, gives 0.  A row whose keys are there and all score -inf (keys that hold
    infinities) has no softmax: it gives NaN.  Any strides will do (the halves of a joint k | v
    projection); heads are read in place where their elements are adjacent and they begin at
    multiples of 4 bytes, and copied otherwise.  float16 is computed in float32 except for single
    tokens (up to 8 rows of queries to a key head, without gradients)."""
    _floating(q, "cross_attention q")
    for t, name in ((k, "k"), (v, "v")):
        _floating(t, "cross_attention " + name)
        _same(q, t, "cross_attention q, " + name)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("cross_attention: q [B, Lq, H, D] and k, v [B, Lk, Hkv, D] are needed, "
                         f"got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lk, Hkv, D = k.shape
    H = q.shape[2]
    if q.shape[0] != B or q.shape[3] != D or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"cross_attention: q {tuple(q.shape)} does not fit k {tuple(k.shape)} "
                         "(batch and head dim equal, query heads a multiple of key heads)")
    if D < 8 or D > 128 or D % 8:
        raise ValueError(f"cross_attention: head dim {D} (a multiple of 8 up to 128)")
    scale = float(scale)
    if not abs(scale) <= _MOST_SCALE:
        raise ValueError(f"cross_attention: scale {scale}")
    keep = None
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor):
            raise TypeError("cross_attention: key_mask is a tensor")
        if key_mask.device != q.device:
            raise ValueError(f"cross_attention: key_mask on {key_mask.device}, q on {q.device}")
        if key_mask.dim() != 2 or key_mask.shape[0] not in (1, B) or key_mask.shape[1] != Lk:
            raise ValueError(f"cross_attention: key_mask {tuple(key_mask.shape)}, "
                             f"needed [{B}, {Lk}]")
    _eager("cross_attention", (q, k, v))
    _on_gpu(q, "cross_attention")
    if scale < 0.0:  # the kernels' running maximum is of unscaled scores
        q, scale = -q, -scale
    grad = (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()
    if q.dtype == torch.float16 and (grad or H // Hkv * q.shape[1] > _FEW_ROWS):
        return cross_attention(q.float(), k.float(), v.float(), key_mask, scale).to(q.dtype)
    if key_mask is not None:
        keep = key_mask if key_mask.dtype == torch.bool else key_mask != 0
        keep = _rows(keep.detach().expand(B, Lk)).view(torch.uint8)
    if grad:
        return _CrossAttention.apply(q, k, v, keep, scale)
    return _xattn_fwd(_heads(q), _heads(k), _heads(v), keep, scale, False)[0]


# ---- log-probabilities and the preference loss -----------------------------------------------------
def _logps_shapes(logits, labels, what):
    _floating(logits, what + " logits")
    if logits.dim() != 3 or logits.shape[2] < 1:
        raise ValueError(f"{what}: logits [S, T, V] are needed, got {tuple(logits.shape)}")
    S, T, V = logits.shape
    if not isinstance(labels, torch.Tensor) or tuple(labels.shape) != (S, T):
        raise ValueError(f"{what}: labels [{S}, {T}] are needed, got "
                         f"{tuple(labels.shape) if isinstance(labels, torch.Tensor) else labels}")


def _label_ids(logits, labels, what):
    return _tokens(labels, logits.device, what + " labels", logits.shape[2], -2 ** 63)


@lru_cache(maxsize=4096)
def _logps_plan(S, T, V):
    """(bytes of the rows' statistics, of dlogps after them, of the workspace at the end)."""
    return 8 * S * T, (4 * S + 7) // 8 * 8, _bytes("mpr_logps_workspace", S, T, V)


def _logps_fwd(logits, labels, pair):
    """(logps, loss, kept); kept: a buffer with the rows' statistics and the loss's derivative by
    logps (and the workspace).  pair: (ref, beta, label_smoothing) or None."""
    S, T, V = logits.shape
    dev = logits.device
    n_stat, n_dlp, n_ws = _logps_plan(S, T, V)
    logps = torch.empty(S, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev) if pair else None
    kept = torch.empty(n_stat + n_dlp + n_ws, dtype=torch.uint8, device=dev)
    ref, beta, smooth = pair or (None, 0.0, 0.0)
    at = kept.data_ptr()
    _call(dev, "mpr_logps_fwd", logits.data_ptr(), _DTYPES[logits.dtype], S, T, V,
          logits.stride(0), logits.stride(1), labels.data_ptr(), _IDS[labels.dtype], T,
          logps.data_ptr(), at, _ptr(ref), beta, smooth, _ptr(loss),
          at + n_stat if pair else None, at + n_stat + n_dlp, n_ws)
    return logps, loss, kept


def _logps_bwd(logits, labels, kept, dlogps, mult):
    """dlogps None: the loss's, which the forward kept."""
    S, T, V = logits.shape
    dx = torch.empty((S, T, V), dtype=logits.dtype, device=logits.device)
    at = kept.data_ptr()
    _call(logits.device, "mpr_logps_bwd", logits.data_ptr(), _DTYPES[logits.dtype], S, T, V,
          logits.stride(0), logits.stride(1), labels.data_ptr(), _IDS[labels.dtype], T, at,
          at + _logps_plan(S, T, V)[0] if dlogps is None else dlogps.data_ptr(), _ptr(mult),
          dx.data_ptr())
    return dx


class _SequenceLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        logits = _rows(logits)
        logps, _, kept = _logps_fwd(logits, labels, None)
        ctx.save_for_backward(logits, labels, kept)
        return logps

    @staticmethod
    @_first_order
    def backward(ctx, dlogps):
        logits, labels, kept = ctx.saved_tensors
        return _logps_bwd(logits, labels, kept, dlogps.contiguous(), None), None


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref, beta, smooth):
        logits = _rows(logits)
        logps, loss, kept = _logps_fwd(logits, labels, (ref, beta, smooth))
        ctx.save_for_backward(logits, labels, kept)
        ctx.mark_non_differentiable(logps)
        ctx.set_materialize_grads(False)  # or torch fills zeros for logps in every backward
        return loss, logps

    @staticmethod
    @_first_order
    def backward(ctx, dloss, _):
        if dloss is None:
            return None, None, None, None, None
        logits, labels, kept = ctx.saved_tensors
        return _logps_bwd(logits, labels, kept, None, dloss), None, None, None, None


def sequence_logps(logits, labels):
    """``sum_t log_softmax(logits[s, t])[labels[s, t]]`` over the positions whose label is not
    negative (-100: ignored, as the trainer's loss does): ``logits`` [S, T, V], ``labels`` [S, T]
    (int32 or int64, device or host) -> [S] float32.

    The rows of ignored positions are not read, and their gradient is 0.  A label >= V on the
    device gives NaN (on the host: IndexError).  Under ``no_grad`` this is the reference model's
    side of ``preference_loss``."""
    _logps_shapes(logits, labels, "sequence_logps")
    _eager("sequence_logps", (logits,))
    labels = _label_ids(logits, labels, "sequence_logps")
    if logits.requires_grad and torch.is_grad_enabled():
        return _SequenceLogps.apply(logits, labels)
    return _logps_fwd(_rows(logits), labels, None)[0]


def preference_loss(logits, labels, ref_logps, beta: float = 0.1, label_smoothing: float = 0.0):
    """The preference loss of P answer pairs: (loss, logps).

    ``logits`` [2P, T, V], ``labels`` [2P, T] (negative: ignored) and ``ref_logps`` [2P], the
    reference model's ``sequence_logps``, hold the chosen answers first, then the rejected ones in
    the same order.  ``margin_p = beta ((logps[p] - logps[P + p]) - (ref[p] - ref[P + p]))`` and
    ``loss = mean_p -(1 - label_smoothing) log sigmoid(margin_p) - label_smoothing log
    sigmoid(-margin_p)``; the margin of an answer that the model rules out (a label's logit of -inf) is
    infinite, and its term the limit.  ``loss`` (a float32 scalar) is differentiable by ``logits``; ``logps``
    [2P] (float32) is for the metrics and is not."""
    _logps_shapes(logits, labels, "preference_loss")
    S = logits.shape[0]
    if S == 0 or S % 2:
        raise ValueError(f"preference_loss: {S} sequences are not pairs")
    if not isinstance(ref_logps, torch.Tensor) or tuple(ref_logps.shape) != (S,):
        raise ValueError(f"preference_loss: ref_logps [{S}] are needed")
    if ref_logps.device != logits.device:
        raise ValueError(f"preference_loss: ref_logps on {ref_logps.device}, logits on "
                         f"{logits.device}")
    beta, smooth = float(beta), float(label_smoothing)
    if not math.isfinite(beta):
        raise ValueError(f"preference_loss: beta {beta}")
    if not 0.0 <= smooth <= 0.5:
        raise ValueError(f"preference_loss: label_smoothing {smooth} (0 to 0.5)")
    _eager("preference_loss", (logits, ref_logps))
    labels = _label_ids(logits, labels, "preference_loss")
    ref = ref_logps.detach().to(torch.float32).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return _PreferenceLoss.apply(logits, labels, ref, beta, smooth)
    logps, loss, _ = _logps_fwd(_rows(logits), labels, (ref, beta, smooth))
    return loss, logps


# ---- gradient clipping ---------------------------------------------------------------------------
def _dense(t) -> bool:
    """Whether the tensor fills its memory without gaps or repeats (in whatever order)."""
    want = 1
    for n, s in sorted(zip(t.shape, t.stride()), key=lambda p: p[1]):
        if n != 1:
            if s != want:
                return False
            want *= n
    return True


_T = torch.Tensor
_dtype_of = attrgetter("dtype")


def _plain(tensors):
    """(dtype codes, device index) of contiguous tensors of the known types on one device, else None.
    A model has hundreds of gradients, so each question goes to all of them in one C loop; what the
    answer None hides is found out and named by the functions below."""
    try:
        codes = list(map(_DTYPES.get, map(_dtype_of, tensors)))
        devices = set(map(_T.get_device, tensors))
        if None in codes or len(devices) != 1 or not all(map(_T.is_contiguous, tensors)):
            return None
    except (TypeError, AttributeError, RuntimeError):
        return None
    return codes, devices.pop()


def _check_grads(grads, what):
    """The dtype codes of the gradients, or the refusal of the first that will not do."""
    codes = [_floating(g, f"{what} gradient {i}") for i, g in enumerate(grads)]
    device = grads[0].device
    for i, g in enumerate(grads):
        if g.device != device or g.layout is not torch.strided:
            raise ValueError(f"{what}: gradient {i} is a {g.layout} tensor on {g.device}, needed "
                             f"dense on {device}")
        if not (g.is_contiguous() or _dense(g)):
            raise ValueError(f"{what}: gradient {i} {tuple(g.shape)} with strides {g.stride()} "
                             "leaves gaps in its memory (clip a .contiguous() copy)")
    return codes


def _check_outs(grads, out, what):
    codes = [_floating(t, f"{what} output {i}") for i, t in enumerate(out)]
    for i, (g, t) in enumerate(zip(grads, out)):
        dense = t.is_contiguous() and g.is_contiguous()
        if t.device != g.device or t.numel() != g.numel() or not (dense or t.shape == g.shape):
            raise ValueError(f"{what}: output {i} is {tuple(t.shape)} on {t.device}, its gradient "
                             f"{tuple(g.shape)} on {g.device}")
        if not dense and t.stride() != g.stride():
            raise ValueError(f"{what}: output {i} is laid out otherwise than its gradient")
    return codes


def _listed(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _clip(grads, out, max_norm, eps, what):
    n = len(grads)
    if out is not None and len(out) != n:
        raise ValueError(f"{what}: {n} gradients and {len(out)} outputs")
    if n == 0:
        return torch.zeros(())
    mine = _plain(grads)
    codes = mine[0] if mine else _check_grads(grads, what)
    counts = array("q", map(_T.numel, grads))
    if out is not None:
        theirs = _plain(out)
        if not (mine and theirs and theirs[1] == mine[1] and
                counts == array("q", map(_T.numel, out))):
            theirs = (_check_outs(grads, out, what),)
    _eager(what, grads)
    if out is not None:
        _eager(what, out)
    _on_gpu(grads[0], what)
    device = grads[0].device
    table = array("q", bytes(40 * n))  # n x {pointer, values, type, output pointer, its type}
    table[0::5] = array("q", map(_T.data_ptr, grads))
    table[1::5] = counts
    table[2::5] = array("q", codes)
    if max_norm is not None:
        table[3::5] = table[0::5] if out is None else array("q", map(_T.data_ptr, out))
        table[4::5] = array("q", codes if out is None else theirs[0])
    desc = (ctypes.c_int64 * (5 * n)).from_buffer(table)
    norm = torch.empty((), dtype=torch.float32, device=device)
    nbytes = ctypes.c_int64()
    _lib.call("mpr_clip_workspace", n, desc, ctypes.byref(nbytes))
    ws = _workspace(nbytes.value, device)
    _call(device, "mpr_clip_grads", n, desc, max_norm or 0.0, eps, _ptr(norm), _ptr(ws),
          nbytes.value)
    return norm


@torch.no_grad()
def grad_norm(grads):
    """The L2 norm of all values of the tensors (or the one tensor) together: a float32 scalar on their
    device, 0 on the host for none.  Squares are summed in 64 bits; a tensor listed twice counts
    twice.  Tensors with gaps in their memory are refused."""
    return _clip(_listed(grads), None, None, 0.0, "grad_norm")


@torch.no_grad()
def clip_grads_(grads, max_norm: float, eps: float = 1e-6, out=None):
    """Scales the gradients by ``min(1, max_norm / (norm + eps))`` and returns ``norm``, their
    global L2 norm before it (``grad_norm``).

    In place, or into ``out``: a tensor for each gradient, of its shape (or, both contiguous, its
    number of values) and any floating type (the optimizer's fp32 buffer for bf16 gradients).
    Gradients below the limit are not written in place at all.  The types may differ between
    tensors, and one tensor alone needs no list.  A norm that is not finite goes through as
    it is: NaN makes every gradient NaN, infinity makes finite ones 0.  Tensors that share memory
    (one gradient listed twice) and gradients with gaps in their memory are refused."""
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"clip_grads_: max_norm {max_norm}, eps {eps}")
    grads = _listed(grads)
    out = None if out is None else _listed(out)
    norm = _clip(grads, out, max_norm, eps, "clip_grads_")
    if grads:
        torch.autograd.graph.increment_version(grads if out is None else out)
    return norm
