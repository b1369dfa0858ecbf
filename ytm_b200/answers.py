"""From clause outputs to an answer, on torch CUDA tensors (include/ytm.h).

  q4_pack, q4_votes   class sums from clause weights held in 4 bits with a
                      scale for every 32, 64 or 128 clauses of a class
  answer              class biases, allowed classes, penalties for classes
                      answered before and a temperature on class sums, with
                      the chosen class and its log-probability
  class_loss          cross entropy of biased, masked, tempered class sums
                      with the gradients of class sums, bias and temperature

The calls launch on the current stream of the tensors' device and return new
tensors; they keep nothing between calls.  Rows may be strided or repeated
(`expand`); a tensor whose rows are not contiguous inside is copied.  Wrong
types, shapes or devices raise TypeError or ValueError before anything is
launched.  The gradients come with the loss; none of the calls records into
autograd, and a tensor that requires grad is refused while grad mode is on.
"""
from __future__ import annotations

import ctypes as ct

import numpy as np
import torch

from . import _lib
from ._lib import AnswerArgs, LossArgs, check

_TYPES = {torch.int32: _lib.YTM_I32, torch.float32: _lib.YTM_F32, torch.float16: _lib.YTM_F16,
          torch.bfloat16: _lib.YTM_BF16}
_SUMS = tuple(_TYPES)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_F32, _I32, _U8 = (torch.float32,), (torch.int32,), (torch.uint8,)
_INDICES = (torch.int32, torch.int64)
_I64 = torch.int64
_f32 = torch.float32
_empty = torch.empty
_grad = torch.is_grad_enabled
_raw_stream = torch._C._cuda_getCurrentRawStream  # of a device index; current_stream() takes 2 us for the same


def _need(t, name: str, dim: int, types, device=None):
    """Checks one tensor; returns it with contiguous rows."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype not in types:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in types)}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension{'s' if dim > 1 else ''}, got {t.dim()}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, got {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if t.requires_grad and _grad():
        raise ValueError(f"{name} requires grad: these operators do not record into autograd (detach it)")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t


def _vector(t, name: str, n: int, types, device):
    t = _need(t, name, 1, types, device)
    if t.shape[0] != n:
        raise ValueError(f"{name} must have {n} values, got {t.shape[0]}")
    return t


def _call(f, what: str, device, *args) -> None:
    """A library call with the tensors' device as the current one, on its
    current stream."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        check(rc, what)


def pack_allowed(allowed, k: int | None = None):
    """Booleans [n, k] or [k] (numpy or torch) -> the int32 bit words [n or 1,
    ceil(k / 32)] that `allowed` arguments take, as a CPU tensor."""
    a = allowed.detach().cpu().numpy() if isinstance(allowed, torch.Tensor) else np.asarray(allowed)
    a = np.atleast_2d(a).astype(bool)
    if k is not None and a.shape[1] != k:
        raise ValueError(f"allowed must have {k} classes, got {a.shape[1]}")
    pad = np.zeros((a.shape[0], -(-a.shape[1] // 32) * 32), dtype=bool)
    pad[:, :a.shape[1]] = a
    return torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32).copy())


# ------------------------------------------------------------------ 4-bit votes

def q4_pack(weights: torch.Tensor, group: int = 64, scale_dtype: torch.dtype = torch.float32):
    """Clause weights [clauses, classes] (int32 or float32, finite) -> (packed
    uint8 [classes, 16 * ceil(clauses / 32)], scales [classes, ceil(clauses /
    group)]): per class and `group` (32, 64, 128) consecutive clauses the scale
    max|w| / 7 and the weights rounded to [-7, 7] of it (half to even)."""
    w = _need(weights, "weights", 2, (torch.int32, torch.float32))
    C, K = w.shape
    if C == 0 or K == 0:
        raise ValueError("weights must have at least one clause and one class")
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    if scale_dtype not in _FLOATS:
        raise TypeError("scale_dtype must be float32, float16 or bfloat16")
    if C > 1 and w.stride(0) < K:
        w = w.contiguous()
    packed = _empty(K, -(-C // 32) * 16, dtype=torch.uint8, device=w.device)
    scales = _empty(K, -(-C // group), dtype=scale_dtype, device=w.device)
    _call(_lib.load().ytm_q4_pack, "ytm_q4_pack", w.device, w.data_ptr(), _TYPES[w.dtype], w.stride(0) if C > 1 else K,
          C, K, group, packed.data_ptr(), scales.data_ptr(), _TYPES[scale_dtype])
    return packed, scales


def q4_votes(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group: int, bias: torch.Tensor | None = None,
             clauses: int | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Class sums [n, classes] of clause activations under 4-bit weights (see
    q4_pack): bias[k] + sum over the groups of scale * sum of (packed - 8) * x,
    summed in fp32.

    x: real activations [n, clauses] (float32, float16, bfloat16), or clause
    outputs as bits, int32 [n, ceil(clauses / 32)] (`CudaEngine.infer_fired`);
    with bits, `clauses` is needed.  bias: float32 [classes]."""
    x = _need(x, "x", 2, _SUMS)
    dev = x.device
    packed = _need(packed, "packed", 2, _U8, dev)
    scales = _need(scales, "scales", 2, _FLOATS, dev)
    n, width = x.shape
    K, row_bytes = packed.shape
    bits = x.dtype is torch.int32
    if clauses is None:
        if bits:
            raise ValueError("clauses must be given with clause bits")
        clauses = width
    if clauses < 1 or K < 1:
        raise ValueError("needs at least one clause and one class")
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    words = (clauses + 31) // 32
    if width != (words if bits else clauses):
        raise ValueError(f"x has {width} columns, {clauses} clauses need {words if bits else clauses}")
    if row_bytes != words * 16 or not packed.is_contiguous():
        raise ValueError(f"packed must be contiguous [classes, {words * 16}] for {clauses} clauses")
    if scales.shape != (K, (clauses + group - 1) // group) or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous [{K}, {-(-clauses // group)}]")
    if out_dtype not in _FLOATS:
        raise TypeError("out_dtype must be float32, float16 or bfloat16")
    if bias is not None:
        bias = _vector(bias, "bias", K, _F32, dev)
    y = _empty(n, K, dtype=out_dtype, device=dev)
    if n == 0:
        return y
    lib, x_type = _lib.load(), _lib.YTM_BITS if bits else _TYPES[x.dtype]
    ws = _empty(lib.ytm_q4_votes_workspace_bytes(x_type, n, clauses, K, group), dtype=torch.uint8, device=dev)
    _call(lib.ytm_q4_votes, "ytm_q4_votes", dev, x.data_ptr(), x_type, x.stride(0) if n > 1 else 0, n, clauses,
          packed.data_ptr(), scales.data_ptr(), _TYPES[scales.dtype], group, K,
          None if bias is None else bias.data_ptr(), y.data_ptr(), _TYPES[out_dtype], ws.data_ptr())
    return y


# -------------------------------------------------------------- adjusted class sums

def _allowed(allowed, n: int, k: int, device):
    """Allowed-class bit words, checked."""
    a = _need(allowed, "allowed", 2, _I32, device)
    if a.shape[1] != (k + 31) // 32 or a.shape[0] not in (1, n):
        raise ValueError(f"allowed must be int32 [{n} or 1, {(k + 31) // 32}], got {list(a.shape)}")
    return a


def _knob(v, name: str, n: int, device, positive: bool):
    """A number, or float32 [n]: (pointer, value for all rows, tensor)."""
    if isinstance(v, torch.Tensor):
        t = _vector(v, name, n, _F32, device)
        return t.data_ptr(), 0.0, t
    v = float(v)
    if positive and not v > 0.0:
        raise ValueError(f"{name} must be positive, got {v}")
    return None, v, None


def answer(cs: torch.Tensor, bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
           history: torch.Tensor | None = None, lengths: torch.Tensor | None = None, repetition=1.0, frequency=0.0,
           presence=0.0, temperature=1.0, adjusted: bool = True):
    """Adjusted class sums and the answer: (choice int64 [n], logprob float32
    [n], adjusted float32 [n, k] or None).

    cs: class sums [n, k] (int32, float32, float16, bfloat16).  With c the
    number of times class k stands in the row's history (index tensor [n, h],
    int32 or int64, of which the first lengths[n], int32, count; indices
    outside [0, k) count for nothing):

        if c > 0: v = (v > 0 ? v / repetition : v * repetition) - frequency * c - presence
        z = (v + bias) / temperature if allowed else -inf

    in 64 bits, rounded once to float32.  bias: float32 [k] or [n, k];
    allowed: bit words, int32 [n or 1, ceil(k / 32)] (`pack_allowed`);
    repetition, frequency, presence, temperature: numbers (used as float32), or
    float32 [n], whose values are not checked.  choice is the lowest class of
    the largest z (NaN above all, as numpy's argmax), -1 where no class is
    allowed; logprob is log softmax(z) at the choice, -inf where no class is
    allowed."""
    cs = _need(cs, "cs", 2, _SUMS)
    n, k = cs.shape
    dev = cs.device
    if k < 1:
        raise ValueError("cs must have at least one class")
    bias_p = allowed_p = hist_p = lens_p = None
    bias_stride = allowed_stride = hist_stride = hist_len = hist_64 = 0
    if bias is not None:
        if isinstance(bias, torch.Tensor) and bias.dim() == 2:
            bias = _need(bias, "bias", 2, _F32, dev)
            if bias.shape != (n, k):
                raise ValueError(f"bias must be [{k}] or [{n}, {k}], got {list(bias.shape)}")
            bias_stride = bias.stride(0) if n > 1 else 0
        else:
            bias = _vector(bias, "bias", k, _F32, dev)
        bias_p = bias.data_ptr()
    if allowed is not None:
        allowed = _allowed(allowed, n, k, dev)
        allowed_p, allowed_stride = allowed.data_ptr(), allowed.stride(0) if allowed.shape[0] > 1 else 0
    if history is not None:
        history = _need(history, "history", 2, _INDICES, dev)
        if history.shape[0] != n:
            raise ValueError(f"history must have {n} rows, got {history.shape[0]}")
        hist_len = history.shape[1]
        if lengths is not None:
            lengths = _vector(lengths, "lengths", n, _I32, dev)
        if hist_len > 2 ** 31 - 1:
            raise ValueError("history must have fewer than 2^31 entries a row")
        if hist_len:
            hist_p, hist_stride, hist_64 = history.data_ptr(), history.stride(0) if n > 1 else 0, history.dtype is _I64
            if lengths is not None:
                lens_p = lengths.data_ptr()
    elif lengths is not None:
        raise ValueError("lengths needs history")
    rep_p, rep, repetition = _knob(repetition, "repetition", n, dev, True)
    fre_p, fre, frequency = _knob(frequency, "frequency", n, dev, False)
    pre_p, pre, presence = _knob(presence, "presence", n, dev, False)
    tem_p, tem, temperature = _knob(temperature, "temperature", n, dev, True)
    choice = _empty(n, dtype=_I64, device=dev)
    logprob = _empty(n, dtype=_f32, device=dev)
    z = _empty(n, k, dtype=_f32, device=dev) if adjusted else None
    args = AnswerArgs(cs.data_ptr(), cs.stride(0) if n > 1 else 0, n, k, _TYPES[cs.dtype], bias_p, bias_stride, allowed_p,
                      allowed_stride, hist_p, hist_stride, hist_len, hist_64, lens_p, rep_p, fre_p, pre_p, tem_p, rep,
                      fre, pre, tem, choice.data_ptr(), logprob.data_ptr(), None if z is None else z.data_ptr())
    _call(_lib.load().ytm_answer, "ytm_answer", dev, ct.byref(args))
    return choice, logprob, z


def class_loss(cs: torch.Tensor, target: torch.Tensor, bias: torch.Tensor | None = None,
               allowed: torch.Tensor | None = None, temperature=1.0, weight: torch.Tensor | None = None):
    """Cross entropy of z = (cs + bias) / temperature over the allowed classes,
    with its gradients: (loss float32 [n], dcs [n, k] of cs's type or None for
    int32 class sums, dbias float32 [k] or None without bias, dtemperature
    float32 [1]).

        loss[n] = weight[n] * (log sum exp z[n] - z[n, target[n]])
        d = weight (softmax z - onehot), dcs = d / temperature,
        dbias = sum_n d / temperature, dtemperature = -sum d z / temperature

    so the gradients are those of loss.sum(); they are summed in a fixed order.
    target: int32 or int64 [n]; rows with a target outside [0, k) or a weight
    of 0 count for nothing.  A target that its mask forbids gives weight * inf
    and no gradient.  bias: float32 [k]; allowed as for `answer`; temperature:
    a positive number or float32 [1], whose value is not checked; weight:
    float32 [n]."""
    cs = _need(cs, "cs", 2, _SUMS)
    n, k = cs.shape
    dev = cs.device
    if k < 1:
        raise ValueError("cs must have at least one class")
    target = _vector(target, "target", n, _INDICES, dev)
    bias_p = allowed_p = weight_p = dcs_p = dbias_p = ws_p = dcs = dbias = None
    allowed_stride = 0
    if bias is not None:
        bias = _vector(bias, "bias", k, _F32, dev)
        bias_p = bias.data_ptr()
    if allowed is not None:
        allowed = _allowed(allowed, n, k, dev)
        allowed_p, allowed_stride = allowed.data_ptr(), allowed.stride(0) if allowed.shape[0] > 1 else 0
    tem_p, tem, temperature = _knob(temperature, "temperature", 1, dev, True)
    if weight is not None:
        weight = _vector(weight, "weight", n, _F32, dev)
        weight_p = weight.data_ptr()
    lib, cs_type, stride = _lib.load(), _TYPES[cs.dtype], cs.stride(0) if n > 1 else 0
    loss = _empty(n, dtype=_f32, device=dev)
    dtem = _empty(1, dtype=_f32, device=dev)
    if cs_type != _lib.YTM_I32:
        dcs = _empty(n, k, dtype=cs.dtype, device=dev)
        dcs_p = dcs.data_ptr()
    if bias is not None:
        dbias = _empty(k, dtype=_f32, device=dev)
        dbias_p = dbias.data_ptr()
    need = lib.ytm_class_loss_workspace_bytes(n, k, cs_type, stride)
    if need:
        ws = _empty(need, dtype=torch.uint8, device=dev)
        ws_p = ws.data_ptr()
    args = LossArgs(cs.data_ptr(), stride, n, k, cs_type, bias_p, allowed_p, allowed_stride, target.data_ptr(), weight_p,
                    tem_p, tem, target.dtype is _I64, loss.data_ptr(), dcs_p, dbias_p, dtem.data_ptr())
    _call(lib.ytm_class_loss, "ytm_class_loss", dev, ct.byref(args), ws_p)
    return loss, dcs, dbias, dtem
