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
autograd, and a tensor that requires grad is refused while grad mode is on, as
is one with a forward-mode tangent.
"""
from __future__ import annotations

import ctypes as ct

import numpy as np
import torch

from . import _lib

try:
    from . import _answers as _bind
except ImportError as e:
    class _Missing:
        """The binding was not built: every call says so."""

        def __init__(self, why):
            self._why = why

        def __getattr__(self, name):
            raise _lib.YTMError(f"ytm_b200/_answers.so cannot be loaded ({self._why}): build it with "
                                "`python -m ytm_b200.build`")

    _bind = _Missing(e)


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
    max|w| / 7 and the weights rounded to [-7, 7] of it (half to even).  float16
    scales hold weights of up to 7 * 65504."""
    return _bind.q4_pack(weights, group, scale_dtype)


def q4_votes(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group: int, bias: torch.Tensor | None = None,
             clauses: int | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Class sums [n, classes] of clause activations under 4-bit weights (see
    q4_pack): bias[k] + sum over the groups of scale * sum of (packed - 8) * x,
    summed in fp32.

    x: real activations [n, clauses] (float32, float16, bfloat16), or clause
    outputs as bits, int32 [n, ceil(clauses / 32)] (`CudaEngine.infer_fired`);
    with bits, `clauses` is needed.  bias: float32 [classes].  float32
    activations, and 16-bit ones of one or two samples, are held to 2^-30 of the
    largest of their 128 neighbouring clauses; several infinities among those
    give NaN."""
    return _bind.q4_votes(x, packed, scales, group, bias, clauses, out_dtype)


def q4_votes_gave_up(device=None) -> int:
    """How many blocks of q4_votes calls that have ended on the device (default:
    the current one) gave up a wait, since the process began.  Their votes are
    NaN; 0 unless the device is in trouble.  Waits for the current stream."""
    out = ct.c_uint64()
    with torch.cuda.device(device):
        _lib.check(_lib.load().ytm_q4_votes_gave_up(ct.byref(out), ct.c_void_p(torch.cuda.current_stream().cuda_stream)),
                   "ytm_q4_votes_gave_up")
    return out.value


# -------------------------------------------------------------- adjusted class sums

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

    in 64 bits (divisions as products with reciprocals), rounded once to
    float32.  bias: float32 [k] or [n, k];
    allowed: bit words, int32 [n or 1, ceil(k / 32)] (`pack_allowed`);
    repetition, frequency, presence, temperature: numbers (used as float32), or
    float32 [n] or [], whose values are not checked.  choice is the lowest class of
    the largest z (NaN above all, as numpy's argmax), -1 where no class is
    allowed; logprob is log softmax(z) at the choice, -inf where no class is
    allowed."""
    return _bind.answer(cs, bias, allowed, history, lengths, repetition, frequency, presence, temperature, adjusted)


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
    a positive number or float32 [1] or [], whose value is not checked; weight:
    float32 [n].  cs + bias is a float32 sum; int32 class sums keep their
    differences at any size.  A NaN or +inf among a row's allowed class sums makes its loss
    and gradients NaN."""
    return _bind.class_loss(cs, target, bias, allowed, temperature, weight)
