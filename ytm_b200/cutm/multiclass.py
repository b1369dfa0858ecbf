"""MultiClassTM — reference src/cutm/multiclass.py:6-59 on the B200 engine."""
from __future__ import annotations

import numpy as np
import torch

from .. import answers
from .base import BaseTM


class MultiClassTM(BaseTM):
    def __init__(self, number_of_clauses_per_class: int, T: int, s: float, dim: tuple[int, int, int],
                 n_classes: int, **opt_args):
        super().__init__(number_of_clauses_per_class=number_of_clauses_per_class, T=T, s=s, dim=dim,
                         n_classes=n_classes, **opt_args)

    def encode_Y(self, Y) -> np.ndarray:
        """+T for the true class, -T for the others (multiclass.py:35-37)."""
        Y = np.asarray(Y)
        return np.where(Y[:, None] == np.arange(self.number_of_outputs)[None, :], self.T, -self.T).astype(np.int32)

    def fit(self, X, Y, is_X_encoded: bool = False, **opt_args):
        Yn = Y.cpu().numpy() if isinstance(Y, torch.Tensor) else np.asarray(Y)
        assert Yn.ndim == 1, "Y must be 1D array (samples,)"
        assert X.shape[0] == Yn.shape[0], "X and Y must have the same number of samples."
        encoded_Y = self.encode_Y(Yn)
        encoded_X = self._literals_device(X, is_X_encoded)
        self._fit(encoded_X, encoded_Y, **opt_args)

    def score(self, X, is_X_encoded: bool, block_size: int | None = None, votes=None):
        """Class sums float32 [samples, classes]; with `votes` (pack_votes)
        those of the weights packed to 4 bits."""
        lits = self._literals_device(X, is_X_encoded)
        return self._score_device(lits, votes=votes).cpu().numpy().astype(np.float32)

    def predict(self, X, is_X_encoded: bool = False, block_size: int | None = None, votes=None):
        class_sums = self.score(X, is_X_encoded, block_size=block_size, votes=votes)
        preds = np.argmax(class_sums, axis=1)
        return preds, class_sums

    def _on_device(self, a, dtype):
        return None if a is None else torch.as_tensor(a).to(device=self.device, dtype=dtype)

    def answer(self, X, is_X_encoded: bool = False, votes=None, bias=None, allowed=None, history=None, lengths=None,
               repetition=1.0, frequency=0.0, presence=0.0, temperature=1.0):
        """predict with class sums adjusted first, on the device: (choice int64
        [samples], log-probability float32 [samples], adjusted class sums
        float32 [samples, classes]).

        bias [classes] or [samples, classes]; allowed: booleans of the same
        shapes (-inf and never chosen where false; choice -1 where all are);
        history [samples, h]: classes answered before (negative entries count
        for nothing), of which the first lengths[sample] count; repetition,
        frequency, presence penalise them, temperature divides: numbers, or one
        per sample (the formula: ytm_b200.answers.answer).  `bias` and
        `temperature` may be those that `calibrate` returns."""
        cs = self._score_device(self._literals_device(X, is_X_encoded), votes=votes)
        if allowed is not None:
            allowed = answers.pack_allowed(allowed, self.number_of_outputs).to(self.device)
        knobs = {name: v if np.ndim(v) == 0 and not isinstance(v, torch.Tensor) else self._on_device(v, torch.float32)
                 for name, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence),
                                 ("temperature", temperature))}
        choice, logprob, z = answers.answer(cs, bias=self._on_device(bias, torch.float32), allowed=allowed,
                                            history=self._on_device(history, torch.int64),
                                            lengths=self._on_device(lengths, torch.int32), **knobs)
        return choice.cpu().numpy(), logprob.cpu().numpy(), z.cpu().numpy()

    def calibrate(self, X, Y, is_X_encoded: bool = False, votes=None, steps: int = 100, lr: float = 0.1,
                  temperature: float | None = None):
        """Fit a class bias and a temperature that make softmax((class sums +
        bias) / temperature) the probabilities of the labels Y (negative: no
        label): `steps` Adam steps on the mean cross entropy of the samples,
        the temperature in its logarithm and the bias in units of the first
        temperature (default T / 4).  The model does not change.  Returns
        (bias float32 [classes], temperature)."""
        Yd = self._on_device(Y, torch.int64)
        assert Yd.dim() == 1 and Yd.shape[0] == X.shape[0], "X and Y must have the same number of samples."
        cs = self._score_device(self._literals_device(X, is_X_encoded), votes=votes)
        t0 = float(self.T) / 4 if temperature is None else float(temperature)
        n = max(1, int(((Yd >= 0) & (Yd < self.number_of_outputs)).sum()))
        weight = torch.full((Yd.shape[0],), 1.0 / n, device=self.device)
        theta = torch.zeros(self.number_of_outputs + 1, device=self.device)  # bias / t0, log(temperature / t0)
        m, v = torch.zeros_like(theta), torch.zeros_like(theta)
        for i in range(1, steps + 1):
            t = t0 * theta[-1:].exp()
            _, _, db, dt = answers.class_loss(cs, Yd, bias=theta[:-1] * t0, temperature=t, weight=weight)
            g = torch.cat([db * t0, dt * t])
            m.lerp_(g, 0.1)
            v.lerp_(g * g, 0.001)
            theta -= lr * (m / (1 - 0.9 ** i)) / ((v / (1 - 0.999 ** i)).sqrt() + 1e-8)
        return (theta[:-1] * t0).cpu().numpy(), float(t0 * theta[-1].exp())
