"""Network equaliser that learns from the soft decisions of a fitted VAE equaliser.

The reference's network equalisers (`CNN`, `WienerHammersteinNN`, lib/torch_components.py:122-222; `TorchConvNNPilot`,
lib/real_equalization.py:232-431) are trained on pilot symbols.  A fitted blind equaliser replaces the pilots here: its posterior over
the constellation is the teacher of a small network that classifies every symbol from a window of received samples, over the joint
constellation (I and Q together) and with nonlinearities beyond second order.

    window of samples -> linear, tanh -> n_blocks x [ h + W_down (silu(W_gate h) * (W_up h)) ] -> linear -> logits per constellation point

The windows are never copied out of the received sequence: they are one matrix whose rows start `samples_per_symbol` samples
apart.  Forward, loss and every gradient run in the package's kernels (`dense_ops`), the update in its Adam-AMSGrad kernel;
parameters are one flat float32 pack (cast once a step if the network computes in a 16-bit type).
"""
from __future__ import annotations

import math

import numpy as np
import torch

from . import ops
from .dense_ops import gated_backward, gated_forward, linear_backward, linear_forward, topk_distillation_step
from .torch_components import _resolve_device


class DistilledEqualiser:
    """fit(y, teacher) / apply(y) / estimate_symbol_probs(y) as the blind equalisers; `teacher` is any fitted VAE equaliser of this
    package (it provides `top_logits` and `joint_constellation`).  `window` (odd) samples per symbol are seen, `top_k` points of
    the teacher's posterior are learned from, at `temperature`."""
    IS_PROBABILISTIC = True

    def __init__(self, constellation, samples_per_symbol, batch_size, learning_rate=1e-3, window=25, hidden=64, inner=128,
                 n_blocks=1, top_k=8, temperature=1.0, dtype=torch.float32, torch_device=None, seed=0) -> None:
        if window % 2 == 0 or window < 1:
            raise ValueError("window: an odd number of samples")
        if min(hidden, inner, top_k, batch_size, samples_per_symbol) < 1 or n_blocks < 0:
            raise ValueError("hidden, inner, top_k, batch_size and samples_per_symbol must be positive, n_blocks not negative")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise NotImplementedError(f"float32, bfloat16 or float16 (got {dtype})")
        self.constellation = np.asarray(constellation)
        self.is_complex = np.iscomplexobj(self.constellation)
        self.samples_per_symbol, self.batch_size, self.window = samples_per_symbol, batch_size, window
        self.n_classes, self.n_blocks = len(self.constellation), n_blocks
        self.top_k, self.temperature = min(top_k, self.n_classes), temperature
        self.learning_rate, self.dtype = learning_rate, dtype
        self.torch_device = _resolve_device(torch_device)
        self.loss_print_interval = 100
        features = window * (2 if self.is_complex else 1)
        self._shapes = {"w_in": (hidden, features), "b_in": (hidden,)}
        for i in range(n_blocks):
            self._shapes.update({f"w_gate{i}": (inner, hidden), f"w_up{i}": (inner, hidden), f"w_down{i}": (hidden, inner)})
        self._shapes.update({"w_out": (self.n_classes, hidden), "b_out": (self.n_classes,)})
        generator = torch.Generator().manual_seed(seed)
        parts = [torch.randn(math.prod(s), generator=generator) * (s[-1] ** -0.5 if len(s) == 2 else 0.0) for s in self._shapes.values()]
        self._pack = torch.cat(parts).to(self.torch_device)
        self.optimizer_state = None

    # ---- parameters
    def _views(self, flat):
        out, at = {}, 0
        for name, shape in self._shapes.items():
            n = math.prod(shape)
            out[name] = flat[at:at + n].view(shape)
            at += n
        return out

    def get_parameters(self):
        """{name: float32 view of the parameter pack}."""
        return self._views(self._pack)

    def initialize_optimizer(self):
        self.optimizer_state = [torch.zeros_like(self._pack) for _ in range(4)] + [0]  # gradient, m, v, running max of v, steps

    # ---- received samples -> window matrix
    def _samples(self, y_input):
        y = np.ascontiguousarray(y_input)
        if np.iscomplexobj(y) != self.is_complex:
            raise ValueError("received samples and constellation must both be real or both complex")
        flat = y.astype(np.complex64).view(np.float32) if self.is_complex else y.astype(np.float32)
        ns, half = (2 if self.is_complex else 1), self.window // 2
        padded = np.concatenate((np.zeros(ns * half, np.float32), flat, np.zeros(ns * (half + self.samples_per_symbol), np.float32)))
        return torch.from_numpy(padded).to(self.torch_device).to(self.dtype)

    def _windows(self, samples, first, count):
        """Rows of `window` samples around symbols first ... first + count - 1: a strided view."""
        ns = 2 if self.is_complex else 1
        hop = self.samples_per_symbol * ns
        return samples.as_strided((count, self.window * ns), (hop, 1), samples.storage_offset() + first * hop)

    # ---- network
    def _forward(self, x, p, keep):
        h, z = linear_forward(x, p["w_in"], p["b_in"], activation="tanh", keep=keep)
        kept = [(x, z)]
        for i in range(self.n_blocks):
            g, gu = gated_forward(h, p[f"w_gate{i}"], p[f"w_up{i}"], keep=keep)
            kept.append((h, gu, g))
            h = linear_forward(g, p[f"w_down{i}"], residual=h)[0]
        logits = linear_forward(h, p["w_out"], p["b_out"])[0]
        return logits, kept + [(h,)]

    def loss_and_gradients(self, x, teacher_logits, teacher_index):
        """(per-symbol losses, {name: gradient of their mean}) for a window matrix and the teacher's top logits."""
        p = self._views(self._pack.to(self.dtype))
        logits, kept = self._forward(x, p, True)
        # float16: gradients of a large batch's mean would lie below its normal range, those of the sum above it; halfway, and
        # the rest in float32
        rest = x.shape[0] ** 0.5 if self.dtype == torch.float16 else 1.0
        weight = torch.full((x.shape[0],), rest / x.shape[0], device=self.torch_device)
        loss, d = topk_distillation_step(logits, teacher_logits, teacher_index, weight, temperature=self.temperature)
        grads = {}
        d, grads["w_out"], grads["b_out"] = linear_backward(d, kept[-1][0], p["w_out"])
        for i in reversed(range(self.n_blocks)):
            h, gu, g = kept[1 + i]
            dg, grads[f"w_down{i}"], _ = linear_backward(d, g, p[f"w_down{i}"], need=(True, True, False))
            dh, grads[f"w_gate{i}"], grads[f"w_up{i}"], _, _ = gated_backward(dg, h, p[f"w_gate{i}"], p[f"w_up{i}"], gu,
                                                                              need=(True, True, True, False, False))
            d = d + dh
        x, z = kept[0]
        _, grads["w_in"], grads["b_in"] = linear_backward(d, x, p["w_in"], z, activation="tanh", need=(False, True, True))
        if rest != 1.0:
            grads = {name: g.float() / rest for name, g in grads.items()}
        return loss, grads

    def _class_map(self, teacher):
        points = np.asarray(teacher.joint_constellation)
        if len(points) != self.n_classes:
            raise ValueError(f"the teacher decides among {len(points)} points, this equaliser among {self.n_classes}")
        order = np.argmin(np.abs(points[:, None] - self.constellation[None, :]), axis=1)
        if len(set(order.tolist())) != len(points) or np.max(np.abs(points - self.constellation[order])) > 1e-4:
            raise ValueError("the teacher's constellation is not this equaliser's")
        return torch.from_numpy(order.astype(np.int32)).to(self.torch_device)

    # ---- training and use
    def fit(self, y_input, teacher):
        """One pass over the sequence in batches of `batch_size` symbols -> (equalised symbols, mean loss of every batch)."""
        if self.optimizer_state is None:
            raise Exception("Optimizer has not been initialized yet. Please call 'initialize_optimizer' before proceeding to 'fit'.")
        S, B = self.samples_per_symbol, self.batch_size
        n_batches = len(y_input) // S // B
        if n_batches * S * B != len(y_input):
            print(f"Warning! Number of samples in receiver signal does not match with a multiplum of the symbol length ({S})")
        t_logits, t_index = teacher.top_logits(y_input, self.top_k)
        t_index = self._class_map(teacher)[t_index.long()]
        samples = self._samples(y_input)
        curve = torch.zeros(max(n_batches, 1), device=self.torch_device)
        grad, m, v, vmax = self.optimizer_state[:4]
        for n in range(n_batches):
            x = self._windows(samples, n * B, B)
            loss, grads = self.loss_and_gradients(x, t_logits[n * B:(n + 1) * B], t_index[n * B:(n + 1) * B])
            for name, view in self._views(grad).items():
                view.copy_(grads[name])
            self.optimizer_state[4] += 1
            ops.adam_amsgrad_(self._pack, grad, m, v, vmax, self.learning_rate, self.optimizer_state[4])
            curve[n] = loss.mean()
            if n % self.loss_print_interval == 0:
                print(f"Batch {n}, Loss: {curve[n].item():.3f}")
        return self.apply(y_input), curve.cpu().numpy()[:n_batches]

    def forward_logits(self, y_input, chunk=1 << 18):
        """Logits [N, points] of every symbol of a received sequence, on the device."""
        n = len(y_input) // self.samples_per_symbol
        samples, p = self._samples(y_input), self._views(self._pack.to(self.dtype))
        out = torch.empty((n, self.n_classes), dtype=self.dtype, device=self.torch_device)
        for first in range(0, n, chunk):
            count = min(chunk, n - first)
            out[first:first + count] = self._forward(self._windows(samples, first, count), p, False)[0]
        return out

    def estimate_symbol_probs(self, y_input):
        """Posteriors [points, N], as the probabilistic equalisers return them."""
        return torch.softmax(self.forward_logits(y_input).float(), dim=1).t().contiguous().cpu().numpy()

    def apply(self, y_input):
        """Equalised symbols: the posterior mean."""
        q = self.estimate_symbol_probs(y_input)
        return np.tensordot(self.constellation, q.astype(np.float64), axes=(0, 0)).astype(np.complex64 if self.is_complex else np.float32)

    def __repr__(self) -> str:
        return "DistilledEqualiser"
