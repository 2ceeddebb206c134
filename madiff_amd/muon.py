"""The Muon step over a flat parameter buffer: momentum, Newton-Schulz orthogonalisation of every weight matrix at once,
decoupled weight decay, update, bf16 shadow and moving average (csrc/ortho.hip).

For a matrix W [rows, cols] with gradient g and momentum M:

    M <- mu M + (1 - mu) g,   U = (1 - mu) g + mu M  (Nesterov) or M
    O = Newton-Schulz(U)                                              (ops.orthogonalize)
    W <- (1 - lr wd) W - lr scale O

The reference trains with Adam (diffuser/utils/training.py:109); this is an alternative next to it, for the matrices only:
gains, shifts, biases and embeddings stay with Adam (trainer.FlatMuonEMA does both).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch

from . import lib, ops


class MuonPlan:
    """Where the matrices of a flat float32 buffer are, and the device tables that let one call update all of them.

    matrices: (offset, rows, cols) in elements, row-major, not overlapping; scales: the factor on lr of each (default 1).
    A plan is immutable; step() takes its workspace from torch's allocator call by call, so steps on several streams, or
    captured into several graphs, do not share one."""

    def __init__(self, matrices: Sequence[Tuple[int, int, int]], device="cuda", scales: Optional[Sequence[float]] = None):
        self.matrices = [tuple(int(v) for v in m) for m in matrices]
        if not self.matrices:
            raise ValueError("MuonPlan: no matrices")
        if scales is not None and len(scales) != len(self.matrices):
            raise ValueError(f"MuonPlan: {len(scales)} scales for {len(self.matrices)} matrices")
        end = 0
        for at, rows, cols in sorted(self.matrices):
            if at < 0 or rows < 1 or cols < 1:
                raise ValueError(f"MuonPlan: a matrix has an offset >= 0 and at least one row and column, not {(at, rows, cols)}")
            if at < end:
                raise ValueError(f"MuonPlan: the matrix at {at} overlaps the one before it, which ends at {end}")
            end = at + rows * cols
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"MuonPlan: the plan has to be on the GPU, not on {self.device}")
        n = len(self.matrices)
        at = (C.c_long * n)(*[m[0] for m in self.matrices])
        rows, cols = ((C.c_int * n)(*[min(m[i], 2 ** 31 - 1) for m in self.matrices]) for i in (1, 2))
        sc = (C.c_float * n)(*[1.0 if scales is None else float(v) for v in (scales or [1.0] * n)])
        need = C.c_long()
        if lib._lib.madiff_muon_plan(n, at, rows, cols, sc, None, 0, C.byref(need)) != 0:
            raise ValueError("MuonPlan: a matrix is out of range (shorter side up to 16384, longer up to 4194304), or all of them have "
                             "more than 2^33 elements")
        self._host = torch.zeros(need.value, dtype=torch.uint8)
        lib.call("madiff_muon_plan", n, at, rows, cols, sc, self._host.data_ptr(), need.value, C.byref(need))
        ws, elements = C.c_long(), C.c_long()
        lib.call("madiff_muon_plan_ws", self._host.data_ptr(), C.byref(ws), C.byref(elements))
        self.ws_bytes, self.elements = ws.value, elements.value
        self._dev = self._host.to(self.device)
        self.device = self._dev.device

    def _check(self, name, t, dtype=torch.float32):
        if not torch.is_tensor(t) or t.device != self.device or t.dtype != dtype or not t.is_contiguous() or t.dim() != 1:
            raise ValueError(f"MuonPlan.step: {name} has to be a contiguous one-dimensional {dtype} tensor on {self.device}")
        if t.numel() < self.elements:
            raise ValueError(f"MuonPlan.step: {name} has {t.numel()} elements, the matrices end at {self.elements}")
        return t.data_ptr()

    @torch.no_grad()
    def step(self, p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, *, lr: float, momentum: float = 0.95, nesterov: bool = True,
             weight_decay: float = 0.0, ema: Optional[torch.Tensor] = None, ema_beta: float = 0.995, do_ema: Optional[int] = None,
             shadow: Optional[torch.Tensor] = None, grad_scale: float = 1.0, zero_grad: bool = False, steps: int = 5,
             coefficients: Sequence[float] = ops.NEWTON_SCHULZ, eps: float = 1e-7, state: Optional[torch.Tensor] = None) -> None:
        """One step, in place, on the current stream: p, g, m (and ema) flat float32, shadow bfloat16.  do_ema: 0 none, 1 lerp
        with ema_beta (the default where ema is given), 2 copy; state (int32[2] on the GPU): the mode is state[1] instead
        (none without ema).
        zero_grad: clear g as it is read.  Elements outside the plan's matrices are not touched."""
        ops._refuse_tangents("MuonPlan.step", p, g, m, ema, shadow)
        ptrs = [self._check(k, t) for k, t in (("p", p), ("g", g), ("m", m))]
        pe = None if ema is None else self._check("ema", ema)
        ps = None if shadow is None else self._check("shadow", shadow, torch.bfloat16)
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (p, g, m, ema, shadow) if t is not None)
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("MuonPlan.step: p, g, m, ema and shadow must not overlap")
        if state is not None and (state.device != self.device or state.dtype != torch.int32 or state.numel() < 2 or not state.is_contiguous()):
            raise ValueError(f"MuonPlan.step: state has to be a contiguous int32[2] on {self.device}")
        do_ema = (0 if ema is None else 1) if do_ema is None else int(do_ema)
        if do_ema not in (0, 1, 2) or (do_ema and ema is None):
            raise ValueError(f"MuonPlan.step: do_ema has to be 0, 1 or 2, and 0 without ema, not {do_ema}")
        lr, momentum, weight_decay, ema_beta = float(lr), float(momentum), float(weight_decay), float(ema_beta)
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"MuonPlan.step: momentum has to be in [0, 1), not {momentum}")
        args = ops._check_newton_schulz("MuonPlan.step", steps, coefficients, eps)
        ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=self.device)
        ops._launch(p, lambda st: lib.call(
            "madiff_muon_step", self._host.data_ptr(), self._dev.data_ptr(), *ptrs, pe, ps, p.numel(), lr, momentum, 1 - momentum,
            int(bool(nesterov)), 1 - lr * weight_decay, float(grad_scale), int(bool(zero_grad)), do_ema, ema_beta, 1 - ema_beta,
            ops._p(state), *args, ws.data_ptr(), self.ws_bytes, st))
