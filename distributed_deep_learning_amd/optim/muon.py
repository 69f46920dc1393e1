"""Muon: momentum whose matrix updates are orthogonalised by Newton-Schulz products.

For every weight that is a matrix (convolution filters flattened to ``[out, in * kh * kw]``):

    M <- mu M + g;   U = g + mu M (Nesterov) or M;   O = orthogonalise(U);   W <- W - lr (s O + wd W),   s = sqrt(max(1, rows / cols))

Everything else (biases, norm parameters, whatever ``use_muon`` declines) is updated by Adam with its own learning rate.

GPU path: ``csrc/ortho.hip``, all matrices of the arena in shared launches (2, and 3 to 6 for every Newton-Schulz step; one in all when
every matrix fits a CU): the momentum update is fused with
the sums of squares, the weight update with the last product, and the bf16 shadow and the cleared gradient are written along.
CPU path: the same mathematics with torch ops.
"""
from __future__ import annotations

import ctypes as C
from typing import Callable, Optional

import numpy as np
import torch

from ..ops import _lib
from ..ops import kernels as K
from ..parallel.arena import ParamArena
from .fused import _ArenaOptimizer, default_no_decay


def is_matrix(name: str, p: torch.Tensor) -> bool:
    """Default choice of what Muon orthogonalises: tensors of two dimensions and more."""
    return p.dim() >= 2


def _geometry(name: str, p: torch.Tensor):
    """``(rows, cols, scale)`` of the matrix as it lies in memory.  The first dimension indexes rows; the order of the others does not
    matter (orthogonalising commutes with permuting columns), so channels-last filters are taken as they are."""
    rows, cols = p.shape[0], p.numel() // p.shape[0]
    scale = max(1.0, rows / cols) ** 0.5
    if rows == 1 or cols == 1 or p.stride(0) == cols:
        return rows, cols, scale
    if p.dim() == 2 and p.stride(0) == 1:                # stored transposed: so is its orthogonal factor
        return cols, rows, scale
    raise ValueError(f"Muon: parameter {name} with strides {tuple(p.stride())} is no matrix over its first dimension in memory")


def _deal(blocks, length, spread: bool) -> np.ndarray:
    """Which block of a shared launch works on which part of which matrix: ``(matrix, part)`` rows.  The matrices' parts are handed out in
    order of their reductions' ``length``, longest first.  ``spread``: the kernels give each XCD a run of this table; where reductions are not
    cut to like lengths (the products with X) the table is laid out so that every XCD gets an equal share of each matrix, its parts one after
    the other, longest matrices first in dispatch order (block ``d`` runs on XCD ``d % 8``): ResNet-50's 121 and 142 us -> 95 and 122.  Else a
    matrix stays on one XCD, whose L2 its tiles share (spread, the square products take 34 us instead of 32)."""
    n = sum(blocks)
    out, at = np.zeros((n, 2), dtype=np.int32), 0
    for i in sorted(range(len(blocks)), key=lambda i: -length[i]):
        pos = np.arange(at, at + blocks[i])
        at += blocks[i]
        out[pos, 0] = i
        out[pos[np.lexsort((pos, pos % 8))] if spread else pos, 1] = np.arange(blocks[i])
    if spread:
        q, r, d = n // 8, n % 8, np.arange(n)
        x = d % 8
        dealt = np.empty_like(out)
        dealt[np.where(x < r, x * (q + 1), r * (q + 1) + (x - r) * q) + d // 8] = out
        out = dealt
    return out


class Muon(_ArenaOptimizer):
    """``momentum`` holds Muon's momentum for matrices and Adam's first moment for the rest; ``exp_avg_sq`` is used by the rest only.

    ``ns_precision``: ``"single"`` (default) multiplies to fp32's accuracy, as fp32 weights and momentum deserve; ``"half"`` uses 11-bit
    operands (a third of the matrix work, 0.2 % error of the update).  ``adam_lr`` is scaled along when a scheduler changes ``lr``.
    Weight decay is decoupled for matrices (``W -= lr wd W``); Adam's part follows :class:`FusedAdam`.

    Whole matrices are needed on every rank: gradients are all-reduced (``sync="allreduce"``); sharded updates are refused."""

    _state_names = ["momentum", "exp_avg_sq"]

    def __init__(self, arena_or_params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 ns_steps: int = K.NS_STEPS, ns_coefficients=K.NS_COEFFICIENTS, ns_eps: float = K.NS_EPS, ns_precision: str = "single",
                 adam_lr: float = 3e-4, adam_betas=(0.9, 0.95), adam_eps: float = 1e-8, use_muon: Callable = is_matrix,
                 no_decay: Optional[Callable] = default_no_decay, **kw):
        if ns_precision not in ("single", "half"):
            raise ValueError("ns_precision must be 'single' or 'half'")
        if lr <= 0.0:
            raise ValueError("Muon: lr must be positive")
        coef = K.check_newton_schulz(ns_steps, ns_coefficients)
        defaults = dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, adam_ratio=adam_lr / lr,
                        adam_betas=tuple(adam_betas), adam_eps=adam_eps)
        super().__init__(arena_or_params, defaults, no_decay=no_decay, **kw)
        a: ParamArena = self.arena
        self.ns_steps, self.ns_coefficients, self.ns_eps, self.ns_precision = int(ns_steps), coef, float(ns_eps), ns_precision
        self.hyper = torch.zeros(16, dtype=torch.float32, device=a.device)       # [0:8] matrices, [8:16] Adam
        self.matrices = []                                                       # (segment, rows, cols, scale)
        adam_seg = a.chunk_seg.clone()
        for n, p, s in zip(a.names, a.params, a.segments):
            if p.numel() > 0 and p.dim() > 0 and use_muon(n, p):
                self.matrices.append((s, *_geometry(n, p)))
                adam_seg[s.offset // _lib.chunk_elems():(s.offset + s.padded) // _lib.chunk_elems()] = -1
        self._adam_seg = adam_seg if len(self.matrices) < len(a.params) else None
        self._plan = None
        if a.device.type == "cuda" and self.matrices:
            self._plan = self._build_plan()

    def _build_plan(self):
        """Device tables of the shared launches: one record per matrix, and for each launch which block works on which part of which
        matrix."""
        lib = _lib.require()
        prod = 3 if self.ns_precision == "single" else 1
        rec = np.dtype([("elem", "<i8"), ("ws", "<i8"), ("slab", "<i8"), ("rows", "<i4"), ("cols", "<i4"), ("seg", "<i4"), ("scale", "<f4"),
                        ("gram_splits", "<i4"), ("square_splits", "<i4")])
        if rec.itemsize != lib.ddl_ns_mat_bytes():
            raise RuntimeError("Muon: matrix record does not match the kernel library")
        table, launches = np.zeros(len(self.matrices), dtype=rec), [[] for _ in range(8)]
        ws, slabs, out = 0, 0, (C.c_int * 10)()
        solo = all(lib.ddl_ns_solo(rows, cols) for _, rows, cols, _ in self.matrices)        # every matrix fits a CU: one launch for all
        sides = [(C.c_int * len(self.matrices))(*(f(rows, cols) for _, rows, cols, _ in self.matrices)) for f in (min, max)]
        chunks = (C.c_int * 2)()
        _lib.check(lib.ddl_ns_chunks(*sides, len(self.matrices), prod, chunks), "ns_chunks")
        for i, (s, rows, cols, scale) in enumerate(self.matrices):
            need = lib.ddl_ns_shape(rows, cols, prod, 1, *chunks, out)
            if need < 0:
                raise RuntimeError(f"Muon: no plan for a {rows} x {cols} matrix")
            table[i] = (s.offset, ws, slabs, rows, cols, s.index, scale, out[0], out[1])
            if not solo:
                ws += lib.ddl_ns_workspace(rows, cols, prod)
                slabs += need
            for m, n in zip(launches, [1] + [0] * 7 if solo else out[2:10]):
                m.append(n)
        dev = self.arena.device
        maps = np.concatenate([_deal(n, sides[0] if k >= 6 else sides[1], k >= 6) for k, n in enumerate(launches)])
        return {"table": torch.from_numpy(table.view(np.uint8).copy()).to(dev), "maps": torch.from_numpy(np.ascontiguousarray(maps)).to(dev),
                "blocks": (C.c_int * 8)(*(sum(m) for m in launches)), "prod": prod,
                "chains": lib.ddl_ns_chains(*sides, len(self.matrices)),
                "solo": max(max(rows, cols) for _, rows, cols, _ in self.matrices) if solo else 0,
                "coef": (C.c_float * 3)(*self.ns_coefficients), "ws": torch.empty(max(ws, 8), dtype=torch.float16, device=dev),
                "slabs": torch.empty(max(slabs, 4), dtype=torch.float32, device=dev),
                "parts": torch.empty(len(self.matrices) * lib.ddl_ns_max_parts(), dtype=torch.float64, device=dev)}

    def shard_state(self, ranges, gather=None) -> None:
        raise NotImplementedError("Muon needs whole matrices on every rank: use gradient all-reduce, not the sharded (ps) mode")

    def _prepare(self) -> None:
        g, t = self.param_groups[0], self.step_count
        b1, b2 = g["adam_betas"]
        vals = [g["lr"], g["momentum"], 1.0 if g["nesterov"] else 0.0, 0.0, self.grad_scale, 0.0, 0.0, 0.0,
                g["lr"] * g["adam_ratio"], b1, b2, g["adam_eps"], self.grad_scale, 1.0 - b1 ** t, 1.0 - b2 ** t, 0.0]
        if vals != self._hyper_host:
            self.hyper.copy_(torch.tensor(vals, dtype=torch.float32), non_blocking=True)
            self._hyper_host = vals

    def _before_ranges(self, ranges) -> None:
        if ranges is not None and [tuple(r) for r in ranges] != [(0, self.arena.total)]:
            raise NotImplementedError("Muon updates the whole arena at once: element ranges would cut matrices")

    def _update(self, clo: int, chi: int, zero_grad: bool) -> None:
        a = self.arena
        if not self._use_kernel():
            return self._update_cpu(zero_grad)
        lib = _lib.require()
        st = self.flat_state
        if self._plan is not None:
            p = self._plan
            _lib.check(lib.ddl_muon_step(p["table"].data_ptr(), p["maps"].data_ptr(), p["blocks"], a.master.data_ptr(), a.grad.data_ptr(),
                                         st["momentum"].data_ptr(), a.shadow.data_ptr() if a.shadow is not None else None,
                                         self.seg_wd.data_ptr(), self.hyper.data_ptr(), p["ws"].data_ptr(), p["parts"].data_ptr(),
                                         p["slabs"].data_ptr(), p["prod"], self.ns_steps, p["coef"], self.ns_eps, int(zero_grad),
                                         p["solo"], p["chains"], _lib.stream_ptr()), "muon_step")
        if self._adam_seg is not None:
            _lib.check(lib.ddl_flat_adam(a.master.data_ptr(), a.grad.data_ptr(), st["momentum"].data_ptr(),
                                         st["exp_avg_sq"].data_ptr(), a.shadow.data_ptr() if a.shadow is not None else None,
                                         self._adam_seg.data_ptr(), self.seg_wd.data_ptr(), self.hyper.data_ptr() + 32, clo, chi,
                                         int(zero_grad), _lib.stream_ptr()), "flat_adam")

    # ---- CPU path
    def _orthogonalize_cpu(self, u: torch.Tensor) -> torch.Tensor:
        a, b, c = self.ns_coefficients
        x = u / (torch.linalg.vector_norm(u.double()).float() + self.ns_eps)
        tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        for _ in range(self.ns_steps):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        return x.t() if tall else x

    def _update_cpu(self, zero_grad: bool) -> None:
        g, a, t = self.param_groups[0], self.arena, self.step_count
        lr, mu, b1, b2 = g["lr"], g["momentum"], *g["adam_betas"]
        mats = {s.index: (rows, cols, scale) for s, rows, cols, scale in self.matrices}
        for s in a.segments:
            lo, hi, wd = s.offset, s.offset + s.numel, float(self._seg_wd_host[s.index])
            w, gr, m = a.master[lo:hi], a.grad[lo:hi] * self.grad_scale, self.flat_state["momentum"][lo:hi]
            if s.index in mats:
                rows, cols, scale = mats[s.index]
                m.mul_(mu).add_(gr)
                u = gr + mu * m if g["nesterov"] else m
                o = self._orthogonalize_cpu(u.view(rows, cols)).reshape(-1)
                w.mul_(1.0 - lr * wd).add_(o, alpha=-lr * scale)
            else:
                v = self.flat_state["exp_avg_sq"][lo:hi]
                gr = gr + wd * w
                m.mul_(b1).add_(gr, alpha=1 - b1)
                v.mul_(b2).addcmul_(gr, gr, value=1 - b2)
                w.addcdiv_(m / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt_().add_(g["adam_eps"]), value=-lr * g["adam_ratio"])
        if a.shadow is not None:
            a.shadow.copy_(a.master)
        if zero_grad:
            a.grad.zero_()
