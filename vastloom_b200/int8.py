"""A MoE layer whose experts are 8-bit integers with a scale a channel, from the router to the combine.

Any expert matrix becomes int8 here: a resident ggml matrix of every storage type (dequantized on the
device, then rounded row by row) or a float32 array. All types then run the same tensor-core products,
where the block formats Q4_K, Q5_K, Q6_K, IQ2_S and MXFP4 otherwise have CUDA-core kernels only; the
price is one byte a weight and the rounding of weights and activations to 8 bits.

    logits -> route -> balance loss and per-expert counts -> plan (pairs by expert)
           -> gate/up product of the pairs' tokens -> SwiGLU and down product -> combine (+ shared)

The layer math is the reference's (moe_forward, deepseek_v4_graph.cpp:1902-2274); the route weight
multiplies a pair's down row. Every step is a call of the public C ABI on device buffers.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Union

import numpy as np

from . import (DTYPE_BF16, SCORE_SQRT_SOFTPLUS, Device, Int8Weights, Matrix, balance_workspace_bytes,
               int8_workspace_bytes)

Expert = Union[Matrix, np.ndarray]


class Int8Experts:
    """`groups` int8 matrices [rows, cols] in one device allocation, filled matrix by matrix."""

    def __init__(self, dev: Device, groups: int, rows: int, cols: int):
        self.dev, self.rows, self.cols = dev, rows, cols
        self.stride = (cols + 15) // 16 * 16
        self._q = dev.buffer(groups * rows * self.stride, "int8-weights")
        try:
            self._s = dev.buffer(groups * rows * 4, "int8-scales")
        except BaseException:
            self._q.free()
            raise
        self.weights = Int8Weights(self._q.address, self._s.address, rows, cols, groups=groups, stride=self.stride)

    def fill(self, group: int, row0: int, source: Expert) -> None:
        """Rounds `source` ([n, cols]) into rows row0 .. row0 + n of a group."""
        dev = self.dev
        if isinstance(source, Matrix):
            n, cols = source.rows, source.cols
        else:
            source = np.ascontiguousarray(source, dtype=np.float32)
            n, cols = source.shape
        if cols != self.cols or not 0 <= row0 <= self.rows - n or not 0 <= group < self.weights.groups:
            raise ValueError(f"a [{n}, {cols}] matrix does not fit rows {row0}.. of [{self.rows}, {self.cols}]")
        wide = dev.buffer(n * cols * 4, "int8-source")
        try:
            if isinstance(source, Matrix):
                dev._check(dev.lib.vlb_dequantize_device(dev.h, source.ptr, wide.ptr, None))
            else:
                wide.upload(source)
            at = group * self.rows + row0
            dev.int8_quantize_device(wide.address, n, cols, self._q.address + at * self.stride,
                                     self._s.address + at * 4, q_stride=self.stride)
            dev.synchronize()
        finally:
            wide.free()

    def free(self) -> None:
        self._q.free()
        self._s.free()


class Int8MoeLayer:
    """One MoE layer on int8 experts: w1, w3 ([I, H]) and w2 ([H, I]) of every expert, optionally a
    shared expert's three. swiglu_limit clamps the routed experts' SwiGLU, shared_swiglu_limit the
    shared one's (None: as the routed ones; 0: no clamp), as the two limits of MoeLayer. The gate and
    up values between the two products are held in bf16 (half of f32's bytes through HBM; their
    rounding, 2^-9, is below that of the 8-bit rows made of them). Every forward also takes the
    balance loss and the counts."""

    def __init__(self, dev: Device, *, router: np.ndarray, w1: Sequence[Expert], w3: Sequence[Expert],
                 w2: Sequence[Expert], top_k: int, score: int = SCORE_SQRT_SOFTPLUS, bias: Optional[np.ndarray] = None,
                 route_scale: float = 1.0, swiglu_limit: float = 0.0,
                 shared: Optional[tuple[Expert, Expert, Expert]] = None, max_tokens: int = 64,
                 shared_swiglu_limit: Optional[float] = None):
        self.dev, self.top_k, self.score, self.route_scale = dev, top_k, score, route_scale
        self.swiglu_limit, self.max_tokens = swiglu_limit, max_tokens
        self.shared_swiglu_limit = swiglu_limit if shared_swiglu_limit is None else shared_swiglu_limit
        router = np.ascontiguousarray(router, dtype=np.float32)
        self.E, self.H = router.shape
        if not len(w1) == len(w3) == len(w2) == self.E:
            raise ValueError("every expert needs w1, w3 and w2")
        self.I = self._shape(w1[0])[0]
        for a, b, c in [*zip(w1, w3, w2), *([shared] if shared else [])]:
            if not self._shape(a) == self._shape(b) == (self.I, self.H) or self._shape(c) != (self.H, self.I):
                raise ValueError(f"an expert's matrices must be [{self.I}, {self.H}] twice and [{self.H}, {self.I}]")
        self._bufs: list = []
        try:
            self._create(router, bias, w1, w3, w2, shared)
        except BaseException:
            self.close()
            raise

    def _create(self, router, bias, w1, w3, w2, shared) -> None:
        dev, E, H, I, T, k = self.dev, self.E, self.H, self.I, self.max_tokens, self.top_k
        self._router = self._keep(dev.to_device(router))
        self._bias = None if bias is None else self._keep(dev.to_device(np.ascontiguousarray(bias, np.float32)))
        self.gate_up = self._keep(Int8Experts(dev, E, 2 * I, H))
        self.down = self._keep(Int8Experts(dev, E, H, I))
        for e in range(E):
            self._fill(self.gate_up, self.down, e, w1[e], w3[e], w2[e])
        self.shared = None
        if shared is not None:
            self.shared = (self._keep(Int8Experts(dev, 1, 2 * I, H)), self._keep(Int8Experts(dev, 1, H, I)))
            self._fill(*self.shared, 0, *shared)
        n = T * k
        sizes = dict(x=T * H * 4, logits=T * E * 4, idx=n * 4, weights=n * 4, row_index=n * 4, row_weight=n * 4,
                     elem_row=n * 4, offsets=(E + 2) * 4, gate_up=max(n, T) * 2 * I * 2, rows=n * H * 4, own=T * H * 4,
                     out=T * H * 4, loss=4, counts=E * 4,
                     plan_ws=int(dev.lib.vlb_ep_workspace_bytes(T, k, E)), balance_ws=balance_workspace_bytes(T, E),
                     ws=max(int8_workspace_bytes(n, max(H, I)), int8_workspace_bytes(T, max(H, I))))
        self._b = {name: self._keep(dev.buffer(max(16, size), f"int8-{name}")) for name, size in sizes.items()}
        self.last_loss, self.last_counts = 0.0, np.zeros(E, np.uint32)

    def _keep(self, buf):
        self._bufs.append(buf)
        return buf

    @staticmethod
    def _shape(m: Expert):
        return (m.rows, m.cols) if isinstance(m, Matrix) else m.shape

    def _fill(self, gate_up: Int8Experts, down: Int8Experts, group: int, w1: Expert, w3: Expert, w2: Expert) -> None:
        gate_up.fill(group, 0, w1)
        gate_up.fill(group, self.I, w3)
        down.fill(group, 0, w2)

    def _products(self, gate_up: Int8Experts, down: Int8Experts, limit: float, rows: int, out, T: int,
                  row_index: int = 0, row_weight: int = 0, offsets: int = 0) -> None:
        """gate/up of `rows` rows of x, SwiGLU, down into `out` (f32)."""
        b, dev = self._b, self.dev
        dev.int8_linear_device(gate_up.weights, b["x"].address, rows, b["gate_up"].address, y_type=DTYPE_BF16, x_rows=T,
                               row_index_ptr=row_index, offsets_ptr=offsets, ws_ptr=b["ws"].address,
                               ws_bytes=b["ws"].nbytes)
        dev.int8_linear_device(down.weights, b["gate_up"].address, rows, out.address, x_type=DTYPE_BF16,
                               x_stride=2 * self.I, up_ptr=b["gate_up"].address + 2 * self.I,
                               swiglu_limit=limit, row_weight_ptr=row_weight, offsets_ptr=offsets,
                               ws_ptr=b["ws"].address, ws_bytes=b["ws"].nbytes)

    def forward(self, x: np.ndarray, logits: Optional[np.ndarray] = None) -> np.ndarray:
        """x f32 [T, H] -> f32 [T, H]. last_loss and last_counts hold the router's balance loss
        (coefficient 1) and the experts' loads of this batch."""
        dev, b, k, E, H = self.dev, self._b, self.top_k, self.E, self.H
        x = np.ascontiguousarray(x, dtype=np.float32)
        T = x.shape[0]
        if x.shape != (T, H) or not 0 < T <= self.max_tokens:
            raise ValueError(f"x must be [1..{self.max_tokens}, {H}]")
        b["x"].upload(x)
        if logits is None:
            dev._check(dev.lib.vlb_router_logits_device(dev.h, b["x"].ptr, self._router.ptr, T, H, E, b["logits"].ptr, None))
        else:
            b["logits"].upload(np.ascontiguousarray(logits, dtype=np.float32).reshape(T, E))
        dev._check(dev.lib.vlb_route_device(dev.h, self.score, 0, b["logits"].ptr,
                                            self._bias.ptr if self._bias else None, None, None, 0, T, E, k,
                                            C.c_float(self.route_scale), b["idx"].ptr, b["weights"].ptr, None))
        dev.balance_loss_device(b["logits"].address, b["idx"].address, T, E, k, counts_ptr=b["counts"].address,
                                ws_ptr=b["balance_ws"].address, ws_bytes=b["balance_ws"].nbytes, score=self.score,
                                loss_ptr=b["loss"].address)
        dev.route_plan_device(b["idx"].address, b["weights"].address, T, k, E, b["plan_ws"].address,
                              b["row_index"].address, b["row_weight"].address, b["elem_row"].address,
                              b["offsets"].address)
        self._products(self.gate_up, self.down, self.swiglu_limit, T * k, b["rows"], T, b["row_index"].address,
                       b["row_weight"].address, b["offsets"].address)
        if self.shared:
            self._products(*self.shared, self.shared_swiglu_limit, T, b["own"], T)
        dev._check(dev.lib.vlb_ep_combine_device(dev.h, b["rows"].ptr, b["elem_row"].ptr, T, k,
                                                 b["own"].ptr if self.shared else None, H, b["out"].ptr, None))
        dev.int8_status()
        self.last_loss = float(b["loss"].download(np.float32, 1)[0])
        self.last_counts = b["counts"].download(np.uint32, E)
        return b["out"].download(np.float32, T * H).reshape(T, H)

    def close(self) -> None:
        for buf in self._bufs:
            buf.free()
        self._bufs = []
