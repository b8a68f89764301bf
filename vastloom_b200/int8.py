"""A MoE layer whose experts are 8-bit integers with a scale a channel, from the router to the combine.

Any expert matrix becomes int8 here: a resident ggml matrix of every storage type (dequantized on the
device, then rounded row by row) or a float32 array. All types then run the same tensor-core products,
where the block formats Q4_K, Q5_K, Q6_K, IQ2_S and MXFP4 otherwise have CUDA-core kernels only; the
price is one byte a weight and the rounding of weights and activations to 8 bits.

    logits -> route -> balance loss and per-expert counts -> plan (pairs by expert)
           -> gate/up product of the pairs' tokens -> SwiGLU and down product -> combine (+ shared)

With an input norm the layer is a residual block, out = x + MoE(RMSNorm(x)), whose rows are 8-bit integers from the norm
on: they are sorted by expert as such, the gate/up products take their SwiGLU in the epilogue, and the residual is added
with the shared expert's down product (or by the combine):

    norm (rows, int8 rows) -> logits -> route -> balance loss and counts -> int8 rows by expert
           -> gate/up product and SwiGLU -> down product -> combine on x (+ shared)

The layer math is the reference's (moe_forward, deepseek_v4_graph.cpp:1902-2274); the route weight
multiplies a pair's down row. Every step is a call of the public C ABI on device buffers.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Union

import numpy as np

from . import (ACT_NONE, ACT_SWIGLU, DTYPE_BF16, DTYPE_I8, SCORE_SQRT_SOFTPLUS, Device, Int8Weights, Matrix,
               balance_workspace_bytes, int8_workspace_bytes, sort_tokens_workspace_bytes)

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
        self._fill(group, row0, [source], None)

    def fill_pairs(self, group: int, gate: Expert, up: Expert) -> None:
        """Rounds two [rows / 2, cols] matrices into a group, row by row in turn: the channel pairs of ACT_SWIGLU."""
        n = self.rows // 2
        order = np.arange(2 * n, dtype=np.uint32).reshape(2, n).T
        self._fill(group, 0, [gate, up], np.ascontiguousarray(order))

    def _fill(self, group: int, row0: int, sources: Sequence[Expert], order: Optional[np.ndarray]) -> None:
        dev = self.dev
        sources = [s if isinstance(s, Matrix) else np.ascontiguousarray(s, dtype=np.float32) for s in sources]
        shapes = [(s.rows, s.cols) if isinstance(s, Matrix) else s.shape for s in sources]
        if any(len(shape) != 2 for shape in shapes):
            raise ValueError(f"a source must be a matrix, not of shape {next(s for s in shapes if len(s) != 2)}")
        n, cols = sum(shape[0] for shape in shapes), shapes[0][1]
        if (any(shape[1] != self.cols for shape in shapes) or not 0 <= row0 <= self.rows - n or
                not 0 <= group < self.weights.groups or (order is not None and (order.size != n or len(set(shapes)) > 1))):
            raise ValueError(f"a [{n}, {cols}] matrix does not fit rows {row0}.. of [{self.rows}, {self.cols}]")
        bufs = [dev.buffer(n * cols * 4, "int8-source")]
        try:
            at = 0
            for source, shape in zip(sources, shapes):
                part = C.c_void_p(bufs[0].address + at * cols * 4)
                if isinstance(source, Matrix):
                    dev._check(dev.lib.vlb_dequantize_device(dev.h, source.ptr, part, None))
                else:
                    dev._check(dev.lib.vlb_memcpy_h2d(dev.h, part, C.c_void_p(source.ctypes.data), source.nbytes))
                at += shape[0]
            if order is not None:
                bufs.append(dev.to_device(order))
            to = group * self.rows + row0
            dev.int8_quantize_device(bufs[0].address, n, cols, self._q.address + to * self.stride,
                                     self._s.address + to * 4, q_stride=self.stride,
                                     row_index_ptr=bufs[1].address if order is not None else 0)
            dev.synchronize()
        finally:
            for buf in bufs:
                buf.free()

    def free(self) -> None:
        self._q.free()
        self._s.free()


class Int8MoeLayer:
    """One MoE layer on int8 experts: w1, w3 ([I, H]) and w2 ([H, I]) of every expert, optionally a
    shared expert's three. swiglu_limit clamps the routed experts' SwiGLU, shared_swiglu_limit the
    shared one's (None: as the routed ones; 0: no clamp), as the two limits of MoeLayer. The gate and
    up values between the two products are held in bf16 (half of f32's bytes through HBM; their
    rounding, 2^-9, is below that of the 8-bit rows made of them). Every forward also takes the
    balance loss and the counts. input_norm (weight f32 [H], eps): a residual block, out = x + MoE(RMSNorm(x)); the
    SwiGLU's values are then what is held in bf16."""

    def __init__(self, dev: Device, *, router: np.ndarray, w1: Sequence[Expert], w3: Sequence[Expert],
                 w2: Sequence[Expert], top_k: int, score: int = SCORE_SQRT_SOFTPLUS, bias: Optional[np.ndarray] = None,
                 route_scale: float = 1.0, swiglu_limit: float = 0.0,
                 shared: Optional[tuple[Expert, Expert, Expert]] = None, max_tokens: int = 64,
                 shared_swiglu_limit: Optional[float] = None, input_norm: Optional[tuple[np.ndarray, float]] = None):
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
        self._norm = None
        if input_norm is not None:
            weight = np.ascontiguousarray(input_norm[0], dtype=np.float32)
            if weight.shape != (self.H,):
                raise ValueError("the norm weight must have one value for each column of x")
            self._norm = (weight, float(input_norm[1]))
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
        if self._norm:
            ld = self.gate_up.stride
            self._norm_weight = self._keep(dev.to_device(self._norm[0]))
            sizes |= dict(normed=T * H * 4, q=T * ld, q_scale=T * 4, q_rows=n * ld, row_scale=n * 4, gate_up=max(n, T) * I * 2,
                          plan_ws=sort_tokens_workspace_bytes(T, k, E))
        self._b = {name: self._keep(dev.buffer(max(16, size), f"int8-{name}")) for name, size in sizes.items()}
        self.last_loss, self.last_counts = 0.0, np.zeros(E, np.uint32)

    def _keep(self, buf):
        self._bufs.append(buf)
        return buf

    @staticmethod
    def _shape(m: Expert):
        return (m.rows, m.cols) if isinstance(m, Matrix) else m.shape

    def _fill(self, gate_up: Int8Experts, down: Int8Experts, group: int, w1: Expert, w3: Expert, w2: Expert) -> None:
        if self._norm:
            gate_up.fill_pairs(group, w1, w3)
        else:
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

    def _block_products(self, gate_up: Int8Experts, down: Int8Experts, limit: float, q, scale, rows: int, out,
                        row_weight: int = 0, offsets: int = 0, residual: int = 0) -> None:
        """gate/up of int8 rows with SwiGLU in the epilogue, down into `out` (f32) on a residual."""
        b, dev = self._b, self.dev
        dev.int8_linear_act_device(gate_up.weights, q.address, rows, b["gate_up"].address, act=ACT_SWIGLU, act_limit=limit,
                                   x_type=DTYPE_I8, y_type=DTYPE_BF16, x_stride=gate_up.stride, x_scale_ptr=scale.address,
                                   offsets_ptr=offsets)
        dev.int8_linear_act_device(down.weights, b["gate_up"].address, rows, out.address, act=ACT_NONE, x_type=DTYPE_BF16,
                                   row_weight_ptr=row_weight, offsets_ptr=offsets, residual_ptr=residual,
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
        rows = b["x"]  # what the router reads
        if self._norm:
            rows = b["normed"]
            dev.add_rms_norm_device(b["x"].address, T, H, weight_ptr=self._norm_weight.address, eps=self._norm[1],
                                    y_ptr=rows.address, q_ptr=b["q"].address, q_stride=self.gate_up.stride,
                                    q_scale_ptr=b["q_scale"].address)
        if logits is None:
            dev._check(dev.lib.vlb_router_logits_device(dev.h, rows.ptr, self._router.ptr, T, H, E, b["logits"].ptr, None))
        else:
            b["logits"].upload(np.ascontiguousarray(logits, dtype=np.float32).reshape(T, E))
        dev._check(dev.lib.vlb_route_device(dev.h, self.score, 0, b["logits"].ptr,
                                            self._bias.ptr if self._bias else None, None, None, 0, T, E, k,
                                            C.c_float(self.route_scale), b["idx"].ptr, b["weights"].ptr, None))
        dev.balance_loss_device(b["logits"].address, b["idx"].address, T, E, k, counts_ptr=b["counts"].address,
                                ws_ptr=b["balance_ws"].address, ws_bytes=b["balance_ws"].nbytes, score=self.score,
                                loss_ptr=b["loss"].address)
        if self._norm:
            return self._block(T)
        dev.route_plan_device(b["idx"].address, b["weights"].address, T, k, E, b["plan_ws"].address,
                              b["row_index"].address, b["row_weight"].address, b["elem_row"].address,
                              b["offsets"].address)
        self._products(self.gate_up, self.down, self.swiglu_limit, T * k, b["rows"], T, b["row_index"].address,
                       b["row_weight"].address, b["offsets"].address)
        if self.shared:
            self._products(*self.shared, self.shared_swiglu_limit, T, b["own"], T)
        dev._check(dev.lib.vlb_ep_combine_device(dev.h, b["rows"].ptr, b["elem_row"].ptr, T, k,
                                                 b["own"].ptr if self.shared else None, H, b["out"].ptr, None))
        return self._result(T)

    def _block(self, T: int) -> np.ndarray:
        dev, b, k, H = self.dev, self._b, self.top_k, self.H
        dev.sort_tokens_device(b["idx"].address, T, k, self.E, x_ptr=b["q"].address, H=self.gate_up.stride, x_type=DTYPE_I8,
                               x_scale_ptr=b["q_scale"].address, weights_ptr=b["weights"].address,
                               rows_ptr=b["q_rows"].address, row_scale_ptr=b["row_scale"].address,
                               row_weight_ptr=b["row_weight"].address, elem_row_ptr=b["elem_row"].address,
                               offsets_ptr=b["offsets"].address, ws_ptr=b["plan_ws"].address, ws_bytes=b["plan_ws"].nbytes)
        self._block_products(self.gate_up, self.down, self.swiglu_limit, b["q_rows"], b["row_scale"], T * k, b["rows"],
                             row_weight=b["row_weight"].address, offsets=b["offsets"].address)
        residual = b["x"]
        if self.shared:
            self._block_products(*self.shared, self.shared_swiglu_limit, b["q"], b["q_scale"], T, b["own"],
                                 residual=residual.address)
            residual = b["own"]
        dev.combine_device(b["rows"].address, b["elem_row"].address, T, k, H, b["out"].address, residual_ptr=residual.address)
        return self._result(T)

    def _result(self, T: int) -> np.ndarray:
        dev, b, E, H = self.dev, self._b, self.E, self.H
        dev.int8_status()
        self.last_loss = float(b["loss"].download(np.float32, 1)[0])
        self.last_counts = b["counts"].download(np.uint32, E)
        return b["out"].download(np.float32, T * H).reshape(T, H)

    def close(self) -> None:
        for buf in self._bufs:
            buf.free()
        self._bufs = []
