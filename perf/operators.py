"""The int8 products and the router's balance loss, as a user's program calls them, and their plain forms.

Three operators, chosen by a case's "op":

  linear   y = x W^T on 8-bit integers: rows of x rounded to int8 with one scale each (or given as int8), int8
           weights with one scale a channel.
  experts  the same product grouped over the experts of a MoE layer: row r belongs to the expert whose range of
           `offsets` holds it and takes token `row_index[r]`'s activations (gate/up entry), or SwiGLU of its own
           gate and up values (down entry, "swiglu").
  balance  the router's load-balance loss, the per-expert counts and the gradient of the logits.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def listed():
    return [
        # one token through the gate/up matrix of a small expert: latency
        {"name": "linear_token", "op": "linear", "M": 1, "K": 2048, "N": 2048, "x": "bf16", "y": "bf16"},
        # a decode batch through a shared expert's gate/up matrix
        {"name": "linear_batch", "op": "linear", "M": 64, "K": 4096, "N": 4096, "x": "bf16", "y": "bf16"},
        # a ragged batch, odd sizes in every dimension, in 32 bits
        {"name": "linear_odd", "op": "linear", "M": 77, "K": 1001, "N": 1411, "x": "f32", "y": "f32"},
        # a prefill through a dense projection
        {"name": "linear_prefill", "op": "linear", "M": 4096, "K": 4096, "N": 4096, "x": "f16", "y": "f16"},
        # rows that an earlier step left in int8 with their scales: the product alone
        {"name": "linear_int8_rows", "op": "linear", "M": 8192, "K": 2048, "N": 4096, "x": "i8", "y": "f32"},
        # one token's eight experts out of 64
        {"name": "experts_token", "op": "experts", "T": 1, "k": 8, "E": 64, "K": 2048, "N": 2048, "x": "bf16", "y": "bf16",
         "skew": 0.0, "swiglu": False},
        # a decode batch over 256 experts: two rows an expert, the weights are what is read
        {"name": "experts_decode", "op": "experts", "T": 64, "k": 8, "E": 256, "K": 4096, "N": 4096, "x": "f32", "y": "f32",
         "skew": 0.0, "swiglu": False},
        # a prefill through 64 experts' gate/up matrices
        {"name": "experts_prefill", "op": "experts", "T": 4096, "k": 8, "E": 64, "K": 2048, "N": 2048, "x": "bf16",
         "y": "bf16", "skew": 0.0, "swiglu": False},
        # the down products of a prefill whose routes are skewed, some experts with no row
        {"name": "experts_down_skewed", "op": "experts", "T": 2048, "k": 8, "E": 64, "K": 1024, "N": 2048, "x": "bf16",
         "y": "bf16", "skew": 1.1, "swiglu": True},
        # a router's smallest training call
        {"name": "balance_small", "op": "balance", "T": 16, "E": 64, "k": 8, "score": "softmax", "x": "f32", "S": 1,
         "masked": 0.0},
        # packed sequences with padding, the balance kept within each sequence
        {"name": "balance_sequences", "op": "balance", "T": 8192, "E": 256, "k": 8, "score": "sqrt_softplus", "x": "bf16",
         "S": 13, "masked": 0.1},
        # a large batch as one
        {"name": "balance_large", "op": "balance", "T": 65536, "E": 256, "k": 8, "score": "sigmoid", "x": "f32", "S": 1,
         "masked": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "experts", "experts", "balance"))
    if op == "balance":
        E, k = _log(rng, 8, 512), rng.randint(1, 8)
        T = _log(rng, 1, min(65536, 65536 * 256 // E))
        return {"op": op, "T": T, "E": E, "k": k, "score": rng.choice(("softmax", "sigmoid", "sqrt_softplus")),
                "x": rng.choice(("f32", "f16", "bf16")), "S": _log(rng, 1, min(64, T)), "masked": rng.choice((0.0, 0.2))}
    K, N = _log(rng, 64, 4096), _log(rng, 64, 4096)
    if op == "linear":
        M = _log(rng, 1, min(16384, (1 << 36) // (K * N)))
        return {"op": op, "M": M, "K": K, "N": N, "x": rng.choice(("f32", "f16", "bf16", "i8")),
                "y": rng.choice(("f32", "f16", "bf16"))}
    E = _log(rng, 4, min(256, (1 << 31) // (K * N)))
    k = rng.randint(1, min(8, E))
    T = _log(rng, 1, min(4096, (1 << 36) // (K * N * k)))
    swiglu = rng.random() < 0.4
    x = rng.choice(("f16", "bf16") if swiglu else ("f32", "f16", "bf16"))
    return {"op": op, "T": T, "k": k, "E": E, "K": K, "N": N, "x": x, "y": x if swiglu else rng.choice(("f32", "f16", "bf16")),
            "skew": rng.choice((0.0, 1.1)), "swiglu": swiglu}


def _stride(K):
    """Weight rows start on 16-byte boundaries, as the entry points' documentation asks for the fast path."""
    return (K + 15) // 16 * 16


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream's own handle


def _routes(T, k, E, skew, g):
    """Top-k routes of random logits, experts' popularity ~ rank^-skew: pairs sorted by expert, then token."""
    logits = torch.randn(T, E, device="cuda", generator=g)
    if skew:
        rank = torch.randperm(E, device="cuda", generator=g) + 1.0
        logits = logits - 2.0 * skew * torch.log(rank)
    idx = torch.topk(logits, k, dim=1).indices
    order = torch.argsort(idx.reshape(-1), stable=True)
    counts = torch.bincount(idx.reshape(-1), minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0)
    return (order // k).to(torch.int32), offsets.to(torch.int32), int(counts.max())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    st = {"case": case, "stream": _stream()}
    if case["op"] == "balance":
        T, E, k, S = case["T"], case["E"], case["k"], case["S"]
        z = 2.0 * torch.randn(T, E, device="cuda", generator=g) - 0.5
        st["idx"] = torch.topk(z, min(k, E), dim=1).indices.to(torch.int32).contiguous()
        st["logits"] = z.to(TYPES[case["x"]])
        st["mask"] = (torch.rand(T, device="cuda", generator=g) >= case["masked"]) if case["masked"] else None
        cuts = torch.sort(torch.randint(0, T + 1, (S - 1,), device="cuda", generator=g)).values if S > 1 else None
        st["offsets"] = None
        if S > 1:  # cuts that fall together leave a sequence without a token
            st["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), T)]).to(torch.int32)
        st["coef"] = 0.01
        st["upstream"] = torch.rand(1, device="cuda", generator=g) + 0.5
        st["loss"] = torch.zeros(1, device="cuda")
        st["counts"] = torch.zeros(S, E, dtype=torch.int32, device="cuda")
        st["grad"] = torch.zeros_like(st["logits"])
        return st
    K, N = case["K"], case["N"]
    E = case.get("E", 1)
    ld = _stride(K)
    st["w"] = torch.randint(-127, 128, (E, N, ld), device="cuda", generator=g, dtype=torch.int8)
    st["w_scale"] = torch.randn(E, N, device="cuda", generator=g).abs() * 0.002
    if case["op"] == "linear":
        rows = case["M"]
        if case["x"] == "i8":
            st["x"] = torch.randint(-127, 128, (rows, ld), device="cuda", generator=g, dtype=torch.int8)
            st["x_scale"] = torch.rand(rows, device="cuda", generator=g) * 0.03 + 0.01
        else:
            st["x"] = torch.randn(rows, K, device="cuda", generator=g).to(TYPES[case["x"]])
    else:
        rows = case["T"] * case["k"]
        st["row_index"], st["offsets"], st["cap"] = _routes(case["T"], case["k"], E, case["skew"], g)
        if case["swiglu"]:  # gate and up side by side, as the product before leaves them
            st["x"] = (2.0 * torch.randn(rows, 2 * K, device="cuda", generator=g)).to(TYPES[case["x"]])
            st["row_weight"] = torch.rand(rows, device="cuda", generator=g)
        else:
            st["x"] = torch.randn(case["T"], K, device="cuda", generator=g).to(TYPES[case["x"]])
    st["rows"] = rows
    st["y"] = torch.zeros(rows, N, device="cuda", dtype=TYPES[case["y"]])
    return st


def run(state):
    return _own(state) if own else _plain(state)


# ---- the plain forms -------------------------------------------------------------------------------------


def _quantized(x):
    """Rows of 32-bit values as whole numbers in [-127, 127], and the rows' scales."""
    top = x.abs().amax(dim=1, keepdim=True)
    full = torch.full_like(top, 127.0)
    step = torch.where(top > 0, full / top, torch.zeros_like(top))
    return torch.round(x * step), top / full


def _plain(st):
    case = st["case"]
    if case["op"] == "balance":
        return _plain_balance(st)
    K = case["K"]
    w = st["w"][:, :, :K].float()
    if case["op"] == "linear":
        if case["x"] == "i8":
            q, s = st["x"][:, :K].float(), st["x_scale"][:, None]
        else:
            q, s = _quantized(st["x"].float())
        return (torch.matmul(q, w[0].t()) * s * st["w_scale"][0]).to(st["y"].dtype)
    rows, ends = st["rows"], st["offsets"].long()
    at = torch.arange(rows, device="cuda")
    expert = torch.bucketize(at, ends[1:], right=True)
    slot = at - ends[expert]
    if case["swiglu"]:
        gate, up = st["x"][:, :K].float(), st["x"][:, K:].float()
        q, s = _quantized(gate / (1.0 + torch.exp(-gate)) * up)
        s = s * st["row_weight"][:, None]
    else:
        q, s = _quantized(st["x"].float()[st["row_index"].long()])
    padded = q.new_zeros(w.shape[0], st["cap"], K)  # every expert's rows, filled up to the longest
    padded[expert, slot] = q
    y = torch.bmm(padded, w.transpose(1, 2))[expert, slot]
    return (y * s * st["w_scale"][expert]).to(st["y"].dtype)


def _plain_balance(st):
    case = st["case"]
    T, E, k, S = case["T"], case["E"], case["k"], case["S"]
    z = st["logits"].float()
    live = st["mask"] if st["mask"] is not None else torch.ones(T, dtype=torch.bool, device="cuda")
    if S > 1:
        seq = torch.bucketize(torch.arange(T, device="cuda"), st["offsets"][1:].long(), right=True)
    else:
        seq = torch.zeros(T, dtype=torch.int64, device="cuda")
    picks = (seq[:, None] * E + st["idx"].long()).reshape(-1)
    hits = live[:, None].expand(T, k).reshape(-1).to(torch.int32)
    counts = torch.zeros(S * E, dtype=torch.int32, device="cuda").scatter_add_(0, picks, hits).view(S, E)
    n = torch.zeros(S, device="cuda").index_add_(0, seq, live.float())
    share = torch.where(n > 0, 1.0 / torch.clamp(n, min=1.0), torch.zeros_like(n)) / torch.clamp((n > 0).sum().float(), min=1.0)
    f = counts.float() * (E / k) / torch.clamp(n, min=1.0)[:, None]
    if case["score"] == "softmax":
        u = torch.exp(z - z.amax(dim=1, keepdim=True))
        slope = torch.ones_like(z)
    elif case["score"] == "sigmoid":
        u = 1.0 / (1.0 + torch.exp(-z))
        slope = 1.0 - u
    else:
        soft = torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))
        u = torch.sqrt(soft)
        slope = 1.0 / (1.0 + torch.exp(-z)) / (2.0 * soft)
    p = u / u.sum(dim=1, keepdim=True)
    d = (p * f[seq]).sum(dim=1, keepdim=True)
    weight = st["coef"] * share[seq][:, None] * live[:, None]
    grad = st["upstream"] * weight * p * (f[seq] - d) * slope
    return {"loss": (weight * d).sum().view(1), "counts": counts, "grad": grad.to(st["logits"].dtype)}


# ---- the framework's operators ---------------------------------------------------------------------------

_handle = None


def _device():
    global _handle
    if _handle is None:
        import vastloom_b200 as vb

        _handle = vb.Device(0, install_codebooks=False)
    return _handle


def _own(st):
    case = st["case"]
    dev = _device()
    if "ws" not in st:
        _own_setup(st)
    if case["op"] == "balance":
        dev.balance_loss_device(st["logits"].data_ptr(), st["idx"].data_ptr(), case["T"], case["E"], case["k"],
                                logits_type=st["x_type"], score=st["score"], coefficient=st["coef"],
                                mask_ptr=st["mask_ptr"], seq_offsets_ptr=st["offsets_ptr"], n_seqs=case["S"],
                                upstream_ptr=st["upstream"].data_ptr(), loss_ptr=st["loss"].data_ptr(),
                                counts_ptr=st["counts"].data_ptr(), dlogits_ptr=st["grad"].data_ptr(),
                                ws_ptr=st["ws"].data_ptr(), ws_bytes=st["ws_bytes"], stream=st["stream"])
        return {"loss": st["loss"], "counts": st["counts"], "grad": st["grad"]}
    x = st["x"].data_ptr()
    if case["op"] == "linear":
        dev.int8_linear_device(st["weights"], x, st["rows"], st["y"].data_ptr(), x_type=st["x_type"], y_type=st["y_type"],
                               x_stride=st["x_stride"], x_scale_ptr=st["scale_ptr"], ws_ptr=st["ws"].data_ptr(),
                               ws_bytes=st["ws_bytes"], stream=st["stream"])
    elif case["swiglu"]:
        dev.int8_linear_device(st["weights"], x, st["rows"], st["y"].data_ptr(), x_type=st["x_type"], y_type=st["y_type"],
                               x_stride=st["x_stride"], up_ptr=x + case["K"] * SIZE[case["x"]],
                               row_weight_ptr=st["row_weight"].data_ptr(), offsets_ptr=st["offsets"].data_ptr(),
                               ws_ptr=st["ws"].data_ptr(), ws_bytes=st["ws_bytes"], stream=st["stream"])
    else:
        dev.int8_linear_device(st["weights"], x, st["rows"], st["y"].data_ptr(), x_type=st["x_type"], y_type=st["y_type"],
                               x_stride=st["x_stride"], x_rows=case["T"], row_index_ptr=st["row_index"].data_ptr(),
                               offsets_ptr=st["offsets"].data_ptr(), ws_ptr=st["ws"].data_ptr(),
                               ws_bytes=st["ws_bytes"], stream=st["stream"])
    return st["y"]


def _own_setup(st):
    """What a program keeps beside its inputs: the weights' description and the workspace."""
    import vastloom_b200 as vb

    case = st["case"]
    kinds = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16, "i8": vb.DTYPE_I8}
    st["x_type"] = kinds[case["x"]]
    if case["op"] == "balance":
        st["score"] = {"softmax": vb.SCORE_SOFTMAX, "sigmoid": vb.SCORE_SIGMOID,
                       "sqrt_softplus": vb.SCORE_SQRT_SOFTPLUS}[case["score"]]
        st["mask_ptr"] = st["mask"].data_ptr() if st["mask"] is not None else 0
        st["offsets_ptr"] = st["offsets"].data_ptr() if st["offsets"] is not None else 0
        st["ws_bytes"] = vb.balance_workspace_bytes(case["T"], case["E"], case["S"])
    else:
        st["y_type"] = kinds[case["y"]]
        st["x_stride"] = st["x"].stride(0)
        st["scale_ptr"] = st["x_scale"].data_ptr() if "x_scale" in st else 0
        st["weights"] = vb.Int8Weights(st["w"].data_ptr(), st["w_scale"].data_ptr(), case["N"], case["K"],
                                       groups=case.get("E", 1), stride=_stride(case["K"]))
        st["ws_bytes"] = vb.int8_workspace_bytes(st["rows"], case["K"])
    st["ws"] = torch.empty(max(1, st["ws_bytes"]), dtype=torch.uint8, device="cuda")


# ---- what a pass cannot do without -----------------------------------------------------------------------


def work(case):
    if case["op"] == "balance":
        T, E, k, S = case["T"], case["E"], case["k"], case["S"]
        nbytes = 2 * T * E * SIZE[case["x"]] + T * k * 4 + S * E * 4 + 8
        return {"bytes": nbytes + (T if case["masked"] else 0), "flops": 12 * T * E}
    K, N = case["K"], case["N"]
    if case["op"] == "linear":
        rows, used, read = case["M"], 1, case["M"] * K * SIZE[case["x"]] + (case["M"] * 4 if case["x"] == "i8" else 0)
    else:
        rows = case["T"] * case["k"]
        # experts with at least one row, were every token's choice even
        used = case["E"] * (1.0 - (1.0 - case["k"] / case["E"]) ** case["T"])
        read = rows * (2 * K * SIZE[case["x"]] + 4) if case["swiglu"] else case["T"] * K * SIZE[case["x"]] + 4 * rows
    return {"bytes": int(read + used * N * (K + 4) + rows * N * SIZE[case["y"]]), "flops": 2 * rows * N * K}


# ---- the definitions in 64 bits --------------------------------------------------------------------------


def _exact_rows(x):
    """The definition's whole numbers: one step size a row, the quotient and the product rounded to 32 bits."""
    top = x.double().abs().max(dim=1).values
    inv = (127.0 / torch.where(top > 0, top, torch.ones_like(top))).float().double() * (top > 0)
    return torch.round((x.double() * inv[:, None]).float().double()), top / 127.0


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "balance":
        return _exact_balance(st)
    K, rows = case["K"], st["rows"]
    out = torch.zeros(rows, case["N"], dtype=torch.float64, device="cuda")
    if case["op"] == "linear":
        if case["x"] == "i8":
            q, s = st["x"][:, :K].double(), st["x_scale"].double()
        else:
            q, s = _exact_rows(st["x"])
        return (q @ st["w"][0, :, :K].double().T) * s[:, None] * st["w_scale"][0].double()
    if case["swiglu"]:
        gate, up = st["x"][:, :K].double(), st["x"][:, K:].double()
        a = gate * torch.sigmoid(gate) * up
        top = a.abs().max(dim=1).values
        q, s = torch.round(a * (127.0 / torch.where(top > 0, top, torch.ones_like(top)))[:, None]), top / 127.0
        s = s * st["row_weight"].double()
    else:
        q, s = _exact_rows(st["x"])
        q, s = q[st["row_index"].long()], s[st["row_index"].long()]
    ends = st["offsets"].tolist()
    for e in range(case["E"]):
        lo, hi = ends[e], ends[e + 1]
        if hi > lo:
            out[lo:hi] = (q[lo:hi] @ st["w"][e, :, :K].double().T) * s[lo:hi, None] * st["w_scale"][e].double()
    return out


def _exact_balance(st):
    case = st["case"]
    T, E, k, S = case["T"], case["E"], case["k"], case["S"]
    z = st["logits"].double().cpu().numpy()
    idx = st["idx"].cpu().numpy()
    live = st["mask"].cpu().numpy() if st["mask"] is not None else np.ones(T, bool)
    cuts = st["offsets"].cpu().numpy() if st["offsets"] is not None else np.array([0, T])
    if case["score"] == "softmax":
        u, slope = np.exp(z - z.max(1, keepdims=True)), np.ones_like(z)
    elif case["score"] == "sigmoid":
        u = 1.0 / (1.0 + np.exp(-z))
        slope = 1.0 / (1.0 + np.exp(z))
    else:
        soft = np.logaddexp(0.0, z)
        u, slope = np.sqrt(soft), 0.5 / (1.0 + np.exp(-z)) / soft
    p = u / u.sum(1, keepdims=True)
    tokens = [np.flatnonzero(live[cuts[s]:cuts[s + 1]]) + cuts[s] for s in range(S)]
    alive = sum(1 for t in tokens if t.size)
    loss, grad, up = 0.0, np.zeros_like(z), float(st["upstream"].double().item())
    for t in tokens:
        if not t.size:
            continue
        f = np.bincount(idx[t].reshape(-1), minlength=E) * (E / (k * t.size))
        d = p[t] @ f
        loss += st["coef"] * d.sum() / (alive * t.size)
        grad[t] = up * st["coef"] / (alive * t.size) * p[t] * (f[None, :] - d[:, None]) * slope[t]
    return {"loss": np.array([loss]), "counts": None, "grad": grad}
