"""The operators around the experts of an int8 MoE block, as a user's program calls them, and their plain forms.

Chosen by a case's "op":

  norm       h = x + residual and its RMS norm with a weight a column.
  norm_grad  the gradient of both: of the sum, and of the weight.
  sort       the (token, slot) pairs of a route in the experts' order, each pair's row, weight and token, and where each
             expert starts. Pairs of masked tokens and of ids past the experts are dropped.
  combine    the experts' rows back to their tokens: a weighted sum over a token's slots, on top of a residual.
  combine_grad  the gradient of that: of the rows, and of the weights.
  linear     y = row_weight * act(x W^T + bias) + residual on 8-bit integers, act also SwiGLU of channel pairs.
  entry      a block's entry as it runs: norm to int8 rows with scales, rows sorted by expert, the experts' gate/up
             products with their SwiGLU.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
EPS = 1e-6


def listed():
    return [
        # one token between attention and experts, the stream kept in f32: latency
        {"name": "norm_token", "op": "norm", "rows": 1, "H": 4096, "x": "bf16", "r": "f32"},
        # a long prompt's rows
        {"name": "norm_prefill", "op": "norm", "rows": 16384, "H": 4096, "x": "bf16", "r": "bf16"},
        # a ragged batch of odd rows in 32 bits
        {"name": "norm_grad_odd", "op": "norm_grad", "rows": 333, "H": 1411, "x": "f32", "r": "f32"},
        # a training batch
        {"name": "norm_grad_batch", "op": "norm_grad", "rows": 8192, "H": 4096, "x": "bf16", "r": "bf16"},
        # a decode batch over 256 experts
        {"name": "sort_decode", "op": "sort", "T": 64, "k": 8, "E": 256, "H": 4096, "x": "bf16", "dropped": 0.0, "skew": 0.0},
        # packed prompts with padding, routes skewed
        {"name": "sort_prefill", "op": "sort", "T": 16384, "k": 8, "E": 64, "H": 2048, "x": "bf16", "dropped": 0.1,
         "skew": 1.1},
        # a decode batch's rows back to their tokens
        {"name": "combine_decode", "op": "combine", "T": 64, "k": 8, "E": 256, "H": 4096, "x": "f32", "y": "f32",
         "dropped": 0.0, "skew": 0.0},
        # a prompt's, onto the stream
        {"name": "combine_prefill", "op": "combine", "T": 16384, "k": 8, "E": 64, "H": 2048, "x": "bf16", "y": "f32",
         "dropped": 0.1, "skew": 1.1},
        # a training batch
        {"name": "combine_grad_batch", "op": "combine_grad", "T": 8192, "k": 8, "E": 64, "H": 2048, "x": "bf16", "y": "bf16",
         "dropped": 0.1, "skew": 0.0},
        # one token through a shared expert's gate/up matrix
        {"name": "linear_token", "op": "linear", "M": 1, "K": 4096, "N": 4096, "x": "bf16", "y": "bf16", "act": "swiglu",
         "bias": False, "residual": False},
        # a prompt through a dense projection with everything on
        {"name": "linear_prefill", "op": "linear", "M": 4096, "K": 4096, "N": 4096, "x": "f16", "y": "f16", "act": "gelu",
         "bias": True, "residual": True},
        # a prompt's entry into 64 experts
        {"name": "entry_prefill", "op": "entry", "T": 4096, "k": 8, "E": 64, "K": 2048, "N": 2048, "x": "bf16", "r": "f32",
         "y": "bf16", "dropped": 0.0, "skew": 0.0},
    ]


ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "swiglu")


def _log(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "sort", "combine", "combine_grad", "linear", "entry"))
    x = rng.choice(("f32", "f16", "bf16"))
    if op in ("norm", "norm_grad"):
        H = _log(rng, 64, 16384)
        return {"op": op, "rows": _log(rng, 1, (1 << 25) // H), "H": H, "x": x, "r": rng.choice((x, "f32"))}
    if op == "linear":
        K, act = _log(rng, 64, 4096), rng.choice(ACTS)
        N = 2 * _log(rng, 32, 2048) if act == "swiglu" else _log(rng, 64, 4096)
        return {"op": op, "M": _log(rng, 1, min(8192, (1 << 35) // (K * N))), "K": K, "N": N, "x": x,
                "y": rng.choice(("f32", "f16", "bf16")), "act": act, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5}
    E = _log(rng, 4, 256)
    k = rng.randint(1, min(8, E))
    more = {"dropped": rng.choice((0.0, 0.15)), "skew": rng.choice((0.0, 1.1))}
    if op == "entry":
        K = _log(rng, 64, 4096)
        E = min(E, (1 << 28) // (K * 4096) + 4)
        k = min(k, E)
        N = 2 * _log(rng, 32, 2048)
        T = _log(rng, 1, min(4096, (1 << 35) // (K * N * k)))
        return {"op": op, "T": T, "k": k, "E": E, "K": K, "N": N, "x": x, "r": rng.choice((x, "f32")),
                "y": rng.choice(("f16", "bf16")), **more}
    H = _log(rng, 64, 8192)
    T = _log(rng, 1, min(32768, (1 << 26) // (H * k)))
    case = {"op": op, "T": T, "k": k, "E": E, "H": H, "x": x, **more}
    if op == "sort":
        case["x"] = rng.choice(("f32", "f16", "bf16", "i8"))
    else:
        case["y"] = rng.choice((x, "f32"))
    return case


# ---- inputs ------------------------------------------------------------------------------------------------


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream's own handle


def _stride(K):
    """Int8 rows start on 16-byte boundaries, as the entry points' documentation asks for the fast path."""
    return (K + 15) // 16 * 16


def _route(case, g, st):
    """Top-k routes of random logits, experts' popularity ~ rank^-skew; a share of the tokens is masked, and as many
    pairs carry an id past the experts (they were dropped)."""
    T, k, E = case["T"], case["k"], case["E"]
    z = torch.randn(T, E, device="cuda", generator=g)
    if case["skew"]:
        z = z - 2.0 * case["skew"] * torch.log(torch.randperm(E, device="cuda", generator=g) + 1.0)
    top = torch.topk(z, k, dim=1)
    st["weights"] = torch.softmax(top.values, dim=1).contiguous()
    idx = top.indices.to(torch.int32)
    st["mask"] = None
    if case["dropped"]:
        st["mask"] = torch.rand(T, device="cuda", generator=g) >= case["dropped"]
        gone = torch.rand(T, k, device="cuda", generator=g) < case["dropped"]
        idx = torch.where(gone, torch.full_like(idx, E), idx)
    st["idx"] = idx.contiguous()


def _places(case, idx, mask):
    """Each pair's row in the experts' order (-1: dropped), each expert's start, and the tokens of the rows."""
    T, k, E = case["T"], case["k"], case["E"]
    live = idx < E
    if mask is not None:
        live = live & mask[:, None]
    key = torch.where(live, idx, torch.full_like(idx, E)).reshape(-1).long()
    order = torch.argsort(key, stable=True)
    row = torch.empty_like(order)
    row[order] = torch.arange(T * k, device="cuda")
    starts = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    starts[1:] = torch.cumsum(torch.zeros(E + 1, dtype=torch.int64, device="cuda").scatter_add_(
        0, key, torch.ones_like(key))[:E], 0)
    elem_row = torch.where(live.reshape(-1), row, torch.full_like(row, -1)).to(torch.int32).view(T, k)
    return elem_row, starts.to(torch.int32), order


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, kind="f32"):
        return torch.randn(*shape, device="cuda", generator=g).to(TYPES[kind])

    def zeros(*shape, kind="f32"):
        return torch.zeros(*shape, device="cuda", dtype=TYPES[kind])

    op = case["op"]
    st = {"case": case, "stream": _stream()}
    if op in ("norm", "norm_grad"):
        rows, H = case["rows"], case["H"]
        st["w"] = 1.0 + 0.2 * randn(H)
        if op == "norm":
            st["x"], st["r"] = randn(rows, H, kind=case["x"]), (4.0 * randn(rows, H)).to(TYPES[case["r"]])
            st["h"], st["y"] = zeros(rows, H, kind=case["r"]), zeros(rows, H, kind=case["x"])
        else:
            st["dy"], st["dh"] = randn(rows, H, kind=case["x"]), randn(rows, H, kind=case["r"])
            st["h"] = (4.0 * randn(rows, H)).to(TYPES[case["r"]])
            st["dx"], st["dw"] = zeros(rows, H, kind=case["x"]), zeros(H)
            st["dr"] = zeros(rows, H, kind=case["r"]) if case["r"] != case["x"] else None
        return st
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        ny = N // 2 if case["act"] == "swiglu" else N
        st["x"] = randn(M, K, kind=case["x"])
        st["w"] = torch.randint(-127, 128, (1, N, _stride(K)), device="cuda", generator=g, dtype=torch.int8)
        st["ws"] = randn(1, N).abs() * (0.02 / math.sqrt(K))
        st["bias"] = randn(1, N) if case["bias"] else None
        st["residual"] = randn(M, ny, kind=case["y"]) if case["residual"] else None
        st["y"] = zeros(M, ny, kind=case["y"])
        return st
    T, k, E = case["T"], case["k"], case["E"]
    _route(case, g, st)
    if op == "entry":
        K, N = case["K"], case["N"]
        st["x"], st["r"] = randn(T, K, kind=case["x"]), (4.0 * randn(T, K)).to(TYPES[case["r"]])
        st["nw"] = 1.0 + 0.2 * randn(K)
        st["w"] = torch.randint(-127, 128, (E, N, _stride(K)), device="cuda", generator=g, dtype=torch.int8)
        st["ws"] = randn(E, N).abs() * (0.02 / math.sqrt(K))
        st["h"], st["y"] = zeros(T, K, kind=case["r"]), zeros(T * k, N // 2, kind=case["y"])
        st["offsets"] = zeros(E + 1).to(torch.int32)
        st["cap"] = int(torch.bincount(st["idx"].reshape(-1).long(), minlength=E + 1)[:E].max())
        return st
    H = case["H"]
    if op == "sort":
        if case["x"] == "i8":
            st["x"] = torch.randint(-127, 128, (T, H), device="cuda", generator=g, dtype=torch.int8)
            st["x_scale"] = torch.rand(T, device="cuda", generator=g) * 0.03 + 0.01
            st["row_scale"] = zeros(T * k)
        else:
            st["x"] = randn(T, H, kind=case["x"])
        st["rows"], st["row_weight"] = zeros(T * k, H, kind=case["x"]), zeros(T * k)
        for name, n in (("elem_row", (T, k)), ("row_index", (T * k,)), ("offsets", (E + 1,))):
            st[name] = zeros(*n).to(torch.int32)
        return st
    st["elem_row"], st["offsets"], _ = _places(case, st["idx"], st["mask"])
    st["rows"] = randn(T * k, H, kind=case["x"])
    if op == "combine":
        st["residual"] = (4.0 * randn(T, H)).to(TYPES[case["y"]])
        st["out"] = zeros(T, H, kind=case["y"])
    else:
        st["dout"] = randn(T, H, kind=case["y"])
        st["drows"], st["dweights"] = zeros(T * k, H, kind=case["x"]), zeros(T, k)
    return st


def run(state):
    return _own(state) if own else _plain(state)


# ---- the plain forms -------------------------------------------------------------------------------------


def _activate(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "swiglu":
        gate, up = z[:, 0::2], z[:, 1::2]
        return gate / (1.0 + torch.exp(-gate)) * up
    return z


def _quantized(x):
    """Rows of 32-bit values as whole numbers in [-127, 127], and the rows' scales."""
    top = x.abs().amax(dim=1, keepdim=True)
    full = torch.full_like(top, 127.0)
    step = torch.where(top > 0, full / top, torch.zeros_like(top))
    return torch.round(x * step), top / full


def _norm(st, w):
    h = st["x"].float() + st["r"].float()
    return h, h * (1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)) * w


def _plain(st):
    case = st["case"]
    op = case["op"]
    if op == "norm":
        h, y = _norm(st, st["w"])
        return {"h": h.to(st["h"].dtype), "y": y.to(st["y"].dtype)}
    if op == "norm_grad":
        h, dy = st["h"].float(), st["dy"].float()
        s = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        n, gy = h * s, dy * st["w"]
        d = s * (gy - n * (gy * n).mean(dim=1, keepdim=True)) + st["dh"].float()
        out = {"dx": d.to(st["dx"].dtype), "dw": (dy * n).sum(dim=0)}
        if st["dr"] is not None:
            out["dr"] = d.to(st["dr"].dtype)
        return out
    if op == "linear":
        q, s = _quantized(st["x"].float())
        z = torch.matmul(q, st["w"][0, :, : case["K"]].float().t()) * s * st["ws"][0]
        if st["bias"] is not None:
            z = z + st["bias"][0]
        y = _activate(z, case["act"])
        if st["residual"] is not None:
            y = y + st["residual"].float()
        return y.to(st["y"].dtype)
    T, k, E = case["T"], case["k"], case["E"]
    if op in ("sort", "entry"):
        elem_row, starts, order = _places(case, st["idx"], st["mask"])
        at = torch.arange(T * k, device="cuda")
        live = at < starts[E]
        token = order // k
    if op == "sort":
        out = {"elem_row": elem_row, "offsets": starts,
               "row_index": torch.where(live, token, torch.zeros_like(token)).to(torch.int32),
               "row_weight": torch.where(live, st["weights"].reshape(-1)[order], torch.zeros_like(st["row_weight"])),
               "rows": torch.where(live[:, None], st["x"][token], torch.zeros_like(st["rows"]))}
        if "x_scale" in st:
            out["row_scale"] = torch.where(live, st["x_scale"][token], torch.zeros_like(st["row_scale"]))
        return out
    if op == "entry":
        h, y = _norm(st, st["nw"])
        q, s = _quantized(y)
        expert = torch.bucketize(at, starts[1:].long(), right=True).clamp(max=E - 1)
        slot = torch.where(live, at - starts[expert], torch.full_like(at, st["cap"]))
        padded = q.new_zeros(E, st["cap"] + 1, case["K"])  # every expert's rows, the dropped ones behind them
        padded[expert, slot] = q[token]
        z = torch.bmm(padded, st["w"][:, :, : case["K"]].float().transpose(1, 2))[expert, slot]
        a = _activate(z * s[token] * st["ws"][expert], "swiglu").to(st["y"].dtype)
        return {"h": h.to(st["h"].dtype), "y": torch.where(live[:, None], a, torch.zeros_like(a)), "offsets": starts}
    gone = st["elem_row"] < 0
    rows = st["rows"].float()[st["elem_row"].clamp(min=0).long()]  # [T, k, H]
    weights = torch.where(gone, torch.zeros_like(st["weights"]), st["weights"])
    if op == "combine":
        return ((rows * weights[:, :, None]).sum(dim=1) + st["residual"].float()).to(st["out"].dtype)
    dout = st["dout"].float()
    dweights = (rows * dout[:, None, :]).sum(dim=2)
    drows = torch.zeros(T * k + 1, case["H"], device="cuda")
    drows[torch.where(gone, torch.full_like(st["elem_row"], T * k), st["elem_row"]).long()] = \
        dout[:, None, :] * weights[:, :, None]
    live = torch.arange(T * k, device="cuda") < st["offsets"][E]
    drows = torch.where(live[:, None], drows[: T * k], torch.zeros_like(rows.view(T * k, -1)))
    return {"drows": drows.to(st["drows"].dtype), "dweights": torch.where(gone, torch.zeros_like(dweights), dweights)}


# ---- the framework's operators ---------------------------------------------------------------------------

_handle = None


def _device():
    global _handle
    if _handle is None:
        import vastloom_b200 as vb

        _handle = vb.Device(0, install_codebooks=False)
    return _handle


def _own_setup(st):
    """What a program keeps beside its inputs: addresses, the weights' description and the workspace."""
    import vastloom_b200 as vb

    case = st["case"]
    op = case["op"]
    kinds = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16, "i8": vb.DTYPE_I8}
    for name in ("x", "r", "y"):
        if name in case:
            st[name + "_type"] = kinds[case[name]]
    nbytes = 0
    if op == "norm_grad":
        nbytes = vb.add_rms_norm_grad_workspace_bytes(case["rows"], case["H"])
    elif op == "linear":
        nbytes = vb.int8_workspace_bytes(case["M"], case["K"])
        st["act"] = getattr(vb, "ACT_" + case["act"].upper())
    elif op in ("sort", "entry"):
        nbytes = vb.sort_tokens_workspace_bytes(case["T"], case["k"], case["E"])
    if op in ("linear", "entry"):
        st["weights_i8"] = vb.Int8Weights(st["w"].data_ptr(), st["ws"].data_ptr(), case["N"], case["K"],
                                          groups=case.get("E", 1), stride=_stride(case["K"]))
    if op == "entry":
        n, ld = case["T"] * case["k"], _stride(case["K"])
        st["act"] = vb.ACT_SWIGLU
        st["q"] = torch.zeros(case["T"], ld, dtype=torch.int8, device="cuda")
        st["q_scale"] = torch.empty(case["T"], device="cuda")
        st["q_rows"] = torch.empty(n, ld, dtype=torch.int8, device="cuda")
        st["q_row_scale"] = torch.empty(n, device="cuda")
        st["elem_row"] = torch.empty(n, dtype=torch.int32, device="cuda")
    st["scratch"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    st["scratch_bytes"] = nbytes
    st["ptr"] = {name: v.data_ptr() for name, v in st.items() if isinstance(v, torch.Tensor)}


def _own(st):
    dev = _device()
    if "ptr" not in st:
        _own_setup(st)
    case, p, stream = st["case"], st["ptr"], st["stream"]
    op, ws = case["op"], {"ws_ptr": p["scratch"], "ws_bytes": st["scratch_bytes"]}
    if op == "norm":
        dev.add_rms_norm_device(p["x"], case["rows"], case["H"], x_type=st["x_type"], residual_type=st["r_type"],
                                residual_ptr=p["r"], weight_ptr=p["w"], eps=EPS, residual_out_ptr=p["h"], y_ptr=p["y"],
                                stream=stream)
        return {"h": st["h"], "y": st["y"]}
    if op == "norm_grad":
        dev.add_rms_norm_grad_device(p["dy"], p["h"], case["rows"], case["H"], x_type=st["x_type"],
                                     residual_type=st["r_type"], weight_ptr=p["w"], eps=EPS, dh_ptr=p["dh"],
                                     dx_ptr=p["dx"], dresidual_ptr=p.get("dr", 0), dweight_ptr=p["dw"], stream=stream,
                                     **ws)
        out = {"dx": st["dx"], "dw": st["dw"]}
        if st["dr"] is not None:
            out["dr"] = st["dr"]
        return out
    if op == "linear":
        dev.int8_linear_act_device(st["weights_i8"], p["x"], case["M"], p["y"], x_type=st["x_type"], y_type=st["y_type"],
                                   act=st["act"], bias_ptr=p.get("bias", 0), residual_ptr=p.get("residual", 0),
                                   stream=stream, **ws)
        return st["y"]
    T, k, E = case["T"], case["k"], case["E"]
    if op == "sort":
        dev.sort_tokens_device(p["idx"], T, k, E, x_ptr=p["x"], H=case["H"], x_type=st["x_type"],
                               x_scale_ptr=p.get("x_scale", 0), weights_ptr=p["weights"], mask_ptr=p.get("mask", 0),
                               rows_ptr=p["rows"], row_scale_ptr=p.get("row_scale", 0), row_index_ptr=p["row_index"],
                               row_weight_ptr=p["row_weight"], elem_row_ptr=p["elem_row"], offsets_ptr=p["offsets"],
                               stream=stream, **ws)
        names = ("elem_row", "offsets", "row_index", "row_weight", "rows", "row_scale")
        return {name: st[name] for name in names if name in st}
    if op == "entry":
        ld = _stride(case["K"])
        dev.add_rms_norm_device(p["x"], T, case["K"], x_type=st["x_type"], residual_type=st["r_type"],
                                residual_ptr=p["r"], weight_ptr=p["nw"], eps=EPS, residual_out_ptr=p["h"], q_ptr=p["q"],
                                q_stride=ld, q_scale_ptr=p["q_scale"], stream=stream)
        dev.sort_tokens_device(p["idx"], T, k, E, x_ptr=p["q"], H=ld, x_type=_I8, x_scale_ptr=p["q_scale"],
                               mask_ptr=p.get("mask", 0), rows_ptr=p["q_rows"], row_scale_ptr=p["q_row_scale"],
                               elem_row_ptr=p["elem_row"], offsets_ptr=p["offsets"], stream=stream, **ws)
        dev.int8_linear_act_device(st["weights_i8"], p["q_rows"], T * k, p["y"], x_type=_I8, y_type=st["y_type"],
                                   x_stride=ld, x_scale_ptr=p["q_row_scale"], offsets_ptr=p["offsets"], act=st["act"],
                                   stream=stream)
        return {"h": st["h"], "y": st["y"], "offsets": st["offsets"]}
    if op == "combine":
        dev.combine_device(p["rows"], p["elem_row"], T, k, case["H"], p["out"], x_type=st["x_type"], y_type=st["y_type"],
                           weights_ptr=p["weights"], residual_ptr=p["residual"], stream=stream)
        return st["out"]
    dev.combine_grad_device(p["dout"], p["elem_row"], T, k, case["H"], x_type=st["x_type"], y_type=st["y_type"],
                            rows_ptr=p["rows"], weights_ptr=p["weights"], drows_ptr=p["drows"],
                            dweights_ptr=p["dweights"], stream=stream)
    return {"drows": st["drows"], "dweights": st["dweights"]}


_I8 = 3  # the 8-bit integers' type code


# ---- what a pass cannot do without -----------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, x, r = case["rows"] * case["H"], SIZE[case["x"]], SIZE[case["r"]]
        if op == "norm":  # x, residual; h, y
            return {"bytes": 2 * n * (x + r) + 4 * case["H"], "flops": 6 * n}
        both = r if case["r"] != case["x"] else 0
        return {"bytes": n * (2 * x + 2 * r + both) + 8 * case["H"], "flops": 12 * n}  # dy, h, dh; dx, dr
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        ny = N // 2 if case["act"] == "swiglu" else N
        out = M * ny * SIZE[case["y"]] * (2 if case["residual"] else 1)
        return {"bytes": M * K * SIZE[case["x"]] + N * (K + 4 + (4 if case["bias"] else 0)) + out, "flops": 2 * M * N * K}
    T, k, E = case["T"], case["k"], case["E"]
    live = T * k * (1.0 - case["dropped"]) ** 2  # pairs
    if op == "entry":
        K, N = case["K"], case["N"]
        used = E * (1.0 - (1.0 - k / E) ** T)  # experts with a row, were every token's choice even
        nbytes = T * K * (SIZE[case["x"]] + 2 * SIZE[case["r"]]) + T * k * 4 + used * N * (K + 4)
        return {"bytes": int(nbytes + live * N // 2 * SIZE[case["y"]]), "flops": int(2 * live * N * K)}
    H, x = case["H"], SIZE[case["x"]]
    small = T * k * 8
    if op == "sort":
        return {"bytes": int(T * H * x + live * (H * x + 8) + small), "flops": 0}
    y = SIZE[case["y"]]
    if op == "combine":
        return {"bytes": int(live * H * x + 2 * T * H * y + small), "flops": int(2 * live * H)}
    return {"bytes": int(2 * live * H * x + T * H * y + small + 4 * T * k), "flops": int(3 * live * H)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------


def _exact_act(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":  # 1 + tanh(u) = 2 sigmoid(2 u)
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "swiglu":
        pairs = z.view(z.shape[0], -1, 2)
        return pairs[:, :, 0] * torch.sigmoid(pairs[:, :, 0]) * pairs[:, :, 1]
    return z


def _exact_norm(x, r, w):
    h = x.double() + r.double()
    return h, h / (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / h.shape[1] + EPS).sqrt() * w.double()


def _exact_rows(x):
    """Rows as whole numbers by the definition, one step size a row (in 32 bits, as the row's values are), and scales."""
    top = x.abs().max(dim=1).values.float()
    inv = torch.where(top > 0, 127.0 / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(top))
    return torch.round((x.float() * inv[:, None])).double(), top.double() / 127.0


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h, y = _exact_norm(st["x"], st["r"], st["w"])
        return {"h": h, "y": y}
    if op == "norm_grad":
        h, dy, w = st["h"].double(), st["dy"].double(), st["w"].double()
        ms = (h ** 2).sum(dim=1, keepdim=True) / case["H"] + EPS
        along = (dy * w * h).sum(dim=1, keepdim=True) / (case["H"] * ms)
        d = (dy * w - h * along) / ms.sqrt() + st["dh"].double()
        out = {"dx": d, "dw": (dy * h / ms.sqrt()).sum(dim=0)}
        if st["dr"] is not None:
            out["dr"] = d
        return out
    if op == "linear":
        K = case["K"]
        q, s = _exact_rows(st["x"].double())
        out = torch.empty(st["y"].shape, dtype=torch.float64, device="cuda")
        for r in range(0, case["M"], 1024):
            z = q[r : r + 1024] @ st["w"][0, :, :K].double().t() * s[r : r + 1024, None] * st["ws"][0].double()
            if st["bias"] is not None:
                z = z + st["bias"][0].double()
            out[r : r + 1024] = _exact_act(z, case["act"])
        return out if st["residual"] is None else out + st["residual"].double()
    T, k, E = case["T"], case["k"], case["E"]
    if op in ("sort", "entry"):
        ids = st["idx"].cpu().numpy().astype("int64")
        if st["mask"] is not None:
            ids[~st["mask"].cpu().numpy()] = E
        flat = ids.reshape(-1)
        order = flat.argsort(kind="stable")
        order = torch.from_numpy(order[flat[order] < E]).cuda()  # the live pairs
        n = order.numel()
    if op == "sort":
        rows, weight = torch.zeros(T * k, case["H"], dtype=torch.float64, device="cuda"), torch.zeros(T * k).double().cuda()
        rows[:n], weight[:n] = st["x"][order // k].double(), st["weights"].reshape(-1)[order].double()
        out = {"elem_row": None, "offsets": None, "row_index": None, "row_weight": weight,
               "rows": None if case["x"] == "i8" else rows}
        if "x_scale" in st:
            out["row_scale"] = torch.zeros_like(weight)
            out["row_scale"][:n] = st["x_scale"][order // k].double()
        return out
    if op == "entry":
        h, y = _exact_norm(st["x"], st["r"], st["nw"])
        q, s = _exact_rows(y)
        out = torch.zeros(T * k, case["N"] // 2, dtype=torch.float64, device="cuda")
        expert = st["idx"].reshape(-1)[order].long()
        at = torch.searchsorted(expert, torch.arange(E + 1, device="cuda")).tolist()
        for e in range(E):
            for lo in range(at[e], at[e + 1], 1024):
                hi = min(at[e + 1], lo + 1024)
                token = order[lo:hi] // k
                z = q[token] @ st["w"][e, :, : case["K"]].double().t() * s[token, None] * st["ws"][e].double()
                out[lo:hi] = _exact_act(z, "swiglu")
        return {"h": h, "y": out, "offsets": None}
    live = st["elem_row"] >= 0
    if op == "combine":
        out = st["residual"].double()
        for s in range(k):
            row = st["rows"][st["elem_row"][:, s].clamp(min=0).long()].double()
            out = out + torch.where(live[:, s, None], row * st["weights"][:, s, None].double(), torch.zeros_like(row))
        return out
    dout = st["dout"].double()
    drows, dweights = torch.zeros(st["drows"].shape).double().cuda(), torch.zeros(T, k).double().cuda()
    for s in range(k):
        on = live[:, s]
        row = st["elem_row"][on, s].long()
        drows[row] = dout[on] * st["weights"][on, s, None].double()
        dweights[on, s] = (dout[on] * st["rows"][row].double()).sum(dim=1)
    return {"drows": drows, "dweights": dweights}
