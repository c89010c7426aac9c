"""The measured cases of the training operators beside the MLP engine: layer norm
(forward, backward), the AdamW step over many tensors (states in 32 or in 8 bits),
quantising to 8-bit floats with a scale for each block of 128, and the matrix
product of such operands.

`own` chooses the side: False runs each operator's plain form (elementary torch
operations), True calls the framework. Sizes are those of the repository's
configurations (1024-4096-4096-4096-1024 at batch 8192, 16 layers of 512 at batch
2048, 8 layers of 8192, 1000-3000-777-10 at batch 4099), single tokens beside them.
"""
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is held as zeros
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8
LR, DECAY = 1e-3, 0.01

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def listed():
    return [
        # the norm in front of a layer while a model answers: a few tokens, latency is all
        {"name": "ln_fwd_16x1024", "op": "ln_fwd", "rows": 16, "cols": 1024, "pad": 0, "dtype": "bf16", "params": "f32"},
        # the same norm on the training batch of the 4096-wide network
        {"name": "ln_fwd_8192x4096", "op": "ln_fwd", "rows": 8192, "cols": 4096, "pad": 0, "dtype": "bf16", "params": "f32"},
        # its backward pass there, with the weight's and the bias's gradients
        {"name": "ln_bwd_8192x4096", "op": "ln_bwd", "rows": 8192, "cols": 4096, "pad": 0, "dtype": "bf16", "params": "f32"},
        # the backward pass behind the ragged network's 777-wide layer: odd rows, odd columns, fp32
        {"name": "ln_bwd_4099x777", "op": "ln_bwd", "rows": 4099, "cols": 777, "pad": 0, "dtype": "f32", "params": "f32"},
        # the optimizer step of the 4096-wide network: fp32 masters, gradients and states, bf16 copies
        {"name": "adamw_f32_4096", "op": "adamw", "dims": "1024,4096,4096,4096,1024", "state": "f32", "grad": "f32", "copy": True},
        # the ragged network's tensors (the smallest of 10 values), states in 8 bits
        {"name": "adamw_e4m3_ragged", "op": "adamw", "dims": "1000,3000,777,10", "state": "e4m3", "grad": "bf16", "copy": True},
        # four layers of 8192, states in 8 bits: what that choice is for
        {"name": "adamw_e4m3_8192", "op": "adamw", "dims": "8192,8192,8192,8192,8192", "state": "e4m3", "grad": "f32", "copy": True},
        # a training batch's activations, for the forward product and transposed for the weight gradient's
        {"name": "quant_act_8192x4096", "op": "quant", "rows": 8192, "cols": 4096, "pad": 0, "dtype": "bf16", "block_rows": 1, "both": True, "q": "e4m3"},
        # weights from their fp32 masters, 128 x 128 blocks, also transposed for the input gradient's product
        {"name": "quant_weight_4096x1024", "op": "quant", "rows": 4096, "cols": 1024, "pad": 0, "dtype": "f32", "block_rows": 128, "both": True, "q": "e4m3"},
        # a linear layer for 8 tokens: the weights have to be read once
        {"name": "gemm_8x4096x4096", "op": "gemm", "m": 8, "n": 4096, "k": 4096, "a": "e4m3", "b": "e4m3", "block_b": 128, "out": "bf16"},
        # the layer on the training batch
        {"name": "gemm_8192x4096x4096", "op": "gemm", "m": 8192, "n": 4096, "k": 4096, "a": "e4m3", "b": "e4m3", "block_b": 128, "out": "bf16"},
        # the weight gradient of the ragged network's first layer: both operands scaled along the batch, fp32 result
        {"name": "gemm_3000x1000x4099", "op": "gemm", "m": 3000, "n": 1000, "k": 4099, "a": "e4m3", "b": "e4m3", "block_b": 1, "out": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "adamw", "quant", "gemm"])
    if op in ("ln_fwd", "ln_bwd"):
        cols = _log(rng, 8, 16384)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        rows = _log(rng, 1, min(65536, max(1, 8192 * 4096 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 0, 8, 24]),
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "params": rng.choice(["f32", "bf16"])}
    if op == "adamw":
        layers = rng.randint(1, 8)
        dims = [_log(rng, 10, 4096) for _ in range(layers + 1)]
        return {"op": op, "dims": ",".join(map(str, dims)), "state": rng.choice(["f32", "e4m3"]),
                "grad": rng.choice(["f32", "bf16"]), "copy": rng.random() < 0.7}
    if op == "quant":
        cols = _log(rng, 16, 16384)
        rows = _log(rng, 1, min(65536, max(1, 8192 * 4096 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 8]), "dtype": rng.choice(["bf16", "bf16", "f32"]),
                "block_rows": rng.choice([1, 128]), "both": rng.random() < 0.5, "q": rng.choice(["e4m3", "e4m3", "e5m2"])}
    n, k = _log(rng, 16, 8192), _log(rng, 32, 8192)
    m = _log(rng, 1, min(65536, max(1, 8192 * 4096 * 4096 // (n * k))))
    return {"op": op, "m": m, "n": n, "k": k, "a": rng.choice(["e4m3", "e4m3", "e5m2"]), "b": "e4m3",
            "block_b": rng.choice([1, 128]), "out": rng.choice(["bf16", "f32"])}


def _up(n, k):
    return -(-n // k) * k


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rows_of(g, rows, cols, ld, dtype):
    """Activations: rows of their own size, a few columns far larger than the rest."""
    x = _normal(g, rows, ld)
    x.mul_(torch.exp(0.5 * _normal(g, rows, 1))).mul_(torch.exp(0.7 * _normal(g, 1, ld))).add_(0.3 * _normal(g, rows, 1))
    return x.to(dtype)


# ---------------------------------------------------------------- states
def _ln_state(case, g):
    rows, cols, t = case["rows"], case["cols"], TYPES[case["dtype"]]
    ld = cols + case["pad"]
    s = {"x": _rows_of(g, rows, cols, ld, t), "eps": 1e-5,
         "gamma": (1 + 0.2 * _normal(g, cols)).to(TYPES[case["params"]]), "beta": (0.2 * _normal(g, cols)).to(TYPES[case["params"]])}
    if case["op"] == "ln_fwd":
        s |= {"y": torch.zeros(rows, cols, dtype=t, device="cuda"), "mean": torch.zeros(rows, device="cuda"), "rstd": torch.zeros(rows, device="cuda")}
    else:
        x = s["x"][:, :cols].double()
        mean = x.mean(1)
        rstd = 1 / torch.sqrt(((x - mean[:, None]) ** 2).mean(1) + s["eps"])
        s |= {"mean": mean.float(), "rstd": rstd.float(), "dy": (1e-2 * _normal(g, rows, cols)).to(t),
              "dx": torch.zeros(rows, cols, dtype=t, device="cuda"),
              "dgamma": torch.zeros(cols, device="cuda"), "dbeta": torch.zeros(cols, device="cuda")}
    return s


def _tensors(case):
    """(offset, size, weight decay) of every tensor in the flat buffers, each at a multiple of 128 values."""
    dims, out, at = [int(d) for d in case["dims"].split(",")], [], 0
    for i in range(len(dims) - 1):
        for n, decay in ((dims[i] * dims[i + 1], DECAY), (dims[i + 1], 0.0)):
            out.append((at, n, decay))
            at += _up(n, BLOCK)
    return out, at


def _adamw_state(case, g):
    tensors, n = _tensors(case)
    live = torch.zeros(n, dtype=torch.bool, device="cuda")
    for at, k, _ in tensors:
        live[at:at + k] = True
    grad = _normal(g, n).mul_(1e-3)
    grad *= torch.exp(_normal(g, n // BLOCK)).repeat_interleave(BLOCK)
    grad *= live
    m, r = _normal(g, n).mul_(3e-4).mul_(live), _normal(g, n).abs_().mul_(1e-3).add_(1e-4).mul_(live)
    s = {"p": _normal(g, n).mul_(0.02).mul_(live), "g": grad.to(TYPES[case["grad"]]), "t": 20, "tensors": tensors}
    if case["state"] == "f32":
        s |= {"m": m, "v": r * r}
    else:
        s["m"], s["m_scale"] = _pack(m.view(-1, BLOCK), torch.float8_e4m3fn)
        s["v"], s["v_scale"] = _pack(r.view(-1, BLOCK), torch.float8_e4m3fn)
    if case["copy"]:
        s["copy"] = s["p"].to(torch.bfloat16)
    return s


def _quant_state(case, g):
    rows, cols, b, q = case["rows"], case["cols"], case["block_rows"], TYPES[case["q"]]
    s = {"x": _rows_of(g, rows, cols, cols + case["pad"], TYPES[case["dtype"]]),
         "q": torch.zeros(rows, _up(cols, 16), device="cuda").to(q), "scale": torch.zeros(-(-cols // BLOCK), -(-rows // b), device="cuda")}
    if case["both"]:
        s |= {"qt": torch.zeros(cols, _up(rows, 16), device="cuda").to(q), "scale_t": torch.zeros(-(-rows // BLOCK), -(-cols // b), device="cuda")}
    return s


def _operand(g, rows, k, dtype, block_rows):
    """What quantising leaves: values that fill the type's range block by block, rows padded to 16 bytes, a scale for each block."""
    x = torch.zeros(rows, _up(k, 16), device="cuda")
    x[:, :k] = _normal(g, rows, k).mul_(100.0 if dtype == torch.float8_e4m3fn else 1e4).clamp_(-448 if dtype == torch.float8_e4m3fn else -57344, 448 if dtype == torch.float8_e4m3fn else 57344)
    scale = torch.exp(0.5 * _normal(g, -(-k // BLOCK), -(-rows // block_rows))).mul_(0.01 if dtype == torch.float8_e4m3fn else 1e-4)
    return x.to(dtype), scale


def _gemm_state(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    a, sa = _operand(g, m, k, TYPES[case["a"]], 1)
    b, sb = _operand(g, n, k, TYPES[case["b"]], case["block_b"])
    return {"a": a, "scale_a": sa, "b": b, "scale_b": sb, "out": torch.zeros(m, n, dtype=TYPES[case["out"]], device="cuda")}


def prepare(case, seed):
    make = {"ln_fwd": _ln_state, "ln_bwd": _ln_state, "adamw": _adamw_state, "quant": _quant_state, "gemm": _gemm_state}[case["op"]]
    return {"case": case, **make(case, _generator(seed))}


# ---------------------------------------------------------------- plain forms
def _pack(x, dtype):
    """Blocks [count, values] -> (8-bit values, scale of each block): scale = largest magnitude / largest value of the type."""
    most = torch.full((x.shape[0], 1), torch.finfo(dtype).max, device=x.device)
    big = x.abs().amax(1, keepdim=True)
    none = big < TINY
    q = x * torch.where(none, torch.zeros_like(big), most / big)
    return q.to(dtype).reshape(-1), torch.where(none, torch.zeros_like(big), big / most).reshape(-1)


def _ln_fwd_plain(s):
    cols = s["case"]["cols"]
    x = s["x"][:, :cols].float()
    mean = x.sum(1) / cols
    x = x - mean[:, None]
    rstd = 1 / torch.sqrt((x * x).sum(1) / cols + s["eps"])
    y = x * rstd[:, None] * s["gamma"].float() + s["beta"].float()
    return {"y": y.to(s["y"].dtype), "mean": mean, "rstd": rstd}


def _ln_bwd_plain(s):
    cols = s["case"]["cols"]
    hat = (s["x"][:, :cols].float() - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dy"].float()
    dgamma, dbeta = (dy * hat).sum(0), dy.sum(0)
    dy = dy * s["gamma"].float()
    dx = s["rstd"][:, None] * (dy - (dy.sum(1) / cols)[:, None] - hat * ((dy * hat).sum(1) / cols)[:, None])
    return {"dx": dx.to(s["dx"].dtype), "dgamma": dgamma, "dbeta": dbeta}


def _adamw_plain(s):
    s["t"] += 1
    g, eight = s["g"].float(), s["case"]["state"] == "e4m3"
    if eight:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        r = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    r = torch.sqrt(v)
    blocks = torch.tensor([_up(n, BLOCK) for _, n, _ in s["tensors"]], device="cuda")
    keep = torch.repeat_interleave(torch.tensor([1 - LR * d for _, _, d in s["tensors"]], device="cuda"), blocks, output_size=g.numel())
    s["p"].copy_(s["p"] * keep - m * (LR / (1 - BETA1 ** s["t"])) / (r * (1 - BETA2 ** s["t"]) ** -0.5 + EPS))
    if eight:
        q, scale = _pack(m.view(-1, BLOCK), torch.float8_e4m3fn)
        s["m"].copy_(q), s["m_scale"].copy_(scale)
        q, scale = _pack(r.view(-1, BLOCK), torch.float8_e4m3fn)
        least = torch.full_like(r, 2.0 ** -9).to(torch.float8_e4m3fn)  # a root above zero stays above zero
        low = (q.float() == 0) & (r > 0) & (scale > 0).repeat_interleave(BLOCK)
        s["v"].copy_(torch.where(low, least.float(), q.float()).to(q.dtype)), s["v_scale"].copy_(scale)
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    if "copy" in s:
        s["copy"].copy_(s["p"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "m", "v", "m_scale", "v_scale", "copy") if k in s}


def _quant_one(x, dtype, block_rows):
    """[rows, cols] -> 8-bit [rows, cols], scale [column blocks, row blocks]."""
    rows, cols = x.shape
    up = torch.zeros(_up(rows, block_rows), _up(cols, BLOCK), device=x.device)
    up[:rows, :cols] = x
    blocks = up.view(-1, block_rows, up.shape[1] // BLOCK, BLOCK).permute(0, 2, 1, 3)
    q, scale = _pack(blocks.reshape(-1, block_rows * BLOCK), dtype)
    q = q.view(blocks.shape).permute(0, 2, 1, 3).reshape(up.shape)[:rows, :cols]
    return q, scale.view(blocks.shape[:2]).t()


def _quant_plain(s):
    case = s["case"]
    x = s["x"][:, :case["cols"]].float()
    q, scale = _quant_one(x, s["q"].dtype, case["block_rows"])
    s["q"][:, :case["cols"]] = q
    out = {"q": s["q"], "scale": scale}
    if case["both"]:
        q, scale = _quant_one(x.t(), s["q"].dtype, case["block_rows"])
        s["qt"][:, :case["rows"]] = q
        out |= {"qt": s["qt"], "scale_t": scale}
    return out


def _spread(scale, rows, k, block_rows):
    return scale.t().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :k]


def _gemm_plain(s):
    case = s["case"]
    m, n, k = case["m"], case["n"], case["k"]
    a = s["a"][:, :k].float() * _spread(s["scale_a"], m, k, 1)
    b = s["b"][:, :k].float() * _spread(s["scale_b"], n, k, case["block_b"])
    return (a @ b.t()).to(s["out"].dtype)


# ---------------------------------------------------------------- the framework's calls
def _ln_desc(s):
    import pkt_b200
    case, x = s["case"], s["x"]
    kind = {"bf16": pkt_b200.DTYPE_BF16, "f32": pkt_b200.DTYPE_F32}
    d = pkt_b200.LayerNormDesc(rows=case["rows"], cols=case["cols"], dtype=kind[case["dtype"]], param_dtype=kind[case["params"]], eps=s["eps"],
                               x=x.data_ptr(), ldx=x.stride(0), gamma=s["gamma"].data_ptr(), mean=s["mean"].data_ptr(), rstd=s["rstd"].data_ptr())
    if case["op"] == "ln_fwd":
        d.beta, d.y, d.ldy = s["beta"].data_ptr(), s["y"].data_ptr(), s["y"].stride(0)
    else:
        d.dy, d.lddy, d.dx, d.lddx = s["dy"].data_ptr(), s["dy"].stride(0), s["dx"].data_ptr(), s["dx"].stride(0)
        d.dgamma, d.dbeta = s["dgamma"].data_ptr(), s["dbeta"].data_ptr()
        s["work"] = torch.empty(pkt_b200.layernorm_backward_workspace(d), dtype=torch.uint8, device="cuda")
        d.workspace, d.workspace_bytes = s["work"].data_ptr(), s["work"].numel()
    return d


def _ln_own(s):
    import pkt_b200
    if "desc" not in s:
        s["desc"] = _ln_desc(s)
    if s["case"]["op"] == "ln_fwd":
        pkt_b200.layernorm_forward(s["desc"])
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    pkt_b200.layernorm_backward(s["desc"])
    return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def _adamw_own(s):
    import pkt_b200
    if "plan" not in s:
        tensors = []
        for at, n, decay in s["tensors"]:
            t = pkt_b200.AdamWTensor(param=s["p"][at:].data_ptr(), grad=s["g"][at:].data_ptr(), m=s["m"][at:].data_ptr(), v=s["v"][at:].data_ptr(), n=n, weight_decay=decay)
            if "m_scale" in s:
                t.m_scale, t.v_scale = s["m_scale"][at // BLOCK:].data_ptr(), s["v_scale"][at // BLOCK:].data_ptr()
            if "copy" in s:
                t.copy_bf16 = s["copy"][at:].data_ptr()
            tensors.append(t)
        s["plan"] = pkt_b200.AdamW(tensors, beta1=BETA1, beta2=BETA2, eps=EPS, grad_dtype=s["case"]["grad"], state_dtype=s["case"]["state"], step=s["t"])
    s["plan"].step(LR)
    return _adamw_outputs(s)


def _quant_own(s):
    import pkt_b200
    if "desc" not in s:
        case = s["case"]
        d = pkt_b200.Fp8QuantizeDesc(rows=case["rows"], cols=case["cols"], dtype=pkt_b200.DTYPE_BF16 if case["dtype"] == "bf16" else pkt_b200.DTYPE_F32,
                                     q_dtype=pkt_b200.DTYPE_E4M3 if case["q"] == "e4m3" else pkt_b200.DTYPE_E5M2, block_rows=case["block_rows"],
                                     x=s["x"].data_ptr(), ldx=s["x"].stride(0), q=s["q"].data_ptr(), ldq=s["q"].stride(0), scale=s["scale"].data_ptr(), ld_scale=s["scale"].stride(0))
        if case["both"]:
            d.qt, d.ldqt, d.scale_t, d.ld_scale_t = s["qt"].data_ptr(), s["qt"].stride(0), s["scale_t"].data_ptr(), s["scale_t"].stride(0)
        s["desc"] = d
    pkt_b200.fp8_quantize(s["desc"])
    return {k: s[k] for k in ("q", "scale", "qt", "scale_t") if k in s}


def _gemm_own(s):
    import pkt_b200
    if "desc" not in s:
        case, kind = s["case"], {"e4m3": pkt_b200.DTYPE_E4M3, "e5m2": pkt_b200.DTYPE_E5M2, "bf16": pkt_b200.DTYPE_BF16, "f32": pkt_b200.DTYPE_F32}
        s["desc"] = pkt_b200.Fp8GemmDesc(M=case["m"], N=case["n"], K=case["k"], a_dtype=kind[case["a"]], b_dtype=kind[case["b"]],
                                         a=s["a"].data_ptr(), lda=s["a"].stride(0), scale_a=s["scale_a"].data_ptr(), ld_scale_a=s["scale_a"].stride(0), a_block_rows=1,
                                         b=s["b"].data_ptr(), ldb=s["b"].stride(0), scale_b=s["scale_b"].data_ptr(), ld_scale_b=s["scale_b"].stride(0), b_block_rows=case["block_b"],
                                         out=s["out"].data_ptr(), ldo=s["out"].stride(0), out_dtype=kind[case["out"]])
    pkt_b200.fp8_gemm(s["desc"])
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ln_fwd": _ln_own, "ln_bwd": _ln_own, "adamw": _adamw_own, "quant": _quant_own, "gemm": _gemm_own}[op](state)
    return {"ln_fwd": _ln_fwd_plain, "ln_bwd": _ln_bwd_plain, "adamw": _adamw_plain, "quant": _quant_plain, "gemm": _gemm_plain}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, es, ps = case["rows"], case["cols"], 2 if case["dtype"] == "bf16" else 4, 2 if case["params"] == "bf16" else 4
        if op == "ln_fwd":
            return {"bytes": rows * cols * 2 * es + 8 * rows + 2 * cols * ps, "flops": 8 * rows * cols}
        return {"bytes": rows * cols * 3 * es + 8 * rows + cols * (ps + 8), "flops": 14 * rows * cols}
    if op == "adamw":
        n = sum(k for _, k, _ in _tensors(case)[0])
        state = 16 if case["state"] == "f32" else 4 + 16 / BLOCK
        return {"bytes": n * (8 + (4 if case["grad"] == "f32" else 2) + state + (2 if case["copy"] else 0)), "flops": 14 * n}
    if op == "quant":
        rows, cols = case["rows"], case["cols"]
        n, sides = rows * cols, 2 if case["both"] else 1
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + sides * (n + 4 * n / (BLOCK * case["block_rows"])), "flops": 3 * sides * n}
    m, n, k = case["m"], case["n"], case["k"]
    scales = 4 * -(-k // BLOCK) * (m + -(-n // case["block_b"]))
    return {"bytes": m * k + n * k + scales + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_blocks(x, dtype, block_rows):
    """The 8-bit values and scales of a [rows, cols] matrix in 64 bits: each block is divided by its largest magnitude over the type's."""
    rows, cols = x.shape
    most = 448.0 if dtype == torch.float8_e4m3fn else 57344.0
    pad = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    big = pad.abs().unflatten(1, (-1, BLOCK)).amax(2).unflatten(0, (-1, block_rows)).amax(1)
    scale = torch.where(big < TINY, torch.zeros_like(big), big / most)
    every = scale.repeat_interleave(block_rows, 0).repeat_interleave(BLOCK, 1)[:rows, :cols]
    return torch.where(every > 0, x / every, torch.zeros_like(x)), scale.t().contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        x = s["x"][:, :case["cols"]].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + s["eps"]).pow(-0.5)
        return {"y": torch.addcmul(s["beta"].double(), (x - mean[:, None]) * rstd[:, None], s["gamma"].double()), "mean": mean, "rstd": rstd}
    if op == "ln_bwd":
        # y_j = gamma_j h_j + beta_j, h = (x - mean) rstd: dL/dx is the projection of rstd gamma dy off the constants and off h
        x, dy = s["x"][:, :case["cols"]].double(), s["dy"].double()
        rstd = s["rstd"].double()[:, None]
        h = x.sub(s["mean"].double()[:, None]).mul(rstd)
        w = dy * s["gamma"].double()
        dx = rstd * (w - w.mean(1, keepdim=True) - h * (w * h).mean(1, keepdim=True))
        return {"dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, h), "dbeta": dy.sum(0)}
    if op == "adamw":
        t, g, eight = s["t"] + 1, s["g"].double(), case["state"] == "e4m3"
        if eight:
            m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
            v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)).square()
        else:
            m, v = s["m"].double(), s["v"].double()
        m, v = torch.lerp(g, m, BETA1), torch.lerp(g.square(), v, BETA2)
        p = s["p"].double()
        for at, n, decay in s["tensors"]:
            p[at:at + n] *= 1 - LR * decay
        p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out = {"p": p}
        if eight:
            root = v.sqrt()
            for name, x in (("m", m), ("v", root)):
                q, scale = _exact_blocks(x.view(-1, BLOCK), torch.float8_e4m3fn, 1)
                q = q.to(torch.float8_e4m3fn).double().view(-1)
                out |= {name: torch.where((q == 0) & (x > 0) & (name == "v"), torch.full_like(q, 2.0 ** -9), q), name + "_scale": scale.view(-1)}
        else:
            out |= {"m": m, "v": v}
        return out | ({"copy": p} if case["copy"] else {})
    if op == "quant":
        x, kind = s["x"][:, :case["cols"]].double(), s["q"].dtype
        out = {}
        for name, y, into in (("", x, s["q"]), ("t", x.t(), s.get("qt"))):
            if into is not None:
                q, scale = _exact_blocks(y, kind, case["block_rows"])
                whole = torch.zeros(into.shape, dtype=torch.float64, device="cuda")
                whole[:, :q.shape[1]] = q.to(kind).double()
                out |= {"q" + name: whole, "scale" + ("_t" if name else ""): scale}
        return out
    a, b = (s[x][:, :case["k"]].double() for x in "ab")
    a.mul_(s["scale_a"].double().t().repeat_interleave(BLOCK, 1)[:, :case["k"]])
    rows = s["scale_b"].double().t().repeat_interleave(BLOCK, 1)[:, :case["k"]]
    b.mul_(rows if case["block_b"] == 1 else rows.repeat_interleave(BLOCK, 0)[:case["n"]])
    return torch.einsum("mk,nk->mn", a, b)
