"""The 8-bit activation checkpoints of the training step and the per-head edge attention, as a user's program calls them.

Cases are dicts; `op` is one of
  mx8    quantise an activation (rows, D) for the backward pass and restore it: MXINT8, 32 channels share a power-of-two scale
  wgrad  weight and bias gradient of a Linear whose input is held in 8 bits: dW = dY^T x, db = column sums of dY
  serve  the per-head edge attention of the `improved` block without a graph (inference)
  train  the same, forward and backward; `ckpt`: its E1 operand is held in 8 bits between the two
`own` chooses between the framework's kernels and the plain form in elementary torch operations."""
import math

import torch

own = False

GROUP = 32
# (in, out) features of the per-pair Linears: align_absorbing (de 64, dx 256, dim_ffE 128) and the tiny test config (de 32, dx 64)
LINEAR_SHAPES = [(i, o) for i in (32, 64, 128, 256) for o in (32, 64, 128, 256) if i * o <= 64 * 256]
# (dx, heads): align_absorbing, the tiny test config and shapes around them
HEAD_SHAPES = [(256, 8), (64, 4), (32, 4), (128, 8), (256, 4), (256, 16), (96, 3), (192, 6), (64, 8)]
LARGEST = 16 * 300 * 300 * 256          # pair-channels of the largest listed attention


def listed():
    train_rows = 16 * 140 * 140          # the training benchmark: 16 graphs of up to 140 nodes
    return [
        # Y of one layer of the training benchmark, the input of e_out
        {"name": "mx8 bf16 train batch", "op": "mx8", "rows": train_rows, "D": 256, "dtype": "bf16", "keep": False},
        # the edge feed-forward's hidden tensor (ReLU: many zeros, kept apart from small values) of a small odd batch, fp32
        {"name": "mx8 fp32 small", "op": "mx8", "rows": 3 * 37 * 37, "D": 128, "dtype": "fp32", "keep": True},
        # e_mul / e_add of the training benchmark, mixed precision
        {"name": "wgrad 64-256 bf16", "op": "wgrad", "rows": train_rows, "in": 64, "out": 256, "dtype": "bf16"},
        # e_out of the training benchmark, fp32
        {"name": "wgrad 256-64 fp32", "op": "wgrad", "rows": train_rows, "in": 256, "out": 64, "dtype": "fp32"},
        # linE2 of a ragged batch (7 graphs of 93 nodes), mixed precision
        {"name": "wgrad 128-64 bf16 odd", "op": "wgrad", "rows": 7 * 93 * 93, "in": 128, "out": 64, "dtype": "bf16"},
        # e_mul of the tiny test config: 4 graphs of 24 nodes, latency
        {"name": "wgrad 32-64 fp32 tiny", "op": "wgrad", "rows": 4 * 24 * 24, "in": 32, "out": 64, "dtype": "fp32"},
        # one product of the tiny test config
        {"name": "serve fp32 one graph", "op": "serve", "B": 1, "n": 24, "dx": 64, "heads": 4, "dtype": "fp32", "cap": 0.0, "mol": False},
        # sampling at the benchmark's graph size, attention inside molecules only
        {"name": "serve bf16 n300", "op": "serve", "B": 8, "n": 300, "dx": 256, "heads": 8, "dtype": "bf16", "cap": 0.0, "mol": True},
        # the training benchmark, mixed precision
        {"name": "train bf16 n140", "op": "train", "B": 16, "n": 140, "dx": 256, "heads": 8, "dtype": "bf16", "cap": 0.0, "mol": False, "ckpt": False},
        # a ragged fp32 batch with capped scores
        {"name": "train fp32 n93 cap", "op": "train", "B": 7, "n": 93, "dx": 256, "heads": 8, "dtype": "fp32", "cap": 30.0, "mol": False, "ckpt": True},
        # the tiny test config's training batch, latency
        {"name": "train fp32 tiny", "op": "train", "B": 4, "n": 24, "dx": 64, "heads": 4, "dtype": "fp32", "cap": 0.0, "mol": True, "ckpt": False},
        # the largest graphs in training, everything on
        {"name": "train bf16 n300 8-bit", "op": "train", "B": 16, "n": 300, "dx": 256, "heads": 8, "dtype": "bf16", "cap": 30.0, "mol": True, "ckpt": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mx8", "wgrad", "serve", "train"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "mx8":
        D = rng.choice([32, 64, 128, 256, 256, rng.randint(1, 300)])
        return {"op": op, "rows": _log(rng, 1, 400_000), "D": D, "dtype": dtype, "keep": rng.random() < 0.5}
    if op == "wgrad":
        i, o = rng.choice(LINEAR_SHAPES)
        return {"op": op, "rows": _log(rng, 1, 400_000), "in": i, "out": o, "dtype": dtype}
    dx, heads = rng.choice(HEAD_SHAPES)
    n = _log(rng, 1, 300)
    B = _log(rng, 1, max(1, min(64, LARGEST // (2 if dtype == "fp32" else 1) // (n * n * dx))))
    case = {"op": op, "B": B, "n": n, "dx": dx, "heads": heads, "dtype": dtype, "cap": rng.choice([0.0, 0.0, 30.0, round(rng.uniform(5.0, 60.0), 2)]),
            "mol": rng.random() < 0.5}
    if op == "train":
        case["ckpt"] = rng.random() < 0.5
    return case


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "mx8":              # in, codes and scales out and back in, out
        D = case["D"]
        return {"bytes": case["rows"] * (2 * e * D + 2 * (D + -(-D // GROUP))), "flops": case["rows"] * D * 6}
    if case["op"] == "wgrad":
        i, o = case["in"], case["out"]
        return {"bytes": case["rows"] * (i + i // GROUP + o * e) + 4 * (i * o + o), "flops": 2 * case["rows"] * i * o}
    nodes, dx = case["B"] * case["n"], case["dx"]
    pc = nodes * case["n"] * dx
    if case["op"] == "serve":            # E1, E2 in, Y out; Q, K, V in, wV out
        return {"bytes": 3 * e * pc + 16 * nodes * dx, "flops": 8 * pc}
    return {"bytes": 6 * e * pc + 32 * nodes * dx, "flops": 26 * pc}     # and dY in, dE1, dE2 out; dwV in, dQ, dK, dV out


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    dev, dt = "cuda", _type(case)
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)
    if case["op"] in ("mx8", "wgrad"):
        R, D = case["rows"], case["D"] if case["op"] == "mx8" else case["in"]
        # an activation: channels of different spread, rows of padded pairs all zero, after a ReLU where zeros are kept apart
        x = rn(R, D) * torch.exp(rn(D))
        x *= (torch.rand(R, 1, device=dev, generator=g) < 0.8)
        if case.get("keep"):
            x = torch.relu(x)
        x = x.to(dt)
        if case["op"] == "mx8":
            return {"case": case, "x": x}
        codes, exps = _quantise(x, False)
        dy = (rn(R, case["out"]) * 1e-2 * torch.exp(rn(R, 1))).to(dt)
        return {"case": case, "codes": codes.to(torch.int8).reshape(R, D), "scales": exps.to(torch.uint8), "dy": dy}
    B, n, dx = case["B"], case["n"], case["dx"]
    real = torch.randint(max(1, n // 2), n + 1, (B, 1), device=dev, generator=g)
    mask = torch.arange(n, device=dev)[None] < real
    # molecules of a reaction: consecutive runs of nodes; padded nodes belong to none
    mol = torch.div(torch.arange(n, device=dev)[None] * torch.randint(2, 6, (B, 1), device=dev, generator=g), real, rounding_mode="floor")
    mol = torch.where(mask, mol, -1).to(torch.int32)
    m = mask[:, :, None].float()
    s = {"case": case, "mask": mask, "mol": mol if case["mol"] else None}
    for k in "QKV":
        s[k] = rn(B, n, dx) * m
    s["E1"], s["E2"] = (rn(B, n, n, dx) * 0.5).to(dt), (rn(B, n, n, dx) * 0.5).to(dt)
    if case["op"] == "train":
        s["dY"], s["dwV"] = (rn(B, n, n, dx) * 0.1).to(dt), rn(B, n, dx)
        for k in ("Q", "K", "V", "E1", "E2"):
            s[k].requires_grad_(True)
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------------------


def _quantise(x, keep):
    """Whole numbers (rows, groups, 32) as floats and the biased exponents (rows, groups) of MXINT8."""
    R, D = x.shape
    G = -(-D // GROUP)
    x = torch.nn.functional.pad(x.float(), (0, G * GROUP - D)).reshape(R, G, GROUP)
    bits = x.abs().amax(-1).view(torch.int32)
    e = ((bits >> 23) + ((bits & 0x7FFFFF) >= 0x7F0000)).clamp(27, 254)       # 127.5 / 64 and more would round to 128
    q = (x * torch.ldexp(torch.ones((), device=x.device), 133 - e)[..., None]).round().clamp(-127, 127)
    if keep:
        q = torch.where((q == 0) & (x != 0), torch.sign(x), q)
    return (q if G * GROUP == D else q.reshape(R, G * GROUP)[:, :D]), e


def _restore(q, e, D):
    """The values of codes (rows, D) with biased exponents (rows, groups), in 32 bits."""
    R, G = e.shape
    f = torch.ldexp(torch.ones((), device=e.device), e.to(torch.int32) - 133)
    q = q.reshape(R, -1).float()
    if G * GROUP == D:
        return (q.reshape(R, G, GROUP) * f[..., None]).reshape(R, D)
    return q * f.repeat_interleave(GROUP, 1)[:, :D]


def _heads(t, H):
    """(B,n,dx) -> (B,H,n,df)"""
    B, n, dx = t.shape
    return t.reshape(B, n, H, dx // H).transpose(1, 2).contiguous()


def _attention(s, E1, E2):
    """Y (32 bits), the capped scores, the probabilities (B,i,j,H) and wV."""
    c = s["case"]
    B, n, dx, H = c["B"], c["n"], c["dx"], c["heads"]
    pm = (s["mask"][:, :, None] & s["mask"][:, None, :])[..., None]
    qk = s["Q"][:, :, None] * s["K"][:, None] * (1 / math.sqrt(dx // H))
    Y = qk * (torch.where(pm, E1, 0) + 1) + torch.where(pm, E2, 0)
    S = Y.reshape(B, n, n, H, dx // H).sum(-1)
    if c["cap"] > 0:
        S = torch.tanh(S / c["cap"]) * c["cap"]
    T = S
    if s["mol"] is not None:
        ok = (s["mol"][:, :, None] == s["mol"][:, None, :]) & (s["mol"] >= 0)[:, :, None]
        T = S.masked_fill(~ok[..., None], -math.inf)
    top = T.amax(2, keepdim=True)
    P = torch.exp(T - torch.where(torch.isinf(top), 0, top))
    total = P.sum(2, keepdim=True)
    P = P / torch.where(total > 0, total, 1)
    wV = torch.matmul(P.permute(0, 3, 1, 2).contiguous(), _heads(s["V"], H)).transpose(1, 2).reshape(B, n, dx)
    return Y, S, P, wV, qk, pm


def _plain(s):
    c = s["case"]
    dt = _type(c)
    if c["op"] == "mx8":
        q, e = _quantise(s["x"], c["keep"])
        return _restore(q, e, c["D"]).to(dt)
    if c["op"] == "wgrad":
        dy = s["dy"].float()
        return dy.t() @ _restore(s["codes"], s["scales"], c["in"]), dy.sum(0)
    E1 = s["E1"].float()
    Y, S, P, wV, qk, pm = _attention(s, E1, s["E2"].float())
    if c["op"] == "serve":
        return Y.to(dt), wV
    B, n, dx, H = c["B"], c["n"], c["dx"], c["heads"]
    df = dx // H
    if c["ckpt"]:
        E1 = _restore(*_quantise(E1.reshape(-1, dx), False), dx).reshape(B, n, n, dx)
    out = Y.to(dt)
    del Y
    do = s["dwV"]
    dP = torch.matmul(_heads(do, H), _heads(s["V"], H).transpose(2, 3).contiguous()).permute(0, 2, 3, 1)
    dS = P * (dP - (do * wV).reshape(B, n, 1, H, df).sum(-1))
    if c["cap"] > 0:
        dS = dS * (1 - (S / c["cap"]) ** 2)
    dY = (s["dY"].float().reshape(B, n, n, H, df) + dS[..., None]).reshape(B, n, n, dx)
    dE1, dE2 = torch.where(pm, dY * qk, 0).to(dt), torch.where(pm, dY, 0).to(dt)
    t = dY * (torch.where(pm, E1, 0) + 1) * (1 / math.sqrt(df))
    dQ, dK = (t * s["K"][:, None]).sum(2), (t * s["Q"][:, :, None]).sum(1)
    dV = torch.matmul(P.permute(0, 3, 2, 1).contiguous(), _heads(do, H)).transpose(1, 2).reshape(B, n, dx)
    return out, wV, dQ, dK, dV, dE1, dE2


# ---- the framework's calls ------------------------------------------------------------------------------------------------------


def _own(s):
    from diffalign_amd import autograd_ops, mx8
    c = s["case"]
    if c["op"] == "mx8":
        return mx8.dequantize(mx8.quantize(s["x"], keep_nonzero=c["keep"]), s["x"].dtype)
    if c["op"] == "wgrad":
        return mx8.linear_wgrad(mx8.Mx8(s["codes"], s["scales"]), s["dy"])
    Y, wV = autograd_ops.head_attention(s["Q"], s["K"], s["V"], s["E1"], s["E2"], s["mask"], c["heads"], cap=c["cap"], groups=s["mol"],
                                        checkpoint="mx8" if c.get("ckpt") else "none")
    if c["op"] == "serve":
        return Y, wV
    return (Y, wV) + torch.autograd.grad((Y, wV), [s[k] for k in ("Q", "K", "V", "E1", "E2")], (s["dY"], s["dwV"]))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---- 64 bits, from the definitions ----------------------------------------------------------------------------------------------


def _exact_values(x, keep):
    """What 8 bits hold of x (rows, D), in 64 bits."""
    x = x.double()
    out = torch.empty_like(x)
    for k in range(0, x.shape[1], GROUP):
        part = x[:, k:k + GROUP]
        m, e = torch.frexp(part.abs().amax(1, keepdim=True))                 # amax = m 2^e, m in [1/2, 1)
        step = torch.exp2((e + (m >= 127.5 / 128).to(e.dtype)).clamp(-99, 128).double() - 7)
        q = torch.clamp(torch.round(part / step), -127, 127)
        if keep:
            q = torch.where((q == 0) & (part != 0), torch.sign(part), q)
        out[:, k:k + GROUP] = q * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "mx8":
            return _exact_values(s["x"], case["keep"])
        if case["op"] == "wgrad":
            e = s["scales"].double().repeat_interleave(GROUP, 1)[:, :case["in"]]
            dy = s["dy"].double()
            return torch.mm((s["codes"].double() * torch.exp2(e - 133)).t(), dy).t().contiguous(), dy.sum(0)
        graphs = [_exact_graph(s, b) for b in range(case["B"])]
        return tuple(torch.stack([x[k] for x in graphs]) for k in range(len(graphs[0])))


def _exact_graph(s, b):
    c = s["case"]
    n, dx, H = c["n"], c["dx"], c["heads"]
    df = dx // H
    Q, K, V = (s[k][b].double().reshape(n, H, df) for k in "QKV")
    pm = s["mask"][b][:, None, None, None] & s["mask"][b][None, :, None, None]
    E1, E2 = (torch.where(pm, s[k][b].double().reshape(n, n, H, df), 0.0) for k in ("E1", "E2"))
    Y = torch.einsum("ihc,jhc->ijhc", Q, K) / math.sqrt(df) * (1 + E1) + E2
    S = Y.sum(-1)
    if c["cap"] > 0:
        S = c["cap"] * torch.tanh(S / c["cap"])
    P = torch.softmax(S, 1)
    if s["mol"] is not None:
        mol = s["mol"][b]
        ok = ((mol[:, None] == mol[None]) & (mol[:, None] >= 0))[..., None]
        P = torch.nan_to_num(torch.softmax(torch.where(ok, S, -math.inf), 1), nan=0.0)
    wV = torch.einsum("ijh,jhc->ihc", P, V)
    flat = lambda t: t.reshape(t.shape[:-2] + (dx,))
    if c["op"] == "serve":
        return flat(Y), flat(wV)
    do, dY = s["dwV"][b].double().reshape(n, H, df), s["dY"][b].double().reshape(n, n, H, df)
    dP = torch.einsum("ihc,jhc->ijh", do, V)
    dS = P * (dP - (P * dP).sum(1, keepdim=True))
    if c["cap"] > 0:
        dS = dS / torch.cosh(torch.atanh((S / c["cap"]).clamp(-1 + 1e-15, 1 - 1e-15))) ** 2
    G = dY + dS[..., None]
    if c["ckpt"]:
        E1 = torch.where(pm, _exact_values(s["E1"][b].reshape(n * n, dx), False).reshape(n, n, H, df), 0.0)
    f = (1 + E1) / math.sqrt(df)
    dE1 = torch.where(pm, G * torch.einsum("ihc,jhc->ijhc", Q, K) / math.sqrt(df), 0.0)
    dE2 = torch.where(pm, G, 0.0)
    dQ, dK = torch.einsum("ijhc,jhc->ihc", G * f, K), torch.einsum("ijhc,ihc->jhc", G * f, Q)
    return (flat(Y), flat(wV), flat(dQ), flat(dK), flat(torch.einsum("ijh,ihc->jhc", P, do)), flat(dE1), flat(dE2))
