"""Timed cases of the dense and few-token operators around the routed experts of a sparse layer.

Four operators, each as a user calls it (``own`` true) and in a plain form of elementary torch
operations (``own`` false):

* ``norm``   the block's boundary: residual + scale * gate * RMSNorm(delta), then the next RMSNorm;
* ``linear`` a product in 8-bit floating point (E4M3) with one power-of-two scale per 1 x 128
             activations and one float32 scale per 128 x 128 weights, activations quantised in the call;
* ``mlp``    the dense shared expert in that arithmetic: gate / up, SwiGLU, quantised again, down;
* ``few``    a whole routed-expert layer for a few tokens: router, NVFP4 experts on bf16 activations
             (no activation quantisation), weighted combine.
"""
import math

import torch

own = False

H, I, E, K = 6144, 2048, 256, 8            # the model's hidden, expert intermediate, experts, top-k
SCALING = 2.5                              # routed scaling factor
EPS = 1e-5


def listed():
    return [
        # decode, one row: the block's boundary between attention and the sparse layer
        {"name": "norm-token", "op": "norm", "rows": 1, "width": H, "form": "pre", "type": "bf16"},
        # a mixed batch through a block with norms on both sides, a gate per channel and a scaled branch
        {"name": "norm-sandwich", "op": "norm", "rows": 333, "width": 5120, "form": "sandwich", "type": "bf16"},
        # float32 residual stream with a gate per row, odd width
        {"name": "norm-f32-odd", "op": "norm", "rows": 1021, "width": 4100, "form": "rowgate", "type": "f32"},
        # a prefill batch at the same boundary as norm-token
        {"name": "norm-prefill", "op": "norm", "rows": 8192, "width": H, "form": "pre", "type": "bf16"},
        # gate|up projection of the shared expert for one decoded token
        {"name": "linear-token", "op": "linear", "rows": 1, "n": 2 * I, "k": H},
        # a ragged projection: no size a multiple of the scale block
        {"name": "linear-odd", "op": "linear", "rows": 197, "n": 1500, "k": 2000},
        # down projection of a prefill batch
        {"name": "linear-prefill", "op": "linear", "rows": 8192, "n": H, "k": I},
        # shared expert beside the decode step, one token and a batch
        {"name": "mlp-token", "op": "mlp", "rows": 1, "hidden": H, "inter": I},
        {"name": "mlp-prefill", "op": "mlp", "rows": 4096, "hidden": H, "inter": I},
        # the sparse layer of one decoded token
        {"name": "few-token", "op": "few", "rows": 1, "hidden": H, "inter": I, "experts": E, "top_k": K, "fold": False},
        # another, smaller shape with odd counts, residual and shared rows folded in
        {"name": "few-small", "op": "few", "rows": 7, "hidden": 1280, "inter": 768, "experts": 40, "top_k": 6, "fold": True},
        # sixteen rows: four sequences with three drafted tokens each, residual and shared rows folded in
        {"name": "few-drafts", "op": "few", "rows": 16, "hidden": H, "inter": I, "experts": E, "top_k": K, "fold": True},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999 * step)))
    return max(lo, min(hi, int(v // step) * step))


def draw(rng):
    op = rng.choice(["norm", "linear", "mlp", "few"])
    if op == "norm":
        width = _log(rng, 256, 16384, 4)
        return {"op": op, "rows": _log(rng, 1, min(8192, 8192 * H // (2 * width))), "width": width,
                "form": rng.choice(["pre", "sandwich", "rowgate", "plain"]), "type": rng.choice(["bf16", "f32"])}
    if op == "linear":
        n, k = _log(rng, 64, 8192, 4), _log(rng, 128, 8192, 16)
        return {"op": op, "rows": _log(rng, 1, max(1, min(8192, 8192 * H * I // (n * k)))), "n": n, "k": k}
    if op == "mlp":
        hidden, inter = _log(rng, 256, H, 16), _log(rng, 128, I, 16)
        return {"op": op, "rows": _log(rng, 1, 4096), "hidden": hidden, "inter": inter}
    experts = rng.choice([8, 24, 64, 128, 256])
    return {"op": op, "rows": _log(rng, 1, 16), "hidden": 256 * rng.randint(2, 24), "inter": 256 * rng.randint(1, 8),
            "experts": experts, "top_k": rng.randint(1, min(8, experts)), "fold": rng.random() < 0.5}


def _type(case):
    return torch.bfloat16 if case.get("type", "bf16") == "bf16" else torch.float32


def _round_fp8_weight(w):
    """float32 [n, k] -> E4M3 codes and one float32 scale per 128 x 128 block (ragged at the edges)."""
    n, k = w.shape
    pad = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).view(-(-n // 128), 128, -(-k // 128), 128)
    scale = pad.abs().amax(dim=(1, 3)).clamp_min(1e-12) / 448.0
    codes = (pad / scale[:, None, :, None]).view(-(-n // 128) * 128, -1)[:n, :k].to(torch.float8_e4m3fn)
    return codes.contiguous(), scale.contiguous()


def _round_nvfp4_weight(w):
    """float32 [..., k] -> packed E2M1 codes (low nibble first), E4M3 scale bytes per 16 values, scale_2."""
    s2 = w.abs().amax() / (6.0 * 448.0)
    blocks = w.view(*w.shape[:-1], -1, 16)
    scale = (blocks.abs().amax(-1) / (6.0 * s2)).to(torch.float8_e4m3fn)
    v = blocks / (scale.float() * s2).clamp_min(1e-30)[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    code = torch.bucketize(v.abs(), edges, out_int32=True).to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
    code = code.view(w.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8), s2


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std

    op, rows = case["op"], case["rows"]
    s = {"case": case}
    if op == "norm":
        t, width, form = _type(case), case["width"], case["form"]
        s["residual"] = normal(rows, width, std=2.0).to(t)
        s["delta"] = None if form == "plain" else normal(rows, width, std=0.5).to(t)
        s["norm_weight"] = (1.0 + normal(width, std=0.1)).to(t)
        s["post_weight"] = (1.0 + normal(width, std=0.1)).to(t) if form == "sandwich" else None
        s["gate"] = {"sandwich": lambda: torch.sigmoid(normal(1, width)).to(t),
                     "rowgate": lambda: torch.sigmoid(normal(rows, 1)).to(t)}.get(form, lambda: None)()
        s["scale"] = 0.25 if form == "sandwich" else 1.0
        return s
    if op == "linear":
        s["x"] = normal(rows, case["k"]).to(torch.bfloat16)
        s["w"] = _round_fp8_weight(normal(case["n"], case["k"], std=0.02))
        return s
    if op == "mlp":
        hidden, inter = case["hidden"], case["inter"]
        s["x"] = normal(rows, hidden).to(torch.bfloat16)
        s["gate"], s["up"] = (_round_fp8_weight(normal(inter, hidden, std=0.02)) for _ in range(2))
        s["down"] = _round_fp8_weight(normal(hidden, inter, std=0.02))
        return s
    hidden, inter, experts, top_k = case["hidden"], case["inter"], case["experts"], case["top_k"]
    s["x"] = normal(rows, hidden).to(torch.bfloat16)
    s["router_w"], s["router_b"] = normal(experts, hidden, std=0.02), normal(experts, std=0.01)
    s["residual"] = normal(rows, hidden, std=2.0).to(torch.bfloat16) if case["fold"] else None
    s["shared"] = normal(rows, hidden, std=0.3).to(torch.bfloat16) if case["fold"] else None
    for name, n, k in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
        codes = torch.empty(experts, n, k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(experts, n, k // 16, dtype=torch.uint8, device="cuda")
        scale2 = torch.empty(experts, device="cuda")
        for e in range(experts):
            codes[e], scales[e], scale2[e] = _round_nvfp4_weight(normal(n, k, std=0.02))
        s[name] = (codes, scales, scale2)
    if own:
        # the handle a program keeps: the same weights, laid out by the library once
        from __graft_entry__ import load_package
        load_package()
        from glmrt_b200.layer import MoeLayer
        layer = MoeLayer(hidden, inter, experts, top_k, max_tokens=16, scaling=SCALING)
        layer.set_router(s["router_w"], s["router_b"])
        s2 = torch.stack([s[n][2] for n in ("gate", "up", "down")], 1).tolist()
        for e in range(experts):
            layer.set_expert(e, *(s[n][j][e] for n in ("gate", "up", "down") for j in range(2)), s2[e])
        s["layer"] = layer
    return s


# ---- plain forms ---------------------------------------------------------------------------------
def _plain_norm(s):
    t = s["residual"].dtype
    r = s["residual"].float()
    if s["delta"] is not None:
        d = s["delta"].float()
        if s["post_weight"] is not None:
            d = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS) * s["post_weight"].float()
        if s["gate"] is not None:
            d = d * s["gate"].float()
        r = r + s["scale"] * d
    y = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * s["norm_weight"].float()
    return [r.to(t), y.to(t)]


def _plain_quantised(x):
    """Rows of x as the E4M3 values they are quantised to: per row and 128 columns one scale, the
    smallest power of two with amax / scale <= 448."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -k % 128)).view(rows, -1, 128)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100) / 448.0)
    scale = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int())
    return ((b / scale).to(torch.float8_e4m3fn).float() * scale).view(rows, -1)[:, :k]


def _plain_fp8_weight(w):
    codes, scale = w
    n, k = codes.shape
    return codes.float() * scale.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _plain_linear(x, w):
    return _plain_quantised(x) @ _plain_fp8_weight(w).T


def _plain_nvfp4(w, idx):
    """The float32 weights of experts idx [...]."""
    codes, scales, scale2 = w
    c = codes[idx]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = values[c.int()].unflatten(-1, (-1, 16)) * scales[idx].view(torch.float8_e4m3fn).float()[..., None]
    return v.flatten(-2) * scale2[idx][..., None, None]


def _plain_few(s):
    c = s["case"]
    score = torch.sigmoid(s["x"].double() @ s["router_w"].double().T)           # 64 bits: neighbours in rank
    idx = torch.sort(score + s["router_b"].double(), dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = score.gather(1, idx)
    w = (w / w.sum(1, keepdim=True) * SCALING).float()
    x = s["x"].float()[:, None, :, None]
    g = (_plain_nvfp4(s["gate"], idx) @ x)[..., 0]
    u = (_plain_nvfp4(s["up"], idx) @ x)[..., 0]
    act = g / (1.0 + torch.exp(-g)) * u * w[..., None]
    out = (_plain_nvfp4(s["down"], idx) @ act[..., None])[..., 0].sum(1)
    if s["residual"] is not None:
        out = s["residual"].float() + (s["shared"].float() + out)
    return out.to(torch.bfloat16)


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "few":
            return s["layer"].forward_few(s["x"], residual_bf16=s["residual"], shared_delta_bf16=s["shared"])
        from __graft_entry__ import load_package
        load_package()
        if op == "norm":
            from glmrt_b200.block_norm import block_norm
            return list(block_norm(s["residual"], s["delta"], norm_weight=s["norm_weight"],
                                   post_weight=s["post_weight"], gate=s["gate"], scale=s["scale"], eps=EPS))
        from glmrt_b200 import fp8
        if op == "linear":
            return fp8.block_linear(s["x"], *s["w"])
        return fp8.gated_mlp(s["x"], *s["gate"], *s["up"], *s["down"])
    if op == "norm":
        return _plain_norm(s)
    if op == "linear":
        return _plain_linear(s["x"], s["w"]).to(torch.bfloat16)
    if op == "mlp":
        g, u = _plain_linear(s["x"], s["gate"]), _plain_linear(s["x"], s["up"])
        return _plain_linear(g / (1.0 + torch.exp(-g)) * u, s["down"]).to(torch.bfloat16)
    return _plain_few(s)


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "norm":
        size = 2 if case.get("type", "bf16") == "bf16" else 4
        streams = 2 if case["form"] == "plain" else 4        # rows in and normalised rows out; with a branch it and the new residual too
        return {"bytes": rows * case["width"] * size * streams, "flops": 10 * rows * case["width"]}
    if op == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": rows * k * 2 + n * k + rows * n * 2, "flops": 2 * rows * n * k}
    if op == "mlp":
        hidden, inter = case["hidden"], case["inter"]
        return {"bytes": 4 * rows * hidden + 3 * hidden * inter, "flops": 6 * rows * hidden * inter}
    hidden, inter, experts, top_k = case["hidden"], case["inter"], case["experts"], case["top_k"]
    # experts that `rows` independent choices of top_k touch, on average
    touched = experts * (1.0 - (1.0 - top_k / experts) ** rows)
    return {"bytes": int(touched * 3 * hidden * inter * 9 / 16) + experts * hidden * 4 + rows * hidden * (8 if case["fold"] else 4),
            "flops": 6 * rows * top_k * hidden * inter + 2 * rows * experts * hidden}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_e4m3(v):
    """Nearest E4M3 value of float64 v, ties to even, from the format's definition."""
    a = v.abs()
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a)[1].clamp(-5, 9) - 4)
    return torch.sign(v) * (torch.round(a / step) * step).clamp_max(448.0)


def _exact_product(x, w):
    """sum over k of e4m3(x / s_x) s_x * w s_w, block by block of 128, s_x a power of two."""
    codes, scale = w
    rows, k = x.shape
    n = codes.shape[0]
    y = torch.zeros(rows, n, dtype=torch.float64, device=x.device)
    block_of = torch.arange(n, device=x.device) // 128
    for b in range(0, k, 128):
        xb = x[:, b:b + 128].double()
        amax = xb.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
        m, e = torch.frexp(amax / 448.0)
        sx = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int())
        y += (_exact_e4m3(xb / sx) @ codes[:, b:b + 128].double().T) * sx * scale[block_of, b // 128].double()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        r = s["residual"].double()
        if s["delta"] is not None:
            d = s["delta"].double()
            if s["post_weight"] is not None:
                d = d / torch.sqrt(torch.sum(d ** 2, 1, keepdim=True) / case["width"] + EPS) * s["post_weight"].double()
            r = r + s["scale"] * (d if s["gate"] is None else d * s["gate"].double())
        return [r, r / torch.sqrt(torch.sum(r ** 2, 1, keepdim=True) / case["width"] + EPS) * s["norm_weight"].double()]
    if op == "linear":
        return _exact_product(s["x"], s["w"])
    if op == "mlp":
        g, u = _exact_product(s["x"], s["gate"]), _exact_product(s["x"], s["up"])
        return _exact_product(g * torch.sigmoid(g) * u, s["down"])
    x = s["x"].double()
    score = torch.sigmoid(x @ s["router_w"].double().T)
    pick = torch.argsort(score + s["router_b"].double(), dim=1, descending=True, stable=True)[:, :case["top_k"]]
    out = torch.zeros_like(x)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    share = score.gather(1, pick)
    share = share / share.sum(1, keepdim=True) * SCALING

    def weights(name, e):
        codes, scales, scale2 = (v[e] for v in s[name])
        nib = torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1).long()
        v = grid[nib & 7] * (1 - 2 * (nib >> 3)).double()
        return v * scales.view(torch.float8_e4m3fn).double().repeat_interleave(16, 1) * scale2.double()

    for e in torch.unique(pick).tolist():
        t, slot = torch.nonzero(pick == e, as_tuple=True)
        g, u = x[t] @ weights("gate", e).T, x[t] @ weights("up", e).T
        out[t] += (g * torch.sigmoid(g) * u) @ weights("down", e).T * share[t, slot][:, None]
    return out if s["residual"] is None else s["residual"].double() + s["shared"].double() + out
