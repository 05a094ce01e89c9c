"""GPU tests of the operators around the routed experts -- block norm, block-scaled FP8 products and
gated MLP, the layer for a few tokens -- against plain implementations in 64 bits.

Tolerances are bounds, written out where they are used: `half(t)` is the largest relative error of one
rounding to type t, and every float32 sum is off by at most (roundings along the longest path) * 2^-23
of the sum of the magnitudes (2^-23 and not 2^-24: tensor cores may truncate).
"""
import math

import numpy as np
import pytest
import torch

from oracle import glmrt_oracle as O

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -23


def half(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def mods(pkg):
    import importlib
    return {m: importlib.import_module("glmrt_b200." + m) for m in ("block_norm", "fp8", "layer", "shared_expert")}


def randn(seed, *shape, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def within(got, ref, tol, what=""):
    assert got.shape == ref.shape
    d = (got.double() - ref).abs()
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / tol.clamp_min(1e-300)).max()):.3g} of the bound"


# ---- block norm ----------------------------------------------------------------------------------
def norm_ref(res, delta, nw, pw, gate, scale, eps):
    """(r, y) in 64 bits and the magnitudes |residual| + |scale * branch| that bound their errors."""
    r = res.double()
    mag = r.abs()
    if delta is not None:
        d = delta.double()
        if pw is not None:
            d = d * torch.rsqrt((d * d).mean(1, keepdim=True) + eps) * pw.double()
        if gate is not None:
            d = d * gate.double()
        r = r + scale * d
        mag = mag + (scale * d).abs()
    rs = torch.rsqrt((r * r).mean(1, keepdim=True) + eps)
    return r, r * rs * nw.double(), mag, mag * rs * nw.double().abs()


def check_norm(mods, res, delta, nw, pw=None, gate=None, scale=1.0, eps=1e-5, **kw):
    r, y, mr, my = norm_ref(res, delta, nw, pw, gate, scale, eps)
    ro, yo = mods["block_norm"].block_norm(res, delta, norm_weight=nw, post_weight=pw, gate=gate, scale=scale, eps=eps, **kw)
    # a thread adds at most 32 squares and 10 more values join: 42 roundings of a sum of positive terms,
    # halved by the root, and a handful of products: below 2^-18 of the magnitudes
    h = half(res.dtype)
    within(ro, r, h * r.abs() + 2 ** -18 * mr + 1e-38, "residual")
    within(yo, y, h * y.abs() + 2 ** -18 * my + 1e-38, "normalized")
    return ro, yo


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 6144), (3, 1), (5, 7), (2, 256), (700, 264), (1, 32768), (3, 32767), (301, 6144),
                                        (2, 1025), (299, 5001), (7, 16384), (4, 4100), (350, 12), (600, 2052), (2, 32764)])
def test_block_norm_sizes(mods, dtype, wdtype, rows, width):
    res, delta = randn(1, rows, width, std=2.0, dtype=dtype), randn(2, rows, width, dtype=dtype)
    nw, pw = 1 + randn(3, width, std=0.1), 1 + randn(4, width, std=0.1)
    nw, pw = nw.to(wdtype), pw.to(wdtype)
    check_norm(mods, res, delta, nw)
    check_norm(mods, res, delta, nw, pw, randn(5, 1, width, dtype=dtype), 0.25)
    check_norm(mods, res, delta, nw, None, randn(6, rows, 1, dtype=dtype), -1.5)
    check_norm(mods, res, delta, nw, pw, randn(7, rows, width, dtype=dtype), 1.0, eps=0.1)
    ro, _ = check_norm(mods, res, None, nw)
    assert ro is res


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float32, torch.bfloat16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,width", [(1183, 4096), (1184, 4096), (1185, 4104), (2371, 520), (4737, 256), (2368, 8192), (1300, 8200), (3001, 6144), (1279, 4100), (17000, 252), (300, 16380)])
def test_block_norm_many_rows(mods, dtype, wdtype, rows, width):
    """The forms for many rows (a ring in shared memory, narrow pieces) at their borders, with every term and in place."""
    res, delta = randn(1, rows, width, std=2.0, dtype=dtype), randn(2, rows, width, dtype=dtype)
    nw, pw = (1 + randn(3, width, std=0.1)).to(wdtype), (1 + randn(4, width, std=0.1)).to(wdtype)
    want = check_norm(mods, res, delta, nw)
    check_norm(mods, res, delta, nw, pw, randn(5, 1, width, dtype=dtype), 0.25)
    check_norm(mods, res, delta, nw, None, randn(6, rows, 1, dtype=dtype), -1.5)
    check_norm(mods, res, delta, nw, pw, randn(7, rows, width, dtype=dtype), 1.0, eps=0.1)
    check_norm(mods, res, None, nw)
    r2, d2 = res.clone(), delta.clone()
    got = mods["block_norm"].block_norm(r2, d2, norm_weight=nw, residual_out=r2, normalized=d2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pad = torch.nn.functional.pad(res, (0, 16))
    out = torch.full((rows, width + 8), 7.0, device="cuda", dtype=dtype)
    got = mods["block_norm"].block_norm(pad[:, :width], delta, norm_weight=nw, normalized=out[:, :width])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (out[:, width:] == 7).all()


def test_block_norm_beyond_32_bit_offsets(mods):
    rows, width = 350300, 6144
    few = randn(1, 1000, width, dtype=torch.bfloat16)
    nw = 1 + randn(2, width, std=0.1, dtype=torch.bfloat16)
    want = mods["block_norm"].block_norm(few.repeat(2, 1), few.repeat(2, 1), norm_weight=nw, scale=0.5)
    many = few.repeat(-(-rows // 1000), 1)[:rows]
    got = mods["block_norm"].block_norm(many, many, norm_weight=nw, scale=0.5)
    for at in range(0, rows, 1000):
        n = min(1000, rows - at)
        assert all(torch.equal(g[at:at + n], v[:n]) for g, v in zip(got, want)), at


def test_block_norm_of_the_most_rows(mods):
    """2^31 - 1 rows of one value: the last ones too."""
    rows, few = 2 ** 31 - 1, 2 ** 20
    x = randn(1, few, 1, dtype=torch.bfloat16)
    nw = torch.full((1,), 1.5, device="cuda")
    want = mods["block_norm"].block_norm(x, norm_weight=nw, eps=0.5)[1]
    y = x.double() * torch.rsqrt(x.double() ** 2 + 0.5) * 1.5
    within(want, y, (half(torch.bfloat16) + 2 ** -18) * y.abs() + 1e-38)
    got = mods["block_norm"].block_norm(x.repeat(2048, 1)[:rows], norm_weight=nw, eps=0.5)[1]
    for at in range(0, rows, 64 * few):
        part = got[at:at + 64 * few]
        assert torch.equal(part, want.repeat(64, 1)[:len(part)]), at


def test_block_norm_strides_and_alignment(mods):
    """Padded rows, rows that start off a 16-byte boundary, an expanded gate."""
    rows, width = 9, 520
    base = randn(1, rows, 3, width + 12, dtype=torch.bfloat16)
    for off in (0, 1, 4, 8):
        res, delta = base[:, 0, off:off + width], base[:, 1, off:off + width]
        out = torch.full((rows, width + 5), 7.0, device="cuda", dtype=torch.bfloat16)
        nw = (1 + randn(2, width + 1, std=0.1)).bfloat16()[1 - off % 2:][:width]
        check_norm(mods, res, delta, nw, normalized=out[:, 2:2 + width])
        assert (out[:, :2] == 7).all() and (out[:, 2 + width:] == 7).all()
    gate = randn(3, 1, 1, dtype=torch.bfloat16)
    check_norm(mods, base[:, 0, :width], base[:, 1, :width], nw, gate=gate.expand(rows, width))


@pytest.mark.parametrize("which", ["residual", "delta"])
def test_block_norm_in_place(mods, which):
    res, delta, nw = randn(1, 400, 1000, dtype=torch.bfloat16), randn(2, 400, 1000, dtype=torch.bfloat16), 1 + randn(3, 1000, std=.1)
    want = mods["block_norm"].block_norm(res, delta, norm_weight=nw)
    r2, d2 = res.clone(), delta.clone()
    kw = {"residual_out": r2, "normalized": d2} if which == "residual" else {"residual_out": d2, "normalized": r2}
    got = mods["block_norm"].block_norm(r2, d2, norm_weight=nw, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = res.clone()
    assert torch.equal(mods["block_norm"].block_norm(x, norm_weight=nw, normalized=x)[1],
                       mods["block_norm"].block_norm(res, norm_weight=nw)[1])


def test_block_norm_zero_rows_inf_and_nan_stay_in_their_rows(mods):
    res, nw = randn(1, 6, 1024), torch.ones(1024, device="cuda")
    delta = randn(2, 6, 1024)
    res[1], delta[1] = 0, 0
    res[2, 5] = float("inf")
    res[3, 7] = float("nan")
    ro, y = mods["block_norm"].block_norm(res, delta, norm_weight=nw)
    assert (y[1] == 0).all() and y[2, 5].isnan() and (y[2, :5] == 0).all() and y[3].isnan().all()
    r, yr, mr, my = norm_ref(res[4:], delta[4:], nw, None, None, 1.0, 1e-5)
    within(y[4:], yr, half(torch.float32) * yr.abs() + 2 ** -18 * my)


def test_block_norm_does_not_depend_on_the_batch_or_the_stream(mods):
    res, delta, nw = randn(1, 5, 6144, dtype=torch.bfloat16), randn(2, 5, 6144, dtype=torch.bfloat16), 1 + randn(3, 6144, std=.1)
    r, y = mods["block_norm"].block_norm(res, delta, norm_weight=nw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        r2, y2 = mods["block_norm"].block_norm(res[:2], delta[:2], norm_weight=nw)
    side.synchronize()
    assert torch.equal(y2, y[:2]) and torch.equal(r2, r[:2])


# ---- FP8 products --------------------------------------------------------------------------------
def pow2(e):
    """2^e, exact (the device's pow and log2 are not)."""
    return torch.ldexp(torch.ones(e.shape, dtype=torch.float64, device=e.device), e)


def floor_log2(v):
    return torch.frexp(v)[1] - 1


def ceil_log2(v):
    m, e = torch.frexp(v)
    return e - (m == 0.5).int()


def rows_ref(x):
    """The quantiser in 64 bits: (codes' values, scales [rows, blocks])."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(rows, -1, 128)
    s = pow2(ceil_log2(b.abs().amax(-1).clamp_min(2.0 ** -100) / 448.0))
    v = b / s[..., None]
    step = pow2(floor_log2(v.abs().clamp_min(2.0 ** -6)) - 3)
    q = torch.round(v / step) * step
    return q.view(rows, -1)[:, :k], s


def weight_ref(codes, scales):
    n, k = codes.shape
    return codes.double() * scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def product_ref(x, w):
    """y and the sum of magnitudes, in 64 bits."""
    q, s = rows_ref(x)
    xq = q * s.repeat_interleave(128, 1)[:, :x.shape[1]]
    return xq @ w.T, xq.abs() @ w.abs().T


def roundings(k):
    # 32 products of one instruction, 4 instructions a block, one addition per block, 8 partial sums joined
    return 32 + 4 + math.ceil(k / 128) + 8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 128), (5, 144), (130, 2000), (1, 6144)])
def test_fp8_row_codes_and_scales_are_exact(mods, dtype, rows, k):
    x = randn(k + rows, rows, k, dtype=dtype)
    x[0, :] *= 2.0 ** -70
    x[-1, 0] = 448.0 * 64                       # exactly at the border between two scales
    q, s = rows_ref(x)
    codes, scales = mods["fp8"].quantize_rows(x)
    assert torch.equal(scales.T.double(), s) and torch.equal(codes.double(), q)
    wide = torch.cat([x, x], 1)                 # rows with a stride
    c2, s2 = mods["fp8"].quantize_rows(wide[:, :k])
    assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2, scales)


def test_fp8_row_blocks_of_zeros_tiny_values_and_non_finite_values(mods):
    x = randn(3, 6, 384, dtype=torch.float32)
    x[0] = 0
    x[1, :128] = 2.0 ** -120
    x[2, 130] = float("inf")
    x[3, 300] = float("nan")
    x[4] = 3.0e38
    codes, scales = mods["fp8"].quantize_rows(x)
    assert (codes[:2].double()[:, :128] == 0).all() and scales.T[0].isfinite().all()
    assert scales.T[2].isnan().tolist() == [False, True, False] and scales.T[3].isnan().tolist() == [False, False, True]
    assert torch.equal(codes[4].double() * float(scales[0, 4]), rows_ref(x[4:5])[0][0] * rows_ref(x[4:5])[1][0, 0])
    w = mods["fp8"].quantize_weight(randn(4, 40, 384, std=0.02))
    y = mods["fp8"].block_linear(x.bfloat16().clamp(-1e30, 1e30).nan_to_num_(0.0).index_fill_(0, torch.tensor([2], device="cuda"), float("nan")), *w)
    assert y[2].isnan().all() and y[[0, 1, 3, 4, 5]].isfinite().all()
    assert (y[0] == 0).all()


LINEAR = [(1, 1, 16), (1, 4096, 6144), (2, 128, 128), (3, 140, 16384), (4, 6144, 2064), (4, 20000, 272), (5, 200, 400), (7, 130, 272), (16, 257, 2048), (17, 384, 144), (33, 1500, 2000),
          (64, 640, 6144), (65, 96, 512), (128, 512, 1040), (129, 1000, 256), (197, 1500, 2000), (300, 6144, 2048),
          (777, 516, 400), (2048, 768, 1024), (1, 8, 16384), (520, 4100, 144)]


@pytest.mark.parametrize("rows,n,k", LINEAR)
def test_fp8_block_linear(mods, rows, n, k):
    x = randn(rows + n, rows, k, dtype=torch.bfloat16)
    x *= torch.pow(2.0, torch.randint(-6, 7, (rows, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(1))).bfloat16()
    codes, scales = mods["fp8"].quantize_weight(randn(k, n, k, std=0.02) * torch.linspace(0.2, 5, k, device="cuda"))
    y, mag = product_ref(x, weight_ref(codes, scales))
    f32 = roundings(k) * ULP * mag
    within(mods["fp8"].block_linear(x, codes, scales, out_dtype=torch.float32), y, f32 + 1e-38, "float32")
    out = torch.full((rows + 1, n), 3.0, device="cuda", dtype=torch.bfloat16)      # what lies behind stays
    got = mods["fp8"].block_linear(x, codes, scales, out=out[:rows])
    within(got, y, half(torch.bfloat16) * (y.abs() + f32) + f32, "bfloat16")
    assert (out[rows] == 3).all()
    assert torch.equal(mods["fp8"].block_linear(x, codes, scales), got), "two calls differ"
    pad = torch.nn.functional.pad(x, (3, 5))
    assert torch.equal(mods["fp8"].block_linear(pad[:, 3:3 + k], codes.view(torch.uint8), scales), got), "strided rows"


def test_fp8_block_linear_empty_rows_and_weight_extremes(mods):
    codes, scales = mods["fp8"].quantize_weight(randn(1, 200, 256))
    assert mods["fp8"].block_linear(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), codes, scales).shape == (0, 200)
    scales[1, 1] = 0.0
    codes.view(torch.uint8)[3, 5] = 0x7f              # NaN code
    codes.view(torch.uint8)[4] = 0x01                 # smallest subnormal
    y = mods["fp8"].block_linear(randn(2, 4, 256, dtype=torch.bfloat16), codes, scales)
    assert y[:, 3].isnan().all() and y.isnan().sum() == 4


@pytest.mark.parametrize("rows", [1, 40])
def test_fp8_calls_on_two_streams_and_in_a_graph(mods, rows):
    x = randn(1, rows, 2048, dtype=torch.bfloat16)
    w = mods["fp8"].quantize_weight(randn(2, 1024, 2048, std=0.02))
    want = mods["fp8"].block_linear(x, *w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [mods["fp8"].block_linear(x, *w) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    xin = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mods["fp8"].block_linear(xin, *w)
    for _ in range(2):
        xin.copy_(x)
        g.replay()
        assert torch.equal(out, want)
        xin.zero_()


@pytest.mark.parametrize("rows,n,k", [(350300, 16, 6144), (140001, 16384, 16)])
def test_fp8_linear_beyond_32_bit_offsets(mods, rows, n, k):
    """More than 2^31 values in the rows, or in the output: every row as it comes out among a few."""
    assert max(rows * n, rows * k) > 2 ** 31
    few = randn(1, 1000, k, dtype=torch.bfloat16)
    w = mods["fp8"].quantize_weight(randn(2, n, k, std=0.02))
    want = mods["fp8"].block_linear(few.repeat(2, 1), *w)[:1000]       # (on the many rows' kernel)
    got = mods["fp8"].block_linear(few.repeat(-(-rows // 1000), 1)[:rows], *w)
    for at in range(0, rows, 1000):
        assert torch.equal(got[at:at + 1000], want[:min(1000, rows - at)]), at


def mlp_ref(x, gate, up, down):
    """y, and a bound on what float32 can change: sums, and codes whose border is within the error."""
    (g, mg), (u, mu) = product_ref(x, weight_ref(*gate)), product_ref(x, weight_ref(*up))
    k, inter = x.shape[1], gate[0].shape[0]
    act = g * torch.sigmoid(g) * u
    # |silu'| <= 1.1; the fast exponential and division add a few units in the last place
    err = 1.1 * roundings(k) * ULP * mg * u.abs() + (g * torch.sigmoid(g)).abs() * roundings(k) * ULP * mu + 2 ** -17 * act.abs()
    q, s = rows_ref(act)
    sw = s.repeat_interleave(128, 1)[:, :inter]
    step = pow2(floor_log2((act / sw).abs().clamp_min(2.0 ** -6)) - 3) * sw
    # a code may change by one step where the error reaches the border; a block's scale may double where its
    # largest value is within the error of the border: then subnormal codes are rounded to twice the step
    near = ((act - q * sw).abs() + err >= step / 2).double() * (2 * step)
    wd = weight_ref(*down)
    xq = q * sw
    pad = torch.nn.functional.pad(act.abs(), (0, -inter % 128)).view(len(x), -1, 128).amax(-1)
    perr = torch.nn.functional.pad(err, (0, -inter % 128)).view(len(x), -1, 128).amax(-1)
    edge = torch.pow(2.0, torch.round(torch.log2(pad.clamp_min(1e-300) / 448))) * 448
    flip = ((pad - edge).abs() <= perr).repeat_interleave(128, 1)[:, :inter].double() * (2.0 ** -9 * sw + 2.0 ** -4 * act.abs())
    return xq @ wd.T, (near + flip) @ wd.abs().T + roundings(inter) * ULP * (xq.abs() @ wd.abs().T)


@pytest.mark.parametrize("rows,hidden,inter", [(1, 6144, 2048), (1, 128, 128), (3, 256, 144), (4, 8192, 1536), (5, 1024, 400), (16, 1024, 400), (40, 528, 640),
                                               (64, 6144, 2048), (65, 512, 272), (300, 2048, 1040), (1030, 1536, 768)])
def test_fp8_gated_mlp(mods, rows, hidden, inter):
    x = randn(rows, rows, hidden, dtype=torch.bfloat16)
    gate, up = (mods["fp8"].quantize_weight(randn(s, inter, hidden, std=0.03)) for s in (1, 2))
    down = mods["fp8"].quantize_weight(randn(3, hidden, inter, std=0.03))
    y, f32 = mlp_ref(x, gate, up, down)
    got = mods["fp8"].gated_mlp(x, *gate, *up, *down)
    within(got, y, half(torch.bfloat16) * (y.abs() + f32) + f32 + 1e-38)
    # the bound above allows changed codes; on the whole they must be rare
    assert float((got.double() - y).norm() / y.norm()) <= half(torch.bfloat16)
    assert torch.equal(mods["fp8"].gated_mlp(x, *gate, *up, *down), got)
    wide = torch.nn.functional.pad(x, (0, 8))
    out = torch.empty_like(got)
    assert mods["fp8"].gated_mlp(wide[:, :hidden], *gate, *up, *down, out=out) is out and torch.equal(out, got)
    assert torch.equal(mods["fp8"].gated_mlp(x, *gate, *up, *down, out=x), got), "in the rows' place"


# ---- the layer for a few tokens ------------------------------------------------------------------
GRID = (0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6)


def layer_weights(ref):
    """[E, rows, cols] float64 weights of a synthetic quantised layer."""
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    out = []
    for t, (c, s) in enumerate(((ref.gate, ref.gate_s), (ref.up, ref.up_s), (ref.down, ref.down_s))):
        sc = torch.from_numpy(np.ascontiguousarray(s)).cuda().view(torch.float8_e4m3fn).double()
        out.append(grid[torch.from_numpy(np.ascontiguousarray(c)).cuda().long()] * sc.repeat_interleave(16, -1)
                   * torch.from_numpy(ref.scale2[:, t].astype(np.float64)).cuda()[:, None, None])
    return out


def few_ref(weights, x, idx, w, residual=None, shared=None):
    """out and a bound on its error before the last rounding."""
    gate, up, down = weights
    out, err = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    x = x.double()
    hidden, inter = x.shape[1], gate.shape[1]
    # a sum of k products: 16 of one instruction, k / 16 instructions at worst in one chain, 16 partial sums joined
    c1, c2 = (16 + hidden // 16 + 16) * ULP, (16 + idx.shape[1] * inter // 16 + 16 + 16) * ULP
    for t in range(x.shape[0]):
        for s in range(idx.shape[1]):
            e = int(idx[t, s])
            if not 0 <= e < gate.shape[0]:
                continue
            g, u = gate[e] @ x[t], up[e] @ x[t]
            mg, mu = gate[e].abs() @ x[t].abs(), up[e].abs() @ x[t].abs()
            silu = g * torch.sigmoid(g)
            act = float(w[t, s]) * silu * u
            # float32 sums, the fast exponential and division, and the rounding to fp16 (2^-11)
            ea = abs(float(w[t, s])) * (1.1 * c1 * mg * u.abs() + silu.abs() * c1 * mu) + (2 ** -17 + 2 ** -11) * act.abs()
            out[t] += down[e] @ act
            err[t] += down[e].abs() @ (ea + c2 * act.abs())
    for more in (shared, residual):
        if more is not None:
            out, err = out + more.double(), err + 2 * ULP * more.double().abs()
    return out, err


def check_few(layer, weights, x, residual=None, shared=None):
    got, idx, w = layer.forward_few(x, residual_bf16=residual, shared_delta_bf16=shared, want_routes=True)
    layer.check()
    ref, err = few_ref(weights, x, idx.cpu(), w.cpu(), residual, shared)
    within(got, ref, half(torch.bfloat16) * (ref.abs() + err) + err + 1e-38)
    return got, idx, w


def make_layer(mods, ref, top_k, engine="tc", max_tokens=16):
    h, i, e = ref.dims
    layer = mods["layer"].MoeLayer(h, i, e, top_k, max_tokens=max_tokens, engine=engine)
    layer.load_quantized_layer(ref)
    return layer


SHAPES = [(256, 256, 4, 1), (512, 256, 16, 4), (1280, 768, 12, 6), (2048, 512, 40, 8), (256, 1280, 3, 3), (768, 256, 20, 16)]


@pytest.mark.parametrize("engine", ["simt", "tc"])
@pytest.mark.parametrize("shape", SHAPES)
def test_few_matches_64_bits(mods, engine, shape):
    h, i, e, top_k = shape
    ref = O.make_layer(h + i, h, i, e)
    layer, weights = make_layer(mods, ref, top_k, engine), layer_weights(ref)
    for rows in (1, 2, 3, 7, 8, 9, 16):
        x = randn(rows, rows, h, dtype=torch.bfloat16)
        got, idx, w = check_few(layer, weights, x)
        fwd_idx = layer.forward(x, want_routes=True)[1]
        assert torch.equal(idx.sort(1).values, fwd_idx.sort(1).values)
        score = torch.sigmoid(x.double() @ torch.from_numpy(ref.router_w).cuda().double().T)
        picked = score.gather(1, idx.long())
        # scores: a float32 dot product of h terms and the exponential; weights: their share of the sum
        share = picked / picked.sum(1, keepdim=True) * 2.5
        assert float((w.double() - share).abs().max()) <= 2.5 * 2 ** -14
        check_few(layer, weights, x, randn(8, rows, h, std=2, dtype=torch.bfloat16), randn(9, rows, h, dtype=torch.bfloat16))
    layer.close()


@pytest.mark.parametrize("engine", ["simt", "tc"])
def test_few_with_given_routes(mods, engine):
    """No route at all, one expert for every row, an expert twice in a row, zero and negative weights."""
    ref = O.make_layer(5, 512, 256, 10)
    layer, weights = make_layer(mods, ref, 4, engine), layer_weights(ref)
    x = randn(1, 16, 512, dtype=torch.bfloat16)
    w = randn(2, 16, 4).abs() + 0.1
    cases = {"none": torch.full((16, 4), -1), "one": torch.full((16, 4), 3),
             "twice": torch.tensor([[1, 1, 2, -1]]).repeat(16, 1), "mixed": torch.arange(64).view(16, 4) % 11 - 1}
    res = randn(3, 16, 512, dtype=torch.bfloat16)
    for name, idx in cases.items():
        for wt in (w, w * torch.tensor([1, 0, -2, 1e-4], device="cuda")):
            got = layer.forward_few_routed(x, idx.cuda(), wt, residual_bf16=res)
            layer.check()
            out, err = few_ref(weights, x, idx, wt.cpu(), res)
            within(got, out, half(torch.bfloat16) * (out.abs() + err) + err, name)
            if name == "none":
                assert torch.equal(got, res)
    layer.close()


@pytest.mark.parametrize("engine", ["simt", "tc"])
def test_few_reports_an_expert_outside_the_layer_and_recovers(mods, pkg, engine):
    from glmrt_b200 import native as N
    ref = O.make_layer(5, 512, 256, 10)
    layer, weights = make_layer(mods, ref, 4, engine), layer_weights(ref)
    x, w = randn(1, 3, 512, dtype=torch.bfloat16), torch.ones(3, 4, device="cuda")
    idx = torch.tensor([[0, 1, 10, 2], [3, 4, 5, 6], [7, 8, 9, 0]])
    got = layer.forward_few_routed(x, idx.cuda(), w)
    with pytest.raises(N.GlmrtError, match="outside the layer"):
        layer.check()
    out, err = few_ref(weights, x, idx, w.cpu())
    within(got, out, half(torch.bfloat16) * (out.abs() + err) + err)
    check_few(layer, weights, x)
    layer.close()


@pytest.mark.parametrize("engine", ["simt", "tc"])
def test_few_small_large_and_non_finite_rows(mods, engine):
    ref = O.make_layer(6, 768, 512, 8)
    layer, weights = make_layer(mods, ref, 2, engine), layer_weights(ref)
    x = randn(1, 9, 768, dtype=torch.bfloat16)
    x[0] *= 2.0 ** -60
    x[1] *= 2.0 ** 40
    x[2, ::2] *= 2.0 ** -30
    x[3] = 0
    idx, w = torch.arange(18).view(9, 2) % 8, torch.ones(9, 2, device="cuda")
    out, err = few_ref(weights, x, idx, w.cpu())
    got = layer.forward_few_routed(x, idx.cuda(), w)
    within(got, out, half(torch.bfloat16) * (out.abs() + err) + err + 2.0 ** -133)   # bf16's smallest step
    x[5, 3] = float("nan")
    x[7, 9] = float("inf")
    bad = layer.forward_few_routed(x, idx.cuda(), w)
    keep = [r for r in range(9) if r not in (5, 7)]
    assert torch.equal(bad[keep], got[keep]) and bad[5].isnan().all() and not bad[7].isfinite().any()
    layer.close()


def test_few_rows_do_not_depend_on_their_batch_and_repeat(mods):
    ref = O.make_layer(7, 1024, 512, 12)
    layer = make_layer(mods, ref, 4)
    x = randn(1, 16, 1024, dtype=torch.bfloat16)
    want = layer.forward_few(x)
    for _ in range(5):
        assert torch.equal(layer.forward_few(x), want)
    for rows in (1, 2, 3, 4, 5, 7, 8, 9, 15):
        assert torch.equal(layer.forward_few(x[:rows]), want[:rows]), rows
    layer.check()
    layer.close()


def test_few_in_place_of_residual_and_after_forward(mods):
    """The output in the residual's place, W4A4 forwards in between, and a lane of its own."""
    ref = O.make_layer(8, 512, 256, 16)
    layer = make_layer(mods, ref, 4, max_tokens=512)
    x, res, sh = (randn(s, 5, 512, dtype=torch.bfloat16) for s in (1, 2, 3))
    big = randn(4, 400, 512, dtype=torch.bfloat16)
    want_big = layer.forward(x).clone()
    want = layer.forward_few(x, residual_bf16=res, shared_delta_bf16=sh)
    layer.forward(big)
    r2, s2 = res.clone(), sh.clone()
    assert torch.equal(layer.forward_few(x, out=r2, residual_bf16=r2, shared_delta_bf16=sh), want)
    assert torch.equal(layer.forward_few(x, out=s2, residual_bf16=res, shared_delta_bf16=s2), want)
    assert torch.equal(layer.forward(x), want_big)
    lane, stacked = layer.create_lane(3), layer.create_stacked()
    stacked.load_quantized_layer(O.make_layer(9, 512, 256, 16))
    first = layer.forward_few(x[:3])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [lane.forward_few(x[:3]) for _ in range(4)]
    mine = [layer.forward_few(x[:3]) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, first) for g in got + mine)
    other = stacked.forward_few(x[:3])
    assert not torch.equal(other, first) and torch.equal(layer.forward_few(x[:3]), first)
    for l in (lane, stacked, layer):
        l.check()
        l.close()


def test_few_replays_from_graphs_that_share_a_workspace(mods):
    ref = O.make_layer(10, 512, 256, 16)
    layer = make_layer(mods, ref, 4)
    xs = [torch.zeros(n, 512, device="cuda", dtype=torch.bfloat16) for n in (1, 6)]
    layer.forward_few(xs[1])
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.forward_few(x))
        graphs.append(g)
    for seed in range(3):
        for x, g, out in zip(xs, graphs, outs):
            x.copy_(randn(seed, *x.shape, dtype=torch.bfloat16))
            g.replay()
            got = out.clone()
            assert torch.equal(layer.forward_few(x), got)
    layer.check()
    layer.close()


def test_few_full_size_layer(mods):
    """The model's own shape, weights made on the device: against 64 bits on the experts it names."""
    h, i, e, top_k = 6144, 2048, 256, 8
    layer = mods["layer"].MoeLayer(h, i, e, top_k, max_tokens=16)
    layer.set_router(randn(1, e, h, std=0.02), randn(2, e, std=0.01))
    layer.fill_synthetic(11)
    x = randn(3, 16, h, dtype=torch.bfloat16)
    res = randn(4, 16, h, dtype=torch.bfloat16)
    got, idx, w = layer.forward_few(x, residual_bf16=res, want_routes=True)
    one, idx1, w1 = layer.forward_few(x[2:3].contiguous(), residual_bf16=res[2:3].contiguous(), want_routes=True)
    layer.check()
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    for t in (2, 15):
        experts = idx[t].tolist()
        parts = [layer.read_expert(v) for v in experts]
        weights = [torch.stack([grid[torch.from_numpy(p[j][0]).cuda().long()]
                                * torch.from_numpy(p[j][1].copy()).cuda().view(torch.float8_e4m3fn).double().repeat_interleave(16, 1) * p[j][2]
                                for p in parts]) for j in range(3)]
        out, err = few_ref(weights, x[t:t + 1], torch.arange(top_k)[None], w[t:t + 1].cpu(), res[t:t + 1])
        within(got[t:t + 1], out, half(torch.bfloat16) * (out.abs() + err) + err, f"row {t}")
        if t == 2:
            assert idx1.tolist() == idx[2:3].tolist()
            within(one, out, half(torch.bfloat16) * (out.abs() + err) + err, "alone")
    layer.close()


def test_few_refuses_what_the_wrapper_cannot_pass(mods):
    """C entry points: too many rows, an output over the rows, buffers off their boundaries."""
    import ctypes as C
    from glmrt_b200 import native as N
    layer = make_layer(mods, O.make_layer(18, 256, 256, 4), 2)
    x, out = randn(1, 17, 256, dtype=torch.bfloat16), torch.empty(17, 256, device="cuda", dtype=torch.bfloat16)
    idx, w = torch.zeros(17, 2, dtype=torch.int32, device="cuda"), torch.ones(17, 2, device="cuda")
    buf, null = lambda t, off=0, less=0: N.DeviceBuffer.of(t.data_ptr() + off, t.nbytes - off - less), N.DeviceBuffer.null()

    def status(name, hidden=buf(x), out=buf(out), idx=buf(idx), w=buf(w), residual=null, rows=4):
        a = N.FewArgs(hidden, residual, null, out, idx, w, rows)
        return layer.lib.call_status(f"glmrt_b200_moe_layer_{name}_async", layer.handle, C.byref(a), None)

    for name in ("forward_few", "forward_few_routed"):
        assert status(name) == 0
        for bad in (dict(rows=17), dict(rows=0), dict(hidden=null), dict(out=null), dict(out=buf(x)), dict(out=buf(x, 512)), dict(hidden=buf(x, 8)),
                    dict(out=buf(out, 2)), dict(residual=buf(out, 512)), dict(idx=buf(idx, 2)), dict(w=buf(w, 1))):
            assert status(name, **bad) == 1, (name, bad)
        for small in (dict(hidden=buf(x, 0, x.nbytes - 4 * 512 + 1)), dict(out=buf(out, 0, out.nbytes - 4 * 512 + 1)), dict(idx=buf(idx, 0, idx.nbytes - 31)),
                      dict(w=buf(w, 0, w.nbytes - 31))):
            assert status(name, **small) == 2, (name, small)
    assert status("forward_few", idx=null, w=null) == 0
    assert status("forward_few_routed", idx=null) == 1 and status("forward_few_routed", w=null) == 1
    layer.check()
    layer.close()


@pytest.mark.parametrize("engine", ["simt", "tc"])
def test_few_writes_either_route_buffer_alone(mods, engine):
    """Through C: indices, weights, both or neither may be asked for."""
    import ctypes as C
    from glmrt_b200 import native as N
    layer = make_layer(mods, O.make_layer(19, 512, 256, 12), 3, engine)
    x = randn(1, 5, 512, dtype=torch.bfloat16)
    want, want_idx, want_w = layer.forward_few(x, want_routes=True)
    buf, null = lambda t: N.DeviceBuffer.of(t.data_ptr(), t.nbytes), N.DeviceBuffer.null()
    for has_idx, has_w in ((True, True), (True, False), (False, True), (False, False)):
        out = torch.zeros_like(x)
        idx, w = torch.full((6, 3), 77, dtype=torch.int32, device="cuda"), torch.full((6, 3), 77.0, device="cuda")
        a = N.FewArgs(buf(x), null, null, buf(out), buf(idx) if has_idx else null, buf(w) if has_w else null, 5)
        assert layer.lib.call_status("glmrt_b200_moe_layer_forward_few_async", layer.handle, C.byref(a), None) == 0
        layer.check()
        assert engine == "simt" or layer.stats().launches_last_forward == 1, "not the one-kernel form"
        assert torch.equal(out, want), (has_idx, has_w)
        assert torch.equal(idx[:5], want_idx) if has_idx else (idx[:5] == 77).all()
        assert torch.equal(w[:5], want_w) if has_w else (w[:5] == 77).all()
        assert (idx[5] == 77).all() and (w[5] == 77).all()
    layer.close()


def test_few_expired_wait_is_reported_once_and_healed(mods):
    """What a barrier that ran out leaves (the word set, the count short) outlives the calls after it: they leave their
    outputs alone, the check reports it, and then everything is right again.  The state is set from the host."""
    from glmrt_b200 import native as N
    import ctypes as C
    ref = O.make_layer(20, 512, 256, 16)
    layer = make_layer(mods, ref, 4, "tc-ordered", max_tokens=300)      # (whose large batches repeat bit by bit)
    stacked = layer.create_stacked()                    # shares the workspace
    stacked.load_quantized_layer(ref)
    lane = layer.create_lane(3)                         # has its own
    x, big = randn(1, 3, 512, dtype=torch.bfloat16), randn(2, 300, 512, dtype=torch.bfloat16)
    want, idx, w = layer.forward_few(x, want_routes=True)
    want_routed = layer.forward_few_routed(x, idx, w)
    want_big = layer.forward(big)
    b = N.DeviceBuffer()
    layer.lib.call("glmrt_b200_moe_layer_debug_buffer", layer.handle, C.c_uint32(N.DEBUG["COUNTERS"]), C.byref(b))
    for short in (1, 7, 147):
        layer.check()
        torch.cuda.synchronize()
        words = np.array([2 ** 32 - short, 1], np.uint32)     # barrier count, expired
        layer.lib.call("glmrt_copy_h2d", N.DeviceBuffer.of(b.ptr + 32, 8), C.c_void_p(words.ctypes.data), C.c_size_t(8))
        out = torch.full_like(x, 7.0)
        for l in (layer, stacked, layer):
            l.forward_few(x, out=out, residual_bf16=x)
            l.forward_few_routed(x, idx, w, out=out)
            assert torch.equal(layer.forward(big), want_big)
        torch.cuda.synchronize()
        assert (out == 7).all()
        assert torch.equal(lane.forward_few(x), want)
        lane.check()
        assert layer.stats().device_error == 1
        with pytest.raises(N.GlmrtError, match="bounded wait"):
            layer.check()
        layer.check()
        assert layer.debug("COUNTERS", np.uint32)[8:10].tolist() == [0, 0]
        for l in (layer, stacked):
            assert torch.equal(l.forward_few(x), want) and torch.equal(l.forward_few_routed(x, idx, w), want_routed)
    layer.check()
    for l in (lane, stacked, layer):
        l.close()


@pytest.mark.parametrize("engine", ["simt", "tc"])
@pytest.mark.parametrize("experts", [20, 300])
def test_few_picks_the_experts_that_the_router_picks(mods, engine, experts):
    """Equal scores go to the lower id; scores or biases that are not finite are never picked, and slots without a
    candidate name expert 0 with weight 0: the rule of the layer's router, whose routes `forward` returns."""
    h, top_k = 512, 6
    ref = O.make_layer(21, h, 256, experts)
    w0, b0 = torch.from_numpy(ref.router_w).cuda(), torch.from_numpy(ref.bias).cuda()
    layer, weights = make_layer(mods, ref, top_k, engine), layer_weights(ref)
    x = randn(1, 16, h, dtype=torch.bfloat16)
    inf, nan = float("inf"), float("nan")

    def equal_rows(w, b):               # every expert the same score
        w[:], b[:] = w[0], 0.0

    def pairs(w, b):                    # neighbours share theirs
        w[1::2], b[1::2] = w[0::2], b[0::2]

    def zero_and_above(w, b):           # sums of score and bias at zero, and one quarter
        w[:], b[:] = 0.0, -0.5
        b[experts // 2:] = -0.25

    def infinite(w, b):
        b[3], b[5], w[7, 2], w[8] = inf, -inf, nan, inf
        b[experts - 1] = nan

    def three_left(w, b):
        b[:], b[[2, 9, experts - 2]] = -inf, torch.tensor([0.1, 0.0, 0.2], device="cuda")

    def zero_and_one_left(w, b):
        b[:], b[[0, 11]] = nan, torch.tensor([0.1, 0.2], device="cuda")

    def none_left(w, b):
        b[:] = inf

    for change in (equal_rows, pairs, zero_and_above, infinite, three_left, zero_and_one_left, none_left):
        w, b = w0.clone(), b0.clone()
        change(w, b)
        layer.set_router(w, b)
        for rows in (1, 2, 16):
            want_idx, want_w = layer.forward(x[:rows], want_routes=True)[1:]
            got, idx, rw = check_few(layer, weights, x[:rows])
            assert engine == "simt" or layer.stats().launches_last_forward == 1, "not the one-kernel form"
            assert torch.equal(idx, want_idx), (change.__name__, rows)
            # weights: float32 logits of h terms in another order, their exponential, and their share of the sum
            assert float((rw - want_w).abs().max()) <= 2.5 * 2 ** -14, (change.__name__, rows)
            assert torch.equal(layer.forward_few_routed(x[:rows], idx, rw), got), (change.__name__, rows)
    layer.set_router(w0, b0)
    bad = x.clone()
    bad[2, 5], bad[4, 7] = nan, -inf
    got, idx, rw = layer.forward_few(bad, want_routes=True)
    want, want_idx, want_w = layer.forward_few(x, want_routes=True)
    assert (idx[2] == 0).all() and (rw[2] == 0).all() and got[2].isnan().all() and not got[4].isfinite().any()
    keep = [r for r in range(16) if r not in (2, 4)]
    assert torch.equal(got[keep], want[keep]) and torch.equal(idx[keep], want_idx[keep]) and torch.equal(rw[keep], want_w[keep])
    layer.close()


def test_few_refuses_route_buffers_over_others(mods):
    """Through C: returned routes over the rows, the residual, the output or each other; an output over given routes."""
    import ctypes as C
    from glmrt_b200 import native as N
    layer = make_layer(mods, O.make_layer(22, 512, 256, 12), 3)
    x, res, sh = (randn(s, 4, 512, dtype=torch.bfloat16) for s in (1, 2, 3))
    out, idx, w = torch.empty_like(x), torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.ones(4, 3, device="cuda")
    buf = lambda t, off=0: N.DeviceBuffer.of(t.data_ptr() + off, t.nbytes - off)

    def status(name, **kw):
        b = {**dict(hidden=buf(x), residual=buf(res), shared=buf(sh), out=buf(out), idx=buf(idx), w=buf(w)), **kw}
        return layer.lib.call_status(f"glmrt_b200_moe_layer_{name}_async", layer.handle, C.byref(N.FewArgs(*b.values(), 4)), None)

    assert status("forward_few") == 0 and status("forward_few_routed") == 0
    for t in (x, res, sh, out):
        for name in ("idx", "w"):
            for off in (0, 512, t.nbytes - 48):
                assert status("forward_few", **{name: buf(t, off)}) == 1 and "overlaps" in layer.lib.last_error(), (name, off)
    assert status("forward_few", w=buf(idx)) == 1 and "overlaps" in layer.lib.last_error()
    for name in ("idx", "w"):
        assert status("forward_few_routed", **{name: buf(out, 1024)}) == 1 and "overlaps" in layer.lib.last_error()
    both = torch.zeros(2, 4, 3, dtype=torch.int32, device="cuda")           # side by side is apart
    assert status("forward_few", idx=buf(both[0]), w=buf(both[1])) == 0
    layer.check()
    layer.close()


def test_few_many_experts_and_most_routes(mods):
    """More than 256 experts, 16 slots, every row its own experts: 256 entries at once."""
    h, i, e, top_k = 512, 256, 330, 16
    ref = O.make_layer(13, h, i, e)
    layer, weights = make_layer(mods, ref, top_k), layer_weights(ref)
    x = randn(1, 16, h, dtype=torch.bfloat16)
    _, idx, _ = check_few(layer, weights, x)
    assert torch.equal(idx.sort(1).values, layer.forward(x, want_routes=True)[1].sort(1).values)
    idx, w = torch.arange(256).view(16, 16) + 70, randn(2, 16, 16).abs() + 0.1
    got = layer.forward_few_routed(x, idx.cuda(), w)
    layer.check()
    out, err = few_ref(weights, x, idx, w.cpu())
    within(got, out, half(torch.bfloat16) * (out.abs() + err) + err)
    layer.close()


def test_few_shapes_beyond_the_fused_kernel(mods):
    """Rows too long for the fused kernel's shared memory: right, and the same for one row as among others."""
    h, i, e = 24576, 256, 3
    ref = O.make_layer(14, h, i, e)
    layer, weights = make_layer(mods, ref, 2), layer_weights(ref)
    x = randn(1, 5, h, dtype=torch.bfloat16)
    got, idx, w = check_few(layer, weights, x)
    for r in range(5):
        assert torch.equal(layer.forward_few_routed(x[r:r + 1], idx[r:r + 1], w[r:r + 1]), got[r:r + 1])
    layer.close()


def test_few_weights_beyond_4_gib(mods):
    """Stacks of more than 2^32 bytes: the experts at their end, against 64 bits."""
    h, i, e = 6144, 2048, 720
    layer = mods["layer"].MoeLayer(h, i, e, 2, max_tokens=4)
    layer.set_router(randn(1, e, h, std=0.02), randn(2, e, std=0.01))
    layer.fill_synthetic(15)
    assert e * h * i // 2 > 2 ** 32
    x, w = randn(3, 3, h, dtype=torch.bfloat16), torch.ones(3, 2, device="cuda")
    experts = [e - 1, 0, 683, e - 2]
    pick = torch.tensor([[0, 1], [2, 3], [3, 0]])
    got = layer.forward_few_routed(x, torch.tensor(experts)[pick].cuda(), w)
    layer.check()
    parts = [layer.read_expert(v) for v in experts]
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    weights = [torch.stack([grid[torch.from_numpy(p[j][0]).cuda().long()]
                            * torch.from_numpy(p[j][1].copy()).cuda().view(torch.float8_e4m3fn).double().repeat_interleave(16, 1) * p[j][2]
                            for p in parts]) for j in range(3)]
    out, err = few_ref(weights, x, pick, w.cpu())
    within(got, out, half(torch.bfloat16) * (out.abs() + err) + err)
    layer.close()


def test_operators_on_three_streams_at_once(mods):
    """Two lanes of a layer, 8-bit products and norms side by side: everybody gets what they get alone."""
    ref = O.make_layer(16, 1024, 512, 32)
    layer = make_layer(mods, ref, 4)
    lane = layer.create_lane(16)
    x, rows = randn(1, 7, 1024, dtype=torch.bfloat16), randn(2, 3000, 4096, dtype=torch.bfloat16)
    w = mods["fp8"].quantize_weight(randn(3, 1000, 4096, std=0.02))
    few, lin = layer.forward_few(x), {m: mods["fp8"].block_linear(rows[:m], *w) for m in (2, 40, 3000)}
    nw = 1 + randn(4, 4096, std=0.1)
    norm = mods["block_norm"].block_norm(rows, rows, norm_weight=nw)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(8):
        for s, l in zip(streams, (layer, lane)):
            with torch.cuda.stream(s):
                got.append((l.forward_few(x), few))
        with torch.cuda.stream(streams[2]):
            got += [(mods["fp8"].block_linear(rows[:m], *w), lin[m]) for m in lin]
            got += zip(mods["block_norm"].block_norm(rows, rows, norm_weight=nw), norm)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g, want in got)
    for l in (lane, layer):
        l.check()
        l.close()
    import importlib
    importlib.import_module("glmrt_b200.launch").check()


def test_operators_from_two_host_threads(mods):
    """Two threads, a stream and a lane each, sizes that take different kernels; one thread's refused calls between."""
    import threading
    from glmrt_b200 import native as N
    ref = O.make_layer(17, 512, 256, 16)
    layer = make_layer(mods, ref, 4)
    lanes = [layer, layer.create_lane(16)]
    w = mods["fp8"].quantize_weight(randn(1, 700, 512, std=0.05))
    xs = {m: randn(m, m, 512, dtype=torch.bfloat16) for m in (1, 6, 16, 90, 1500)}
    nw = torch.ones(512, device="cuda")

    def work(l):
        out = []
        for m, x in xs.items():
            out += [mods["fp8"].block_linear(x, *w), *mods["block_norm"].block_norm(x, x, norm_weight=nw)]
            if m <= 16:
                out.append(l.forward_few(x))
        return out

    want = work(layer)
    torch.cuda.synchronize()
    failures = []

    def run(l, refused):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = work(l)
                if refused:
                    try:
                        mods["fp8"].block_linear(xs[6], *w, out=torch.empty(6, 699, device="cuda", dtype=torch.bfloat16))
                        failures.append("not refused")
                    except ValueError:
                        pass
                    try:
                        l.forward_few(xs[16].repeat(2, 1))
                        failures.append("not refused")
                    except N.GlmrtError:
                        pass
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(g, v) for g, v in zip(got, want)):
                    failures.append("differs")

    threads = [threading.Thread(target=run, args=(l, i == 1)) for i, l in enumerate(lanes)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for l in reversed(lanes):
        l.check()
        l.close()


def test_first_calls_of_a_process_may_be_captured(pkg):
    """Nothing has to run before a capture: every operator's first call is inside one."""
    import os
    import subprocess
    import sys
    code = """
import torch
from __graft_entry__ import load_package
load_package()
from glmrt_b200 import fp8
from glmrt_b200.block_norm import block_norm
x = {m: torch.ones(m, 6144, device="cuda", dtype=torch.bfloat16) for m in (1, 40, 100, 2000)}
w = fp8.quantize_weight(torch.linspace(-1, 1, 640 * 6144, device="cuda").view(640, 6144))
d = fp8.quantize_weight(torch.linspace(-1, 1, 6144 * 640, device="cuda").view(6144, 640))
nw = torch.ones(6144, device="cuda")
def run():
    return [t for v in x.values() for t in (fp8.block_linear(v, *w), fp8.gated_mlp(v, *w, *w, *d), *block_norm(v, v, norm_weight=nw))]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


def test_first_few_row_calls_of_a_process_may_be_captured(pkg):
    """The few-row layer's first calls, routes chosen and routes given, inside a capture (the layer is made before)."""
    import os
    import subprocess
    import sys
    code = """
import torch
from __graft_entry__ import load_package
load_package()
from glmrt_b200.layer import MoeLayer
layer = MoeLayer(512, 256, 16, 4, max_tokens=16)
layer.set_router(torch.linspace(-1, 1, 16 * 512, device="cuda").sin().view(16, 512), torch.zeros(16, device="cuda"))
layer.fill_synthetic(3)
x = {m: torch.linspace(-2, 2, m * 512, device="cuda").cos().view(m, 512).bfloat16() for m in (1, 5, 16)}
idx = {m: torch.arange(4 * m, device="cuda", dtype=torch.int32).view(m, 4) % 16 for m in x}
w = {m: torch.full((m, 4), 0.5, device="cuda") for m in x}
def run():
    return [t for m in x for t in (*layer.forward_few(x[m], want_routes=True), layer.forward_few_routed(x[m], idx[m], w[m], residual_bf16=x[m]))]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
for _ in range(2):
    for t in got:
        t.zero_()
    g.replay()
    layer.check()
    assert layer.stats().launches_last_forward == 1
    assert all(torch.equal(a, b) for a, b in zip(got, run())) and any(t.any() for t in got)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


def test_few_rows_of_the_full_size_layer_do_not_depend_on_their_batch(mods):
    """The model's own shape: outputs, indices and weights bit by bit, alone and among others, routes chosen and given."""
    h, e = 6144, 256
    layer = mods["layer"].MoeLayer(h, 2048, e, 8, max_tokens=16)
    layer.set_router(randn(1, e, h, std=0.02), randn(2, e, std=0.01))
    layer.fill_synthetic(23)
    x, res = randn(3, 16, h, dtype=torch.bfloat16), randn(4, 16, h, dtype=torch.bfloat16)
    want = layer.forward_few(x, residual_bf16=res, want_routes=True)
    layer.check()
    for at, rows in ((0, 1), (2, 1), (15, 1), (3, 2), (5, 3), (9, 7), (0, 16)):
        part = slice(at, at + rows)
        got = layer.forward_few(x[part], residual_bf16=res[part], want_routes=True)
        assert all(torch.equal(g, v[part]) for g, v in zip(got, want)), (at, rows)
        assert torch.equal(layer.forward_few_routed(x[part], want[1][part], want[2][part], residual_bf16=res[part]), want[0][part]), (at, rows)
    layer.check()
    layer.close()


# ---- all of them together ------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 5, 16, 17, 200])
def test_sparse_block_runs_the_operators_together(mods, rows):
    """The block against its parts in 64 bits (few rows), and against the layer's own path (more rows);
    eager, replayed from a graph, and for a block on the W4A4 path alone."""
    se, h, i = mods["shared_expert"], 512, 256
    ref = O.make_layer(12, h, i, 16)
    layer, weights = make_layer(mods, ref, 4, max_tokens=256), layer_weights(ref)
    g, u, d = randn(1, i, h, std=.05), randn(2, i, h, std=.05), randn(3, h, i, std=.05)
    nw = 1 + randn(4, h, std=0.1)
    shared = se.DenseSharedExpert(g, u, d, dtype=torch.float8_e4m3fn)
    block = se.SparseBlock(layer, shared, nw)
    res, delta = randn(5, rows, h, std=2, dtype=torch.bfloat16), randn(6, rows, h, dtype=torch.bfloat16)
    r, x = mods["block_norm"].block_norm(res, delta, norm_weight=nw)
    sh = shared.delta(x)
    y, f32 = mlp_ref(x, shared.gate, shared.up, shared.down)
    within(sh, y, half(torch.bfloat16) * (y.abs() + f32) + f32, "shared")
    # against unquantised weights: E4M3 on both sides of two products in a row; three roundings of at most
    # 2^-4 each, whose errors have random signs, stay below their sum in the norm
    xd = x.double()
    full = (torch.nn.functional.silu(xd @ g.double().T) * (xd @ u.double().T)) @ d.double().T
    assert float((sh.double() - full).norm() / full.norm()) <= 3 * 2 ** -4
    got = block.forward(res, delta)
    layer.check()
    if rows <= 16:
        _, idx, w = layer.forward_few(x, want_routes=True)
        out, err = few_ref(weights, x, idx.cpu(), w.cpu(), r, sh)
        within(got, out, half(torch.bfloat16) * (out.abs() + err) + err, "block")
    else:
        assert torch.equal(got, layer.forward_residual(x, r, sh))
    plain = se.SparseBlock(layer, shared, nw, few_rows=0)
    assert torch.equal(plain.forward(res, delta), layer.forward_residual(x, r, sh))
    rin, din = res.clone(), delta.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gout = block.forward(rin, din)
    graph.replay()
    assert torch.equal(gout, got)
    rin.copy_(din)
    graph.replay()
    assert torch.equal(gout, block.forward(delta, delta))
    assert block.forward(res[:0], delta[:0]).shape == (0, h)
    layer.close()
