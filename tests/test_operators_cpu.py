"""Refusals of the operators around the routed experts: nothing here reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib(pkg):
    from glmrt_b200 import native as N
    return N.library()


def norm_args(N, rows=4, width=64, **kw):
    a = N.BlockNormArgs()
    size = rows * width * 2
    a.residual, a.delta = N.DeviceBuffer.of(0x10000, size), N.DeviceBuffer.of(0x20000, size)
    a.norm_weight = N.DeviceBuffer.of(0x30000, width * 2)
    a.residual_out, a.normalized = N.DeviceBuffer.of(0x40000, size), N.DeviceBuffer.of(0x50000, size)
    a.rows, a.width, a.scale, a.eps = rows, width, 1.0, 1e-5
    for n in ("residual", "delta", "residual_out", "normalized"):
        setattr(a, n + "_stride", width)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_block_norm_refusals(lib):
    from glmrt_b200 import native as N
    buf = N.DeviceBuffer.of

    def status(**kw):
        return lib.call_status("glmrt_b200_block_norm_async", C.byref(norm_args(N, **kw)), None)

    assert lib.call_status("glmrt_b200_block_norm_async", None, None) == 1
    for bad in (dict(dtype=2), dict(weight_dtype=7), dict(width=32769), dict(eps=-1.0), dict(eps=float("nan")),
                dict(scale=float("inf")), dict(rows=1 << 33), dict(residual_stride=63), dict(normalized_stride=0)):
        assert status(**bad) == 1, bad
    assert lib.call_status("glmrt_b200_block_norm_async", C.byref(norm_args(N, width=0)), None) == 1
    assert lib.call_status("glmrt_b200_block_norm_async", C.byref(norm_args(N, rows=0)), None) == 0
    for name in ("residual", "residual_out", "normalized", "norm_weight"):
        assert status(**{name: N.DeviceBuffer.null()}) == 1, name
    for name in ("residual", "delta", "residual_out", "normalized"):
        assert status(**{name: buf(0x100000, 4 * 64 * 2 - 1)}) == 2, name
        assert status(**{name: buf(0x100001, 4 * 64 * 2)}) == 1, name
        assert status(**{name + "_stride": 1 << 62}) == 2, name
    assert status(norm_weight=buf(0x30000, 127)) == 2
    # a null delta takes no branch arguments
    null = N.DeviceBuffer.null()
    assert status(delta=null) == 1 and "need a delta" in lib.last_error()
    # overlaps: outputs with each other, an output with part of an input, with a weight, with the gate
    assert status(residual_out=buf(0x50000 + 64, 512)) == 1
    assert status(normalized=buf(0x10000 + 16, 512)) == 1
    assert status(normalized=buf(0x10000, 1024), normalized_stride=128) == 1
    assert status(normalized=buf(0x30000, 512)) == 1
    gate = buf(0x60000, 512)
    assert status(gate=gate, gate_col_stride=2) == 1
    assert status(gate=gate, gate_row_stride=64, gate_col_stride=1, residual_out=buf(0x60000, 512)) == 1
    assert status(gate=buf(0x60000, 6), gate_row_stride=1) == 2
    assert status(post_weight=buf(0x70000, 100)) == 2


def test_fp8_refusals(lib):
    from glmrt_b200 import native as N
    Z = C.c_size_t
    buf, null = N.DeviceBuffer.of, N.DeviceBuffer.null()
    need = Z(0)
    assert lib.call_status("glmrt_b200_fp8_block_linear_workspace", Z(4), Z(64), Z(128), None) == 1
    for rows, n, k in ((4, 0, 128), (4, 64, 0), (4, 64, 120), (1 << 25, 64, 128), (4, 1 << 25, 128), (4, 64, 1 << 25)):
        assert lib.call_status("glmrt_b200_fp8_block_linear_workspace", Z(rows), Z(n), Z(k), C.byref(need)) == 1
    assert lib.call_status("glmrt_b200_fp8_block_linear_workspace", Z(4), Z(64), Z(128), C.byref(need)) == 0 and need.value == 0
    assert lib.call_status("glmrt_b200_fp8_block_linear_workspace", Z(17), Z(64), Z(128), C.byref(need)) == 0 and need.value > 0
    ws = buf(0x100000, need.value)

    def linear(x=buf(0x10000, 17 * 256), c=buf(0x20000, 64 * 128), s=buf(0x30000, 4), o=buf(0x40000, 17 * 128), w=ws, rows=17, n=64, k=128,
               stride=128, dtype=0):
        return lib.call_status("glmrt_b200_fp8_block_linear_async", C.byref(N.Fp8BlockLinearArgs(x, c, s, o, w, rows, n, k, stride, dtype)), None)

    assert linear(rows=0) == 0
    assert linear(dtype=2) == 1 and linear(stride=127) == 1 and linear(k=120) == 1
    for name in "xcsow":
        assert linear(**{name: null}) == 1, name
    assert linear(x=buf(0x10000, 17 * 256 - 1)) == 2 and linear(c=buf(0x20000, 8191)) == 2 and linear(s=buf(0x30000, 3)) == 2
    assert linear(o=buf(0x40000, 17 * 128 - 1)) == 2 and linear(w=buf(0x100000, need.value - 1)) == 2
    assert linear(o=buf(0x40000, 17 * 128), dtype=1) == 2
    assert linear(c=buf(0x20008, 64 * 128)) == 1 and linear(w=buf(0x100010, need.value)) == 1

    def rows(x=buf(0x10000, 1024), c=buf(0x20000, 512), s=buf(0x30000, 16), n=4, cols=128, stride=128, dtype=0):
        return lib.call_status("glmrt_b200_fp8_quantize_rows_async", C.byref(N.Fp8QuantizeRowsArgs(x, c, s, n, cols, stride, dtype)), None)

    assert rows(n=0) == 0 and rows(cols=100) == 1 and rows(dtype=3) == 1 and rows(stride=100) == 1
    assert rows(x=null) == 1 and rows(dtype=1) == 2 and rows(c=buf(0x20000, 511)) == 2 and rows(s=buf(0x30000, 15)) == 2
    assert rows(c=buf(0x20004, 512)) == 1

    assert lib.call_status("glmrt_b200_fp8_gated_mlp_workspace", Z(4), Z(128), Z(72), C.byref(need)) == 1
    assert lib.call_status("glmrt_b200_fp8_gated_mlp_workspace", Z(4), Z(128), Z(64), C.byref(need)) == 0
    names = ["x", "gc", "gs", "uc", "us", "dc", "ds", "o", "w"]
    good = dict(zip(names, (buf(0x10000, 1024), buf(0x20000, 8192), buf(0x30000, 4), buf(0x40000, 8192), buf(0x50000, 4),
                            buf(0x60000, 8192), buf(0x70000, 4), buf(0x80000, 1024), buf(0x100000, need.value))))

    def mlp(rows=4, stride=128, **kw):
        b = {**good, **kw}
        return lib.call_status("glmrt_b200_fp8_gated_mlp_async", C.byref(N.Fp8GatedMlpArgs(*[b[n] for n in names], rows, 128, 64, stride)), None)

    assert mlp(rows=0) == 0 and mlp(stride=64) == 1
    for name in names:
        assert mlp(**{name: null}) == 1, name
        assert mlp(**{name: buf(good[name].ptr, good[name].bytes - 1)}) == 2, name


def test_fp8_refuses_outputs_over_inputs(lib):
    from glmrt_b200 import native as N
    Z = C.c_size_t
    buf = N.DeviceBuffer.of
    need = Z(0)
    assert lib.call_status("glmrt_b200_fp8_block_linear_workspace", Z(17), Z(128), Z(128), C.byref(need)) == 0
    places = dict(x=buf(0x10000, 17 * 256), c=buf(0x20000, 128 * 128), s=buf(0x30000, 4), w=buf(0x100000, need.value))

    def linear(o, rows=17, w=places["w"]):
        return lib.call_status("glmrt_b200_fp8_block_linear_async",
                               C.byref(N.Fp8BlockLinearArgs(places["x"], places["c"], places["s"], o, w, rows, 128, 128, 128, 0)), None)

    for rows in (1, 17):
        for name in ("x", "c", "s"):
            assert linear(buf(places[name].ptr, 17 * 256), rows) == 1 and "overlaps" in lib.last_error(), (rows, name)
            assert linear(buf(places[name].ptr - 2, 17 * 256), rows) == 1 and "overlaps" in lib.last_error(), (rows, name)
    assert linear(buf(places["w"].ptr + 512, 17 * 256)) == 1 and "overlaps" in lib.last_error()
    assert linear(buf(0x40000, 17 * 256), w=buf(0x10000, need.value)) == 1 and "overlaps" in lib.last_error()

    def rows(x=buf(0x10000, 1024), c=buf(0x20000, 512), s=buf(0x30000, 16)):
        return lib.call_status("glmrt_b200_fp8_quantize_rows_async", C.byref(N.Fp8QuantizeRowsArgs(x, c, s, 4, 128, 128, 0)), None)

    for bad in (dict(c=buf(0x10000, 512)), dict(s=buf(0x10400 - 4, 16)), dict(s=buf(0x20000 + 508, 16))):
        assert rows(**bad) == 1 and "overlaps" in lib.last_error(), bad

    assert lib.call_status("glmrt_b200_fp8_gated_mlp_workspace", Z(4), Z(128), Z(64), C.byref(need)) == 0
    names = ["x", "gc", "gs", "uc", "us", "dc", "ds", "o", "w"]
    good = dict(zip(names, (buf(0x10000, 1024), buf(0x20000, 8192), buf(0x30000, 4), buf(0x40000, 8192), buf(0x50000, 4),
                            buf(0x60000, 8192), buf(0x70000, 4), buf(0x80000, 1024), buf(0x100000, need.value))))
    for out, others in (("o", names[1:7] + ["w"]), ("w", names[:8])):
        for name in others:
            b = {**good, out: buf(good[name].ptr & ~0xff, good[out].bytes)}
            assert lib.call_status("glmrt_b200_fp8_gated_mlp_async",
                                   C.byref(N.Fp8GatedMlpArgs(*[b[n] for n in names], 4, 128, 64, 128)), None) == 1, (out, name)
            assert "overlaps" in lib.last_error(), (out, name)


def test_packed_arguments_have_the_layout_of_the_structs(pkg):
    """The wrappers pack their arguments with struct; the C side reads the structs of the header."""
    from glmrt_b200 import block_norm, fp8, layer, native as N
    import ctypes
    for packer, cls, nbuf in ((block_norm._ARGS, N.BlockNormArgs, 7), (fp8._QUANT_ARGS, N.Fp8QuantizeRowsArgs, 3),
                              (fp8._LINEAR_ARGS, N.Fp8BlockLinearArgs, 5), (fp8._MLP_ARGS, N.Fp8GatedMlpArgs, 9),
                              (layer.MoeLayer._FEW_ARGS, N.FewArgs, 6)):
        assert packer.size == ctypes.sizeof(cls)
        values = [0] * (4 * nbuf)
        for i in range(nbuf):
            values[4 * i:4 * i + 4] = [1000 + i, 2000 + i, 0, 0]
        rest = [n for n, _ in cls._fields_[nbuf:]]
        got = cls.from_buffer_copy(packer.pack(*values, *range(1, len(rest) + 1)))
        assert [(getattr(got, n).ptr, getattr(got, n).bytes) for n, _ in cls._fields_[:nbuf]] == [(1000 + i, 2000 + i) for i in range(nbuf)]
        assert [getattr(got, n) for n in rest] == list(range(1, len(rest) + 1))


def test_null_argument_structs(lib):
    for name in ("fp8_quantize_rows", "fp8_block_linear", "fp8_gated_mlp"):
        assert lib.call_status(f"glmrt_b200_{name}_async", None, None) == 1


def test_few_refusals(lib):
    from glmrt_b200 import native as N
    for name in ("forward_few", "forward_few_routed"):
        assert lib.call_status(f"glmrt_b200_moe_layer_{name}_async", None, None, None) == 1
        assert lib.call_status(f"glmrt_b200_moe_layer_{name}_async", None, C.byref(N.FewArgs(rows=1)), None) == 1
        assert "null" in lib.last_error()


def test_wrappers_refuse_host_tensors_and_wrong_shapes(pkg):
    from glmrt_b200 import block_norm, fp8
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        block_norm.block_norm(x, norm_weight=w)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        block_norm.block_norm(x.half(), norm_weight=w)
    with pytest.raises(ValueError, match="rows"):
        block_norm.block_norm(x[0], norm_weight=w)
    codes, scales = fp8.quantize_weight(torch.randn(70, 64))
    assert codes.shape == (70, 64) and scales.shape == (1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.block_linear(x, codes, scales)
    with pytest.raises(ValueError, match="must be"):
        fp8.block_linear(x[:, :32], codes, scales)
    with pytest.raises(ValueError, match="out_dtype"):
        fp8.block_linear(x, codes, scales, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize_rows(x)


def test_quantize_weight_against_the_definition(pkg):
    from glmrt_b200 import fp8
    w = torch.randn(200, 272, generator=torch.Generator().manual_seed(1)) * 0.02
    w[130:, :128] = 0
    codes, scales = fp8.quantize_weight(w)
    for i in range(2):
        for j in range(3):
            b = w[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            s = float(b.abs().max()) / 448 or 1.0
            assert abs(float(scales[i, j]) - s) <= 2 ** -22 * s
            back = codes[128 * i:128 * i + 128, 128 * j:128 * j + 128].float() * scales[i, j]
            # half a step of E4M3: 2^-4 of the value, or half the smallest step (2^-10) of the scale
            assert ((back - b).abs() <= 2 ** -4 * b.abs() * 1.001 + 2 ** -10 * s).all()


def test_few_wrapper_raises_on_rows_and_routes_it_cannot_pass(pkg, monkeypatch):
    """ValueError, also where asserts are off, before anything reaches the library."""
    import types
    from glmrt_b200 import launch
    from glmrt_b200.layer import MoeLayer
    layer = object.__new__(MoeLayer)
    layer.hidden, layer.top_k, layer.lib, layer.handle = 64, 2, None, None
    layer.device = types.SimpleNamespace(index=-1)              # what get_device says of a host tensor
    calls = []
    monkeypatch.setattr(launch, "call", lambda lib, symbol, packed, index, *handle: calls.append(symbol))
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    layer.forward_few(x, out=x, residual_bf16=x, shared_delta_bf16=x)
    assert len(calls) == 1
    for bad in (x[0], x[:, :32], x.float(), x.T.contiguous().T, x.view(torch.float16)):
        with pytest.raises(ValueError, match="forward_few"):
            layer.forward_few(bad)
    for bad in (x[:2], x.float(), torch.zeros(3, 128, dtype=torch.bfloat16)[:, :64]):
        for name in ("out", "residual_bf16", "shared_delta_bf16"):
            with pytest.raises(ValueError, match="forward_few"):
                layer.forward_few(x, **{name: bad})
    idx, w = torch.zeros(3, 2, dtype=torch.int64), torch.ones(3, 2)
    layer.device = torch.device("cpu")
    for i, v in ((idx[:2], w), (idx, w[:, :1]), (idx.float(), w), (idx.bool(), w), (idx.to("meta"), w), (idx, w.to("meta"))):
        with pytest.raises(ValueError, match="forward_few_routed"):
            layer.forward_few_routed(x, i, v)
    assert len(calls) == 1


def test_few_wrapper_keeps_ids_outside_32_bits_outside(pkg, monkeypatch):
    from glmrt_b200.layer import MoeLayer
    layer = object.__new__(MoeLayer)
    layer.hidden, layer.top_k, layer.device, layer.lib, layer.handle = 64, 4, torch.device("cpu"), None, None
    seen = []
    monkeypatch.setattr(MoeLayer, "_few", lambda self, symbol, hidden, out, residual, shared, idx, w: seen.append(idx))
    layer.forward_few_routed(torch.zeros(1, 64, dtype=torch.bfloat16), torch.tensor([[2 ** 32, -2 ** 32 - 1, -1, 5]]), torch.ones(1, 4))
    assert seen[0].dtype == torch.int32 and seen[0].tolist() == [[2 ** 31 - 1, -2 ** 31, -1, 5]]


def test_quantize_weight_of_blocks_below_the_smallest_scale(pkg):
    """Largest magnitudes whose 448th part rounds to zero in float32: zeros stay zeros and nothing is NaN."""
    from glmrt_b200 import fp8
    w = torch.zeros(130, 256)
    w[0, 0], w[1, 1], w[129, 3], w[0, 200] = 1e-44, -3e-43, 2e-40, 1.0
    codes, scales = fp8.quantize_weight(w)
    assert codes.float().isfinite().all() and (scales > 0).all()
    back = codes.float() * scales.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)
    # E4M3's half step, and float32's smallest value: half of it per code of a scale that is itself subnormal
    assert ((back - w).abs().double() <= 2 ** -4 * w.abs().double() + 448 * 2.0 ** -150).all()
