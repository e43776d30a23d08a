"""4-bit operators: quantiser (bit-exact), dequantiser, scale tiles, W4A4 GEMM and linear against
plain NumPy in 64 bits (fp4_ref.py), their refusals, streams and graphs.

Tolerances. The quantiser's rule fixes every rounding, so codes, scales and values are equal. The
GEMM accumulates K/64 MMA steps in fp32: each step rounds (or truncates) a partial sum that is at
most S = sum |a b| by 2^-23 of it, the 64 products inside a step likewise (aligned to the largest):
|acc - exact| <= 2 (K/64 + 1) 2^-23 S. Scaling and bias round three times (2^-24 each), the output
once (half a step of its type)."""
import ctypes

import numpy as np
import pytest

import fp4_ref as f
import w4a6_oracle as o

torch = pytest.importorskip("torch")

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def lib():
    from bitdance_b200 import _lib, build
    build.build_library()
    return _lib.load()


def matrix(rows, K, dtype, seed, spread=2.0):
    """Blocks of very different size, a few zeros, outlier elements."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, K)) * np.repeat(
        np.exp(spread * rng.standard_normal((rows, K // 16))), 16, axis=1)
    x[rng.random((rows, K)) < 0.02] = 0.0
    return torch.from_numpy(x).to(dtype)


def tie_matrix(K=256):
    """Rows of exact E2M1 values and midpoints times powers of two and E4M3 scales; zero rows and
    blocks, signed zeros, block maxima at and one ulp beside 6 x scale, tiny and huge rows."""
    rng = np.random.default_rng(3)
    grid = np.concatenate([f.E2M1, f.MID, [6.0]])
    x = np.zeros((24, K), np.float32)
    for r in range(8):
        for b in range(K // 16):
            s = np.float32(2.0 ** (b % 7 - 3) * (1 + (b % 8) / 8 if r % 2 else 1))
            x[r, 16 * b:16 * b + 16] = grid * s * np.where(rng.random(16) < .5, -1, 1)
        x[r, 0] = 2688.0 * 2.0 ** (r - 4)      # the row scale is a power of two: ties stay exact
    for r in (8, 9, 10):
        for b in range(K // 16):
            m = np.float32(6 * (1 + (b % 8) / 8) * 2.0 ** (b % 5))
            m = [m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(1e9))][r - 8]
            x[r, 16 * b:16 * b + 16] = m * rng.uniform(-1, 1, 16)
            x[r, 16 * b + b % 16] = -m
        x[r, 5] = 2688.0 * 4
    x[12, ::2] = -0.0
    x[13] = rng.standard_normal(K) * 1e-30
    x[14] = rng.standard_normal(K) * 1e-39      # float32 subnormals
    x[15] = rng.standard_normal(K) * 1e37
    x[16, 7] = 1e-44
    x[17, K - 1] = -3.0e38
    x[18] = 2.0 ** -46 * rng.standard_normal(K)  # MXFP4 exponent clamped at -40
    x[19] = 2.0 ** 50 * rng.standard_normal(K)   # ... and at 40
    x[20, :32] = 1.0
    return torch.from_numpy(x)


# --------------------------------------------------------------------------------------- CPU


def test_mxfp4_rule_is_the_reference_quantiser():
    x = np.concatenate([tie_matrix().numpy(), matrix(16, 256, torch.float32, 1).numpy()])
    x = x[np.abs(x).max(axis=1) < 1e36]
    codes, byte, _ = f.quantize(x, "mxfp4")
    sign, idx, _, exp, _ = o.quantize_codes(x.astype(np.float64).reshape(-1, 32), o.E8M0, o.E2M1_POS,
                                            32)
    want = (np.asarray(idx).reshape(x.shape) |
            (np.asarray(sign).reshape(x.shape).astype(np.int64) << 3)).astype(np.uint8)
    # beyond the largest exponent the reference saturates the same way
    assert np.array_equal(codes, want)
    assert np.array_equal(byte.reshape(-1), (np.asarray(exp).reshape(-1) + 127).astype(np.uint8))


def test_nvfp4_rule_is_the_weight_quantisers_up_to_the_division():
    """Same scales, and the same codes except where x / (s B) lies within the three roundings of
    1/s, (1/s)/B and their product with x (3 * 2^-24 relative, one more for the weight rule's x/s)
    of a midpoint. Where the row's scales are powers of two nothing rounds: all codes are equal."""
    x = tie_matrix().numpy()[:8]
    for r in range(8):
        codes, byte, s = f.quantize(x[r:r + 1], "nvfp4")
        oc, ob, ot = o.quantize_b_nvfp4(x[r:r + 1], block=16)
        assert float(ot) == s[0]
        assert np.array_equal(byte, ob)
        if r % 2 == 0:
            assert np.array_equal(codes, oc)
            continue
        y = np.abs(x[r].astype(np.float64)) / s[0] / np.repeat(f.scale_values(byte[0], "nvfp4"), 16)
        near = np.abs(y[:, None] / f.MID - 1).min(axis=1) <= 4 * 2.0 ** -24
        assert np.array_equal(codes[0][~near], oc[0][~near])
        assert (np.abs((codes[0] & 7).astype(int) - (oc[0] & 7)) <= near).all()


def test_c_abi_refusals():
    L = lib()
    P = ctypes.c_void_p
    ok = P(4096)  # never dereferenced
    q = L.bd_quantize_fp4
    assert q(ok, 0, 0, ok, None, ok, ok, 4, 64, 2, None) == -1     # unknown flag
    assert q(ok, 3, 0, ok, None, ok, ok, 4, 64, 0, None) == -1     # dtype
    assert q(ok, 0, 2, ok, None, ok, ok, 4, 64, 0, None) == -1     # format
    assert q(ok, 0, 0, ok, None, None, ok, 4, 64, 0, None) == -1   # no scales
    assert q(ok, 0, 0, ok, None, ok, None, 4, 64, 0, None) == -1   # NVFP4 without row scales
    assert q(ok, 0, 0, ok, None, ok, ok, 4, 48, 0, None) == -2     # K % 32
    assert q(ok, 0, 0, ok, None, ok, ok, -1, 64, 0, None) == -2
    assert q(None, 0, 0, None, None, None, None, 0, 64, 0, None) == 0
    assert q(P(4100), 0, 0, ok, None, ok, ok, 4, 64, 0, None) == -3
    assert q(ok, 0, 0, ok, None, P(4104), ok, 4, 64, 0, None) == -3
    d = L.bd_dequantize_fp4
    assert d(ok, ok, None, 1.0, ok, 3, 0, 4, 64, 0, None) == -1
    assert d(ok, None, None, 1.0, ok, 2, 0, 4, 64, 0, None) == -1
    assert d(ok, ok, None, 1.0, ok, 2, 0, 4, 40, 0, None) == -2
    assert d(ok, ok, None, 1.0, P(4104), 2, 0, 4, 64, 0, None) == -3
    t = L.bd_tile_scales_fp4
    assert t(ok, ok, 4, 64, 7, None) == -1
    assert t(ok, ok, 4, 33, 0, None) == -2
    assert t(ok, P(4097), 4, 64, 0, None) == -3
    g = L.bd_w4a4_gemm
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 0, 0, 4, None) == -1  # flag
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 5, 0, 0, 0, None) == -1
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 3, 0, 0, None) == -1
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 0, 1, 0, None) == -1  # no bias
    assert g(ok, None, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 0, 0, 0, None) == -1
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 80, 0, 0, 0, 0, None) == -2
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 4, 0, 64, 0, 0, 0, 0, None) == -2
    assert g(ok, P(4104), ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 0, 0, 0, None) == -3
    assert g(P(4097), ok, ok, None, ok, ok, None, 1.0, None, 4, 8, 64, 0, 0, 0, 0, None) == -3
    assert g(ok, ok, ok, None, ok, ok, None, 1.0, None, 0, 8, 64, 0, 0, 0, 0, None) == 0
    li = L.bd_w4a4_linear
    need = L.bd_query_w4a4_linear_workspace(5, 96, 0)
    assert li(ok, ok, 9, ok, ok, None, 1.0, None, 5, 8, 96, 0, 0, 0, ok, need, None) == -1
    assert li(ok, ok, 0, ok, ok, None, 1.0, None, 5, 8, 96, 0, 0, 0, ok, need - 1, None) == -6
    assert li(ok, ok, 0, ok, ok, None, 1.0, None, 5, 8, 96, 0, 0, 0, P(4112), need, None) == -3
    assert L.bd_query_fp4_scales(129, 96, 0) == 2 * 2 * 512
    assert L.bd_query_fp4_scales(129, 96, 1) == 2 * 1 * 512
    assert L.bd_query_fp4_scales(4, 40, 0) == 0


def test_python_sizes_match_the_library():
    from bitdance_b200 import fp4
    L = lib()
    for fmt, code in fp4.FP4_FORMATS.items():
        for rows, K in ((1, 32), (128, 64), (129, 1056), (8192, 14336)):
            assert fp4._scale_bytes(rows, K, fmt) == L.bd_query_fp4_scales(rows, K, code)
            assert fp4._linear_workspace(rows, K, fmt) == \
                L.bd_query_w4a4_linear_workspace(rows, K, code)


def test_python_refusals():
    import bitdance_b200 as bd
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="format"):
        bd.quantize_fp4(x, "fp4")
    with pytest.raises(TypeError, match="CUDA"):
        bd.quantize_fp4(x)
    with pytest.raises(ValueError, match="2-D"):
        bd.quantize_fp4(x[0])
    with pytest.raises(TypeError, match="float32"):
        bd.quantize_fp4(x.double())
    a = bd.Fp4Operand(x, x, 4, 64, "nvfp4")
    with pytest.raises(ValueError, match="format mismatch"):
        bd.w4a4_gemm(a, bd.Fp4Operand(x, x, 4, 64, "mxfp4"))
    with pytest.raises(ValueError, match="K mismatch"):
        bd.w4a4_gemm(a, bd.Fp4Operand(x, x, 4, 96, "nvfp4"))
    with pytest.raises(TypeError):
        bd.dequantize_fp4(a)


def test_operands_off_the_gpu_are_refused():
    import bitdance_b200 as bd
    u8 = torch.zeros(4096, dtype=torch.uint8)
    op = bd.Fp4Operand(u8[:1024].view(4, 256), u8[:4096], 4, 512, "nvfp4", torch.ones(4))
    for call in (lambda: bd.dequantize_fp4(op), lambda: bd.w4a4_gemm(op, op)):
        with pytest.raises(TypeError, match="CUDA"):
            call()


# --------------------------------------------------------------------------------------- GPU

gpu = pytest.mark.gpu


def operand(x, fmt):
    """Quantised on the GPU and, from the same values, by the 64-bit form: equal."""
    import bitdance_b200 as bd
    op = bd.quantize_fp4(x.cuda(), fmt)
    code, byte, s = f.quantize(x.double().numpy(), fmt)
    assert np.array_equal(op.codes.cpu().numpy(), f.pack(code))
    own = f.tile_rows(*byte.shape)
    assert np.array_equal(op.scales.cpu().numpy()[own], f.tile(byte)[own])
    if fmt == "nvfp4":
        assert np.array_equal(op.row_scale.cpu().numpy(), s.astype(np.float32))
    return op, code, byte, s


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,K", [(1, 32), (9, 64), (130, 96), (257, 1024), (2, 1056), (3, 14336),
                                    (1300, 2048)])
def test_quantise_and_back(rows, K, fmt, dtype):
    import bitdance_b200 as bd
    op, code, byte, s = operand(matrix(rows, K, dtype, rows + K), fmt)
    want = (f.values(code, byte, fmt) * s[:, None]).astype(np.float32)
    assert np.array_equal(bd.dequantize_fp4(op).cpu().numpy(), want)
    for out in (torch.bfloat16, torch.float16):
        assert torch.equal(bd.dequantize_fp4(op, out).cpu(), torch.from_numpy(want).to(out))
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype,rows,K", [
    (torch.float32, 600, 1056), (torch.bfloat16, 600, 1056), (torch.float16, 601, 1056),
    (torch.bfloat16, 593, 9248), (torch.float32, 4737, 1056), (torch.bfloat16, 4737, 1088)])
def test_quantise_many_rows(rows, K, fmt, dtype):
    import bitdance_b200 as bd
    op, code, byte, s = operand(matrix(rows, K, dtype, 3), fmt)
    want = (f.values(code, byte, fmt) * s[:, None]).astype(np.float32)
    assert np.array_equal(bd.dequantize_fp4(op).cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantise_ties_zeros_and_extremes(fmt):
    import bitdance_b200 as bd
    x = tie_matrix()
    operand(x, fmt)
    operand(x[:13].to(torch.bfloat16), fmt)
    if fmt == "mxfp4":
        c, e = bd.quantize_mxfp4(x.cuda())
        code, byte, _ = f.quantize(x.double().numpy(), fmt)
        assert np.array_equal(c.cpu().numpy(), f.pack(code)) and np.array_equal(e.cpu().numpy(), byte)
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("K", [96, 4096])
def test_non_finite_input_is_reported_and_stays_in_its_row(fmt, bad, K):
    import bitdance_b200 as bd
    from bitdance_b200 import _lib
    x = matrix(5, K, torch.float32, 8)
    clean = bd.quantize_fp4(x.cuda(), fmt)
    x[3, K - 7] = bad
    op = bd.quantize_fp4(x.cuda(), fmt)
    assert bd.device_error() == _lib.BD_DEVERR_NONFINITE
    keep = [0, 1, 2, 4]
    assert torch.equal(op.codes[keep], clean.codes[keep])
    w = bd.quantize_fp4(matrix(128, K, torch.float32, 9).cuda(), fmt)
    assert torch.equal(bd.w4a4_gemm(op, w)[keep], bd.w4a4_gemm(clean, w)[keep])
    bd.device_error()


@gpu
def test_scale_tiles_of_natural_scales():
    import bitdance_b200 as bd
    rng = np.random.default_rng(0)
    for fmt, block in (("nvfp4", 16), ("mxfp4", 32)):
        for rows, K in ((1, 32), (128, 256), (200, 1056)):
            byte = rng.integers(0, 256, (rows, K // block), dtype=np.uint8)
            codes = torch.zeros((rows, K // 2), dtype=torch.uint8, device="cuda")
            op = bd.pack_fp4(codes, torch.from_numpy(byte).cuda(), fmt)
            own = f.tile_rows(*byte.shape)
            assert np.array_equal(op.scales.cpu().numpy()[own], f.tile(byte)[own])


def gemm_check(c, av, wv, K, dtype, bias=None, act=lambda v: v, lipschitz=1.0):
    exact = av @ wv.T + (0.0 if bias is None else bias)
    mag = np.abs(av) @ np.abs(wv).T
    pre = 2 * (K // 64 + 1) * 2.0 ** -23 * mag + 4 * 2.0 ** -24 * (mag + np.abs(exact) + (
        0.0 if bias is None else np.abs(bias)))
    want = act(exact)
    # activations: Lipschitz constant times the error of their input, expf / tanhf within 2^-20
    bound = lipschitz * pre + HALF_STEP[dtype] * np.abs(want) + 1e-30
    if act is not gemm_check.__defaults__[1]:
        bound = bound + 2.0 ** -20 * np.abs(exact)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of fp16's subnormals
    got = c.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[0], got[bad][:3], want[bad][:3])


def value_of(code, byte, s, fmt):
    return f.values(code, byte, fmt) * s[:, None]


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,N,K", [
    (1, 128, 32), (1, 1, 64), (3, 257, 96), (16, 384, 256), (17, 128, 1056), (32, 1000, 4096),
    (33, 128, 14336), (64, 136, 288), (65, 640, 2048), (128, 256, 512), (129, 130, 544),
    (256, 512, 1024), (257, 8, 4128), (300, 384, 320), (1, 4096, 8192), (520, 776, 800)])
def test_gemm(M, N, K, fmt):
    import bitdance_b200 as bd
    a, *an = operand(matrix(M, K, torch.bfloat16, 1, 0.7), fmt)
    w, *wn = operand(matrix(N, K, torch.float32, 2, 0.7), fmt)
    av, wv = value_of(*an, fmt), value_of(*wn, fmt)
    bias = torch.linspace(-2, 2, N).to(torch.bfloat16)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M + 2, N), 7.0, dtype=dtype, device="cuda")
        c = bd.w4a4_gemm(a, w, out_dtype=dtype, out=out[1:M + 1])
        gemm_check(c, av, wv, K, dtype)
        assert (out[0] == 7).all() and (out[M + 1] == 7).all()  # nothing beyond the rows
    c = bd.w4a4_gemm(a, w, bias=bias.cuda(), epilogue="bias", out_dtype=torch.float32)
    gemm_check(c, av, wv, K, torch.float32, bias.double().numpy())
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("epilogue,act,lip", [
    ("bias_relu", lambda v: np.maximum(v, 0), 1.0),
    ("bias_silu", lambda v: v / (1 + np.exp(-np.clip(v, -700, None))), 1.1),
    ("bias_gelu", lambda v: .5 * v * (1 + np.tanh(.7978845608028654 * (v + .044715 * v ** 3))), 1.2)])
@pytest.mark.parametrize("M", [5, 200])
def test_gemm_epilogues_and_tensor_scales(epilogue, act, lip, M):
    import bitdance_b200 as bd
    N, K = 200, 288
    a, *an = operand(matrix(M, K, torch.float16, 3, 0.3), "nvfp4")
    wq = f.quantize(matrix(N, K, torch.float32, 4, 0.3).double().numpy(), "nvfp4")
    w = bd.pack_fp4(torch.from_numpy(f.pack(wq[0])).cuda(), torch.from_numpy(wq[1]).cuda(), "nvfp4",
                    tensor_scale=2.0 ** -9)
    bias = (torch.randn(N, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16)
    c = bd.w4a4_gemm(a, w, bias=bias.cuda(), epilogue=epilogue, out_dtype=torch.float16)
    gemm_check(c, value_of(*an, "nvfp4"), f.values(wq[0], wq[1], "nvfp4") * 2.0 ** -9, K,
               torch.float16, bias.double().numpy(), act, lip)


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,N,K", [
    (9473, 8, 96), (2500, 1000, 1056), (1300, 1801, 320), (300, 4900, 288), (2560, 1024, 64),
    (257, 4864, 2592), (5121, 513, 512)])
def test_gemm_of_many_tiles(M, N, K, fmt):
    """Products that CTA pairs share, with ragged last tiles and stages."""
    import bitdance_b200 as bd
    a, *an = operand(matrix(M, K, torch.bfloat16, 1, 0.7), fmt)
    w, *wn = operand(matrix(N, K, torch.float32, 2, 0.7), fmt)
    av, wv = value_of(*an, fmt), value_of(*wn, fmt)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M + 2, N), 7.0, dtype=dtype, device="cuda")
        c = bd.w4a4_gemm(a, w, out_dtype=dtype, out=out[1:M + 1])
        gemm_check(c, av, wv, K, dtype)
        assert (out[0] == 7).all() and (out[M + 1] == 7).all()
    bias = torch.linspace(-2, 2, N).to(torch.bfloat16)
    c = bd.w4a4_gemm(a, w, bias=bias.cuda(), epilogue="bias_silu", out_dtype=torch.float16)
    gemm_check(c, av, wv, K, torch.float16, bias.double().numpy(),
               lambda v: v / (1 + np.exp(-np.clip(v, -700, None))), 1.1)
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,N,K", [(1, 512, 2048), (40, 300, 1056), (600, 1024, 512)])
def test_linear_is_quantise_then_gemm(M, N, K, fmt):
    import bitdance_b200 as bd
    x = matrix(M, K, torch.bfloat16, 5, 0.5).cuda()
    w = bd.quantize_weights_fp4(matrix(N, K, torch.float32, 6, 0.5).cuda(), fmt)
    want = bd.w4a4_gemm(bd.quantize_fp4(x, fmt), w)
    for _ in range(3):
        assert torch.equal(bd.w4a4_linear(x, w), want)
    assert bd.device_error() == 0


@gpu
def test_empty_batch():
    import bitdance_b200 as bd
    w = bd.quantize_fp4(matrix(128, 64, torch.float32, 6).cuda())
    x = torch.empty((0, 64), device="cuda")
    assert bd.w4a4_linear(x, w).shape == (0, 128)
    assert bd.w4a4_gemm(bd.quantize_fp4(x), w).shape == (0, 128)
    assert bd.dequantize_fp4(bd.quantize_fp4(x)).shape == (0, 64)


@gpu
def test_streams_and_graph_replay():
    """Two linears on two streams at once, and a captured one replayed on new inputs."""
    import bitdance_b200 as bd
    w = bd.quantize_weights_fp4(matrix(512, 1024, torch.float32, 6, 0.5).cuda())
    xs = [matrix(24, 1024, torch.bfloat16, s, 0.5).cuda() for s in range(4)]
    want = [bd.w4a4_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        for j, s in enumerate(streams):
            got.append((j + 2 * (i % 2), bd.w4a4_linear(xs[j + 2 * (i % 2)], w, stream=s)))
    torch.cuda.synchronize()
    for j, c in got:
        assert torch.equal(c, want[j])
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = bd.w4a4_linear(static, w)
    for j in (1, 3, 0):
        static.copy_(xs[j])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want[j])
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_linear_right_behind_its_weights(fmt):
    """Weights written by the launch just before the linear: its early loads wait for them."""
    import bitdance_b200 as bd
    x = matrix(3, 2048, torch.bfloat16, 1, 0.5).cuda()
    ws = [matrix(4096, 2048, torch.float32, s, 0.5).cuda() for s in range(3)]
    want = []
    for w in ws:
        q = bd.quantize_fp4(w, fmt)
        torch.cuda.synchronize()
        want.append(bd.w4a4_linear(x, q))
        torch.cuda.synchronize()
    del q
    got = []
    for i in range(24):  # the operand's memory is reused from turn to turn
        got.append(bd.w4a4_linear(x, bd.quantize_fp4(ws[i % 3], fmt, overlap_prev=i % 2 == 1)))
    for i, c in enumerate(got):
        assert torch.equal(c, want[i % 3])


@gpu
def test_a_refused_launch_leaves_no_error_behind():
    """A launch into the legacy stream while a blocking stream is being captured is refused by the
    runtime; the next call is not."""
    import bitdance_b200 as bd
    L = lib()
    x = torch.randn(4, 64, device="cuda")
    want = bd.quantize_fp4(x)
    codes, scales = torch.zeros_like(want.codes), torch.zeros_like(want.scales)
    row_scale = torch.zeros_like(want.row_scale)
    torch.cuda.synchronize()

    def quantize(stream):
        P = ctypes.c_void_p
        return L.bd_quantize_fp4(P(x.data_ptr()), 0, 0, P(codes.data_ptr()), None,
                                 P(scales.data_ptr()), P(row_scale.data_ptr()), 4, 64, 0, P(stream))
    rt = ctypes.CDLL("libcudart.so.12")
    s, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(s)) == 0
    assert rt.cudaStreamBeginCapture(s, 0) == 0
    refused = quantize(1)  # the legacy stream
    rt.cudaStreamEndCapture(s, ctypes.byref(graph))
    rt.cudaGetLastError()
    assert refused == -5
    assert quantize(s.value) == 0
    torch.cuda.synchronize()
    assert torch.equal(codes, want.codes) and torch.equal(row_scale, want.row_scale)
    assert rt.cudaStreamDestroy(s) == 0


@gpu
@pytest.mark.parametrize("which", ["codes", "scales", "row_scale"])
def test_one_tensor_off_the_gpu_is_refused(which):
    import bitdance_b200 as bd
    good = bd.quantize_fp4(torch.ones(4, 512, device="cuda"))
    bad = bd.Fp4Operand(good.codes, good.scales, 4, 512, "nvfp4", good.row_scale)
    setattr(bad, which, getattr(good, which).cpu())
    x = torch.ones(1, 512, device="cuda")
    for call in (lambda: bd.dequantize_fp4(bad), lambda: bd.w4a4_gemm(good, bad),
                 lambda: bd.w4a4_linear(x, bad),
                 lambda: bd.w4a4_linear(x, good, bias=torch.ones(4, dtype=torch.bfloat16)),
                 lambda: bd.w4a4_linear(x.cpu(), good),
                 lambda: bd.dequantize_fp4(good, out=torch.empty(4, 512))):
        with pytest.raises(TypeError, match="CUDA"):
            call()
