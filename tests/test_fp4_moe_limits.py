"""4-bit operators and the mixture-of-experts layer at the edges of what their documentation allows:
offsets beyond 32 bits, outputs that no vector store may take, NaN in places that nothing reads, graphs
and streams side by side. Where an answer has to equal another call's, it does bit for bit: rows are
quantised on their own, and an expert's products do not depend on which number it has."""
import numpy as np
import pytest

import fp4_ref as f

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantiser_and_dequantiser_beyond_two_to_the_31(fmt):
    import bitdance_b200 as bd
    rows, K, tail = 150016, 14336, 200
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    part = torch.randn(tail, K, dtype=torch.bfloat16, device="cuda", generator=g)
    x[-tail:] = part
    x[:tail] = part
    op = bd.quantize_fp4(x, fmt)
    del x
    code, byte, s = f.quantize(part.double().cpu().numpy(), fmt)
    want = torch.from_numpy(f.pack(code)).cuda()
    assert torch.equal(op.codes[-tail:], want) and torch.equal(op.codes[:tail], want)
    values = torch.from_numpy((f.values(code, byte, fmt) * s[:, None]).astype(np.float32)).bfloat16()
    out = bd.dequantize_fp4(op, torch.bfloat16)
    assert torch.equal(out[-tail:].cpu(), values) and torch.equal(out[:tail].cpu(), values)
    assert not out[tail:-tail:1000].any()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_product_beyond_two_to_the_31(fmt):
    import bitdance_b200 as bd
    from test_fp4 import gemm_check, matrix, operand, value_of
    M, N, K, tail = 139998, 16381, 64, 300
    x = matrix(tail, K, torch.bfloat16, 1, 0.5)
    _, *an = operand(x, fmt)
    w, *wn = operand(matrix(N, K, torch.float32, 2, 0.5), fmt)
    full = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    full[-tail:] = x.cuda()
    c = bd.w4a4_gemm(bd.quantize_fp4(full, fmt), w)
    gemm_check(c[-tail:], value_of(*an, fmt), value_of(*wn, fmt), K, torch.bfloat16)
    assert not c[:-tail:997].any()
    assert bd.device_error() == 0


def test_expert_weights_beyond_two_to_the_32():
    """The last of 512 experts against the same matrices as the only ones."""
    import bitdance_b200 as bd
    E, H, I, T, k, last = 512, 4096, 2048, 5, 3, 12
    g = torch.Generator(device="cuda").manual_seed(0)

    def matrix(n, K):
        codes = torch.zeros(E, n, K // 2, dtype=torch.uint8, device="cuda")
        scales = torch.full((E, n, K // 16), 0x38, dtype=torch.uint8, device="cuda")
        codes[-last:] = torch.randint(0, 256, (last, n, K // 2), dtype=torch.uint8, device="cuda",
                                      generator=g)
        scales[-last:] = torch.randint(0x30, 0x40, (last, n, K // 16), dtype=torch.uint8,
                                       device="cuda", generator=g)
        return codes, scales, torch.rand(E, device="cuda", generator=g) * 0.01

    w = bd.MoeWeights(*matrix(2 * I, H), *matrix(H, I))
    few = bd.MoeWeights(*(getattr(w, n)[-last:].clone() for n in (
        "gate_up", "gate_up_scales", "gate_up_tensor_scale", "down", "down_scales",
        "down_tensor_scale")))
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    ids = torch.stack([torch.randperm(last, device="cuda", generator=g)[:k] for _ in range(T)]).int()
    weight = torch.rand(T, k, device="cuda", generator=g)
    y = bd.moe_experts(x, ids + (E - last), weight, w, out_dtype=torch.float32)
    assert torch.equal(y, bd.moe_experts(x, ids, weight, few, out_dtype=torch.float32))
    assert y.any()
    assert bd.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(7, 256, 512), (100, 264, 288), (1280, 2048, 256)])
def test_outputs_off_the_vector_alignment(M, N, K, dtype):
    """An output that starts one element into its memory: nothing beside it is written."""
    import bitdance_b200 as bd
    from test_fp4 import matrix
    a = bd.quantize_fp4(matrix(M, K, torch.bfloat16, 1, 0.5).cuda())
    w = bd.quantize_fp4(matrix(N, K, torch.float32, 2, 0.5).cuda())
    memory = torch.full((M * N + 2,), 7.0, dtype=dtype, device="cuda")
    c = bd.w4a4_gemm(a, w, out_dtype=dtype, out=memory[1:-1].view(M, N))
    assert torch.equal(c, bd.w4a4_gemm(a, w, out_dtype=dtype))
    assert memory[0] == 7 and memory[-1] == 7
    if dtype == torch.float32 or M > 64:
        return
    from test_moe import Case
    case = Case(M, N, 128, 4, seed=1)
    memory = torch.full((M * N + 2,), 7.0, dtype=dtype, device="cuda")
    y = bd.moe_layer(case.x, case.router, case.w, 2, out_dtype=dtype, out=memory[1:-1].view(M, N))
    assert torch.equal(y, bd.moe_layer(case.x, case.router, case.w, 2, out_dtype=dtype))
    assert memory[0] == 7 and memory[-1] == 7


def test_weights_of_empty_slots_are_not_read():
    import bitdance_b200 as bd
    from test_moe import Case
    for T, k in ((3, 4), (20, 6)):  # up to 32 pairs, and more
        case = Case(T, 256, 128, 8, seed=T)
        g = torch.Generator(device="cuda").manual_seed(T)
        ids = torch.randint(-1, 8, (T, k), device="cuda", dtype=torch.int32, generator=g)
        ids[0] = -1
        w = torch.rand(T, k, device="cuda", generator=g)
        want = bd.moe_experts(case.x, ids, w, case.w)
        for bad in (float("nan"), float("inf")):
            assert torch.equal(bd.moe_experts(case.x, ids, torch.where(ids < 0, bad, w), case.w), want)
        assert not want[0].any()


def test_two_graphs_of_a_layer_replayed_at_once():
    """Captured apart, replayed on two streams: each has its own workspace."""
    import bitdance_b200 as bd
    from test_moe import Case
    cases = [Case(6, 512, 384, 8, seed=1), Case(6, 512, 384, 8, seed=2)]
    dense = bd.quantize_weights_fp4(torch.randn(384, 512, device="cuda") * 0.05)
    want = []
    for c in cases:
        y = bd.moe_layer(c.x, c.router, c.w, 2)
        want.append((y, bd.w4a4_linear(y, dense)))
    graphs, got = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = bd.moe_layer(c.x, c.router, c.w, 2)
            z = bd.w4a4_linear(y, dense)
        graphs.append(graph)
        got.append((y, z))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(30):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (y, z), (wy, wz) in zip(got, want):
        assert torch.equal(y, wy) and torch.equal(z, wz)
    assert bd.device_error() == 0


def test_every_entry_point_on_a_raw_stream_handle():
    """stream= as an integer handle, the operands made on that stream too."""
    import bitdance_b200 as bd
    from test_moe import Case
    case = Case(5, 256, 128, 4, seed=1)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(40, 256, device="cuda", generator=g)
    w = torch.randn(96, 256, device="cuda", generator=g)
    gate_up = torch.randn(2, 256, 128, device="cuda", generator=g)
    down = torch.randn(2, 128, 128, device="cuda", generator=g)
    ids = torch.tensor([[0, 1]] * 5, dtype=torch.int32, device="cuda")
    weight = torch.rand(5, 2, device="cuda", generator=g)

    def run(**kw):
        a = bd.quantize_fp4(x, **kw)
        m, e = bd.quantize_mxfp4(x, **kw)
        q = [bd.quantize_weights_fp4(w, fmt, **kw) for fmt in ("nvfp4", "mxfp4")]
        p = bd.pack_fp4(m, e, "mxfp4", **kw)
        experts = bd.quantize_moe_weights(gate_up, down, **kw)
        return [bd.w4a4_gemm(a, q[0], **kw), bd.w4a4_gemm(p, q[1], **kw), bd.w4a4_linear(x, q[1], **kw),
                bd.dequantize_fp4(a, **kw), bd.dequantize_fp4(p, torch.bfloat16, **kw),
                bd.moe_layer(case.x, case.router, case.w, 2, **kw),
                bd.moe_experts(case.x, ids, weight, case.w, **kw), experts.gate_up, experts.down_scales]

    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s.cuda_stream, s, torch.cuda.default_stream().cuda_stream):
        for _ in range(3):
            got = run(stream=stream)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert bd.device_error() == 0
