"""Kernels launched to overlap one another: weights quantised two launches before a product that streams
its weights early (weights_static: the launch just before it does not write them)."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def middles():
    """Launches that may start before the one ahead of them has ended, and let the next one start."""
    import bitdance_b200 as bd
    from bitdance_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(4, 256, device="cuda", generator=g)
    a4, w4 = bd.quantize_fp4(x), bd.quantize_fp4(torch.randn(128, 256, device="cuda", generator=g))
    a6, w6 = ops.quantize_activations(x), ops.quantize_weights(
        torch.randn(128, 256, device="cuda", generator=g))
    big = bd.quantize_fp4(torch.randn(1024, 256, device="cuda", generator=g))
    wide = bd.quantize_fp4(torch.randn(5120, 256, device="cuda", generator=g))
    ws = ops.Workspace()
    return {
        "w4a4": lambda: bd.w4a4_gemm(a4, w4, overlap_prev=True),
        "w4a4 in large tiles": lambda: bd.w4a4_gemm(big, wide, overlap_prev=True),
        "w4a6": lambda: ops.w4a6_gemm(a6, w6, workspace=ws, overlap_prev=True),
        "w4a6 quantiser": lambda: ops.quantize_activations(x, overlap_prev=True),
        "quantiser": lambda: bd.quantize_fp4(x, overlap_prev=True)}


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("middle", ["w4a4", "w4a4 in large tiles", "w4a6", "w4a6 quantiser", "quantiser"])
def test_weights_written_two_launches_before(middle, fmt):
    import bitdance_b200 as bd
    between = middles()[middle]
    g = torch.Generator(device="cuda").manual_seed(1)
    ws = [torch.randn(4096, 8192, device="cuda", generator=g).bfloat16() for _ in range(3)]
    a = bd.quantize_fp4(torch.randn(3, 8192, device="cuda", generator=g), fmt)
    want = []
    for w in ws:
        q = bd.quantize_fp4(w, fmt)
        torch.cuda.synchronize()
        want.append(bd.w4a4_gemm(a, q))
        torch.cuda.synchronize()
    del q
    got = []
    for i in range(30):  # the operand's memory is reused from turn to turn
        torch.cuda._sleep(400_000)  # all three launches are queued before the first one starts
        q = bd.quantize_fp4(ws[i % 3], fmt)
        kept = between()
        got.append(bd.w4a4_gemm(a, q, overlap_prev=True, weights_static=True))
        del q, kept
    for i, c in enumerate(got):
        assert torch.equal(c, want[i % 3]), i
    assert bd.device_error() == 0
