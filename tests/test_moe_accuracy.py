"""Accuracy of the mixture-of-experts layer's activations, element by element: weights that pick one
activation at a time, rows whose blocks differ widely in size, and experts with more tokens than one
pass takes.

Bound of an activation v (x or a hidden value): D(v) = 2^-17 of its 16-block's largest magnitude or
2^-34 of its row's. A product with a one-hot weight row has one term, so nothing else is added up; what
follows rounds a handful of times (silu's expf and a few products: 2^-20 of the value)."""
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu


def block_max(v):
    return v.abs().view(v.shape[0], -1, 16).amax(dim=2).repeat_interleave(16, dim=1)


def D(v):
    return 2.0 ** -17 * block_max(v) + 2.0 ** -34 * v.abs().amax(dim=1, keepdim=True)


def one_hot_codes(rows, K, at):
    """(rows, K/2) E2M1 codes: 1.0 (nibble 2) at element at[r] of row r."""
    n = torch.zeros(rows, K, dtype=torch.uint8)
    n[torch.arange(rows), at] = 2
    return n[:, 0::2] | (n[:, 1::2] << 4)


def picking_experts(E, K):
    """Experts with h_i = silu(x_0) x_i and y = h (H = I = K)."""
    import bitdance_b200 as bd
    own = torch.arange(K)
    gate_up = torch.cat([one_hot_codes(K, K, torch.zeros(K, dtype=torch.long)),
                         one_hot_codes(K, K, own)])
    one = 0x38  # E4M3 1.0
    return bd.MoeWeights(
        gate_up.expand(E, -1, -1).contiguous().cuda(),
        torch.full((E, 2 * K, K // 16), one, dtype=torch.uint8, device="cuda"),
        torch.ones(E, device="cuda"),
        one_hot_codes(K, K, own).expand(E, -1, -1).contiguous().cuda(),
        torch.full((E, K, K // 16), one, dtype=torch.uint8, device="cuda"),
        torch.ones(E, device="cuda"))


def spread_rows(T, K, dtype, seed, steps):
    """Row t: x_0 a power of two, the row's largest; block b of size 2^-s(b) of it, s in 0..steps."""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(T, K // 16, 16, generator=g) * 0.5 + 0.5
    x = x * torch.where(torch.rand(x.shape, generator=g) < 0.5, -1.0, 1.0)
    x[:, :, 1::3] *= torch.rand(T, K // 16, 5, generator=g)  # smaller elements inside a block too
    for t in range(T):
        s = torch.randperm(K // 16, generator=g) % (steps + 1)
        s[0] = 0
        top = 2.0 ** (t % 5)
        x[t] *= (top * 2.0 ** -s.double()).float()[:, None]
        x[t, 0] *= 0.9
        x[t, 0, 0] = top
    return x.view(T, K).to(dtype)


@gpu
@pytest.mark.parametrize("dtype,steps", [(torch.bfloat16, 31), (torch.float16, 20)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (11, 4, 1), (16, 1, 1), (24, 2, 2), (50, 1, 1)])
def test_one_activation_at_a_time(T, E, k, dtype, steps):
    """Every block exponent from the row's largest down: 16-token and 24-token passes."""
    import bitdance_b200 as bd
    K = 512
    x = spread_rows(T, K, dtype, T, steps).cuda()
    ids = torch.stack([(torch.arange(T) + s) % E for s in range(k)], dim=1).int().cuda()
    y = bd.moe_experts(x, ids, torch.full((T, k), 1.0 / k, device="cuda"), picking_experts(E, K),
                       out_dtype=torch.float32)
    v = x.double()
    s = v[:, :1] * torch.sigmoid(v[:, :1])
    want = s * v
    bound = s * D(v) + D(want) * (1 + 2.0 ** -10) + 2.0 ** -20 * want.abs()
    bad = ~((y.double() - want).abs() <= bound)
    assert not bad.any(), (torch.nonzero(bad)[0], y[bad][:4], want[bad][:4], bound[bad][:4])
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("ratio", [8, 11, 14])
@pytest.mark.parametrize("T,E,k", [(3, 6, 2), (30, 2, 1)])
def test_an_outlier_channel_does_not_coarsen_the_rest(ratio, T, E, k):
    """One channel 2^ratio above the others, in a 16-block that no weight row reads: the outputs keep
    the accuracy of the other blocks."""
    import bitdance_b200 as bd
    from test_moe import HALF_STEP, Case
    case = Case(T, 2048, 256, E, seed=ratio, spread=0.5)
    case.x[:, 37] = 2.0 ** ratio * case.x.abs().amax(dim=1)
    case.w.gate_up[:, :, 16:24] = 0  # elements 32..47
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(T)]).int()
    w = torch.rand(T, k, device="cuda", generator=g) + 0.5
    y = bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32)

    def product(v, verr, weight):
        aw = weight.abs()
        block = block_max(v)
        steps = 2 * (v.shape[1] / 64 + 1) * 2.0 ** -23
        return v @ weight.t(), (D(v) + verr + steps * (v.abs() + block)) @ aw.t()

    want, err = torch.zeros_like(y, dtype=torch.float64), torch.zeros_like(y, dtype=torch.float64)
    for e in range(E):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        xe, wt = case.x[t].double(), w[t, slot].double()[:, None]
        both, berr = product(xe, torch.zeros_like(xe), case.value(0, e))
        gate, up, ge, ue = both[:, :256], both[:, 256:], berr[:, :256], berr[:, 256:]
        silu = gate * torch.sigmoid(gate)
        h = silu * up * wt
        herr = (1.1 * ge * (up.abs() + ue) + silu.abs() * ue) * wt + 2.0 ** -21 * h.abs()
        d, derr = product(h, herr, case.value(1, e))
        want.index_add_(0, t, d)
        err.index_add_(0, t, derr + 2.0 ** -21 * d.abs())
    bound = err + HALF_STEP[torch.float32] * want.abs()
    bad = ~((y.double() - want).abs() <= bound)
    assert not bad.any(), (torch.nonzero(bad)[0], y[bad][:4], want[bad][:4], bound[bad][:4])


@gpu
@pytest.mark.parametrize("T", [17, 33, 64])
@pytest.mark.parametrize("H,I", [(256, 384), (640, 128)])
def test_one_expert_with_more_tokens_than_a_pass(T, H, I):
    """Few tokens per expert on average (passes of 16), and one expert that every token names: two to
    four passes over its weights."""
    import bitdance_b200 as bd
    from test_moe import Case, check
    E = 64
    case = Case(T, H, I, E, seed=T)
    ids = torch.full((T, 3), -1, dtype=torch.int32, device="cuda")
    ids[:, 1] = 41
    ids[::3, 0] = torch.arange(0, T, 3, device="cuda", dtype=torch.int32) % 40
    w = torch.rand(T, 3, device="cuda") + 0.25
    y = bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32)
    check(y, case, ids, w)
    assert bd.device_error() == 0


@gpu
def test_experts_that_finish_far_apart_repeat_their_bits():
    """One expert with every token beside many with one: down tasks wait for digits made long apart."""
    import bitdance_b200 as bd
    from test_moe import Case, check
    T, E = 64, 96
    case = Case(T, 1024, 768, E, seed=2)
    ids = torch.stack([torch.full((T,), 95), torch.arange(T), torch.full((T,), 3)], dim=1).int().cuda()
    w = torch.rand(T, 3, device="cuda") + 0.25
    want = bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32)
    check(want, case, ids, w)
    for _ in range(100):
        assert torch.equal(bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32), want)
    assert bd.device_error() == 0
