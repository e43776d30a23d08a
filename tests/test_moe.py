"""Mixture-of-experts layer for a few tokens (bd_moe_layer, bd_moe_experts) against the definition in
64 bits, its refusals, empty slots and repeated experts, streams and graphs.

Tolerances. The kernels multiply by digits of the activations: what six digits leave of a value is at
most 2^-17 of its 16-block's largest magnitude, or 2^-20 of its row's (digits below the smallest
scale are dropped). A sum over K is accumulated in fp32 in K/64 MMA steps of partial sums at most
S = sum |w| (|x| + block max) (the digits of a value add up to at most that), two roundings of
2^-23 each step. These bounds go through silu(g) u (|silu'| < 1.1) and the down product; what
follows rounds a handful of times (2^-21 of the value covers silu's expf and eight products), the
partial sums of k experts k times, the output once."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E2M1 = (0.0, .5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def lib():
    from bitdance_b200 import _lib, build
    build.build_library()
    return _lib.load()


# --------------------------------------------------------------------------------------- CPU


def test_digits_leave_2_to_the_minus_17():
    """The digit rule restated: E2M1 digits of a value |v| <= 4, each time eight times what is left."""
    rng = np.random.default_rng(0)
    v = np.concatenate([rng.uniform(-4, 4, 200000), [4.0, -4.0, 0.0, 2.5, 3.5, 1.75, 0.25]])
    book = np.array(E2M1)
    left, total = v.copy(), np.zeros_like(v)
    for p in range(6):
        a = np.abs(left)
        assert a.max() <= 4.0
        d = book[np.abs(a[:, None] - book).argmin(axis=1)] * np.sign(left)
        total += d * 8.0 ** -p
        left = (left - d) * 8
    # amax > 2 in units of the scale, so 2^-16 of the scale is 2^-17 of the block's largest
    assert np.abs(total - v).max() <= 2.0 ** -16


def test_c_abi_refusals():
    L = lib()
    P = ctypes.c_void_p
    ok = P(4096)  # never dereferenced
    ws = L.bd_query_moe_workspace(4, 256, 128, 8, 2)
    assert ws > 0

    def layer(y=ok, ids=ok, w=ok, x=ok, xd=1, r=ok, rd=1, sb=None, sc=0, T=4, H=256, I=128, E=8, k=2,
              od=0, work=ok, nb=ws, gu=ok, gus=ok):
        return L.bd_moe_layer(y, ids, w, x, xd, r, rd, sb, sc, 1, 1.0, gu, gus, ok, ok, ok, ok, T, H, I,
                              E, k, od, work, nb, None)

    def experts(**kw):
        a = dict(y=ok, x=ok, xd=1, ids=ok, w=ok, T=4, H=256, I=128, E=8, k=2, od=0, work=ok, nb=ws)
        a.update(kw)
        return L.bd_moe_experts(a["y"], a["x"], a["xd"], a["ids"], a["w"], ok, ok, ok, ok, ok, ok,
                                a["T"], a["H"], a["I"], a["E"], a["k"], a["od"], a["work"], a["nb"],
                                None)

    for call in (layer, experts):
        assert call(xd=0) == -1            # fp32 activations
        assert call(od=3) == -1
        assert call(x=None) == -1
        assert call(ids=None) == -1
        assert call(H=192) == -2
        assert call(I=64) == -2
        assert call(T=65) == -2
        assert call(T=-1) == -2
        assert call(E=513) == -2
        assert call(E=1) == -2             # top_k > E
        assert call(k=17, E=32) == -2
        assert call(k=0) == -2
        assert call(nb=ws - 1) == -6
        assert call(work=None) == -6
        assert call(work=P(4096 + 16)) == -3
        assert call(x=P(4104)) == -3
        assert call(T=0, x=None, work=None) == 0
    assert layer(sc=2) == -1
    assert layer(rd=2) == -1               # router of another 16-bit type
    assert layer(r=None) == -1
    assert layer(r=P(4098)) == -3
    assert layer(gu=P(4104)) == -3
    assert layer(gus=P(4100)) == -3
    assert L.bd_query_moe_workspace(65, 256, 128, 8, 2) == 0
    assert L.bd_query_moe_workspace(0, 256, 128, 8, 2) == 0


def test_python_workspace_matches_the_library():
    from bitdance_b200 import moe
    L = lib()
    for T, H, I, E, k in ((1, 128, 128, 1, 1), (64, 4096, 14336, 8, 2), (7, 1408, 384, 512, 16),
                          (33, 2048, 768, 500, 8)):
        assert moe._workspace_bytes(T, H, I, E, k) == L.bd_query_moe_workspace(T, H, I, E, k)


def test_python_refusals():
    import bitdance_b200 as bd
    u8 = torch.zeros
    w = bd.MoeWeights(u8(4, 256, 64, dtype=torch.uint8), u8(4, 256, 8, dtype=torch.uint8), u8(4),
                      u8(4, 128, 64, dtype=torch.uint8), u8(4, 128, 8, dtype=torch.uint8), u8(4))
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    r = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="scoring"):
        bd.moe_layer(x, r, w, 2, scoring="relu")
    with pytest.raises(TypeError, match="bfloat16"):
        bd.moe_layer(x.float(), r, w, 2)
    with pytest.raises(TypeError, match="CUDA"):
        bd.moe_layer(x, r, w, 2)
    with pytest.raises(ValueError, match="2-D"):
        bd.moe_layer(x[0], r, w, 2)
    with pytest.raises(ValueError, match="tokens, top_k"):
        bd.moe_experts(x, torch.zeros(3, 2), torch.zeros(3, 2), w)
    with pytest.raises(ValueError, match="do not match"):
        bd.quantize_moe_weights(torch.zeros(4, 256, 128), torch.zeros(4, 128, 64))


# --------------------------------------------------------------------------------------- GPU

gpu = pytest.mark.gpu


class Case:
    """Weights with scales over E4M3's range (subnormal ones too), router, activations; the values in
    64 bits on the GPU."""

    def __init__(self, T, H, I, E, dtype=torch.bfloat16, seed=0, spread=1.0, subnormal=False):
        import bitdance_b200 as bd
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.T, self.H, self.I, self.E = T, H, I, E

        def matrix(n, k):
            codes = torch.randint(0, 256, (E, n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
            lo = 0 if subnormal else 0x30
            byte = torch.randint(lo, 0x40, (E, n, k // 16), dtype=torch.uint8, device="cuda", generator=g)
            scale = torch.rand(E, device="cuda", generator=g) * 0.2 + 0.9
            return codes, byte, scale / (3.0 * k ** 0.5)

        parts = matrix(2 * I, H) + matrix(H, I)
        self.w = bd.MoeWeights(*parts)
        x = torch.randn(T, H, device="cuda", generator=g)
        x = x * torch.exp(spread * torch.randn(T, H // 16, 1, device="cuda", generator=g)).expand(
            T, H // 16, 16).reshape(T, H)
        self.x = x.to(dtype)
        self.router = (torch.randn(E, H, device="cuda", generator=g) / H ** 0.5).to(dtype)

    def value(self, which, e):
        codes, byte, scale = ((self.w.gate_up, self.w.gate_up_scales, self.w.gate_up_tensor_scale)
                              if which == 0 else
                              (self.w.down, self.w.down_scales, self.w.down_tensor_scale))
        c = torch.stack((codes[e] & 15, codes[e] >> 4), dim=-1).flatten(-2).long()
        book = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device="cuda")
        b = byte[e].long()
        s = torch.where(b >> 3 == 0, (b & 7) * 2.0 ** -9, (1 + (b & 7) / 8.0) * 2.0 ** ((b >> 3) - 7.0))
        return book[c] * s.double().repeat_interleave(16, dim=1) * scale[e].double()


def bmax(v):
    """Largest magnitude of each 16-block, for every element, and of each row."""
    a = v.abs().view(v.shape[0], -1, 16).amax(dim=2).repeat_interleave(16, dim=1)
    return a, a.amax(dim=1, keepdim=True)


def product(v, verr, w):
    """v . w^T and its error bound."""
    block, row = bmax(v)
    aw = w.abs()
    err = (2.0 ** -17 * block + 2.0 ** -20 * row + verr) @ aw.t()
    steps = 2 * (v.shape[1] / 64 + 1) * 2.0 ** -23
    return v @ w.t(), err + steps * ((v.abs() + block) @ aw.t())


def reference(case, ids, weights):
    """y and its error bound before the output's rounding, from ids and weights (T, k)."""
    x = case.x.double()
    y, err, terms = (torch.zeros_like(x) for _ in range(3))
    for e in sorted(set(ids.flatten().tolist())):
        if not 0 <= e < case.E:
            continue
        t, s = torch.nonzero(ids == e, as_tuple=True)
        wt = weights[t, s].double()[:, None]
        xe = x[t]
        gu, gerr = product(xe, torch.zeros_like(xe), case.value(0, e))
        g, u, ge, ue = gu[:, :case.I], gu[:, case.I:], gerr[:, :case.I], gerr[:, case.I:]
        silu = g * torch.sigmoid(g)
        h = silu * u * wt
        herr = (1.1 * ge * (u.abs() + ue) + silu.abs() * ue) * wt.abs() + 2.0 ** -21 * h.abs()
        d, derr = product(h, herr, case.value(1, e))
        y.index_add_(0, t, d)
        err.index_add_(0, t, derr + 2.0 ** -22 * d.abs())
        terms.index_add_(0, t, d.abs())
    return y, err + ids.shape[1] * 2.0 ** -23 * terms


def check(got, case, ids, weights):
    y, err = reference(case, ids, weights)
    bound = err + HALF_STEP[got.dtype] * (y.abs() + err) + (2.0 ** -24 if got.dtype == torch.float16
                                                          else 1e-30)
    bad = ~((got.double() - y).abs() <= bound)
    assert not bad.any(), (torch.nonzero(bad)[0], got[bad][:3], y[bad][:3], bound[bad][:3])


def routing(case, k, scoring="softmax", bias=None, renormalize=True, scale=1.0, router=None):
    """The selection in 64 bits."""
    logits = case.x.double() @ (case.router if router is None else router).double().t()
    score = torch.sigmoid(logits) if scoring == "sigmoid" else torch.softmax(logits, dim=1)
    by = logits if bias is None else score + bias.double()
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :k]
    w = score.gather(1, ids)
    if renormalize:
        w = w / w.sum(dim=1, keepdim=True)
    return ids.int(), w * scale


def weights_match(got, want, case, router=None):
    """A logit is a sum of groups of eight products, each group rounded eight times in fp32 (the sum
    over the groups is in 64 bits): |error| <= d = 8 * 2^-24 sum |w x|. Every score and every sum of
    scores then changes by a factor within exp(+-d), their quotient within exp(+-2 d); one rounding."""
    r = (case.router if router is None else router).double()
    d = 8 * 2.0 ** -24 * (case.x.double().abs() @ r.abs().t()).amax(dim=1, keepdim=True)
    return bool(((got.double() - want).abs() <= want * (torch.expm1(2 * d) + 2.0 ** -24)).all())


@gpu
@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 128, 128, 1, 1), (1, 256, 128, 4, 4), (1, 2048, 768, 16, 8), (2, 384, 640, 3, 2),
    (7, 1408, 384, 512, 6), (8, 640, 128, 64, 16), (9, 256, 1408, 8, 2), (17, 128, 256, 5, 1),
    (24, 1024, 512, 2, 2), (33, 512, 896, 8, 3), (48, 2176, 128, 40, 8), (64, 256, 256, 1, 1),
    (64, 768, 512, 8, 2), (64, 128, 2048, 300, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(T, H, I, E, k, dtype):
    import bitdance_b200 as bd
    case = Case(T, H, I, E, dtype, seed=T + H + E)
    for out_dtype in (None, torch.float32):
        y, ids, weights = bd.moe_layer(case.x, case.router, case.w, k, out_dtype=out_dtype,
                                       return_routing=True)
        want_ids, want_w = routing(case, k)
        assert torch.equal(ids, want_ids)
        assert weights_match(weights, want_w, case)
        check(y, case, ids, weights)
    assert torch.equal(bd.moe_layer(case.x, case.router, case.w, k, out_dtype=torch.float32), y)
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("router", [torch.bfloat16, torch.float32])
def test_scorings(scoring, renormalize, with_bias, router):
    import bitdance_b200 as bd
    case = Case(5, 512, 128, 37, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    bias = torch.randn(37, device="cuda", generator=g) * 0.1 if with_bias else None
    if bias is not None:
        bias[5] = float("-inf")
        bias[6] = 9.0
    r = (torch.randn(37, 512, device="cuda", generator=g) / 16).to(router)
    y, ids, weights = bd.moe_layer(case.x, r, case.w, 4, scoring=scoring, renormalize=renormalize,
                                   selection_bias=bias, routed_scale=2.5, return_routing=True)
    want_ids, want_w = routing(case, 4, scoring, bias, renormalize, 2.5, r)
    assert torch.equal(ids, want_ids)
    if with_bias:
        assert (ids[:, 0] == 6).all() and not (ids == 5).any()
    assert weights_match(weights, want_w, case, r)
    check(y, case, ids, weights)


@gpu
@pytest.mark.parametrize("T", [1, 16, 17, 33])
@pytest.mark.parametrize("H,E", [(2048, 32), (2176, 7), (2048, 33)])
def test_routing_where_experts_are_few_and_rows_long(T, H, E):
    """The router may split K there; the sigmoid of every chosen logit shows in its weight."""
    import bitdance_b200 as bd
    case = Case(T, H, 128, E, torch.bfloat16, seed=T + H + E)
    y, ids, weights = bd.moe_layer(case.x, case.router, case.w, 5, scoring="sigmoid",
                                   renormalize=False, return_routing=True)
    want_ids, want = routing(case, 5, "sigmoid", renormalize=False)
    assert torch.equal(ids, want_ids)
    assert weights_match(weights, want, case)
    check(y, case, ids, weights)


@gpu
def test_equal_scores_take_the_lowest_experts():
    import bitdance_b200 as bd
    case = Case(6, 256, 128, 48, seed=4)
    case.router[:] = case.router[0]
    _, ids, weights = bd.moe_layer(case.x, case.router, case.w, 5, return_routing=True)
    assert torch.equal(ids, torch.arange(5, device="cuda", dtype=torch.int32).expand(6, 5))
    assert (weights == 0.2).all()


@gpu
def test_given_routing_empty_slots_repeats_and_bad_ids():
    import bitdance_b200 as bd
    from bitdance_b200 import _lib
    case = Case(6, 512, 384, 8, seed=5)
    ids = torch.tensor([[0, 3, 7], [-1, -1, -1], [2, -1, 2], [5, 5, 5], [-1, 1, -1], [7, 0, 3]],
                       dtype=torch.int32, device="cuda")
    w = torch.rand(6, 3, device="cuda") - 0.3
    out = torch.full((8, 512), 7.0, dtype=torch.float32, device="cuda")
    y = bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32, out=out[1:7])
    assert (y[1] == 0).all()
    check(y, case, ids, w)
    assert (out[0] == 7).all() and (out[7] == 7).all()
    assert bd.device_error() == 0
    bad = ids.clone()
    bad[0, 1], bad[5, 0] = 8, -2
    y = bd.moe_experts(case.x, bad, w, case.w, out_dtype=torch.float32)
    check(y, case, bad, w)          # ids outside count as none
    assert bd.device_error() == _lib.BD_DEVERR_RANGE
    none = torch.full_like(ids, -1)
    assert (bd.moe_experts(case.x, none, w, case.w) == 0).all()
    assert bd.device_error() == 0


@gpu
@pytest.mark.parametrize("T,k,E", [(1, 16, 16), (2, 16, 16), (8, 4, 5), (11, 3, 3), (33, 4, 6), (64, 16, 20)])
def test_random_routing_with_repeats_and_empty_slots(T, k, E):
    """Both ways of sorting the pairs by expert (up to 32 pairs, and more)."""
    import bitdance_b200 as bd
    case = Case(T, 256, 256, E, seed=T)
    g = torch.Generator(device="cuda").manual_seed(T + k)
    ids = torch.randint(-1, E, (T, k), device="cuda", dtype=torch.int32, generator=g)
    w = torch.rand(T, k, device="cuda", generator=g) - 0.3
    y = bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32)
    check(y, case, ids, w)
    assert torch.equal(bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32), y)
    assert bd.device_error() == 0


@gpu
def test_largest_counts():
    import bitdance_b200 as bd
    case = Case(64, 128, 128, 512, seed=9)
    y, ids, weights = bd.moe_layer(case.x, case.router, case.w, 16, return_routing=True)
    want_ids, want_w = routing(case, 16)
    assert torch.equal(ids, want_ids)
    assert weights_match(weights, want_w, case)
    check(y, case, ids, weights)
    assert bd.device_error() == 0


@gpu
def test_two_layers_and_a_linear_at_once_on_three_streams():
    import bitdance_b200 as bd
    cases = [Case(9, 512, 256, 12, seed=1), Case(40, 256, 512, 6, seed=2)]
    w4 = bd.quantize_weights_fp4(torch.randn(1024, 512, device="cuda"))
    calls = [lambda s=None, c=c: bd.moe_layer(c.x, c.router, c.w, 3, stream=s) for c in cases]
    calls.append(lambda s=None: bd.w4a4_linear(cases[0].x, w4, stream=s))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [(i, call(s)) for _ in range(20) for i, (call, s) in enumerate(zip(calls, streams))]
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])
    assert bd.device_error() == 0


@gpu
def test_one_tensor_off_the_gpu_is_refused():
    import dataclasses

    import bitdance_b200 as bd
    case = Case(2, 128, 128, 4)
    ids, w = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, 2)
    calls = [lambda: bd.moe_layer(case.x, case.router.cpu(), case.w, 2),
             lambda: bd.moe_layer(case.x.cpu(), case.router, case.w, 2),
             lambda: bd.moe_layer(case.x, case.router, case.w, 2, selection_bias=torch.zeros(4)),
             lambda: bd.moe_layer(case.x, case.router, case.w, 2, out=torch.empty(2, 128).bfloat16()),
             lambda: bd.moe_experts(case.x, ids, w.cuda(), case.w),
             lambda: bd.moe_experts(case.x, ids.cuda(), w, case.w)]
    for field in dataclasses.fields(case.w):
        bad = dataclasses.replace(case.w, **{field.name: getattr(case.w, field.name).cpu()})
        calls.append(lambda bad=bad: bd.moe_layer(case.x, case.router, bad, 2))
    for call in calls:
        with pytest.raises(TypeError, match="CUDA"):
            call()


@gpu
def test_no_tokens():
    import bitdance_b200 as bd
    case = Case(2, 128, 128, 4)
    y, ids, w = bd.moe_layer(case.x[:0], case.router, case.w, 2, return_routing=True)
    assert y.shape == (0, 128) and ids.shape == (0, 2) and w.shape == (0, 2)


@gpu
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 90), (torch.bfloat16, 2.0 ** -90),
                                        (torch.float16, 2.0 ** -14), (torch.float16, 1024.0)])
def test_large_and_small_activations(dtype, size):
    """Rows of very different size and wide blocks (no overflow of the products in fp32: the up
    projection is scaled down for the large ones)."""
    import bitdance_b200 as bd
    case = Case(5, 512, 256, 4, dtype, seed=6, spread=0.5)
    case.x[::2] = (case.x[::2].double() * size).to(dtype)
    if size > 1e20:
        case.w.gate_up_tensor_scale *= 2.0 ** -80
    ids, w = routing(case, 2, "sigmoid")
    w = torch.rand(5, 2, device="cuda") + 0.5
    check(bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32), case, ids, w)


@gpu
def test_subnormal_scales():
    import bitdance_b200 as bd
    case = Case(4, 256, 384, 4, seed=7, subnormal=True)
    ids, w = routing(case, 3)
    w = w.float()
    check(bd.moe_experts(case.x, ids, w, case.w, out_dtype=torch.float32), case, ids, w)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_token_stays_alone(bad):
    import bitdance_b200 as bd
    case = Case(9, 512, 256, 8, seed=8)
    want = bd.moe_layer(case.x, case.router, case.w, 2)
    case.x[4, 77] = bad
    y, ids, _ = bd.moe_layer(case.x, case.router, case.w, 2, return_routing=True)
    assert ids.min() >= 0 and ids.max() < 8
    assert torch.isnan(y[4]).all()
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(y[keep], want[keep])


@gpu
def test_quantised_weights_through_the_layer():
    import bitdance_b200 as bd
    g = torch.Generator(device="cuda").manual_seed(2)
    w = bd.quantize_moe_weights(torch.randn(3, 512, 384, device="cuda", generator=g) * 0.05,
                                torch.randn(3, 384, 256, device="cuda", generator=g) * 0.05)
    case = Case(4, 384, 256, 3, seed=9)
    case.w = w
    y, ids, weights = bd.moe_layer(case.x, case.router, w, 2, return_routing=True)
    check(y, case, ids, weights)


@gpu
def test_streams_graphs_and_repeats_give_the_same_bits():
    """Two layers on two streams at once, a captured one replayed on new inputs, and the dense 4-bit
    linear of the same values after it, as a model runs them."""
    import bitdance_b200 as bd
    cases = [Case(T, 512, 384, 16, seed=20 + T) for T in (1, 5, 20, 64)]
    dense = bd.quantize_weights_fp4(torch.randn(256, 512, device="cuda") * 0.05)
    want = [bd.moe_layer(c.x, c.router, c.w, 3) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(24):
        for j, s in enumerate(streams):
            c = (i + j) % 4
            got.append((c, bd.moe_layer(cases[c].x, cases[c].router, cases[c].w, 3, stream=s)))
    torch.cuda.synchronize()
    for c, y in got:
        assert torch.equal(y, want[c])
    c = cases[2]
    x = c.x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = bd.moe_layer(x, c.router, c.w, 3)
        z = bd.w4a4_linear(y, dense)
    for shift in (0, 3, 7):
        x.copy_(c.x.roll(shift, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[2].roll(shift, 0))
        assert torch.equal(z, bd.w4a4_linear(want[2].roll(shift, 0), dense))
    assert bd.device_error() == 0
