"""The mixture-of-experts router's selection where logits are equal or nearly so: sums of large terms
that cancel, whose 64-bit value does not depend on the order (every partial sum fits 53 bits)."""
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu


def cancelling_rows(E, H, x_dtype, router_dtype, seed):
    """Rows that are permutations of one another over the first H - 8 columns, and x constant there:
    equal exact logits. Entries have at most 23 bits above 2^-20 (8 or 11 for the 16-bit types), the
    constant 8 or 11, the sum of 2048 at most 11 more."""
    g = torch.Generator().manual_seed(seed)
    r = torch.randn(H - 8, generator=g) * 2.0 ** torch.randint(-6, 7, (H - 8,), generator=g)
    r = (r * 2.0 ** 20).round() / 2.0 ** 20 if router_dtype == torch.float32 else r.to(router_dtype)
    rows = torch.zeros(E, H, dtype=router_dtype)
    for e in range(E):
        rows[e, :H - 8] = r[torch.randperm(H - 8, generator=g)]
    x = torch.full((5, H), 1 + 2.0 ** (-7 if x_dtype == torch.bfloat16 else -10), dtype=x_dtype)
    x[:, H - 8:] = 1.0
    x[1::2] = -x[1::2]
    return rows, x


def experts(E, H):
    import bitdance_b200 as bd
    I = 128
    return bd.MoeWeights(torch.zeros(E, 2 * I, H // 2, dtype=torch.uint8, device="cuda"),
                         torch.full((E, 2 * I, H // 16), 0x38, dtype=torch.uint8, device="cuda"),
                         torch.ones(E, device="cuda"),
                         torch.zeros(E, H, I // 2, dtype=torch.uint8, device="cuda"),
                         torch.full((E, H, I // 16), 0x38, dtype=torch.uint8, device="cuda"),
                         torch.ones(E, device="cuda"))


@gpu
@pytest.mark.parametrize("E,H", [(8, 2048), (32, 2176), (40, 1024), (130, 2048)])
@pytest.mark.parametrize("x_dtype,router_dtype", [
    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
    (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_equal_and_nearly_equal_logits(E, H, x_dtype, router_dtype):
    import bitdance_b200 as bd
    rows, x = cancelling_rows(E, H, x_dtype, router_dtype, E)
    w = experts(E, H)
    k = 4
    _, ids, weights = bd.moe_layer(x.cuda(), rows.cuda(), w, k, return_routing=True)
    assert torch.equal(ids.cpu(), torch.arange(k, dtype=torch.int32).expand(5, k))
    assert (weights == 1.0 / k).all()
    # one column apart by multiples of 2^-20 (2^-14 where fp16 has no smaller): the order is theirs
    g = torch.Generator().manual_seed(1)
    order = torch.randperm(E, generator=g)
    rows[:, H - 1] = (order * (2.0 ** -14 if router_dtype == torch.float16 else 2.0 ** -20)).to(rows.dtype)
    _, ids, _ = bd.moe_layer(x.cuda(), rows.cuda(), w, k, return_routing=True)
    best = torch.argsort(order, descending=True).int()
    for t in range(5):  # x is negative in the odd rows
        want = best[:k] if t % 2 == 0 else best.flip(0)[:k]
        assert torch.equal(ids[t].cpu(), want)


@gpu
@pytest.mark.parametrize("size", [2.0 ** 66, 2.0 ** -80])
def test_products_beyond_fp32(size):
    """bf16 activations and router weights whose products leave fp32's range: the order stands."""
    import bitdance_b200 as bd
    E, H = 16, 256
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(3, H, generator=g) * size).to(torch.bfloat16)
    r = (torch.randn(E, H, generator=g) * size).to(torch.bfloat16)
    _, ids, weights = bd.moe_layer(x.cuda(), r.cuda(), experts(E, H), 3, return_routing=True)
    logits = x.double() @ r.double().t()
    assert torch.equal(ids.cpu(), torch.argsort(logits, dim=1, descending=True)[:, :3].int())
    score = torch.softmax(logits, dim=1).gather(1, ids.cpu().long())
    want = score / score.sum(dim=1, keepdim=True)
    # fp32 rounding, and logits of 2^140 leave the first alone
    assert ((weights.cpu().double() - want).abs() <= 2.0 ** -23 * want).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_zero_rows_in_a_batch(dtype):
    """Rows of zeros, as a padded batch has them: every logit is equal, the output row is zero."""
    import bitdance_b200 as bd
    from test_moe import Case, check, routing
    case = Case(6, 256, 128, 9, dtype, seed=3)
    case.x[1] = 0
    case.x[4] = -0.0
    y, ids, weights = bd.moe_layer(case.x, case.router, case.w, 4, return_routing=True)
    want_ids, _ = routing(case, 4)
    assert torch.equal(ids, want_ids)
    for t in (1, 4):
        assert ids[t].tolist() == [0, 1, 2, 3] and (weights[t] == 0.25).all() and (y[t] == 0).all()
    check(y, case, ids, weights)


@gpu
@pytest.mark.parametrize("renormalize", [True, False])
def test_a_nan_logit_shows_in_the_softmax_weights(renormalize):
    """softmax over the experts of logits with a NaN is NaN, whether that expert is chosen or not."""
    import bitdance_b200 as bd
    E, H = 12, 256
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, H, generator=g).to(torch.bfloat16)
    r = torch.randn(E, H, generator=g).to(torch.bfloat16)
    r[5, 100] = float("nan")
    _, ids, weights = bd.moe_layer(x.cuda(), r.cuda(), experts(E, H), 3, renormalize=renormalize,
                                   return_routing=True)
    assert weights.isnan().all()
    assert not (ids == 5).any()  # a NaN ranks last
    _, ids, weights = bd.moe_layer(x.cuda(), r.cuda(), experts(E, H), 3, scoring="sigmoid",
                                   return_routing=True)
    assert weights.isfinite().all() and not (ids == 5).any()
