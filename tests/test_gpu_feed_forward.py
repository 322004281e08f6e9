"""The A8W8 product with a fused epilogue, gated expert products, routing, expert sort and the sum over choices on the GPU,
against 64-bit forms.  Bounds count roundings (oracle/feed_forward.py); whole numbers are equal."""
import pytest
import torch

from oracle import feed_forward as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(out, value, bound):
    bad = ~((out.double() - value).abs() <= bound)
    bad &= ~((out.double() == value) | (torch.isnan(out) & torch.isnan(value)))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, the first at {bad.nonzero()[0].tolist()}"


def gemm_case(m, n, k, gated, bias, residual, out_ty, seed=0, row_dt=torch.float16, col_dt=torch.float32, bias_dt=None):
    g = _gen(seed)
    rows = 2 * n if gated else n
    c = dict(a=torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8),
             b=torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8),
             row=(torch.rand(m, generator=g, device="cuda") * 0.015 + 0.005).to(row_dt),
             col=((torch.rand(rows, generator=g, device="cuda") + 0.5) / (0.0125 * 5376 * max(k, 1) ** 0.5)).to(col_dt))
    c["bias"] = torch.randn(rows, generator=g, device="cuda").to(bias_dt or out_ty) if bias else None
    c["residual"] = torch.randn(m, n, generator=g, device="cuda").to(out_ty) if residual else None
    return c


def run_gemm(c, act, gated, out_ty):
    import flashnn_b200
    from flashnn_b200 import _lib
    out = flashnn_b200.GemmA8W8Epilogue(out_ty, activation=act, gated=gated)(c["a"], c["b"], c["row"], c["col"], bias=c["bias"],
                                                                             residual=c["residual"])
    assert _lib.device_status() == 0
    return out


def check_gemm(c, act, gated, out_ty):
    out = run_gemm(c, act, gated, out_ty)
    within(out, *O.gemm_epilogue(c["a"], c["b"], c["row"], c["col"], c["bias"], act, gated, c["residual"], out_ty))
    return out


# ---------------------------------------------------------------------------------------------------------------
# product with a fused epilogue
# ---------------------------------------------------------------------------------------------------------------
# (m, n, k): the streaming kernel (up to 8 tokens, K a multiple of 4096), the single-CTA kernel with each number of
# resident rows, the CTA-pair kernel; sizes around 16, 32, 64, 128 and 256, odd ones, one K block and less
SHAPES = [(1, 512, 4096), (3, 1000, 8192), (8, 528, 4096), (5, 24, 4096), (1, 1, 64), (9, 97, 64), (16, 4096, 1024), (17, 31, 16),
          (64, 257, 272), (65, 33, 144), (128, 1000, 512), (129, 300, 144), (300, 1111, 208), (1000, 2000, 512), (513, 3000, 256),
          (2000, 4099, 128)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_epilogue_over_shapes(shape, gated):
    m, n, k = shape
    i = SHAPES.index(shape)
    act = O.ACTIVATIONS[(i + 3 * gated) % 6]
    out_ty = DTYPES[(i + gated) % 2]
    check_gemm(gemm_case(m, n, k, gated, i % 3 != 0, i % 2 == 0, out_ty, seed=i), act, gated, out_ty)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(2, 68, 17696), (16, 64, 512), (5, 301, 1040), (64, 33, 4112), (100, 130, 2048), (129, 70, 4112),
                                   (300, 100, 8192), (17, 1000, 1040), (128, 200, 28672), (1, 5, 8208)], ids=str)
def test_epilogue_with_the_k_blocks_shared_by_a_cluster(shape, gated):
    """Few tiles and a long K: two, four or eight CTAs per tile, uneven shares of the K blocks, ragged rows and columns."""
    m, n, k = shape
    for i, out_ty in enumerate(DTYPES):
        check_gemm(gemm_case(m, n, k, gated, i == 0, i == 1, out_ty, seed=n), O.ACTIVATIONS[(n + i) % 6], gated, out_ty)


@pytest.mark.parametrize("m", [2, 33, 260])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", O.ACTIVATIONS)
def test_every_activation_on_every_kernel(act, gated, m):
    for out_ty in DTYPES:
        c = gemm_case(m, 512, 4096, gated, True, True, out_ty, seed=m)
        c["col"] *= 4  # into the activations' flat ends
        check_gemm(c, act, gated, out_ty)


@pytest.mark.parametrize("k", [128, 2304])  # with 16 and with 8 epilogue warps
def test_every_width_of_the_pair_tile_is_reached(k):
    """The shape table's widths for the plain product decide the fused one's too; each of them runs here."""
    from flashnn_b200 import _lib
    seen = set()
    for m, n in [(4096, 8192), (4096, 7168), (764, 8192), (2048, 4736), (1024, 4700), (1024, 4400), (512, 4736), (300, 9400)]:
        kernel, width = _lib.a8w8_plan(m, n, k)
        if kernel == 1 and width not in seen:
            seen.add(width)
            check_gemm(gemm_case(m, n, k, False, True, True, torch.bfloat16, seed=width), "silu", False, torch.bfloat16)
    assert len(seen) >= 3
    for m, n in [(4096, 4096), (764, 4096), (512, 2368), (1024, 2200)]:
        check_gemm(gemm_case(m, n, k, True, True, True, torch.bfloat16, seed=n), "silu", True, torch.bfloat16)
    check_gemm(gemm_case(700, 4999, k, False, False, True, torch.float16, seed=k), "gelu", False, torch.float16)  # an output that takes no TMA stores


@pytest.mark.parametrize("m", [4, 40, 400])
@pytest.mark.parametrize("gated", [False, True])
def test_scale_and_bias_dtypes(gated, m):
    f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
    for row_dt, col_dt, bias_dt, out_ty in [(f16, f16, f32, f16), (bf16, bf16, f16, bf16), (f32, f32, bf16, f16), (f32, f16, f32, bf16)]:
        check_gemm(gemm_case(m, 520, 4096, gated, True, False, out_ty, seed=m, row_dt=row_dt, col_dt=col_dt, bias_dt=bias_dt),
                   "gelu", gated, out_ty)


def test_no_epilogue_gives_the_plain_products_bits():
    import flashnn_b200
    for m, n, k in [(3, 512, 4096), (40, 300, 208), (500, 1000, 256)]:
        for out_ty in DTYPES:
            c = gemm_case(m, n, k, False, False, False, out_ty, seed=n)
            plain = flashnn_b200.GemmA8W8(out_ty)(c["a"], c["b"], c["row"], c["col"])
            assert torch.equal(run_gemm(c, None, False, out_ty), plain)


@pytest.mark.parametrize("m", [3, 70, 300])
def test_views_strides_and_misaligned_operands(m):
    out_ty, n, k = torch.bfloat16, 513, 4096
    base = gemm_case(m, n, k, True, True, True, out_ty, seed=m)
    ref = check_gemm(base, "silu", True, out_ty)

    def padded(t, cols, off):  # the same values in rows of `cols`, starting at column `off`
        p = torch.full((t.shape[0], cols), 77, dtype=t.dtype, device="cuda")
        p[:, off:off + t.shape[1]] = t
        return p[:, off:off + t.shape[1]]

    for change in (dict(a=padded(base["a"], k + 32, 16)), dict(b=padded(base["b"], k + 16, 0)), dict(a=padded(base["a"], k + 5, 3)),
                   dict(b=padded(base["b"], k + 1, 1)), dict(a=base["a"].t().contiguous().t()),
                   dict(residual=padded(base["residual"], n + 7, 3)), dict(residual=base["residual"].t().contiguous().t()),
                   dict(row=base["row"].view(m, 1), col=base["col"].view(1, -1), bias=base["bias"].view(1, -1)),
                   dict(bias=torch.stack([base["bias"], base["bias"]], 1)[:, 0])):
        assert torch.equal(run_gemm(dict(base, **change), "silu", True, out_ty), ref)
    one_row = base["residual"][:1].expand(m, n)  # a residual that is broadcast over the tokens
    c = dict(base, residual=one_row)
    out = check_gemm(c, "silu", True, out_ty)
    assert torch.equal(out, run_gemm(dict(base, residual=one_row.contiguous()), "silu", True, out_ty))


def test_broadcast_operands():
    import flashnn_b200 as F
    c = gemm_case(6, 520, 4096, True, False, False, torch.float16, seed=8)
    want = run_gemm(dict(c, a=c["a"][:1].expand(6, -1).contiguous(), b=c["b"][:1].expand(1040, -1).contiguous()), "silu", True, torch.float16)
    got = run_gemm(dict(c, a=c["a"][:1].expand(6, -1), b=c["b"][:1].expand(1040, -1)), "silu", True, torch.float16)
    assert torch.equal(got, want)
    x = torch.randn(1, 40, device="cuda")
    f = F.MoeRouting(40, 4)
    assert all(torch.equal(a, b) for a, b in zip(f(x.expand(9, -1)), f(x.expand(9, -1).contiguous())))


def test_empty_and_degenerate_sizes():
    for m, n, k in [(0, 8, 64), (5, 0, 64)]:
        assert run_gemm(gemm_case(m, n, k, True, True, True, torch.float16), "silu", True, torch.float16).shape == (m, n)
    for gated in (False, True):  # no products at all: the bias alone goes through
        check_gemm(gemm_case(5, 40, 0, gated, True, True, torch.float16), "gelu_tanh", gated, torch.float16)


def _call_c(c, act, gated, out, ldo, residual, ldr):
    from flashnn_b200 import _lib
    dt = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
    m, k = c["a"].shape
    n = c["b"].shape[0] // (2 if gated else 1)
    _lib.check(_lib.lib().fnn_gemm_a8w8_epilogue(
        c["a"].data_ptr(), k, c["b"].data_ptr(), k, c["row"].data_ptr(), dt[c["row"].dtype], c["col"].data_ptr(), dt[c["col"].dtype],
        c["bias"].data_ptr(), dt[c["bias"].dtype], _lib.ACTIVATIONS[act], int(gated), residual.data_ptr(), ldr, out.data_ptr(),
        dt[out.dtype], ldo, m, n, k, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k,ldo", [(3, 520, 4096, 528), (70, 100, 144, 107), (70, 96, 144, 104), (300, 1000, 144, 1008), (300, 333, 144, 334), (16, 200, 4096, 203),
                                       (700, 5000, 2304, 5008)])
def test_writes_stay_inside_and_the_residual_may_be_the_output(m, n, k, ldo, gated):
    c = gemm_case(m, n, k, gated, True, True, torch.bfloat16, seed=ldo)
    value, bound = O.gemm_epilogue(c["a"], c["b"], c["row"], c["col"], c["bias"], "silu", gated, c["residual"], torch.bfloat16)
    for in_place in (False, True):
        buf = torch.full((m + 2, ldo), 3.0, dtype=torch.bfloat16, device="cuda")
        out = buf[1:m + 1]
        if in_place:
            out[:, :n] = c["residual"]
        _call_c(c, "silu", gated, out, ldo, out if in_place else c["residual"], ldo if in_place else n)
        torch.cuda.synchronize()
        within(out[:, :n], value, bound)
        assert (buf[0] == 3).all() and (buf[m + 1] == 3).all() and (out[:, n:] == 3).all()


@pytest.mark.parametrize("m", [4, 40, 400])
def test_non_finite_values_stay_where_they_are(m):
    nan, inf = float("nan"), float("inf")
    for act in O.ACTIVATIONS:
        c = gemm_case(m, 512, 4096, True, True, True, torch.float16, seed=1)
        ref = run_gemm(c, act, True, torch.float16)
        c["row"][1], c["bias"][7], c["bias"][512 + 9], c["residual"][2, 11] = nan, nan, inf, -inf
        out = run_gemm(c, act, True, torch.float16)
        assert torch.isnan(out[1]).all() and torch.isnan(out[:, 7]).all() and out[2, 11] == -inf
        assert not torch.isfinite(out[0, 9])
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1], keep[:, 7], keep[:, 9], keep[2, 11] = False, False, False, False
        assert torch.equal(out[keep], ref[keep])


def test_large_sums_are_exact():
    """|sum| > 2^24, where an fp32 accumulator would lose units; the output takes the rounding of the exact sum."""
    for m in (2, 50, 300):
        c = gemm_case(m, 512, 8192, True, False, False, torch.float16, seed=m)
        c["a"].fill_(127)
        c["b"][:512] = 127
        c["b"][512:, ::2] = -127
        c["row"].fill_(2 ** -14)
        c["col"].fill_(2 ** -12)
        check_gemm(c, "none", True, torch.float16)


# ---------------------------------------------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------------------------------------------
def check_route(logits, top_k, bias=None, **kw):
    import flashnn_b200
    w, ids = flashnn_b200.MoeRouting(logits.shape[1], top_k, **kw)(logits, bias)
    rw, rids = O.route(logits.cpu(), top_k, None if bias is None else bias.float().cpu().double(), **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.cpu(), rids)
    # fp32 scores: below 1.6e-5 of the value under the softmax, whose argument is rounded, and 2^-20 under the sigmoid; the
    # weights' sum and division at most 34 roundings more
    rtol = (1.6e-5 if kw.get("scoring", "softmax") == "softmax" else 2 ** -20) * 2 + 34 * O.U32
    within(w.cpu(), rw, rw.abs() * rtol + 1e-44)
    return w, ids


ROUTES = [(1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (7, 5, 5, 1, 1), (64, 60, 4, 1, 1), (33, 64, 6, 8, 3), (50, 160, 6, 8, 3), (129, 256, 8, 8, 4),
          (20, 384, 8, 1, 1), (9, 1000, 32, 1, 1), (16, 1024, 16, 32, 5), (40, 72, 3, 12, 4), (30, 32, 32, 32, 32), (11, 96, 7, 3, 2),
          (50, 448, 15, 8, 5), (21, 60, 5, 4, 3), (17, 510, 8, 3, 2), (40, 120, 12, 8, 4), (13, 250, 9, 2, 1), (35, 36, 16, 1, 1)]


@pytest.mark.parametrize("shape", ROUTES, ids=str)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_routing(shape, scoring, with_bias):
    m, e, k, groups, tg = shape
    for i, dt in enumerate([torch.float32, torch.bfloat16, torch.float16]):
        g = _gen(e + i)
        x = (2 * torch.randn(m, e, generator=g, device="cuda")).to(dt)
        bias = torch.rand(e, generator=g, device="cuda") - 0.5 if with_bias else None
        for gs in ("max", "top2") if groups > 1 else ("max",):
            check_route(x, k, bias, scoring=scoring, num_groups=groups, topk_groups=tg, group_score=gs, renormalize=(i != 1),
                        scale=1.0 if i == 0 else 2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing_ties_go_to_the_lowest_index(scoring):
    x = torch.zeros(4, 40, device="cuda")
    x[1, ::2] = 1
    x[2] = torch.arange(40, device="cuda") // 8
    x[3] = torch.where(torch.arange(40, device="cuda") % 2 == 0, 0.0, -0.0)
    zero = torch.zeros(40, device="cuda")
    for bias in (None, zero, -zero):
        for kw in (dict(), dict(num_groups=5, topk_groups=2), dict(num_groups=5, topk_groups=2, group_score="top2"),
                   dict(num_groups=10, topk_groups=7, group_score="top2")):
            check_route(x, 8, bias, scoring=scoring, **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing_near_ties_are_decided_in_64_bits(scoring):
    """Keys one step of fp32 apart, and logits whose scores are equal in fp32 but not in 64 bits."""
    g = _gen(3)
    x = torch.full((64, 64), 0.5, device="cuda")
    x = (x.view(torch.int32) + torch.randint(-2, 3, (64, 64), generator=g, device="cuda", dtype=torch.int32)).view(torch.float32)
    y = 17 + torch.randn(64, 64, generator=g, device="cuda")       # sigmoid within 2^-24 of 1
    z = -120 - 10 * torch.rand(64, 64, generator=g, device="cuda")  # scores that fp32 cannot hold
    z[:, 0] = 0 if scoring == "softmax" else -125
    bias = torch.rand(64, generator=g, device="cuda") * 2 ** -22
    for logits in (x, y, z):
        for b in (None, torch.zeros(64, device="cuda"), bias):
            check_route(logits, 6, b, scoring=scoring, num_groups=8, topk_groups=4, group_score="top2", renormalize=scoring == "sigmoid")
            check_route(logits, 6, b, scoring=scoring, renormalize=scoring == "sigmoid")


def test_routing_masked_and_non_finite_rows():
    import flashnn_b200
    inf, nan = float("inf"), float("nan")
    g = _gen(4)
    x = torch.randn(8, 24, generator=g, device="cuda")
    x[0] = -inf                      # nothing left
    x[1, 3:] = -inf                  # fewer than top_k left
    x[2, ::2] = -inf
    x[3, 8:16] = -inf                # a whole group
    x[4, 5] = -1e30
    for kw in (dict(), dict(num_groups=3, topk_groups=2), dict(num_groups=3, topk_groups=2, group_score="top2")):
        w, ids = check_route(x, 5, None, **kw)
        assert (w[0] == 0).all()
        check_route(x, 5, torch.zeros(24, device="cuda"), **kw)
        check_route(x, 5, None, scoring="sigmoid", **kw)
    x[5, 7], x[6, 2] = nan, inf
    w, ids = flashnn_b200.MoeRouting(24, 5)(x)
    assert torch.isnan(w[5]).all() and 7 not in ids[5].tolist() and len(set(ids[5].tolist())) == 5
    assert ids[6, 0] == 2 and torch.isnan(w[6, 0])
    assert torch.isfinite(w[[0, 1, 2, 3, 4, 7]]).all()
    ids = flashnn_b200.MoeRouting(24, 24, scoring="sigmoid")(x)[1]
    assert (ids.sort(1).values == torch.arange(24, device="cuda")).all()


@pytest.mark.parametrize("e,k", [(40, 12), (200, 6)])
def test_many_rows_that_fp32_does_not_decide(e, k):
    """The same doubtful row 50000 times: every copy is decided alike, in 64 bits, by both forms of the kernel."""
    import flashnn_b200
    g = _gen(e)
    x = torch.randn(1, e, generator=g, device="cuda").abs() * 2 ** -20
    bias = torch.rand(e, generator=g, device="cuda") * 2 ** -20
    w, ids = check_route(x, k, bias, scoring="sigmoid")
    many = flashnn_b200.MoeRouting(e, k, scoring="sigmoid")(x.expand(50000, -1), bias)
    assert (many[0] == w).all() and (many[1] == ids).all()


def test_equal_logits_choose_the_first_experts():
    import flashnn_b200
    for e, k in ((8, 2), (256, 8), (64, 6), (1000, 20)):  # a router that has learnt nothing yet
        w, ids = flashnn_b200.MoeRouting(e, k)(torch.zeros(300, e, device="cuda", dtype=torch.bfloat16))
        assert (ids == torch.arange(k, device="cuda")).all() and torch.allclose(w, torch.full_like(w, 1 / k), rtol=1e-6)


def test_routing_strided_logits_and_empty_batch():
    import flashnn_b200
    f = flashnn_b200.MoeRouting(40, 4)
    x = torch.randn(9, 40, device="cuda")
    ref = f(x)
    for y in (torch.cat([x, x], 1)[:, :40], x.t().contiguous().t(), torch.stack([x, -x], 1)[:, 0]):
        assert all(torch.equal(p, q) for p, q in zip(f(y), ref))
    w, ids = f(x[:0])
    assert w.shape == ids.shape == (0, 4)
    bias = torch.rand(40, device="cuda", dtype=torch.float64)
    assert torch.equal(f(x, bias)[1], f(x, bias.float())[1])


# ---------------------------------------------------------------------------------------------------------------
# expert sort
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,e,bm", [(1, 1, 1), (1, 8, 16), (2, 8, 16), (31, 3, 16), (1000, 60, 32), (4096, 8, 128), (4097, 256, 64),
                                    (20001, 512, 256), (131072, 256, 128), (70000, 1024, 16), (50000, 7, 100), (300000, 100, 64)])
def test_expert_sort(n, e, bm):
    import flashnn_b200
    g = _gen(n)
    ids = torch.randint(0, e, (n, 1), generator=g, device="cuda", dtype=torch.int32)
    if e > 4:
        ids[ids == 2] = 3  # an expert without tokens
    for first, dropped in ((0, False), (5, True)):
        x = ids + first
        if dropped:
            x = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.3, torch.randint(-2 ** 31, 5, (n, 1), generator=g, device="cuda", dtype=torch.int32), x)
            x[: n // 10] = first + e
        out = flashnn_b200.moe_sort_tokens(x, e, bm, first_expert=first)
        for got, want in zip(out, O.sort_slots(x, e, bm, first)):
            assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


def test_expert_sort_one_expert_takes_all_and_none_at_all():
    import flashnn_b200
    for n in (100, 40000):
        for value in (6, -1, 2 ** 31 - 1):
            x = torch.full((n // 4, 4), value, device="cuda", dtype=torch.int32)
            for got, want in zip(flashnn_b200.moe_sort_tokens(x, 8, 64), O.sort_slots(x, 8, 64)):
                assert torch.equal(got.cpu(), want)
    slots, experts, used = flashnn_b200.moe_sort_tokens(torch.zeros(0, 2, device="cuda", dtype=torch.int64), 8, 64)
    assert slots.numel() == experts.numel() == 0 and used.tolist() == [0]
    x = torch.tensor([[-2 ** 63, 2 ** 32, 2 ** 32 + 3, 2 ** 63 - 1, 3, -1]], device="cuda")  # 64-bit numbers that are no experts
    slots, experts, used = flashnn_b200.moe_sort_tokens(x, 8, 4)
    assert used.tolist() == [4] and slots[:4].tolist() == [4, 6, 6, 6] and experts[0] == 3
    c = torch.randn(1, 6, 16, device="cuda").half()
    assert torch.equal(flashnn_b200.moe_combine(c, topk_ids=x, num_experts=8)[0], c[0, 4])
    x = torch.randint(0, 8, (50, 6), device="cuda")
    for a, b in zip(flashnn_b200.moe_sort_tokens(x[:, ::2], 8, 16), flashnn_b200.moe_sort_tokens(x[:, ::2].int().contiguous(), 8, 16)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------
# sum over the choices
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (3, 2, 64), (5, 8, 4096), (70, 3, 1001), (257, 16, 520), (2, 40, 24)])
def test_combine(m, k, n, dt):
    import flashnn_b200
    g = _gen(n)
    c = torch.randn(m, k, n, generator=g, device="cuda").to(dt)
    w = torch.rand(m, k, generator=g, device="cuda")
    r = torch.randn(m, n, generator=g, device="cuda").to(dt)
    ids = torch.randint(-1, 7, (m, k), generator=g, device="cuda", dtype=torch.int32)
    for weights, residual in ((None, None), (w, r), (w, None), (None, r)):
        within(flashnn_b200.moe_combine(c, weights, residual=residual), *O.combine(c, weights, residual=residual))
        d = c.clone()
        d[(ids < 2) | (ids >= 6)] = float("nan")  # rows that no expert here has written
        out = flashnn_b200.moe_combine(d, weights, ids, 4, first_expert=2, residual=residual)
        within(out, *O.combine(d, weights, ids, 4, 2, residual))


def test_combine_strides():
    import flashnn_b200
    m, k, n = 37, 3, 200
    c = torch.randn(m, k, n, device="cuda").half()
    r = torch.randn(m, n, device="cuda").half()
    w = torch.rand(m, k, device="cuda")
    ref = flashnn_b200.moe_combine(c, w, residual=r)
    wide = torch.randn(m, k + 1, n + 9, device="cuda").half()
    wide[:, 1:, 5:5 + n] = c
    for x in (wide[:, 1:, 5:5 + n], c.permute(1, 0, 2).contiguous().permute(1, 0, 2), c.permute(0, 2, 1).contiguous().permute(0, 2, 1)):
        assert torch.equal(flashnn_b200.moe_combine(x, w, residual=r), ref)
    assert torch.equal(flashnn_b200.moe_combine(c, w.t().contiguous().t(), residual=r.t().contiguous().t()), ref)
    same = r[:1].expand(m, n)
    assert torch.equal(flashnn_b200.moe_combine(c, w, residual=same), flashnn_b200.moe_combine(c, w, residual=same.contiguous()))
    assert flashnn_b200.moe_combine(c[:0], w[:0], residual=r[:0]).shape == (0, n)
    assert torch.equal(flashnn_b200.moe_combine(c[:, :0]), torch.zeros(m, n, device="cuda").half())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 257, 511, 513, 1002, 1025, 1026, 2050, 2305])
def test_combine_narrow_columns(n, dt):
    """Rows of columns that no 16-byte access fits: each width of access and the rows' ends; nothing beside them is written."""
    import flashnn_b200
    m, k = 5, 3
    g = _gen(n)
    c = torch.randn(m, k, n, generator=g, device="cuda").to(dt)
    w = torch.rand(m, k, generator=g, device="cuda")
    r = torch.randn(m, n, generator=g, device="cuda").to(dt)
    want = flashnn_b200.moe_combine(c, w, residual=r)
    within(want, *O.combine(c, w, residual=r))
    ids = torch.randint(0, 4, (m, k), generator=g, device="cuda", dtype=torch.int32)
    d = c.clone()
    d[ids >= 2] = float("nan")
    within(flashnn_b200.moe_combine(d, w, ids, 2, residual=r), *O.combine(d, w, ids, 2, 0, r))
    odd = torch.randn(m * k * n + 1, generator=g, device="cuda").to(dt)[1:].view(m, k, n)  # one element off every boundary
    odd.copy_(c)
    assert torch.equal(flashnn_b200.moe_combine(odd, w, residual=r), want)


def test_combine_offsets_beyond_32_bits():
    import flashnn_b200
    m, k, n = 3, 2, 8192
    big = torch.empty((2 ** 31 // n + 16) * n, dtype=torch.float16, device="cuda")
    c = big.as_strided((m, k, n), ((2 ** 30 // n + 3) * n, n, 1))
    c.copy_(torch.randn(m, k, n, device="cuda"))
    within(flashnn_b200.moe_combine(c), *O.combine(c))


# ---------------------------------------------------------------------------------------------------------------
# gated expert products
# ---------------------------------------------------------------------------------------------------------------
def experts_case(m, e, n, k, top_k, bias, out_ty, seed, dropped=0.0):
    g = _gen(seed)
    c = dict(a=torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8),
             b=torch.randint(-127, 128, (e, 2 * n, k), generator=g, device="cuda", dtype=torch.int8),
             row=(torch.rand(m, generator=g, device="cuda") * 0.015 + 0.005).half(),
             col=(torch.rand(e, 2 * n, generator=g, device="cuda") + 0.5) / (0.0125 * 5376 * k ** 0.5))
    c["bias"] = torch.randn(e, 2 * n, generator=g, device="cuda").to(out_ty) if bias else None
    ids = torch.argsort(torch.rand(m, e, generator=g, device="cuda"), 1)[:, :top_k].int()
    c["ids"] = torch.where(torch.rand(m, top_k, generator=g, device="cuda") < dropped, torch.full_like(ids, -1), ids).contiguous()
    return c


def check_experts(c, act, bm, out_ty):
    import flashnn_b200
    from flashnn_b200 import _lib
    (m, top_k), (e, rows, _) = c["ids"].shape, c["b"].shape
    plan = flashnn_b200.moe_sort_tokens(c["ids"], e, bm)
    out = torch.full((m, top_k, rows // 2), 7.0, dtype=out_ty, device="cuda")
    got = flashnn_b200.fused_moe_a8w8_gated_forward(c["a"], c["b"], out, c["row"], c["col"], c["ids"], *plan, top_k, bm, activation=act,
                                                    bias=c["bias"])
    assert got is out and _lib.device_status() == 0
    value, bound = O.experts_gated(c["a"], c["b"], c["row"], c["col"], c["bias"], act, c["ids"], out_ty)
    gone = c["ids"] < 0
    assert (out[gone] == 7).all()
    within(out[~gone], value[~gone], bound[~gone])
    return out


@pytest.mark.parametrize("m,e,n,k,top_k,bm", [
    (1, 4, 16, 64, 1, 16), (5, 4, 40, 64, 2, 16), (33, 8, 48, 128, 2, 16), (7, 3, 33, 32, 1, 32), (64, 8, 64, 96, 4, 64), (64, 8, 1024, 512, 2, 16),
    (300, 8, 1024, 512, 2, 128), (100, 60, 256, 1024, 4, 16), (513, 4, 272, 144, 2, 256), (50, 4, 100, 80, 2, 48), (3, 64, 129, 208, 3, 16)])
def test_gated_experts(m, e, n, k, top_k, bm):
    for i, out_ty in enumerate(DTYPES):
        act = O.ACTIVATIONS[(m + i) % 6]
        check_experts(experts_case(m, e, n, k, top_k, bool(i), out_ty, seed=m, dropped=0.25 * i), act, bm, out_ty)


@pytest.mark.parametrize("m,e,n,k,top_k,bm", [(2000, 4, 512, 512, 2, 256), (1800, 6, 509, 272, 2, 256), (4400, 8, 384, 128, 1, 512)])
def test_gated_experts_on_the_cta_pair_kernel(m, e, n, k, top_k, bm):
    for i, out_ty in enumerate(DTYPES):
        check_experts(experts_case(m, e, n, k, top_k, not i, out_ty, seed=m, dropped=0.2 * i), "silu", bm, out_ty)


def test_gated_experts_strided_output_and_token_rows():
    import flashnn_b200
    c = experts_case(50, 4, 64, 96, 2, True, torch.float16, seed=1)
    plan = flashnn_b200.moe_sort_tokens(c["ids"], 4, 16)
    ref = check_experts(c, "silu", 16, torch.float16)
    buf = torch.full((50, 2, 72), 3.0, dtype=torch.float16, device="cuda")
    out = buf[:, :, :64]
    rows = torch.full((50, 112), 9, dtype=torch.int8, device="cuda")
    rows[:, :96] = c["a"]
    flashnn_b200.fused_moe_a8w8_gated_forward(rows[:, :96], c["b"], out, c["row"], c["col"], c["ids"], *plan, 2, 16, bias=c["bias"])
    assert torch.equal(out, ref) and (buf[:, :, 64:] == 3).all()
    # blocks whose expert does not exist write nothing
    plan[1][:] = torch.where(plan[1] == 2, torch.full_like(plan[1], 99), plan[1])
    out = torch.full_like(ref, 3.0)
    flashnn_b200.fused_moe_a8w8_gated_forward(c["a"], c["b"], out, c["row"], c["col"], c["ids"], *plan, 2, 16, bias=c["bias"])
    other = (c["ids"] != 2)
    assert torch.equal(out[other], ref[other]) and (out[~other] == 3).all()


def test_gated_experts_refuse_what_does_not_fit():
    import flashnn_b200
    c = experts_case(8, 4, 64, 96, 2, False, torch.float16, seed=1)
    plan = flashnn_b200.moe_sort_tokens(c["ids"], 4, 16)
    out = torch.zeros(8, 2, 64, dtype=torch.float16, device="cuda")

    def call(out=out, ids=c["ids"], top_k=2, plan=plan, **kw):
        return flashnn_b200.fused_moe_a8w8_gated_forward(c["a"], c["b"], out, c["row"], c["col"], ids, *plan, top_k, 16, **kw)
    for bad in (dict(out=out[:, :1]), dict(out=out.float()), dict(top_k=1), dict(ids=c["ids"][:4]), dict(activation="swish"),
                dict(bias=torch.zeros(4, 64, device="cuda")), dict(plan=(plan[0], plan[1][:1], plan[2]))):
        with pytest.raises(AssertionError):
            call(**bad)


# ---------------------------------------------------------------------------------------------------------------
# together, as a model runs them
# ---------------------------------------------------------------------------------------------------------------
def moe_layer(x, gate_w, up, up_col, down, down_col, top_k, bm, bias=None):
    """A mixture-of-experts feed-forward layer in int8: quantise, route, sort, gated experts, quantise, experts, sum."""
    import flashnn_b200 as F
    m, (e, hidden, inter) = x.shape[0], down.shape
    q, s = F.DynamicQuantize()(x)
    w, ids = F.MoeRouting(e, top_k, scoring="sigmoid")(x.float() @ gate_w.t(), bias)
    plan = F.moe_sort_tokens(ids, e, bm)
    h = torch.empty(m, top_k, inter, dtype=x.dtype, device=x.device)
    F.fused_moe_a8w8_gated_forward(q, up, h, s, up_col, ids, *plan, top_k, bm)
    hq, hs = F.DynamicQuantize()(h.view(m * top_k, inter))
    y = torch.empty(m * top_k, 1, hidden, dtype=x.dtype, device=x.device)
    # the second product's rows are the choices: one each
    F.fused_moe_a8w8_forward(hq, down, y, hs, down_col, w.view(-1, 1), ids.view(-1, 1), *plan, True, 1, bm)
    return F.moe_combine(y.view(m, top_k, hidden), topk_ids=ids, num_experts=e, residual=x), (q, s, w, ids, h, hq, hs, y)


def layer_case(m, hidden=256, inter=320, e=8, dt=torch.bfloat16, seed=0):
    g = _gen(seed)

    def w8(*shape):
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    return (torch.randn(m, hidden, generator=g, device="cuda").to(dt), torch.randn(e, hidden, generator=g, device="cuda") / 16,
            w8(e, 2 * inter, hidden), torch.full((e, 2 * inter), 1 / (73 * 16.0), device="cuda"),
            w8(e, hidden, inter), torch.full((e, hidden), 1 / (73 * 18.0), device="cuda"))


@pytest.mark.parametrize("m,bm", [(1, 16), (37, 16), (500, 128)])
def test_a_whole_layer(m, bm):
    x, gate_w, up, up_col, down, down_col = args = layer_case(m)
    out, (q, s, w, ids, h, hq, hs, y) = moe_layer(*args, top_k=2, bm=bm)
    # each stage against 64 bits on the stage's own inputs
    _, rids = O.route((x.float() @ gate_w.t()).cpu(), 2, scoring="sigmoid")
    assert torch.equal(ids.cpu(), rids)
    within(h, *O.experts_gated(q, up, s, up_col, None, "silu", ids, x.dtype))
    exact = torch.stack([(hq[i].double() @ down[int(j)].double().t()) * hs[i].double() * down_col[int(j)].double() * v.double()
                         for i, (j, v) in enumerate(zip(ids.view(-1), w.view(-1)))])
    # two roundings to 16 bits (fp16, then bf16) and three in fp32; fp16's smallest step below its normal range
    within(y.view(-1, 256), exact, exact.abs() * (2 ** -11 + 2 ** -8 + 2 ** -18) + 2 ** -24)
    within(out, *O.combine(y.view(m, 2, 256), None, ids, 8, 0, x))


def test_a_dense_layer_with_norm_and_residual():
    """RMSNorm + quantise, gated product, quantise, product + residual: each product against 64 bits on its own inputs."""
    import flashnn_b200 as F
    g = _gen(1)
    for m in (1, 16, 200):
        x = torch.randn(m, 512, generator=g, device="cuda").to(torch.bfloat16)
        up = torch.randint(-127, 128, (2 * 1024, 512), generator=g, device="cuda", dtype=torch.int8)
        down = torch.randint(-127, 128, (512, 1024), generator=g, device="cuda", dtype=torch.int8)
        uc, dc = torch.full((2048,), 1 / (73 * 22.0), device="cuda"), torch.full((512,), 1 / (73 * 32.0), device="cuda")
        q, s = F.RMSNormDquant(512).cuda()(x)
        h = F.GemmA8W8Epilogue(x.dtype, "silu", gated=True)(q, up, s, uc)
        within(h, *O.gemm_epilogue(q, up, s, uc, None, "silu", True, None, x.dtype))
        hq, hs = F.DynamicQuantize()(h)
        y = F.GemmA8W8Epilogue(x.dtype)(hq, down, hs, dc, residual=x)
        within(y, *O.gemm_epilogue(hq, down, hs, dc, None, "none", False, x, x.dtype))


def test_a_layer_in_two_captured_graphs_and_on_two_streams():
    """Two graphs of the layer replayed on two streams at once, next to eager calls on the stream of the capture: nothing is
    shared between them."""
    cases = [layer_case(40, seed=s) for s in (1, 2, 3)]
    want = [moe_layer(*c, top_k=2, bm=16)[0].clone() for c in cases]
    static = [layer_case(40, seed=9), layer_case(40, seed=10)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for c in static:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            moe_layer(*c, top_k=2, bm=16)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            # (its second product keeps a workspace of its own per stream: left to the products with a fused epilogue)
            import flashnn_b200 as F
            q, s = F.DynamicQuantize()(c[0])
            w, ids = F.MoeRouting(8, 2, scoring="sigmoid")(c[0].float() @ c[1].t())
            plan = F.moe_sort_tokens(ids, 8, 16)
            h = torch.zeros(40, 2, 320, dtype=torch.bfloat16, device="cuda")
            F.fused_moe_a8w8_gated_forward(q, c[2], h, s, c[3], ids, *plan, 2, 16)
            out = F.moe_combine(h, w)
        graphs.append(g)
        outs.append(out)
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for rep in range(3):
        for c, src in zip(static, (cases[rep], cases[(rep + 1) % 3])):
            for a, b in zip(c, src):
                a.copy_(b)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, (first, second)):
                with torch.cuda.stream(st):
                    g.replay()
            with torch.cuda.stream(side):
                eager = moe_layer(*cases[0], top_k=2, bm=16)[0]
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for out, src in zip(outs, (cases[rep], cases[(rep + 1) % 3])):
            _, (q, s, w, ids, h, *_) = moe_layer(*src, top_k=2, bm=16)
            within(out, *O.combine(h, w))


def test_the_product_captured_and_replayed_on_new_inputs():
    """Each kernel of the product in one graph (streaming, cluster, single CTA, CTA pair), replayed twice beside eager calls."""
    import flashnn_b200 as F
    shapes = [(2, 512, 4096), (16, 200, 4096), (100, 2000, 256), (400, 1000, 512)]
    f = F.GemmA8W8Epilogue(torch.bfloat16, "silu", gated=True)

    def call(c):
        return f(c["a"], c["b"], c["row"], c["col"], bias=c["bias"], residual=c["residual"])
    cases = [[gemm_case(*s, True, True, True, torch.bfloat16, seed=i) for s in shapes] for i in range(3)]
    want = [[call(c) for c in row] for row in cases]
    static = cases[0]
    static = [{k: v.clone() for k, v in c.items()} for c in static]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        outs = [call(c) for c in static]
    for i in (1, 2):
        for c, new in zip(static, cases[i]):
            for k in c:
                c[k].copy_(new[k])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        eager = [call(c) for c in cases[0]]  # on the default stream, at the same time
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i])) and all(torch.equal(a, b) for a, b in zip(eager, want[0]))


def test_an_expert_chosen_twice_by_one_token():
    c = experts_case(20, 4, 64, 96, 3, True, torch.bfloat16, seed=6)
    c["ids"][:, 2] = c["ids"][:, 0]
    out = check_experts(c, "silu", 16, torch.bfloat16)
    assert torch.equal(out[:, 2], out[:, 0])


# ---------------------------------------------------------------------------------------------------------------
# offsets that pass 32 bits
# ---------------------------------------------------------------------------------------------------------------
def test_outputs_and_residual_beyond_32_bit_offsets():
    m, n, k = 36000, 60000, 64  # 2.16e9 outputs
    c = gemm_case(m, n, k, False, True, False, torch.bfloat16, seed=1)
    c["residual"] = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 17, m // 2, m - 1], device="cuda")
    c["residual"][rows] = torch.randn(4, n, device="cuda").bfloat16()
    out = run_gemm(c, "relu", False, torch.bfloat16)
    within(out[rows], *O.gemm_epilogue(c["a"][rows], c["b"], c["row"][rows], c["col"], c["bias"], "relu", False, c["residual"][rows], torch.bfloat16))


def test_expert_weights_and_outputs_beyond_32_bit_offsets():
    import flashnn_b200 as F
    e, n, k, top_k = 40, 14336, 4096, 2  # 4.7e9 bytes of weights
    g = _gen(0)
    b = torch.randint(-127, 128, (e, 2 * n, k), generator=g, device="cuda", dtype=torch.int8)
    ids = torch.tensor([[39, 0], [1, 38], [39, 37]], device="cuda", dtype=torch.int32)
    c = dict(a=torch.randint(-127, 128, (3, k), generator=g, device="cuda", dtype=torch.int8), b=b, row=torch.full((3,), 0.01, device="cuda"),
             col=torch.full((e, 2 * n), 1 / (0.01 * 5376 * 64), device="cuda"), bias=None, ids=ids)
    check_experts(c, "silu", 16, torch.bfloat16)
    # 2.2e9 outputs: 80000 tokens, few of them checked
    m, n = 80000, 14000
    c = experts_case(m, 3, n, 64, 2, False, torch.float16, seed=3)
    out = torch.empty(m, 2, n, dtype=torch.float16, device="cuda")
    plan = F.moe_sort_tokens(c["ids"], 3, 256)
    F.fused_moe_a8w8_gated_forward(c["a"], c["b"], out, c["row"], c["col"], c["ids"], *plan, 2, 256)
    rows = torch.tensor([0, 5, m // 2, m - 1], device="cuda")
    within(out[rows], *O.experts_gated(c["a"][rows], c["b"], c["row"][rows], c["col"], None, "silu", c["ids"][rows], torch.float16))
    del out, plan, b
    torch.cuda.empty_cache()


def test_logits_beyond_32_bit_offsets():
    m, e = 2 ** 23 + 37, 256
    x = torch.randn(m, e, device="cuda", dtype=torch.bfloat16)
    import flashnn_b200 as F
    w, ids = F.MoeRouting(e, 4)(x)
    rows = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
    rw, rids = O.route(x[rows].cpu(), 4)
    assert torch.equal(ids[rows].cpu(), rids)
    within(w[rows].cpu(), rw, rw.abs() * 4e-5)
    del x
    torch.cuda.empty_cache()


def test_calls_on_a_stream_that_is_not_the_default():
    x = layer_case(64, seed=5)
    want = moe_layer(*x, top_k=2, bm=16)[0]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [moe_layer(*x, top_k=2, bm=16)[0] for _ in range(3)]
    st.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_results_do_not_change_from_call_to_call():
    import flashnn_b200 as F
    c = experts_case(1000, 16, 256, 256, 4, True, torch.bfloat16, seed=2)
    first = None
    for _ in range(5):
        plan = F.moe_sort_tokens(c["ids"], 16, 64)
        out = torch.zeros(1000, 4, 256, dtype=torch.bfloat16, device="cuda")
        F.fused_moe_a8w8_gated_forward(c["a"], c["b"], out, c["row"], c["col"], c["ids"], *plan, 4, 64, bias=c["bias"])
        now = [t.clone() for t in (*plan, out, F.moe_combine(out))]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))
