"""The feed-forward operators where rounding, choice of kernel or sharing of memory shows: tails of the activations, zeros' signs,
every tile width, runs of expert blocks, waits that run out, captured graphs side by side."""
import ctypes
import time

import pytest
import torch

from oracle import feed_forward as O
from tests.test_gpu_feed_forward import DTYPES, check_experts, check_gemm, check_route, experts_case, gemm_case, run_gemm, within

pytestmark = pytest.mark.gpu


# streaming, cluster, single-CTA and CTA-pair kernel, and the generic one (no products)
KERNELS = [(2, 512, 4096), (16, 200, 4096), (100, 2000, 256), (400, 1000, 512), (3, 40, 0)]


@pytest.mark.parametrize("m,n,k", KERNELS)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "sigmoid"])
def test_negative_tails_are_relatively_exact(act, m, n, k):
    """The products are 0 and the bias is what the activation sees: the result is off by the output's half step and the few
    roundings that the bound counts, relative to a value that falls to the smallest of the type."""
    for out_ty in DTYPES:
        for gated in (False, True):
            c = gemm_case(m, n, k, gated, True, False, out_ty, bias_dt=torch.float32)
            c["a"].zero_()
            c["bias"][:n] = torch.linspace(-14, 1, n, device="cuda")
            if gated:
                c["bias"][n:] = 4096.0  # the other factor brings the tail back into fp16's normal range
            v = c["bias"].double().expand(m, -1)  # (exactly what the activation sees: no error to carry through it)
            within(run_gemm(c, act, gated, out_ty), *O.finish(v, torch.zeros_like(v), gated, act, None, out_ty))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [s for s in KERNELS if s[2]])
def test_every_kernel_gives_the_generic_kernels_bits(m, n, k, gated):
    """The choice of kernel does not show, not even in the sign of a zero: the generic kernel, which a misaligned operand takes,
    computes one output at a time."""
    for i, act in enumerate(O.ACTIVATIONS):
        for j in range(4):
            out_ty = DTYPES[(i + j) % 2]
            c = gemm_case(m, n, k, gated, j & 1, j & 2, out_ty, seed=i)
            c["a"][::2] = 0
            c["row"][1] *= -1
            c["col"][::3] *= -1
            off = torch.zeros(m, k + 5, dtype=torch.int8, device="cuda")[:, 3:3 + k]
            off.copy_(c["a"])
            fast, generic = run_gemm(c, act, gated, out_ty), run_gemm(dict(c, a=off), act, gated, out_ty)
            assert torch.equal(fast.view(torch.int16), generic.view(torch.int16)), (act, j)
    c = gemm_case(m, n, k, gated, False, False, torch.float16)
    c["a"].zero_()
    c["col"].neg_()
    out = run_gemm(c, None, gated, torch.float16)
    assert (torch.signbit(out) == (not gated)).all()  # (gated: -0 times -0)


@pytest.mark.parametrize("k", [128, 2304])  # with 16 and with 8 epilogue warps
def test_all_widths_of_the_pair_tile(k):
    """Every width that the plan can choose, by name: five without a gate, three with one (half a tile is whole chunks of 32 columns;
    where the plan for the accumulator columns takes one of the three, the gated plan takes it too)."""
    from flashnn_b200 import _lib
    for gated, widths, shapes in ((False, (128, 160, 192, 224, 256), [(136, 4744), (136, 9480), (136, 11848), (257, 7112), (257, 8296)]),
                                  (True, (128, 192, 256), [(136, 2372), (136, 5924), (257, 4148)])):
        for width, (m, n) in zip(widths, shapes):
            assert _lib.a8w8_plan(m, 2 * n if gated else n, k) == (1, width)
            for i, out_ty in enumerate(DTYPES):
                check_gemm(gemm_case(m, n - i, k, gated, True, not i, out_ty, seed=width), "silu" if i else "gelu", gated, out_ty)


# ---------------------------------------------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,tg", [(24, 1, 1), (24, 3, 2), (96, 1, 1), (96, 8, 3), (448, 8, 5)])
def test_masked_experts_and_a_bias_that_is_not_zero(e, groups, tg, scoring):
    """A logit of -inf leaves an expert its bias, a bias of -inf takes it out: single experts, a group, all but a few."""
    g = torch.Generator(device="cuda").manual_seed(e)
    x = torch.randn(60, e, generator=g, device="cuda")
    out = torch.zeros(e, dtype=torch.bool, device="cuda")
    out[torch.randperm(e, generator=g, device="cuda")[: e // 5]] = True
    x[:20, out] = -float("inf")
    x[20:30, : e // max(groups, 2)] = -float("inf")
    x[30:33, 3:] = -float("inf")
    for gs in ("max", "top2") if groups > 1 else ("max",):
        kw = dict(scoring=scoring, num_groups=groups, topk_groups=tg, group_score=gs)
        for lo, hi in ((-0.5, 0.5), (0.0, 0.2), (-0.2, 0.0)):
            bias = torch.rand(e, generator=g, device="cuda") * (hi - lo) + lo
            check_route(x, 5, bias, **kw)
            bias[out] = -float("inf")
            _, ids = check_route(x[33:], 5, bias, **kw)
            assert not out[ids.long()].any()
            check_route(x, 5, bias, **kw)
            bias[: e // max(groups, 2)] = -float("inf")
            check_route(x, 5, bias, **kw)
            bias[2:] = -float("inf")
            check_route(x, 5, bias, **kw)


def test_experts_up_to_the_largest_number():
    import flashnn_b200 as F
    top = 2 ** 31 - 1
    ids = torch.tensor([[top - 1, -2 ** 31], [top, top - 2], [-1, 0]], device="cuda")
    for x in (ids, ids.int(), torch.where(ids == top, 2 ** 40, ids)):  # 2^31 - 1 and all above are no expert
        slots, experts, used = F.moe_sort_tokens(x, 2, 2, first_expert=top - 2)
        assert used.tolist() == [4] and slots[:4].tolist() == [3, 6, 0, 6] and experts[:2].tolist() == [0, 1]
        c = torch.arange(1, 7, device="cuda").half().view(3, 2, 1)
        assert F.moe_combine(c, topk_ids=x, num_experts=2, first_expert=top - 2).flatten().tolist() == [1, 4, 0]
        for call in (lambda: F.moe_sort_tokens(x, 3, 2, first_expert=top - 2),
                     lambda: F.moe_combine(c, topk_ids=x, num_experts=3, first_expert=top - 2)):
            with pytest.raises(AssertionError, match="2\\^31"):
                call()


# ---------------------------------------------------------------------------------------------------------------
# gated expert products: runs of an expert's blocks
# ---------------------------------------------------------------------------------------------------------------
# By the rule of the launch, on 148 SMs: a mean of up to 48 choices per expert and blocks of up to 32 slots make runs of up to 64 rows, else
# 128; the widest of 256, 128 and 64 accumulator columns that gives every SM a tile.  n: 2500 -> 256, 1300 -> 128, 300 -> 64.
@pytest.mark.parametrize("n", [2500, 1300, 301])
@pytest.mark.parametrize("m,bm", [(64, 16), (150, 32), (40, 5), (512, 16), (700, 64), (600, 48), (257, 32)])
def test_runs_of_every_height_and_width(m, bm, n):
    for i, out_ty in enumerate(DTYPES):
        c = experts_case(m, 8, n, 144, 2, not i, out_ty, seed=m + n, dropped=0.1 * i)
        if i:
            c["ids"][: m // 2] = 6  # more than half of the choices are one expert's, so that it has several runs
        check_experts(c, "silu", bm, out_ty)


@pytest.mark.parametrize("m,blocks", [(8132, 1024), (8140, 1025), (20000, 2507)])
def test_slot_lists_around_the_longest_that_is_gathered_into_runs(m, blocks):
    """Up to 1024 blocks are gathered into runs; a longer list has a tile for every block."""
    from flashnn_b200 import _lib
    assert _lib.lib().fnn_moe_sort_slots(2 * m, 8, 16) == 16 * blocks
    check_experts(experts_case(m, 8, 70, 80, 2, True, torch.bfloat16, seed=m, dropped=0.1), "silu", 16, torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------
# waits that run out
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(16, 200, 4096), (64, 130, 4112), (128, 200, 28672)])
def test_a_wait_of_the_cluster_kernel_runs_out(m, n, k, gated):
    """A test option shortens the waits of one launch and leaves out the loads of one K block in the first CTA of every cluster.  The
    launch ends, the host reads the status once, and the same call then gives the same right answer as before."""
    from flashnn_b200 import _lib
    L = _lib.lib()
    c = gemm_case(m, n, k, gated, True, True, torch.bfloat16, seed=n)
    want = check_gemm(c, "silu", gated, torch.bfloat16)
    _lib.set_option(_lib.OPT_TEST_STALL_US, 20000)
    try:
        start = time.perf_counter()
        with pytest.raises(_lib.FlashNNError) as err:
            run_gemm(c, "silu", gated, torch.bfloat16)  # (reads the device status after its call)
        assert time.perf_counter() - start < 2.0
    finally:
        _lib.set_option(_lib.OPT_TEST_STALL_US, 0)
    assert err.value.status == 8 and "bounded wait" in err.value.message
    code = ctypes.c_int(0)
    assert L.fnn_device_status(ctypes.byref(code)) == 0 and code.value == 0
    assert torch.equal(check_gemm(c, "silu", gated, torch.bfloat16), want)
