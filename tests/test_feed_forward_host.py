"""Feed-forward operators without a GPU: refusals of every entry point before the device is touched, sizes, names."""
import pytest
import torch

import flashnn
import flashnn_b200
from flashnn_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from flashnn_b200 import build
    build.build()
    return _lib.lib()


def test_names_are_exported():
    for name in ("GemmA8W8Epilogue", "MoeRouting", "moe_sort_tokens", "fused_moe_a8w8_gated_forward", "moe_combine"):
        assert getattr(flashnn, name) is getattr(flashnn_b200, name) and name in flashnn_b200.__all__


def test_gemm_epilogue_refusals(lib):
    def call(M=4, N=32, K=64, lda=64, ldb=64, rdt=_lib.F16, cdt=_lib.F32, bias=None, bdt=0, act=3, gated=0, res=None, ldr=0,
             odt=_lib.BF16, ldo=32):
        return lib.fnn_gemm_a8w8_epilogue(None, lda, None, ldb, None, rdt, None, cdt, bias, bdt, act, gated, res, ldr, None, odt,
                                          ldo, M, N, K, None)

    assert call() == 1 and b"null" in lib.fnn_last_error_string()
    assert call(M=0) == 0 and call(N=0, ldo=0) == 0
    assert call(M=-1) == 3 and call(lda=63) == 3 and call(ldb=63) == 3 and call(ldo=31) == 3
    assert call(res=16, ldr=-1) == 3
    assert call(N=2 ** 30 + 1, ldo=2 ** 31) == 3  # 2 N weight rows
    assert call(odt=_lib.F32) == 2 and call(rdt=3) == 2 and call(cdt=-1) == 2 and call(bias=16, bdt=7) == 2
    assert call(act=6) == 5 and call(act=-1) == 5


def test_experts_gated_refusals(lib):
    def call(E=4, N=32, K=64, lda=64, rdt=_lib.F16, cdt=_lib.F32, bias=None, bdt=0, act=3, EM=32, valid=16, top_k=2, bm=16,
             odt=_lib.BF16, ldo=32, p=None, ws=None, wsb=0):
        return lib.fnn_fused_moe_a8w8_gated(p, lda, p, E, N, K, p, rdt, p, cdt, bias, bdt, act, p, EM, p, p, valid, top_k, bm, p,
                                            odt, ldo, ws, wsb, None)

    assert call() == 1
    assert call(EM=0) == 0 and call(valid=0) == 0
    assert call(E=0) == 3 and call(lda=63) == 3 and call(ldo=31) == 3 and call(top_k=0) == 3 and call(EM=33) == 3
    assert call(E=2 ** 20, N=2 ** 10, ldo=2 ** 10) == 3  # 2 E N weight rows
    assert call(bm=144, EM=144) == 5 and call(act=9) == 5
    assert call(odt=_lib.F32) == 2 and call(rdt=4) == 2 and call(bias=16, bdt=4) == 2
    assert call(p=16, K=40) == 4          # K not a multiple of 16
    assert call(p=16) == 6                # no workspace
    assert call(p=16, ws=128, wsb=1 << 20) == 4


def test_route_refusals(lib):
    def call(dt=_lib.F32, ldl=16, M=4, E=16, scoring=0, groups=1, tg=1, gs=0, k=2):
        return lib.fnn_moe_route(None, dt, ldl, M, E, None, scoring, 1, groups, tg, gs, 1.0, k, None, None, None)

    assert call() == 1
    assert call(M=0) == 0
    assert call(M=-1) == 3 and call(E=0) == 3 and call(ldl=15) == 3 and call(k=0) == 3 and call(k=17) == 3
    assert call(groups=3) == 3 and call(groups=4, tg=5) == 3 and call(groups=4, tg=0) == 3 and call(groups=4, tg=1, k=5) == 3
    assert call(E=1025, ldl=1025) == 5 and call(E=64, ldl=64, k=33) == 5 and call(E=128, ldl=128, groups=64, tg=64) == 5
    assert call(dt=3) == 2 and call(scoring=2) == 5 and call(gs=2) == 5


def test_sort_refusals_and_slot_count(lib):
    def call(n=8, E=4, first=0, bm=16, em=None):
        return lib.fnn_moe_sort(None, n, E, first, bm, None, lib.fnn_moe_sort_slots(n, E, bm) if em is None else em, None, None, None)

    assert call() == 1
    assert call(n=0) == 1  # the count of slots in use is written all the same
    assert call(n=-1, em=0) == 3 and call(E=0, em=0) == 3 and call(bm=0, em=0) == 3 and call(em=16) == 3
    assert call(first=2 ** 40) == 3 and call(E=1025) == 5 and call(n=2 ** 31) == 3
    # no choice of experts fills more: n experts with one choice each, the rest in whole blocks
    assert lib.fnn_moe_sort_slots(0, 8, 16) == 0
    assert lib.fnn_moe_sort_slots(2, 8, 16) == 32
    for n, e, bm in [(5, 3, 2), (7, 2, 4), (6, 6, 1), (4, 8, 3)]:
        from itertools import combinations_with_replacement
        most = max(sum(-(-pick.count(x) // bm) for x in set(pick)) for pick in combinations_with_replacement(range(e), n))
        assert lib.fnn_moe_sort_slots(n, e, bm) == most * bm


def test_combine_refusals(lib):
    def call(dt=_lib.BF16, ldm=64, ldk=32, M=4, k=2, N=32, ids=None, E=1, first=0, res=None, ldr=0, ldo=32):
        return lib.fnn_moe_combine(None, dt, ldm, ldk, M, k, N, None, ids, E, first, res, ldr, None, ldo, None)

    assert call() == 1
    assert call(M=0) == 0 and call(N=0) == 0
    assert call(M=-1) == 3 and call(k=-1) == 3 and call(ldo=31) == 3 and call(ids=16, E=0) == 3 and call(res=16, ldr=-1) == 3
    assert call(ids=16, first=2 ** 40) == 3
    assert call(dt=_lib.F32) == 2


def test_modules_check_their_arguments():
    with pytest.raises(AssertionError, match="unknown activation"):
        flashnn_b200.GemmA8W8Epilogue(activation="swish")
    for bad in (dict(scoring="relu"), dict(group_score="mean"), dict(num_groups=3), dict(num_groups=4, topk_groups=5),
                dict(num_groups=4, topk_groups=1, top_k=5), dict(top_k=0), dict(top_k=17)):
        with pytest.raises(AssertionError):
            flashnn_b200.MoeRouting(**dict(dict(num_experts=16, top_k=2), **bad))


def test_cpu_tensors_are_rejected():
    a = torch.zeros(4, 64, dtype=torch.int8)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: flashnn_b200.GemmA8W8Epilogue()(a, a, torch.ones(4), torch.ones(4)),
                 lambda: flashnn_b200.MoeRouting(8, 2)(torch.zeros(4, 8)),
                 lambda: flashnn_b200.moe_sort_tokens(ids, 8, 16),
                 lambda: flashnn_b200.moe_combine(torch.zeros(4, 2, 8).half()),
                 lambda: flashnn_b200.fused_moe_a8w8_gated_forward(a, a.view(2, 2, 64), torch.zeros(4, 2, 1).half(), torch.ones(4),
                                                                   torch.ones(2, 2), ids, ids.view(-1), ids.view(-1), ids.view(-1), 2, 16)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_the_oracle_against_elementary_forms():
    """The 64-bit forms that the GPU tests use, where a few lines of torch say the same."""
    from oracle import feed_forward as O
    g = torch.Generator().manual_seed(0)
    x = torch.randn(16, 12, generator=g)
    w, ids = O.route(x, 3)
    p, i = torch.softmax(x.double(), 1).topk(3)
    assert torch.equal(i.int(), ids) and torch.allclose(w, p / p.sum(1, keepdim=True), rtol=1e-12, atol=0)
    v = torch.linspace(-30, 30, 601, dtype=torch.float64)
    f = torch.nn.functional
    for name, fn in (("relu", f.relu), ("sigmoid", torch.sigmoid), ("silu", f.silu), ("gelu", f.gelu),
                     ("gelu_tanh", lambda t: f.gelu(t, approximate="tanh"))):
        assert torch.allclose(O.activate(v, name), fn(v), rtol=1e-9, atol=1e-14)
        assert ((O.activate(v[1:], name) - O.activate(v[:-1], name)).abs() <= 1.13 * (v[1] - v[0])).all()  # the steepness the bounds use
    ids = torch.randint(-1, 5, (9, 2), generator=g)
    slots, experts, used = O.sort_slots(ids, 4, 4)
    for s in range(int(used)):
        if slots[s] < 18:
            assert ids.view(-1)[slots[s]] == experts[s // 4]
