"""The scratch that the products keep per stream, and the calls that must not share it: those captured into graphs."""
import types

import pytest
import torch


def test_a_captured_call_gets_a_workspace_of_its_own(monkeypatch):
    from flashnn_b200 import quant_gemm as Q
    capturing = [False]
    monkeypatch.setattr(Q, "_workspaces", type(Q._workspaces)())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing[0], raising=False)
    cpu = torch.device("cpu")
    eager = Q._workspace(cpu, 100)
    assert Q._workspace(cpu, 200) is eager  # one buffer for the stream
    capturing[0] = True
    first, second = Q._workspace(cpu, 100), Q._workspace(cpu, 100)
    assert len({t.data_ptr() for t in (eager, first, second)}) == 3 and first.numel() >= 100
    capturing[0] = False
    assert Q._workspace(cpu, 100) is eager and list(Q._workspaces.values()) == [eager]


def _layer(x, gate_w, up, up_col, down, down_col):
    """The whole int8 mixture-of-experts layer, second product with its routing weights and all."""
    import flashnn_b200 as F
    m, (e, hidden, inter) = x.shape[0], down.shape
    q, s = F.DynamicQuantize()(x)
    w, ids = F.MoeRouting(e, 2, scoring="sigmoid")(x.float() @ gate_w.t())
    plan = F.moe_sort_tokens(ids, e, 16)
    h = torch.empty(m, 2, inter, dtype=x.dtype, device=x.device)
    F.fused_moe_a8w8_gated_forward(q, up, h, s, up_col, ids, *plan, 2, 16)
    hq, hs = F.DynamicQuantize()(h.view(m * 2, inter))
    y = torch.empty(m * 2, 1, hidden, dtype=x.dtype, device=x.device)
    F.fused_moe_a8w8_forward(hq, down, y, hs, down_col, w.view(-1, 1), ids.view(-1, 1), *plan, True, 1, 16)
    return F.moe_combine(y.view(m, 2, hidden), topk_ids=ids, num_experts=e, residual=x)


@pytest.mark.gpu
def test_two_graphs_of_calls_with_workspaces_replay_side_by_side():
    """A layer whose second product gathers its rows into a workspace and a weight-only product whose zero-points need one, captured
    twice on one stream and replayed on two beside eager calls."""
    import flashnn_b200 as F
    from flashnn_b200 import _lib
    from tests.test_gpu_feed_forward import layer_case
    m, n, k = 512, 1024, 512

    def problem(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        wo = (torch.randn(m, k, generator=g, device="cuda").half(), torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8),
              torch.rand(n, generator=g, device="cuda").half() * 0.01, None, torch.randint(-3, 4, (n,), generator=g, device="cuda").half())
        return layer_case(200, seed=seed), wo

    def run(p):
        return [_layer(*p[0]), F.GemmWeightOnly(torch.float16)(*p[1])]
    assert _lib.lib().fnn_gemm_weight_only_workspace_bytes(m, n, k, 8, 0) > 0
    problems = [problem(s) for s in range(3)]
    want = [[t.clone() for t in run(p)] for p in problems]
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in problems[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(run(p))
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(side):
            eager = run(problems[2])
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
        for out in outs:
            for t in out:
                t.zero_()
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_a_captured_hand_over_of_partial_sums_in_memory_that_the_graph_reuses():
    """The product whose CTA pairs hand partial sums over keeps flags in its workspace, which needs no initialisation: replayed alone,
    with other tensors in the same memory between its two calls and behind them."""
    import flashnn_b200 as F
    from flashnn_b200 import _lib
    m, n, k = 4096, 2048, 16384
    need = _lib.lib().fnn_gemm_a8w8_workspace_bytes(m, n, k)
    assert need > 0
    g = torch.Generator(device="cuda").manual_seed(0)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
    row, col = torch.rand(m, generator=g, device="cuda") * 0.01, torch.rand(n, generator=g, device="cuda") * 0.001
    f = F.GemmA8W8(torch.bfloat16)
    want = [f(a, b, row, col).clone(), f(a.flip(0), b, row, col).clone()]
    rev = a.flip(0).contiguous()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = f(a, b, row, col)
        torch.ones(need // 8, dtype=torch.int64, device="cuda")
        second = f(rev, b, row, col)
        torch.full((need // 8,), -1, dtype=torch.int64, device="cuda")
    for _ in range(4):
        first.zero_()
        second.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want[0]) and torch.equal(second, want[1])
    assert _lib.device_status() == 0
