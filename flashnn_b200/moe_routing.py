"""The two ends of a mixture-of-experts layer: MoeRouting turns router logits into each token's experts and weights,
moe_sort_tokens turns those into the block-aligned slot list that the expert products (fused_moe_a8w8_forward,
fused_moe_a8w8_gated_forward, fused_moe_a16w4_forward) read, and moe_combine sums their [M, top_k, N] output over a
token's choices."""
import torch

from . import _lib
from .kernel_backend import BackendKernel
from .quant_gemm import _DT, _flat, _launch, _one_device


def _ids32(t):
    """Expert numbers as int32; what does not fit stays outside every range of experts."""
    return t if t.dtype == torch.int32 else t.clamp(-1, 2 ** 31 - 1).to(torch.int32)


class MoeRouting(BackendKernel):
    """forward(logits [M, E] fp16/bf16/fp32, bias=None or [E]) -> (topk_weights [M, top_k] fp32, topk_ids [M, top_k] int32)

    score = softmax(logits) or sigmoid(logits); the experts with the `top_k` largest score + bias are chosen, best first,
    equal ones by the lowest index; their weights are the scores (without the bias), divided by their sum if `renormalize`,
    times `scale`.  With num_groups > 1 only the experts of the best `topk_groups` groups of E / num_groups consecutive ones
    can be chosen; a group's score is the largest score + bias in it ("max") or the sum of its two largest ("top2").
    The order is that of 64-bit arithmetic; the bias is taken in fp32.

    Taking an expert out: without a bias by a logit of -inf; with one by a bias of -inf, under either scoring.  With a bias a logit of
    -inf only makes the score 0: the expert still competes with bias[e], ahead of live experts whose score + bias is below that,
    and has the weight 0 if it wins.  An expert that is out is chosen only where fewer than top_k others can be."""

    def __init__(self, num_experts: int, top_k: int, scoring: str = "softmax", renormalize: bool = True, num_groups: int = 1,
                 topk_groups: int = 1, group_score: str = "max", scale: float = 1.0):
        super().__init__()
        assert scoring in _lib.SCORINGS, f"unknown scoring {scoring!r}"
        assert group_score in _lib.GROUP_SCORES, f"unknown group score {group_score!r}"
        assert num_groups >= 1 and num_experts % num_groups == 0, "num_groups must divide num_experts"
        assert 1 <= topk_groups <= num_groups, "topk_groups must be between 1 and num_groups"
        assert 1 <= top_k <= topk_groups * (num_experts // num_groups), "top_k must not exceed the experts of the chosen groups"
        self.num_experts, self.top_k = num_experts, top_k
        self.scoring, self.renormalize, self.scale = scoring, bool(renormalize), float(scale)
        self.num_groups, self.topk_groups, self.group_score = num_groups, topk_groups, group_score
        self._scoring, self._group_score = _lib.SCORINGS[scoring], _lib.GROUP_SCORES[group_score]

    def _cuda_impl(self, logits, bias=None):
        index = _one_device(logits, bias)
        assert logits.dim() == 2 and logits.shape[1] == self.num_experts, "logits must be [M, num_experts]"
        dt = _DT.get(logits.dtype)
        assert dt is not None, "logits must be float16, bfloat16 or float32"
        m, e = logits.shape
        ldl = e
        if not logits.is_contiguous():
            if e > 1 and logits.stride(1) != 1 or m > 1 and logits.stride(0) < e:  # (or a broadcast one)
                logits = logits.contiguous()
            elif m > 1:
                ldl = logits.stride(0)
        bias_ptr = None
        if bias is not None:
            assert bias.numel() == e and bias.is_floating_point(), "bias must be [num_experts]"
            bias = _flat(bias if bias.dtype == torch.float32 else bias.float())
            bias_ptr = bias.data_ptr()
        weights = logits.new_empty((m, self.top_k), dtype=torch.float32)
        ids = logits.new_empty((m, self.top_k), dtype=torch.int32)
        _launch(index, _lib.lib().fnn_moe_route, logits.data_ptr(), dt, ldl, m, e, bias_ptr, self._scoring, self.renormalize,
                self.num_groups, self.topk_groups, self._group_score, self.scale, self.top_k, weights.data_ptr(), ids.data_ptr())
        return weights, ids

    def forward(self, logits, bias=None):
        return BackendKernel.forward(self, logits, bias)


def moe_sort_tokens(topk_ids, num_experts, BM, first_expert=0):
    """topk_ids [M, top_k] -> (sorted_token_ids [EM], expert_ids [EM / BM], num_tokens_post_padded [1]), int32: the flat
    (token, choice) indices grouped by expert in ascending order, every group padded to a multiple of BM with M * top_k.

    Experts are first_expert .. first_expert + num_experts - 1 and numbered from 0 in expert_ids; a choice of any other
    expert (one of another device, or -1) gets no slot.  EM depends on the sizes alone: the most slots that any choice of
    experts fills."""
    index = _one_device(topk_ids)
    assert topk_ids.dtype in (torch.int32, torch.int64), "topk_ids must be int32 or int64"
    assert num_experts >= 1 and BM >= 1, "num_experts and BM must be positive"
    assert first_expert >= 0, "first_expert must not be negative"
    assert first_expert + num_experts < 2 ** 31, "expert numbers must be below 2^31 - 1"  # (64-bit ones are cut off there)
    ids = _ids32(topk_ids)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    n = ids.numel()
    used = min(n, num_experts)
    blocks = used + (n - used) // BM  # fnn_moe_sort_slots
    em = blocks * BM
    # one allocation, three views
    sorted_ids, experts, in_use = ids.new_empty(em + blocks + 1).split((em, blocks, 1))
    _launch(index, _lib.lib().fnn_moe_sort, ids.data_ptr(), n, num_experts, first_expert, BM, sorted_ids.data_ptr(), em,
            experts.data_ptr(), in_use.data_ptr())
    return sorted_ids, experts, in_use


def moe_combine(C, topk_weights=None, topk_ids=None, num_experts=None, first_expert=0, residual=None):
    """C [M, top_k, N] fp16/bf16 -> [M, N] in C's dtype: the sum over a token's choices, times topk_weights [M, top_k] where
    given (the expert products can have applied them), plus residual [M, N], in fp32 and rounded once.

    With topk_ids [M, top_k] choices of experts outside first_expert .. first_expert + num_experts - 1 are left out: the
    expert products did not write their rows of C, which are not read."""
    index = _one_device(C, topk_weights, topk_ids, residual)
    dt = _DT.get(C.dtype)
    assert C.dim() == 3 and dt is not None and dt != _lib.F32, "C must be [M, top_k, N] in float16 or bfloat16"
    m, k, n = C.shape
    ldm, ldk = k * n, n
    if not C.is_contiguous():
        if n > 1 and C.stride(2) != 1:
            C = C.contiguous()
        else:
            ldm, ldk = C.stride(0) if m > 1 else ldm, C.stride(1) if k > 1 else n
    w_ptr = ids_ptr = res_ptr = None
    if topk_weights is not None:
        assert topk_weights.shape == (m, k) and topk_weights.dtype in _DT, "topk_weights must be [M, top_k] in a float dtype"
        topk_weights = topk_weights if topk_weights.dtype == torch.float32 else topk_weights.float()
        if not topk_weights.is_contiguous():
            topk_weights = topk_weights.contiguous()
        w_ptr = topk_weights.data_ptr()
    experts = 1
    if topk_ids is not None:
        assert topk_ids.shape == (m, k) and num_experts is not None and num_experts >= 1, "topk_ids must be [M, top_k], with num_experts"
        assert topk_ids.dtype in (torch.int32, torch.int64), "topk_ids must be int32 or int64"
        assert first_expert >= 0, "first_expert must not be negative"
        assert first_expert + num_experts < 2 ** 31, "expert numbers must be below 2^31 - 1"
        topk_ids, experts = _ids32(topk_ids), num_experts
        if not topk_ids.is_contiguous():
            topk_ids = topk_ids.contiguous()
        ids_ptr = topk_ids.data_ptr()
    ldr = n
    if residual is not None:
        assert residual.shape == (m, n) and residual.dtype == C.dtype, "residual must be [M, N] in C's dtype"
        if not residual.is_contiguous():
            if n > 1 and residual.stride(1) != 1:
                residual = residual.contiguous()
            elif m > 1:
                ldr = residual.stride(0)
        res_ptr = residual.data_ptr()
    out = C.new_empty((m, n))
    _launch(index, _lib.lib().fnn_moe_combine, C.data_ptr(), dt, ldm, ldk, m, k, n, w_ptr, ids_ptr, experts, first_expert,
            res_ptr, ldr, out.data_ptr(), n)
    return out
