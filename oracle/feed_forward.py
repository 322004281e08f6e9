"""Feed-forward operators in 64 bits, from their definitions: the A8W8 product with a fused epilogue, gated expert products,
routing, the expert sort and the sum over a token's choices.  Test infrastructure: nothing in the package imports it."""
import math

import torch

ACTIVATIONS = ("none", "relu", "sigmoid", "silu", "gelu", "gelu_tanh")
U32 = 2.0 ** -24  # half a step of fp32, relative


def activate(v, name):
    sig = torch.special.expit
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "sigmoid":
        return sig(v)
    if name == "silu":
        return v * sig(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    if name == "gelu_tanh":
        return v * sig(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def activation_error(v, y, name):
    """How far an fp32 evaluation at v may be off y = activate(v): the hardware exponential is within 2 + 1.173 |x| steps of
    2^-23, reciprocal, sum and products within 6 more; where the sigmoid, also the one that gelu_tanh multiplies v by, is below 2^-126
    (|v| < 2^7) it may be taken as 0.
    GELU: v times a tail whose error is relative to itself: the exponential 4 roundings of 2^-24 and its argument at most 2 v^2, the
    reciprocal 2 and its argument 1 (either weighs at most 1.7 in the tail), the fit 1.6, Horner's scheme and the products 6;
    below 20 + 2 v^2 together.  Near 0, where half of that goes into Phi, an evaluation in 32 bits with the reciprocal one step
    off either way is within 3.5 |v| roundings.  Where e^(-v^2 / 2) is below 2^-126 the result may be 0."""
    if name in ("sigmoid", "silu"):
        return y.abs() * 2 * U32 * (8 + 1.2 * v.abs()) + 2.0 ** -119
    if name == "gelu":
        return torch.minimum(v.abs() * 4 * U32, y.abs() * U32 * (20 + 2 * v * v) + 2.0 ** -119)
    if name == "gelu_tanh":
        t = math.sqrt(8 / math.pi) * (v.abs() + 0.044715 * v.abs() ** 3)
        return y.abs() * 2 * U32 * (8 + 4 * t) + 2.0 ** -119  # the argument's own four roundings included
    return torch.zeros_like(y)


def scale_of(alpha_row, alpha_col, rounded_alike=True):
    """[M, N] in 64 bits: row scale * column scale, rounded to their dtype where both share a 16-bit one (exactly as the plain
    A8W8 product takes it), otherwise unrounded."""
    s = alpha_row.reshape(-1, 1).double() * alpha_col.reshape(1, -1).double()
    if rounded_alike and alpha_row.dtype == alpha_col.dtype and alpha_row.dtype != torch.float32:
        s = s.float().to(alpha_row.dtype).double()
    return s


def finish(v, err, gated, act, residual, out_ty):
    """(value, bound) of the epilogue on v +- err in 64 bits; v has the gate's columns first.  No activation here is steeper
    than 1.13."""
    n = v.shape[-1] // 2 if gated else v.shape[-1]
    g, eg = v[..., :n], err[..., :n]
    y = activate(g, act)
    e = 1.13 * eg + activation_error(g, y, act)
    if gated:
        u, eu = v[..., n:], err[..., n:]
        e = e * (u.abs() + eu) + y.abs() * eu
        y = y * u
        e = e + y.abs() * U32
    if residual is not None:
        y = y + residual.double()
        e = e + y.abs() * U32
    # the rounding to the output type: half a step, or half the smallest subnormal
    info = torch.finfo(out_ty)
    return y, e * 1.01 + (y.abs() + e) * (info.eps / 2) + info.smallest_normal * info.eps / 2


def gemm_epilogue(a, b, alpha_row, alpha_col, bias, act, gated, residual, out_ty):
    """(value, bound): every element of a right fp32 evaluation is within `bound` of `value`."""
    acc = a.double() @ b.double().t()
    p = acc * scale_of(alpha_row, alpha_col)
    # float(acc), the scales' product, their product: one rounding each; adding the bias rounds once more
    err = 3 * U32 * p.abs()
    if bias is not None:
        p = p + bias.reshape(1, -1).double()
        err = err + p.abs() * U32
    return finish(p, err, gated, act, residual, out_ty)


def experts_gated(a, b, alpha_row, alpha_col, bias, act, topk_ids, out_ty):
    """(value, bound) [M, top_k, N]; NaN in the rows of choices that are not in [0, E)."""
    m, k = topk_ids.shape
    n = b.shape[1] // 2
    value = torch.full((m * k, n), math.nan, dtype=torch.float64, device=a.device)
    bound = torch.zeros_like(value)
    flat = topk_ids.reshape(-1).to(a.device)
    for e in range(b.shape[0]):
        at = (flat == e).nonzero().flatten()
        if not at.numel():
            continue
        tok = at // k
        p = (a[tok].double() @ b[e].double().t()) * scale_of(alpha_row[tok], alpha_col[e], rounded_alike=False)
        err = 3 * U32 * p.abs()
        if bias is not None:
            p = p + bias[e].reshape(1, -1).double()
            err = err + p.abs() * U32
        value[at], bound[at] = finish(p, err, True, act, None, out_ty)
    return value.view(m, k, n), bound.view(m, k, n)


def route(logits, top_k, bias=None, scoring="softmax", renormalize=True, num_groups=1, topk_groups=1, group_score="max", scale=1.0):
    """(weights in 64 bits, ids), row by row."""
    weights, ids = [], []
    e = logits.shape[1]
    for row in logits.double().tolist():
        if scoring == "softmax":
            top = max((v for v in row if v == v), default=0.0)
            top = 0.0 if math.isinf(top) else top
            p = [math.exp(v - top) if v < math.inf else v for v in row]
            total = sum(p)
            p = [v / (total if total != 0 else 1.0) if not (v == total == math.inf) else math.nan for v in p]
        else:
            p = [1 / (1 + math.exp(-v)) if v > -700 else (v if v != v else math.exp(v)) for v in row]
        summed = num_groups > 1 and group_score == "top2"
        if bias is None and not summed:
            key = row
        else:
            key = [v if bias is None else v + float(bias[i]) for i, v in enumerate(p)]
        key = [-math.inf if v != v else v for v in key]
        allowed = range(e)
        if num_groups > 1:
            size = e // num_groups
            score = []
            for g in range(num_groups):
                best = sorted(key[g * size:(g + 1) * size], reverse=True)
                score.append(best[0] + best[1] if summed and size > 1 else best[0])
            score = [-math.inf if v != v else v for v in score]
            chosen = sorted(range(num_groups), key=lambda g: (-score[g], g))[:topk_groups]
            allowed = [i for i in range(e) if i // size in chosen]
        best = sorted(allowed, key=lambda i: (-key[i], i))[:top_k]
        w = [p[i] for i in best]
        if renormalize:
            total = sum(w)
            w = [v / (total if total != 0 else 1.0) for v in w]
        weights.append([v * scale for v in w])
        ids.append(best)
    return torch.tensor(weights, dtype=torch.float64).reshape(-1, top_k), torch.tensor(ids, dtype=torch.int32).reshape(-1, top_k)


def sort_slots(topk_ids, num_experts, bm, first_expert=0):
    flat = topk_ids.reshape(-1).tolist()
    slots, experts = [], []
    for e in range(num_experts):
        mine = [i for i, v in enumerate(flat) if v == e + first_expert]
        blocks = -(-len(mine) // bm)
        slots += mine + [len(flat)] * (blocks * bm - len(mine))
        experts += [e] * blocks
    in_use = len(slots)
    used = min(len(flat), num_experts)
    blocks = used + (len(flat) - used) // bm if flat else 0
    slots += [len(flat)] * (blocks * bm - in_use)
    experts += [0] * (blocks - len(experts))
    i32 = dict(dtype=torch.int32)
    return torch.tensor(slots, **i32), torch.tensor(experts, **i32), torch.tensor([in_use], **i32)


def combine(c, topk_weights=None, topk_ids=None, num_experts=None, first_expert=0, residual=None):
    """(value, bound)."""
    m, k, n = c.shape
    x = c.double()
    if topk_ids is not None:
        here = (topk_ids >= first_expert) & (topk_ids < first_expert + num_experts)
        x = torch.where(here[:, :, None], x, torch.zeros_like(x))
    if topk_weights is not None:
        x = x * topk_weights.double()[:, :, None]
    size = x.abs().sum(1)
    v = x.sum(1)
    if residual is not None:
        v = v + residual.double()
        size = size + residual.double().abs()
    info = torch.finfo(c.dtype)
    err = (k + 1) * U32 * size  # one rounding per fused multiply-add of at most `size`
    return v, 1.01 * err + (v.abs() + err) * (info.eps / 2) + info.smallest_normal * info.eps / 2
