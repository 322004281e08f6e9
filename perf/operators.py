"""Cases of the feed-forward operators: the int8 product with bias, activation, gate and residual in its epilogue, the
gated expert products, expert routing, the expert sort and the sum over a token's choices.

`run` computes them with elementary torch operations where `own` is false and with the framework's operators where it
is true, from the same inputs.  `exact` gives the same results in 64 bits from the definitions."""
import math

import torch

own = False

if torch.cuda.is_available():
    DEVICE = torch.device("cuda")
else:
    DEVICE = torch.device("cpu")

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = ("none", "relu", "sigmoid", "silu", "gelu", "gelu_tanh")


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through the gate/up projection of the 70B-shaped feed-forward layer: a decode step
        dict(name="gemm decode gated", op="gemm", m=1, n=28672, k=8192, act="silu", gated=True, bias=False, residual=False, dtype="bf16"),
        # sixteen tokens, a small projection with everything in the epilogue
        dict(name="gemm 16 tokens", op="gemm", m=16, n=4096, k=4096, act="gelu", gated=False, bias=True, residual=True, dtype="fp16"),
        # the down projection of a ragged prefill batch, added to the residual stream
        dict(name="gemm down ragged", op="gemm", m=1037, n=8192, k=28672, act="none", gated=False, bias=False, residual=True, dtype="bf16"),
        # the gate/up projection of a prefill batch
        dict(name="gemm prefill gated", op="gemm", m=4096, n=28672, k=8192, act="silu", gated=True, bias=False, residual=False, dtype="bf16"),
        # a decode batch over eight experts, two choices each: bound by the expert weights
        dict(name="experts decode", op="experts", m=64, n=14336, k=4096, e=8, top_k=2, bm=16, act="silu", bias=False, dropped=0.0, dtype="bf16"),
        # a prefill batch over the same experts
        dict(name="experts prefill", op="experts", m=4096, n=14336, k=4096, e=8, top_k=2, bm=256, act="silu", bias=False, dropped=0.0, dtype="bf16"),
        # one token, softmax over eight experts
        dict(name="route one token", op="route", m=1, e=8, top_k=2, scoring="softmax", groups=1, topk_groups=1, group_score="max",
             bias=False, masked=0.0, dtype="bf16"),
        # a prefill batch, sigmoid scores with a balancing bias and group-limited choice
        dict(name="route grouped", op="route", m=16384, e=256, top_k=8, scoring="sigmoid", groups=8, topk_groups=4, group_score="top2",
             bias=True, masked=0.0, dtype="fp32"),
        # the slot list of a decode batch
        dict(name="sort decode", op="sort", m=64, e=8, top_k=2, bm=16, first=0, dropped=0.0),
        # the slot list of a prefill batch over many experts
        dict(name="sort prefill", op="sort", m=16384, e=256, top_k=8, bm=128, first=0, dropped=0.0),
        # a decode batch's choices added up, the routing weights applied already
        dict(name="combine decode", op="combine", m=64, n=4096, top_k=2, weights=False, residual=True, dropped=0.0, dtype="bf16"),
        # a prefill batch with many choices per token, some of them on another device
        dict(name="combine prefill", op="combine", m=4096, n=4096, top_k=8, weights=True, residual=True, dropped=0.125, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "experts", "route", "sort", "combine"])
    sixteen = rng.choice(["bf16", "fp16"])
    if op == "gemm":
        # any number of tokens and output columns, K in steps of 16 bytes; at most the prefill case's work
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 16, 28672), 16 * _log(rng, 4, 1792)
            if rng.random() < 0.5:
                n = -(-n // 16) * 16
            if rng.random() < 0.25:
                k = 4096 * rng.randint(1, 7)
            gated = rng.random() < 0.5
            if m * n * (2 if gated else 1) * k <= 4096 * 57344 * 8192:
                break
        return dict(op=op, m=m, n=n, k=k, act=rng.choice(ACTIVATIONS), gated=gated, bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5, dtype=sixteen)
    if op == "experts":
        while True:
            m, n, k, e = _log(rng, 1, 4096), 16 * _log(rng, 1, 896), 16 * _log(rng, 4, 512), _log(rng, 2, 64)
            top_k, bm = rng.randint(1, min(8, e)), rng.choice([16, 32, 64, 128, 256])
            # the plain form works block by block: no more block-sized weights than the prefill case has
            if (min(m * top_k, e) + m * top_k // bm) * 2 * n * k <= 40 * 28672 * 4096 and m * top_k * n * k <= 8192 * 14336 * 4096:
                break
        return dict(op=op, m=m, n=n, k=k, e=e, top_k=top_k, bm=bm, act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5,
                    dropped=rng.choice([0.0, 0.0, 0.3]), dtype=sixteen)
    if op == "route":
        m, groups = _log(rng, 1, 16384), rng.choice([1, 1, 2, 4, 8])
        e = groups * max(2, _log(rng, 4, 512) // groups)
        topk_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, topk_groups * (e // groups)))
        return dict(op=op, m=m, e=e, top_k=top_k, scoring=rng.choice(["softmax", "sigmoid"]), groups=groups, topk_groups=topk_groups,
                    group_score=rng.choice(["max", "top2"]), bias=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.2]),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "sort":
        return dict(op=op, m=_log(rng, 1, 16384), e=_log(rng, 2, 512), top_k=rng.randint(1, 8), bm=rng.choice([16, 32, 64, 128, 256]),
                    first=rng.choice([0, 0, 5]), dropped=rng.choice([0.0, 0.0, 0.3]))
    while True:
        m, n, top_k = _log(rng, 1, 16384), _log(rng, 64, 8192), rng.randint(1, 16)
        if m * n * top_k <= 4096 * 4096 * 8:
            break
    return dict(op=op, m=m, n=n, top_k=top_k, weights=rng.random() < 0.5, residual=rng.random() < 0.5,
                dropped=rng.choice([0.0, 0.0, 0.3]), dtype=sixteen)


def work(c):
    m = c["m"]
    if c["op"] == "gemm":
        rows = c["n"] * (2 if c["gated"] else 1)  # weight rows
        out = m * c["n"] * 2
        nbytes = m * c["k"] + rows * c["k"] + 2 * m + 4 * rows + out * (2 if c["residual"] else 1) + (2 * rows if c["bias"] else 0)
        return dict(bytes=nbytes, flops=2 * m * rows * c["k"])
    if c["op"] == "experts":
        rows, choices = 2 * c["n"], m * c["top_k"]
        used = min(c["e"], choices)
        nbytes = m * c["k"] + used * rows * (c["k"] + 4) + choices * c["n"] * 2 + (2 * used * rows if c["bias"] else 0)
        return dict(bytes=nbytes, flops=2 * choices * rows * c["k"])
    if c["op"] == "route":
        size = DTYPES[c["dtype"]].itemsize
        return dict(bytes=m * c["e"] * size + m * c["top_k"] * 8 + (4 * c["e"] if c["bias"] else 0), flops=4 * m * c["e"])
    if c["op"] == "sort":
        slots = _blocks(m * c["top_k"], c["e"], c["bm"]) * c["bm"]
        return dict(bytes=4 * (m * c["top_k"] + slots + slots // c["bm"] + 1), flops=m * c["top_k"])
    rows = c["top_k"] + 1 + int(c["residual"])
    return dict(bytes=rows * m * c["n"] * 2 + m * c["top_k"] * (8 if c["weights"] else 4), flops=2 * m * c["n"] * c["top_k"])


def _blocks(choices, e, bm):
    """Most blocks of bm slots that `choices` choices among e experts can fill."""
    used = min(choices, e)
    return used + (choices - used) // bm


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
class _Inputs:
    """Seeded inputs on the device."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEVICE)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device=DEVICE) * (hi - lo) + lo

    def int8(self, *shape):
        return torch.randint(-127, 128, shape, generator=self.g, device=DEVICE, dtype=torch.int8)

    def choices(self, m, e, top_k, dropped):
        """[m, top_k] different experts per token, a share of them -1 (their experts are on another device)."""
        ids = torch.argsort(torch.rand((m, e), generator=self.g, device=DEVICE), dim=1)[:, :top_k].to(torch.int32)
        if dropped:
            ids[torch.rand((m, top_k), generator=self.g, device=DEVICE) < dropped] = -1
        return ids.contiguous()


def prepare(case, seed):
    c, r = dict(case), _Inputs(seed)
    m = c["m"]
    if c["op"] in ("gemm", "experts"):
        n, k = c["n"], c["k"]
        rows = n * (2 if c["op"] == "experts" or c["gated"] else 1)
        lead = (c["e"],) if c["op"] == "experts" else ()
        dtype = DTYPES[c["dtype"]]
        s = dict(c, a=r.int8(m, k), b=r.int8(*lead, rows, k))
        # the scales a quantiser gives such rows: products come out near N(0, 1)
        s["alpha_row"] = r.uniform(0.005, 0.02, m).half()
        s["alpha_col"] = r.uniform(0.5, 1.5, *lead, rows) / (0.0125 * 5376 * math.sqrt(k))
        s["b_bias"] = r.normal(*lead, rows).to(dtype) if c["bias"] else None
        if c["op"] == "gemm":
            s["r"] = r.normal(m, n).to(dtype) if c["residual"] else None
            if own:
                import flashnn_b200
                s["f"] = flashnn_b200.GemmA8W8Epilogue(dtype, activation=c["act"], gated=c["gated"])
        else:
            s["ids"] = r.choices(m, c["e"], c["top_k"], c["dropped"])
            s["plan"] = _plain_sort(s["ids"], c["e"], c["bm"], 0)
            s["c"] = torch.full((m, c["top_k"], n), 7.0, dtype=dtype, device=DEVICE)  # rows of dropped choices stay
        return s
    if c["op"] == "route":
        s = dict(c, x=(2 * r.normal(m, c["e"])).to(DTYPES[c["dtype"]]), b=r.uniform(-0.2, 0.2, c["e"]) if c["bias"] else None, scale=2.5)
        if c["masked"]:
            s["x"][:, torch.rand(c["e"], generator=r.g, device=DEVICE) < c["masked"]] = -math.inf  # experts taken out
        if own:
            import flashnn_b200
            s["f"] = flashnn_b200.MoeRouting(c["e"], c["top_k"], scoring=c["scoring"], renormalize=True, num_groups=c["groups"],
                                             topk_groups=c["topk_groups"], group_score=c["group_score"], scale=2.5)
        return s
    if c["op"] == "sort":
        # experts are not equally popular
        weight = torch.exp(0.5 * r.normal(c["e"])).expand(m * c["top_k"], -1)
        ids = torch.multinomial(weight[0], m * c["top_k"], replacement=True, generator=r.g).to(torch.int32) + c["first"]
        ids = torch.where(r.uniform(0, 1, m * c["top_k"]) < c["dropped"], torch.full_like(ids, -1), ids)
        return dict(c, ids=ids.view(m, c["top_k"]))
    dtype = DTYPES[c["dtype"]]
    s = dict(c, c=r.normal(m, c["top_k"], c["n"]).to(dtype), r=r.normal(m, c["n"]).to(dtype) if c["residual"] else None)
    s["w"] = r.uniform(0.0, 1.0, m, c["top_k"]) if c["weights"] else None
    s["ids"] = torch.randint(0, 64, (m, c["top_k"]), generator=r.g, device=DEVICE, dtype=torch.int32)
    if c["dropped"]:
        gone = r.uniform(0, 1, m, c["top_k"]) < c["dropped"]
        s["ids"][gone] = -1
        s["c"][gone] = math.nan  # rows that nothing has written
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _act(v, name):
    if name == "relu":
        return torch.clamp_min(v, 0)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_gemm(s):
    v = s["a"].float() @ s["b"].float().t()
    v = v * (s["alpha_row"].float()[:, None] * s["alpha_col"].float()[None, :])
    if s["b_bias"] is not None:
        v = v + s["b_bias"].float()
    v = _act(v[:, :s["n"]], s["act"]) * v[:, s["n"]:] if s["gated"] else _act(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(DTYPES[s["dtype"]])


def _plain_experts(s):
    slots, experts, _ = s["plan"]
    choices, bm, n = s["m"] * s["top_k"], s["bm"], s["n"]
    here = slots < choices
    rows = torch.where(here, slots, 0).long() // s["top_k"]
    e = experts.long()
    v = torch.bmm(s["a"][rows].float().view(-1, bm, s["k"]), s["b"][e].float().transpose(1, 2))
    v = v * s["alpha_row"].float()[rows].view(-1, bm, 1) * s["alpha_col"].float()[e][:, None, :]
    if s["b_bias"] is not None:
        v = v + s["b_bias"].float()[e][:, None, :]
    v = _act(v[..., :n], s["act"]) * v[..., n:]
    # slots without a choice write to a row behind the last, which is dropped
    flat = torch.cat([s["c"].view(choices, n), s["c"].new_zeros(1, n)])
    flat[torch.where(here, slots, choices).long()] = v.view(-1, n).to(flat.dtype)
    s["c"].copy_(flat[:choices].view_as(s["c"]))
    return s["c"]


def _plain_route(s):
    x = s["x"].double()
    if s["scoring"] == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
    else:
        p = 1 / (1 + torch.exp(-x))
    summed = s["groups"] > 1 and s["group_score"] == "top2"
    key = p + s["b"].double() if s["b"] is not None else p if summed else x
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    if s["groups"] > 1:
        g = key.view(s["m"], s["groups"], -1)
        g = torch.sort(g, dim=2, descending=True).values
        g = g[..., 0] + g[..., 1] if summed else g[..., 0]
        best = torch.sort(g, dim=1, descending=True, stable=True).indices[:, :s["topk_groups"]]
        allowed = torch.zeros_like(g).scatter_(1, best, 1.0).repeat_interleave(s["e"] // s["groups"], dim=1)
        # experts of the chosen groups first, in the order they have
        first = torch.sort(allowed.gather(1, order), dim=1, descending=True, stable=True).indices
        order = order.gather(1, first)
    ids = order[:, :s["top_k"]]
    w = p.gather(1, ids)
    total = w.sum(1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0) * s["scale"]
    return w.float(), ids.to(torch.int32)


def _plain_sort(topk_ids, e, bm, first):
    ids = topk_ids.reshape(-1).long() - first
    choices = ids.numel()
    blocks = _blocks(choices, e, bm)
    ids = torch.where((ids >= 0) & (ids < e), ids, e)
    order = torch.argsort(ids, stable=True)
    counts = torch.zeros(e + 1, dtype=torch.long, device=ids.device).scatter_add_(0, ids, torch.ones_like(ids))
    padded = (counts[:e] + bm - 1) // bm * bm
    ends = torch.cumsum(padded, 0)
    before = torch.cumsum(counts, 0) - counts
    begin = torch.cat([ends - padded, ends.new_full((1,), blocks * bm)])
    in_order = ids[order]
    to = begin[in_order] + torch.arange(choices, device=ids.device) - before[in_order]
    slots = ids.new_full((blocks * bm + 1,), choices)
    slots[torch.clamp_max(to, blocks * bm)] = torch.where(in_order < e, order, choices)
    block_begin = torch.arange(blocks, device=ids.device) * bm
    experts = torch.searchsorted(ends, block_begin, right=True)
    experts = torch.where(block_begin < ends[-1], experts, 0)
    return slots[:-1].to(torch.int32), experts.to(torch.int32), ends[-1:].to(torch.int32)


def _plain_combine(s):
    v = s["c"].float()
    if s["w"] is not None:
        v = v * s["w"][:, :, None]
    v = torch.where((s["ids"] >= 0)[:, :, None], v, 0.0).sum(1)
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(s["c"].dtype)


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _own(s):
    import flashnn_b200
    if s["op"] == "gemm":
        return s["f"](s["a"], s["b"], s["alpha_row"], s["alpha_col"], bias=s["b_bias"], residual=s["r"])
    if s["op"] == "experts":
        return flashnn_b200.fused_moe_a8w8_gated_forward(s["a"], s["b"], s["c"], s["alpha_row"], s["alpha_col"], s["ids"], *s["plan"],
                                                         s["top_k"], s["bm"], activation=s["act"], bias=s["b_bias"])
    if s["op"] == "route":
        return s["f"](s["x"], bias=s["b"])
    if s["op"] == "sort":
        return flashnn_b200.moe_sort_tokens(s["ids"], s["e"], s["bm"], first_expert=s["first"])
    return flashnn_b200.moe_combine(s["c"], topk_weights=s["w"], topk_ids=s["ids"], num_experts=64, residual=s["r"])


def run(s):
    if own:
        return _own(s)
    if s["op"] == "gemm":
        return _plain_gemm(s)
    if s["op"] == "experts":
        return _plain_experts(s)
    if s["op"] == "route":
        return _plain_route(s)
    if s["op"] == "sort":
        return _plain_sort(s["ids"], s["e"], s["bm"], s["first"])
    return _plain_combine(s)


# ---------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_act(v, name):
    sig = torch.special.expit
    return {"none": lambda: v, "relu": lambda: torch.relu(v), "sigmoid": lambda: sig(v), "silu": lambda: v * sig(v),
            "gelu": lambda: v * torch.special.ndtr(v),
            "gelu_tanh": lambda: v * sig(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))}[name]()


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if s["op"] == "gemm":
        parts = []
        for half in range(2 if s["gated"] else 1):
            rows = slice(half * s["n"], (half + 1) * s["n"])
            v = torch.matmul(s["a"].to(f64), s["b"][rows].to(f64).mT)
            v *= s["alpha_row"].to(f64).unsqueeze(1)
            v *= s["alpha_col"][rows].to(f64)
            parts.append(v if s["b_bias"] is None else v + s["b_bias"][rows].to(f64))
        v = _exact_act(parts[0], s["act"])
        if s["gated"]:
            v = v * parts[1]
        return v if s["r"] is None else v + s["r"].to(f64)
    if s["op"] == "experts":
        out = s["c"].to(f64).view(-1, s["n"])
        ids = s["ids"].flatten()
        for e in range(s["e"]):
            flat = (ids == e).nonzero().flatten()
            token = flat // s["top_k"]
            v = torch.matmul(s["a"][token].to(f64), s["b"][e].to(f64).mT)
            v *= s["alpha_row"][token].to(f64).unsqueeze(1) * s["alpha_col"][e].to(f64)
            if s["b_bias"] is not None:
                v += s["b_bias"][e].to(f64)
            out[flat] = _exact_act(v[:, :s["n"]], s["act"]) * v[:, s["n"]:]
        return out.view(s["m"], s["top_k"], s["n"])
    if s["op"] == "route":
        x = s["x"].to(f64)
        p = torch.softmax(x, 1).nan_to_num(0.0) if s["scoring"] == "softmax" else torch.special.expit(x)
        key = p if s["b"] is None else p + s["b"].to(f64)
        if s["b"] is None and not (s["groups"] > 1 and s["group_score"] == "top2"):
            key = x
        if s["groups"] > 1:
            g = key.unflatten(1, (s["groups"], -1))
            g = g.topk(2, dim=2).values.sum(2) if s["group_score"] == "top2" else g.max(2).values
            out = torch.ones_like(g, dtype=torch.bool).scatter_(1, g.topk(s["topk_groups"], dim=1).indices, False)
            key = key.masked_fill(out.repeat_interleave(s["e"] // s["groups"], 1), -math.inf)
        w = torch.take_along_dim(p, key.topk(s["top_k"], dim=1).indices, 1)
        return (w / w.sum(1, keepdim=True).clamp_min(1e-300) * s["scale"], None)
    if s["op"] == "combine":
        w = torch.ones(s["ids"].shape, dtype=f64, device=DEVICE) if s["w"] is None else s["w"].to(f64)
        w = w.masked_fill(s["ids"] < 0, 0.0)
        v = torch.einsum("mk,mkn->mn", w, s["c"].to(f64).nan_to_num(0.0))
        return v if s["r"] is None else v + s["r"].to(f64)
    return None  # a slot list has whole numbers only
