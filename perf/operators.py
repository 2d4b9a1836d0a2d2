"""The operators of 8-bit expert layers: what is timed, on which inputs, and what they have to give.

Four operators, each with its directions:

  route      router with sigmoid or softmax scores, a bias for balance that only the selection sees, expert groups,
             top-k, renormalised and scaled weights
  route_bwd  gradient of the routing weights with respect to the logits
  fp8        block quantisation to e4m3 with one power-of-two scale for 128 values: rows (1 x 128 blocks), rows copied
             to their expert-major places while they are quantised, weights (128 x 128 blocks), and reading rows back
  gemm       grouped matrix product of e4m3 operands with those scales: bf16 output ("none"), or SwiGLU whose result
             is quantised again ("swiglu_fp8", with the gate|up values too where a backward pass follows); the weight
             as [G,N,K] (NK, forward) or [G,K,N] (KN, gradient of the input)

8-bit tensors are returned in their own types (float8_e4m3fn values and float8_e8m0fnu scales), whose elements stand
for numbers. With `own` false run() is the plain form in elementary torch operations, with `own` true the framework's.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
BLK = 128
FMAX = 448.0  # largest e4m3 value


def _pkg():
    """This repository's package (its folder is not a Python identifier, so it is put on the path)."""
    root = str(Path(__file__).resolve().parent.parent / "1188b-reference-kernels_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import moe_b200
    return moe_b200


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small batch: launch latency
        dict(name="route decode", op="route", T=4, E=256, k=8, score="sigmoid", groups=8, keep=4, group_score="top2",
             bias=True, renorm=True, scale=2.5),
        # the layer's prompt batch, group-limited with a balance bias
        dict(name="route prompt", op="route", T=16384, E=256, k=8, score="sigmoid", groups=8, keep=4,
             group_score="top2", bias=True, renorm=True, scale=2.5),
        # softmax scores, no renormalisation, an odd batch and expert count
        dict(name="route_bwd odd", op="route_bwd", T=333, E=160, k=6, score="softmax", renorm=False, scale=16.0,
             grad="vals"),
        # backward of the prompt batch from the dense gate gradient that the layer's backward gives
        dict(name="route_bwd prompt", op="route_bwd", T=16384, E=256, k=8, score="sigmoid", renorm=True, scale=2.5,
             grad="probs"),
        # a few tokens on their way to their experts
        dict(name="permute_fp8 decode", op="fp8", dir="permuted", T=16, K=7168, E=256, k=8, dtype="bf16"),
        # the prompt batch on its way to its experts
        dict(name="permute_fp8 prompt", op="fp8", dir="permuted", T=8192, K=7168, E=256, k=8, dtype="bf16"),
        # a layer's weights after an optimiser step
        dict(name="weight to fp8", op="fp8", dir="weight", G=16, N=4096, K=7168, dtype="bf16"),
        # saved 8-bit activations read back for the weight gradient
        dict(name="rows from fp8", op="fp8", dir="read", T=16384, K=2048, dtype="bf16"),
        # a decode step of the first expert product: a few rows, every weight block read once
        dict(name="fc1 decode", op="gemm", R=32, G=32, N=4096, K=7168, layout="NK", epilogue="swiglu_fp8", pre=False,
             skew=0.0),
        # the first expert product of a prompt batch, skewed expert loads
        dict(name="fc1 prompt", op="gemm", R=32768, G=32, N=4096, K=7168, layout="NK", epilogue="swiglu_fp8",
             pre=False, skew=0.5),
        # the second one
        dict(name="fc2 prompt", op="gemm", R=32768, G=32, N=7168, K=2048, layout="NK", epilogue="none", pre=False,
             skew=0.5),
        # gradient of the first product's input, ragged groups, some of them empty
        dict(name="fc1 dgrad ragged", op="gemm", R=8191, G=40, N=5120, K=4096, layout="KN", epilogue="none",
             pre=False, skew=1.0),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route_bwd", "fp8", "gemm", "gemm"])
    if op in ("route", "route_bwd"):
        groups = rng.choice([1, 2, 4, 8])
        size = rng.choice([2, 4, 8, 16, 20, 24, 32, 40]) if groups > 1 else rng.choice([8, 40, 60, 64, 128, 160, 256, 320])
        e = groups * size
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, keep * size))
        t = _logu(rng, 1, 16384)
        score = rng.choice(["sigmoid", "softmax"])
        renorm = rng.random() < 0.7
        scale = rng.choice([1.0, 2.5, 16.0])
        if op == "route":
            return dict(op=op, T=t, E=e, k=k, score=score, groups=groups, keep=keep,
                        group_score=rng.choice(["top2", "max"]), bias=rng.random() < 0.7, renorm=renorm, scale=scale)
        return dict(op=op, T=t, E=e, k=k, score=score, renorm=renorm, scale=scale, grad=rng.choice(["vals", "probs"]))
    if op == "fp8":
        d = rng.choice(["rows", "permuted", "weight", "read"])
        k = 16 * _logu(rng, 4, 448)
        if d == "weight":
            return dict(op=op, dir=d, G=_logu(rng, 1, 16), N=_logu(rng, 8, 512) * 8, K=k, dtype=rng.choice(["bf16", "fp32"]))
        if d == "permuted":
            e = rng.choice([8, 64, 256, 320])
            return dict(op=op, dir=d, T=_logu(rng, 1, 8192), K=k, E=e, k=rng.randint(1, 8), dtype="bf16")
        return dict(op=op, dir=d, T=_logu(rng, 1, 16384), K=k, dtype=rng.choice(["bf16", "fp32"]) if d == "rows" else "bf16")
    layout = rng.choice(["NK", "NK", "KN"])
    epilogue = rng.choice(["none", "swiglu_fp8"]) if layout == "NK" else "none"
    n = 256 * _logu(rng, 1, 16) if epilogue == "swiglu_fp8" else (16 * _logu(rng, 8, 448) if layout == "KN" else 8 * _logu(rng, 16, 896))
    k = 16 * _logu(rng, 8, 448)
    most = max(1, 32 * 4096 * 7168 // (n * k))  # no more weights than the largest listed case has
    return dict(op=op, R=_logu(rng, 1, 16384), G=min(most, _logu(rng, 1, 40)), N=n, K=k, layout=layout, epilogue=epilogue,
                pre=epilogue == "swiglu_fp8" and rng.random() < 0.5, skew=rng.choice([0.0, 0.5, 1.5]))


# ------------------------------------------------------------------------------------------------- quantisation, plainly
def _exponent(amax):
    """e of the smallest power of two with amax <= 448 * 2^e, within the scale type's range; 0 for a block of zeros."""
    m, ex = torch.frexp(amax)  # amax = m * 2^ex with m in [0.5, 1); 448 = 0.875 * 2^9
    e = ex - 9 + (m > 0.875).to(torch.int32)
    return torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e))


def _pad(x, dim):
    n = -x.shape[dim] % BLK
    if not n:
        return x
    shape = list(x.shape)
    shape[dim] = n
    return torch.cat([x, x.new_zeros(shape)], dim)


def _to_rows(x):
    """x [M,K] -> (e4m3 [M,K], e8m0 [M,ceil(K/128)]): one scale for 128 values of a row."""
    m, k = x.shape
    b = _pad(x.float(), 1).view(m, -1, BLK)
    e = _exponent(b.abs().amax(2))
    q = torch.ldexp(b, -e[:, :, None]).view(m, -1)[:, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _to_blocks(w):
    """w [G,N,K] -> (e4m3 [G,N,K], e8m0 [G,ceil(N/128),ceil(K/128)]): one scale for a block of 128 x 128 values."""
    g, n, k = w.shape
    p = _pad(_pad(w.float(), 1), 2)
    b = p.view(g, p.shape[1] // BLK, BLK, p.shape[2] // BLK, BLK)
    e = _exponent(b.abs().amax(4).amax(2))
    q = torch.ldexp(b, -e[:, :, None, :, None]).view(p.shape)[:, :n, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_rows(q, s):
    f = s.float().repeat_interleave(BLK, 1)[:, : q.shape[1]]
    return q.float() * f


def _from_blocks(q, s):
    p = _pad(_pad(q.float(), 1), 2)
    b = p.view(p.shape[0], p.shape[1] // BLK, BLK, p.shape[2] // BLK, BLK) * s.float()[:, :, None, :, None]
    return b.view(p.shape)[:, : q.shape[1], : q.shape[2]]


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _counts(rows, groups, skew, seed):
    """Rows of each group: a Zipf law of exponent `skew` in a drawn order, every row somewhere."""
    g = torch.Generator().manual_seed(seed)
    p = torch.arange(1, groups + 1, dtype=torch.float64) ** -skew
    p = p[torch.randperm(groups, generator=g)]
    return torch.bincount(torch.multinomial(p, rows, replacement=True, generator=g), minlength=groups)


def _activations(shape, g, dtype=torch.bfloat16):
    """Activations of a transformer: rows of different size, a few columns much larger than the rest."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    x *= torch.exp2(torch.randint(-3, 3, (shape[0], 1), generator=g, device=DEV).to(torch.bfloat16))
    hot = torch.randint(0, shape[1], (max(1, shape[1] // 512),), generator=g, device=DEV)
    x[:, hot] *= 16
    return x.to(dtype)


def _logits(t, e, g):
    """Router logits: N(0,1) and a per-expert offset 1.5 * log of a Zipf law, so that loads are skewed."""
    zipf = -1.5 * torch.log(torch.arange(1, e + 1, device=DEV, dtype=torch.float32)) * 0.2
    return torch.randn((t, e), generator=g, device=DEV) + zipf[torch.randperm(e, generator=g, device=DEV)]


def _row_map(idx, t, e):
    """Destinations [T,E] int64 (-1: not routed) of tokens in expert-major order, as the framework's row-id map."""
    on = torch.zeros((t, e), dtype=torch.int64, device=DEV).scatter_(1, idx, 1)
    place = torch.cumsum(on.t().reshape(-1), 0).view(e, t).t() - 1
    return torch.where(on > 0, place, -1).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    op = case["op"]
    if op in ("route", "route_bwd"):
        t, e, k = case["T"], case["E"], case["k"]
        st["logits"] = _logits(t, e, g)
        if op == "route":
            st["bias"] = torch.randn(e, generator=g, device=DEV) * 0.1 if case["bias"] else None
            return st
        st["idx"] = torch.sort(st["logits"], dim=1, descending=True, stable=True).indices[:, :k].contiguous()
        st["grad"] = torch.randn((t, k), generator=g, device=DEV)
        if case["grad"] == "probs":
            st["grad"] = torch.zeros((t, e), device=DEV).scatter_(1, st["idx"], st["grad"])
        return st
    if op == "fp8":
        dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        if case["dir"] == "weight":
            st["w"] = (torch.randn((case["G"], case["N"], case["K"]), generator=g, device=DEV, dtype=torch.bfloat16) * 0.02).to(dt)
            return st
        st["x"] = _activations((case["T"], case["K"]), g, dt)
        if case["dir"] == "permuted":
            st["idx"] = torch.topk(_logits(case["T"], case["E"], g), case["k"], dim=1).indices
            st["map"] = _row_map(st["idx"], case["T"], case["E"])
        if case["dir"] == "read":
            st["q"], st["s"] = _to_rows(st.pop("x"))
        return st
    r, n, k = case["R"], case["N"], case["K"]
    counts = _counts(r, case["G"], case["skew"], seed)
    st["counts"] = counts.to(device=DEV, dtype=torch.int32)
    st["host_counts"] = counts.tolist()
    st["x"] = _to_rows(_activations((r, k), g))
    shape = (case["G"], n, k) if case["layout"] == "NK" else (case["G"], k, n)
    st["w"] = _to_blocks(torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16) * 0.02)
    # where the rows of each group lie when every group is laid out with as many rows as the largest
    most = max(1, int(counts.max()))
    start = torch.cumsum(counts, 0) - counts
    group = torch.repeat_interleave(torch.arange(case["G"]), counts)
    st["slot"] = (group * most + torch.arange(r) - start[group]).to(DEV)
    st["most"] = most
    st["plan"] = {}  # the group table that a program keeps between steps
    return st


# --------------------------------------------------------------------------------------------------------- plain forms
def _scores(logits, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    return p / p.sum(1, keepdim=True)


def _weights(s, renorm, scale):
    if renorm:
        total = s.sum(1, keepdim=True)
        s = torch.where(total > 0, s / total, torch.zeros_like(s))
    return s * scale


def _route_plain(st):
    """In 64 bits: which expert is selected hangs on the last bits of its score."""
    c = st["case"]
    s = _scores(st["logits"].double(), c["score"])
    sel = s if st["bias"] is None else s + st["bias"].double()
    t, e = s.shape
    by_group = sel.view(t, c["groups"], -1)
    top = torch.sort(by_group, dim=2, descending=True).values
    rank = top[:, :, :2].sum(2) if c["group_score"] == "top2" else top[:, :, 0]
    kept = torch.zeros((t, c["groups"]), dtype=torch.bool, device=s.device)
    kept.scatter_(1, torch.sort(rank, dim=1, descending=True, stable=True).indices[:, : c["keep"]], True)
    kept = kept.repeat_interleave(e // c["groups"], 1)
    order = torch.sort(sel, dim=1, descending=True, stable=True).indices
    inside = torch.sort(kept.gather(1, order).to(torch.int32), dim=1, descending=True, stable=True).indices
    idx = order.gather(1, inside)[:, : c["k"]]
    w = _weights(s.gather(1, idx), c["renorm"], c["scale"]).float()
    on = torch.zeros((t, e), dtype=torch.bool, device=s.device).scatter_(1, idx, True)
    return {"vals": w, "idx": idx, "map": on, "probs": torch.zeros((t, e), device=s.device).scatter_(1, idx, w)}


def _route_bwd_plain(st):
    c = st["case"]
    s = _scores(st["logits"], c["score"])
    idx = st["idx"]
    g = (st["grad"] if c["grad"] == "vals" else st["grad"].gather(1, idx)) * c["scale"]
    sk = s.gather(1, idx)
    if c["renorm"]:
        total = sk.sum(1, keepdim=True)
        g = g / total - (g * sk).sum(1, keepdim=True) / (total * total)
    ds = torch.zeros_like(s).scatter_(1, idx, g)
    if c["score"] == "sigmoid":
        return ds * s * (1 - s)
    return s * (ds - (ds * s).sum(1, keepdim=True))


def _fp8_plain(st):
    c = st["case"]
    if c["dir"] == "weight":
        return _to_blocks(st["w"])
    if c["dir"] == "read":
        return _from_rows(st["q"], st["s"]).to(torch.bfloat16)
    q, s = _to_rows(st["x"])
    if c["dir"] == "permuted":
        rows = st["map"].gather(1, st["idx"]).view(-1)
        token = torch.empty_like(rows)
        token[rows] = torch.arange(rows.numel(), device=rows.device) // c["k"]
        return q[token], s.view(torch.uint8)[token].view(torch.float8_e8m0fnu)
    return q, s


def _gemm_plain(st):
    c = st["case"]
    x, w = _from_rows(*st["x"]), _from_blocks(*st["w"])
    laid = x.new_zeros((c["G"] * st["most"], c["K"]))
    laid[st["slot"]] = x
    laid = laid.view(c["G"], st["most"], c["K"])
    y = torch.bmm(laid, w.transpose(1, 2) if c["layout"] == "NK" else w).view(c["G"] * st["most"], c["N"])[st["slot"]]
    if c["epilogue"] == "none":
        return y.to(torch.bfloat16)
    gate, up = y[:, : c["N"] // 2], y[:, c["N"] // 2:]
    q, s = _to_rows(gate / (1 + torch.exp(-gate)) * up)
    return (q, s, y.to(torch.bfloat16)) if c["pre"] else (q, s)


# ------------------------------------------------------------------------------------------------- the framework's calls
def _route_own(st):
    c = st["case"]
    r = _pkg().router_group_topk(st["logits"], c["k"], score=c["score"], num_groups=c["groups"], topk_groups=c["keep"],
                                 group_score=c["group_score"], bias=st["bias"], renorm=c["renorm"], scale=c["scale"])
    return {"vals": r.topk_vals, "idx": r.topk_idx, "map": r.routing_map, "probs": r.probs}


def _route_bwd_own(st):
    c = st["case"]
    grad = {"grad_vals": st["grad"]} if c["grad"] == "vals" else {"grad_probs": st["grad"]}
    return _pkg().router_topk_backward(st["logits"], st["idx"], score=c["score"], renorm=c["renorm"], scale=c["scale"],
                                       **grad)


def _fp8_own(st):
    m, c = _pkg(), st["case"]
    if c["dir"] == "weight":
        return tuple(m.quantize_fp8_weight(st["w"]))
    if c["dir"] == "read":
        return m.dequantize_fp8(m.Fp8Tensor(st["q"], st["s"]))
    if c["dir"] == "permuted":
        return tuple(m.permute_fp8(st["x"], st["map"], st["idx"], c["T"] * c["k"]))
    return tuple(m.quantize_fp8(st["x"]))


def _gemm_own(st):
    m, c = _pkg(), st["case"]
    if "plan" not in st["plan"]:
        st["plan"]["plan"] = m.GroupedGemmPlan(c["G"], st["counts"].device)
    plan = st["plan"]["plan"].from_splits(st["counts"])
    out = m.grouped_gemm_fp8(m.Fp8Tensor(*st["x"]), m.Fp8Tensor(*st["w"]), epilogue=c["epilogue"], plan=plan,
                             w_layout=c["layout"], return_pre=c["pre"])
    if c["epilogue"] == "none":
        return out
    return (*out[0], out[1]) if c["pre"] else tuple(out)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"route": _route_own, "route_bwd": _route_bwd_own, "fp8": _fp8_own, "gemm": _gemm_own}[op](state)
    return {"route": _route_plain, "route_bwd": _route_bwd_plain, "fp8": _fp8_plain, "gemm": _gemm_plain}[op](state)


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["T"], case["E"], case["k"]
        return {"bytes": t * e * (4 + 1 + 4) + t * k * 12 + (4 * e if case["bias"] else 0), "flops": 8 * t * e}
    if op == "route_bwd":
        t, e, k = case["T"], case["E"], case["k"]
        read = t * e * 4 if case["score"] == "softmax" else t * k * 4  # a sigmoid needs the selected logits alone
        return {"bytes": read + t * k * (8 + 4) + t * e * 4, "flops": 8 * t * (e if case["score"] == "softmax" else k)}
    size = 4 if case.get("dtype") == "fp32" else 2
    kb = -(-case["K"] // BLK)
    if op == "fp8":
        k = case["K"]
        if case["dir"] == "weight":
            m = case["G"] * case["N"]
            return {"bytes": m * k * (size + 1) + case["G"] * -(-case["N"] // BLK) * kb, "flops": 2 * m * k}
        m = case["T"]
        if case["dir"] == "permuted":
            return {"bytes": m * k * 2 + m * case["k"] * (k + kb + 16), "flops": 2 * m * k}
        return {"bytes": m * k * (size + 1) + m * kb, "flops": 2 * m * k}
    r, g, n, k = case["R"], case["G"], case["N"], case["K"]
    p = [i ** -case["skew"] for i in range(1, g + 1)]
    used = sum(1 - (1 - v / sum(p)) ** r for v in p)  # groups with rows, on average: the others' weights are not read
    nb = -(-n // BLK)
    out = r * n * 2 if case["epilogue"] == "none" else r * (n // 2 + n // 2 // BLK) + (r * n * 2 if case["pre"] else 0)
    return {"bytes": r * (k + kb) + used * (n * k + nb * kb) + out, "flops": 2 * r * n * k}


# --------------------------------------------------------------------------------------------- the definition in 64 bits
def _grid(v):
    """v rounded to the nearest e4m3 value, ties to even: steps of 2^-3 of the leading power of two, 2^-9 below 2^-6."""
    lead = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -40))).clamp_min(-6)
    step = torch.exp2(lead - 3)
    return torch.round(v / step) * step


def _blocks64(a, rows, rounded=True):
    """(values, scales) in 64 bits of a [G,N,K] quantised with 128 x 128 blocks, or of [1,M,K] with 1 x 128 (rows);
    not `rounded`: the scaled values before they are rounded to 8 bits."""
    hi = 1 if rows else BLK
    g, n, k = a.shape
    nb, kb = -(-n // hi), -(-k // BLK)
    p = torch.zeros((g, nb * hi, kb * BLK), dtype=torch.float64, device=a.device)
    p[:, :n, :k] = a
    amax = p.abs().view(g, nb, hi, kb * BLK).amax(2).view(g, nb, kb, BLK).amax(3)
    e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / FMAX))
    e = torch.where(amax > FMAX * torch.exp2(e), e + 1, e)  # the logarithm's own rounding, next to a power of two
    e = torch.where(amax <= FMAX * torch.exp2(e - 1), e - 1, e)
    s = torch.exp2(torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e)))
    full = s.repeat_interleave(hi, 1).repeat_interleave(BLK, 2)
    q = p / full
    return (_grid(q) if rounded else q)[:, :n, :k], s


def _exact_route(st):
    c = st["case"]
    x = st["logits"].double()
    s = 0.5 + 0.5 * torch.tanh(x / 2) if c["score"] == "sigmoid" else torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
    left = s + (0 if st["bias"] is None else st["bias"].double())
    t, e = x.shape
    size = e // c["groups"]
    best = left.view(t, c["groups"], size).topk(min(size, 2 if c["group_score"] == "top2" else 1), dim=2).values.sum(2)
    out = torch.ones((t, c["groups"]), dtype=torch.bool, device=x.device)
    for _ in range(c["keep"]):
        j = best.argmax(1, keepdim=True)
        out.scatter_(1, j, False)
        best.scatter_(1, j, -math.inf)
    left = left.masked_fill(out.repeat_interleave(size, 1), -math.inf)
    got = []
    for _ in range(c["k"]):
        got.append(left.argmax(1, keepdim=True))
        left.scatter_(1, got[-1], -math.inf)
    idx = torch.cat(got, 1)
    w = s.gather(1, idx)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["scale"]
    return {"vals": w, "idx": None, "map": None, "probs": torch.zeros_like(s).scatter_(1, idx, w)}


def _exact_route_bwd(st):
    """By automatic differentiation of the weights in 64 bits."""
    c = st["case"]
    x = st["logits"].double().requires_grad_(True)
    s = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, 1)
    w = s.gather(1, st["idx"])
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    g = st["grad"].double() if c["grad"] == "vals" else st["grad"].double().gather(1, st["idx"])
    (w * c["scale"] * g).sum().backward()
    return x.grad


def _exact_fp8(st):
    c = st["case"]
    if c["dir"] == "weight":
        return _blocks64(st["w"].double(), False)
    if c["dir"] == "read":
        col = torch.arange(c["K"], device=DEV) // BLK
        return st["q"].double() * st["s"].double()[:, col]
    q, s = (a[0] for a in _blocks64(st["x"].double()[None], True))
    if c["dir"] == "permuted":
        at = torch.argsort(torch.where(st["map"].t() >= 0, st["map"].t(), 1 << 40).reshape(-1))[: c["T"] * c["k"]]
        q, s = q[at % c["T"]], s[at % c["T"]]
    return q, s


def _exact_gemm(st):
    c = st["case"]
    (xq, xs), (wq, ws) = st["x"], st["w"]
    col = torch.arange(c["K"], device=DEV) // BLK
    y = torch.zeros((c["R"], c["N"]), dtype=torch.float64, device=DEV)
    at = 0
    for g, m in enumerate(st["host_counts"]):
        if m:
            x = xq[at: at + m].double() * xs[at: at + m].double()[:, col]
            w, s = wq[g].double(), ws[g].double()
            w = w * s[torch.arange(w.shape[0], device=DEV) // BLK][:, torch.arange(w.shape[1], device=DEV) // BLK]
            y[at: at + m] = x @ (w.t() if c["layout"] == "NK" else w)
        at += m
    if c["epilogue"] == "none":
        return y
    f = c["N"] // 2
    h = y[:, :f] * torch.sigmoid(y[:, :f]) * y[:, f:]
    # as for an output in 16 bits, the value before its last rounding: a computed number next to a border of two 8-bit
    # values has no one right rounding
    q, s = (a[0] for a in _blocks64(h[None], True, rounded=False))
    return (q, s, y) if c["pre"] else (q, s)


def exact(case, seed):
    st = prepare(case, seed)
    return {"route": _exact_route, "route_bwd": _exact_route_bwd, "fp8": _exact_fp8, "gemm": _exact_gemm}[case["op"]](st)
