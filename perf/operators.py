"""8-bit block-scaled projections, the routing of frames to experts, and the experts' FeedForward, as cases that can be
timed and checked.

  linear   y = W q(x) + b. W [out, in] is held as e4m3 codes with one power of two for each 128 x 128 block, and q(x)
           rounds the activations to e4m3 with one power of two for each row's 128 inputs.
  route    per frame: scores of the experts (softmax or sigmoid of the gate's logits), the choice of top_k by score plus
           balance bias, within the best groups of experts, and the chosen scores as weights.
  experts  y = residual + s * sum_j w_j FF_{e_j}(x), FF_e(x) = W2_e q(silu(W1_e q(x) + b1_e)) + b2_e, for the experts e_j
           that routing chose for the frame (-1: none).

The power of two of a block is the smallest 2^e with max |v| <= 448 * 2^e over its values (448: the largest e4m3 value),
e >= -127. Sizes are those of the 0.6B model (d_model 1024, FeedForward 4096) and the large one (512, 2048) at 12.5
frames a second, with 8 to 256 experts.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
SCORES = ("softmax", "sigmoid")
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _linear(name, rows, d_in, d_out, x, out, bias=True):
    return {"name": name, "op": "linear", "rows": rows, "in": d_in, "out": d_out, "x": x, "y": out, "bias": bias}


def _route(name, rows, experts, top_k, score, dtype, bias=False, groups=1, kept=1, renorm=True, padded=0.0):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "top_k": top_k, "score": score, "x": dtype,
            "bias": bias, "groups": groups, "kept": kept, "renorm": renorm, "padded": padded}


def _experts(name, rows, experts, top_k, d, ff, bias=False, residual=False, skew=0.0, padded=0.0):
    return {"name": name, "op": "experts", "rows": rows, "experts": experts, "top_k": top_k, "d": d, "ff": ff,
            "bias": bias, "residual": residual, "skew": skew, "padded": padded}


def listed():
    return [
        # one frame of one stream through a FeedForward's first projection: latency
        _linear("linear_token", 1, 1024, 4096, "bfloat16", "bfloat16"),
        # a 14-frame chunk of 8 streams, whose activations are f32
        _linear("linear_stream_f32", 112, 512, 2048, "float32", "float32"),
        # the token head over one utterance of an odd length: 1024 tokens and a blank, f32 logits
        _linear("linear_head", 203, 640, 1025, "bfloat16", "float32"),
        # a server's batch of 30 s utterances through a FeedForward's first projection
        _linear("linear_batch", 3000, 1024, 4096, "bfloat16", "bfloat16"),
        # recordings of 10 minutes through its second
        _linear("linear_long", 15000, 4096, 1024, "bfloat16", "bfloat16"),
        # one frame to 2 of 8 experts
        _route("route_token", 1, 8, 2, "softmax", "float32"),
        # the batch of 30 s to 4 of 64 experts by sigmoid scores with a balance bias; padding frames choose none
        _route("route_batch", 3000, 64, 4, "sigmoid", "bfloat16", bias=True, padded=0.1),
        # a large batch to 8 of 256 experts in the 4 best of 8 groups
        _route("route_long", 30001, 256, 8, "sigmoid", "float32", bias=True, groups=8, kept=4, padded=0.05),
        # one frame through 2 of 8 experts: two experts' weights are read once
        _experts("experts_token", 1, 8, 2, 1024, 4096),
        # a chunk of 8 streams through the large model's experts as the block's half step
        _experts("experts_stream", 112, 32, 2, 512, 2048, bias=True, residual=True),
        # the batch of 30 s through 2 of 16 experts as the block's half step
        _experts("experts_batch", 3000, 16, 2, 1024, 4096, bias=True, residual=True, skew=0.3, padded=0.1),
        # recordings of 10 minutes, an odd number of frames, 4 of 64 experts, some of them far more often than others
        _experts("experts_long", 15001, 64, 4, 1024, 4096, residual=True, skew=0.7, padded=0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "route", "experts"))
    if op == "linear":
        while True:
            rows, d_in, d_out = _log(rng, 1, 16000), _log(rng, 100, 4096), _log(rng, 100, 4096)
            if rng.random() < 0.5:  # half of the projections have whole blocks, as the models have
                d_in, d_out = -(-d_in // BLOCK) * BLOCK, -(-d_out // BLOCK) * BLOCK
            if rows * d_in * d_out <= 15000 * 4096 * 1024:
                x, y = rng.choice((("bfloat16", "bfloat16"), ("float32", "float32"), ("bfloat16", "float32")))
                c = _linear("", rows, d_in, d_out, x, y, rng.random() < 0.5)
                break
    elif op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * rng.choice((2, 4, 5, 8, 16, 32)) if groups > 1 else rng.choice((4, 8, 12, 16, 32, 60, 64, 128, 160, 256))
        kept = rng.randint(1, groups)
        top_k = rng.randint(1, min(8, kept * (experts // groups)))
        c = _route("", _log(rng, 1, 30000), experts, top_k, rng.choice(SCORES), rng.choice(("float32", "bfloat16")),
                   rng.random() < 0.5, groups, kept, rng.random() < 0.7, rng.choice((0.0, 0.05, 0.3)))
    else:
        while True:
            experts, top_k = rng.choice((4, 8, 12, 16, 32, 48, 64)), rng.randint(1, 4)
            d = rng.choice((256, 512, 640, 1024))
            c = _experts("", _log(rng, 1, 15000), experts, top_k, d, rng.choice((2, 4)) * d, rng.random() < 0.5,
                         rng.random() < 0.5, rng.choice((0.0, 0.3, 0.7)), rng.choice((0.0, 0.05, 0.3)))
            if c["rows"] * top_k * d * c["ff"] <= 15001 * 4 * 1024 * 4096:
                break
    del c["name"]
    return c


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _exponent(amax):
    """The smallest e >= -127 with amax <= 448 * 2^e (0 for a block of zeros)."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp_min(-127)


def _weights(g, lead, n, k):
    """Codes [*lead, n, k] (float8_e4m3fn) and biased exponents [*lead, ceil(n/128), ceil(k/128)] (uint8) of weights of
    the usual size."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(*lead, nb * BLOCK, kb * BLOCK, device="cuda")
    w[..., :n, :k] = torch.randn(*lead, n, k, device="cuda", generator=g) / math.sqrt(k)
    w = w.view(*lead, nb, BLOCK, kb, BLOCK)
    e = _exponent(w.abs().amax((-3, -1)))
    codes = torch.ldexp(w, -e[..., :, None, :, None]).reshape(*lead, nb * BLOCK, kb * BLOCK)[..., :n, :k]
    return codes.to(torch.float8_e4m3fn).contiguous(), (e + 127).to(torch.uint8)


def _frames(g, rows, d):
    """Normalised activations: a few channels are larger than the others, as after a LayerNorm with its weight."""
    gain = torch.exp(0.5 * torch.randn(d, device="cuda", generator=g))
    return torch.randn(rows, d, device="cuda", generator=g) * gain


def _library():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-nemo-rs_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import relpos_mhsa
    return relpos_mhsa


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    rows = case["rows"]
    if case["op"] == "linear":
        s["x"] = _frames(g, rows, case["in"]).to(DTYPES[case["x"]])
        s["codes"], s["scales"] = _weights(g, (), case["out"], case["in"])
        s["b"] = 0.1 * torch.randn(case["out"], device="cuda", generator=g) if case["bias"] else None
        if own:
            s["layer"] = _library().Fp8Linear(case["in"], case["out"], case["bias"])
            s["layer"].load_codes(s["codes"], s["scales"], s["b"])
    elif case["op"] == "route":
        logits = 1.5 * torch.randn(rows, case["experts"], device="cuda", generator=g)
        logits[rows - int(case["padded"] * rows):] = -math.inf  # the frames behind the utterances' ends
        s["logits"] = logits.to(DTYPES[case["x"]])
        s["bias"] = 0.05 * torch.randn(case["experts"], device="cuda", generator=g) if case["bias"] else None
    else:
        e, k, d, ff = case["experts"], case["top_k"], case["d"], case["ff"]
        s["x"] = _frames(g, rows, d).to(torch.bfloat16)
        s["codes1"], s["scales1"] = _weights(g, (e,), ff, d)
        s["codes2"], s["scales2"] = _weights(g, (e,), d, ff)
        s["b1"] = 0.1 * torch.randn(e, ff, device="cuda", generator=g) if case["bias"] else None
        s["b2"] = 0.1 * torch.randn(e, d, device="cuda", generator=g) if case["bias"] else None
        often = -case["skew"] * torch.log(torch.arange(1, e + 1, device="cuda").float())
        often = often[torch.randperm(e, device="cuda", generator=g)]
        gate = torch.randn(rows, e, device="cuda", generator=g) + often
        top, idx = gate.topk(k, dim=-1)
        idx[rows - int(case["padded"] * rows):] = -1  # padding frames
        s["idx"], s["w"] = idx.to(torch.int32), torch.softmax(top, -1)
        s["r"] = torch.randn(rows, d, device="cuda", generator=g).to(torch.bfloat16) if case["residual"] else None
        if own:
            s["layer"] = _library().ExpertFeedForward(e, d, ff, case["bias"])
            s["layer"].load_codes(s["codes1"], s["scales1"], s["codes2"], s["scales2"], s["b1"], s["b2"])
    return s


def _rounded(x):
    """x [..., k] in f32 as its e4m3 codes and block scales stand for it."""
    k = x.shape[-1]
    kb = -(-k // BLOCK)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).unflatten(-1, (kb, BLOCK))
    e = _exponent(p.abs().amax(-1, keepdim=True))
    return torch.ldexp(torch.ldexp(p, -e).to(torch.float8_e4m3fn).float(), e).flatten(-2)[..., :k]


def _values(codes, scales):
    """Weights in f32 as their codes and scales stand for them."""
    n, k = codes.shape[-2:]
    s = torch.ldexp(torch.ones((), device=codes.device), scales.to(torch.int32) - 127)
    s = s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return codes.float() * s


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_linear(s):
    y = _rounded(s["x"].float()) @ _values(s["codes"], s["scales"]).T
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["case"]["y"]])


def _plain_route(s):
    c, x = s["case"], s["logits"].double()  # in 64 bits: a choice between near scores is a rounding away from the other
    there = x > -math.inf
    if c["score"] == "softmax":
        score = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min))
        total = score.sum(-1, keepdim=True)
        score = score / torch.where(total > 0, total, 1)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = torch.where(there, choice, -math.inf)
    if c["groups"] > 1:
        by_group = choice.unflatten(-1, (c["groups"], -1))
        best = by_group.sort(dim=-1, descending=True).values[..., :2]
        best = torch.where(best[..., 1] > -math.inf, best.sum(-1), best[..., 0])
        kept = torch.zeros_like(best, dtype=torch.bool)
        kept.scatter_(-1, best.sort(dim=-1, descending=True, stable=True).indices[..., :c["kept"]], True)
        choice = torch.where(kept[..., None], by_group, -math.inf).flatten(-2)
    top, idx = choice.sort(dim=-1, descending=True, stable=True)
    top, idx = top[..., :c["top_k"]], idx[..., :c["top_k"]]
    w = torch.where(top > -math.inf, score.gather(-1, idx), 0)
    idx = torch.where(top > -math.inf, idx, -1)
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0)
    return {"idx": idx.to(torch.int32), "w": w.float()}


def _plain_experts(s):
    c, k = s["case"], s["case"]["top_k"]
    x = _rounded(s["x"].float())
    pair = s["idx"].flatten().long()
    at = torch.nonzero(pair >= 0).flatten()
    y = torch.zeros(pair.numel(), c["d"], device=x.device)
    if at.numel():
        used, e, count = torch.unique(pair[at], return_inverse=True, return_counts=True)
        at = at[torch.argsort(e, stable=True)]  # the pairs, those of an expert side by side
        e = e.sort().values
        place = torch.arange(e.numel(), device=x.device) - (count.cumsum(0) - count)[e]
        size = min(int(count.max()), 512)  # batches of up to 512 pairs of one expert, so that rare experts pad little
        batches = (count + size - 1) // size
        batch, place = (batches.cumsum(0) - batches)[e] + place // size, place % size
        used = used.repeat_interleave(batches)
        a = torch.zeros(used.numel(), size, c["d"], device=x.device)
        a[batch, place] = x[at // k]
        h = torch.bmm(a, _values(s["codes1"][used], s["scales1"][used]).transpose(1, 2).contiguous())
        if s["b1"] is not None:
            h = h + s["b1"][used][:, None]
        h = _rounded(_silu(h))
        o = torch.bmm(h, _values(s["codes2"][used], s["scales2"][used]).transpose(1, 2).contiguous())
        if s["b2"] is not None:
            o = o + s["b2"][used][:, None]
        y[at] = o[batch, place]
    y = (y.view(c["rows"], k, c["d"]) * s["w"][..., None]).sum(1)
    if s["r"] is not None:
        y = s["r"].float() + 0.5 * y
    return y.to(torch.bfloat16)


def run(state):
    c = state["case"]
    if not own:
        return {"linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}[c["op"]](state)
    if c["op"] == "linear":
        return state["layer"].forward(state["x"], out_dtype=DTYPES[c["y"]])
    if c["op"] == "route":
        idx, w = _library().route(state["logits"], c["top_k"], score=c["score"], bias=state["bias"],
                                  n_groups=c["groups"], topk_groups=c["kept"], renormalize=c["renorm"])
        return {"idx": idx, "w": w}
    return state["layer"].forward(state["x"], state["idx"], state["w"], residual=state["r"],
                                  res_scale=0.5 if c["residual"] else 1.0)


def work(case):
    size = {"float32": 4, "bfloat16": 2}
    rows = case["rows"]
    if case["op"] == "linear":
        k, n = case["in"], case["out"]
        return {"bytes": rows * k * size[case["x"]] + n * k + rows * n * size[case["y"]], "flops": 2.0 * rows * n * k}
    if case["op"] == "route":
        return {"bytes": rows * (case["experts"] * size[case["x"]] + 8 * case["top_k"]), "flops": 0}
    e, k, d, ff = case["experts"], case["top_k"], case["d"], case["ff"]
    live = rows - int(case["padded"] * rows)
    used = e * (1 - (1 - min(1.0, k / e)) ** live)  # experts that some frame chooses
    return {"bytes": rows * d * (6 if case["residual"] else 4) + rows * k * 8 + used * 2 * d * ff,
            "flops": 4.0 * live * k * d * ff}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_round(v):
    """Blocks of the last axis rounded to e4m3 steps of their power of two: to nearest, ties to the even step."""
    out = torch.zeros_like(v)
    for lo in range(0, v.shape[-1], BLOCK):
        b = v[..., lo:lo + BLOCK]
        top = b.abs().max(-1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0))
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)  # log2 rounds
        e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp_min(-127)
        t = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)  # 2^-9 below the smallest normal
        out[..., lo:lo + BLOCK] = torch.round(t / step) * step * torch.exp2(e)
    return out


def _exact_weight(codes, scales):
    w = codes.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= 2.0 ** (int(scales[i, j]) - 127)
    return w


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = _exact_round(s["x"].double()) @ _exact_weight(s["codes"], s["scales"].cpu()).T
        return y if s["b"] is None else y + s["b"].double()
    if case["op"] == "route":
        if case["rows"] > 4000:
            return None
        x = s["logits"].double().cpu().tolist()
        bias = [0.0] * case["experts"] if s["bias"] is None else s["bias"].double().cpu().tolist()
        size, weights = case["experts"] // case["groups"], []
        for row in x:
            if case["score"] == "softmax":
                top = max(row)
                p = [math.exp(v - top) if v > -math.inf else 0.0 for v in row]
                total = math.fsum(p) or 1.0
                p = [v / total for v in p]
            else:
                p = [1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in row]
            choice = [p[i] + bias[i] if row[i] > -math.inf else -math.inf for i in range(len(row))]
            if case["groups"] > 1:
                best = []
                for j in range(case["groups"]):
                    two = sorted(choice[j * size:(j + 1) * size], reverse=True)[:2]
                    best.append(two[0] if len(two) < 2 or two[1] == -math.inf else two[0] + two[1])
                kept = sorted(range(case["groups"]), key=lambda j: (-best[j], j))[:case["kept"]]
                choice = [v if i // size in kept else -math.inf for i, v in enumerate(choice)]
            order = sorted(range(len(row)), key=lambda i: (-choice[i], i))[:case["top_k"]]
            w = [p[i] if choice[i] > -math.inf else 0.0 for i in order]
            total = math.fsum(w)
            weights.append([v / total if total > 0 else 0.0 for v in w] if case["renorm"] else w)
        return {"idx": None, "w": torch.tensor(weights, dtype=torch.float64)}
    x, idx, w = _exact_round(s["x"].double()), s["idx"].long(), s["w"].double()
    y = torch.zeros(case["rows"], case["d"], dtype=torch.float64, device=x.device)
    scales1, scales2 = s["scales1"].cpu(), s["scales2"].cpu()
    for e in sorted(set(idx.flatten().tolist()) - {-1}):
        row, slot = torch.nonzero(idx == e, as_tuple=True)
        h = x[row] @ _exact_weight(s["codes1"][e], scales1[e]).T
        if s["b1"] is not None:
            h = h + s["b1"][e].double()
        o = _exact_round(h * torch.sigmoid(h)) @ _exact_weight(s["codes2"][e], scales2[e]).T
        if s["b2"] is not None:
            o = o + s["b2"][e].double()
        y[row] += w[row, slot][:, None] * o  # a frame chooses an expert once
    return y if s["r"] is None else s["r"].double() + 0.5 * y
