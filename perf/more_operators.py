"""A residual's addition with its norm, low-rank adapters beside a shared 8-bit projection, and the log probabilities of
tokens, as cases that can be timed and checked.

  norm      v = x + a d, sum = v; y = v / sqrt(mean v^2 + eps) * w ("rms") or (v - mean) / sqrt(var + eps) * w + b
            ("layer"); y as floats or as e4m3 codes with one power of two for each row's 128 values.
  adapters  y = W q(x) + b + s_a B_a (A_a x), a = which[row] (-1: none); W as e4m3 codes with a power of two for each
            128 x 128 block, q(x) the activations rounded to e4m3 in the same way, A_a [rank, in] and B_a [out, rank] bf16.
  scores    of logits z / T: log p of a given token, the entropy, and the top_k tokens with their log p, ties to the lower
            index (-1: no token there; a given token of -1 has 0).

The power of two of a block is the smallest 2^e with max |v| <= 448 * 2^e over its values (448: the largest e4m3 value),
e >= -127. Sizes are those of the 0.6B model (d_model 1024, FeedForward 4096) and the large one (512, 2048) at 12.5
frames a second, the transducer's 1024 tokens and a blank, and vocabularies of text models.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "bfloat16": 2}
EPS = 1e-5


def _norm(name, rows, d, x, kind="rms", delta=True, out="codes"):
    return {"name": name, "op": "norm", "rows": rows, "d": d, "x": x, "kind": kind, "delta": delta, "out": out}


def _adapters(name, rows, d_in, d_out, adapters, rank, requests, x, out, bias=False):
    return {"name": name, "op": "adapters", "rows": rows, "in": d_in, "out": d_out, "adapters": adapters, "rank": rank,
            "requests": requests, "x": x, "y": out, "bias": bias}


def _scores(name, rows, vocab, top_k, dtype, temperature=1.0, masked=0.0):
    return {"name": name, "op": "scores", "rows": rows, "vocab": vocab, "top_k": top_k, "x": dtype,
            "temperature": temperature, "masked": masked}


def listed():
    return [
        # one frame of one stream ahead of an 8-bit projection: latency
        _norm("norm_token", 1, 1024, "bfloat16"),
        # a 14-frame chunk of 8 streams, f32, the block's own LayerNorm
        _norm("norm_stream", 112, 512, "float32", "layer", out="float32"),
        # a server's batch of 30 s utterances
        _norm("norm_batch", 3000, 1024, "bfloat16"),
        # recordings of 10 minutes at a FeedForward's width
        _norm("norm_long", 15001, 4096, "bfloat16"),
        # one frame of a stream with its speaker's adapter
        _adapters("adapters_token", 1, 1024, 4096, 8, 16, 1, "bfloat16", "bfloat16"),
        # a 14-frame chunk of 8 streams, f32, an adapter for each
        _adapters("adapters_stream", 112, 512, 2048, 32, 16, 8, "float32", "float32", bias=True),
        # a batch of utterances of different lengths, packed, from customers with adapters and without
        _adapters("adapters_batch", 3000, 1024, 4096, 16, 32, 9, "bfloat16", "bfloat16", bias=True),
        # recordings of 10 minutes in pieces of some 375 frames through a FeedForward's second projection
        _adapters("adapters_long", 15001, 4096, 1024, 64, 64, 40, "bfloat16", "bfloat16"),
        # one step of a transducer's decoder: a token's confidence and 4 alternatives
        _scores("scores_token", 1, 1025, 4, "float32"),
        # every frame of a batch, for confidences and lists of alternatives
        _scores("scores_batch", 3000, 1025, 8, "float32"),
        # one step of 64 requests of a text model, a part of the vocabulary ruled out
        _scores("scores_step", 64, 128000, 20, "bfloat16", masked=0.3),
        # prompts scored whole, an odd vocabulary, f32
        _scores("scores_prompt", 4001, 50001, 5, "float32", temperature=0.7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "adapters", "scores"))
    if op == "norm":
        while True:
            rows, d = _log(rng, 1, 30000), _log(rng, 64, 8192)
            if rng.random() < 0.5:  # half of the widths are whole blocks, as the models' are
                d = -(-d // BLOCK) * BLOCK
            if rows * d <= 15001 * 4096:
                break
        c = _norm("", rows, d, rng.choice(tuple(DTYPES)), rng.choice(("rms", "layer")), rng.random() < 0.8,
                  rng.choice(("codes", "codes", "float32", "bfloat16")))
    elif op == "adapters":
        while True:
            rows, d_in, d_out = _log(rng, 1, 15000), _log(rng, 128, 4096), _log(rng, 128, 4096)
            if rng.random() < 0.7:
                d_in, d_out = -(-d_in // BLOCK) * BLOCK, -(-d_out // BLOCK) * BLOCK
            if rows * d_in * d_out <= 15001 * 4096 * 1024:
                break
        x, y = rng.choice((("bfloat16", "bfloat16"), ("float32", "float32"), ("bfloat16", "float32")))
        c = _adapters("", rows, d_in, d_out, rng.choice((1, 4, 8, 16, 64)), rng.choice((4, 8, 16, 24, 32, 64)),
                      min(rows, _log(rng, 1, 100)), x, y, rng.random() < 0.5)
    else:
        while True:
            rows, vocab = _log(rng, 1, 30000), _log(rng, 100, 200000)
            if rows * vocab <= 4001 * 50001:
                break
        c = _scores("", rows, vocab, rng.choice((0, 1, 4, 5, 8, 20, 32)), rng.choice(tuple(DTYPES)),
                    rng.choice((1.0, 1.0, 0.7, 1.3)), rng.choice((0.0, 0.0, 0.3, 0.9)))
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


def _weights(g, n, k):
    """Codes [n, k] (float8_e4m3fn) and biased exponents [ceil(n/128), ceil(k/128)] (uint8) of weights of the usual size."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    w[:n, :k] = torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)
    w = w.view(nb, BLOCK, kb, BLOCK)
    e = _exponent(w.abs().amax((-3, -1)))
    codes = torch.ldexp(w, -e[:, None, :, None]).reshape(nb * BLOCK, kb * BLOCK)[:n, :k]
    return codes.to(torch.float8_e4m3fn).contiguous(), (e + 127).to(torch.uint8)


def _frames(g, rows, d):
    """Activations: a few channels are larger than the others, as after a norm with its weight."""
    gain = torch.exp(0.5 * torch.randn(d, device="cuda", generator=g))
    return torch.randn(rows, d, device="cuda", generator=g) * gain


def _library():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-nemo-rs_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import relpos_mhsa
    return relpos_mhsa


def _rank(case, i):
    """Adapter i's rank: every third has half of the largest."""
    return max(1, case["rank"] // 2) if i % 3 == 2 else case["rank"]


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    rows = case["rows"]
    if case["op"] == "norm":
        d, t = case["d"], DTYPES[case["x"]]
        s["x"] = (3 * _frames(g, rows, d)).to(t)
        s["delta"] = _frames(g, rows, d).to(t) if case["delta"] else None
        s["w"] = torch.exp(0.3 * torch.randn(d, device="cuda", generator=g))
        s["b"] = 0.1 * torch.randn(d, device="cuda", generator=g) if case["kind"] == "layer" else None
    elif case["op"] == "adapters":
        k, n, na, r = case["in"], case["out"], case["adapters"], case["rank"]
        s["x"] = _frames(g, rows, k).to(DTYPES[case["x"]])
        s["codes"], s["scales"] = _weights(g, n, k)
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        s["a"] = (torch.randn(na, r, k, device="cuda", generator=g) / math.sqrt(k)).to(torch.bfloat16)
        s["b"] = (0.3 * torch.randn(na, n, r, device="cuda", generator=g) / math.sqrt(r)).to(torch.bfloat16)
        for i in range(na):
            s["a"][i, _rank(case, i):] = 0
            s["b"][i, :, _rank(case, i):] = 0
        s["s"] = 0.5 + torch.rand(na, device="cuda", generator=g)
        # requests one behind the other, of different lengths, one in eight without an adapter
        ends = torch.sort(torch.randint(0, rows + 1, (case["requests"] - 1,), device="cuda", generator=g)).values
        of = torch.searchsorted(ends, torch.arange(rows, device="cuda"), right=True)
        which = torch.randint(0, na, (case["requests"],), device="cuda", generator=g)
        which[torch.rand(case["requests"], device="cuda", generator=g) < 0.125] = -1
        s["which"] = which[of].to(torch.int32)
        if own:
            m = _library()
            s["layer"] = m.Fp8Linear(k, n, case["bias"])
            s["layer"].load_codes(s["codes"], s["scales"], s["bias"])
            s["adapters"] = m.LowRankAdapters(k, n, na, r)
            for i, scale in enumerate(s["s"].tolist()):
                s["adapters"].load(i, s["a"][i, :_rank(case, i)], s["b"][i, :, :_rank(case, i)], scale)
    else:
        v, t = case["vocab"], DTYPES[case["x"]]
        # peaked and flat rows, as decoders are sure of some tokens and not of others
        z = torch.randn(rows, v, device="cuda", generator=g) * (1 + 3 * torch.rand(rows, 1, device="cuda", generator=g))
        if case["masked"]:
            z[:, torch.rand(v, device="cuda", generator=g) < case["masked"]] = -math.inf
            z[:, 0] = 0.0  # the end of the text is never ruled out
        s["logits"] = z.to(t)
        # half of the given tokens are the likeliest, the last rows are padding
        some = torch.randint(0, v, (rows,), device="cuda", generator=g)
        tokens = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.5, z.argmax(-1), some)
        tokens[rows - rows // 16:] = -1
        s["tokens"] = tokens.to(torch.int32)
    return s


def _coded(y):
    """Codes (e4m3) and powers of two of rows of 128 values in f32."""
    k = y.shape[-1]
    kb = -(-k // BLOCK)
    p = torch.nn.functional.pad(y, (0, kb * BLOCK - k)).unflatten(-1, (kb, BLOCK))
    e = _exponent(p.abs().amax(-1, keepdim=True))
    return torch.ldexp(p, -e).to(torch.float8_e4m3fn), e


def _plain_norm(s):
    c = s["case"]
    v = s["x"].float()
    out = {}
    if s["delta"] is not None:
        v = v + 0.5 * s["delta"].float()
        out["sum"] = v.to(s["x"].dtype)
    if c["kind"] == "rms":
        y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["w"]
    else:
        u = v - v.mean(-1, keepdim=True)
        y = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * s["w"] + s["b"]
    if c["out"] == "codes":
        codes, e = _coded(y)
        out["codes"] = codes.flatten(-2)[..., :c["d"]]
        out["scales"] = (e[..., 0] + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    else:
        out["out"] = y.to(DTYPES[c["out"]])
    return out


def _plain_adapters(s):
    c = s["case"]
    x, k, n = s["x"].float(), c["in"], c["out"]
    codes, e = _coded(x)
    q = torch.ldexp(codes.float(), e).flatten(-2)[..., :k]
    w = torch.ldexp(torch.ones((), device=x.device), s["scales"].to(torch.int32) - 127)
    w = s["codes"].float() * w.repeat_interleave(BLOCK, -2)[:n].repeat_interleave(BLOCK, -1)[:, :k]
    y = q @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    na, r, which = c["adapters"], c["rank"], s["which"].long()
    if c["rows"] * k <= 256 * 1024:  # few rows: each one's adapter gathered
        a, b = s["a"][which.clamp_min(0)].float(), s["b"][which.clamp_min(0)].float()
        scale = torch.where(which >= 0, s["s"][which.clamp_min(0)], 0)
        y = y + ((a * x[:, None]).sum(-1)[:, None] * b).sum(-1) * scale[:, None]
    else:  # every adapter's product, those of other rows struck out
        t = (x @ s["a"].float().flatten(0, 1).T).view(-1, na, r)
        mine = which[:, None] == torch.arange(na, device=x.device)
        t = t * (mine * s["s"])[..., None]
        y = y + t.flatten(1) @ s["b"].float().transpose(1, 2).reshape(na * r, n)
    return y.to(DTYPES[c["y"]])


def _plain_scores(s):
    c, v = s["case"], s["case"]["vocab"]
    x = s["logits"].float()
    z = x / c["temperature"]
    m = z.amax(-1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    tokens = s["tokens"].long()[:, None]
    given = z.gather(-1, tokens.clamp_min(0)) - lse
    out = {"log_probs": torch.where(tokens >= 0, given, 0)[:, 0],
           "entropy": (torch.log(total) - torch.where(e > 0, d * e, 0).sum(-1, keepdim=True) / total)[:, 0]}
    if c["top_k"]:
        bits = (x + 0.0).view(torch.int32)  # (+ 0: the two zeros are alike)
        bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)  # in the order of the values
        key = (bits.long() << 32) + (v - 1 - torch.arange(v, device=x.device))  # larger for the lower index
        top = key.topk(c["top_k"], dim=-1).values
        idx = v - 1 - (top & 0xFFFFFFFF)
        there = x.gather(-1, idx) > -math.inf
        out["top_log_probs"] = z.gather(-1, idx) - lse
        out["top_indices"] = torch.where(there, idx, -1).to(torch.int32)
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"norm": _plain_norm, "adapters": _plain_adapters, "scores": _plain_scores}[c["op"]](state)
    m = _library()
    if c["op"] == "norm":
        codes = c["out"] == "codes"
        r = m.add_norm(state["x"], state["delta"], state["w"], state["b"], kind=c["kind"], eps=EPS, scale=0.5,
                       want="codes" if codes else "out", out_dtype=None if codes else DTYPES[c["out"]])
        out = {} if r.sum is None else {"sum": r.sum}
        if codes:
            out["codes"] = r.codes.codes.view(torch.float8_e4m3fn)[:, :c["d"]]
            out["scales"] = r.codes.scales.view(torch.float8_e8m0fnu)[:, :-(-c["d"] // BLOCK)]
        else:
            out["out"] = r.out
        return out
    if c["op"] == "adapters":
        return state["layer"].forward(state["x"], out_dtype=DTYPES[c["y"]], adapters=state["adapters"], which=state["which"])
    r = m.token_log_probs(state["logits"], state["tokens"], top_k=c["top_k"], temperature=c["temperature"])
    out = {"log_probs": r.log_probs, "entropy": r.entropy}
    if c["top_k"]:
        out["top_log_probs"], out["top_indices"] = r.top_log_probs, r.top_indices
    return out


def work(case):
    rows = case["rows"]
    if case["op"] == "norm":
        d, es = case["d"], SIZES[case["x"]]
        out = 1 + 1 / BLOCK if case["out"] == "codes" else SIZES[case["out"]]
        return {"bytes": rows * d * ((3 if case["delta"] else 1) * es + out) + d * (8 if case["kind"] == "layer" else 4),
                "flops": 0}
    if case["op"] == "adapters":
        k, n, r = case["in"], case["out"], case["rank"]
        used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** (0.875 * case["requests"]))  # that some request has
        return {"bytes": rows * k * SIZES[case["x"]] + n * k + used * 2 * r * (k + n) + rows * n * SIZES[case["y"]] + 4 * rows,
                "flops": 2.0 * rows * (n * k + 0.875 * r * (n + k))}
    return {"bytes": rows * (case["vocab"] * SIZES[case["x"]] + 12 + 8 * case["top_k"]), "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_codes(v):
    """Blocks of the last axis as e4m3 steps of their power of two (to nearest, ties to the even step), and the powers."""
    codes, powers = torch.zeros_like(v), []
    for lo in range(0, v.shape[-1], BLOCK):
        b = v[..., lo:lo + BLOCK]
        top = b.abs().max(-1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0))
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)  # log2 rounds
        e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp_min(-127)
        e = torch.where(top > 0, e, 0)
        t = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)  # 2^-9 below the smallest normal
        codes[..., lo:lo + BLOCK] = torch.round(t / step) * step
        powers.append(torch.exp2(e))
    return codes, torch.cat(powers, -1)


def _exact_norm(s):
    c = s["case"]
    v, out = s["x"].double(), {}
    if s["delta"] is not None:
        v = v + s["delta"].double() / 2
        out["sum"] = v
    mean = v.sum(-1, keepdim=True) / c["d"] if c["kind"] == "layer" else 0.0
    var = (v - mean).pow(2).sum(-1, keepdim=True) / c["d"]
    y = (v - mean) / torch.sqrt(var + EPS) * s["w"].double()
    if s["b"] is not None:
        y = y + s["b"].double()
    if c["out"] == "codes":
        out["codes"], out["scales"] = _exact_codes(y)
    else:
        out["out"] = y
    return out


def _exact_adapters(s):
    c, x = s["case"], s["x"].double()
    codes, powers = _exact_codes(x)
    q = codes * powers.repeat_interleave(BLOCK, -1)[..., :c["in"]]
    w, scales = s["codes"].double(), s["scales"].cpu()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= 2.0 ** (int(scales[i, j]) - 127)
    y = q @ w.T
    if s["bias"] is not None:
        y += s["bias"].double()
    for i in range(c["adapters"]):
        at = torch.nonzero(s["which"] == i).flatten()
        if at.numel():
            r = _rank(c, i)
            y[at] += float(s["s"][i]) * (x[at] @ s["a"][i, :r].double().T) @ s["b"][i, :, :r].double().T
    return y


def _exact_scores(s):
    c, parts = s["case"], []
    step = max(1, (1 << 27) // c["vocab"])
    for lo in range(0, c["rows"], step):
        z = s["logits"][lo:lo + step].double() / c["temperature"]
        lp = torch.log_softmax(z, -1)
        tok = s["tokens"][lo:lo + step].long()
        given = lp[torch.arange(len(tok), device=tok.device), tok.clamp_min(0)]
        part = [torch.where(tok < 0, 0.0, given), torch.special.entr(lp.exp()).sum(-1)]
        if c["top_k"]:
            part.append(lp.topk(c["top_k"], -1).values)
        parts.append(part)
    cat = [torch.cat(p) for p in zip(*parts)]
    out = {"log_probs": cat[0], "entropy": cat[1]}
    if c["top_k"]:
        out["top_log_probs"], out["top_indices"] = cat[2], None
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "adapters": _exact_adapters, "scores": _exact_scores}[case["op"]](s)
