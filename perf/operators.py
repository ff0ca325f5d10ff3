"""The operators of a Transformer's training step around the framework's attention and Dense layers, as cases to
measure: the embedding lookup and its gradient, the norm / gate / residual step between two blocks and its gradient,
and the AdamW step over all tensors of a model with its states in 32 or in 8 bits.

``run`` computes each in elementary torch operations, or (``own``) through the framework's layers."""
import math

import torch

own = False

INDEX_DTYPES = {"int32": torch.int32, "int64": torch.int64, "fp32": torch.float32}
EPSILON = 1e-5
BLOCK = 256                                    # elements that share a scale in the 8-bit states
BETA1, BETA2, ADAM_EPS, RATE = 0.9, 0.999, 1e-8, 1e-3


# ------------------------------------------------------------------------------------------------ cases
def _embedding_case(name, backward, tokens, vocab, dim, index, padding=False, accumulate=False):
    return {"name": name, "op": "embedding_backward" if backward else "embedding_forward", "tokens": tokens, "vocab": vocab,
            "dim": dim, "index": index, "padding": padding, "accumulate": accumulate}


def _norm_case(name, backward, rows, dim, norm, post_norm="none", block=True, gate_rows=0, residual_scale=1.0):
    return {"name": name, "op": "norm_backward" if backward else "norm_forward", "rows": rows, "dim": dim, "norm": norm,
            "post_norm": post_norm, "block": block, "gate_rows": gate_rows, "residual_scale": residual_scale}


def _adam_case(name, bits, width, layers, vocab, step):
    return {"name": name, "op": "adam", "bits": bits, "width": width, "layers": layers, "vocab": vocab, "step": step}


def listed():
    return [
        # the next token of one sequence enters the model: latency
        _embedding_case("embed one token", False, 1, 32768, 4096, "int32"),
        # a training batch of 32 sequences of 512 tokens
        _embedding_case("embed a batch", False, 16384, 32768, 1024, "int64"),
        # a padded batch over a small vocabulary, indices held as floats as the framework's tensors do, odd sizes,
        # added to a gradient that is there already (input and output embedding share their weights)
        _embedding_case("embed gradient, ragged", True, 4999, 10007, 333, "fp32", padding=True, accumulate=True),
        # the gradient of a training batch
        _embedding_case("embed gradient, batch", True, 16384, 32768, 1024, "int64"),
        # a large batch over a large vocabulary
        _embedding_case("embed gradient, long", True, 262144, 131072, 1024, "int32"),
        # one token between two blocks, norms on both sides of the block and a gate per channel: latency
        _norm_case("norm one token", False, 1, 4096, "rms", "rms", gate_rows=1),
        # residual + LayerNorm after a block of a training batch
        _norm_case("norm, batch", False, 16384, 4096, "layer"),
        # the multi-head attention batch of the benchmark: 32 x 128 tokens of 512
        _norm_case("norm gradient, attention", True, 4096, 512, "layer"),
        # a gate per sequence (7 of 211 steps), odd width, scaled residual
        _norm_case("norm gradient, ragged", True, 1477, 777, "rms", "rms", gate_rows=7, residual_scale=0.70710677),
        # everything at once on a large batch
        _norm_case("norm gradient, large", True, 16384, 4096, "rms", "layer", gate_rows=1),
        # four blocks of width 512: 64 tensors from 512 to a million elements
        _adam_case("adam 32 bits, blocks", 32, 512, 4, 0, 10),
        # twelve blocks of width 1024 and an embedding: 193 tensors, 185 million parameters
        _adam_case("adam 8 bits, model", 8, 1024, 12, 32768, 1000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("embedding_forward", "embedding_backward", "embedding_backward", "norm_forward", "norm_backward",
                     "norm_backward", "adam", "adam"))
    if op.startswith("embedding"):
        dim = _log(rng, 16, 4096)
        if rng.random() < 0.5:
            dim = dim // 4 * 4
        tokens, vocab = _log(rng, 1, min(262144, (1 << 27) // dim)), _log(rng, 2, min(131072, (1 << 27) // dim))
        c = _embedding_case("", op == "embedding_backward", tokens, vocab, dim, rng.choice(sorted(INDEX_DTYPES)),
                       rng.random() < 0.3, op == "embedding_backward" and rng.random() < 0.4)
    elif op.startswith("norm"):
        dim = _log(rng, 16, 8192)
        if rng.random() < 0.6:
            dim = dim // 4 * 4
        groups = rng.choice((0, 0, 1, 1, _log(rng, 2, 64)))
        per_group = _log(rng, 1, max(1, min(32768, (1 << 25) // dim) // max(1, groups)))
        block = groups > 0 or rng.random() < 0.8
        c = _norm_case("", op == "norm_backward", per_group * max(1, groups), dim, rng.choice(("layer", "rms")),
                  rng.choice(("none", "none", "layer", "rms")) if block else "none", block, groups,
                  rng.choice((1.0, 0.70710677, 2.0)) if block else 1.0)
    else:
        bits, width = rng.choice((8, 32)), _log(rng, 48, 1024)
        c = _adam_case("", bits, width, rng.randint(1, 8 if bits == 8 else 6), rng.choice((0, _log(rng, 100, 32768))), rng.choice((1, 7, 100, 5000)))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tensor_sizes(case):
    """The parameter tensors of a model: (elements, whether weight decay applies)."""
    w = case["width"]
    sizes = [(case["vocab"] * w, True)] if case["vocab"] else []
    for _ in range(case["layers"]):
        for _ in range(4):
            sizes += [(w * w, True), (w, False)]
        sizes += [(4 * w * w, True), (4 * w, False), (4 * w * w, True), (w, False)] + [(w, False)] * 4
    return sizes


def _gate_rows(case):
    """The row of the gate that each row of the batch uses."""
    return torch.arange(case["rows"], device="cuda") // max(1, case["rows"] // max(1, case["gate_rows"]))


def _statistics(t, kind):
    t = t.double()
    mean = t.mean(1) if kind == "layer" else torch.zeros(t.shape[0], dtype=torch.float64, device="cuda")
    rstd = torch.rsqrt((t - mean[:, None]).square().mean(1) + EPSILON)
    return torch.stack((mean, rstd), 1)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(mean)

    if case["op"].startswith("embedding"):
        n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        # word frequencies fall with the rank (Zipf): the logarithm of rank + 1 is uniform
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        ids = (torch.exp(u * math.log(vocab + 1)) - 1).floor().clamp_(0, vocab - 1).long()
        if case["padding"]:
            ids[torch.rand(n, device="cuda", generator=g) < 0.2] = 0
        s["ids"] = ids.to(INDEX_DTYPES[case["index"]])
        s["scale"] = math.sqrt(dim)
        s["padding"] = 0 if case["padding"] else -1
        if case["op"] == "embedding_forward":
            s["table"], s["y"] = normal(vocab, dim, scale=0.02), torch.zeros(n, dim, device="cuda")
        else:
            s["dy"] = normal(n, dim, scale=1e-2)
            s["dtable"] = normal(vocab, dim, scale=1e-2) if case["accumulate"] else torch.zeros(vocab, dim, device="cuda")
    elif case["op"].startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        affine = lambda kind, mean: normal(dim, scale=0.1, mean=mean) if kind else None  # noqa: E731
        s["gamma"], s["beta"] = affine(True, 1.0), affine(case["norm"] == "layer", 0.0)
        post = case["post_norm"] != "none"
        s["post_gamma"], s["post_beta"] = affine(post, 1.0), affine(case["post_norm"] == "layer", 0.0)
        s["gate"] = normal(case["gate_rows"], dim, scale=0.3, mean=0.5) if case["gate_rows"] else None
        s["h"] = normal(rows, dim, scale=1.5, mean=0.2) if case["block"] else None
        if case["op"] == "norm_forward":
            s["x"] = normal(rows, dim, scale=2.0, mean=0.3)
            s["y"] = torch.zeros(rows, dim, device="cuda")
            s["r"] = torch.zeros(rows, dim, device="cuda") if case["block"] else None
            s["stats"], s["post_stats"] = torch.zeros(rows, 2, device="cuda"), torch.zeros(rows, 2, device="cuda") if post else None
        else:
            s["r"] = normal(rows, dim, scale=2.5, mean=0.3)                   # what the forward pass left
            s["stats"] = _statistics(s["r"], case["norm"]).float()
            s["post_stats"] = _statistics(s["h"], case["post_norm"]).float() if post else None
            s["dy"], s["dr"] = normal(rows, dim, scale=1e-2), normal(rows, dim, scale=1e-2)
            s["dx"] = torch.zeros(rows, dim, device="cuda")
            s["dh"] = torch.zeros(rows, dim, device="cuda") if case["block"] else None
            for p in ("gamma", "beta", "post_gamma", "post_beta", "gate"):
                s["d_" + p] = None if s[p] is None else torch.zeros_like(s[p])
    else:
        # the tensors of the model in one buffer each for weights, gradients and states, every tensor at a multiple
        # of BLOCK elements; the gaps hold zeros and stay zero
        s["sizes"] = _tensor_sizes(case)
        blocks = [-(-n // BLOCK) for n, _ in s["sizes"]]
        s["starts"] = [BLOCK * sum(blocks[:i]) for i in range(len(blocks))]
        total = BLOCK * sum(blocks)
        counts = torch.tensor(blocks, device="cuda")
        ordinal = torch.repeat_interleave(torch.arange(len(blocks), device="cuda"), counts)       # tensor of each block
        first = torch.repeat_interleave(counts.cumsum(0) - counts, counts)
        s["ordinal"], s["block"] = ordinal, torch.arange(total // BLOCK, device="cuda") - first   # block within its tensor
        elements = torch.tensor([n for n, _ in s["sizes"]], device="cuda")[ordinal]
        s["decay"] = torch.tensor([float(d) for _, d in s["sizes"]], device="cuda")[ordinal]
        live = s["block"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < elements[:, None]
        scale = torch.exp(normal(total // BLOCK, 1)) * 1e-3                   # gradients differ from row to row
        s["W"] = normal(total // BLOCK, BLOCK, scale=0.02).mul_(live)
        s["dW"] = normal(total // BLOCK, BLOCK).mul_(scale).mul_(live)
        v = normal(total // BLOCK, BLOCK, scale=0.3).mul_(scale).mul_(live)
        r = normal(total // BLOCK, BLOCK).abs_().mul_(scale).mul_(live)      # the root of the second moment
        if case["bits"] == 8:
            s["v_scale"], s["s_scale"] = _power_of_two(v.abs().amax(1)), _power_of_two(r.amax(1))
            s["v"], s["s"] = (t.mul_(_inverse(c)[:, None]).to(torch.float8_e4m3fn) for t, c in ((v, s["v_scale"]), (r, s["s_scale"])))
        else:
            s["v"], s["s"] = v, r.square_()
        s["t"] = case["step"] - 1
        if case["step"] == 1:                                                 # the first step: no history
            s.update({k: torch.zeros_like(s[k], dtype=torch.uint8 if k in "vs" and case["bits"] == 8 else None).view(s[k].dtype)
                      for k in ("v", "s", "v_scale", "s_scale") if k in s})
    if own:
        _bind(s)
    return s


def _bind(s):
    """The layer or optimizer object of the user's program, around the tensors that are there."""
    from sharpnet_b200.embedding import EmbeddingLayer
    from sharpnet_b200.normalization import ResidualNorm
    from sharpnet_b200.optimizers import AdamGroup
    from sharpnet_b200.tensor import GPUTensor, GPUWrapper
    w, c = GPUWrapper.FromDeviceId(0), s["case"]
    tensor = lambda t, shape=None: None if t is None else GPUTensor(shape or t.shape, None, w, t.view(-1))  # noqa: E731
    if c["op"].startswith("embedding"):
        s["layer"] = EmbeddingLayer(c["vocab"], c["dim"], w, scale=s["scale"], paddingIndex=s["padding"],
                                    weights=tensor(s.get("table")), weightGradients=tensor(s.get("dtable")))
        s["x"] = tensor(s["ids"]) if c["index"] == "fp32" else s["ids"]
        s["out"] = tensor(s.get("y")) if c["op"] == "embedding_forward" else tensor(s["dy"])
    elif c["op"].startswith("norm"):
        names = ("gamma", "beta", "post_gamma", "post_beta", "gate")
        s["layer"] = ResidualNorm(c["dim"], w, norm=c["norm"], post_norm=c["post_norm"], gate_rows=c["gate_rows"],
                                  residual_scale=c["residual_scale"], epsilon=EPSILON,
                                  parameters={p: tensor(s[p]) for p in names},
                                  gradients={p: tensor(s.get("d_" + p)) for p in names})
        s["layer"].SetStatistics(tensor(s["stats"]), tensor(s["post_stats"]))
        s["tensors"] = {k: tensor(s.get(k)) for k in ("x", "h", "r", "y", "dy", "dr", "dx", "dh")}
    else:
        def part(name, i, per=1):
            n, at = s["sizes"][i][0], s["starts"][i]
            return s[name].view(-1)[at // per: at // per + -(-n // per)]

        n = len(s["sizes"])
        states = ("v", "s", "v_scale", "s_scale") if c["bits"] == 8 else ("v", "s")
        s["group"] = AdamGroup(w, BETA1, BETA2, ADAM_EPS, 0.01,
                               [tensor(part("W", i)) for i in range(n)], [tensor(part("dW", i)) for i in range(n)],
                               decays=[float(d) for _, d in s["sizes"]], state_bits=c["bits"],
                               states=[tuple(part(k, i, BLOCK if "scale" in k else 1) for k in states) for i in range(n)],
                               timestep=s["t"])


# ------------------------------------------------------------------------------------------------ plain forms
def _normalized(t, stats):
    return (t - stats[:, :1]) * stats[:, 1:]


def _plain_statistics(t, kind):
    mean = t.mean(1, keepdim=True) if kind == "layer" else torch.zeros(t.shape[0], 1, device="cuda")
    return torch.cat((mean, 1 / ((t - mean).square().mean(1, keepdim=True) + EPSILON).sqrt()), 1)


def _affine(t, gamma, beta):
    t = t if gamma is None else t * gamma
    return t if beta is None else t + beta


def _norm_input_gradient(g, xhat, rstd, kind):
    if kind == "layer":
        g = g - g.mean(1, keepdim=True)
    return rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))


def _norm_forward(s):
    c, r, h = s["case"], s["x"] * s["case"]["residual_scale"], s["h"]
    if h is not None:
        u = h if c["post_norm"] == "none" else _affine(_normalized(h, _plain_statistics(h, c["post_norm"])), s["post_gamma"], s["post_beta"])
        r = r + (u if s["gate"] is None else u * s["gate"][_gate_rows(c)])
    y = _affine(_normalized(r, _plain_statistics(r, c["norm"])), s["gamma"], s["beta"])
    return {"y": y, "r": r} if h is not None else {"y": y}


def _norm_backward(s):
    c, dy, h = s["case"], s["dy"], s["h"]
    xhat = _normalized(s["r"], s["stats"])
    out = {"gamma": (dy * xhat).sum(0)}
    if s["beta"] is not None:
        out["beta"] = dy.sum(0)
    dr = s["dr"] + _norm_input_gradient(dy * s["gamma"], xhat, s["stats"][:, 1:], c["norm"])
    out["dx"] = c["residual_scale"] * dr
    if h is None:
        return out
    post = c["post_norm"] != "none"
    hhat = _normalized(h, s["post_stats"]) if post else h
    du = dr
    if s["gate"] is not None:
        u = _affine(hhat, s["post_gamma"], s["post_beta"])
        out["gate"] = (dr * u).view(c["gate_rows"], -1, c["dim"]).sum(1)
        du = dr * s["gate"][_gate_rows(c)]
    if post:
        out["post_gamma"] = (du * hhat).sum(0)
        if s["post_beta"] is not None:
            out["post_beta"] = du.sum(0)
        du = _norm_input_gradient(du * s["post_gamma"], hhat, s["post_stats"][:, 1:], c["post_norm"])
    out["dh"] = du
    return out


def _exponent(t):
    """floor(log2(t)) of positive normal numbers."""
    return (t.view(torch.int32) >> 23) - 127


def _power_of_two(largest):
    """The scale of a block of 8-bit states whose largest magnitude is given: the power of two that brings it to
    [128, 256); 0 for a block of zeros."""
    scale = ((_exponent(largest) - 7 + 127) << 23).view(torch.float32)
    return torch.where(largest < 2.0 ** -100, torch.zeros_like(scale), scale)


def _inverse(scale):
    inverse = ((254 << 23) - scale.view(torch.int32)).view(torch.float32)
    return torch.where(scale == 0, torch.zeros_like(scale), inverse)


def _random20(s, seed):
    """20 random bits for every element: of the tensor's ordinal, the pair of elements and the step's seed; the first
    element of a pair takes the low bits of the hash, the second the high ones."""
    m = 0xFFFFFFFF
    pair = s["block"][:, None] * (BLOCK // 2) + torch.arange(BLOCK // 2, device="cuda")
    x = (seed * 0x9E3779B1 + s["ordinal"][:, None] * 0x85EB9A77 + pair) & m
    x = ((x ^ (x >> 16)) * 0x6C8E9CF5) & m
    x = ((x ^ (x >> 12)) * 0xB5297A4D) & m
    x = x ^ (x >> 15)
    return torch.stack(((x & 0xFFFF) << 4, (x >> 16) << 4), 2).view(-1, BLOCK).int()


def _adam(s):
    c = s["case"]
    s["t"] += 1
    t = s["t"]
    factor = RATE * math.sqrt(1 - BETA2 ** t) / (1 - BETA1 ** t)
    # the coefficients as 32-bit numbers, and each operation rounded to 32 bits: that defines the 8-bit states
    b1, b2 = torch.tensor([BETA1, BETA2], device="cuda")
    v, r, W, g = s["v"], s["s"], s["W"], s["dW"]
    if c["bits"] == 8:
        v, r = v.float() * s["v_scale"][:, None], r.float() * s["s_scale"][:, None]
        r = r * r
    v = b1 * v + (1 - b1) * g
    sq = b2 * r + ((1 - b2) * g) * g
    root = sq.sqrt()
    W.copy_(W - (factor * v / (root + ADAM_EPS) + (0.01 * s["decay"])[:, None] * W))
    if c["bits"] == 32:
        s["v"].copy_(v)
        s["s"].copy_(sq)
        return {"W": W, "v": s["v"], "s": s["s"]}
    s["v_scale"].copy_(_power_of_two(v.abs().amax(1)))
    s["s_scale"].copy_(_power_of_two(root.amax(1)))
    s["v"].copy_((v * _inverse(s["v_scale"])[:, None]).to(torch.float8_e4m3fn))
    # the root is rounded up or down at random in proportion: in the normal range of the 8 bits by adding the random
    # bits below the three that stay, below 2^-6 on the fixed grid of 2^-9; never to zero unless it is zero
    x, rnd = root * _inverse(s["s_scale"])[:, None], _random20(s, t)
    high = ((x.view(torch.int32) + rnd) & ~0xFFFFF).view(torch.float32)
    low = (x * 512 + rnd * 2.0 ** -20).floor().clamp(min=1) * 2.0 ** -9
    s["s"].copy_(torch.where(x < 2.0 ** -6, torch.where(x > 0, low, torch.zeros_like(x)), high).to(torch.float8_e4m3fn))
    return {"W": W, "v": s["v"], "s": s["s"], "v_scale": s["v_scale"], "s_scale": s["s_scale"]}


def run(state):
    s, c = state, state["case"]
    if own:
        if c["op"] == "embedding_forward":
            s["layer"].ForwardPropagation(s["x"], s["out"])
            return s["y"]
        if c["op"] == "embedding_backward":
            s["layer"].BackwardPropagation(s["x"], s["out"], accumulate=c["accumulate"])
            return s["dtable"]
        if c["op"] == "norm_forward":
            t = s["tensors"]
            s["layer"].ForwardPropagation(t["x"], t["h"], t["r"], t["y"])
            return {"y": s["y"], "r": s["r"]} if c["block"] else {"y": s["y"]}
        if c["op"] == "norm_backward":
            t = s["tensors"]
            s["layer"].BackwardPropagation(t["r"], t["h"], t["dy"], t["dr"], t["dx"], t["dh"])
            out = {p: s["d_" + p] for p in ("gamma", "beta", "post_gamma", "post_beta", "gate") if s["d_" + p] is not None}
            return {**out, "dx": s["dx"], "dh": s["dh"]} if c["block"] else {**out, "dx": s["dx"]}
        s["group"].UpdateWeights(RATE, RATE)
        return {k: s[k] for k in ("W", "v", "s", "v_scale", "s_scale") if k in s}
    if c["op"] == "embedding_forward":
        return s["table"][s["ids"].long()] * s["scale"]
    if c["op"] == "embedding_backward":
        ids = s["ids"].long()
        kept = s["dy"] * (ids != s["padding"])[:, None]
        # the sums of the frequent words are long: in 64 bits
        sums = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device="cuda").index_add_(0, ids, kept.double()) * s["scale"]
        return s["dtable"].copy_(s["dtable"] + sums if c["accumulate"] else sums)
    if c["op"] == "norm_forward":
        return _norm_forward(s)
    if c["op"] == "norm_backward":
        return _norm_backward(s)
    return _adam(s)


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    c = case
    if c["op"].startswith("embedding"):
        n, index = c["tokens"] * c["dim"], c["tokens"] * (8 if c["index"] == "int64" else 4)
        # how many words are expected to occur in the batch
        word = torch.arange(c["vocab"], dtype=torch.float64)
        never = (1 - torch.log((word + 2) / (word + 1)) / math.log(c["vocab"] + 1)) ** c["tokens"]
        rows = round(float((1 - never).sum())) * c["dim"]
        if c["op"] == "embedding_forward":
            return {"bytes": 4 * (n + rows) + index, "flops": n}
        # the table's gradient is written whole, or the rows of the batch are read and written
        return {"bytes": 4 * n + index + (8 * rows if c["accumulate"] else 4 * c["vocab"] * c["dim"]), "flops": 2 * n}
    if c["op"].startswith("norm"):
        n = c["rows"] * c["dim"]
        if c["op"] == "norm_forward":                    # x, h -> r, y
            return {"bytes": 4 * n * (4 if c["block"] else 2), "flops": 16 * n}
        # dy, dr, r, h -> dx, dh; h itself is needed for its norm and for the gate's gradient alone
        reads = 3 + (c["block"] and (c["gate_rows"] > 0 or c["post_norm"] != "none"))
        return {"bytes": 4 * n * (reads + 1 + c["block"]), "flops": 30 * n}
    n = sum(k for k, _ in _tensor_sizes(c))
    return {"bytes": n * (28 if c["bits"] == 32 else 16) + (0 if c["bits"] == 32 else n // BLOCK * 16), "flops": 14 * n}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def _exact_norm(t, kind, gamma, beta):
    if kind == "none":
        return t
    t = t - t.mean(1, keepdim=True) if kind == "layer" else t
    t = t / (t.square().sum(1, keepdim=True) / t.shape[1] + EPSILON).sqrt()
    t = t if gamma is None else gamma * t
    return t if beta is None else beta + t


def _exact_block(c, p, x, h):
    r = c["residual_scale"] * x
    if h is None:
        return r
    u = _exact_norm(h, c["post_norm"], p["post_gamma"], p["post_beta"])
    if p["gate"] is not None:
        u = (u.view(c["gate_rows"], -1, c["dim"]) * p["gate"][:, None, :]).view_as(u)
    return r + u


def _exact_norm_backward(c, s, p):
    """By the chain rule of the two functions that the forward pass is made of, differentiated by torch."""
    # dx and dh depend on r = residual_scale x + ... alone, so x is taken as what gives this r
    dr, out = s["dr"].double(), {}
    r = s["r"].double().requires_grad_()
    leaves = [p[k].requires_grad_() for k in ("gamma", "beta") if p[k] is not None]
    y = _exact_norm(r, c["norm"], p["gamma"], p["beta"])
    found = torch.autograd.grad(y, [r] + leaves, s["dy"].double())
    dr = dr + found[0]
    out.update(zip([k for k in ("gamma", "beta") if p[k] is not None], found[1:]))
    out["dx"] = c["residual_scale"] * dr
    if s["h"] is not None:
        h = s["h"].double().requires_grad_()
        names = [k for k in ("post_gamma", "post_beta", "gate") if p[k] is not None]
        block = _exact_block(c, {k: None if v is None else v.requires_grad_() for k, v in p.items()}, torch.zeros_like(dr), h)
        found = torch.autograd.grad(block, [h] + [p[k] for k in names], dr)
        out["dh"] = found[0]
        out.update(zip(names, found[1:]))
    return out


def _round32(t):
    """To the nearest 32-bit number (one operation on 32-bit numbers in 64 bits, rounded so, is the 32-bit operation)."""
    return t.float().double()


def _exact_scale(largest):
    m, e = torch.frexp(largest)                          # largest = m 2^e, m in [0.5, 1)
    return torch.where(largest < 2.0 ** -100, torch.zeros_like(largest), torch.ldexp(torch.ones_like(largest), e - 8))


def _exact_e4m3(t):
    """The nearest 8-bit number (4 bits of exponent, 3 of mantissa, subnormals in steps of 2^-9), ties to even."""
    _, e = torch.frexp(t)
    grid = torch.ldexp(torch.ones_like(t), (e - 4).clamp(min=-9))
    return torch.round(t / grid) * grid


def _exact_adam(c, s):
    t = c["step"]
    factor = RATE * math.sqrt(1 - BETA2 ** t) / (1 - BETA1 ** t)
    b1, b2 = (float(torch.tensor(b, dtype=torch.float32)) for b in (BETA1, BETA2))
    one_b1, one_b2 = (float(torch.tensor(1 - b, dtype=torch.float32)) for b in (b1, b2))
    eight = c["bits"] == 8
    near = _round32 if eight else (lambda x: x)
    g = s["dW"].double()
    v = s["v"].float().double() * (s["v_scale"].double()[:, None] if eight else 1)
    r = near(s["s"].float().double() * (s["s_scale"].double()[:, None] if eight else 1))
    sq = near(r * r) if eight else r
    v = near(near(b1 * v) + near(one_b1 * g))
    sq = near(near(b2 * sq) + near(near(one_b2 * g) * g))
    root = near(sq.sqrt())
    W = s["W"].double()
    out = {"W": W - (factor * v / (root + ADAM_EPS) + 0.01 * s["decay"].double()[:, None] * W)}
    if not eight:
        return {**out, "v": v, "s": sq}
    out["v_scale"], out["s_scale"] = _exact_scale(v.abs().amax(1)), _exact_scale(root.amax(1))
    inverse = [torch.where(k == 0, k, 1 / k)[:, None] for k in (out["v_scale"], out["s_scale"])]
    out["v"] = _exact_e4m3(v * inverse[0])
    # stochastic: the value's place between its two neighbours, counted in 2^20ths, plus the random bits, cut off
    x, rnd = root * inverse[1], _random20(s, t).double()
    _, e = torch.frexp(x)
    grid = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    place = torch.where(x < 2.0 ** -6, _round32(x * 512 + rnd * 2.0 ** -20), x / grid + rnd * 2.0 ** -20)
    out["s"] = torch.where(x > 0, place.floor().clamp(min=1) * grid, torch.zeros_like(x))
    return out


def exact(case, seed):
    global own
    c, kept = case, own
    own = False
    s = prepare(case, seed)
    own = kept
    if c["op"] == "embedding_forward":
        return s["table"].double()[s["ids"].long()] * s["scale"]
    if c["op"] == "embedding_backward":
        # sorted by word; the sum of a word's rows is the difference of two running sums over all rows
        ids, order = s["ids"].long().sort()
        rows = s["dy"].double()[order]
        rows[ids == s["padding"]] = 0
        running = torch.cat((torch.zeros(1, c["dim"], dtype=torch.float64, device="cuda"), rows.cumsum_(0)))
        words = torch.arange(c["vocab"], device="cuda")
        sums = running[torch.searchsorted(ids, words, right=True)] - running[torch.searchsorted(ids, words)]
        return s["dtable"].double() + s["scale"] * sums if c["accumulate"] else s["scale"] * sums
    p = {k: None if s.get(k) is None else s[k].double() for k in ("gamma", "beta", "post_gamma", "post_beta", "gate")}
    if c["op"] == "norm_forward":
        r = _exact_block(c, p, s["x"].double(), None if s["h"] is None else s["h"].double())
        y = _exact_norm(r, c["norm"], p["gamma"], p["beta"])
        return {"y": y, "r": r} if s["h"] is not None else {"y": y}
    if c["op"] == "norm_backward":
        return _exact_norm_backward(c, s, p)
    return _exact_adam(c, s)
