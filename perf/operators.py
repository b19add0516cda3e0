"""Products with 4-bit weights: what a model does with the codes, scales and zero points that quantization_amd computes.

Four operators over a weight held as 4-bit codes with float16 scales (and, asymmetric, float16 zero points) per group of
input channels, each in its plain form and as the framework's call:

  linear         y = x W^T + b                    packed_linear(x, weight, bias)
  linear_train   the same with dx = dy W, db       ... and its backward pass (the weight is frozen)
  experts        y[r] = x[r] W[e(r)]^T + b[e(r)]   packed_expert_linear(x, weight, counts, bias), rows sorted by expert
  experts_train  the same with dx, db              ... and its backward pass

with W[n, k] = scale[n, k // g] * (q[n, k] - zero[n, k // g]); q an integer or a value of a 4-bit table.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_TABLES = {"fp4": [1, 2, 3, 4, 6, 8, 12], "flint4": [1, 2, 3, 4, 6, 8, 16]}
_FORMATS = ["int4", "int4_asym", "fp4", "flint4"]
_MOST_FLOPS = 4.9e11   # of the largest listed case: what a drawn one may cost
_MOST_WEIGHTS = 5.3e8


def _case(op, rows, n, k, group, fmt, dtype, bias=False, experts=1, skew=0.0, spare=0):
    return {"op": op, "rows": rows, "n": n, "k": k, "group": group, "format": fmt, "dtype": dtype, "bias": bias,
            "experts": experts, "skew": skew, "spare": spare}


def listed():
    """Weight shapes of TinyLlama-1.1B (2048, 5632), Llama-3-8B (4096, 14336, 128256) and, for the experts, generic ones."""
    return [
        # decoding one token of one sequence: the smallest projection, where the launch counts ...
        dict(_case("linear", 1, 2048, 2048, 128, "int4", "fp16"), name="token_2048x2048"),
        # ... and the up projection of a large layer, where reading the weight counts
        dict(_case("linear", 1, 14336, 4096, 128, "int4_asym", "bf16"), name="token_14336x4096_asym"),
        # a batch of sequences decoding together, small groups, the long contraction of a down projection
        dict(_case("linear", 16, 4096, 14336, 32, "int4", "fp16"), name="batch16_4096x14336_g32"),
        # a few draft tokens through the vocabulary's projection, a value table
        dict(_case("linear", 5, 128256, 4096, 64, "fp4", "bf16"), name="draft5_128256x4096_fp4"),
        # a short prompt of odd length, one scale per row, a bias
        dict(_case("linear", 77, 5632, 2048, 0, "flint4", "fp16", bias=True), name="prompt77_5632x2048_rows"),
        # a long prompt: bound by the matrix cores
        dict(_case("linear", 2000, 14336, 4096, 128, "int4", "bf16"), name="prompt2000_14336x4096"),
        # adapters trained on a frozen 4-bit weight: a micro-batch of 2048 tokens ...
        dict(_case("linear_train", 2048, 4096, 4096, 64, "int4_asym", "bf16"), name="train2048_4096x4096_asym"),
        # ... and a ragged one through a narrower layer, with the bias trained
        dict(_case("linear_train", 509, 2048, 5632, 128, "fp4", "fp16", bias=True), name="train509_2048x5632_fp4"),
        # decoding with many small experts: most of them get a row or two, some none
        dict(_case("experts", 96, 1024, 2048, 64, "int4_asym", "fp16", experts=64, skew=0.7), name="experts64_96x1024x2048"),
        # a prompt through few large experts, unevenly loaded, the row buffer longer than the rows in use
        dict(_case("experts", 4096, 14336, 4096, 128, "int4", "bf16", experts=8, skew=0.5, spare=40), name="experts8_4096x14336x4096"),
        # adapters trained on frozen experts: a small micro-batch ...
        dict(_case("experts_train", 250, 1024, 2048, 128, "int4", "fp16", bias=True, experts=8, skew=1.0), name="experts8_train250"),
        # ... and a large one over many experts
        dict(_case("experts_train", 4096, 2048, 2048, 64, "int4", "bf16", experts=32, skew=0.3), name="experts32_train4096"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["linear", "linear", "linear_train", "experts", "experts_train"])
        experts = _log_int(rng, 2, 64) if op.startswith("experts") else 1
        group = rng.choice([0, 32, 64, 128, 128, 256])
        n, k = _log_int(rng, 48, 16384), _log_int(rng, 64, 16384)
        if group:
            k = max(group, k // group * group)
        c = _case(op, _log_int(rng, 1, 4096), n, k, group, rng.choice(_FORMATS), rng.choice(["fp16", "bf16"]),
                  rng.random() < 0.4, experts, round(rng.uniform(0, 1.5), 2) if experts > 1 else 0.0,
                  rng.choice([0, 0, 1, 17, 100]) if experts > 1 else 0)
        if work(c)["flops"] <= _MOST_FLOPS and experts * n * k <= _MOST_WEIGHTS:
            return c


def _counts(case):
    """Rows of each expert, the busiest first; they add up to case["rows"]."""
    w = [(1.0 + e) ** -case["skew"] for e in range(case["experts"])]
    c = [int(case["rows"] * v / sum(w)) for v in w]
    for i in range(case["rows"] - sum(c)):
        c[i % len(c)] += 1
    return c


def work(case):
    m, n, k = case["rows"], case["n"], case["k"]
    g = case["group"] or k
    used = sum(c > 0 for c in _counts(case))
    params = 4 if "asym" in case["format"] else 2                      # float16 scale, and float16 zero point
    train = case["op"].endswith("_train")
    total = m + case["spare"]
    by = used * n * (k / 2 + k // g * params)                          # weights of the experts that have rows
    by += 2 * (m * k + total * n) * (2 if train else 1)                # x, y; dy, dx
    by += 2 * case["experts"] * n * (2 if train else 1) if case["bias"] else 0
    return {"bytes": by, "flops": 2.0 * m * n * k * (2 if train else 1)}


def _quantized(case, g, gen):
    """Codes, scales and zero points of a random weight [E, N, K], as the framework's quantizers return them."""
    e, n, k = case["experts"], case["n"], case["k"]
    w = torch.randn(e, n, k // g, g, generator=gen, device="cuda") * 0.02
    if case["format"] == "int4_asym":
        lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
        s = ((hi - lo) / 15).half()
        z = (-lo / s.float()).round_().clamp_(0, 15)
        q = w.div_(s.float()).round_().add_(z).clamp_(0, 15).to(torch.uint8)
        return q.view(e, n, k), s.view(e, n, k // g), z.half().view(e, n, k // g)
    table = _TABLES.get(case["format"])
    top = max(table) if table else 7
    s = (w.abs().amax(-1, keepdim=True) / top).half()
    w = w.div_(s.float())
    if not table:
        return w.round_().clamp_(-7, 7).to(torch.int8).view(e, n, k), s.view(e, n, k // g), None
    values = torch.tensor([-v for v in table[::-1]] + [0] + table, dtype=torch.float32, device="cuda")
    q = values.half()[torch.bucketize(w.view(e, n, k), (values[1:] + values[:-1]) / 2)]
    return q, s.view(e, n, k // g), None


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    m, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
    dt = _DTYPES[case["dtype"]]
    q, scale, zero = _quantized(case, case["group"] or k, gen)
    # activations with a few channels that stand out, as behind a norm
    x = torch.randn(m + case["spare"], k, generator=gen, device="cuda")
    x *= 1 + 9 * (torch.rand(k, generator=gen, device="cuda") < 0.01)
    order = torch.randperm(e, generator=torch.Generator().manual_seed(int(seed)))
    counts = torch.tensor(_counts(case))[order]
    return {"q": q, "scale": scale, "zero": zero, "x": x.to(dt), "counts": counts,
            "bias": torch.randn(e, n, generator=gen, device="cuda").to(dt) if case["bias"] else None,
            "dy": (torch.randn(m + case["spare"], n, generator=gen, device="cuda") * 0.01).to(dt)
            if case["op"].endswith("_train") else None}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["experts"], s["train"] = case["op"].startswith("experts"), case["op"].endswith("_train")
    s["split"] = s["counts"].tolist() + [case["spare"]]
    if not s["experts"]:
        s["q"], s["scale"] = s["q"][0], s["scale"][0]
        s["zero"] = None if s["zero"] is None else s["zero"][0]
        s["bias"] = None if s["bias"] is None else s["bias"][0]
    if own:
        from quantization_amd import packed
        s["calls"] = packed
        scale, zero = s.pop("scale"), s.pop("zero")
        if not case["group"]:   # one scale per row: without the groups' axis
            scale, zero = scale[..., 0], None if zero is None else zero[..., 0]
        s["weight"] = packed.pack_codes(s.pop("q"), scale, zero, wq_bits=4, datatype=case["format"],
                                        group_size=case["group"] or None)
        s["counts"] = s["counts"].to(device="cuda", dtype=torch.int32)
        s["leaves"] = [t.requires_grad_() for t in (s["x"], s["bias"]) if t is not None] if s["train"] else []
    return s


def _own(s):
    if s["experts"]:
        y = s["calls"].packed_expert_linear(s["x"], s["weight"], s["counts"], s["bias"])
    else:
        y = s["calls"].packed_linear(s["x"], s["weight"], s["bias"])
    if not s["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, s["leaves"], s["dy"])
    return dict(zip(("y", "dx", "db"), (y, *grads)))


def _weights(s):
    """The weights in float32: [N, K] or [E, N, K]."""
    q, scale = s["q"], s["scale"]
    w = q.float().view(*scale.shape, -1)
    if s["zero"] is not None:
        w = w - s["zero"].float().unsqueeze(-1)
    return (w * scale.float().unsqueeze(-1)).view(q.shape)


def _plain_linear(s):
    w, x = _weights(s), s["x"].float()
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out = {"y": y.to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float()
        out["dx"] = (dy @ w).to(s["x"].dtype)
        if s["bias"] is not None:
            out["db"] = dy.sum(0).to(s["x"].dtype)
    return out


def _plain_experts(s):
    w, bias, parts = _weights(s), s["bias"], s["x"].float().split(s["split"])
    y = [p @ v.t() for p, v in zip(parts, w)]
    if bias is not None:
        y = [p + b for p, b in zip(y, bias.float())]
    # rows behind the last expert's belong to nobody: zeros
    out = {"y": torch.cat(y + [w.new_zeros(s["split"][-1], w.shape[1])]).to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float().split(s["split"])
        dx = [p @ v for p, v in zip(dy, w)] + [w.new_zeros(s["split"][-1], w.shape[2])]
        out["dx"] = torch.cat(dx).to(s["x"].dtype)
        if bias is not None:
            out["db"] = torch.stack([p.sum(0) for p in dy[:-1]]).to(s["x"].dtype)
    return out


def run(state):
    if own:
        return _own(state)
    return _plain_experts(state) if state["experts"] else _plain_linear(state)


def exact(case, seed):
    """The definition in float64, expert by expert: every weight spelled out, every sum over the whole axis."""
    s = _inputs(case, seed)
    m, n, k, g = case["rows"] + case["spare"], case["n"], case["k"], case["group"] or case["k"]
    train = case["op"].endswith("_train")
    at = torch.arange(k, device="cuda") // g
    x = s["x"].double()
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    dx = torch.zeros(m, k, dtype=torch.float64, device="cuda")
    db = torch.zeros(case["experts"], n, dtype=torch.float64, device="cuda")
    first = 0
    for e, c in enumerate(s["counts"].tolist()):
        if c:
            w = s["q"][e].double()
            if s["zero"] is not None:
                w -= s["zero"][e].double()[:, at]
            w *= s["scale"][e].double()[:, at]
            y[first:first + c] = torch.mm(x[first:first + c], w.t())
            if s["bias"] is not None:
                y[first:first + c] += s["bias"][e].double()
            if train:
                d = s["dy"][first:first + c].double()
                dx[first:first + c] = torch.mm(d, w)
                db[e] = d.sum(0)
            first += c
    out = {"y": y}
    if train:
        out["dx"] = dx
        if case["bias"]:
            out["db"] = db if case["op"] == "experts_train" else db[0]
    return out
