"""What the int8 path of a decoder layer costs: its operators at the sizes that decode steps, serving batches and
prompts call them with, in a plain form (elementary torch operations) and through this package.

Four kinds of case, each one pass:

  product   int8_matmul: int8 tokens with a scale each, times int8 weights with a scale for each output channel.
  linear    a linear layer on float activations: optional RMS norm, quantize_tokens, int8_matmul.
  norms     residual_norms: a block's output normalised, gated and scaled, added to the residual stream, and the
            norm that the next block reads.
  mlp       the MLP block from end to end: RMS norm and quantisation, gate and up projections in one product,
            silu_mul_tokens, down projection, residual_norms.

Tokens are quantised as quantize(w, K, bits=8) quantises a row: scale = amax / 127 (1 for a row of zeros),
q = rint(x / scale).
"""
import math

import torch

own = False

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
LARGEST_FLOPS = 2.0 * 8192 * 14336 * 4096
LARGEST_VALUES = 8192 * 8192


def _product(m, k, n, out="f16", scales="f32", name=None):
    case = {"kind": "product", "m": m, "k": k, "n": n, "out": out, "scales": scales}
    return dict(case, name=name) if name else case


def _linear(m, k, n, x="f16", norm=True, scales="f32", name=None):
    # the output goes on in 16 bits, as everything between two quantised layers does
    case = {"kind": "linear", "m": m, "k": k, "n": n, "x": x, "out": "f16" if x == "f32" else x, "norm": norm, "scales": scales}
    return dict(case, name=name) if name else case


def _norms(rows, n, x="f16", post=True, gate=1, name=None):
    # gate: how many rows the gate has (0: no gate; 1: one value a channel; else each row of it serves rows / gate tokens)
    case = {"kind": "norms", "rows": rows, "n": n, "x": x, "post": post, "gate": gate}
    return dict(case, name=name) if name else case


def _mlp(m, hidden, inter, x="f16", name=None):
    case = {"kind": "mlp", "m": m, "hidden": hidden, "inter": inter, "x": x}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence, an attention projection of SmolLM2-1.7B: latency is all there is
        _product(1, 2048, 2048, name="product_decode_small"),
        # a full decode batch on the MLP up projection of a 70B-class model: the stream of the weights
        _product(16, 8192, 28672, scales="f16", name="product_batch16_70b"),
        # no round size at all, K no multiple of 16 bytes, the output kept in float32
        _product(333, 4104, 5003, out="f32", name="product_ragged"),
        # a short prompt through the MLP up projection of an 8B-class model
        _product(512, 4096, 14336, out="bf16", name="product_prompt_512"),
        # the longest prompt: the largest case
        _product(8192, 14336, 4096, out="bf16", name="product_prompt_8192"),
        # one token from the residual stream to the vocabulary of SmolLM2-135M: final norm and lm_head
        _linear(1, 576, 49152, name="linear_decode_head"),
        # a prompt's attention output through the o projection of an 8B-class model
        _linear(2048, 4096, 4096, x="bf16", norm=False, name="linear_prompt_2048"),
        # one token of SmolLM2-135M after a block
        _norms(1, 576, name="norms_decode"),
        # a long prompt of a model that is 8192 wide, one gate value a channel: the largest
        _norms(8192, 8192, x="bf16", name="norms_prompt_8192"),
        # four sequences of 300 tokens with a gate of their own each, odd width, float32
        _norms(1200, 1537, x="f32", gate=4, name="norms_gate_by_sequence"),
        # a decode batch through the MLP of an 8B-class model
        _mlp(8, 4096, 14336, name="mlp_batch_8"),
        # a prompt of no round length through the MLP of SmolLM2-1.7B
        _mlp(1000, 2048, 8192, x="bf16", name="mlp_prompt_1000"),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    what = rng.choices(("product", "linear", "norms", "mlp"), (5, 2, 4, 1))[0]
    if what in ("product", "linear"):
        step = rng.choice((1, 16, 64, 128))
        m, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 14336, step)
        n = _log_int(rng, 64, min(49152, 8192 * 28672 // k))
        while 2.0 * m * k * n > LARGEST_FLOPS:
            m //= 2
        scales = rng.choice(("f32", "f32", "f16"))
        if what == "product":
            return _product(m, k, n, out=rng.choice(("f16", "bf16", "f32")), scales=scales)
        return _linear(m, k, n, x=rng.choice(("f16", "bf16", "f32")), norm=rng.random() < 0.5, scales=scales)
    if what == "norms":
        rows, n = _log_int(rng, 1, 8192), _log_int(rng, 64, 14336, rng.choice((1, 8, 64)))
        while rows * n > LARGEST_VALUES // 2:
            rows //= 2
        divisors = [d for d in range(1, min(rows, 64) + 1) if rows % d == 0]
        return _norms(rows, n, x=rng.choice(("f16", "bf16", "f32")), post=rng.random() < 0.7,
                      gate=rng.choice((0, 1, rng.choice(divisors), rows)))
    hidden = _log_int(rng, 576, 4096, 64)
    return _mlp(_log_int(rng, 1, 2048), hidden, _log_int(rng, 2.5 * hidden, 3.5 * hidden, 64), x=rng.choice(("f16", "bf16")))


# ------------------------------------------------------------------------------------------ inputs
def _weights(gen, n, k, scales):
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=gen)
    s = torch.rand(n, 1, device="cuda", generator=gen).mul_(0.5).add_(0.5).mul_(1.0 / (73.0 * math.sqrt(k)))
    return w, s.to(KINDS[scales])          # products of unit variance with tokens of unit variance


def _activations(gen, rows, n, kind):
    """The residual stream: N(0, 1) with a few channels that are ten times as large."""
    x = torch.randn(rows, n, device="cuda", generator=gen)
    x[:, torch.randint(0, n, (max(1, n // 500),), device="cuda", generator=gen)] *= 10.0
    return x.to(KINDS[kind])


def _norm_weight(gen, n, kind):
    return (1.0 + 0.1 * torch.randn(n, device="cuda", generator=gen)).to(KINDS[kind])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "product":
        s["w"], s["ws"] = _weights(gen, case["n"], case["k"], case["scales"])
        s["q"] = torch.randn(case["m"], case["k"], device="cuda", generator=gen).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
        s["qs"] = torch.rand(case["m"], device="cuda", generator=gen).mul_(0.02).add_(0.02)
    elif case["kind"] == "linear":
        s["w"], s["ws"] = _weights(gen, case["n"], case["k"], case["scales"])
        s["input"] = _activations(gen, case["m"], case["k"], case["x"])
        s["weight"] = _norm_weight(gen, case["k"], case["x"]) if case["norm"] else None
    elif case["kind"] == "norms":
        rows, n, kind = case["rows"], case["n"], case["x"]
        s["hidden"] = _activations(gen, rows, n, kind)
        s["delta"] = torch.randn(rows, n, device="cuda", generator=gen).mul_(3.0).to(KINDS[kind])
        s["post_weight"] = _norm_weight(gen, n, kind) if case["post"] else None
        s["gate_values"] = torch.randn(case["gate"], n, device="cuda", generator=gen).mul_(0.5).to(KINDS[kind]) if case["gate"] else None
        s["weight"] = _norm_weight(gen, n, kind)
        s["hidden_out"] = torch.empty_like(s["hidden"])
    else:
        hidden, inter, kind = case["hidden"], case["inter"], case["x"]
        s["input"] = _activations(gen, case["m"], hidden, kind)
        s["hidden_out"] = torch.empty_like(s["input"])
        s["w1"], s["s1"] = _weights(gen, 2 * inter, hidden, "f32")
        s["w2"], s["s2"] = _weights(gen, hidden, inter, "f32")
        for name in ("in_weight", "post_weight", "weight"):
            s[name] = _norm_weight(gen, hidden, kind)
    return s


# ------------------------------------------------------------------------------------------ the plain form
def _norm(v, weight):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * weight.float()


def _quantized(v):
    amax = v.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), torch.ones_like(amax))
    return torch.round(v / scale), scale


def _int8_product(q, scale, w, ws):
    """Sums of products of whole numbers pass 2^24: in 64 bits."""
    acc = (q.double() @ w.double().t()).float()
    return acc * scale.reshape(-1, 1).float() * ws.reshape(1, -1).float()


def _residual(hidden, delta, post_weight, gate, scale, weight, kind):
    y = delta if post_weight is None else _norm(delta, post_weight)
    if gate is not None:
        y = y * gate.float().repeat_interleave(hidden.shape[0] // gate.shape[0], dim=0)
    hidden = (hidden.float() + scale * y).to(KINDS[kind])      # as it is stored, and read by the norm
    return hidden, _norm(hidden.float(), weight).to(KINDS[kind])


def _plain(s):
    if s["kind"] == "product":
        return _int8_product(s["q"], s["qs"], s["w"], s["ws"]).to(KINDS[s["out"]])
    if s["kind"] == "linear":
        x = s["input"].float()
        q, scale = _quantized(_norm(x, s["weight"]) if s["norm"] else x)
        return _int8_product(q, scale, s["w"], s["ws"]).to(KINDS[s["out"]])
    if s["kind"] == "norms":
        return _residual(s["hidden"], s["delta"].float(), s["post_weight"], s["gate_values"], 0.5, s["weight"], s["x"])
    inter = s["inter"]
    gate_up = _int8_product(*_quantized(_norm(s["input"].float(), s["in_weight"])), s["w1"], s["s1"])
    g, u = gate_up[:, :inter], gate_up[:, inter:]
    down = _int8_product(*_quantized(g * torch.sigmoid(g) * u), s["w2"], s["s2"])
    return _residual(s["input"], down, s["post_weight"], None, 0.5, s["weight"], s["x"])


# ------------------------------------------------------------------------------------------ the package's calls
def _own(s):
    import locomp_b200 as L
    if s["kind"] == "product":
        return L.int8_matmul(s["q"], s["qs"], s["w"], s["ws"], out_dtype=s["out"])
    if s["kind"] == "linear":
        t = L.quantize_tokens(s["input"], s["weight"], EPS)
        return L.int8_matmul(t.q, t.scales, s["w"], s["ws"], out_dtype=s["out"])
    if s["kind"] == "norms":
        normed = L.residual_norms(s["hidden"], s["delta"], s["weight"], EPS, post_weight=s["post_weight"], gate=s["gate_values"],
                                  scale=0.5, hidden_out=s["hidden_out"])
        return s["hidden_out"], normed
    t = L.quantize_tokens(s["input"], s["in_weight"], EPS)
    gate_up = L.int8_matmul(t.q, t.scales, s["w1"], s["s1"], out_dtype="f32")      # to be quantised next: 16 bits would move q by a step here and there
    t = L.silu_mul_tokens(gate_up[:, :s["inter"]], gate_up[:, s["inter"]:])
    down = L.int8_matmul(t.q, t.scales, s["w2"], s["s2"], out_dtype="f32")         # to be normalised and added: rounded once, as the stream is stored
    normed = L.residual_norms(s["input"], down, s["weight"], EPS, post_weight=s["post_weight"], scale=0.5, hidden_out=s["hidden_out"])
    return s["hidden_out"], normed


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_norm(v, weight):
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.double()


def _exact_product(v, w, ws):
    """Tokens in 64 bits, quantised and multiplied by the weights as the values that they stand for."""
    amax = v.abs().amax(-1, keepdim=True)
    step = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    return torch.matmul((v / step).round() * step, (w.double() * ws.double().reshape(-1, 1)).t())


def _exact_residual(hidden, y, post_weight, gate, weight, kind):
    if post_weight is not None:
        y = _exact_norm(y, post_weight)
    if gate is not None:
        y = (y.reshape(gate.shape[0], -1, y.shape[1]) * gate.double().unsqueeze(1)).reshape(y.shape)
    hidden = hidden.double() + 0.5 * y
    return hidden, _exact_norm(hidden.to(KINDS[kind]).double(), weight)      # the norm reads the stream as it is stored


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        x = s["q"].double() * s["qs"].double().unsqueeze(1)
        return torch.matmul(x, (s["w"].double() * s["ws"].double().reshape(-1, 1)).t())
    if case["kind"] == "linear":
        x = s["input"].double()
        return _exact_product(_exact_norm(x, s["weight"]) if case["norm"] else x, s["w"], s["ws"])
    if case["kind"] == "norms":
        return _exact_residual(s["hidden"], s["delta"].double(), s["post_weight"], s["gate_values"], s["weight"], case["x"])
    gate_up = _exact_product(_exact_norm(s["input"].double(), s["in_weight"]), s["w1"], s["s1"])
    g, u = gate_up.split(case["inter"], dim=1)
    down = _exact_product(g / (1 + torch.exp(-g)) * u, s["w2"], s["s2"])
    return _exact_residual(s["input"], down, s["post_weight"], None, s["weight"], case["x"])


def work(case):
    """Each input read once, each output written once."""
    if case["kind"] in ("product", "linear"):
        m, k, n = case["m"], case["k"], case["n"]
        weights = n * k + n * BYTES[case["scales"]]
        if case["kind"] == "product":
            return {"bytes": weights + m * k + 4 * m + m * n * BYTES[case["out"]], "flops": 2.0 * m * n * k}
        size = BYTES[case["x"]]
        return {"bytes": weights + (m * k + (k if case["norm"] else 0)) * size + m * n * BYTES[case["out"]], "flops": 2.0 * m * n * k}
    if case["kind"] == "norms":
        rows, n = case["rows"], case["n"]
        return {"bytes": (4 * rows * n + (1 + case["post"] + case["gate"]) * n) * BYTES[case["x"]], "flops": 12.0 * rows * n}
    m, hidden, inter = case["m"], case["hidden"], case["inter"]
    return {"bytes": 3 * hidden * inter + 4 * (2 * inter + hidden) + (3 * m * hidden + 3 * hidden) * BYTES[case["x"]],
            "flops": 6.0 * m * hidden * inter}
