"""Cases and plain forms of the operators at the output end of a network and of its 4-bit layers.

Four operators: log probabilities of given tokens with entropy and top alternatives
(gonngpu_token_logprobs), distillation from a teacher's top logits (gonngpu_distill_forward,
_backward, _step), microscaled 4-bit quantisation (gonngpu_mxfp4_quantize, _dequantize) and the
linear layer on 4-bit operands (gonngpu_mxfp4_linear).

With `own` false, run() computes them in elementary torch operations in 32 bits; with `own` true it
makes the library's calls.  exact() is the definition again in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BLOCK = 32       # elements that share a scale
ACT_NONE, ACT_RELU = -1, 0
NEG_INF = float("-inf")


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # scoring the classes of the MLP configuration (batch 512, 10 outputs): the smallest call, latency only
        dict(name="logprobs_classes", op="logprobs", rows=512, vocab=10, given=1, top=3, masked=False),
        # one serving step of a small batch over a large vocabulary, 20 alternatives for the client;
        # some tokens are ruled out by a grammar
        dict(name="logprobs_step", op="logprobs", rows=4, vocab=128000, given=1, top=20, masked=True),
        # log probabilities of a prompt's own tokens, odd vocabulary
        dict(name="logprobs_prompt", op="logprobs", rows=1021, vocab=50001, given=1, top=5, masked=False),
        # a teacher's pass over a training batch: its top alternatives are kept for the student
        dict(name="logprobs_teacher", op="logprobs", rows=2048, vocab=64000, given=0, top=64, masked=False),
        # validation loss of a student, soft targets alone
        dict(name="distill_forward", op="distill_forward", rows=1000, vocab=32001, top=32, temperature=2.0,
             soft=1.0, masked=False),
        # gradient of the same loss mixed with the hard labels, from saved statistics
        dict(name="distill_backward", op="distill_backward", rows=2048, vocab=32000, top=16, temperature=2.0,
             soft=0.5, masked=True),
        # loss and gradient of a training step in one call, large vocabulary: the largest state
        dict(name="distill_step", op="distill_step", rows=4096, vocab=128000, top=64, temperature=1.0, soft=0.75,
             masked=False),
        # activations of a short prompt on their way into a 4-bit layer
        dict(name="quantize_rows", op="quantize", rows=333, cols=4096, transposed=False),
        # a layer's weights [in, out], quantised along `in` (across the rows of the stored matrix)
        dict(name="quantize_weights", op="quantize", rows=4096, cols=16384, transposed=True),
        # a single token through a layer: the weights' bytes are the cost
        dict(name="linear_token", op="linear", batch=1, inputs=4096, outputs=16384, bias=True, act=ACT_NONE),
        # the first hidden layer of the MLP configuration (inputs not a multiple of the block), ReLU
        dict(name="linear_mlp", op="linear", batch=512, inputs=784, outputs=1024, bias=True, act=ACT_RELU),
        # the square product of the fp16 configuration, in 4 bits
        dict(name="linear_square", op="linear", batch=8192, inputs=8192, outputs=8192, bias=False, act=ACT_NONE),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "distill_forward", "distill_backward", "distill_step", "quantize",
                     "linear", "linear"])
    if op == "quantize":
        rows = _spread(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=_spread(rng, 1, min(16384, (1 << 26) // rows)),
                    transposed=rng.random() < 0.5)
    if op == "linear":
        batch = _spread(rng, 1, 8192)
        inputs = _spread(rng, 16, 16384)
        most = max(8, min(16384, (1 << 38) // (batch * inputs)))
        return dict(op=op, batch=batch, inputs=inputs, outputs=_spread(rng, 8, most), bias=rng.random() < 0.5,
                    act=rng.choice([ACT_NONE, ACT_RELU]))
    vocab = _spread(rng, 2, 200000)
    rows = _spread(rng, 1, max(1, min(8192, (1 << 27) // vocab)))
    masked = rng.random() < 0.5
    if op == "logprobs":
        return dict(op=op, rows=rows, vocab=vocab, given=rng.choice([0, 1, 1, 3]), top=rng.randint(1, min(vocab, 64)),
                    masked=masked)
    return dict(op=op, rows=rows, vocab=vocab, top=rng.randint(1, min(vocab, 64)),
                temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), soft=rng.choice([0.0, 0.5, 0.9, 1.0]), masked=masked)


# ---------------------------------------------------------------------------------- inputs
def _logits(case, gen):
    """Logits with a normal body and a few strong tokens a row, as a trained network gives; with `masked`
    about a tenth of the vocabulary is ruled out (-inf)."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device=DEVICE)
    x.mul_(2.0)
    strong = torch.randint(0, vocab, (rows, 4), generator=gen, device=DEVICE)
    x.scatter_(1, strong, 8.0 + 3.0 * torch.randn(rows, 4, generator=gen, device=DEVICE))
    if case["masked"]:
        out = torch.rand(vocab, generator=gen, device=DEVICE) < 0.1
        out[0] = False
        x.masked_fill_(out, NEG_INF)
    return x


def _teacher(case, logits, gen):
    """`top` different tokens a row with a teacher's logits; a tenth of the rows give fewer (token -1), one
    row in twenty has no label (-1).  Labels and teacher tokens are never ruled out for the student."""
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    wide = vocab // top
    first = torch.arange(top, device=DEVICE) * wide
    tokens = first + torch.randint(0, wide, (rows, top), generator=gen, device=DEVICE)
    teacher = 2.0 + 2.0 * torch.randn(rows, top, generator=gen, device=DEVICE)
    agree = 0.8 * teacher + torch.randn(rows, top, generator=gen, device=DEVICE)
    logits.scatter_(1, tokens, agree)
    labels = tokens[:, 0].clone()
    labels[torch.rand(rows, generator=gen, device=DEVICE) < 0.05] = -1
    short = torch.rand(rows, 1, generator=gen, device=DEVICE) < 0.1
    late = torch.arange(top, device=DEVICE) >= (top + 1) // 2
    tokens = tokens.masked_fill(short & late, -1)
    return tokens.to(torch.int32), teacher, labels.to(torch.int32)


def _pow2(e):
    """2 ** e as float32 for whole e in [-126, 127], from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(v):
    """[rows, cols] -> [rows, blocks, 32], the last block filled up with zeros."""
    rows, cols = v.shape
    n = -(-cols // BLOCK)
    if n * BLOCK != cols:
        v = torch.nn.functional.pad(v, (0, n * BLOCK - cols))
    return v.reshape(rows, n, BLOCK)


def _quantize(v):
    """Codes (0..15, sign in bit 3) and exponents of blocks of 32 along the last dimension."""
    b = _blocks(v)
    largest = b.abs().amax(dim=-1)
    _, up = torch.frexp(largest)                       # largest = f 2**up with f in [0.5, 1)
    e = torch.where(largest > 0, up - 3, -127).clamp(-127, 125)
    a = b * _pow2(-e)[..., None]
    mag = a.abs()
    code = ((mag > 0.25).to(torch.uint8) + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75) + (mag > 2.5) + (mag >= 3.5)
            + (mag > 5.0))
    return code + 8 * torch.signbit(a).to(torch.uint8), e


def _values(code, e):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=code.device)
    half = torch.div(e, 2, rounding_mode="floor")
    return table[code.int()] * _pow2(half)[..., None] * _pow2(e - half)[..., None]


def _packed_bytes(rows, cols):
    n = -(-cols // BLOCK)
    codes = -(-rows * n * 16 // 512) * 512
    return codes, codes + -(-rows // 128) * -(-n // 4) * 512


def _pack(code, e, rows, cols):
    """The library's packed layout: two codes a byte (the even one low), then one byte a scale in tiles of
    128 rows x 4 blocks, padded with zeros."""
    n = -(-cols // BLOCK)
    at, size = _packed_bytes(rows, cols)
    out = torch.zeros(size, dtype=torch.uint8, device=code.device)
    pairs = code.reshape(rows, n * 16, 2)
    out[:rows * n * 16] = (pairs[..., 0] | (pairs[..., 1] << 4)).reshape(-1)
    tall, wide = -(-rows // 128), -(-n // 4)
    s = torch.zeros(tall * 128, wide * 4, dtype=torch.uint8, device=code.device)
    s[:rows, :n] = (e + 127).to(torch.uint8)
    out[at:] = s.reshape(tall, 4, 32, wide, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return out


def _unpack(packed, rows, cols):
    n = -(-cols // BLOCK)
    at, _ = _packed_bytes(rows, cols)
    byte = packed[:rows * n * 16].reshape(rows, n, 16, 1)
    code = torch.cat([byte & 15, byte >> 4], dim=-1).reshape(rows, n, BLOCK)
    tall, wide = -(-rows // 128), -(-n // 4)
    s = packed[at:].reshape(tall, wide, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tall * 128, wide * 4)
    return code, s[:rows, :n].int() - 127


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    s = {"case": dict(case)}
    op = case["op"]
    if op == "quantize":
        # activations and weights: a normal body, and some channels that are much larger
        s["x"] = torch.randn(case["rows"], case["cols"], generator=gen, device=DEVICE)
        s["x"][:, torch.rand(case["cols"], generator=gen, device=DEVICE) < 0.01] *= 20.0
        r, c = (case["cols"], case["rows"]) if case["transposed"] else (case["rows"], case["cols"])
        s["packed"] = torch.empty(_packed_bytes(r, c)[1], dtype=torch.uint8, device=DEVICE)
        s["values"] = torch.empty(r, c, device=DEVICE)
        return s
    if op == "linear":
        m, k, n = case["batch"], case["inputs"], case["outputs"]
        s["x"] = torch.randn(m, k, generator=gen, device=DEVICE)
        s["x"][:, torch.rand(k, generator=gen, device=DEVICE) < 0.01] *= 20.0
        w = torch.randn(n, k, generator=gen, device=DEVICE) / math.sqrt(k)
        s["weights"] = _pack(*_quantize(w), n, k)      # quantised once, kept with the model
        s["bias"] = torch.randn(n, generator=gen, device=DEVICE) if case["bias"] else None
        s["y"] = torch.empty(m, n, device=DEVICE)
        return s
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    s["logits"] = _logits(case, gen)
    if op == "logprobs":
        given = case["given"]
        s["tokens"] = torch.randint(0, vocab, (rows, given), generator=gen, device=DEVICE, dtype=torch.int32)
        s["logprobs"] = torch.empty(rows, given, device=DEVICE)
        s["entropy"] = torch.empty(rows, device=DEVICE)
        s["top_tokens"] = torch.empty(rows, top, dtype=torch.int32, device=DEVICE)
        s["top_logprobs"] = torch.empty(rows, top, device=DEVICE)
        return s
    s["teacher_tokens"], s["teacher_logits"], s["labels"] = _teacher(case, s["logits"], gen)
    s["loss"] = torch.empty(rows, device=DEVICE)
    s["stats"] = torch.empty(rows, 3, device=DEVICE)
    if op != "distill_forward":
        s["grad"] = torch.empty(rows, vocab, device=DEVICE)
    if op == "distill_backward":
        s["grad_loss"] = torch.rand(rows, generator=gen, device=DEVICE) + 0.5
        x = s["logits"]                                # statistics that the forward pass left
        largest = x.amax(dim=1, keepdim=True)
        s["stats"][:, :1] = largest
        s["stats"][:, 1] = ((x - largest) / case["temperature"]).exp_().sum(dim=1)
        s["stats"][:, 2] = (x - largest).exp_().sum(dim=1)
    return s


# ---------------------------------------------------------------------------------- plain forms
def _ordered(x, vocab):
    """Whole-number keys that order like (value, lowest index first): unique within a row."""
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    return (bits << 32) | (vocab - 1 - torch.arange(vocab, device=x.device))


def _plain_logprobs(s):
    c, x = s["case"], s["logits"]
    largest = x.amax(dim=1, keepdim=True)
    d = x - largest
    e = d.exp()
    total = e.sum(dim=1, keepdim=True)
    log_total = total.log()
    weighted = (e * d.clamp(min=-1e30)).sum(dim=1)
    key = _ordered(x, c["vocab"]).topk(c["top"], dim=1, sorted=True).values
    best = c["vocab"] - 1 - (key & 0xFFFFFFFF)
    return {"logprobs": d.gather(1, s["tokens"].long()) - log_total,
            "entropy": log_total[:, 0] - weighted / total[:, 0],
            "top_tokens": best.to(torch.int32),
            "top_logprobs": d.gather(1, best) - log_total}


def _plain_targets(s, dtype=torch.float32):
    """The teacher's distribution over its tokens, which of them are there, and which rows have a label."""
    c = s["case"]
    there = s["teacher_tokens"] >= 0
    z = (s["teacher_logits"].to(dtype) / c["temperature"]).masked_fill(~there, NEG_INF)
    z = z - z.amax(dim=1, keepdim=True)
    q = z.exp()
    total = q.sum(dim=1, keepdim=True)
    return q / total, z - total.log(), there, s["teacher_tokens"].clamp(min=0).long(), s["labels"] >= 0


def _plain_forward(s):
    c, x = s["case"], s["logits"]
    t, w = c["temperature"], c["soft"]
    largest = x.amax(dim=1, keepdim=True)
    d = x - largest
    total = (d / t).exp().sum(dim=1, keepdim=True)
    total1 = d.exp().sum(dim=1, keepdim=True)
    q, log_q, there, tokens, labelled = _plain_targets(s)
    far = torch.where(there, q * (log_q - (d.gather(1, tokens) / t - total.log())), 0.0).sum(dim=1)
    hard = total1.log()[:, 0] - d.gather(1, s["labels"].clamp(min=0).long()[:, None])[:, 0]
    loss = (w * t * t) * far + (1.0 - w) * torch.where(labelled, hard, 0.0)
    return loss, torch.cat([largest, total, total1], dim=1)


def _plain_backward(s, stats, scale):
    c, x = s["case"], s["logits"]
    t, w = c["temperature"], c["soft"]
    largest, total, total1 = stats[:, :1], stats[:, 1:2], stats[:, 2:]
    q, _, there, tokens, labelled = _plain_targets(s)
    soft = scale * (w * t)
    hard = torch.where(labelled, scale[:, 0] * (1.0 - w), 0.0)[:, None]
    d = x - largest
    grad = (d / t).exp() * (soft / total)
    grad += d.exp_() * (hard / total1)
    grad.scatter_add_(1, tokens, torch.where(there, -soft * q, 0.0))
    grad.scatter_add_(1, s["labels"].clamp(min=0).long()[:, None], -hard)
    return grad


def _step_scale(case):
    return 1.0 / case["rows"]                          # the mean over the rows


def _activate(y, act):
    return y.clamp(min=0.0) if act == ACT_RELU else y


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "logprobs":
        return _plain_logprobs(s)
    if op == "distill_forward":
        loss, stats = _plain_forward(s)
        return {"loss": loss, "stats": stats}
    if op == "distill_backward":
        return {"grad": _plain_backward(s, s["stats"], s["grad_loss"][:, None])}
    if op == "distill_step":
        loss, stats = _plain_forward(s)
        scale = torch.full_like(stats[:, :1], _step_scale(c))
        return {"loss": loss, "grad": _plain_backward(s, stats, scale)}
    if op == "quantize":
        x = s["x"].t() if c["transposed"] else s["x"]
        rows, cols = x.shape
        return {"values": _values(*_quantize(x)).reshape(rows, -1)[:, :cols].contiguous()}
    m, k, n = c["batch"], c["inputs"], c["outputs"]
    w = _values(*_unpack(s["weights"], n, k)).reshape(n, -1)
    x = _values(*_quantize(s["x"])).reshape(m, -1)
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"]
    return {"y": _activate(y, c["act"])}


# ---------------------------------------------------------------------------------- the library's calls
_library = None


def _binding():
    global _library
    if _library is None:
        here = os.path.join(os.getcwd(), "go-nngpu_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import gonngpu
        gonngpu.lib().gonngpu_set_device(torch.cuda.current_device())
        gonngpu.lib().gonngpu_set_blocking(0)          # a pipelined caller: calls only enqueue
        _library = gonngpu
    return _library


def _own(s):
    g = _binding()
    c = s["case"]
    op = c["op"]
    if "handles" not in s:                             # a program wraps its tensors once
        s["handles"] = {k: g.Buffer.wrap(v.data_ptr(), v.numel() * v.element_size(), v)
                        for k, v in s.items() if isinstance(v, torch.Tensor) and v.numel()}
    h = s["handles"]
    if op == "logprobs":
        g.token_logprobs(h["logits"], c["rows"], c["vocab"], tokens=h.get("tokens"), n_tokens=c["given"],
                         logprobs=h.get("logprobs"), entropy=h["entropy"], top_n=c["top"],
                         top_tokens=h["top_tokens"], top_logprobs=h["top_logprobs"])
        return {k: s[k] for k in ("logprobs", "entropy", "top_tokens", "top_logprobs")}
    if op == "quantize":
        r, n = (c["cols"], c["rows"]) if c["transposed"] else (c["rows"], c["cols"])
        g.mxfp4_quantize(h["x"], c["rows"], c["cols"], c["transposed"], h["packed"])
        g.mxfp4_dequantize(h["packed"], r, n, h["values"])
        return {"values": s["values"]}
    if op == "linear":
        g.mxfp4_linear(h["x"], c["batch"], c["inputs"], h["weights"], c["outputs"], h.get("bias"), c["act"], 0.0,
                       h["y"])
        return {"y": s["y"]}
    args = (h["logits"], c["rows"], c["vocab"], h["teacher_tokens"], h["teacher_logits"], c["top"], h["labels"],
            c["temperature"], c["soft"])
    if op == "distill_forward":
        g.distill_forward(*args, loss=h["loss"], stats=h["stats"])
        return {"loss": s["loss"], "stats": s["stats"]}
    if op == "distill_backward":
        g.distill_backward(*args, stats=h["stats"], grad_loss=h["grad_loss"], grad_scale=1.0, grad=h["grad"])
        return {"grad": s["grad"]}
    g.distill_step(*args, grad_loss=None, grad_scale=_step_scale(c), loss=h["loss"], grad=h["grad"])
    return {"loss": s["loss"], "grad": s["grad"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n + 17 * n / 32, "flops": 4 * n}
    if op == "linear":
        m, k, n = case["batch"], case["inputs"], case["outputs"]
        return {"bytes": 4 * m * k + 17 * n * k / 32 + 4 * m * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    cells = rows * vocab
    if op == "logprobs":
        return {"bytes": 4 * cells + rows * (8 * case["given"] + 4 + 8 * top), "flops": 5 * cells}
    small = rows * (8 * top + 8)
    if op == "distill_forward":
        return {"bytes": 4 * cells + small + 12 * rows, "flops": 5 * cells}
    return {"bytes": 8 * cells + small + 12 * rows, "flops": (8 if op == "distill_step" else 5) * cells}


# ---------------------------------------------------------------------------------- 64 bits
def _exact_values(x):
    """What the 4-bit codes stand for, by rounding to the step of each value's binade."""
    rows, cols = x.shape
    b = _blocks(x.double())
    largest = b.abs().amax(dim=-1, keepdim=True)
    e = torch.where(largest > 0, largest.log2().floor(), -125.0)
    e = torch.where(torch.exp2(e) > largest, e - 1, torch.where(torch.exp2(e + 1) <= largest, e + 1, e))
    e = (e - 2).clamp(-127, 125)
    a = b / torch.exp2(e)
    step = torch.exp2(a.abs().clamp(min=1.0).log2().floor().clamp(max=2.0) - 1)
    return ((a / step).round() * step).clamp(-6, 6).mul_(torch.exp2(e)).reshape(rows, -1)[:, :cols]


def _exact_logprobs(s):
    c, x = s["case"], s["logits"].double()
    lse = torch.logsumexp(x, dim=1, keepdim=True)
    logp = x - lse
    best = x.topk(c["top"], dim=1, sorted=True).values
    return {"logprobs": logp.gather(1, s["tokens"].long()),
            "entropy": -torch.special.xlogy(logp.exp(), logp.exp()).sum(dim=1),
            "top_tokens": None, "top_logprobs": best - lse}


def _exact_distill(s):
    c, x = s["case"], s["logits"].double()
    t, w = c["temperature"], c["soft"]
    there = s["teacher_tokens"] >= 0
    q = torch.softmax((s["teacher_logits"].double() / t).masked_fill(~there, NEG_INF), dim=1)
    tokens = s["teacher_tokens"].clamp(min=0).long()
    labelled = (s["labels"] >= 0).double()[:, None]
    label = s["labels"].clamp(min=0).long()[:, None]
    lse_t = torch.logsumexp(x / t, dim=1, keepdim=True)
    lse = torch.logsumexp(x, dim=1, keepdim=True)
    log_p = x.gather(1, tokens) / t - lse_t
    far = torch.where(there, torch.special.xlogy(q, q) - q * log_p, 0.0).sum(dim=1)
    loss = w * t * t * far + (1 - w) * (labelled * (lse - x.gather(1, label)))[:, 0]
    out = {"loss": loss}
    if c["op"] == "distill_forward":
        largest = x.amax(dim=1, keepdim=True)
        out["stats"] = torch.cat([largest, (lse_t - largest / t).exp(), (lse - largest).exp()], dim=1)
        return out
    grad = (x / t - lse_t).exp_().mul_(w * t)
    grad.scatter_add_(1, tokens, torch.where(there, -w * t * q, 0.0))
    if w < 1:
        grad += (x - lse).exp_().mul_((1 - w) * labelled)
        grad.scatter_add_(1, label, -(1 - w) * labelled)
    if c["op"] == "distill_backward":
        return {"grad": grad * s["grad_loss"].double()[:, None]}
    out["grad"] = grad * _step_scale(c)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        return _exact_logprobs(s)
    if op == "quantize":
        return {"values": _exact_values(s["x"].t() if case["transposed"] else s["x"]).contiguous()}
    if op == "linear":
        m, k, n = case["batch"], case["inputs"], case["outputs"]
        code, e = _unpack(s["weights"], n, k)
        low = (code & 7).double()
        size = torch.where(low < 2, low / 2, (1 + 0.5 * (low % 2)) * torch.exp2(torch.floor(low / 2) - 1))
        w = (torch.where(code >= 8, -size, size) * torch.exp2(e.double())[..., None]).reshape(n, -1)[:, :k]
        y = _exact_values(s["x"]) @ w.t()
        if s["bias"] is not None:
            y += s["bias"].double()
        return {"y": _activate(y, case["act"])}
    return _exact_distill(s)
