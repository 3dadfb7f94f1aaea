"""Cases of the dropout, layer-norm and scaled-embedding operators of a pre-norm training step.

Every case is one call: ``layernorm`` (forward, backward), ``dropout`` (forward with an optional residual, backward),
``dropout_add_layernorm`` (forward, backward) and ``embedding`` (scaled lookup with dropout, and its gradient). ``run``
computes it with elementary torch operations, or through ``cgpt_b200.ops`` where ``own`` is set; ``exact`` computes it in 64 bits.

Dropout masks: element ``e`` of a tensor (row-major index) is decided by 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
"Parallel random numbers: as easy as 1, 2, 3", 2011) with key = seed (low, high word) and counter = (e // 8, site, step low,
step high): of the four words, word ``(e % 8) // 2``, its low half for even ``e`` and its high half for odd. The element is kept
where those bits are >= round(p * 65536) and then multiplied by 65536 / (65536 - round(p * 65536)). ``state`` holds (seed, step).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPSILON = 1e-5
SITE = 3          # which dropout of the step the call is


def listed():
    return [
        # one micro-batch of the tiny configuration: latency decides
        dict(name="layernorm fwd f16 tiny", op="layernorm", backward=False, dtype="f16", rows=64, hidden=256),
        # the 104m training step: 32 x 1024 tokens
        dict(name="layernorm fwd bf16 104m", op="layernorm", backward=False, dtype="bf16", rows=32768, hidden=1024),
        # the 1.3B configuration, half a step's tokens, with the residual branch's gradient added in the same pass
        dict(name="layernorm bwd bf16 1.3b", op="layernorm", backward=True, dtype="bf16", rows=16384, hidden=2048, residual=True),
        # rows that no vector load fits, fp32 parity runs
        dict(name="layernorm bwd f32 odd", op="layernorm", backward=True, dtype="f32", rows=4099, hidden=1001, residual=False),
        # a branch's output dropped and added to the residual stream, 1.3B width: the largest case
        dict(name="dropout fwd bf16 1.3b", op="dropout", backward=False, dtype="bf16", rows=32768, hidden=2048, residual=True, p=0.1),
        # gradient of a small, ragged activation
        dict(name="dropout bwd f32 ragged", op="dropout", backward=True, dtype="f32", rows=1, hidden=1000003, residual=False, p=0.25),
        # sub-layer boundary of the 104m step, forward and backward
        dict(name="dropout add norm fwd 104m", op="dropout_add_layernorm", backward=False, dtype="f16", rows=32768, hidden=1024, p=0.1),
        dict(name="dropout add norm bwd 104m", op="dropout_add_layernorm", backward=True, dtype="f16", rows=32768, hidden=1024, p=0.1),
        # the same at the small preset's width and one short sequence
        dict(name="dropout add norm bwd small", op="dropout_add_layernorm", backward=True, dtype="bf16", rows=128, hidden=512, p=0.1),
        # input embedding of the 104m step, word frequencies falling off as 1 / rank
        dict(name="embedding fwd bf16 104m", op="embedding", backward=False, dtype="bf16", tokens=32768, vocab=32000, hidden=1024, p=0.1, padded=False),
        dict(name="embedding bwd bf16 104m", op="embedding", backward=True, dtype="bf16", tokens=32768, vocab=32000, hidden=1024, p=0.1, padded=False),
        # a short padded batch of a small model without dropout
        dict(name="embedding bwd f32 padded", op="embedding", backward=True, dtype="f32", tokens=777, vocab=1000, hidden=250, p=0.0, padded=True),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["layernorm", "dropout", "dropout_add_layernorm", "embedding"])
    case = dict(op=op, backward=rng.random() < 0.5, dtype=rng.choice(["f16", "bf16", "f32"]))
    size = 4 if case["dtype"] == "f32" else 2
    most = 380_000_000 // (5 * size)          # elements a tensor, with up to five of them a call
    hidden = _log_uniform(rng, 32, 8192)
    if rng.random() < 0.6:
        hidden = max(32, hidden // 8 * 8)     # most models' widths are multiples of a vector load; the others are not
    if op == "embedding":
        case.update(tokens=_log_uniform(rng, 1, min(65536, most // hidden)), vocab=_log_uniform(rng, 64, min(131072, most // hidden)), hidden=hidden,
                    p=rng.choice([0.0, round(rng.uniform(0.02, 0.5), 3)]), padded=rng.random() < 0.3)
        return case
    case.update(rows=_log_uniform(rng, 1, min(65536, most // hidden)), hidden=hidden)
    if op != "layernorm":
        case["p"] = round(rng.uniform(0.02, 0.5), 3)
    if op == "dropout" or op == "layernorm" and case["backward"]:
        case["residual"] = rng.random() < 0.5 and not (op == "dropout" and case["backward"])
    return case


# ---------------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Everything the call reads. Activations have a few wide channels and rows of different scale and offset, as a residual
    stream has; gradients are of the size that a loss scale leaves."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)
    d = {"state": torch.tensor([(seed * 0x9E3779B97F4A7C15 + 0x1234567) & 0x7fffffffffffffff, (1 << 32) + seed], dtype=torch.int64, device="cuda")}
    hidden = case["hidden"]
    if case["op"] == "embedding":
        tokens, vocab = case["tokens"], case["vocab"]
        u = torch.rand(tokens, device="cuda", generator=g, dtype=torch.float64)
        ids = (torch.exp(u * math.log(vocab)).floor().long() - 1).clamp_(0, vocab - 1)   # P(id) ~ 1 / (id + 1)
        if case["padded"]:
            ids[torch.rand(tokens, device="cuda", generator=g) < 0.2] = vocab - 1
        d["ids"] = ids.to(torch.int32)
        if case["backward"]:
            d["grad"] = (0.05 * normal(tokens, hidden)).to(dt)
        else:
            d["weight"] = (0.02 * normal(vocab, hidden)).to(dt)
        return d
    rows = case["rows"]

    def activation():
        x = normal(rows, hidden)
        x *= 0.5 + torch.rand(rows, 1, device="cuda", generator=g)
        x[:, :: max(1, hidden // 7)] *= 8
        x += 0.5 * normal(rows, 1)
        return x.to(dt)

    if case["op"] != "dropout":
        d["weight"] = (1 + 0.1 * normal(hidden)).to(dt)
        d["bias"] = (0.1 * normal(hidden)).to(dt)
    if case["backward"]:
        d["grad"] = (0.05 * normal(rows, hidden)).to(dt)
        if case["op"] != "dropout":
            d["input"] = activation()
    else:
        d["input"] = activation()
    if case["op"] == "dropout_add_layernorm" or case.get("residual"):
        d["residual"] = (0.05 * normal(rows, hidden)).to(dt) if case["backward"] else activation()
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    like = s.get("input", s.get("grad"))
    op, backward = case["op"], case["backward"]
    out = {}
    if op == "embedding":
        rows = case["vocab"] if backward else case["tokens"]
        out["grad_weight" if backward else "output"] = torch.empty(rows, case["hidden"], device="cuda", dtype=DTYPES[case["dtype"]])
    else:
        out["grad_input" if backward else "output"] = torch.empty_like(like)
        if op == "dropout_add_layernorm":
            out["grad_residual" if backward else "sum"] = torch.empty_like(like)
        if op != "dropout" and backward:
            out["grad_weight"], out["grad_bias"] = torch.empty_like(s["weight"]), torch.empty_like(s["weight"])
    s["out"] = out
    return s


# ------------------------------------------------------------------------------------------------------ plain form
_LOW = 0xffffffff


def _philox_halves(state, blocks, device):
    """[blocks, 8] 16-bit numbers as int64. Products of two 32-bit words wrap in a signed 64-bit word, whose two halves are
    the product's all the same once the shifted-in sign is masked off."""
    c0 = torch.arange(blocks, device=device, dtype=torch.int64) & _LOW
    c1 = torch.full_like(c0, SITE)
    c2 = torch.zeros_like(c0) + (state[1] & _LOW)
    c3 = torch.zeros_like(c0) + ((state[1] >> 32) & _LOW)
    k0, k1 = state[0] & _LOW, (state[0] >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], dim=1)
    return torch.stack([words & 0xffff, words >> 16], dim=2).reshape(blocks, 8)


def _dropped(x, p, state):
    """The dropout map of a 32-bit tensor."""
    threshold = int(round(p * 65536))
    n = x.numel()
    keep = (_philox_halves(state, (n + 7) // 8, x.device).reshape(-1)[:n] >= threshold).reshape(x.shape)
    return torch.where(keep, x * (65536.0 / (65536 - threshold)), torch.zeros_like(x))


def _statistics(x):
    mean = x.mean(dim=1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPSILON)
    return centred * rstd, rstd


def _norm_backward(grad, x, weight):
    xhat, rstd = _statistics(x)
    g = grad * weight
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    return dx, (grad * xhat).sum(dim=0), grad.sum(dim=0)


def _plain(s):
    case = s["case"]
    dt, op, backward = DTYPES[case["dtype"]], case["op"], case["backward"]
    state, p = s["state"], case.get("p", 0.0)
    if op == "embedding":
        scale = math.sqrt(case["hidden"])
        ids = s["ids"].long()
        if not backward:
            out = s["weight"].float()[ids] * scale
            return {"output": (_dropped(out, p, state) if p else out).to(dt)}
        grad = s["grad"].float()
        grad = (_dropped(grad, p, state) if p else grad) * scale
        if case["padded"]:
            grad = torch.where((ids == case["vocab"] - 1)[:, None], torch.zeros_like(grad), grad)
        table = torch.zeros(case["vocab"], case["hidden"], device=grad.device)
        return {"grad_weight": table.index_add_(0, ids, grad).to(dt)}
    if op == "dropout":
        if backward:
            return {"grad_input": _dropped(s["grad"].float(), p, state).to(dt)}
        out = _dropped(s["input"].float(), p, state)
        return {"output": (out + s["residual"].float() if case["residual"] else out).to(dt)}
    weight, bias = s["weight"].float(), s["bias"].float()
    if backward:
        dx, dw, db = _norm_backward(s["grad"].float(), s["input"].float(), weight)
        if op == "layernorm":
            dx = dx + s["residual"].float() if case["residual"] else dx
            return {"grad_input": dx.to(dt), "grad_weight": dw.to(dt), "grad_bias": db.to(dt)}
        d = dx + s["residual"].float()
        return {"grad_input": _dropped(d, p, state).to(dt), "grad_residual": d.to(dt), "grad_weight": dw.to(dt), "grad_bias": db.to(dt)}
    if op == "layernorm":
        return {"output": (_statistics(s["input"].float())[0] * weight + bias).to(dt)}
    total = (_dropped(s["input"].float(), p, state) + s["residual"].float()).to(dt)   # the norm is of the sum as it is stored
    return {"output": (_statistics(total.float())[0] * weight + bias).to(dt), "sum": total}


# ------------------------------------------------------------------------------------------------ framework's calls
def _framework(s):
    from cgpt_b200 import ops
    case, out = s["case"], s["out"]
    op, backward = case["op"], case["backward"]
    if op == "layernorm":
        if backward:
            ops.layernorm_backward(out["grad_input"], out["grad_weight"], out["grad_bias"], s["grad"], s["input"], s["weight"], EPSILON,
                                   residual=s.get("residual"))
        else:
            ops.layernorm_forward(out["output"], s["input"], s["weight"], s["bias"], EPSILON)
        return out
    if op == "embedding":
        options = ops.ScaledEmbeddingOptions(scale=math.sqrt(case["hidden"]), padding_id=case["vocab"] - 1 if case["padded"] else None,
                                             dropout=ops.DropoutOptions(case["p"], SITE))
        if backward:
            ops.scaled_embedding_backward(out["grad_weight"], s["grad"], s["ids"], case["tokens"], s["state"], options=options)
        else:
            ops.scaled_embedding_forward(out["output"], s["ids"], case["tokens"], s["weight"], s["state"], options=options)
        return out
    options = ops.DropoutOptions(case["p"], SITE)
    if op == "dropout":
        if backward:
            ops.dropout_backward(out["grad_input"], s["grad"], s["state"], options=options)
        else:
            ops.dropout_forward(out["output"], s["input"], s["state"], options=options, residual=s.get("residual"))
    elif backward:
        ops.dropout_add_layernorm_backward(out["grad_input"], out["grad_residual"], out["grad_weight"], out["grad_bias"], s["grad"],
                                           s["residual"], s["input"], s["weight"], EPSILON, s["state"], options=options)
    else:
        ops.dropout_add_layernorm_forward(out["output"], out["sum"], s["input"], s["residual"], s["weight"], s["bias"], EPSILON,
                                          s["state"], options=options)
    return out


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    hidden = case["hidden"]
    if case["op"] == "embedding":
        tokens, vocab = case["tokens"], case["vocab"]
        if case["backward"]:     # every gradient row read, every table row written
            rows = tokens + vocab
        else:                    # every row that occurs read (expected number of them), every output row written
            v = np.arange(1, vocab, dtype=np.float64)
            share = np.log1p(1 / v) / math.log(vocab)
            kept = 0.8 if case["padded"] else 1.0
            rows = tokens + float(np.sum(-np.expm1(tokens * kept * np.log1p(-np.minimum(share, 1 - 1e-12))))) + (1 if case["padded"] else 0)
        return {"bytes": 4 * tokens + rows * hidden * size, "flops": 2 * tokens * hidden}
    n = case["rows"] * hidden
    if case["op"] == "dropout":
        return {"bytes": (2 + bool(case["residual"])) * n * size, "flops": (1 + bool(case["residual"])) * n}
    if case["op"] == "layernorm":
        tensors = 3 + bool(case["residual"]) if case["backward"] else 2
    else:
        tensors = 5 if case["backward"] else 4
    vectors = 3 if case["backward"] else 2
    return {"bytes": (tensors * n + vectors * hidden) * size, "flops": (16 if case["backward"] else 8) * n}


# ----------------------------------------------------------------------------------------------------------- exact
def _keep_mask(n, p, state):
    """Which of the first n elements stay, with the generator in unsigned 64-bit numpy words."""
    seed, step = (int(v) & 0xffffffffffffffff for v in state.tolist())
    m32 = np.uint64(0xffffffff)
    ctr = [np.arange((n + 7) // 8, dtype=np.uint64) & m32, np.uint64(SITE), np.uint64(step & 0xffffffff), np.uint64(step >> 32)]
    key = [seed & 0xffffffff, seed >> 32]
    for r in range(10):
        k = [np.uint64((key[0] + r * 0x9E3779B9) & 0xffffffff), np.uint64((key[1] + r * 0xBB67AE85) & 0xffffffff)]
        first, second = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = [(second >> np.uint64(32)) ^ ctr[1] ^ k[0], second & m32, (first >> np.uint64(32)) ^ ctr[3] ^ k[1], first & m32]
    bits = np.empty((ctr[0].size, 4, 2), dtype=np.uint16)
    for w in range(4):
        bits[:, w, 0] = ctr[w] & np.uint64(0xffff)
        bits[:, w, 1] = ctr[w] >> np.uint64(16)
    return torch.from_numpy(bits.reshape(-1)[:n] >= int(round(p * 65536))).cuda()


def exact(case, seed):
    d = _inputs(case, seed)
    f = {k: v.double() for k, v in d.items() if v.is_floating_point()}
    op, p = case["op"], case.get("p", 0.0)

    def drop(x):
        if not p:
            return x
        q = int(round(p * 65536)) / 65536
        return (x / (1 - q)).masked_fill(~_keep_mask(x.numel(), p, d["state"]).view(x.shape), 0.0)

    if op == "embedding":
        ids, scale = d["ids"].long(), math.sqrt(case["hidden"])
        if not case["backward"]:
            return {"output": drop(f["weight"].index_select(0, ids) * scale)}
        grad = drop(f["grad"]) * scale
        if case["padded"]:
            grad[ids == case["vocab"] - 1] = 0
        order = torch.argsort(ids, stable=True)
        counts = torch.bincount(ids, minlength=case["vocab"])
        return {"grad_weight": torch.segment_reduce(grad[order], "sum", lengths=counts, axis=0, unsafe=True)}
    if op == "dropout":
        out = drop(f["grad"] if case["backward"] else f["input"])
        return {"grad_input": out} if case["backward"] else {"output": out + f["residual"] if case["residual"] else out}
    x = f["input"]
    total = None
    if op == "dropout_add_layernorm" and not case["backward"]:
        total = drop(x) + f["residual"]
        x = total.to(DTYPES[case["dtype"]]).double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    root = torch.sqrt(var + EPSILON)
    xhat = (x - mean) / root
    if not case["backward"]:
        y = torch.addcmul(f["bias"], xhat, f["weight"])
        return {"output": y} if total is None else {"output": y, "sum": total}
    g = f["grad"] * f["weight"]
    hidden = case["hidden"]
    dx = (g - (g.sum(1, keepdim=True) + xhat * torch.linalg.vecdot(g, xhat, dim=1)[:, None]) / hidden) / root
    vectors = {"grad_weight": torch.einsum("rh,rh->h", f["grad"], xhat), "grad_bias": f["grad"].sum(0)}
    if op == "layernorm":
        return {"grad_input": dx + f["residual"] if case["residual"] else dx, **vectors}
    d_sum = dx + f["residual"]
    return {"grad_input": drop(d_sum), "grad_residual": d_sum, **vectors}
