"""Workloads of the 8-bit floating point operators: their inputs, their plain
form in elementary torch operations, and the work they cannot do without.

Four operators, all over e4m3 values with one f32 scale per block of 128:

- quantize: f32 / f16 / bf16 activation rows -> e4m3, a scale per row and 128
  columns;
- prepare: a weight (dense, or ggml Q4_K / Q5_K / Q6_K blocks) -> e4m3, a
  scale per 128 x 128 block;
- matmul: activations quantised as above times a prepared weight;
- moe: a mixture-of-experts layer for a few tokens over prepared expert
  weights (router, top-k, gate / up, SiLU, down, weighted sum).

``own`` selects the framework's calls instead of the plain form.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"q4_k": 4, "q5_k": 5, "q6_k": 6}
BLOCK_BYTES = {"q4_k": 144, "q5_k": 176, "q6_k": 210}


# ---- cases -----------------------------------------------------------------

def listed():
    return [
        # the activations of one prompt of 512 tokens, hidden size 2048
        {"name": "quantize_prompt", "op": "quantize", "m": 512, "k": 2048, "type": "f32"},
        # a long batch in front of the largest weight
        {"name": "quantize_batch", "op": "quantize", "m": 16384, "k": 8192, "type": "bf16"},
        # a GGUF weight on its first use
        {"name": "prepare_q4k", "op": "prepare", "n": 5632, "k": 2048, "count": 1, "type": "q4_k"},
        # the gate weights of eight experts, dense
        {"name": "prepare_experts", "op": "prepare", "n": 5632, "k": 2048, "count": 8, "type": "bf16"},
        # one decode token through an up projection: latency counts
        {"name": "matmul_decode", "op": "matmul", "m": 1, "k": 2048, "n": 5632, "type": "f32"},
        # a decode batch through the largest weight: HBM-bound
        {"name": "matmul_batch16", "op": "matmul", "m": 16, "k": 8192, "n": 28672, "type": "bf16"},
        # a ragged prompt through an up projection
        {"name": "matmul_prompt333", "op": "matmul", "m": 333, "k": 1536, "n": 8960, "type": "f32"},
        # a prefill batch through the largest weight: tensor-bound
        {"name": "matmul_prefill", "op": "matmul", "m": 4096, "k": 8192, "n": 28672, "type": "bf16"},
        # one decode token, two of eight experts
        {"name": "moe_decode", "op": "moe", "t": 1, "h": 2048, "f": 5632, "e": 8, "top": 2, "type": "f32",
         "router": True, "renorm": True},
        # one decode token, eight of 64 small experts
        {"name": "moe_decode_fine", "op": "moe", "t": 1, "h": 2048, "f": 1024, "e": 64, "top": 8, "type": "bf16",
         "router": True, "renorm": False},
        # a ragged batch with routing from outside; some slots and one token empty
        {"name": "moe_routed13", "op": "moe", "t": 13, "h": 1536, "f": 2240, "e": 16, "top": 4, "type": "f16",
         "router": False, "renorm": False},
        # the largest decode batch: every expert active
        {"name": "moe_batch64", "op": "moe", "t": 64, "h": 4096, "f": 8192, "e": 8, "top": 2, "type": "bf16",
         "router": True, "renorm": True},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "prepare", "matmul", "matmul", "moe", "moe"])
    if op == "quantize":
        return {"op": op, "m": _log(rng, 1, 16384), "k": _log(rng, 100, 8192), "type": rng.choice(list(DTYPES))}
    if op == "prepare":
        kind = rng.choice(list(DTYPES) + list(KINDS))
        k = _log(rng, 256, 8192, 256) if kind in KINDS else _log(rng, 200, 8192)
        return {"op": op, "n": _log(rng, 64, 8192), "k": k, "count": 1 if kind in KINDS else rng.choice([1, 1, 2, 5]),
                "type": kind}
    if op == "matmul":
        return {"op": op, "m": _log(rng, 1, 4096), "k": _log(rng, 200, 8192), "n": _log(rng, 200, 28672),
                "type": rng.choice(list(DTYPES))}
    e = rng.choice([4, 8, 16, 24, 64])
    router = rng.random() < 0.7
    return {"op": op, "t": _log(rng, 1, 64), "h": _log(rng, 512, 4096, 16), "f": _log(rng, 256, 4096, 16), "e": e,
            "top": rng.randint(1, min(e, 8)), "type": rng.choice(list(DTYPES)), "router": router,
            "renorm": router and rng.random() < 0.5}


# ---- inputs ----------------------------------------------------------------

def _blocks(n):
    return (n + 127) // 128


def _activations(m, k, dtype, g):
    """N(0, 1) with one channel in a hundred 20 times larger."""
    a = torch.randn((m, k), device="cuda", generator=g)
    big = torch.rand(k, device="cuda", generator=g) < 0.01
    return torch.where(big, a * 20.0, a).to(dtype)


def _weights(shape, g):
    """e4m3 codes as a block-wise quantiser leaves N(0, 0.02^2) weights (the
    largest of a block near 448), and the blocks' scales.  Row pitch a
    multiple of 16 bytes."""
    *lead, n, k = shape
    k16 = (k + 15) // 16 * 16
    w = torch.empty((*lead, n, k16), device="cuda", dtype=torch.float8_e4m3fn)
    flat = w.view(-1, k16)
    rows = max(1, (1 << 28) // k16)
    for i in range(0, flat.shape[0], rows):
        part = flat[i:i + rows]
        part.copy_((torch.randn(part.shape, device="cuda", generator=g) * 110.0).clamp_(-E4M3_MAX, E4M3_MAX))
    s = (torch.rand((*lead, _blocks(n), _blocks(k)), device="cuda", generator=g) + 0.5) * (0.02 / 110.0)
    return w[..., :k], s


def _kquant_blocks(kind, count, g):
    """Valid superblocks: random codes and sub-scales, small positive d and dmin."""
    b = torch.randint(0, 256, (count, BLOCK_BYTES[kind]), device="cuda", generator=g, dtype=torch.uint8)
    d = (torch.rand(count, device="cuda", generator=g) * 2e-3 + 1e-4).half().view(torch.uint8).view(count, 2)
    if kind == "q6_k":
        b[:, 208:210] = d
    else:
        b[:, 0:2] = d
        b[:, 2:4] = (torch.rand(count, device="cuda", generator=g) * 2e-3).half().view(torch.uint8).view(count, 2)
    return b.reshape(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    op = case["op"]
    if op == "quantize":
        s["a"] = _activations(case["m"], case["k"], DTYPES[case["type"]], g)
    elif op == "prepare":
        if case["type"] in KINDS:
            s["blocks"] = _kquant_blocks(case["type"], case["n"] * (case["k"] // 256), g)
        else:
            shape = (case["count"], case["n"], case["k"])
            s["w"] = (torch.randn(shape, device="cuda", generator=g) * 0.02).to(DTYPES[case["type"]])
    elif op == "matmul":
        s["a"] = _activations(case["m"], case["k"], DTYPES[case["type"]], g)
        s["w"], s["ws"] = _weights((case["n"], case["k"]), g)
        if own:  # the scratch memory a program keeps for this shape
            from rocknpu_b200 import device as dev
            s["workspace"] = dev.new_workspace(dev.matmul_f8_workspace_bytes(case["m"], case["n"], case["k"]))
    else:
        t, h, f, e, top = (case[x] for x in ("t", "h", "f", "e", "top"))
        s["x"] = _activations(t, h, DTYPES[case["type"]], g)
        s["gate"], s["gate_s"] = _weights((e, f, h), g)
        s["up"], s["up_s"] = _weights((e, f, h), g)
        s["down"], s["down_s"] = _weights((e, h, f), g)
        s["router"] = s["ids"] = s["weights"] = None
        if case["router"]:
            s["router"] = torch.randn((e, h), device="cuda", generator=g) * (1.0 / math.sqrt(h))
        else:
            s["ids"] = torch.rand((t, e), device="cuda", generator=g).argsort(dim=1)[:, :top].int()
            s["weights"] = torch.rand((t, top), device="cuda", generator=g)
            empty = torch.rand((t, top), device="cuda", generator=g) < 0.1
            empty[t // 2] = t > 1
            s["ids"] = torch.where(empty, -1, s["ids"]).int().contiguous()
        if own:  # the scratch memory a program keeps for this layer
            from rocknpu_b200 import device as dev
            s["workspace"] = dev.new_workspace(dev.moe_f8_workspace_bytes(t, h, f, e, top, DTYPES[case["type"]]))
    return s


# ---- the operators ---------------------------------------------------------

def _scale(amax):
    return torch.where(amax == 0, torch.ones_like(amax), (amax / E4M3_MAX).clamp_min(SCALE_MIN))


def _quantize(a):
    """e4m3 rows and a scale per 128 columns."""
    m, k = a.shape
    kb = _blocks(k)
    x = torch.nn.functional.pad(a.float(), (0, kb * 128 - k)).view(m, kb, 128)
    s = _scale(x.abs().amax(dim=2))
    q = (x / s[:, :, None]).to(torch.float8_e4m3fn).view(m, kb * 128)[:, :k]
    return q, s


def _spread(s, n, k):
    """128 x 128 block scales -> one value per element."""
    return s.repeat_interleave(128, dim=-2)[..., :n, :].repeat_interleave(128, dim=-1)[..., :k]


def _values(w, s):
    return w.float() * _spread(s, w.shape[-2], w.shape[-1])


def _six_bit(b):
    """The eight 6-bit scales and mins of Q4_K / Q5_K's 12 packed bytes."""
    lo, mid, hi = b[:, 0:4], b[:, 4:8], b[:, 8:12]
    sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], dim=1)
    mn = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], dim=1)
    return sc.float(), mn.float()


def _half(b):
    return b.contiguous().view(torch.float16).float()


def _dequant(kind, blocks, n, k):
    """ggml superblocks of 256 -> f32 [n, k]."""
    b = blocks.view(-1, BLOCK_BYTES[kind])
    if kind == "q6_k":
        ql, qh, sc = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 1, 32), b[:, 192:208].view(torch.int8)
        low = torch.stack([ql & 15, ql >> 4], dim=2).view(-1, 2, 4, 32)
        high = torch.cat([(qh >> 0) & 3, (qh >> 2) & 3, (qh >> 4) & 3, (qh >> 6) & 3], dim=2)
        q = (low | (high << 4)).float() - 32.0
        v = (_half(b[:, 208:210]) * sc.float()).view(-1, 16, 1) * q.view(-1, 16, 16)
        return v.view(n, k)
    sc, mn = _six_bit(b[:, 4:16])
    qs = b[:, 48:176] if kind == "q5_k" else b[:, 16:144]
    qs = qs.view(-1, 4, 1, 32)
    q = torch.cat([qs & 15, qs >> 4], dim=2).view(-1, 8, 32)
    if kind == "q5_k":
        bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(1, 8, 1)
        q = q | (((b[:, 16:48].view(-1, 1, 32) >> bit) & 1) << 4)
    v = (_half(b[:, 0:2]) * sc)[:, :, None] * q.float() - (_half(b[:, 2:4]) * mn)[:, :, None]
    return v.view(n, k)


def _prepare(w):
    """Dense [count, n, k] -> e4m3 and a scale per 128 x 128 block."""
    c, n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    x = torch.nn.functional.pad(w.float(), (0, kb * 128 - k, 0, nb * 128 - n)).view(c, nb, 128, kb, 128)
    s = _scale(x.abs().amax(dim=(2, 4)))
    q = (x / s[:, :, None, :, None]).to(torch.float8_e4m3fn).view(c, nb * 128, kb * 128)
    return q[:, :n, :k], s


def _moe(s):
    case = s["case"]
    t, e, top = case["t"], case["e"], case["top"]
    x = s["x"].float()
    if case["router"]:
        # logits in 64 bits: the selection is a comparison of neighbours
        logits = s["x"].double() @ s["router"].double().t()
        order = torch.sort(logits, dim=1, descending=True, stable=True)
        ids = order.indices[:, :top].int()
        p = torch.softmax(logits, dim=1).gather(1, ids.long())
        p = (p / p.sum(dim=1, keepdim=True) if case["renorm"] else p).float()
        weights = p
    else:
        ids, weights = s["ids"], s["weights"]
        p = torch.where(ids >= 0, weights, torch.zeros_like(weights))
    at = ids.clamp_min(0).long()
    if t * top <= e:  # few slots: each with its own expert's weights
        at = at.view(-1)
        xs = x.repeat_interleave(top, dim=0)[:, :, None]
        gate = torch.bmm(_values(s["gate"][at], s["gate_s"][at]), xs)
        up = torch.bmm(_values(s["up"][at], s["up_s"][at]), xs)
        y = torch.bmm(_values(s["down"][at], s["down_s"][at]), gate * torch.sigmoid(gate) * up)
        y = (y.view(t, top, -1) * p[:, :, None]).sum(dim=1)
    else:  # every expert on every token, weighted by 0 where it was not chosen
        dense = torch.zeros((t, e), device=x.device).scatter_add_(1, at, p)
        gate = x @ _values(s["gate"], s["gate_s"]).transpose(1, 2)
        up = x @ _values(s["up"], s["up_s"]).transpose(1, 2)
        y = (gate * torch.sigmoid(gate) * up) @ _values(s["down"], s["down_s"]).transpose(1, 2)
        y = (y * dense.t()[:, :, None]).sum(dim=0)
    return y.to(s["x"].dtype), ids, weights


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from rocknpu_b200 import device as dev
        if op == "quantize":
            return dev.quantize_rows_f8(s["a"], s["status"])
        if op == "prepare":
            if case["type"] in KINDS:
                return dev.prepare_f8_q(KINDS[case["type"]], s["blocks"], case["k"], case["n"], s["status"])
            return dev.prepare_f8(s["w"], s["status"])
        if op == "matmul":
            return dev.matmul_f8(s["a"], s["w"], s["ws"], s["status"], s["workspace"])
        return dev.moe_f8(s["x"], (s["gate"], s["gate_s"]), (s["up"], s["up_s"]), (s["down"], s["down_s"]),
                          s["status"], s["workspace"], router=s["router"], top_k=case["top"],
                          renormalize=case["renorm"], ids=s["ids"], weights=s["weights"])
    if op == "quantize":
        return _quantize(s["a"])
    if op == "prepare":
        if case["type"] in KINDS:
            q, sc = _prepare(_dequant(case["type"], s["blocks"], case["n"], case["k"])[None])
            return q[0], sc[0]
        return _prepare(s["w"])
    if op == "matmul":
        m, k = s["a"].shape
        q, sc = _quantize(s["a"])
        a = q.float() * sc.repeat_interleave(128, dim=1)[:, :k]
        return (a @ _values(s["w"], s["ws"]).t()).to(s["a"].dtype)
    return _moe(s)


# ---- work ------------------------------------------------------------------

def _active(case):
    """Experts that a pass reads: the expected number that t choices of `top` name."""
    return round(case["e"] * (1.0 - (1.0 - case["top"] / case["e"]) ** case["t"]))


def work(case):
    op = case["op"]
    if op == "quantize":
        m, k, b = case["m"], case["k"], 4 if case["type"] == "f32" else 2
        return {"bytes": m * k * (b + 1) + 4 * m * _blocks(k), "flops": 3 * m * k}
    if op == "prepare":
        n, k, c = case["n"], case["k"], case["count"]
        read = n * (k // 256) * BLOCK_BYTES[case["type"]] if case["type"] in KINDS else \
            c * n * k * (4 if case["type"] == "f32" else 2)
        return {"bytes": read + c * (n * k + 4 * _blocks(n) * _blocks(k)), "flops": 3 * c * n * k}
    b = 4 if case["type"] == "f32" else 2
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + 4 * _blocks(n) * _blocks(k) + b * m * (n + k), "flops": 2 * m * n * k}
    t, h, f, e, top = (case[x] for x in ("t", "h", "f", "e", "top"))
    weights = 3 * h * f + 12 * _blocks(h) * _blocks(f)
    return {"bytes": _active(case) * weights + 2 * b * t * h + (4 * e * h if case["router"] else 0) + 8 * t * top,
            "flops": 6 * t * top * h * f + (2 * t * e * h if case["router"] else 0)}


# ---- the definition in 64 bits ---------------------------------------------

def _near(v):
    """Nearest e4m3 value of 64-bit values within +-448 (ties to even)."""
    mag = v.abs()
    step = torch.exp2(torch.floor(torch.log2(mag.clamp_min(2.0 ** -6))) - 3.0)
    return torch.sign(v) * torch.minimum(torch.round(mag / step) * step, torch.full_like(mag, E4M3_MAX))


def _block_max(x, rows, cols):
    """Largest magnitude of each rows x cols block of the last two axes, spread back over its elements."""
    n, k = x.shape[-2:]
    i = torch.arange(n, device=x.device) // rows
    j = torch.arange(k, device=x.device) // cols
    top = torch.zeros((*x.shape[:-2], n, int(j[-1]) + 1), device=x.device, dtype=x.dtype)
    top.scatter_reduce_(-1, j.expand(x.shape), x.abs(), "amax")
    best = torch.zeros((*x.shape[:-2], int(i[-1]) + 1, top.shape[-1]), device=x.device, dtype=x.dtype)
    best.scatter_reduce_(-2, i[:, None].expand(top.shape), top, "amax")
    return best, i, j


def _exact_quantized(x, rows):
    best, i, j = _block_max(x, rows, 128)
    s = torch.where(best > 0, torch.maximum(best / E4M3_MAX, torch.full_like(best, SCALE_MIN)), torch.ones_like(best))
    return _near(x / s[..., i, :][..., j]), s, i, j


def _exact_kquant(kind, raw, n, k):
    """Superblock values from the format's definition, one 32-value group at a time."""
    b = raw.view(-1, BLOCK_BYTES[kind]).long()

    def f16(at):
        return raw.view(-1, BLOCK_BYTES[kind])[:, at:at + 2].contiguous().view(torch.float16).double()[:, 0]

    out = torch.empty((b.shape[0], 256), device=raw.device, dtype=torch.float64)
    if kind == "q6_k":
        d = f16(208)
        for y in range(256):
            half, r = divmod(y, 128)
            quarter, l = divmod(r, 32)
            byte = b[:, 64 * half + 32 * (quarter % 2) + l]
            low = byte % 16 if quarter < 2 else byte // 16
            high = (b[:, 128 + 32 * half + l] // 4 ** quarter) % 4
            sc = b[:, 192 + y // 16]
            sc = torch.where(sc > 127, sc - 256, sc)
            out[:, y] = d * sc * (low + 16 * high - 32)
        return out.view(n, k)
    d, dmin = f16(0), f16(2)
    for j in range(8):
        if j < 4:
            sc, mn = b[:, 4 + j] % 64, b[:, 8 + j] % 64
        else:
            sc = b[:, 8 + j] % 16 + 16 * (b[:, j] // 64)
            mn = b[:, 8 + j] // 16 + 16 * (b[:, 4 + j] // 64)
        base = (48 if kind == "q5_k" else 16) + 32 * (j // 2)
        byte = b[:, base:base + 32]
        q = byte % 16 if j % 2 == 0 else byte // 16
        if kind == "q5_k":
            q = q + 16 * ((b[:, 16:48] // 2 ** j) % 2)
        out[:, 32 * j:32 * j + 32] = (d * sc)[:, None] * q - (dmin * mn)[:, None]
    return out.view(n, k)


def _exact_weight(w, s):
    i = torch.arange(w.shape[-2], device=w.device) // 128
    j = torch.arange(w.shape[-1], device=w.device) // 128
    return w.float().double() * s.double()[i][:, j]


def exact(case, seed):
    op = case["op"]
    if op == "matmul" and 2.0 * case["m"] * case["n"] * case["k"] > 2e14:
        return None
    s = prepare(case, seed)
    if op == "quantize":
        q, sc, _, _ = _exact_quantized(s["a"].double(), 1)
        return q, sc
    if op == "prepare":
        if case["type"] in KINDS:
            return _exact_quantized(_exact_kquant(case["type"], s["blocks"], case["n"], case["k"]), 128)[:2]
        qs, scs = zip(*(_exact_quantized(w.double(), 128)[:2] for w in s["w"]))
        return torch.stack(qs), torch.stack(scs)
    if op == "matmul":
        q, sc, _, j = _exact_quantized(s["a"].double(), 1)
        a = q * sc[:, j]
        out = torch.empty((case["m"], case["n"]), device="cuda", dtype=torch.float64)
        for r in range(0, case["n"], 4096):
            out[:, r:r + 4096] = a @ _exact_weight(s["w"][r:r + 4096], s["ws"][r // 128:r // 128 + 32]).t()
        return out
    t, top = case["t"], case["top"]
    x = s["x"].double()
    if case["router"]:
        logits = (x[:, None, :] * s["router"].double()[None]).sum(dim=2)
        left = logits.clone()
        ids = torch.empty((t, top), device="cuda", dtype=torch.int32)
        for k in range(top):
            ids[:, k] = left.argmax(dim=1)
            left.scatter_(1, ids[:, k:k + 1].long(), float("-inf"))
        chosen = logits.gather(1, ids.long())
        norm = torch.logsumexp(chosen if case["renorm"] else logits, dim=1, keepdim=True)
        weights = torch.exp(chosen - norm)
    else:
        ids, weights = s["ids"], s["weights"].double()
    y = torch.zeros_like(x)
    for e in range(case["e"]):
        p = torch.where(ids == e, weights, torch.zeros_like(weights)).sum(dim=1, keepdim=True)
        rows = (ids == e).any(dim=1).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        gate = x[rows] @ _exact_weight(s["gate"][e], s["gate_s"][e]).t()
        up = x[rows] @ _exact_weight(s["up"][e], s["up_s"][e]).t()
        h = gate / (1.0 + torch.exp(-gate)) * up
        y[rows] += p[rows] * (h @ _exact_weight(s["down"][e], s["down_s"][e]).t())
    return y, ids, weights
