"""Timed cases of the gradient operators: the global norm over many tensors,
clipping by it, microscaled 4-bit quantisation and the fold of such payloads.

`own = False` runs each operator in its plain form (elementary torch
operations); `own = True` calls gloo_amd.

A microscaled (MXFP4) payload of n elements: ceil(n / 32) blocks of 16 bytes
(32 codes of 4 bits, the even element in the low half), then one scale byte a
block (2^(byte - 127); 255: the block is NaN), zero bytes up to a multiple of 16.
"""
import random

import torch

own = False

DTYPES = {"float64": torch.float64, "float32": torch.float32, "float16": torch.float16,
          "bfloat16": torch.bfloat16}
EPS = 1e-6  # the clip coefficient is max_norm / (norm + EPS), at most 1
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # a small model's gradients (or one rank's shard of them): latency
        dict(name="norm_small_f32", op="norm", numel=40961, tensors=24, dtype="float32",
             p="2", packed=True),
        # bf16 gradients as ragged, back-to-back views of a 128 MiB bucket
        dict(name="norm_bf16", op="norm", numel=(64 << 20) + 77, tensors=148, dtype="bfloat16",
             p="2", packed=True),
        # 1 GiB of f32 gradients, the repository's largest message, as separate tensors
        dict(name="norm_f32_1GiB", op="norm", numel=256 << 20, tensors=291, dtype="float32",
             p="2", packed=False),
        # clipping a small model: latency
        dict(name="clip_small_bf16", op="clip", numel=100003, tensors=20, dtype="bfloat16",
             p="2", packed=True),
        # the repository's main size (256 MiB of f32), clipped out of the exchange
        # bucket into the optimizer's
        dict(name="clip_f32_256MiB", op="clip", numel=64 << 20, tensors=148, dtype="float32",
             p="2", packed=False),
        # bf16 matrices with f32 norms and biases among them, 1 GiB and more
        dict(name="clip_mixed_large", op="clip", numel=(400 << 20) + 5, tensors=291, dtype="mixed",
             p="2", packed=True),
        # a small odd message, squeezed and opened again
        dict(name="quant_small_f32", op="quant", numel=20011, dtype="float32", feedback=False),
        # a 256 MiB bf16 bucket
        dict(name="quant_bf16_256MiB", op="quant", numel=(128 << 20) + 9, dtype="bfloat16",
             feedback=False),
        # the 1 GiB f32 bucket with error feedback
        dict(name="quant_f32_ef_1GiB", op="quant", numel=256 << 20, dtype="float32",
             feedback=True),
        # two ranks' small messages
        dict(name="fold_small_f32", op="fold", numel=40009, sources=2, dtype="float32"),
        # one hop of a compressed exchange: four payloads into one
        dict(name="fold4_requant", op="fold", numel=(128 << 20) - 31, sources=4, dtype="payload"),
        # eight ranks' payloads of a 1 GiB f32 bucket into its mean
        dict(name="fold8_f32_1GiB", op="fold", numel=256 << 20, sources=8, dtype="float32"),
    ]


def _size(rng, low, high):
    """Log-uniform in [low, high], odd as often as not."""
    v = int(low * (high / low) ** rng.random())
    return max(low, min(high, v + rng.randrange(2)))


def draw(rng):
    op = rng.choice(("norm", "clip", "quant", "fold"))
    if op in ("norm", "clip"):
        dtype = rng.choice(("float32", "bfloat16", "float16", "mixed", "float64"))
        numel = _size(rng, 1000, 128 << 20)
        return dict(op=op, numel=numel, tensors=min(numel, _size(rng, 1, 400)), dtype=dtype,
                    p=rng.choice(("2", "2", "1", "inf")), packed=rng.random() < 0.5)
    if op == "quant":
        return dict(op=op, numel=_size(rng, 33, 200 << 20),
                    dtype=rng.choice(("float32", "bfloat16", "float16")),
                    feedback=rng.random() < 0.5)
    k = rng.randrange(1, 17)
    return dict(op=op, numel=_size(rng, 33, (512 << 20) // max(k, 4)), sources=k,
                dtype=rng.choice(("float32", "bfloat16", "float16", "payload")))


# ---- inputs -----------------------------------------------------------------

def _split(numel, tensors):
    """Sizes of `tensors` tensors of numel elements in all: a few large ones, many small."""
    rng = random.Random(numel * 1009 + tensors)
    w = [rng.lognormvariate(0, 1.5) for _ in range(tensors)]
    rest, total, sizes = numel - tensors, sum(w), []
    for x in w:
        sizes.append(1 + int(rest * x / total))
    sizes[sizes.index(max(sizes))] += numel - sum(sizes)
    return sizes


def _buckets(case):
    """[(dtype, [(offset, size)], bucket elements)] of a case's tensors."""
    sizes = _split(case["numel"], case["tensors"])
    if case["dtype"] == "mixed":  # every fourth tensor in f32
        parts = [("bfloat16", [s for i, s in enumerate(sizes) if i % 4 != 3]),
                 ("float32", [s for i, s in enumerate(sizes) if i % 4 == 3])]
    else:
        parts = [(case["dtype"], sizes)]
    out = []
    for dtype, part in parts:
        if not part:
            continue
        at, spans = 0, []
        for s in part:
            spans.append((at, s))
            at += s if case["packed"] else -(-s // 128) * 128
        out.append((DTYPES[dtype], spans, at))
    return out


def _normal(n, dtype, gen, spread):
    """Normal values whose magnitude varies by `spread` octaves over stretches of 1024 elements."""
    x = torch.randn(n, generator=gen, device="cuda", dtype=torch.float32)
    m = torch.exp2(spread * torch.randn(-(-n // 1024), generator=gen, device="cuda"))
    full = n // 1024 * 1024
    x[:full].view(-1, 1024).mul_(m[:n // 1024, None])
    x[full:].mul_(m[-1])
    return x.mul_(0.02).to(dtype)


def payload_bytes(n):
    nb = -(-n // 32)
    return -(-nb * 17 // 16) * 16


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case=case, n=case["numel"])
    if case["op"] in ("norm", "clip"):
        s["p"] = float(case["p"])
        s["buckets"], s["grads"], s["outs"], s["out_buckets"] = [], [], [], []
        for dtype, spans, total in _buckets(case):
            b = _normal(total, dtype, gen, 1.0)
            s["buckets"].append(b)
            s["grads"] += [b[at:at + n] for at, n in spans]
            if case["op"] == "clip":
                o = torch.zeros_like(b)
                s["out_buckets"].append(o)
                s["outs"] += [o[at:at + n] for at, n in spans]
        s["max_norm"] = 0.01 if case["p"] == "inf" else 1.0
        s["wide"] = any(g.dtype == torch.float64 for g in s["grads"])
        if own:
            import gloo_amd
            s["handle"] = gloo_amd.Gradients(s["grads"], outs=s["outs"] or None)
    elif case["op"] == "quant":
        dtype = DTYPES[case["dtype"]]
        s["x"] = _normal(s["n"], dtype, gen, 1.0)
        s["payload"] = torch.empty(payload_bytes(s["n"]), dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty_like(s["x"])
        s["residual"] = s["residual_out"] = None
        if case["feedback"]:
            s["residual"] = _normal(s["n"], torch.float32, gen, 1.0).mul_(0.1)
            s["residual_out"] = torch.empty_like(s["residual"])
    else:
        k = case["sources"]
        s["payloads"] = torch.empty(k, payload_bytes(s["n"]), dtype=torch.uint8, device="cuda")
        for row in s["payloads"]:
            row.copy_(_pack(*_encode(_normal(s["n"], torch.float32, gen, 1.0)), s["n"]))
        s["rows"] = list(s["payloads"])
        s["scale"] = float(torch.tensor(1.0 / k, dtype=torch.float32))
        if case["dtype"] == "payload":
            s["payload"] = torch.empty_like(s["rows"][0])
            s["values"] = torch.empty(s["n"], device="cuda")
        else:
            s["values"] = torch.empty(s["n"], device="cuda", dtype=DTYPES[case["dtype"]])
    return s


# ---- plain forms ------------------------------------------------------------

def _power_sum(grads, p):
    """The sum of |g|^p in 64 bits over all tensors (the maximum for p = inf)."""
    wide = [g if g.dtype == torch.float64 else g.float() for g in grads]
    if p == float("inf"):
        return torch.stack([g.abs().max().double() for g in wide]).max()
    if p == 1:
        return torch.stack([g.abs().sum(dtype=torch.float64) for g in wide]).sum()
    return torch.stack([g.square().sum(dtype=torch.float64) for g in wide]).sum()


def _norm(s):
    t = _power_sum(s["grads"], s["p"])
    return t.sqrt() if s["p"] == 2 else t


def _clip(s):
    total = _norm(s)
    c = (s["max_norm"] / (total + EPS)).clamp(max=1.0)
    for g, o in zip(s["grads"], s["outs"]):
        o.copy_(g * c if g.dtype == torch.float64 else g.float() * c.float())
    return total


def _pow2(e):
    """2^(e - 127) for a biased exponent e in 0..254, from its bits."""
    return torch.where(e > 0, e << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _encode(y):
    """(codes [blocks, 32], scale bytes [blocks]) of f32 values y."""
    n = y.numel()
    nb = -(-n // 32)
    b = y if n == nb * 32 else torch.cat([y, y.new_zeros(nb * 32 - n)])
    b = b.view(nb, 32)
    bits = b.view(torch.int32)
    e = (bits & 0x7fffffff).amax(1) >> 23
    bad = e == 255
    e = (e - 2).clamp(min=0)
    a = (b / _pow2(e)[:, None]).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5))
    code = torch.where(bits < 0, code + 8, code)
    code = torch.where(bad[:, None], torch.zeros_like(code), code)
    return code, torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)


def _pack(code, scale, n):
    out = torch.zeros(payload_bytes(n), dtype=torch.uint8, device=code.device)
    nb = scale.numel()
    out[:nb * 16] = (code[:, 0::2] | (code[:, 1::2] << 4)).reshape(-1)
    out[nb * 16:nb * 17] = scale
    return out


def _unpack(payload, n):
    """The f32 values of payloads [..., bytes]: [..., n]."""
    nb = -(-n // 32)
    table = torch.tensor(FP4 + tuple(-v for v in FP4), device=payload.device)
    codes = payload[..., :nb * 16]
    scale = payload[..., nb * 16:nb * 17].int()
    pair = torch.stack([codes & 15, codes >> 4], -1).int()
    v = table[pair].view(*payload.shape[:-1], nb, 32)
    v = v * torch.where(scale == 255, float("nan"), _pow2(scale.clamp(max=254)))[..., None]
    return v.view(*payload.shape[:-1], nb * 32)[..., :n]


def _quant(s):
    y = s["x"].float()
    if s["residual"] is not None:
        y = y + s["residual"]
    code, scale = _encode(y)
    s["payload"].copy_(_pack(code, scale, s["n"]))
    v = _unpack(s["payload"], s["n"])
    s["values"].copy_(v)
    if s["residual"] is not None:
        s["residual_out"].copy_(torch.where(v.isnan(), 0.0, y - v))


def _fold(s):
    acc = _unpack(s["rows"][0], s["n"])
    for row in s["rows"][1:]:
        acc = acc + _unpack(row, s["n"])
    acc = acc * s["scale"]
    if s["case"]["dtype"] == "payload":
        s["payload"].copy_(_pack(*_encode(acc), s["n"]))
        acc = _unpack(s["payload"], s["n"])
    s["values"].copy_(acc)


# ---- one pass ---------------------------------------------------------------

def run(state):
    s = state
    op = s["case"]["op"]
    if op == "norm":
        if own:
            return {"norm": s["handle"].norm(s["p"])}
        return {"norm": _norm(s).to(torch.float64 if s["wide"] else torch.float32)}
    if op == "clip":
        if own:
            total = s["handle"].clip_norm(s["max_norm"], s["p"])
        else:
            total = _clip(s).to(torch.float64 if s["wide"] else torch.float32)
        return {"norm": total, "clipped": s["out_buckets"]}
    if op == "quant":
        # the payload is given back as the values that it stands for
        if own:
            from gloo_amd import mx
            mx.quantize(s["x"], s["payload"], residual=s["residual"],
                        residual_out=s["residual_out"])
            mx.dequantize(s["values"], s["payload"])
        else:
            _quant(s)
        return {"values": s["values"], "residual": s["residual_out"]}
    if own:
        from gloo_amd import mx
        if s["case"]["dtype"] == "payload":
            mx.requantize_n(s["payload"], s["rows"], s["n"], scale=s["scale"])
            mx.dequantize(s["values"], s["payload"])
        else:
            mx.reduce_n(s["values"], s["rows"], scale=s["scale"])
    else:
        _fold(s)
    return {"values": s["values"]}


def work(case):
    n = case["numel"]
    if case["op"] in ("norm", "clip"):
        size = sum(sum(m for _, m in spans) * torch.empty(0, dtype=d).element_size()
                   for d, spans, _ in _buckets(case))
        clip = case["op"] == "clip"
        return {"bytes": size * (2 if clip else 1), "flops": n * (3 if clip else 2)}
    pay = payload_bytes(n)
    if case["op"] == "quant":
        es = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
        # x read, the payload and its values written; both residuals
        return {"bytes": n * es * 2 + pay + (n * 8 if case["feedback"] else 0), "flops": n * 4}
    k = case["sources"]
    if case["dtype"] == "payload":
        return {"bytes": pay * (k + 1) + n * 4, "flops": n * (2 * k + 3)}
    es = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    return {"bytes": pay * k + n * es, "flops": n * (2 * k + 1)}


# ---- the definitions in 64 bits ---------------------------------------------

def _two64(e):
    """2^e in 64 bits, from its bits: pow() may be off in the last place, which moves ties."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(y):
    """What y (f64 holding f32 values) stands for after quantisation: per block of
    32 the step below the largest power of two, round half to even."""
    n = y.numel()
    b = torch.nn.functional.pad(y, (0, -n % 32)).view(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    e = torch.frexp(top)[1] - 1  # top = m 2^e, 1 <= m < 2
    scale = _two64((e - 2).clamp(-127, 127))
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    a = b.abs() / scale
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = ((a / step).round() * step).clamp(max=6.0) * scale
    q = torch.where(top.isfinite(), torch.copysign(q, b), float("nan"))
    return q.view(-1)[:n]


def _open64(row, n):
    """The values of one payload in 64 bits."""
    nb = -(-n // 32)
    c = torch.empty(nb * 32, dtype=torch.int64, device=row.device)
    c[0::2] = row[:nb * 16].long() % 16
    c[1::2] = row[:nb * 16].long() // 16
    exp, man = (c % 8) // 2, (c % 2).double()
    mag = torch.where(exp == 0, man / 2, (1 + man / 2) * _two64(exp - 1))
    mag = torch.where(c >= 8, -mag, mag).view(nb, 32)
    s = row[nb * 16:nb * 17].long()
    s = torch.where(s == 255, float("nan"), _two64(s - 127))
    return (mag * s[:, None]).view(-1)[:n]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] in ("norm", "clip"):
        p = s["p"]
        parts = [g.double().abs() for g in s["buckets"]] if case["packed"] else \
            [g.double().abs() for g in s["grads"]]
        if p == float("inf"):
            total = max(float(g.max()) for g in parts)
        else:
            total = sum(float((g ** p).sum()) for g in parts) ** (1 / p)
        norm = torch.tensor(total, dtype=torch.float64)
        if case["op"] == "norm":
            return {"norm": norm}
        c = min(1.0, s["max_norm"] / (total + EPS))
        clipped = []
        for b, (_, spans, _) in zip(s["buckets"], _buckets(case)):
            o = torch.zeros(b.numel(), dtype=torch.float64, device=b.device)
            for at, n in spans:
                o[at:at + n] = b[at:at + n].double() * c
            clipped.append(o)
        return {"norm": norm, "clipped": clipped}
    if case["op"] == "quant":
        y = s["x"].double()
        if s["residual"] is not None:
            # the sum is held in 32 bits, as the residual is, before it is quantised
            y = (y + s["residual"].double()).float().double()
        v = _values64(y)
        return {"values": v, "residual": None if s["residual"] is None else y - v}
    acc = _open64(s["rows"][0], s["n"])
    for row in s["rows"][1:]:
        acc += _open64(row, s["n"])
    acc *= s["scale"]
    if case["dtype"] == "payload":
        acc = _values64(acc.float().double())
    return {"values": acc}
