"""The operators around a forest's leaf values, each in its plain form and as the framework's
own call: the embedding lookup with scaling, its gradient by sorted tokens, and the AdamW step
over many tensors at once.

A leaf is a token: a forest of T trees with L leaves each is a table of T * L rows, a row of the
data set is a bag of T tokens, and its prediction is the sum of the rows its tokens name.  The
same lookup with one token a bag and wide rows is the embedding of category codes.
"""
import math

import numpy as np
import torch

own = False  # True: run() makes the framework's calls instead of the plain form

BLOCK = 128  # elements of a block that shares a scale; a tensor's slot starts at a multiple of it
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.95, 1e-8, 0.1
STEPS_BEFORE, SEED = 100, 7
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one token of a served model: launch latency
        dict(name="lookup one", op="lookup", bags=1, per_bag=1, rows=32768, dim=4096, type="bf16", index=64, spread="even"),
        # the tokens of a training batch
        dict(name="lookup batch", op="lookup", bags=16384, per_bag=1, rows=131072, dim=4096, type="bf16", index=64, spread="even"),
        # prediction of a forest: a million rows, 128 trees of 256 leaves, one value a leaf
        dict(name="lookup forest", op="lookup", bags=1000000, per_bag=128, rows=32768, dim=1, type="fp32", index=32, spread="forest"),
        # bags of category codes, some slots empty (-1), rows of an odd width
        dict(name="lookup bags", op="lookup", bags=20011, per_bag=12, rows=50021, dim=100, type="fp16", index=32, spread="padded"),
        # a handful of tokens
        dict(name="grad few", op="grad", bags=64, per_bag=1, rows=4096, dim=512, type="fp32", out="fp32", index=64, spread="zipf", add=False),
        # the tokens of a training batch: few frequent ones, many rare ones, most rows untouched
        dict(name="grad batch", op="grad", bags=16384, per_bag=1, rows=131072, dim=4096, type="bf16", out="bf16", index=64, spread="zipf", add=False),
        # leaf values of a forest: the tokens stay the same from step to step, their order is kept
        dict(name="grad forest", op="grad", bags=1000000, per_bag=128, rows=32768, dim=1, type="fp32", out="fp32", index=32, spread="forest", add=False),
        # odd sizes, added to the gradient of the batches before
        dict(name="grad odd", op="grad", bags=9001, per_bag=1, rows=30011, dim=770, type="fp16", out="fp32", index=32, spread="zipf", add=True),
        # the leaf values of 500 trees of depth 8: one small tensor a tree, launch latency
        dict(name="step forest", op="step", tensors=500, elements=128000, mix="even", type="fp32", grad="fp32", bits=32, master=False),
        # half-precision weights with their single-precision copy
        dict(name="step master", op="step", tensors=40, elements=64000000, mix="odd", type="bf16", grad="bf16", bits=32, master=True),
        # half-precision weights, both moments in 8 bits
        dict(name="step 8 bits", op="step", tensors=60, elements=128000000, mix="odd", type="bf16", grad="bf16", bits=8, master=False),
        # many tensors of odd sizes, both moments in 8 bits
        dict(name="step 8 bits small", op="step", tensors=333, elements=2000003, mix="odd", type="fp32", grad="fp32", bits=8, master=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "step"])
    if op == "step":
        bits = rng.choice([8, 32])
        kind = rng.choice(["fp32", "bf16", "fp16"])
        master = bits == 32 and kind != "fp32" and rng.random() < 0.7
        tensors = _log(rng, 1, 600)
        return dict(op=op, tensors=tensors, elements=max(2 * tensors, _log(rng, 1000, 40000000)), mix=rng.choice(["even", "odd"]),
                    type=kind, grad=rng.choice([kind, "fp32"]), bits=bits, master=master)
    kind = rng.choice(["fp32", "bf16", "fp16"])
    spread = rng.choice(["even", "zipf", "padded", "forest"])
    if spread == "forest":
        per_bag = _log(rng, 2, 200)
        rows = per_bag * rng.choice([8, 32, 64, 256])
        case = dict(op=op, bags=_log(rng, 100, 100000000 // per_bag // 2), per_bag=per_bag, rows=rows, dim=rng.choice([1, 1, 2, 3]), type="fp32",
                    index=32, spread=spread)
        case["bags"] = max(1, case["bags"] // case["dim"])
    else:
        per_bag = _log(rng, 2, 40) if spread == "padded" else 1
        dim = rng.choice([_log(rng, 8, 6000), 8 * _log(rng, 1, 700)])
        rows = _log(rng, 10, min(200000, 200000000 // dim))
        case = dict(op=op, bags=_log(rng, 1, min(65536, 100000000 // dim // per_bag)), per_bag=per_bag, rows=rows, dim=dim, type=kind,
                    index=rng.choice([32, 64]), spread=spread)
    if op == "grad":
        case.update(out=rng.choice([case["type"], "fp32"]), add=spread != "forest" and rng.random() < 0.3)
    return case


# ---- inputs ----------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(case, g):
    n, t, v = case["bags"], case["per_bag"], case["rows"]
    kind = torch.int32 if case["index"] == 32 else torch.int64
    if case["spread"] == "forest":  # tree after tree, as the forest walk leaves them
        leaves = v // t
        # the leaves of a tree are not equally full
        leaf = (torch.rand((t, n), generator=g, device="cuda") ** 1.5 * leaves).to(torch.int32).clamp_(max=leaves - 1)
        leaf += torch.arange(t, dtype=torch.int32, device="cuda")[:, None] * leaves
        return leaf.to(kind).t()
    u = torch.rand((n, t), generator=g, device="cuda", dtype=torch.float64)
    if case["spread"] == "zipf":  # frequency falls as 1 / rank; ranks are spread over the table
        rank = (torch.exp(u * math.log(v + 1.0)) - 1).to(torch.int64).clamp_(0, v - 1)
        # a permutation of 0 .. v - 1: an odd multiplier that has no factor in common with v
        m = next(k for k in range(max(3, int(v * 0.618)) | 1, 4 * v + 64, 2) if math.gcd(k, v) == 1)
        tok = rank * m % v
    else:
        tok = (u * v).to(torch.int64).clamp_(max=v - 1)
    if case["spread"] == "padded":
        used = torch.randint(0, t + 1, (n, 1), generator=g, device="cuda")
        tok = torch.where(torch.arange(t, device="cuda") < used, tok, -1)
    return tok.to(kind)


def _scale(case):
    return math.sqrt(case["dim"]) if case["dim"] > 4 else 0.1


def _sizes(case):
    """Sizes of the tensors of one step, the same for every seed; none is empty."""
    n, total = case["tensors"], case["elements"]
    if case["mix"] == "even":
        share = np.full(n, total / n)
    else:  # a few matrices hold most of it, between them vectors and odd sizes
        share = np.exp(np.random.RandomState(n).uniform(0, 9, n))
        share *= total / share.sum()
    return [max(1, int(s)) for s in share]


def _layout(sizes):
    """Start of every tensor's slot in a flat buffer, and the buffer's length."""
    pad = [(s + BLOCK - 1) // BLOCK * BLOCK for s in sizes]
    begin = np.concatenate([[0], np.cumsum(pad)]).tolist()
    return begin[:-1], begin[-1]


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["op"] == "lookup":
        s["tokens"] = _tokens(case, g)
        s["table"] = (torch.randn((case["rows"], case["dim"]), generator=g, device="cuda") * 0.02).to(TYPES[case["type"]])
    elif case["op"] == "grad":
        s["tokens"] = _tokens(case, g)
        s["grad"] = torch.randn((case["bags"], case["dim"]), generator=g, device="cuda").to(TYPES[case["type"]])
        if case["add"]:
            s["sum"] = torch.randn((case["rows"], case["dim"]), generator=g, device="cuda").to(TYPES[case["out"]])
        if own and case["spread"] == "forest":
            import arboretum_b200
            s["order"] = arboretum_b200.token_order(s["tokens"], case["rows"], pooled=True)
    else:
        sizes = _sizes(case)
        begin, length = _layout(sizes)
        kept = torch.zeros(length, dtype=torch.bool, device="cuda")
        for b, n in zip(begin, sizes):
            kept[b:b + n] = True
        normal = lambda std: torch.randn(length, generator=g, device="cuda") * std * kept  # noqa: E731
        weights = normal(0.02)
        s["param"] = weights.to(TYPES[case["type"]])
        if case["master"]:
            s["master"] = weights
        s["grad"] = normal(1e-3).to(TYPES[case["grad"]])
        m, root = normal(2e-4), normal(1e-3).abs()
        if case["bits"] == 8:
            index = torch.arange(length, dtype=torch.int64, device="cuda")
            s["m"], s["m_scale"] = _to_8_bits(m, index, STEPS_BEFORE, 0)
            s["v"], s["v_scale"] = _to_8_bits(root, index, STEPS_BEFORE, 16)
        else:
            s["m"], s["v"] = m, root * root
        s["step"] = STEPS_BEFORE
        if own:
            import arboretum_b200
            cut = lambda x: [x[b:b + n] for b, n in zip(begin, sizes)]  # noqa: E731
            s["optimizer"] = arboretum_b200.AdamW(cut(s["param"]), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                                  state_bits=case["bits"], master=case["master"], seed=SEED)
            state = dict(step=STEPS_BEFORE, moment1=s["m"], moment2=s["v"])
            if case["bits"] == 8:
                state.update(scale1=s["m_scale"], scale2=s["v_scale"])
            if case["master"]:
                state.update(master=s["master"])
            s["optimizer"].load_state_dict(state)
            s["grads"] = cut(s["grad"])
    return s


# ---- one pass --------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    if case["op"] == "lookup":
        return _plain_lookup(s, case)
    if case["op"] == "grad":
        return _plain_grad(s, case)
    return _plain_step(s, case)


def _own(s, case):
    import arboretum_b200
    pooled = case.get("per_bag", 1) > 1
    if case["op"] == "lookup":
        return arboretum_b200.embedding(s["tokens"] if pooled else s["tokens"].view(-1), s["table"], scale=_scale(case), pooled=pooled)
    if case["op"] == "grad":
        if "order" in s:
            tokens = s["order"]
        else:
            tokens = s["tokens"] if pooled else s["tokens"].view(-1)
        return arboretum_b200.embedding_grad(s["grad"], tokens, case["rows"], scale=_scale(case), pooled=pooled,
                                             out=s.get("sum"), out_dtype=TYPES[case["out"]], accumulate=case["add"])
    o = s["optimizer"]
    o.step(s["grads"])
    return _state(s["param"], o.moment1, o.moment2, o.scale1, o.scale2, o.master)


def _state(param, m, v, m_scale, v_scale, master):
    out = dict(param=param, moment1=m, moment2=v)
    if m_scale is not None:
        out.update(scale1=m_scale, scale2=v_scale)
    if master is not None:
        out.update(master=master)
    return out


def _plain_lookup(s, case):
    tok, table = s["tokens"], s["table"]
    inside = (tok >= 0) & (tok < case["rows"])
    rows = table[torch.where(inside, tok, 0)].float() * inside[..., None]
    return (rows.sum(1) * _scale(case)).to(table.dtype)


def _plain_grad(s, case):
    n, t, v, dim = case["bags"], case["per_bag"], case["rows"], case["dim"]
    tok = s["tokens"].reshape(-1)
    tok = torch.where((tok >= 0) & (tok < v), tok, v)
    long = n * t >= 64 * v  # sums over thousands of rows
    g = s["grad"].to(torch.float64 if long else torch.float32)
    g = g[:, None].expand(n, t, dim).reshape(n * t, dim)
    total = torch.zeros((v + 1, dim), dtype=g.dtype, device="cuda").index_add_(0, tok, g)[:v] * _scale(case)
    if case["add"]:
        return s["sum"].copy_(s["sum"].to(total.dtype) + total)
    return total.to(TYPES[case["out"]])


def _plain_step(s, case):
    s["step"] += 1
    t = s["step"]
    p, g = s.get("master", s["param"]).float(), s["grad"].float()
    if case["bits"] == 8:
        m, root = _from_8_bits(s["m"], s["m_scale"]), _from_8_bits(s["v"], s["v_scale"])
        v = root * root
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = v.sqrt()
    below = root * (1 / math.sqrt(1 - BETA2 ** t)) + EPS
    p = p * (1 - LR * DECAY) - (m / below) * (LR / (1 - BETA1 ** t))
    s["param"].copy_(p)
    if case["master"]:
        s["master"].copy_(p)
    if case["bits"] == 8:
        index = torch.arange(p.numel(), dtype=torch.int64, device="cuda")
        s["m"], s["m_scale"] = _to_8_bits(m, index, t, 0)
        s["v"], s["v_scale"] = _to_8_bits(root, index, t, 16)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _state(s["param"], s["m"], s["v"], s.get("m_scale"), s.get("v_scale"), s.get("master"))


# ---- the moments in 8 bits -------------------------------------------------------------------
# A block of 128 values shares a power of two; a value is that times an e4m3 number.  Rounding is
# dithered: an element is rounded up with the probability of its remainder, by 16 bits of a hash of
# (element, step, seed), so that a moment that changes by less than half a step still moves on average.
def _hash(index, step):
    low = 0xFFFFFFFF
    x = (index & low) ^ ((index >> 32) * 0x9E3779B1 & low) ^ (step * 0x85EBCA6B & low) ^ (SEED * 0xC2B2AE35 & low)
    x = (x ^ (x >> 16)) * 0x7FEB352D & low
    x = (x ^ (x >> 15)) * 0x846CA68B & low
    return x ^ (x >> 16)


def _power(exponent):
    """2 ** (exponent - 127) as float32, exponent in 1 .. 254"""
    return (exponent << 23).to(torch.int32).view(torch.float32)


def _to_8_bits(x, index, step, shift):
    blocks = x.view(-1, BLOCK)
    top = blocks.abs().max(1).values.view(torch.int32).to(torch.int64)
    # the largest code stands for 448 = 1.75 * 2^8
    e = (((top + 0x1FFFFF) >> 23) - 8).clamp(1, 246)
    y = blocks.abs() * _power(254 - e)[:, None]  # exact
    bits = (y * 2.0 ** -120).view(torch.int32).view(-1).to(torch.int64)  # e4m3's exponents become float32's smallest
    u = ((_hash(index, step) >> shift & 0xFFFF) << 4) + 8
    code = ((bits + u) >> 20).clamp(max=126)
    if shift:  # no value above zero becomes zero: it is divided by
        code = torch.maximum(code, (x > 0).to(torch.int64))
    code = code | (x < 0).to(torch.int64) << 7
    return code.to(torch.uint8).view(torch.float8_e4m3fn), _power(e)


def _from_8_bits(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


# ---- what a pass cannot do without -----------------------------------------------------------
def _distinct(case):
    """Expected number of different tokens."""
    n, v = case["bags"] * case["per_bag"], case["rows"]
    if case["spread"] == "zipf":
        k = np.arange(v, dtype=np.float64)
        p = np.log((k + 2) / (k + 1)) / math.log(v + 1.0)
    else:
        p = np.float64(1 / v)
    if case["spread"] == "padded":
        n = n / 2
    each = -np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12)))
    return float(each.sum() if each.ndim else each * v)


def work(case):
    if case["op"] == "step":
        n = sum(_sizes(case))
        moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * n / BLOCK
        weights = (8 + SIZE[case["type"]]) * n if case["master"] else 2 * SIZE[case["type"]] * n
        return {"bytes": moments + weights + SIZE[case["grad"]] * n, "flops": 16 * n}
    n, t, v, dim = case["bags"], case["per_bag"], case["rows"], case["dim"]
    tokens = n * t * case["index"] // 8
    size = SIZE[case["type"]]
    if case["op"] == "lookup":
        return {"bytes": tokens + (_distinct(case) + n) * dim * size, "flops": n * t * dim}
    written = 2 * _distinct(case) if case["add"] else v
    return {"bytes": tokens + n * dim * size + written * dim * SIZE[case["out"]], "flops": n * t * dim}


# ---- the definitions in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        return _exact_lookup(s, case)
    if case["op"] == "grad":
        return _exact_grad(s, case)
    return _exact_step(s, case)


def _exact_lookup(s, case):
    v = case["rows"]
    table = torch.cat([s["table"].double(), torch.zeros((1, case["dim"]), dtype=torch.float64, device="cuda")])
    total = torch.zeros((case["bags"], case["dim"]), dtype=torch.float64, device="cuda")
    for t in range(case["per_bag"]):
        tok = s["tokens"][:, t].long()
        tok[(tok < 0) | (tok >= v)] = v
        total += table[tok]
    return total * _scale(case)


def _exact_grad(s, case):
    n, t, v, dim = case["bags"], case["per_bag"], case["rows"], case["dim"]
    if case["spread"] == "forest":
        total = torch.zeros((v, dim), dtype=torch.float64, device="cuda")
        for k in range(t):
            for d in range(dim):
                total[:, d] += torch.bincount(s["tokens"][:, k].long(), weights=s["grad"][:, d].double(), minlength=v)
        return total * _scale(case)
    tok, order = torch.sort(s["tokens"].reshape(-1).long(), stable=True)
    row = torch.div(order, t, rounding_mode="floor")
    total = torch.empty((v, dim), dtype=torch.float64, device="cuda")
    edge = torch.searchsorted(tok, torch.arange(v + 1, device="cuda"))
    for d in range(0, dim, 512):  # differences of the running sum over the sorted tokens
        run_sum = torch.zeros((n * t + 1, min(512, dim - d)), dtype=torch.float64, device="cuda")
        torch.cumsum(s["grad"][:, d:d + 512].double()[row], 0, out=run_sum[1:])
        total[:, d:d + 512] = run_sum[edge[1:]] - run_sum[edge[:-1]]
    total *= _scale(case)
    return total + s["sum"].double() if case["add"] else total


def _exact_step(s, case):
    t = STEPS_BEFORE + 1
    p, g = s.get("master", s["param"]).double(), s["grad"].double()
    if case["bits"] == 8:
        wide = lambda code, scale: code.double() * scale.double().repeat_interleave(BLOCK)  # noqa: E731
        m, v = wide(s["m"], s["m_scale"]), wide(s["v"], s["v_scale"]) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = (1 - LR * DECAY) * p - LR / (1 - BETA1 ** t) * m / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    out = dict(param=p, moment1=m, moment2=v)
    if case["master"]:
        out["master"] = p
    if case["bits"] == 8:
        index = torch.arange(p.numel(), dtype=torch.int64, device="cuda")
        out["moment1"], out["scale1"] = _exact_8_bits(m, _hash(index, t) & 0xFFFF)
        out["moment2"], out["scale2"] = _exact_8_bits(v ** 0.5, _hash(index, t) >> 16 & 0xFFFF)
        out["moment2"] = torch.where((v > 0) & (out["moment2"] == 0), 2.0 ** -9, out["moment2"])
    return out


def _exact_8_bits(x, random):
    top = x.view(-1, BLOCK).abs().amax(1)
    part, power = torch.frexp(top)  # top = part * 2^power, part in [0.5, 1); 448 = 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(top), torch.where(part > 0.875, power - 8, power - 9))
    scale = torch.where(top > 0, scale, 0.0).clamp(min=2.0 ** -126)
    y = x.abs() / scale.repeat_interleave(BLOCK)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    q = torch.floor(y / step + (random.double() + 0.5) / 65536) * step
    return torch.copysign(q.clamp(max=448.0), x), scale
