"""Cases of the operators around a fused RMSNorm -> Linear layer, in a plain form and as the framework's calls.

linear          y = act(x W^T + bias) + residual
qk_norm_rope    RMSNorm of every query and key head and the rotation by position, from the fused QKV projection
kv_cache_write  keys and values into a paged e4m3 cache, one fp32 scale per token and head
kv_cache_read   the pages of every sequence back as bf16, packed one behind the other
"""
import math
import random  # noqa: F401  (draw takes a random.Random)

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100   # rows of zeros get a scale as well
EPS = 1e-6
MAX_POSITION = 32768


def listed():
    return [
        # one token through the output projection, added to the residual stream
        {"name": "linear_out_1", "op": "linear", "tokens": 1, "n": 4096, "k": 4096, "bias": False, "act": "none", "residual": True},
        # a full decode batch through a biased up projection
        {"name": "linear_up_64", "op": "linear", "tokens": 64, "n": 14336, "k": 4096, "bias": True, "act": "gelu_tanh", "residual": False},
        # a short prompt on a layer with odd sizes, everything switched on
        {"name": "linear_odd_333", "op": "linear", "tokens": 333, "n": 1001, "k": 1144, "bias": True, "act": "silu", "residual": True},
        # a long prompt through the down projection
        {"name": "linear_down_8192", "op": "linear", "tokens": 8192, "n": 4096, "k": 14336, "bias": False, "act": "none", "residual": True},
        # decode batch, 32 query and 8 key heads behind a 6144-channel QKV projection
        {"name": "qk_decode_16", "op": "qk", "tokens": 16, "hq": 32, "hk": 8, "d": 128, "rot": 128, "inter": False, "gamma": True},
        # long prompt on the same heads
        {"name": "qk_prefill_16384", "op": "qk", "tokens": 16384, "hq": 32, "hk": 8, "d": 128, "rot": 128, "inter": False, "gamma": True},
        # heads of 80 with 32 rotated channels in neighbouring pairs
        {"name": "qk_partial_1021", "op": "qk", "tokens": 1021, "hq": 6, "hk": 3, "d": 80, "rot": 32, "inter": True, "gamma": False},
        # one decode step of 64 sequences
        {"name": "write_decode_64", "op": "write", "tokens": 64, "h": 8, "d": 128, "page": 16, "pad": 0},
        # a long prompt, some padding tokens among it
        {"name": "write_prefill_16384", "op": "write", "tokens": 16384, "h": 8, "d": 128, "page": 64, "pad": 37},
        # one short sequence
        {"name": "read_one_100", "op": "read", "seqs": 1, "mean": 100, "h": 8, "d": 128, "page": 16, "pad": 0},
        # ragged batch, odd heads, pages that end inside sequences, rows behind the last one
        {"name": "read_ragged_7", "op": "read", "seqs": 7, "mean": 300, "h": 5, "d": 96, "page": 24, "pad": 5},
        # long contexts
        {"name": "read_long_32", "op": "read", "seqs": 32, "mean": 4096, "h": 8, "d": 128, "page": 64, "pad": 0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "qk", "write", "read"])
    if op == "linear":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 8, 16384), 8 * _log(rng, 1, 2048)
            if m * n * k <= 8192 * 4096 * 14336:
                break
        return {"op": op, "tokens": m, "n": n, "k": k, "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "residual": rng.random() < 0.5}
    d = rng.choice([64, 80, 96, 128, 128, 192, 256, 8 * rng.randint(2, 32)])
    if op == "qk":
        inter = rng.random() < 0.5
        step = 8 if inter else 16
        rot = d // step * step if rng.random() < 0.5 else step * rng.randint(1, d // step)
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 7, 8])
        tokens = _log(rng, 1, max(1, min(16384, 16384 * 40 * 128 // ((hq + hk) * d))))
        return {"op": op, "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": rot, "inter": inter, "gamma": rng.random() < 0.7}
    h = rng.choice([1, 2, 3, 4, 5, 8, 16])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128, 256])
    if op == "write":
        tokens = _log(rng, 1, max(1, min(16384, 16384 * 8 * 128 // (h * d))))
        return {"op": op, "tokens": tokens, "h": h, "d": d, "page": page, "pad": rng.choice([0, rng.randint(0, tokens)])}
    total = _log(rng, 1, max(1, min(131072, 131072 * 8 * 128 // (h * d))))
    seqs = min(total, _log(rng, 1, 128))
    return {"op": op, "seqs": seqs, "mean": max(1, total // seqs), "h": h, "d": d, "page": page, "pad": rng.choice([0, 3])}


def _table(rot, device):
    """cos, then sin, of every position: angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=F64, device=device) / rot)
    ang = torch.arange(MAX_POSITION, dtype=F64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(F32)


def _lengths(case, seed):
    """Sequence lengths of a ragged batch (an empty one and a single token among them), the same total every time."""
    b, mean = case["seqs"], case["mean"]
    r = random.Random(seed * 7919 + b)
    if b == 1:
        return [mean]
    cuts = sorted(r.randint(0, b * mean) for _ in range(b - 1))
    return [hi - lo for lo, hi in zip([0] + cuts, cuts + [b * mean])]


def _quantise(x):
    a = x.to(F32).abs().amax(-1).clamp(min=AMAX_FLOOR)
    return (x.to(F32) * E4M3_MAX / a[..., None]).to(E4M3), a / E4M3_MAX


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(1000003 * seed + 17)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=F32) * scale).to(BF16)

    s = dict(case)
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        s["x"] = normal(m, k)
        s["W"] = normal(n, k, scale=k ** -0.5)
        s["bias_v"] = normal(n) if case["bias"] else None
        s["res_v"] = normal(m, n) if case["residual"] else None
        return s
    d = case["d"]
    if case["op"] == "qk":
        t, hq, hk = case["tokens"], case["hq"], case["hk"]
        # what the fused QKV projection writes: q, k and v side by side
        qkv = normal(t, (hq + 2 * hk) * d).view(t, hq + 2 * hk, d)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        s["gq"] = 1 + normal(d, scale=0.1) if case["gamma"] else None
        s["gk"] = 1 + normal(d, scale=0.1) if case["gamma"] else None
        s["positions"] = torch.randint(0, MAX_POSITION, (t,), generator=g, device=dev)
        s["table"] = _table(case["rot"], dev)
        return s
    h, page = case["h"], case["page"]
    if case["op"] == "write":
        t = case["tokens"]
        pages = -(-t // page) + 3
        kv = normal(t, 3 * h, d)   # queries in front, as the projection writes them
        s["k"], s["v"] = kv[:, h:2 * h], kv[:, 2 * h:]
        slots = torch.randperm(pages * page, generator=g, device=dev)[:t]
        if case["pad"]:
            slots[torch.randperm(t, generator=g, device=dev)[:case["pad"]]] = -1
        s["slots"] = slots
        s["cache"] = _cache(pages, page, h, d, dev)
        return s
    lens = _lengths(case, seed)
    used = [-(-x // page) for x in lens]
    pages = sum(used) + 2
    s["cache"] = _cache(pages, page, h, d, dev)
    for codes, scales in (s["cache"][:2], s["cache"][2:]):
        q, a = _quantise(normal(pages, page, h, d))
        codes.view(torch.uint8).copy_(q.view(torch.uint8))
        scales.copy_(a)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(max(used), 1)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    s["pages"] = table
    ends = [0]
    for x in lens:
        ends.append(ends[-1] + x)
    s["cu"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    s["total"] = ends[-1] + case["pad"]
    return s


def _cache(pages, page, h, d, dev):
    """Codes and scales of the keys, then of the values."""
    made = []
    for _ in range(2):
        made += [torch.zeros(pages, page, h, d, dtype=torch.uint8, device=dev).view(E4M3),
                 torch.zeros(pages, page, h, dtype=F32, device=dev)]
    return made


# ------------------------------------------------------------------ the plain forms

def _activation(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear(s):
    z = s["x"].to(F32) @ s["W"].to(F32).t()
    if s["bias_v"] is not None:
        z = z + s["bias_v"].to(F32)
    z = _activation(z, s["act"])
    if s["res_v"] is not None:
        z = z + s["res_v"].to(F32)
    return z.to(BF16)


def _plain_rotate(x, gamma, cos, sin, inter):
    x = x.to(F32)
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if gamma is not None:
        n = n * gamma.to(F32)
    half = cos.shape[-1]
    rot, rest = n[..., :2 * half], n[..., 2 * half:]
    cos, sin = cos[:, None], sin[:, None]
    if inter:
        a, b = rot[..., 0::2], rot[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(BF16)


def _plain_qk(s):
    cs = s["table"][s["positions"]]
    half = s["rot"] // 2
    cos, sin = cs[:, :half], cs[:, half:]
    return (_plain_rotate(s["q"], s["gq"], cos, sin, s["inter"]), _plain_rotate(s["k"], s["gk"], cos, sin, s["inter"]))


def _plain_write(s):
    kept = s["slots"] >= 0
    slots = s["slots"][kept]
    for x, codes, scales in ((s["k"], s["cache"][0], s["cache"][1]), (s["v"], s["cache"][2], s["cache"][3])):
        q, a = _quantise(x[kept])
        codes.view(torch.uint8).flatten(0, 1)[slots] = q.view(torch.uint8)
        scales.flatten(0, 1)[slots] = a
    return list(s["cache"])


def _plain_read(s):
    i = torch.arange(s["total"], device=s["cu"].device, dtype=torch.int32)
    held = i < s["cu"][-1]
    b = torch.searchsorted(s["cu"][1:].contiguous(), i, right=True).clamp(max=s["cu"].numel() - 2)
    pos = torch.where(held, i - s["cu"][b], 0).long()
    page = torch.where(held, s["pages"][b, pos // s["page"]], 0).long()
    out = []
    for codes, scales in (s["cache"][:2], s["cache"][2:]):
        c = codes.view(torch.uint8)[page, pos % s["page"]].view(E4M3).to(F32)
        x = c * scales[page, pos % s["page"]][..., None]
        out.append(torch.where(held[:, None, None], x, 0).to(BF16))
    return out


def run(s):
    if own:
        import kernel_benchmarking_b200 as kb
        if s["op"] == "linear":
            return kb.linear(s["x"], s["W"], s["bias_v"], activation=None if s["act"] == "none" else s["act"], residual=s["res_v"])
        if s["op"] == "qk":
            return kb.qk_norm_rope(s["q"], s["k"], s["gq"], s["gk"], s["table"], s["positions"], EPS, interleaved=s["inter"])
        if s["op"] == "write":
            kb.kv_cache_write(s["k"], s["v"], s["slots"], *s["cache"])
            return list(s["cache"])
        return list(kb.kv_cache_read(*s["cache"], s["pages"], s["cu"], s["total"]))
    return {"linear": _plain_linear, "qk": _plain_qk, "write": _plain_write, "read": _plain_read}[s["op"]](s)


def work(case):
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        b = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        return {"bytes": 2 * b, "flops": 2 * m * n * k}
    d = case["d"]
    if case["op"] == "qk":
        t, rows = case["tokens"], case["tokens"] * (case["hq"] + case["hk"])
        return {"bytes": 4 * rows * d + 4 * t * case["rot"] + 8 * t + (4 * d if case["gamma"] else 0), "flops": 10 * rows * d}
    if case["op"] == "write":
        rows = 2 * (case["tokens"] - case["pad"]) * case["h"]
        return {"bytes": rows * (2 * d + d + 4) + 8 * case["tokens"], "flops": 4 * rows * d}
    total = case["seqs"] * case["mean"]
    rows = 2 * total * case["h"]
    return {"bytes": rows * (d + 4 + 2 * d) + 4 * (total // case["page"]) + 4 * case["pad"] * case["h"] * d, "flops": 2 * rows * d}


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", s["x"].double(), s["W"].double())
        if s["bias_v"] is not None:
            z += s["bias_v"].double()[None, :]
        if case["act"] == "relu":
            z = torch.where(z > 0, z, torch.zeros((), dtype=F64, device=z.device))
        elif case["act"] == "gelu":   # z times the normal distribution's area below z
            z = z * torch.special.erfc(-z / 2.0 ** 0.5) / 2
        elif case["act"] == "gelu_tanh":   # (1 + tanh u) / 2 is the logistic function of 2 u
            z = z * torch.sigmoid((8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        return z + s["res_v"].double() if s["res_v"] is not None else z
    if case["op"] == "qk":
        t, half = case["tokens"], case["rot"] // 2
        turn = s["table"][s["positions"]].double()
        turn = torch.complex(turn[:, :half], turn[:, half:])[:, None, :]
        out = []
        for x, gamma in ((s["q"], s["gq"]), (s["k"], s["gk"])):
            y = x.double()
            y = y / ((y ** 2).sum(-1, keepdim=True) / case["d"] + EPS).sqrt()
            y = y * gamma.double() if gamma is not None else y
            pairs = y[..., :2 * half]
            # a rotated pair is a complex number times its turn
            z = (pairs.reshape(t, -1, half, 2) if case["inter"] else pairs.reshape(t, -1, 2, half).transpose(2, 3)).contiguous()
            z = torch.view_as_real(torch.view_as_complex(z) * turn)
            z = z if case["inter"] else z.transpose(2, 3)
            out.append(torch.cat([z.reshape(t, -1, 2 * half), y[..., 2 * half:]], dim=-1))
        return tuple(out)
    if case["op"] == "write":
        out = [c.to(F32).double() if c.dtype == E4M3 else c.double() for c in s["cache"]]
        at = [(t, x) for t, x in enumerate(s["slots"].tolist()) if x >= 0]
        src = torch.tensor([t for t, _ in at], dtype=torch.long, device=s["k"].device)
        dst = torch.tensor([x for _, x in at], dtype=torch.long, device=s["k"].device)
        for i, x in ((0, s["k"]), (2, s["v"])):
            rows = x.double().index_select(0, src)
            top = torch.linalg.vector_norm(rows, ord=math.inf, dim=-1).clamp(min=AMAX_FLOOR)
            out[i].view(-1, case["h"], case["d"]).index_copy_(0, dst, E4M3_MAX * rows / top[..., None])
            out[i + 1].view(-1, case["h"]).index_copy_(0, dst, top / E4M3_MAX)
        return out
    ends = s["cu"].tolist()
    out = []
    for codes, scales in (s["cache"][:2], s["cache"][2:]):
        parts = []
        for b in range(case["seqs"]):
            n = ends[b + 1] - ends[b]
            mine = s["pages"][b, :-(-n // case["page"])].long() if n else s["pages"][b, :0].long()
            c = codes.view(torch.uint8)[mine].view(E4M3).to(F32).double() * scales[mine].double()[..., None]
            parts.append(c.flatten(0, 1)[:n])
        parts.append(torch.zeros(case["pad"], case["h"], case["d"], dtype=F64, device=s["cu"].device))
        out.append(torch.cat(parts))
    return out
