"""The attention side of a decoder layer, around the MoE block: norms and rotary positions of
queries and keys, a cache of keys and values in 4, 8 or 16 bits, attention of single tokens over
that cache, and causal attention over packed prompts.

`own` chooses between the plain form (elementary torch operations) and the package's entry points.
Head counts and widths are GPT-OSS's (64 query heads on 8 of 64), Qwen3's (32 on 4 of 128, with
norms) and Coder-Next's (16 on 2 of 256, a quarter of each head rotated), and generic ones in draw().
"""
import math
import os
import sys

import torch

own = False
DEVICE = "cuda"

GPT_OSS = {"q_heads": 64, "kv_heads": 8, "dim": 64}
QWEN3 = {"q_heads": 32, "kv_heads": 4, "dim": 128}
CODER = {"q_heads": 16, "kv_heads": 2, "dim": 256}

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one sequence: a decode step's rotation, base frequencies stretched for long contexts
        dict(GPT_OSS, name="rope_step", op="rope", tokens=1, src="f32", dst="bf16", norm=False, rotary=64,
             layout="half", base=150000.0, scaling="yarn_exact", factor=32.0, orig=4096, far=131072),
        # a prompt with norms of queries and keys
        dict(QWEN3, name="rope_prompt_4096", op="rope", tokens=4096, src="f32", dst="bf16", norm=True, rotary=128,
             layout="half", base=1e6, scaling="none", factor=1.0, orig=0, far=4096),
        # part of each head, neighbouring pairs, out of a fused projection, far positions
        dict(CODER, name="rope_partial_777", op="rope", tokens=777, src="bf16", dst="f16", norm=True, rotary=64,
             layout="interleaved", base=1e7, scaling="linear", factor=4.0, orig=0, far=1000000),
        # 64 sequences step together: one token each into its own page
        dict(GPT_OSS, name="cache_step_64", op="cache", tokens=64, src="f32", format="mxfp4", page=64, scattered=True),
        # a long prompt goes into the cache and comes back for the next part of it
        dict(QWEN3, name="cache_prompt_8191", op="cache", tokens=8191, src="bf16", format="mxint8", page=256,
             scattered=False),
        # one user, a short conversation: a layer with a window and sinks
        dict(GPT_OSS, name="decode_one_700", op="decode", seqs=1, least=700, most=700, src="bf16", format="mxfp4",
             page=64, window=128, sinks=True),
        # a full serving batch, lengths from nothing (a slot without a request) to 24000
        dict(QWEN3, name="decode_batch_32", op="decode", seqs=32, least=0, most=24000, src="bf16", format="mxfp4",
             page=256, window=0, sinks=False),
        # one long document
        dict(CODER, name="decode_one_100001", op="decode", seqs=1, least=100001, most=100001, src="f16",
             format="mxint8", page=256, window=0, sinks=False),
        # a short question
        dict(GPT_OSS, name="prompt_61", op="prompt", seqs=1, least=61, most=61, past=0, src="bf16", window=128,
             sinks=True),
        # prompts of different lengths packed, one layer with a window and sinks
        dict(GPT_OSS, name="prompt_packed_window", op="prompt", seqs=9, least=1, most=2048, past=0, src="bf16",
             window=128, sinks=True),
        # the second parts of prompts whose first parts are keys and values already
        dict(CODER, name="prompt_packed_past", op="prompt", seqs=3, least=300, most=1500, past=2000, src="f16",
             window=0, sinks=False),
        # one long prompt
        dict(QWEN3, name="prompt_8192", op="prompt", seqs=1, least=8192, most=8192, past=0, src="bf16", window=0,
             sinks=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: an operator, a shape (a configured one or a generic one) and sizes over the whole range."""
    if rng.random() < 0.5:
        shape = dict(rng.choice([GPT_OSS, QWEN3, CODER]))
    else:
        kv = rng.choice([1, 2, 3, 4, 5, 8])
        shape = {"kv_heads": kv, "q_heads": kv * rng.choice([1, 2, 3, 4, 6, 8, 12, 16]), "dim": rng.choice([64, 128, 256])}
    op = rng.choice(["rope", "cache", "decode", "prompt"])
    if op == "rope":
        d = shape["dim"]
        # at most twice the bytes of the longest listed prompt
        most = min(4096, 28000000 // ((shape["q_heads"] + shape["kv_heads"]) * d))
        return dict(shape, op=op, tokens=_log_int(rng, 1, most), src=rng.choice(["f32", "f32", "f16", "bf16"]),
                    dst=rng.choice(["f16", "bf16", "f32"]), norm=rng.random() < 0.6,
                    rotary=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["half", "half", "interleaved"]),
                    base=float(rng.choice([10000, 150000, 1000000])),
                    scaling=rng.choice(["none", "linear", "yarn", "yarn_exact"]), factor=float(rng.choice([2, 8, 32])),
                    orig=4096, far=_log_int(rng, 4096, 1000000))
    fmt = rng.choice(["mxfp4", "mxfp4", "mxint8", "f16"])
    page = rng.choice([64, 128, 256])
    if op == "cache":
        return dict(shape, op=op, tokens=_log_int(rng, 1, 8192), src=rng.choice(["f32", "f16", "bf16"]), format=fmt,
                    page=page, scattered=rng.random() < 0.5)
    window, sinks = rng.choice([0, 0, 128, 1000]), rng.random() < 0.4
    if op == "decode":
        seqs = _log_int(rng, 1, 64)
        # at most as many cached bytes as the longest listed batch
        bits = {"mxfp4": 4, "mxint8": 8, "f16": 16}[fmt]
        room = 32 * 12000 * 4 * 128 * 4 // (shape["kv_heads"] * shape["dim"] * bits)
        most = _log_int(rng, 16, max(17, min(65536, room // seqs)))
        return dict(shape, op=op, seqs=seqs, least=rng.choice([0, 1, most // 2, most]), most=most,
                    src=rng.choice(["f16", "bf16"]), format=fmt, page=page, window=window, sinks=sinks)
    seqs = _log_int(rng, 1, 32)
    # scores of the longest listed prompt: 32 heads of 128 over 8192 * 8192 / 2 pairs
    area = 32 * 128 * 8192 * 8192 // (shape["q_heads"] * shape["dim"])
    rows = 50000000 // ((shape["q_heads"] + 2 * shape["kv_heads"]) * shape["dim"])
    most = _log_int(rng, 1, max(1, min(8192, int(math.sqrt(area / (3 * seqs))), rows // seqs)))
    return dict(shape, op=op, seqs=seqs, least=rng.choice([1, most, (most + 1) // 2]), most=most,
                past=rng.choice([0, 0, most]), src=rng.choice(["f16", "bf16"]), window=window, sinks=sinks)


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed, *ids):
    for i in ids:
        seed = (seed * 1000003 + i + 1) % (1 << 62)
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _keys(shape, g):
    """Projected keys: about N(0, 1), one channel in 16 four times as wide."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    x[..., 5::16] *= 4.0
    return x


def _lengths(case):
    """The sequences' lengths: the longest first, the others spread over the range."""
    n, lo, hi = case["seqs"], case["least"], case["most"]
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((5 * i + 3) % n) // (n - 1) if i else hi for i in range(n)]


def _rope_inputs(case, seed):
    g = _gen(seed)
    T, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    # one row a token: queries, keys, values, as a fused projection leaves them
    qkv = _keys((T, hq + 2 * hk, d), g).to(TYPES[case["src"]])
    start = int(torch.randint(0, max(1, case["far"] - T), (1,), generator=g, device=DEVICE))
    pos = (start + torch.arange(T, device=DEVICE)).to(torch.int32)
    w = [1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE) for _ in range(2)] if case["norm"] else [None, None]
    return {"qkv": qkv, "pos": pos, "q_norm": w[0], "k_norm": w[1]}


def _frequencies(case):
    """Radians a position turns each pair by, and the factor on cosine and sine (YaRN: Peng et al., 2023)."""
    n, base = case["rotary"], case["base"]
    f = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if case["scaling"] == "linear":
        return [v / case["factor"] for v in f], 1.0
    if case["scaling"] in ("yarn", "yarn_exact"):
        def pair(turns):
            return n * math.log(case["orig"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low, high = pair(32.0), pair(1.0)
        if case["scaling"] == "yarn":
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0.0), min(high, n - 1.0)
        if low == high:
            high += 0.001
        ramp = [min(1.0, max(0.0, (i - low) / (high - low))) for i in range(n // 2)]
        return [v / case["factor"] * r + v * (1.0 - r) for v, r in zip(f, ramp)], 0.1 * math.log(case["factor"]) + 1.0
    return f, 1.0


def _cache_inputs(case, seed):
    g = _gen(seed)
    T, hk, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    k = _keys((T, hk, d), g).to(TYPES[case["src"]])
    v = torch.randn((T, hk, d), generator=g, device=DEVICE).to(TYPES[case["src"]])
    if case["scattered"]:  # a token a page, anywhere in it
        pages = T
        slots = torch.randperm(pages, generator=g, device=DEVICE) * page
        slots = slots + torch.randint(0, page, (T,), generator=g, device=DEVICE)
    else:  # one sequence over pages in any order
        pages = (T + page - 1) // page
        order = torch.randperm(pages, generator=g, device=DEVICE)
        t = torch.arange(T, device=DEVICE)
        slots = order[t // page] * page + t % page
    return {"k": k, "v": v, "slots": slots.to(torch.int32), "pages": pages}


def _decode_inputs(case, seed):
    """Queries, lengths and pages; the cached keys and values of sequence i come from _history(case, seed, i)."""
    g = _gen(seed)
    n, page = case["seqs"], case["page"]
    lens = _lengths(case)
    counts = [(L + page - 1) // page for L in lens]
    order = torch.randperm(sum(counts) + 1, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros((n, max(1, max(counts))), dtype=torch.int32, device=DEVICE)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    q = torch.randn((n, case["q_heads"], case["dim"]), generator=g, device=DEVICE).to(TYPES[case["src"]])
    sinks = torch.randn(case["q_heads"], generator=g, device=DEVICE) if case["sinks"] else None
    return {"q": q, "sinks": sinks, "lens": lens, "table": table, "pages": sum(counts) + 1,
            "len": torch.tensor(lens, dtype=torch.int32, device=DEVICE)}


def _history(case, seed, i, n):
    g = _gen(seed, i)
    shape = (n, case["kv_heads"], case["dim"])
    return _keys(shape, g), torch.randn(shape, generator=g, device=DEVICE)


def _slots(case, s, i):
    t = torch.arange(s["lens"][i], device=DEVICE)
    return s["table"][i][t // case["page"]].long() * case["page"] + t % case["page"]


def _prompt_inputs(case, seed):
    g = _gen(seed)
    hq, hk, d, t = case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["src"]]
    lens = _lengths(case)
    cu_q, cu_k = [0], [0]
    for L in lens:
        cu_q.append(cu_q[-1] + L)
        cu_k.append(cu_k[-1] + L + case["past"])
    s = {"q": torch.randn((cu_q[-1], hq, d), generator=g, device=DEVICE).to(t), "k": _keys((cu_k[-1], hk, d), g).to(t),
         "v": torch.randn((cu_k[-1], hk, d), generator=g, device=DEVICE).to(t),
         "sinks": torch.randn(hq, generator=g, device=DEVICE) if case["sinks"] else None, "lens_q": cu_q, "lens_k": cu_k}
    for name, c in (("cu_q", cu_q), ("cu_k", cu_k)):
        s[name] = torch.tensor(c, dtype=torch.int32, device=DEVICE)
    return s


# ---- the plain form ------------------------------------------------------------------------------
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _quantise(fmt, x):
    """Codes (whole numbers as int8) and exponents [.., dim / 32] of the blocks of 32; f16: the values themselves."""
    if fmt == "f16":
        return x.float().clamp(-65504.0, 65504.0).half(), None
    b = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))  # m in [0.5, 1): amax = 2m * 2^(e-1)
    if fmt == "mxfp4":
        e = e - 3 + (m > 0.875).int()
    else:
        e = e - 7 + (m >= 0.99609375).int()
    e = torch.where(m == 0, -16, e).clamp(-16, 13 if fmt == "mxfp4" else 9)
    y = torch.ldexp(b, -e[..., None])
    if fmt == "mxint8":
        return y.round().clamp(-127, 127).to(torch.int8).flatten(-2), e.to(torch.int8)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    return torch.where(y < 0, -code, code).to(torch.int8).flatten(-2), e.to(torch.int8)


def _values(fmt, code, e):
    """What codes and exponents stand for, in float32."""
    if fmt == "f16":
        return code.float()
    b = code.unflatten(-1, (-1, 32))
    if fmt == "mxfp4":
        v = torch.tensor(FP4, device=DEVICE)[b.abs().int()] * torch.sign(b.float())
    else:
        v = b.float()
    return torch.ldexp(v, e.int()[..., None]).flatten(-2)


def _plain_rope(s):
    case, x = s["case"], s["qkv"]
    hq, hk, n = case["q_heads"], case["kv_heads"], case["rotary"]
    f, mul = _frequencies(case)
    angle = s["pos"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEVICE)
    cos, sin = (torch.cos(angle) * mul).float()[:, None], (torch.sin(angle) * mul).float()[:, None]
    out = []
    for y, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hk], s["k_norm"])):
        y = y.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        r = y[..., :n]
        a, b = (r[..., :n // 2], r[..., n // 2:]) if case["layout"] == "half" else (r[..., 0::2], r[..., 1::2])
        c, d = a * cos - b * sin, b * cos + a * sin
        r = torch.cat([c, d], -1) if case["layout"] == "half" else torch.stack([c, d], -1).flatten(-2)
        out.append(torch.cat([r, y[..., n:]], -1).to(TYPES[case["dst"]]))
    return out


def _plain_cache(s):
    fmt, slots = s["case"]["format"], s["slots"].long()
    out = []
    for name in ("k", "v"):
        code, e = _quantise(fmt, s[name])
        s[name + "_code"][slots] = code
        if e is not None:
            s[name + "_exp"][slots] = e
        out.append(_values(fmt, s[name + "_code"][slots], None if e is None else s[name + "_exp"][slots]).half())
    return out


def _attend(q, k, v, scale, sinks, allowed):
    """softmax(q k^T * scale) v of the heads [h, g, rows, dim] that share keys [h, keys, dim]; `allowed`: rows x keys
    or None; a sink is one more score with no value; rows with nothing allowed are zero."""
    x = torch.matmul(q, k.transpose(-1, -2)[:, None]) * scale
    if allowed is not None:
        x = x.masked_fill(~allowed, -math.inf)
    m = x.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    if sinks is not None:
        z = z + torch.exp(sinks - m)
    return torch.matmul(p, v[:, None]) / torch.where(z == 0, torch.ones_like(z), z)


def _plain_decode(s):
    case, kind = s["case"], s["q"].dtype
    hk, d = case["kv_heads"], case["dim"]
    out = torch.zeros_like(s["q"])
    sinks = None if s["sinks"] is None else s["sinks"].view(hk, -1, 1, 1)
    for i, n in enumerate(s["lens"]):
        if n == 0:
            continue
        slots = _slots(case, s, i)
        if case["window"]:
            slots = slots[-case["window"]:]
        k, v = (_values(case["format"], s[a + "_code"][slots], s[a + "_exp"][slots] if s[a + "_exp"] is not None else None)
                .transpose(0, 1) for a in ("k", "v"))
        q = s["q"][i].float().view(hk, -1, 1, d)
        out[i] = _attend(q, k, v, d ** -0.5, sinks, None).reshape(-1, d).to(kind)
    return out


def _allowed(case, n, m):
    """Which of m keys each of the last n positions sees."""
    i = torch.arange(m - n, m, device=DEVICE)[:, None]
    j = torch.arange(m, device=DEVICE)
    a = j <= i
    return a & (i - j < case["window"]) if case["window"] else a


def _prompts(s, kind, sinks):
    """Attention of each packed sequence in `kind`, one key head at a time; yields (rows, query heads, result)."""
    case = s["case"]
    hk, d = case["kv_heads"], case["dim"]
    group = case["q_heads"] // hk
    for i in range(case["seqs"]):
        a, b, c, e = s["lens_q"][i], s["lens_q"][i + 1], s["lens_k"][i], s["lens_k"][i + 1]
        if a == b:
            continue
        allowed = _allowed(case, b - a, e - c)
        for h in range(hk):
            q = s["q"][a:b, h * group:(h + 1) * group].to(kind).permute(1, 0, 2)[None]
            sk = None if sinks is None else sinks.to(kind)[h * group:(h + 1) * group].view(1, group, 1, 1)
            y = _attend(q, s["k"][c:e, h].to(kind)[None], s["v"][c:e, h].to(kind)[None], d ** -0.5, sk, allowed)
            yield slice(a, b), slice(h * group, (h + 1) * group), y[0].permute(1, 0, 2)


def _plain_prompt(s):
    out = torch.zeros_like(s["q"])
    for rows, heads, y in _prompts(s, torch.float32, s["sinks"]):
        out[rows, heads] = y.to(out.dtype)
    return out


# ---- the package's entry points ------------------------------------------------------------------
_ctx = None


def _package():
    root = os.path.join(os.getcwd(), "moe-stream_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import moe_rocm

    return moe_rocm


def _context():
    """The program's one context, on torch's stream."""
    global _ctx
    if _ctx is None:
        _ctx = _package().Context(0)
    _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def _heads(x):
    M = _package()
    kind = {torch.float32: M.F32, torch.float16: M.F16, torch.bfloat16: M.BF16}[x.dtype]
    return M.Heads(x.data_ptr(), x.shape[1], kind, x.stride(0), x.stride(1))


class _Cache:
    """A cache handle that goes with the state."""

    def __init__(self, case, pages):
        M = _package()
        fmt = {"mxfp4": M.KV_MXFP4, "mxint8": M.KV_MXINT8, "f16": M.KV_F16}[case["format"]]
        self.kv = M.KvCache(_context(), fmt, pages, case["page"], case["kv_heads"], case["dim"])

    def __del__(self):
        try:
            self.kv.close()
        except (AttributeError, TypeError):  # half-made, or at the interpreter's end
            pass


class _Rope:
    def __init__(self, case):
        M = _package()
        self.rope = M.Rope(
            _context(), case["dim"], rotary_dim=case["rotary"], base=case["base"],
            layout=M.ROPE_HALF if case["layout"] == "half" else M.ROPE_INTERLEAVED,
            scaling={"none": M.ROPE_PLAIN, "linear": M.ROPE_LINEAR, "yarn": M.ROPE_YARN,
                     "yarn_exact": M.ROPE_YARN_EXACT}[case["scaling"]],
            factor=case["factor"], orig_context=case["orig"])

    def __del__(self):
        try:
            self.rope.close()
        except (AttributeError, TypeError):
            pass


def prepare(case, seed):
    op = case["op"]
    if op == "rope":
        s = _rope_inputs(case, seed)
        if own:
            s["rope"] = _Rope(case)
            T, d, t = case["tokens"], case["dim"], TYPES[case["dst"]]
            s["out"] = [torch.empty((T, case[h], d), dtype=t, device=DEVICE) for h in ("q_heads", "kv_heads")]
    elif op == "prompt":
        s = _prompt_inputs(case, seed)
        if own:
            s["out"] = torch.zeros_like(s["q"])
    else:
        s = _cache_inputs(case, seed) if op == "cache" else _decode_inputs(case, seed)
        hk, d, fmt, n = case["kv_heads"], case["dim"], case["format"], s["pages"] * case["page"]
        if own:
            s["cache"] = _Cache(case, s["pages"])
        else:
            for a in ("k", "v"):
                s[a + "_code"] = torch.zeros((n, hk, d), dtype=torch.float16 if fmt == "f16" else torch.int8, device=DEVICE)
                s[a + "_exp"] = None if fmt == "f16" else torch.zeros((n, hk, d // 32), dtype=torch.int8, device=DEVICE)
        if op == "cache" and own:
            s["out"] = [torch.empty((case["tokens"], hk, d), dtype=torch.float16, device=DEVICE) for _ in range(2)]
        if op == "decode":
            if own:
                s["out"] = torch.zeros_like(s["q"])
            for i, n in enumerate(s["lens"]):
                if n == 0:
                    continue
                slots = _slots(case, s, i)
                kv = _history(case, seed, i, n)
                if own:
                    slots = slots.to(torch.int32)
                    s["cache"].kv.write(_heads(kv[0]), _heads(kv[1]), n, slots.data_ptr())
                    continue
                for a, x in zip(("k", "v"), kv):
                    code, e = _quantise(fmt, x)
                    s[a + "_code"][slots] = code
                    if e is not None:
                        s[a + "_exp"][slots] = e
    s["case"] = case
    torch.cuda.synchronize()
    return s


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"rope": _plain_rope, "cache": _plain_cache, "decode": _plain_decode, "prompt": _plain_prompt}[op](s)
    M, ctx = _package(), _context()
    if op == "rope":
        hq, hk = case["q_heads"], case["kv_heads"]
        M.qk_norm_rope(ctx, s["rope"].rope, _heads(s["qkv"][:, :hq]), _heads(s["qkv"][:, hq:hq + hk]),
                       case["tokens"], s["pos"].data_ptr(), _heads(s["out"][0]), _heads(s["out"][1]), eps=1e-6,
                       q_norm=s["q_norm"].data_ptr() if case["norm"] else None,
                       k_norm=s["k_norm"].data_ptr() if case["norm"] else None)
    elif op == "cache":
        kv, slots = s["cache"].kv, s["slots"].data_ptr()
        kv.write(_heads(s["k"]), _heads(s["v"]), case["tokens"], slots)
        kv.read(case["tokens"], slots, _heads(s["out"][0]), _heads(s["out"][1]))
    elif op == "decode":
        s["cache"].kv.attend(_heads(s["q"]), case["seqs"], s["len"].data_ptr(), s["table"].data_ptr(),
                             s["table"].shape[1], _heads(s["out"]), window=case["window"],
                             sinks=s["sinks"].data_ptr() if case["sinks"] else None)
    else:
        M.attn_prefill(ctx, case["dim"], _heads(s["q"]), _heads(s["k"]), _heads(s["v"]), s["q"].shape[0],
                       s["k"].shape[0], case["seqs"], s["cu_q"].data_ptr(), s["cu_k"].data_ptr(), _heads(s["out"]),
                       window=case["window"], sinks=s["sinks"].data_ptr() if case["sinks"] else None)
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    hq, hk, d, op = case["q_heads"], case["kv_heads"], case["dim"], case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if op == "rope":
        n = case["tokens"] * (hq + hk) * d
        return {"bytes": n * (size[case["src"]] + size[case["dst"]]) + 4 * case["tokens"], "flops": 8 * n}
    # bytes of a cached token: keys and values, and the blocks' exponents
    token = 0
    if op != "prompt":
        bits = {"mxfp4": 4, "mxint8": 8, "f16": 16}[case["format"]]
        token = 2 * hk * (d * bits // 8 + (0 if bits == 16 else d // 32))
    if op == "cache":
        n = case["tokens"] * 2 * hk * d
        return {"bytes": n * (size[case["src"]] + 2) + 2 * token * case["tokens"], "flops": 4 * n}
    lens = _lengths(case)
    if op == "decode":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        return {"bytes": seen * token + 4 * case["seqs"] * hq * d, "flops": 4 * seen * hq * d}
    pairs = 0
    for n in lens:
        m, w = n + case["past"], case["window"]
        for lo, hi in ((m - n + 1, m),):  # the i-th position of a sequence sees min(i, window) keys
            if w and hi > w:
                part = max(0, min(hi, w) - lo + 1)
                pairs += part * (lo + min(hi, w)) // 2 if part else 0
                pairs += (hi - max(lo, w + 1) + 1) * w
            else:
                pairs += (hi - lo + 1) * (lo + hi) // 2
    rows = sum(lens)
    nbytes = 2 * (2 * rows * hq * d + 2 * (rows + case["seqs"] * case["past"]) * hk * d)
    return {"bytes": nbytes, "flops": 4 * pairs * hq * d}


# ---- the same in 64 bits -------------------------------------------------------------------------
def _nearest(fmt, x):
    """The values a cache holds for x, in 64 bits, by distance to every value of the format; a tie goes to the even code."""
    x = x.double()
    if fmt == "f16":
        return x.clamp(-65504.0, 65504.0).half().double()
    grid = torch.tensor(FP4 if fmt == "mxfp4" else range(128), dtype=torch.float64, device=DEVICE)
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    # the least scale whose largest value is the nearest one to the block's largest magnitude
    limit, low, high = (7.0, -16, 13) if fmt == "mxfp4" else (127.5, -16, 9)
    scale = torch.full_like(top, 2.0 ** low)
    for e in range(low, high):
        over = top > limit * 2.0 ** e if fmt == "mxfp4" else top >= limit * 2.0 ** e
        scale = torch.where(over, torch.full_like(top, 2.0 ** (e + 1)), scale)
    y = b / scale
    a = y.abs().clamp(max=float(grid[-1]))
    at = torch.searchsorted(grid, a.contiguous()).clamp(1, len(grid) - 1)
    lo, hi = grid[at - 1], grid[at]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (at % 2 == 0))
    return (torch.where(up, hi, lo) * torch.sign(y) * scale).flatten(-2)


def _exact_rope(case, seed):
    s = _rope_inputs(case, seed)
    n, hq, hk = case["rotary"], case["q_heads"], case["kv_heads"]
    f, mul = _frequencies(case)
    turn = torch.polar(torch.full((), mul, dtype=torch.float64, device=DEVICE),
                       s["pos"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEVICE))[:, None]
    out = []
    for y, w in ((s["qkv"][:, :hq].double(), s["q_norm"]), (s["qkv"][:, hq:hq + hk].double(), s["k_norm"])):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()
        half = case["layout"] == "half"
        first, second = (slice(0, n // 2), slice(n // 2, n)) if half else (slice(0, n, 2), slice(1, n, 2))
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out


def exact(case, seed):
    op = case["op"]
    if op == "rope":
        return _exact_rope(case, seed)
    if op == "cache":
        s = _cache_inputs(case, seed)
        return [_nearest(case["format"], s["k"]), _nearest(case["format"], s["v"])]
    hk, d, w = case["kv_heads"], case["dim"], case["window"]
    group = case["q_heads"] // hk
    if op == "decode":
        s = _decode_inputs(case, seed)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for i, n in enumerate(s["lens"]):
            if n == 0:
                continue
            k, v = _history(case, seed, i, n)
            first = max(0, n - w) if w else 0
            k, v = _nearest(case["format"], k[first:]), _nearest(case["format"], v[first:])
            for h in range(case["q_heads"]):
                x = k[:, h // group] @ s["q"][i, h].double() / math.sqrt(d)
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][h:h + 1].double()])
                out[i, h] = torch.softmax(x, 0)[:n - first] @ v[:, h // group]
        return out
    s = _prompt_inputs(case, seed)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i in range(case["seqs"]):
        a, b, c, e = s["lens_q"][i], s["lens_q"][i + 1], s["lens_k"][i], s["lens_k"][i + 1]
        behind = (e - c) - (b - a)
        gap = torch.arange(b - a, device=DEVICE)[:, None] + behind - torch.arange(e - c, device=DEVICE)
        hidden = (gap < 0) | (gap >= w) if w else gap < 0
        for h in range(case["q_heads"]):
            x = s["q"][a:b, h].double() @ s["k"][c:e, h // group].double().T / math.sqrt(d)
            x[hidden] = -math.inf
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(b - a, 1)], 1)
            out[a:b, h] = torch.softmax(x, 1)[:, :e - c] @ s["v"][c:e, h // group].double()
    return out
