"""New tokens of many sequences over what those sequences keep: attention of packed chunks over the paged
cache, and, for layers whose attention is linear, the short causal convolution and the gated delta rule over
per-sequence states. Single tokens, drafts of a few, and long prompts go through the same calls.

`own` chooses between the plain form (elementary torch operations) and the package's entry points.
Attention shapes are GPT-OSS's (64 query heads on 8 of 64), Qwen3's (32 on 4 of 128) and Coder-Next's (16 on 2
of 256); linear layers have 32 value heads of 128 on 16 key heads of 128. Generic ones are in draw().
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
LINEAR = {"key_heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128}

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user, four drafted tokens checked at once: a layer with a window and sinks
        dict(GPT_OSS, name="extend_draft_one", op="extend", seqs=1, first=4, least=4, most=4, past_least=700,
             past_most=700, src="bf16", format="mxfp4", page=64, window=128, sinks=True),
        # drafts of five for a full serving batch, behind nothing to 24000 tokens
        dict(QWEN3, name="extend_draft_32", op="extend", seqs=32, first=5, least=5, most=5, past_least=0,
             past_most=24000, src="bf16", format="mxfp4", page=256, window=0, sinks=False),
        # one prompt goes on by 1000 tokens while 32 sequences step by one each
        dict(GPT_OSS, name="extend_mixed_33", op="extend", seqs=33, first=1000, least=1, most=1, past_least=100,
             past_most=6000, src="bf16", format="mxint8", page=128, window=0, sinks=True),
        # four prompts at different places, the next parts of them
        dict(QWEN3, name="extend_parts_4", op="extend", seqs=4, first=511, least=300, most=511, past_least=0,
             past_most=8001, src="bf16", format="f16", page=256, window=0, sinks=False),
        # the next 2048 tokens of one long document
        dict(CODER, name="extend_chunk_2048", op="extend", seqs=1, first=2048, least=2048, most=2048,
             past_least=30001, past_most=30001, src="f16", format="mxint8", page=256, window=0, sinks=False),
        # one user's token through a linear layer
        dict(LINEAR, name="delta_step_1", op="delta", seqs=1, first=1, least=1, most=1, src="bf16", raw=True, fresh=0),
        # a serving batch, a token each
        dict(LINEAR, name="delta_step_48", op="delta", seqs=48, first=1, least=1, most=1, src="bf16", raw=True, fresh=0),
        # drafts of five
        dict(LINEAR, name="delta_draft_16", op="delta", seqs=16, first=5, least=5, most=5, src="f16", raw=False, fresh=0),
        # one prompt from its beginning
        dict(LINEAR, name="delta_prompt_4096", op="delta", seqs=1, first=4096, least=4096, most=4096, src="bf16",
             raw=True, fresh=1),
        # prompts of odd lengths, new ones and next parts, narrower keys
        dict(key_heads=4, value_heads=12, key_dim=64, value_dim=128, name="delta_packed_7", op="delta", seqs=7,
             first=1500, least=1, most=1207, src="f16", raw=False, fresh=3),
        # the convolution in front of a linear layer: queries, keys and values of a serving batch's tokens
        dict(name="conv_step_48", op="conv", channels=8192, width=4, seqs=48, first=1, least=1, most=1, src="bf16",
             dst="bf16", bias=False, fresh=0),
        # the same for packed prompts
        dict(name="conv_packed_7", op="conv", channels=8192, width=4, seqs=7, first=1500, least=1, most=1207, src="f32",
             dst="bf16", bias=False, fresh=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: an operator, a shape (a configured one or a generic one) and sizes over the whole range."""
    op = rng.choice(["extend", "extend", "delta", "delta", "conv"])
    if op == "extend":
        if rng.random() < 0.5:
            shape = dict(rng.choice([GPT_OSS, QWEN3, CODER]))
        else:
            kv = rng.choice([1, 2, 3, 4, 5, 8])
            shape = {"kv_heads": kv, "q_heads": kv * rng.choice([1, 2, 3, 4, 6, 8, 12, 16]), "dim": rng.choice([64, 128, 256])}
        seqs = _log_int(rng, 1, 48)
        bits = {"mxfp4": 4, "mxint8": 8, "f16": 16}
        fmt = rng.choice(["mxfp4", "mxint8", "f16"])
        # at most as many cached bytes as the longest listed batch
        room = 32 * 12000 * 4 * 128 * 4 // (shape["kv_heads"] * shape["dim"] * bits[fmt])
        past = _log_int(rng, 16, max(17, min(32000, room // seqs)))
        # and a third of the longest chunk's operations
        area = 16 * 256 * 2048 * 31000 // (3 * shape["q_heads"] * shape["dim"])
        first = _log_int(rng, 1, max(1, min(2048, area // (past + 2048))))
        least = rng.choice([1, 1, min(5, first)])
        most = max(least, rng.choice([1, 5, min(first, max(1, area // (seqs * (past + 2048))))]))
        return dict(shape, op=op, seqs=seqs, first=first, least=least, most=most, past_least=rng.choice([0, 1, past // 2]),
                    past_most=past, src=rng.choice(["f16", "bf16"]), format=fmt, page=rng.choice([64, 128, 256]),
                    window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.4)
    seqs = _log_int(rng, 1, 48)
    first = _log_int(rng, 1, 4096)
    least = rng.choice([1, 1, min(5, first)])
    most = max(least, rng.choice([1, 5, max(1, min(first, 4096 // seqs))]))
    first = max(1, min(first, 4096 - (seqs - 1) * (least + most) // 2))
    fresh = rng.choice([0, 0, seqs, seqs // 2])
    if op == "conv":
        return dict(op=op, channels=rng.choice([8192, 64, 520, 2056, 6144]), width=rng.choice([2, 3, 4, 4]), seqs=seqs,
                    first=first, least=least, most=most, src=rng.choice(["f32", "f16", "bf16"]),
                    dst=rng.choice(["f32", "f16", "bf16"]), bias=rng.random() < 0.3, fresh=fresh)
    if rng.random() < 0.5:
        shape = dict(LINEAR)
    else:
        kh = rng.choice([1, 2, 3, 4, 8])
        shape = {"key_heads": kh, "value_heads": kh * rng.choice([1, 2, 3, 4]), "key_dim": rng.choice([64, 128]),
                 "value_dim": rng.choice([64, 128])}
    return dict(shape, op=op, seqs=seqs, first=first, least=least, most=most, src=rng.choice(["f16", "bf16"]),
                raw=rng.random() < 0.5, fresh=fresh)


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed, *ids):
    for i in ids:
        seed = (seed * 1000003 + i + 1) % (1 << 62)
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _spread(n, first, lo, hi):
    """n numbers: the first one, the others over the range."""
    return [first] + [lo + (hi - lo) * ((5 * i + 3) % n) // max(1, n - 1) for i in range(1, n)]


def _new(case):
    return _spread(case["seqs"], case["first"], case["least"], case["most"])


def _lengths(case):
    """Tokens of each sequence in the cache, its new ones among them."""
    past = _spread(case["seqs"], case["past_most"], case["past_least"], case["past_most"])
    return [p + n for p, n in zip(past, _new(case))]


def _offsets(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu, torch.tensor(cu, dtype=torch.int32, device=DEVICE)


def _keys(shape, g):
    """Projected keys: about N(0, 1), one channel in 16 four times as wide."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    x[..., 5::16] *= 4.0
    return x


def _extend_inputs(case, seed):
    """Queries, lengths and pages; the cached keys and values of sequence i come from _history(case, seed, i)."""
    g = _gen(seed)
    page, lens = case["page"], _lengths(case)
    counts = [(n + page - 1) // page for n in lens]
    order = torch.randperm(sum(counts) + 1, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros((case["seqs"], max(counts)), dtype=torch.int32, device=DEVICE)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    cu, cu_q = _offsets(_new(case))
    q = torch.randn((cu[-1], case["q_heads"], case["dim"]), generator=g, device=DEVICE).to(TYPES[case["src"]])
    sinks = torch.randn(case["q_heads"], generator=g, device=DEVICE) if case["sinks"] else None
    return {"q": q, "sinks": sinks, "cu": cu, "cu_q": cu_q, "lens": lens, "table": table, "pages": sum(counts) + 1,
            "len": torch.tensor(lens, dtype=torch.int32, device=DEVICE)}


def _history(case, seed, i, n):
    g = _gen(seed, i)
    shape = (n, case["kv_heads"], case["dim"])
    return _keys(shape, g), torch.randn(shape, generator=g, device=DEVICE)


def _slots(case, s, i):
    t = torch.arange(s["lens"][i], device=DEVICE)
    return s["table"][i][t // case["page"]].long() * case["page"] + t % case["page"]


def _states(case, shape, g):
    """States of the sequences, and where each reads and writes its own: new sequences start from zeros; the old
    states stay, as drafts need them that are not taken."""
    n = case["seqs"]
    states = torch.zeros((2 * n, *shape), device=DEVICE)
    states[:n] = torch.randn((n, *shape), generator=g, device=DEVICE)
    source = torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)
    target = source + n
    source[n - case["fresh"]:] = -1
    return states, source, target


def _delta_inputs(case, seed):
    g = _gen(seed)
    kh, vh, dk, dv, t = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"], TYPES[case["src"]]
    cu, cu_q = _offsets(_new(case))
    T = cu[-1]
    # one row a token, as a convolution with SiLU leaves them
    x = torch.randn((T, 2 * kh * dk + vh * dv), generator=g, device=DEVICE) * 1.5
    x = x * torch.sigmoid(x)
    q, k, v = x[:, :kh * dk].view(T, kh, dk), x[:, kh * dk:2 * kh * dk].view(T, kh, dk), x[:, 2 * kh * dk:].view(T, vh, dv)
    a, b = (torch.randn((T, vh), generator=g, device=DEVICE) for _ in range(2))
    s = {"cu": cu, "cu_q": cu_q}
    a_log = torch.log(1 + 15 * torch.rand(vh, generator=g, device=DEVICE))
    dt = torch.exp(math.log(0.001) + (math.log(0.1) - math.log(0.001)) * torch.rand(vh, generator=g, device=DEVICE))
    dt_bias = dt + torch.log(-torch.expm1(-dt))
    if case["raw"]:
        s.update(q=q.to(t), k=k.to(t), v=v.to(t), a=a, b=b, a_log=a_log, dt_bias=dt_bias)
    else:
        unit = [y / y.square().sum(-1, keepdim=True).sqrt() for y in (q, k)]
        g_log = -torch.exp(a_log) * torch.nn.functional.softplus(a + dt_bias)
        s.update(q=unit[0].to(t), k=unit[1].to(t), v=v.to(t), a=g_log, b=torch.sigmoid(b), a_log=None, dt_bias=None)
    s["states"], s["source"], s["target"] = _states(case, (vh, dk, dv), g)
    s["states"] *= 0.1
    return s


def _conv_inputs(case, seed):
    g = _gen(seed)
    c, w = case["channels"], case["width"]
    cu, cu_q = _offsets(_new(case))
    s = {"cu": cu, "cu_q": cu_q, "x": torch.randn((cu[-1], c), generator=g, device=DEVICE).to(TYPES[case["src"]]),
         "w": torch.randn((c, w), generator=g, device=DEVICE) / math.sqrt(w),
         "bias": torch.randn(c, generator=g, device=DEVICE) * 0.1 if case["bias"] else None}
    s["states"], s["source"], s["target"] = _states(case, (w - 1, c), g)
    s["states"] = s["states"].to(TYPES[case["src"]]).float()  # earlier inputs
    return s


# ---- the plain form ------------------------------------------------------------------------------
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _quantise(fmt, x):
    """Codes (whole numbers as int8) and exponents [.., dim / 32] of the blocks of 32; f16: the values themselves."""
    if fmt == "f16":
        return x.clamp(-65504.0, 65504.0).half(), None
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))  # m in [0.5, 1): amax = 2m * 2^(e-1)
    e = e - 3 + (m > 0.875).int() if fmt == "mxfp4" else e - 7 + (m >= 0.99609375).int()
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
    v = torch.tensor(FP4, device=DEVICE)[b.abs().int()] * torch.sign(b.float()) if fmt == "mxfp4" else b.float()
    return torch.ldexp(v, e.int()[..., None]).flatten(-2)


def _plain_extend(s):
    case = s["case"]
    hk, d, fmt = case["kv_heads"], case["dim"], case["format"]
    out = torch.zeros_like(s["q"])
    for i, n in enumerate(s["lens"]):
        a, b = s["cu"][i], s["cu"][i + 1]
        slots = _slots(case, s, i)
        lo = max(0, n - (b - a) + 1 - case["window"]) if case["window"] else 0  # what the first row sees
        k, v = (_values(fmt, s[x + "_code"][slots[lo:]], None if s[x + "_exp"] is None else s[x + "_exp"][slots[lo:]])
                .transpose(0, 1)[:, None] for x in ("k", "v"))
        q = s["q"][a:b].float().unflatten(1, (hk, -1)).permute(1, 2, 0, 3)  # key head, its heads, rows, dim
        x = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
        behind = torch.arange(n - (b - a), n, device=DEVICE)[:, None] - torch.arange(lo, n, device=DEVICE)
        seen = (behind >= 0) & (behind < case["window"]) if case["window"] else behind >= 0
        x = x.masked_fill(~seen, -math.inf)
        m = x.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sinks = s["sinks"].view(hk, -1, 1, 1)
            m = torch.maximum(m, sinks)
        p = torch.exp(x - m)
        z = p.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            z = z + torch.exp(sinks - m)
        y = torch.matmul(p, v) / z
        out[a:b] = y.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
    return out


def _start(states, source):
    """The states that the sequences start from: zeros for new ones."""
    return states[source.clamp(min=0).long()] * (source >= 0).view(-1, *[1] * (states.dim() - 1))


def _rows(s, step):
    """The packed row of each sequence's i-th token, in whole steps, and whether there is one."""
    n = torch.tensor(_new(s["case"]), device=DEVICE)[:, None]
    longest = max(_new(s["case"]))
    i = torch.arange((longest + step - 1) // step * step, device=DEVICE)
    there = i < n
    return torch.where(there, s["cu_q"][:-1, None].long() + i, 0), there


def _plain_delta(s):
    """Steps of up to 64 tokens at a time: within a step the tokens' corrections of the state solve a triangular
    system, so that it takes products of whole steps; the steps follow each other."""
    case = s["case"]
    vh, group = case["value_heads"], case["value_heads"] // case["key_heads"]
    step = min(64, max(_new(case)))
    rows, there = _rows(s, step)
    seqs = rows.shape[0]

    def take(x):  # sequence, head, step, token of it, elements
        x = x.float()[rows] * there.view(*there.shape, *[1] * (x.dim() - 1))
        return x.unflatten(1, (-1, step)).movedim(3, 1)

    q, k, v = (take(s[x]) for x in ("q", "k", "v"))
    if case["raw"]:
        q, k = (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6) for x in (q, k))
        g = -torch.exp(s["a_log"]) * torch.log1p(torch.exp(s["a"] + s["dt_bias"]))
        beta = torch.sigmoid(s["b"])
    else:
        g, beta = s["a"], s["b"]
    q, k = (x.repeat_interleave(group, 1) for x in (q, k))
    beta = take(beta)[..., None]
    g = take(g).double().cumsum(-1)
    lower = torch.ones((step, step), dtype=torch.bool, device=DEVICE).tril()
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~lower, -math.inf)).float()
    rise, fall = torch.exp(g).float()[..., None], torch.exp(g[..., -1:] - g).float()[..., None]
    mix = torch.matmul(beta * k, k.transpose(-1, -2)) * decay
    inverse = torch.eye(step, device=DEVICE).expand_as(mix).contiguous()
    for i in range(1, step):
        inverse[..., i, :i] = -torch.matmul(mix[..., i:i + 1, :i], inverse[..., :i, :i])[..., 0, :]
    u, w = torch.matmul(inverse, beta * v), torch.matmul(inverse, beta * rise * k)
    scale = case["key_dim"] ** -0.5
    look = torch.matmul(q, k.transpose(-1, -2)) * decay * scale
    q, k = q * rise * scale, (k * fall).transpose(-1, -2)
    state = _start(s["states"], s["source"])
    out = torch.empty_like(v)
    for n in range(v.shape[2]):
        new = u[:, :, n] - torch.matmul(w[:, :, n], state)
        out[:, :, n] = torch.matmul(q[:, :, n], state) + torch.matmul(look[:, :, n], new)
        state = state * rise[:, :, n, -1:] + torch.matmul(k[:, :, n], new)
    s["states"][s["target"].long()] = state
    out = out.movedim(1, 3).flatten(1, 2)  # sequence, token, head, elements
    return [out[there].to(s["v"].dtype), s["states"][seqs:]]


def _plain_conv(s):
    case, x = s["case"], s["x"].float()
    w = case["width"]
    counts = torch.tensor(_new(case), device=DEVICE)
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device=DEVICE), counts)
    place = torch.arange(len(x), device=DEVICE) - s["cu_q"].long()[seq]  # of a token in its sequence
    start = _start(s["states"], s["source"])

    def earlier(seq, place, back):  # the inputs `back` tokens earlier
        i = place - back
        row = (s["cu_q"].long()[seq] + i).clamp(min=0, max=len(x) - 1)
        return torch.where((i >= 0)[:, None], x[row], start[seq, (w - 1 + i).clamp(0, w - 2)])

    y = x * s["w"][:, w - 1]
    for back in range(1, w):
        y = y + earlier(seq, place, back) * s["w"][:, w - 1 - back]
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y * torch.sigmoid(y)
    every = torch.arange(case["seqs"], device=DEVICE)
    s["states"][s["target"].long()] = torch.stack([earlier(every, counts, w - 1 - j) for j in range(w - 1)], 1)
    return [y.to(TYPES[case["dst"]]), s["states"][case["seqs"]:]]


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


def _kind(x):
    M = _package()
    return {torch.float32: M.F32, torch.float16: M.F16, torch.bfloat16: M.BF16}[x.dtype]


def _heads(x):
    return _package().Heads(x.data_ptr(), x.shape[1], _kind(x), x.stride(0), x.stride(1))


def _matrix(x):
    return _package().Rows(x.data_ptr(), x.shape[1], _kind(x), x.stride(0))


class _Handle:
    """A handle of the package that goes with the state."""

    def __init__(self, make):
        self.h = make()

    def __del__(self):
        try:
            self.h.close()
        except (AttributeError, TypeError):  # half-made, or at the interpreter's end
            pass


def prepare(case, seed):
    op = case["op"]
    s = {"extend": _extend_inputs, "delta": _delta_inputs, "conv": _conv_inputs}[op](case, seed)
    s["case"] = case
    M = _package() if own else None
    if op == "extend":
        hk, d, fmt, n = case["kv_heads"], case["dim"], case["format"], s["pages"] * case["page"]
        if own:
            kind = {"mxfp4": M.KV_MXFP4, "mxint8": M.KV_MXINT8, "f16": M.KV_F16}[fmt]
            s["cache"] = _Handle(lambda: M.KvCache(_context(), kind, s["pages"], case["page"], hk, d))
            s["out"] = torch.zeros_like(s["q"])
        else:
            for a in ("k", "v"):
                s[a + "_code"] = torch.zeros((n, hk, d), dtype=torch.float16 if fmt == "f16" else torch.int8, device=DEVICE)
                s[a + "_exp"] = None if fmt == "f16" else torch.zeros((n, hk, d // 32), dtype=torch.int8, device=DEVICE)
        for i, n in enumerate(s["lens"]):
            slots = _slots(case, s, i)
            kv = _history(case, seed, i, n)
            if own:
                slots = slots.to(torch.int32)
                s["cache"].h.write(_heads(kv[0]), _heads(kv[1]), n, slots.data_ptr())
                continue
            for a, x in zip(("k", "v"), kv):
                code, e = _quantise(fmt, x)
                s[a + "_code"][slots] = code
                if e is not None:
                    s[a + "_exp"][slots] = e
    elif own and op == "delta":
        s["rule"] = _Handle(lambda: M.DeltaRule(
            _context(), case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"],
            unit_eps=1e-6 if case["raw"] else 0.0, a_log=s["a_log"].data_ptr() if case["raw"] else None,
            dt_bias=s["dt_bias"].data_ptr() if case["raw"] else None))
        s["out"] = torch.empty_like(s["v"], memory_format=torch.contiguous_format)
    elif own:
        s["out"] = torch.empty(s["x"].shape, dtype=TYPES[case["dst"]], device=DEVICE)
    torch.cuda.synchronize()
    return s


def run(s):
    case = s["case"]
    op, n = case["op"], case["seqs"]
    if not own:
        return {"extend": _plain_extend, "delta": _plain_delta, "conv": _plain_conv}[op](s)
    M, ctx = _package(), _context()
    cu = s["cu_q"].data_ptr()
    if op == "extend":
        s["cache"].h.extend(_heads(s["q"]), s["q"].shape[0], n, cu, s["len"].data_ptr(), s["table"].data_ptr(),
                            s["table"].shape[1], _heads(s["out"]), window=case["window"],
                            sinks=s["sinks"].data_ptr() if case["sinks"] else None)
        return s["out"]
    states = dict(states=s["states"].data_ptr(), n_slots=2 * n, source=s["source"].data_ptr(), target=s["target"].data_ptr())
    if op == "delta":
        s["rule"].h.forward(_heads(s["q"]), _heads(s["k"]), _heads(s["v"]), s["a"].data_ptr(), s["b"].data_ptr(),
                            s["v"].shape[0], n, cu, _heads(s["out"]), **states)
    else:
        M.causal_conv(ctx, _matrix(s["x"]), s["w"].data_ptr(), case["width"], s["x"].shape[0], n, cu, _matrix(s["out"]),
                      bias=s["bias"].data_ptr() if case["bias"] else None, silu=True, **states)
    return [s["out"], s["states"][n:]]


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    op, new = case["op"], _new(case)
    if op == "extend":
        hq, hk, d, w = case["q_heads"], case["kv_heads"], case["dim"], case["window"]
        bits = {"mxfp4": 4, "mxint8": 8, "f16": 16}[case["format"]]
        token = 2 * hk * (d * bits // 8 + (0 if bits == 16 else d // 32))  # keys, values and the blocks' exponents
        seen = pairs = 0
        for n, m in zip(new, _lengths(case)):
            seen += min(m, n + w - 1) if w else m
            # the i-th position of a sequence sees min(i, window) keys
            lo, full = m - n + 1, min(m, w) if w else m
            if full >= lo:
                pairs += (full - lo + 1) * (lo + full) // 2
            pairs += (m - max(full, lo - 1)) * w
        return {"bytes": seen * token + 4 * sum(new) * hq * d, "flops": 4 * pairs * hq * d}
    T, kept = sum(new), 2 * case["seqs"] - case["fresh"]
    if op == "delta":
        kh, vh, dk, dv = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
        # what a state has for the key, the correction of it, and what it has for the query
        return {"bytes": T * (2 * size[case["src"]] * (kh * dk + vh * dv) + 8 * vh) + 4 * kept * vh * dk * dv,
                "flops": 6 * T * vh * dk * dv}
    c, w = case["channels"], case["width"]
    return {"bytes": c * (T * (size[case["src"]] + size[case["dst"]]) + 4 * w + 4 * kept * (w - 1)), "flops": T * c * (2 * w + 4)}


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


def _exact_extend(case, seed):
    s = _extend_inputs(case, seed)
    hq, d, w = case["q_heads"], case["dim"], case["window"]
    group = hq // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(s["lens"]):
        a, b = s["cu"][i], s["cu"][i + 1]
        k, v = (_nearest(case["format"], x) for x in _history(case, seed, i, n))
        gap = torch.arange(b - a, device=DEVICE)[:, None] + (n - (b - a)) - torch.arange(n, device=DEVICE)
        hidden = (gap < 0) | (gap >= w) if w else gap < 0
        for h in range(hq):
            x = s["q"][a:b, h].double() @ k[:, h // group].T / math.sqrt(d)
            x[hidden] = -math.inf
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(b - a, 1)], 1)
            out[a:b, h] = torch.softmax(x, 1)[:, :n] @ v[:, h // group]
    return out


def _exact_delta(case, seed):
    """A sequence at a time, all its tokens as one triangular system."""
    s = _delta_inputs(case, seed)
    group, n = case["value_heads"] // case["key_heads"], case["seqs"]
    q, k, v, a, beta = (s[x].double() for x in ("q", "k", "v", "a", "b"))
    if case["raw"]:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
        a = a + s["dt_bias"].double()
        a = -torch.exp(s["a_log"].double()) * (a.clamp(min=0) + torch.log1p(torch.exp(-a.abs())))
        beta = 1 / (1 + torch.exp(-beta))
    out, states = torch.zeros_like(v), s["states"][n:].double()
    for i in range(n):
        lo, hi = s["cu"][i], s["cu"][i + 1]
        kept = int(s["source"][i])
        start = s["states"][kept].double() if kept >= 0 else torch.zeros_like(states[0])
        at = torch.arange(hi - lo, device=DEVICE)
        for h in range(case["value_heads"]):
            x, y, z, e = q[lo:hi, h // group], k[lo:hi, h // group], v[lo:hi, h], beta[lo:hi, h, None]
            total = torch.cumsum(a[lo:hi, h], 0)[:, None]
            apart = total - total.T
            apart[at[:, None] < at] = -math.inf
            fade = torch.exp(apart)
            system = torch.tril(e * (y @ y.T) * fade, -1)
            system[at, at] = 1.0
            wanted = e * (z - torch.exp(total) * (y @ start[h]))
            new = torch.linalg.solve_triangular(system, wanted, upper=False, unitriangular=True)
            out[lo:hi, h] = (torch.exp(total) * (x @ start[h]) + (x @ y.T * fade) @ new) / math.sqrt(case["key_dim"])
            states[int(s["target"][i]) - n, h] = torch.exp(total[-1]) * start[h] + (y * torch.exp(total[-1] - total)).T @ new
    return [out, states]


def _exact_conv(case, seed):
    s = _conv_inputs(case, seed)
    n, w = case["seqs"], case["width"]
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEVICE)
    states = s["states"][n:].double()
    for i in range(n):
        lo, hi = s["cu"][i], s["cu"][i + 1]
        kept = int(s["source"][i])
        before = s["states"][kept].double() if kept >= 0 else torch.zeros_like(states[0])
        line = torch.cat([before, s["x"][lo:hi].double()])
        y = (line.unfold(0, w, 1) * s["w"].double()).sum(-1)
        if s["bias"] is not None:
            y = y + s["bias"].double()
        out[lo:hi] = y / (1 + torch.exp(-y))
        states[int(s["target"][i]) - n] = line[len(line) - (w - 1):]
    return [out, states]


def exact(case, seed):
    return {"extend": _exact_extend, "delta": _exact_delta, "conv": _exact_conv}[case["op"]](case, seed)
