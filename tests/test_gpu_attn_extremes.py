"""The attention-side operators on the GPU where sums run out of bits: scores of any finite size, weights far below
the largest, sinks at the ends of their range; parts of a split sequence with sinks and with missing pages; and which
keys each row of a long sequence sees, counted."""
import numpy as np
import pytest

import moe_rocm as M

import attnref as R
from test_gpu_attn import FORMATS, TYPES, Cached, sync_error

pytestmark = pytest.mark.gpu


def decode(ctx, kv, q, dtype, lens, table, **kw):
    """One call over the cache `kv`: q [n_seqs, heads, D]."""
    H, D = q.shape[1:]
    dq, out = R.Rows(ctx, q, dtype), R.Rows(ctx, None, dtype, len(lens), H, D)
    dl, dt = R.i32(ctx, lens), R.i32(ctx, table)
    sinks = kw.pop("sinks", None)
    ds = None if sinks is None else ctx.to_device(np.asarray(sinks, np.float32))
    kv.attend(dq.heads, len(lens), dl, dt, table.shape[1], out.heads, sinks=ds, **kw)
    try:
        ctx.sync()
        return out.get()
    finally:
        for b in (dq, out, dl, dt, ds):
            if b is not None:
                b.free()


def prompt(ctx, q, k, v, dtype, cu_q, cu_k, **kw):
    D = q.shape[2]
    dq, dk, dv = (R.Rows(ctx, x, dtype) for x in (q, k, v))
    out = R.Rows(ctx, None, dtype, *q.shape)
    dcq, dck = R.i32(ctx, cu_q), R.i32(ctx, cu_k)
    sinks = kw.pop("sinks", None)
    ds = None if sinks is None else ctx.to_device(np.asarray(sinks, np.float32))
    M.attn_prefill(ctx, D, dq.heads, dk.heads, dv.heads, len(q), len(k), len(cu_q) - 1, dcq, dck, out.heads, sinks=ds, **kw)
    ctx.sync()
    y = out.get()
    for b in (dq, dk, dv, out, dcq, dck, ds):
        if b is not None:
            b.free()
    return y


def filled(ctx, fmt, seqs, page=64):
    """A cache with the sequences (k, v) [n, heads, D] on pages one after the other -> (cache, table)."""
    H, D = seqs[0][0].shape[1:]
    counts = [max(1, -(-len(k) // page)) for k, _ in seqs]
    kv = M.KvCache(ctx, fmt, sum(counts), page, H, D)
    table = np.zeros((len(seqs), max(counts)), np.int32)
    at = 0
    for i, ((k, v), c) in enumerate(zip(seqs, counts)):
        table[i, :c] = at + np.arange(c)
        if len(k):
            dk, dv = R.Rows(ctx, k, M.F32), R.Rows(ctx, v, M.F32)
            ds = R.i32(ctx, at * page + np.arange(len(k)))
            kv.write(dk.heads, dv.heads, len(k), ds)
            ctx.sync()
            dk.free(), dv.free(), ds.free()
        at += c
    return kv, table


# ---- scores of any finite size ---------------------------------------------------------------------
def check_one_of(got, q, k, v, scale, dtype):
    """A row whose scores are so large that 32 bits hold them to whole powers of e or worse. On one key it is the key's
    value. With the largest score clear of the others by more than the scores' own error (D products summed in 32 bits
    and three more roundings: (D + 4) 2^-24 of the sum of magnitudes, at either key) and 40 (e^-40 for each of 700 others at
    most: nothing, in 16 bits of output), it is that key's value too. Else weights are whatever the error makes them,
    but they are weights: the row lies between the least and the largest value, give or take the output's rounding and the
    weights' (each off by half a step of 16 bits of weight, in sum and divisor)."""
    q, k = q.astype(np.float64), k.astype(np.float64)
    s = k @ q * scale
    err = (len(q) + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)) * abs(scale)
    top = int(s.argmax())
    clear = all(s[top] - s[j] > err[top] + err[j] + 40 for j in range(len(s)) if j != top)
    if clear:
        assert (got == R.rounded(v[top], dtype)).all(), (len(s), got[:4], v[top][:4])
    else:
        room = (2 * R.HALF[dtype] + 2.0 ** -10) * np.abs(v).max()
        assert (got >= v.min(0) - room).all() and (got <= v.max(0) + room).all(), (len(s), got[:4])
    return clear


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,q_size,k_size,scale", [("f16", 8000, 8000, 0.0), ("f16", 60000, 60000, 0.0), ("bf16", 20000, 3e4, -0.3),
                                                       ("bf16", 1e6, 100.0, 1.0), ("f16", 500, 500, 1e6), ("bf16", 1e30, 6e4, 1e-24),
                                                       ("f16", 6e4, 6e4, 1e25)])
def test_decode_scores_beyond_the_bits_of_the_base(gpu_ctx, fmt, D, dtype, q_size, k_size, scale):
    dtype, fmt = TYPES[dtype], FORMATS[fmt]
    rng = np.random.default_rng(D)
    lens, hk, group = [1] * 12 + [2, 3, 5, 70, 700], 2, 3
    seqs = [((rng.uniform(-1, 1, (n, hk, D)) * k_size).astype(np.float32), rng.normal(size=(n, hk, D)).astype(np.float32)) for n in lens]
    kv, table = filled(gpu_ctx, fmt, seqs)
    q = R.rounded(rng.uniform(-1, 1, (len(lens), hk * group, D)) * q_size, dtype)
    got = decode(gpu_ctx, kv, q, dtype, lens, table, scale=scale)
    n_clear = 0
    for i, (k, v) in enumerate(seqs):
        k, v = R.stored(k, fmt), R.stored(v, fmt)
        for h in range(hk * group):
            n_clear += check_one_of(got[i, h], q[i, h], k[:, h // group], v[:, h // group], scale or D ** -0.5, dtype)
    assert n_clear >= 12 * hk * group
    kv.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 256])
def test_decode_of_a_split_sequence_with_large_scores(gpu_ctx, fmt, D):
    """The parts' bases differ by less than their own last bits: the key that takes all weight lies in any part."""
    fmt = FORMATS[fmt]
    rng = np.random.default_rng(D)
    n = 9000
    k, v = (rng.uniform(-1, 1, (n, 1, D)) * 2.0).astype(np.float32), rng.normal(size=(n, 1, D)).astype(np.float32)
    at = np.array([0, 4000, 8999, 77])
    q = np.zeros((1, 4, D), np.float32)
    for h, a in enumerate(at):  # a key that lies along the query, larger than all others
        k[a, 0] = np.sign(rng.normal(size=D)) * 64
        q[0, h] = np.sign(k[a, 0]) * 16384
    kv, table = filled(gpu_ctx, fmt, [(k, v)], page=256)
    ks, vs = R.stored(k, fmt), R.stored(v, fmt)
    for scale in (1.0, 1e4):
        got = decode(gpu_ctx, kv, q, M.F16, [n], table, scale=scale)
        for h in range(4):
            assert check_one_of(got[0, h], q[0, h], ks[:, 0], vs[:, 0], scale, M.F16)
            assert int((ks[:, 0] @ q[0, h]).argmax()) == at[h]
    kv.close()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,q_size,k_size,scale", [("f16", 8000, 8000, 0.0), ("f16", 60000, 60000, 0.0), ("bf16", 1e4, 1e5, -0.3),
                                                       ("bf16", 1e9, 1e7, 0.0), ("f16", 500, 500, 1e6), ("bf16", 1e25, 1e6, 1e-20),
                                                       ("f16", 6e4, 6e4, 1e25)])
@pytest.mark.parametrize("window", [0, 1, 30])
def test_prefill_scores_beyond_the_bits_of_the_base(gpu_ctx, D, dtype, q_size, k_size, scale, window):
    dtype = TYPES[dtype]
    rng = np.random.default_rng(D + window)
    lens, hk, group = [1, 1, 1, 2, 3, 40, 150], 1, 2
    cu = np.concatenate([[0], np.cumsum(lens)])
    q = R.rounded(rng.uniform(-1, 1, (cu[-1], hk * group, D)) * q_size, dtype)
    k = R.rounded(rng.uniform(-1, 1, (cu[-1], hk, D)) * k_size, dtype)
    v = R.rounded(rng.normal(size=(cu[-1], hk, D)), dtype)
    got = prompt(gpu_ctx, q, k, v, dtype, cu, cu, scale=scale, window=window)
    n_clear = 0
    for a, b in zip(cu[:-1], cu[1:]):
        for r in range(a, b):
            first = max(a, r - window + 1) if window else a
            for h in range(hk * group):
                n_clear += check_one_of(got[r, h], q[r, h], k[first:r + 1, h // group], v[first:r + 1, h // group],
                                        scale or D ** -0.5, dtype)
    assert n_clear >= len(lens) * hk * group


# ---- weights far below the largest -----------------------------------------------------------------
def fine_bound(y, size_v, size_s, n, D, out_type, p_half, least):
    """How far a result may be off. The output's own rounding (and half of the smallest step of f16). Each weight is off
    by p_half of itself or by `least` of the largest weight, in the sum of values and in the divisor; its score, D products
    summed in 32 bits and four more roundings, by `ds`, each an error of p relative to p; the sums' own by n roundings."""
    ds = (D + 6) * 2.0 ** -24 * size_s + 8 * 2.0 ** -24
    return (R.HALF[out_type] * np.abs(y) + (p_half + 2 * ds + n * 2.0 ** -24) * (size_v + np.abs(y))
            + least * n * (np.abs(y) + 1.0) * 4 + 2.0 ** -25)


def tail(rng, n, H, D, lead, scale_q):
    """n keys with scores of about 0 (spread 0.3) against q = scale_q * ones, and values about 1 (spread 0.3); with
    `lead`, the first one's score is that and its value zero."""
    k = (rng.normal(size=(n, H, D)) * 0.3 / scale_q).astype(np.float32)  # scores sum over D, times D^-1/2
    v = (1 + 0.3 * rng.normal(size=(n, H, D))).astype(np.float32)
    if lead is not None:
        k[0], v[0] = lead * D ** -0.5 / scale_q, 0.0
    return k, v


def far_below(q, k, v, scale, sink):
    """The row by 64 bits -> (row, sum p |v|, largest sum of magnitudes of a score's terms, keys)."""
    return R.attend(q, k, v, scale, 0, len(k) - 1, sink)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,lead,sink", [(24000, 16.0, None), (24000, 18.0, None), (1000, 18.0, None), (24000, None, 18.0), (1000, 15.0, 17.0)])
def test_decode_of_a_long_tail_far_below_the_largest(gpu_ctx, fmt, D, dtype, n, lead, sink):
    """One key (a first token, say) or a sink takes nearly all weight and has no value: the rest is the result."""
    dtype, fmt = TYPES[dtype], FORMATS[fmt]
    rng = np.random.default_rng(D)
    k, v = tail(rng, n, 1, D, lead, 1.0)
    kv, table = filled(gpu_ctx, fmt, [(k, v)], page=256)
    k, v = R.stored(k, fmt)[:, 0], R.stored(v, fmt)[:, 0]
    q = np.ones((1, 2, D), np.float32)
    got = decode(gpu_ctx, kv, q, dtype, [n], table, sinks=None if sink is None else [sink, sink])
    for h in range(2):
        y, av, ss, cnt = far_below(q[0, h], k, v, D ** -0.5, sink)
        # weights in f16, the largest of them 2^14: half of the smallest step is 2^-39 of it
        tol = fine_bound(y, av, ss, cnt, D, dtype, 2.0 ** -11, 2.0 ** -39)
        assert (np.abs(got[0, h] - y) <= tol).all(), float((np.abs(got[0, h] - y) / tol).max())
        assert (tol <= 0.05 * np.abs(y) + 2.0 ** -25).all()  # the bound sees a lost tail
    kv.close()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,lead,sink", [(20000, 16.0, None), (20000, 18.0, None), (300, None, 16.0), (20000, None, 18.0), (20000, 12.0, 17.0)])
def test_prefill_of_a_long_tail_far_below_the_largest(gpu_ctx, D, dtype, n, lead, sink):
    dtype = TYPES[dtype]
    rng = np.random.default_rng(D)
    k, v = (R.rounded(x, dtype) for x in tail(rng, n, 1, D, lead, 1.0))
    q = np.ones((40, 2, D), np.float32)
    got = prompt(gpu_ctx, q, k, v, dtype, [0, 40], [0, n], sinks=None if sink is None else [sink, sink])
    for r in (0, 1, 31, 32, 39):
        for h in range(2):
            seen = n - 40 + r + 1
            y, av, ss, cnt = far_below(q[r, h], k[:seen, 0], v[:seen, 0], D ** -0.5, sink)
            # f16: the largest weight is 2^7 or more, half of the smallest step 2^-25; bf16: the range of 32 bits
            tol = fine_bound(y, av, ss, cnt, D, dtype, R.HALF[dtype], 2.0 ** -32 if dtype == M.F16 else 0.0)
            assert (np.abs(got[r, h] - y) <= tol).all(), (r, float((np.abs(got[r, h] - y) / tol).max()))
            assert (tol <= 0.15 * np.abs(y) + 2.0 ** -25).all()


# ---- sinks ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
def test_sinks_at_the_ends_of_their_range(gpu_ctx, D):
    """-inf is no sink, 3e38 or any that is far above the scores leaves nothing, inf and NaN have no result: the same
    over the cache, whole and split, and over a prompt."""
    rng = np.random.default_rng(D)
    sinks = np.array([-np.inf, np.inf, np.nan, 200.0, -1e30, 1e38], np.float32)
    H = len(sinks)
    for n in (3, 90, 5000):
        k, v = rng.normal(size=(n, 1, D)).astype(np.float32), rng.normal(size=(n, 1, D)).astype(np.float32)
        q = R.rounded(rng.normal(size=(1, H, D)), M.F16)
        kv, table = filled(gpu_ctx, M.KV_F16, [(k, v)])
        k, v = R.stored(k, M.KV_F16), R.stored(v, M.KV_F16)
        got = [decode(gpu_ctx, kv, q, M.F16, [n], table, sinks=sinks)[0], prompt(gpu_ctx, q, k, v, M.F16, [0, 1], [0, n], sinks=sinks)[0],
               prompt(gpu_ctx, q, k, v, M.BF16, [0, 1], [0, n], sinks=sinks)[0]]
        for g, dtype in zip(got, (M.F16, M.F16, M.BF16)):
            assert np.isnan(g[1:3]).all() and (g[[3, 5]] == 0).all(), (n, g[1:, :2])
            for h in (0, 4):
                x, kk, vv = (R.rounded(a, dtype) for a in (q[0, h], k[:, 0], v[:, 0]))
                y, av, ss, cnt = R.attend(x, kk, vv, D ** -0.5, 0, n - 1)
                assert (np.abs(g[h] - y) <= R.attention_bound(y, av, ss, cnt, D, dtype, R.HALF[dtype])).all()
        kv.close()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_sinks_of_rows_that_see_nothing(gpu_ctx, D):
    """With no key a sink that has a weight takes it all: zeros; one that is not a number or infinite has no result."""
    sinks = [0.5, -np.inf, np.inf, np.nan]
    q, k = np.ones((3, 4, D), np.float32), np.ones((1, 1, D), np.float32)
    got = prompt(gpu_ctx, q, k, k, M.F16, [0, 3], [0, 1], sinks=sinks)
    assert (got[:2, :2] == 0).all() and np.isnan(got[:2, 2:]).all()
    kv, table = filled(gpu_ctx, M.KV_F16, [(k, k)])
    got = decode(gpu_ctx, kv, q[:1], M.F16, [0], table, sinks=sinks)
    assert (got[0, :2] == 0).all() and np.isnan(got[0, 2:]).all()
    kv.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,hk,group", [(64, 8, 8), (128, 4, 8), (256, 2, 8), (64, 1, 20), (128, 2, 3)])
@pytest.mark.parametrize("window", [0, 4097])
def test_decode_of_split_sequences_with_sinks(gpu_ctx, fmt, D, hk, group, window):
    lens = [9000, 0, 1500, 20, 5011]
    c = Cached(gpu_ctx, FORMATS[fmt], lens, hk, D, 256, D + group)
    rng = np.random.default_rng(4)
    H = hk * group
    q = R.rounded(rng.normal(size=(len(lens), H, D)), M.BF16)
    sinks = rng.normal(size=H).astype(np.float32) * 3
    sinks[0], sinks[-1], sinks[H // 2] = -np.inf, 40.0, 8.0
    got = decode(gpu_ctx, c.kv, q, M.BF16, lens, c.table, window=window, sinks=sinks)
    c.check(got, q, M.BF16, group, D ** -0.5, window, sinks)
    c.close()


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("D,hk,group", [(64, 2, 4), (256, 1, 3)])
def test_decode_of_split_sequences_with_pages_missing(gpu_ctx, D, hk, group, sink):
    """Pages out of range in places, in a row longer than any part, and all of them; lengths out of range."""
    lens = [20000, 6000, 3000]
    c = Cached(gpu_ctx, M.KV_MXINT8, lens, hk, D, 64, 3)
    rng = np.random.default_rng(4)
    H = hk * group
    q = R.rounded(rng.normal(size=(3, H, D)), M.F16)
    sinks = rng.normal(size=H).astype(np.float32) if sink else None
    table = c.table.copy()
    there = [np.ones(n, bool) for n in lens]
    for page in [0, 7, *range(20, 290)]:
        table[0, page] = -1
        there[0][64 * page:64 * page + 64] = False
    table[1, :] = int(c.kv.desc.n_pages)
    there[1][:] = False
    dq, out, dl, dt = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, None, M.F16, 3, H, D), R.i32(gpu_ctx, lens), R.i32(gpu_ctx, table)
    ds = gpu_ctx.to_device(sinks) if sink else None
    c.kv.attend(dq.heads, 3, dl, dt, table.shape[1], out.heads, sinks=ds)
    sync_error(gpu_ctx, "block_table")
    got = out.get()
    assert (got[1] == 0).all()
    c.check(got, q, M.F16, group, D ** -0.5, 0, sinks, there)
    # a length beyond the table's: its pages behind the sequence's are out of range; one below zero: none
    dl.upload(np.array([2 ** 31 - 1, -3, 3000], np.int32)), dt.upload(c.table)
    c.kv.attend(dq.heads, 3, dl, dt, table.shape[1], out.heads, sinks=ds)
    sync_error(gpu_ctx, "seq_len block_table")
    got = out.get()
    assert (got[1] == 0).all() and np.isfinite(got).all()
    c.lens, c.k, c.v = [3000], c.k[2:], c.v[2:]
    c.check(got[2:], q[2:], M.F16, group, D ** -0.5, 0, sinks)
    for b in (dq, out, dl, dt, ds):
        if b is not None:
            b.free()
    c.close()


# ---- which keys a row sees, counted ----------------------------------------------------------------
def counted(n, H, D):
    """Values that count: key j has a one in column j % D."""
    v = np.zeros((n, H, D), np.float32)
    v[np.arange(n), :, np.arange(n) % D] = 1.0
    return v


def shares(first, last, D):
    """Of keys first..last (arrays), the part in each column."""
    d = np.arange(D)
    upto = lambda x: np.maximum(0, (x[:, None] - d) // D + 1)  # noqa: E731  keys 0..x in the column
    n = upto(last) - upto(first - 1)
    return n / np.maximum(last - first + 1, 1)[:, None]


@pytest.mark.parametrize("D,hk,group,dtype", [(128, 4, 8, "bf16"), (64, 8, 8, "bf16"), (256, 2, 8, "f16"), (128, 3, 1, "f16"),
                                              (64, 2, 6, "f16"), (256, 9, 2, "bf16")])
@pytest.mark.parametrize("lens,past,window", [([8192], 0, 0), ([8192], 0, 128), ([5000, 1, 2100], 700, 0), ([3001, 777, 4100], 64, 1000)])
def test_prefill_sees_every_key_of_a_long_prompt_once(gpu_ctx, D, hk, group, dtype, lens, past, window):
    """Scores of zero: a row is the mean of the values it sees, whose columns count them. A key too many or too few is a
    part in 128 of a column or more at 8192 keys and D = 64. All weights are one power of two, so that only the quotient (2 steps
    of 32 bits) and the output are rounded."""
    dtype = TYPES[dtype]
    cu_q = np.concatenate([[0], np.cumsum(lens)])
    cu_k = np.concatenate([[0], np.cumsum([n + past for n in lens])])
    H = hk * group
    rng = np.random.default_rng(0)
    q = np.zeros((cu_q[-1], H, D), np.float32)
    k = R.rounded(rng.normal(size=(cu_k[-1], hk, D)), dtype)
    v = np.concatenate([counted(n + past, hk, D) for n in lens])
    got = prompt(gpu_ctx, q, k, v, dtype, cu_q, cu_k, window=window)
    for s, n in enumerate(lens):
        last = past + np.arange(n)
        first = np.maximum(0, last - window + 1) if window else np.zeros(n, int)
        y = shares(first, last, D)[:, None]
        d = np.abs(got[cu_q[s]:cu_q[s + 1]] - y)
        assert (d <= (R.HALF[dtype] + 2.0 ** -22) * y + (2.0 ** -25 if dtype == M.F16 else 0)).all(), (s, np.argwhere(d.max(-1) == d.max())[0])


def check_decode_counted(ctx, fmt, D, hk, group, lens, window):
    rng = np.random.default_rng(1)
    seqs = [(rng.normal(size=(n, hk, D)).astype(np.float32), counted(n, hk, D)) for n in lens]
    kv, table = filled(ctx, fmt, seqs, page=128)
    got = decode(ctx, kv, np.zeros((len(lens), hk * group, D), np.float32), M.F16, lens, table, window=window)
    last = np.array(lens) - 1
    first = np.maximum(0, last - window + 1) if window else np.zeros(len(lens), int)
    y = shares(first, last, D)[:, None]
    assert (np.abs(got - y) <= (2.0 ** -11 + 2.0 ** -21) * y + 2.0 ** -25).all()
    kv.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,hk,group", [(64, 8, 8), (128, 4, 8), (256, 2, 8), (128, 1, 33)])
@pytest.mark.parametrize("lens,window", [([24000, 0, 1, 700, 9000], 0), ([24000, 64, 8193], 5000), ([1] * 30 + [7000], 0)])
def test_decode_sees_every_key_once(gpu_ctx, fmt, D, hk, group, lens, window):
    check_decode_counted(gpu_ctx, FORMATS[fmt], D, hk, group, lens, window)


def test_decode_of_more_sequences_than_are_split_sees_every_key_once(gpu_ctx):
    check_decode_counted(gpu_ctx, M.KV_MXFP4, 64, 1, 4, [300] * 1030 + [5000], 0)


# ---- offsets of many sequences -----------------------------------------------------------------------
@pytest.mark.parametrize("n_seqs", [513, 1500])
@pytest.mark.parametrize("at,value", [(0, -1), (1, 2 ** 31 - 1), (448, -7), (512, 0), (-1, 10 ** 6)])
def test_offsets_out_of_range_among_many_sequences(gpu_ctx, n_seqs, at, value):
    """One key offset out of range, or below the one before, anywhere: reported, and the sequences that do not have it are as
    they are without."""
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(1, 4, n_seqs)
    cu = np.concatenate([[0], np.cumsum(lens)])
    bad = cu.copy()
    bad[at] = value
    D, T = 64, int(cu[-1])
    q, k, v = (R.rounded(rng.normal(size=(T, 1, D)), M.F16) for _ in range(3))
    want = prompt(gpu_ctx, q, k, v, M.F16, cu, cu)
    rows = [R.Rows(gpu_ctx, x, M.F16) for x in (q, k, v)] + [R.Rows(gpu_ctx, None, M.F16, T, 1, D), R.i32(gpu_ctx, cu), R.i32(gpu_ctx, bad)]
    dq, dk, dv, out, dcq, dck = rows
    M.attn_prefill(gpu_ctx, D, dq.heads, dk.heads, dv.heads, T, T, n_seqs, dcq, dck, out.heads)
    sync_error(gpu_ctx, "cu_q or cu_k")
    got, at = out.get(), at % (n_seqs + 1)
    first, last = cu[max(at - 1, 0)], cu[min(at + 1, n_seqs)]
    assert (got[:first] == want[:first]).all() and (got[last:] == want[last:]).all()
    for b in rows:
        b.free()


# ---- sinks whose powers of two leave 32 bits ---------------------------------------------------------
@pytest.mark.parametrize("n", [3, 5000])
def test_finite_sinks_near_the_largest_number(gpu_ctx, n):
    """Finite sinks up to the largest have a result: nothing is left beside one, nothing is taken by a least one."""
    D, sinks = 64, np.array([3e38, np.finfo(np.float32).max, -3e38, np.finfo(np.float32).min], np.float32)
    rng = np.random.default_rng(n)
    q, k, v = (R.rounded(rng.normal(size=s), M.F16) for s in ((1, 4, D), (n, 1, D), (n, 1, D)))
    kv, table = filled(gpu_ctx, M.KV_F16, [(k, v)])
    for got in (decode(gpu_ctx, kv, q, M.F16, [n], table, sinks=sinks), prompt(gpu_ctx, q, k, v, M.F16, [0, 1], [0, n], sinks=sinks)):
        assert (got[0, :2] == 0).all()
        for h in (2, 3):
            y, av, ss, cnt = R.attend(q[0, h], k[:, 0], v[:, 0], D ** -0.5, 0, n - 1)
            assert (np.abs(got[0, h] - y) <= R.attention_bound(y, av, ss, cnt, D, M.F16, 2.0 ** -11)).all()
    kv.close()
