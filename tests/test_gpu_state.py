"""The operators over kept states on the GPU against plain 64-bit forms (attnref.py, stateref.py), at the lengths, strides, masks
and index entries where they can go wrong. Tolerances are derived where they stand."""
import numpy as np
import pytest

import moe_rocm as M

import attnref as R
import stateref as S
from test_gpu_attn import FORMATS, TYPES, sync_error

pytestmark = pytest.mark.gpu


def offsets(counts, start=0):
    return np.concatenate([[start], start + np.cumsum(counts)]).astype(np.int32)


# ---- attention of new tokens over the cache ------------------------------------------------------
class Cached:
    """A cache with sequences of the given lengths in pages in any order, and what it holds of them."""

    def __init__(self, ctx, fmt, page, hk, D, lens, rng, scale=1.0):
        self.counts = [(n + page - 1) // page for n in lens]
        n_pages = sum(self.counts) + 2
        self.kv = M.KvCache(ctx, fmt, n_pages, page, hk, D)
        order = rng.permutation(n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(1, max(self.counts, default=1))), -1, np.int32)  # unused entries: no page
        self.k, self.v, at = [], [], 0
        for i, n in enumerate(lens):
            self.table[i, :self.counts[i]] = order[at:at + self.counts[i]]
            at += self.counts[i]
            k, v = rng.normal(size=(n, hk, D)).astype(np.float32) * scale, rng.normal(size=(n, hk, D)).astype(np.float32)
            self.k.append(R.stored(k, fmt)), self.v.append(R.stored(v, fmt))
            if n == 0:
                continue
            t = np.arange(n)
            bk, bv = R.Rows(ctx, k, M.F32), R.Rows(ctx, v, M.F32)
            slots = R.i32(ctx, self.table[i][t // page] * page + t % page)
            self.kv.write(bk.heads, bv.heads, n, slots)
            ctx.sync()
            for b in (bk, bv, slots):
                b.free()


def extend_ref(q, cache, new, lens, scale, window, sinks, out_type, there=None):
    """-> (rows, bound); weights are f16 (half a step of 2^-11), see attnref.attention_bound."""
    T, hq, D = q.shape
    y, tol = np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for s, n in enumerate(new):
        hk = cache.k[s].shape[1]
        for i in range(n):
            pos = lens[s] - n + i
            for h in range(hq):
                first = max(0, pos - window + 1) if window else 0
                k, v = cache.k[s][:, h // (hq // hk)], cache.v[s][:, h // (hq // hk)]
                keep = np.arange(len(k))
                if there is not None:
                    keep = keep[there[s][:len(k)]]
                sel = keep[(keep >= first) & (keep <= pos)]
                a, size_v, size_s, seen = R.attend(q[at + i, h], k[sel], v[sel], scale, 0, len(sel) - 1,
                                                   None if sinks is None else sinks[h])
                y[at + i, h] = a
                tol[at + i, h] = R.attention_bound(a, size_v, size_s, max(seen, 1), D, out_type, 2.0 ** -11)
        at += n
    return y, tol


CASES = [
    # D, key heads, heads of each, page, new tokens, lengths, window, sinks
    (64, 2, 8, 64, [1], [1], 0, False),
    (64, 1, 1, 64, [1, 1, 1], [1, 64, 65], 0, True),
    (64, 2, 3, 128, [3, 0, 5, 1], [3, 10, 200, 0], 0, True),
    (64, 2, 8, 64, [4, 1, 2], [700, 129, 2], 128, True),
    (128, 2, 8, 64, [5, 2, 1, 7], [300, 2, 127, 193], 0, False),
    (128, 1, 5, 256, [13, 1], [13, 1000], 100, False),
    (128, 1, 16, 64, [9], [777], 0, True),
    (256, 2, 4, 64, [3, 4], [70, 400], 0, True),
    (256, 1, 8, 128, [1, 17], [600, 17], 33, False),
    (64, 1, 64, 64, [2, 1], [90, 3], 0, False),
    (128, 3, 1, 64, [40, 2], [150, 64], 0, True),
    (64, 1, 4, 64, [5], [3], 0, True),            # more new tokens than cached ones: the first rows see nothing
    (64, 2, 8, 64, [70, 1], [170, 500], 0, True),
    (128, 1, 8, 64, [90], [91], 64, False),
    (256, 1, 8, 64, [33, 1], [40, 200], 0, False),
    (64, 1, 2, 64, [130], [1300], 1, False),      # only itself
    (128, 1, 4, 64, [200, 3], [264, 320], 200, True),
    (64, 1, 8, 64, [6, 5], [500, 64], 0, True),
    (64, 2, 4, 128, [9, 13, 0, 16], [2000, 13, 5, 700], 0, False),
    (128, 1, 8, 64, [6, 8, 5], [3000, 40, 5], 0, True),
    (256, 1, 8, 64, [5, 6, 7], [400, 130, 7], 0, True),
    (256, 2, 8, 64, [3], [1500], 100, False),
]


@pytest.mark.parametrize("D,hk,group,page,new,lens,window,sinks", CASES)
@pytest.mark.parametrize("fmt,kind", [("mxfp4", "bf16"), ("mxint8", "f16"), ("f16", "bf16")])
def test_extend(gpu_ctx, D, hk, group, page, new, lens, window, sinks, fmt, kind):
    rng = np.random.default_rng(D + sum(new) + sum(lens))
    kind = TYPES[kind]
    cache = Cached(gpu_ctx, FORMATS[fmt], page, hk, D, lens, rng)
    T, hq = sum(new), hk * group
    before, after = 2, 3  # rows in no sequence
    q = R.rounded(rng.normal(size=(before + T + after, hq, D)), kind)
    sk = rng.normal(size=hq).astype(np.float32) if sinks else None
    bq, out = R.Rows(gpu_ctx, q, kind, pad=1, first=1), R.Rows(gpu_ctx, None, kind, before + T + after, hq, D, pad=2, first=1)
    dev = [R.i32(gpu_ctx, a) for a in (offsets(new, before), lens, cache.table)]
    ds = gpu_ctx.to_device(sk) if sinks else None
    for _ in range(2):
        cache.kv.extend(bq.heads, before + T + after, len(new), dev[0], dev[1], dev[2], cache.table.shape[1], out.heads,
                        window=window, sinks=ds)
        gpu_ctx.sync()
        got = out.get()
        y, tol = extend_ref(q[before:before + T], cache, new, lens, D ** -0.5, window, sk, kind)
        assert (np.abs(got[before:before + T] - y) <= tol).all(), float((np.abs(got[before:before + T] - y) / tol).max())
        mark = R.from_bits(np.array([out.mark]), kind)[0]
        assert (got[:before] == mark).all() and (got[before + T:] == mark).all()
    for b in (bq, out, *dev):
        b.free()
    if ds is not None:
        ds.free()
    cache.kv.close()


def test_extend_of_single_tokens_is_decode(gpu_ctx):
    rng = np.random.default_rng(3)
    lens = [1, 0, 700, 1300, 64]
    cache = Cached(gpu_ctx, M.KV_MXFP4, 64, 2, 128, lens, rng)
    q = R.rounded(rng.normal(size=(5, 16, 128)), M.BF16)
    bq, o1, o2 = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, 5, 16, 128), R.Rows(gpu_ctx, None, M.BF16, 5, 16, 128)
    cu, dl, dt = (R.i32(gpu_ctx, a) for a in (offsets([1] * 5), lens, cache.table))
    cache.kv.attend(bq.heads, 5, dl, dt, cache.table.shape[1], o1.heads)
    cache.kv.extend(bq.heads, 5, 5, cu, dl, dt, cache.table.shape[1], o2.heads)
    gpu_ctx.sync()
    # the same sums in other orders: a step of the outputs' type at most
    a, b = o1.get(), o2.get()
    assert (np.abs(a - b) <= 2 * 2.0 ** -8 * np.abs(a) + 1e-6).all()
    for x in (bq, o1, o2, cu, dl, dt):
        x.free()
    cache.kv.close()


def test_extend_entries_out_of_range(gpu_ctx):
    rng = np.random.default_rng(5)
    lens, new = [200, 130], [4, 2]
    cache = Cached(gpu_ctx, M.KV_MXINT8, 64, 1, 64, lens, rng)
    q = R.rounded(rng.normal(size=(6, 4, 64)), M.BF16)
    bq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, 6, 4, 64)
    mp = cache.table.shape[1]

    def run(cu, ln, table):
        dev = [R.i32(gpu_ctx, a) for a in (cu, ln, table)]
        cache.kv.extend(bq.heads, 6, 2, *dev, mp, out.heads)
        return dev

    # a page that is not there: its tokens are left out
    table = cache.table.copy()
    table[0, 1] = 10 ** 6
    dev = run(offsets(new), lens, table)
    sync_error(gpu_ctx, "block_table")
    there = [np.ones(200, bool), np.ones(130, bool)]
    there[0][64:128] = False
    y, tol = extend_ref(q, cache, new, lens, 0.125, 0, None, M.BF16, there)
    assert (np.abs(out.get() - y) <= tol).all()
    # a length beyond the table is the table's: the queries stand at its end, pages there are missing
    dev += run(offsets(new), [10 ** 9, 130], cache.table)
    sync_error(gpu_ctx, "seq_len")
    # offsets out of range and out of order
    for cu in ([0, 4, 9], [-3, 4, 6], [5, 2, 6]):
        dev += run(np.array(cu, np.int32), lens, cache.table)
        sync_error(gpu_ctx, "cu_q")
    for b in (bq, out, *dev):
        b.free()
    cache.kv.close()


@pytest.mark.parametrize("new", [1, 12, 30])
def test_extend_of_overlapping_offsets(gpu_ctx, new):
    """Every other sequence claims all rows: an error, rows that hold some sequence's result or none, and nothing written elsewhere."""
    n_seqs, n = 60, 3000
    T = new * n_seqs
    rng = np.random.default_rng(new)
    cache = Cached(gpu_ctx, M.KV_MXFP4, 64, 1, 64, [n], rng)
    table = np.repeat(cache.table, n_seqs, 0)
    q = R.rounded(rng.normal(size=(T, 4, 64)), M.BF16)
    bq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, T, 4, 64)
    cu = np.array([T * (s & 1) for s in range(n_seqs + 1)], np.int32)
    dev = [R.i32(gpu_ctx, a) for a in (cu, [n] * n_seqs, table)]
    cache.kv.extend(bq.heads, T, n_seqs, *dev, table.shape[1], out.heads)
    sync_error(gpu_ctx, "cu_q")
    assert np.isfinite(out.get()).all()
    # the same call with offsets in order
    dev[0].upload(offsets([new] * n_seqs))
    cache.kv.extend(bq.heads, T, n_seqs, *dev, table.shape[1], out.heads)
    gpu_ctx.sync()
    some = slice(7 * new, 8 * new)
    y, tol = extend_ref(q[some], cache, [new], [n], 0.125, 0, None, M.BF16)
    assert (np.abs(out.get()[some] - y) <= tol).all()
    for b in (bq, out, *dev):
        b.free()
    cache.kv.close()


# ---- causal convolution --------------------------------------------------------------------------
@pytest.mark.parametrize("C_,new", [(8, [1]), (64, [1, 1, 1, 1, 1]), (520, [2, 0, 5, 1, 33]), (2056, [16, 17, 15, 4, 3]),
                                    (4104, [100, 1]), (64, [0, 0, 3])])
@pytest.mark.parametrize("taps,silu,bias,src,dst", [(4, True, False, "bf16", "bf16"), (4, False, True, "f32", "f32"),
                                                    (3, True, True, "f16", "f32"), (2, True, False, "f32", "f16")])
@pytest.mark.parametrize("in_place", [False, True])
def test_conv(gpu_ctx, C_, new, taps, silu, bias, src, dst, in_place):
    rng = np.random.default_rng(C_ + taps)
    src, dst, n = TYPES[src], TYPES[dst], len(new)
    T, before, after, P = sum(new), 1, 2, taps - 1
    x = R.rounded(rng.normal(size=(before + T + after, 1, C_)) * 2, src)
    w = (rng.normal(size=(C_, taps)) / 2).astype(np.float32)
    b = rng.normal(size=C_).astype(np.float32) if bias else None
    states = rng.normal(size=(2 * n + 1, P, C_)).astype(np.float32)
    source = rng.permutation(n).astype(np.int32)
    source[n // 2] = -1
    target = source.copy() if in_place else (np.arange(n) + n).astype(np.int32)
    if not in_place:
        target[n - 1] = -1
    bx, out = R.Rows(gpu_ctx, x, src, pad=1), R.Rows(gpu_ctx, None, dst, before + T + after, 1, C_, pad=2)
    dw, db, dst_states = gpu_ctx.to_device(w), gpu_ctx.to_device(b) if bias else None, gpu_ctx.to_device(states)
    dev = [R.i32(gpu_ctx, a) for a in (offsets(new, before), source, target)]
    M.causal_conv(gpu_ctx, M.Rows(bx.buf, C_, src, bx.width), dw, taps, before + T + after, n, dev[0],
                  M.Rows(out.buf, C_, dst, out.width), bias=db, silu=silu, states=dst_states, n_slots=2 * n + 1,
                  source=dev[1], target=dev[2])
    gpu_ctx.sync()
    got, kept = out.get()[:, 0], dst_states.download(np.float32).reshape(states.shape)
    want, at = states.astype(np.float64).copy(), before
    for s, m in enumerate(new):
        old = states[source[s]] if source[s] >= 0 else np.zeros((P, C_))
        y, off, last = S.conv(x[at:at + m, 0], w, b, silu, old)
        tol = off + R.HALF[dst] * np.abs(y) * 1.01 * (dst != M.F32) + 2.0 ** -25 * (dst == M.F16)
        assert (np.abs(got[at:at + m] - y) <= tol).all(), (s, float((np.abs(got[at:at + m] - y) / tol).max()))
        if target[s] >= 0:
            want[target[s]] = last
        at += m
    assert (kept == want).all()  # inputs, as they are
    mark = R.from_bits(np.array([out.mark]), dst)[0]
    assert (got[:before] == mark).all() and (got[before + T:] == mark).all()
    for a in (bx, out, dw, dst_states, *dev):
        a.free()
    if bias:
        db.free()


# ---- gated delta rule ----------------------------------------------------------------------------
class Delta:
    """Inputs of a call, its device copies, and a run of it."""

    def __init__(self, ctx, kh, vh, dk, dv, new, kind, raw, rng, states=None, strong=False):
        self.ctx, self.kh, self.vh, self.dk, self.dv, self.new, self.kind, self.raw = ctx, kh, vh, dk, dv, new, kind, raw
        T = self.T = sum(new) + 3
        self.q, self.k = (R.rounded(rng.normal(size=(T, kh, dk)), kind) for _ in range(2))
        self.v = R.rounded(rng.normal(size=(T, vh, dv)) * 2, kind)
        self.a, self.b = (rng.normal(size=(T, vh + 2)).astype(np.float32) for _ in range(2))
        self.a_log = rng.uniform(-1, 2, vh).astype(np.float32) if raw else None
        self.dt_bias = rng.uniform(-4, 0, vh).astype(np.float32) if raw else None
        self.eps = 1e-6 if raw else 0.0
        if not raw:
            self.a = -np.abs(self.a) * np.float32(20.0 if strong else 0.3)
            self.b = (1 / (1 + np.exp(-self.b))).astype(np.float32)
            self.q, self.k = (R.rounded(x / np.sqrt((x * x).sum(-1, keepdims=True)), kind) for x in (self.q, self.k))
        n = len(new)
        self.states = (rng.normal(size=(2 * n + 1, vh, dk, dv)) if states is None else states).astype(np.float32)
        self.source = rng.permutation(n).astype(np.int32)
        self.target = (np.arange(n) + n).astype(np.int32)

    def run(self, in_place=False, start=1, cu=None, error=None):
        c, n = self.ctx, len(self.new)
        if in_place:
            self.target = self.source.copy()
        self.start = start
        rows = [R.Rows(c, self.q, self.kind, pad=self.kh + self.vh, first=0), R.Rows(c, self.k, self.kind, pad=1, first=1),
                R.Rows(c, self.v, self.kind), R.Rows(c, None, self.kind, self.T, self.vh, self.dv, pad=1, first=1)]
        flat = [c.to_device(x) for x in (self.a, self.b, self.states)]
        gate = [c.to_device(x) for x in (self.a_log, self.dt_bias)] if self.raw else [None, None]
        dev = [R.i32(c, x) for x in (offsets(self.new, start) if cu is None else cu, self.source, self.target)]
        rule = M.DeltaRule(c, self.kh, self.vh, self.dk, self.dv, unit_eps=self.eps, gate_stride=self.vh + 2, a_log=gate[0],
                           dt_bias=gate[1])
        rule.forward(rows[0].heads, rows[1].heads, rows[2].heads, flat[0], flat[1], self.T, n, dev[0], rows[3].heads,
                     states=flat[2], n_slots=len(self.states), source=dev[1], target=dev[2])
        if error:
            sync_error(c, error)
        else:
            c.sync()
        self.mark = R.from_bits(np.array([rows[3].mark]), self.kind)[0]
        self.out, self.kept = rows[3].get(), flat[2].download(np.float32).reshape(self.states.shape)
        rule.close()
        for x in (*rows, *flat, *dev):
            x.free()
        for x in gate:
            if x is not None:
                x.free()

    def check(self):
        g, beta, g_off, b_off = S.gates(self.a[:, :self.vh], self.b[:, :self.vh], self.a_log, self.dt_bias)
        want, bound, at = self.states.astype(np.float64), np.zeros(self.states.shape), self.start
        half = R.HALF[self.kind]
        for s, n in enumerate(self.new):
            for h in range(self.vh):
                hk = h // (self.vh // self.kh)
                old = self.states[self.source[s], h] if self.source[s] >= 0 else np.zeros((self.dk, self.dv))
                i = slice(at, at + n)
                y, off, last, e = S.delta(self.q[i, hk], self.k[i, hk], self.v[i, h], g[i, h], beta[i, h], old, self.dk ** -0.5,
                                          self.eps, g_off[i, h], b_off[i, h])
                tol = off * (1 + half) + half * np.abs(y) * 1.01 + 2.0 ** -25 * (self.kind == M.F16)
                d = np.abs(self.out[i, h] - y)
                assert (d <= tol).all(), (s, h, n, float((d / tol).max()))
                if self.target[s] >= 0:
                    want[self.target[s], h], bound[self.target[s], h] = last, e + 1e-37
            at += n
        d = np.abs(self.kept - want)
        assert (d <= bound).all(), float((d / np.maximum(bound, 1e-37)).max())
        assert (self.out[:self.start] == self.mark).all() and (self.out[at:] == self.mark).all()
        return float((d / np.maximum(bound, 1e-37)).max())


LENGTHS = [[1], [1, 1, 1], [2, 0, 5, 1], [9, 17, 8], [64, 1, 65, 63], [130, 3], [128, 127], [200]]


@pytest.mark.parametrize("new", LENGTHS)
@pytest.mark.parametrize("kh,vh,dk,dv", [(1, 1, 128, 128), (2, 4, 128, 128), (1, 3, 64, 128), (2, 2, 128, 64), (1, 2, 64, 64)])
@pytest.mark.parametrize("kind,raw", [("bf16", True), ("f16", False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_delta(gpu_ctx, new, kh, vh, dk, dv, kind, raw, in_place):
    rng = np.random.default_rng(sum(new) + 7 * dk + dv)
    c = Delta(gpu_ctx, kh, vh, dk, dv, new, TYPES[kind], raw, rng)
    c.source[len(new) // 2] = -1  # starts from zeros
    c.run(in_place)
    if not in_place and len(new) > 1:
        assert (c.kept[:len(new)] == c.states[:len(new)]).all()  # the states before stay
    c.check()


# lengths about the one up to which sequences go token by token: 12 and more, by the number of sequences and heads
@pytest.mark.parametrize("new", [[11], [12], [13], [14], [12, 13, 14], [32, 33, 31], [13] * 9])
@pytest.mark.parametrize("kh,vh,dk,dv,kind", [(1, 2, 128, 128, "bf16"), (1, 2, 64, 128, "f16"), (4, 16, 64, 64, "bf16")])
def test_delta_at_the_border_of_its_paths(gpu_ctx, new, kh, vh, dk, dv, kind):
    c = Delta(gpu_ctx, kh, vh, dk, dv, new, TYPES[kind], False, np.random.default_rng(sum(new) + vh))
    c.run()
    c.check()


@pytest.mark.parametrize("new", [[1, 3], [150, 70]])
def test_delta_decays_of_any_size(gpu_ctx, new):
    rng = np.random.default_rng(8)
    c = Delta(gpu_ctx, 1, 2, 128, 128, new, M.BF16, False, rng, strong=True)
    c.a[::5] = -np.inf  # forgets all
    c.a[1::7] = -1000.0
    c.a[2::9] = 0.0
    c.b[3::11] = 0.0
    c.b[4::11] = 1.0
    c.run()
    c.check()


def test_delta_of_no_state(gpu_ctx):
    """Without slots sequences start from zeros and nothing is kept."""
    rng = np.random.default_rng(9)
    c = Delta(gpu_ctx, 1, 1, 64, 64, [5, 100], M.F16, False, rng)
    rows = [R.Rows(gpu_ctx, x, M.F16) for x in (c.q, c.k, c.v)] + [R.Rows(gpu_ctx, None, M.F16, c.T, 1, 64)]
    a, b, cu = gpu_ctx.to_device(c.a), gpu_ctx.to_device(c.b), R.i32(gpu_ctx, offsets(c.new, 1))
    rule = M.DeltaRule(gpu_ctx, 1, 1, 64, 64, gate_stride=3)
    rule.forward(rows[0].heads, rows[1].heads, rows[2].heads, a, b, c.T, 2, cu, rows[3].heads)
    gpu_ctx.sync()
    c.out, c.kept, c.start, c.mark = rows[3].get(), c.states, 1, -7.5
    c.source[:], c.target[:] = -1, -1
    c.check()
    rule.close()
    for x in (*rows, a, b, cu):
        x.free()


def test_delta_slots_out_of_range(gpu_ctx):
    rng = np.random.default_rng(10)
    for new in ([2, 3], [90, 70]):
        c = Delta(gpu_ctx, 1, 1, 64, 64, new, M.BF16, False, rng)
        c.source[0], c.target[1] = 5, 10 ** 9  # 5 slots
        c.run(error="source or target")
        c.source[0], c.target[1] = -1, -1
        c.check()


@pytest.mark.parametrize("what", ["value", "key", "beta", "decay", "query"])
@pytest.mark.parametrize("at", [0, 20, 63, 64, 100])
def test_delta_what_is_not_finite_reaches_no_earlier_token(gpu_ctx, what, at):
    """A value that is not finite reaches its column from its token on, a key, decay or beta all columns, a query its row."""
    rng = np.random.default_rng(at)
    n, dv = 140, 64
    c = Delta(gpu_ctx, 1, 2, 64, dv, [n], M.BF16, False, rng)
    row = at + 1
    clean = c.v.copy(), c.k.copy(), c.b.copy(), c.a.copy(), c.q.copy()
    if what == "value":
        c.v[row, 1, 5] = np.inf
    if what == "key":
        c.k[row, 0, 3] = np.nan
    if what == "beta":
        c.b[row, 1] = np.nan
    if what == "decay":
        c.a[row, 1] = np.inf
    if what == "query":
        c.q[row, 0, 9] = np.nan
    c.run()
    out, kept, target = c.out, c.kept, c.target
    c.v, c.k, c.b, c.a, c.q = clean
    c.run()
    c.check()
    hit = np.zeros(out.shape, bool)
    if what == "value":
        hit[row:n + 1, 1, 5] = True
    if what == "key":
        hit[row:n + 1] = True
    if what in ("beta", "decay"):
        hit[row:n + 1, 1] = True
    if what == "query":
        hit[row] = True
    assert not np.isfinite(out[hit]).any()
    assert (out[~hit] == c.out[~hit]).all()
    assert not np.isfinite(kept[target[0]][hit[n].nonzero()[0][:1]]).all() if what in ("key", "beta", "decay") else True
    if what == "query":
        assert (kept == c.kept).all()
    if what == "value":
        assert not np.isfinite(kept[target[0], 1, :, 5]).any()
        mask = np.ones((2, 64, dv), bool)
        mask[1, :, 5] = False
        assert (kept[target[0]][mask] == c.kept[target[0]][mask]).all()


def test_delta_of_more_chunks_than_the_workspace_holds(gpu_ctx):
    """256 heads of 128 leave room for about ten chunks at once: two sequences cross from one launch to the next."""
    rng = np.random.default_rng(11)
    new = [40, 1000, 3, 700, 65]
    c = Delta(gpu_ctx, 256, 256, 128, 128, new, M.BF16, False, rng, states=np.zeros((11, 256, 128, 128)))
    c.source[:] = -1
    c.run()
    heads = [0, 100, 255]
    g, beta, g_off, b_off = S.gates(c.a[:, :256], c.b[:, :256], None, None)
    at = 1
    for s, n in enumerate(new):
        for h in heads:
            i = slice(at, at + n)
            y, off, last, e = S.delta(c.q[i, h], c.k[i, h], c.v[i, h], g[i, h], beta[i, h], np.zeros((128, 128)), 128 ** -0.5, 0.0,
                                      g_off[i, h], b_off[i, h])
            assert (np.abs(c.out[i, h] - y) <= off * 1.01 + 2.0 ** -8 * np.abs(y)).all(), (s, h)
            assert (np.abs(c.kept[c.target[s], h] - last) <= e + 1e-37).all(), (s, h)
        at += n


@pytest.mark.parametrize("cu", [[0, 2, 400], [-3, 4, 160], [100, 0, 120], [160, 160, 0], [2 ** 30, -2 ** 31, 2 ** 31 - 1]])
@pytest.mark.parametrize("most", [20, 160])
def test_offsets_out_of_range(gpu_ctx, cu, most):
    """They end in an error, whichever path takes them, and what is right in them has its result."""
    rng = np.random.default_rng(11)
    cu = np.array([min(x, x * most // 160) if abs(x) < 1000 else x for x in cu], np.int32)
    c = Delta(gpu_ctx, 1, 1, 64, 64, [most - 3], M.BF16, False, rng)
    c.new, c.source, c.target = [0, 0], np.array([-1, -1], np.int32), np.array([0, 1], np.int32)
    c.run(cu=cu, error="cu")
    x = R.rounded(rng.normal(size=(most, 1, 64)), M.BF16)
    w, bx, out = gpu_ctx.to_device(np.ones((64, 4), np.float32)), R.Rows(gpu_ctx, x, M.BF16), R.Rows(gpu_ctx, None, M.F32, most, 1, 64)
    dev = R.i32(gpu_ctx, cu)
    M.causal_conv(gpu_ctx, M.Rows(bx.buf, 64, M.BF16), w, 4, most, 2, dev, M.Rows(out.buf, 64))
    sync_error(gpu_ctx, "cu")
    got = out.get()[:, 0]
    first, last = np.clip(cu[:2], 0, most)
    if first == 0 and last > 0:
        y, off, _ = S.conv(x[:last, 0], np.ones((64, 4)), None, False, np.zeros((3, 64)))
        assert (np.abs(got[:last] - y) <= off).all()
    for b in (w, bx, out, dev):
        b.free()


def test_kernel_names(gpu_ctx):
    """The documented names count launches."""
    rng = np.random.default_rng(13)
    l = Layer(gpu_ctx, rng, 2, 130, [3000, 2])
    l.set([100, 2], [3000, 2])
    gpu_ctx.set_option(M.OPT_PROFILE, 1)
    gpu_ctx.profile_reset()
    l.call()
    gpu_ctx.sync()
    counts = {k: gpu_ctx.profile_read(k)[0] for k in ("attn_extend", "extend_join", "causal_conv", "delta_step", "delta_prepare", "delta_chunks")}
    gpu_ctx.set_option(M.OPT_PROFILE, 0)
    assert all(n == 1 for n in counts.values()), counts
    l.close()


@pytest.mark.parametrize("n", [40, 70, 108, 109, 110, 130])  # 14 * 8 rows, 3 of them in no sequence, are the most that all go token by token
def test_delta_of_one_long_sequence_among_empty_ones(gpu_ctx, n):
    rng = np.random.default_rng(12)
    c = Delta(gpu_ctx, 1, 1, 64, 64, [0] * 20 + [n] + [0] * 19, M.BF16, False, rng)
    c.run()
    c.check()


@pytest.mark.parametrize("n_seqs", [70, 1100])
def test_many_sequences(gpu_ctx, n_seqs):
    """More sequences than a wave has lanes, and than are looked through one by one: some long, most short."""
    rng = np.random.default_rng(n_seqs)
    new = rng.integers(0, 4, n_seqs)
    new[[3, n_seqs // 2, n_seqs - 1]] = [80, 40, 130]
    new = new.tolist()
    c = Delta(gpu_ctx, 1, 1, 64, 64, new, M.F16, False, rng)
    c.run()
    c.check()

    T, P, C_ = sum(new), 3, 64
    x = R.rounded(rng.normal(size=(T, 1, C_)), M.BF16)
    w = rng.normal(size=(C_, 4)).astype(np.float32)
    states = rng.normal(size=(n_seqs, P, C_)).astype(np.float32)
    bx, out = R.Rows(gpu_ctx, x, M.BF16), R.Rows(gpu_ctx, None, M.F32, T, 1, C_)
    dev = [gpu_ctx.to_device(w), gpu_ctx.to_device(states), R.i32(gpu_ctx, offsets(new)), R.i32(gpu_ctx, np.arange(n_seqs))]
    M.causal_conv(gpu_ctx, M.Rows(bx.buf, C_, M.BF16), dev[0], 4, T, n_seqs, dev[2], M.Rows(out.buf, C_), states=dev[1],
                  n_slots=n_seqs, source=dev[3], target=dev[3])
    gpu_ctx.sync()
    got, kept, at = out.get()[:, 0], dev[1].download(np.float32).reshape(states.shape), 0
    for s, m in enumerate(new):
        y, off, last = S.conv(x[at:at + m, 0], w, None, False, states[s])
        assert (np.abs(got[at:at + m] - y) <= off).all() and (kept[s] == last).all()
        at += m
    for b in (bx, out, *dev):
        b.free()

    lens = [n + int(k) for n, k in zip(new, rng.integers(0, 100, n_seqs))]
    lens[3] = 900
    cache = Cached(gpu_ctx, M.KV_MXFP4, 64, 1, 64, lens, rng)
    q = R.rounded(rng.normal(size=(T, 2, 64)), M.BF16)
    bq, o = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, T, 2, 64)
    idx = [R.i32(gpu_ctx, a) for a in (offsets(new), lens, cache.table)]
    cache.kv.extend(bq.heads, T, n_seqs, *idx, cache.table.shape[1], o.heads)
    gpu_ctx.sync()
    y, tol = extend_ref(q, cache, new, lens, 0.125, 0, None, M.BF16)
    assert (np.abs(o.get() - y) <= tol).all()
    for b in (bq, o, *idx):
        b.free()
    cache.kv.close()


def test_extend_of_a_page_behind_4_gib(gpu_ctx):
    rng = np.random.default_rng(14)
    hk, D, pages = 8, 256, 8400  # pages of 512 KiB
    assert M.KvCache.nbytes(M.KV_F16, pages, 64, hk, D) > 2 ** 32
    kv = M.KvCache(gpu_ctx, M.KV_F16, pages, 64, hk, D)
    n, table = 130, np.array([[pages - 1, 3, pages - 2]], np.int32)
    k, v = (rng.normal(size=(n, hk, D)).astype(np.float32) for _ in range(2))
    t = np.arange(n)
    bk, bv, slots = R.Rows(gpu_ctx, k, M.F32), R.Rows(gpu_ctx, v, M.F32), R.i32(gpu_ctx, table[0][t // 64] * 64 + t % 64)
    kv.write(bk.heads, bv.heads, n, slots)
    for new in (1, 5, 90):
        q = R.rounded(rng.normal(size=(new, hk * 2, D)), M.BF16)
        bq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, new, hk * 2, D)
        dev = [R.i32(gpu_ctx, a) for a in ([0, new], [n], table)]
        kv.extend(bq.heads, new, 1, *dev, 3, out.heads)
        gpu_ctx.sync()
        c = type("C", (), {"k": [R.stored(k, M.KV_F16)], "v": [R.stored(v, M.KV_F16)]})
        y, tol = extend_ref(q, c, [new], [n], D ** -0.5, 0, None, M.BF16)
        assert (np.abs(out.get() - y) <= tol).all()
        for b in (bq, out, *dev):
            b.free()
    for b in (bk, bv, slots):
        b.free()
    kv.close()


# scores that 16 bits do not hold, scores far apart, sinks and queries that are not finite
@pytest.mark.parametrize("new", [1, 3, 12, 40])  # each form of the kernel
@pytest.mark.parametrize("D", [64, 256])
def test_extend_extremes(gpu_ctx, new, D):
    rng = np.random.default_rng(new)
    n, group = 300, 4
    cache = Cached(gpu_ctx, M.KV_F16, 64, 1, D, [n], rng)
    q = rng.normal(size=(new, group, D))
    q[:, 1] *= 1e6      # scores of 10^6 and more: nearly one key each
    q[:, 2] *= 1e-30    # all keys alike
    q = R.rounded(q, M.BF16)
    q[0, 3, 5] = np.nan
    sinks = np.array([-np.inf, 3.0, 1.0, 0.0], np.float32)
    bq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, new, group, D)
    dev = [R.i32(gpu_ctx, a) for a in ([0, new], [n], cache.table)]
    for s, scale in ((sinks, 0.0), (None, 0.0), (sinks, -0.3), (None, 1e-30)):
        ds = gpu_ctx.to_device(s) if s is not None else None
        cache.kv.extend(bq.heads, new, 1, *dev, cache.table.shape[1], out.heads, scale=scale, sinks=ds)
        gpu_ctx.sync()
        got = out.get()
        assert np.isnan(got[0, 3]).all()
        q1 = np.where(np.isnan(q), 0, q)
        y, tol = extend_ref(q1, cache, [new], [n], scale or D ** -0.5, 0, s, M.BF16)
        ok = np.abs(got - y) <= tol
        ok[0, 3] = True
        assert ok.all(), np.argwhere(~ok)[:4]
        if ds is not None:
            ds.free()
    for bad in (np.inf, np.nan):
        s = np.array([1.0, bad, 0.0, 0.0], np.float32)
        ds = gpu_ctx.to_device(s)
        cache.kv.extend(bq.heads, new, 1, *dev, cache.table.shape[1], out.heads, sinks=ds)
        gpu_ctx.sync()
        got = out.get()
        assert np.isnan(got[:, 1]).all() and np.isfinite(got[:, 0]).all() and np.isfinite(got[:, 2]).all()
        ds.free()
    for b in (bq, out, *dev):
        b.free()
    cache.kv.close()


@pytest.mark.parametrize("new", [1, 12, 40])
def test_extend_weights_far_below_the_largest(gpu_ctx, new):
    """A first key 17 above the rest that has no value: the rest's weights, 2^-24.5 of the largest, keep their bits."""
    n, D, group = 2000, 64, 4
    rng = np.random.default_rng(1)
    cache = Cached(gpu_ctx, M.KV_F16, 64, 1, D, [n], rng, scale=0.0)
    k, v = np.zeros((1, 1, D), np.float32), np.zeros((1, 1, D), np.float32)
    k[0, 0, 0] = 17.0
    bk, bv, slot = R.Rows(gpu_ctx, k, M.F32), R.Rows(gpu_ctx, v, M.F32), R.i32(gpu_ctx, [cache.table[0, 0] * 64])
    cache.kv.write(bk.heads, bv.heads, 1, slot)
    cache.k[0][0], cache.v[0][0] = k[0], 0.0
    q = np.zeros((new, group, D))
    q[..., 0] = 1.0
    bq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, new, group, D)
    dev = [R.i32(gpu_ctx, a) for a in ([0, new], [n], cache.table)]
    cache.kv.extend(bq.heads, new, 1, *dev, cache.table.shape[1], out.heads, scale=1.0)
    gpu_ctx.sync()
    y, _ = extend_ref(q, cache, [new], [n], 1.0, 0, None, M.BF16)
    # a weight is off by 2^-11 of itself (its sum too), the output by its own rounding
    w = np.abs(cache.v[0]).mean() * n * np.exp(-17.0)
    assert (np.abs(out.get() - y) <= 2.0 ** -8 * np.abs(y) + 2.0 ** -10 * w).all()
    for b in (bk, bv, slot, bq, out, *dev):
        b.free()
    cache.kv.close()


# ---- graphs, streams, as they are used ----------------------------------------------------------------
class Layer:
    """A linear layer's convolution and rule, and an attention layer's cache, over the same new tokens."""

    def __init__(self, ctx, rng, n_seqs, most, lens):
        self.ctx, self.n, self.T, self.kh, self.vh, self.D = ctx, n_seqs, most, 2, 4, 64
        C_ = self.C = (2 * self.kh + self.vh) * self.D
        self.w = (rng.normal(size=(C_, 4)) / 2).astype(np.float32)
        self.x = R.rounded(rng.normal(size=(most, 1, C_)), M.BF16)
        self.g, self.b = -np.abs(rng.normal(size=(most, self.vh))).astype(np.float32), rng.uniform(0.1, 0.9, (most, self.vh)).astype(np.float32)
        self.conv_states = rng.normal(size=(2 * n_seqs, 3, C_)).astype(np.float32)
        self.states = (rng.normal(size=(2 * n_seqs, self.vh, self.D, self.D)) * 0.1).astype(np.float32)
        self.q = R.rounded(rng.normal(size=(most, 8, 64)), M.BF16)
        self.cache = Cached(ctx, M.KV_MXINT8, 64, 2, 64, lens, rng)
        self.rule = M.DeltaRule(ctx, self.kh, self.vh, self.D, self.D, unit_eps=1e-6)
        up = ctx.to_device
        self.d = dict(w=up(self.w), x=R.Rows(ctx, self.x, M.BF16), y=R.Rows(ctx, None, M.BF16, most, 1, C_), g=up(self.g), b=up(self.b),
                      cs=up(self.conv_states), s=up(self.states), o=R.Rows(ctx, None, M.BF16, most, self.vh, self.D),
                      q=R.Rows(ctx, self.q, M.BF16), a=R.Rows(ctx, None, M.BF16, most, 8, 64), cu=R.i32(ctx, np.zeros(n_seqs + 1)),
                      len=R.i32(ctx, np.zeros(n_seqs)), table=R.i32(ctx, self.cache.table), src=R.i32(ctx, np.arange(n_seqs)),
                      dst=R.i32(ctx, np.arange(n_seqs) + n_seqs))

    def call(self):
        d, D, s = self.d, self.D, 2
        M.causal_conv(self.ctx, M.Rows(d["x"].buf, self.C, M.BF16), d["w"], 4, self.T, self.n, d["cu"], M.Rows(d["y"].buf, self.C, M.BF16),
                      silu=True, states=d["cs"], n_slots=2 * self.n, source=d["src"], target=d["dst"])
        at = lambda first, heads: M.Heads(d["y"].buf.ptr + first * D * s, heads, M.BF16, self.C, D)  # noqa: E731
        self.rule.forward(at(0, self.kh), at(self.kh, self.kh), at(2 * self.kh, self.vh), d["g"], d["b"], self.T, self.n, d["cu"],
                          d["o"].heads, states=d["s"], n_slots=2 * self.n, source=d["src"], target=d["dst"])
        self.cache.kv.extend(d["q"].heads, self.T, self.n, d["cu"], d["len"], d["table"], self.cache.table.shape[1], d["a"].heads)

    def set(self, new, lens):
        self.ctx.sync()
        for name, x in (("cu", offsets(new)), ("len", lens)):
            self.d[name].upload(np.asarray(x, np.int32))
        for name in ("y", "o", "a"):
            self.d[name].buf.upload(np.full(self.d[name].buf.nbytes // 2, self.d[name].mark, np.uint16))
        self.d["cs"].upload(self.conv_states), self.d["s"].upload(self.states)

    def results(self):
        self.ctx.sync()
        return [self.d[n].all().copy() for n in ("y", "o", "a")] + [self.d[n].download(np.float32).copy() for n in ("cs", "s")]

    def close(self):
        self.rule.close(), self.cache.kv.close()
        for x in self.d.values():
            x.free()


def test_graphs_see_present_offsets_and_share_their_scratch(gpu_ctx):
    """Two captured graphs of all three calls, replayed in turn with other offsets and lengths, and eager calls between: the same bits."""
    rng = np.random.default_rng(20)
    layers = [Layer(gpu_ctx, rng, 3, 160, [900, 400, 64]), Layer(gpu_ctx, rng, 2, 90, [1500, 200])]
    plans = [[([1, 1, 1], [900, 300, 1]), ([100, 0, 60], [500, 7, 60]), ([40, 33, 2], [41, 400, 64])],
             [([90, 0], [1500, 0]), ([1, 5], [1300, 200]), ([33, 57], [33, 199])]]
    want = []
    for l, plan in zip(layers, plans):
        want.append([])
        for new, lens in plan:
            l.set(new, lens)
            l.call()
            want[-1].append(l.results())
    graphs = []
    for l in layers:
        gpu_ctx.graph_begin()
        l.call()
        graphs.append(gpu_ctx.graph_end())
    for step in (0, 2, 1, 0, 1):
        for l, plan in zip(layers, plans):
            l.set(*plan[step])
        for g in graphs:
            g.launch()
        for l, w in zip(layers, want):
            for a, b in zip(l.results(), w[step]):
                assert np.array_equal(a, b, equal_nan=True)
        layers[0].set(*plans[0][step])
        layers[0].call()  # eager, on the same scratch
        for a, b in zip(layers[0].results(), want[0][step]):
            assert np.array_equal(a, b, equal_nan=True)
    for g in graphs:
        g.close()
    for l in layers:
        l.close()


def test_parts_of_a_prompt_follow_each_other(gpu_ctx):
    """A prompt in one call and in parts, states and cache carried on: the same to the rounding of what is carried, which is none (conv)
    or that of 32-bit sums (rule); attention over the cache does not carry at all."""
    rng = np.random.default_rng(21)
    n = 150
    l = Layer(gpu_ctx, rng, 1, n, [n])
    l.conv_states[:], l.states[:] = 0, 0
    l.set([n], [n])
    l.call()
    whole = l.results()
    l.set([n], [n])
    d, at = l.d, 0
    d["src"].upload(np.array([-1], np.int32))
    for part in (1, 64, 3, 40, 33, 9):
        x, y, o = (l.d[k].buf.ptr + at * w for k, w in (("x", l.C * 2), ("y", l.C * 2), ("o", l.vh * l.D * 2)))
        cu, ln = R.i32(gpu_ctx, [0, part]), R.i32(gpu_ctx, [at + part])
        kw = dict(n_slots=2, source=d["src"], target=d["dst"])
        M.causal_conv(gpu_ctx, M.Rows(x, l.C, M.BF16), d["w"], 4, part, 1, cu, M.Rows(y, l.C, M.BF16), silu=True, states=d["cs"], **kw)
        h = lambda first, heads: M.Heads(y + first * l.D * 2, heads, M.BF16, l.C, l.D)  # noqa: E731, B023
        l.rule.forward(h(0, 2), h(2, 2), h(4, 4), d["g"].ptr + at * 16, d["b"].ptr + at * 16, part, 1, cu, M.Heads(o, 4, M.BF16), states=d["s"], **kw)
        l.cache.kv.extend(M.Heads(d["q"].buf.ptr + at * 1024, 8, M.BF16), part, 1, cu, ln, d["table"], l.cache.table.shape[1],
                          M.Heads(d["a"].buf.ptr + at * 1024, 8, M.BF16))
        gpu_ctx.sync()
        d["src"].upload(np.array([1], np.int32))
        cu.free(), ln.free()
        at += part
    parts = l.results()
    assert (parts[0] == whole[0]).all() and (parts[3][l.C * 3:] == whole[3][l.C * 3:]).all()
    o1, o2 = (R.from_bits(x[1], M.BF16).reshape(n, -1) for x in (whole, parts))
    # each token adds (2 * 64 + 32) half steps to a column at most (stateref.delta), and does not let it grow; both sides' outputs are rounded
    near = 2 * 160 * n * S.U
    s1, s2 = (x[4].reshape(2, l.vh, l.D, l.D)[1].astype(np.float64) for x in (whole, parts))
    norm = np.sqrt((s1 * s1).sum(1)).max()
    assert np.sqrt(((s1 - s2) ** 2).sum(1)).max() <= near * norm
    assert (np.abs(o1 - o2) <= 2.0 ** -7 * np.abs(o1) + near * max(np.abs(o1).max(), norm)).all()
    a1, a2 = (R.from_bits(x[2], M.BF16) for x in (whole, parts))
    # two forms of the kernel: weights and their sum off by 2^-11 each, the outputs by their rounding
    assert (np.abs(a1 - a2) <= 2.0 ** -7 * np.abs(a1) + 4 * 2.0 ** -11 * np.abs(l.cache.v[0]).max()).all()
    l.close()


def test_another_stream(gpu_ctx):
    """The calls run on the context's stream, whichever that is, behind what is on it."""
    import ctypes as C

    hip = C.CDLL("libamdhip64.so")
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    got = []
    for own in (True, False):
        with M.Context() as ctx:
            if not own:
                ctx.set_stream(stream.value)
            l = Layer(ctx, np.random.default_rng(22), 2, 100, [300, 90])
            l.set([60, 40], [300, 90])
            l.call()
            l.call()  # from the same states again
            got.append(l.results())
            l.close()
    assert hip.hipStreamDestroy(stream) == 0
    for a, b in zip(*got):
        assert np.array_equal(a, b)
