"""The attention-side operators on the GPU against plain 64-bit forms (attnref.py), at the sizes, strides,
masks and index entries where they can go wrong. Tolerances are derived where they stand."""
import numpy as np
import pytest

import moe_rocm as M

import attnref as R

pytestmark = pytest.mark.gpu

FORMATS = {"mxfp4": M.KV_MXFP4, "mxint8": M.KV_MXINT8, "f16": M.KV_F16}
TYPES = {"f32": M.F32, "f16": M.F16, "bf16": M.BF16}


def sync_error(ctx, text):
    """The next sync reports an entry out of range, the one after it nothing."""
    with pytest.raises(M.MoeRocmError) as ei:
        ctx.sync()
    assert ei.value.status == M.MR_E_INVAL and text in ei.value.message, ei.value.message
    ctx.sync()


# ---- rotary positions ------------------------------------------------------------------------
@pytest.mark.parametrize("D,n,hq,hk,T", [(64, 64, 64, 8, 1), (128, 128, 32, 4, 7), (256, 64, 16, 2, 3), (8, 8, 3, 1, 5),
                                         (96, 96, 5, 5, 2), (512, 512, 2, 1, 3), (72, 40, 33, 0, 4), (128, 8, 1, 1, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dst,norm", [("f32", "f32", True), ("f32", "bf16", False), ("bf16", "f16", True),
                                          ("f16", "f32", False)])
def test_rope(gpu_ctx, D, n, hq, hk, T, interleaved, src, dst, norm):
    rng = np.random.default_rng(D * 7 + T)
    src, dst = TYPES[src], TYPES[dst]
    x = R.rounded(rng.normal(size=(T, hq + hk, D)) * 3, src)
    pos = rng.integers(-5, 200000, T).astype(np.int32)
    pos[0] = 2 ** 31 - 1
    rope = M.Rope(gpu_ctx, D, rotary_dim=n, base=150000.0, layout=int(interleaved), scaling=M.ROPE_YARN, factor=8.0,
                  orig_context=4096)
    f, mul = rope.frequencies()
    w = [1 + 0.2 * rng.normal(size=D).astype(np.float32) for _ in range(2)]
    dw = [gpu_ctx.to_device(a.astype(np.float32)) for a in w]
    # queries and keys out of one projection row, with room around the outputs
    q, k = R.Rows(gpu_ctx, x[:, :hq], src, pad=hk + 1, first=1), R.Rows(gpu_ctx, x[:, hq:], src) if hk else None
    qo = R.Rows(gpu_ctx, None, dst, T, hq, D, pad=2, first=1)
    ko = R.Rows(gpu_ctx, None, dst, T, hk, D) if hk else None
    dp = R.i32(gpu_ctx, pos)
    kw = dict(q_norm=dw[0], k_norm=dw[1] if hk else None, eps=1e-6) if norm else {}
    M.qk_norm_rope(gpu_ctx, rope, q.heads, k.heads if hk else None, T, dp, qo.heads, ko.heads if hk else None, **kw)
    gpu_ctx.sync()
    for got, a, weight in ((qo, x[:, :hq], w[0]), (ko, x[:, hq:], w[1])):
        if got is None:
            continue
        y, size = R.rope(a, pos, f, mul, interleaved, weight if norm else None, 1e-6)
        # relative to the pair: the norm's sum of squares (8 terms in a lane, up to 6 steps across lanes; half of
        # it under the root), root, division, two products; the angle (a fraction of a turn in f32: 2 pi 2^-25), sine
        # and cosine (2 steps), the factor; two products and a sum
        tol = 26 * 2.0 ** -24 * size + R.HALF[dst] * np.abs(y) * (dst != M.F32) + 2.0 ** -25 * (dst == M.F16)
        assert (np.abs(got.get() - y) <= tol).all(), float((np.abs(got.get() - y) / tol).max())
    for b in (q, k, qo, ko, dp, *dw):
        if b is not None:
            b.free()
    rope.close()


def test_rope_in_place_and_without_norm_of_keys(gpu_ctx):
    rng = np.random.default_rng(1)
    T, H, D = 33, 5, 64
    x = R.rounded(rng.normal(size=(T, H + 2, D)), M.BF16)
    rope = M.Rope(gpu_ctx, D)
    pos = R.i32(gpu_ctx, np.arange(T))
    w = gpu_ctx.to_device(np.full(D, 2.0, np.float32))
    outs = []
    for place in (False, True):
        q, k = R.Rows(gpu_ctx, x[:, :H], M.BF16), R.Rows(gpu_ctx, x[:, H:], M.BF16)
        qo, ko = (q, k) if place else (R.Rows(gpu_ctx, None, M.BF16, T, H, D), R.Rows(gpu_ctx, None, M.BF16, T, 2, D))
        M.qk_norm_rope(gpu_ctx, rope, q.heads, k.heads, T, pos, qo.heads, ko.heads, q_norm=w, eps=0.0)
        gpu_ctx.sync()
        outs.append((qo.get(), ko.get()))
        for b in {q, k, qo, ko}:
            b.free()
    assert all((a == b).all() for a, b in zip(*outs))
    f, mul = rope.frequencies()
    y, size = R.rope(x[:, H:], np.arange(T), f, mul, False)
    assert (np.abs(outs[0][1] - y) <= 26 * 2.0 ** -24 * size + 2.0 ** -8 * np.abs(y)).all()
    pos.free(), w.free(), rope.close()


# ---- the cache ---------------------------------------------------------------------------------
def _values(rng, shape):
    """Values over the whole range of block exponents: normal ones, ties, zeros, tiny and huge ones."""
    x = rng.normal(size=shape).astype(np.float32) * np.exp2(rng.integers(-24, 20, shape[:-1] + (1,))).astype(np.float32)
    x[rng.random(shape) < 0.1] = 0
    y = rng.integers(-56, 57, shape).astype(np.float32) / 8  # ties of MXFP4's codes, and of MXINT8's below
    x = np.where(rng.random(shape[:-1] + (1,)) < 0.4, y, x)
    z = rng.integers(-255, 256, shape).astype(np.float32) / 2
    return np.where(rng.random(shape[:-1] + (1,)) < 0.3, z, x)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,H,page", [(64, 3, 64), (128, 1, 256), (256, 2, 128)])
@pytest.mark.parametrize("src", ["f32", "bf16", "f16"])
def test_write_then_read(gpu_ctx, fmt, D, H, page, src):
    rng = np.random.default_rng(D + page)
    fmt, src = FORMATS[fmt], TYPES[src]
    pages, T = 3, 2 * page + 37
    kv = M.KvCache(gpu_ctx, fmt, pages, page, H, D)
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    slots[5] = -1
    x, y = (R.rounded(_values(rng, (T, H, D)), src) for _ in range(2))
    if src == M.F32:
        x[7, 0, 3], y[8, 0, 40], x[9, 0, 1] = np.inf, -np.inf, np.nan
    dk, dv = R.Rows(gpu_ctx, x, src, pad=1), R.Rows(gpu_ctx, y, src, pad=2, first=1)
    ds = R.i32(gpu_ctx, slots)
    kv.write(dk.heads, dv.heads, T, ds)
    # every slot of the cache, and a negative one: those never written are zeros
    order = np.concatenate([[-3], rng.permutation(pages * page)]).astype(np.int32)
    ko, vo = (R.Rows(gpu_ctx, None, M.F32, len(order), H, D, pad=1) for _ in range(2))
    do = R.i32(gpu_ctx, order)
    kv.read(len(order), do, ko.heads, vo.heads)
    gpu_ctx.sync()
    at = {int(s): t for t, s in enumerate(slots) if s >= 0}
    for got, a in ((ko.get(), x), (vo.get(), y)):
        want = np.zeros((len(order), H, D))
        held = R.stored(a, fmt)
        for i, s in enumerate(order):
            if int(s) in at:
                want[i] = held[at[int(s)]]
        assert (got == want).all(), np.argwhere(got != want)[:5]
    # a second write of one token leaves its neighbours as they are; types of k and v apart, out as f16
    one = rng.normal(size=(1, H, D))
    a, b = R.Rows(gpu_ctx, one, M.F16), R.Rows(gpu_ctx, one, M.F32)
    slots1 = np.array([slots[2]], np.int32)
    d1 = R.i32(gpu_ctx, slots1)
    kv.write(a.heads, b.heads, 1, d1)
    kv.read(len(order), do, None, vo.heads)
    ko2 = R.Rows(gpu_ctx, None, M.F16, len(order), H, D)
    kv.read(len(order), do, ko2.heads, None)
    gpu_ctx.sync()
    i = int(np.argwhere(order == slots1[0])[0, 0])
    v2, k2 = vo.get(), ko2.get()
    assert (v2[i] == R.stored(R.rounded(one, M.F32), fmt)[0]).all() and (k2[i] == R.stored(R.rounded(one, M.F16), fmt)[0]).all()
    rest = np.arange(len(order)) != i
    assert (v2[rest] == want[rest]).all() and (k2[rest] == ko.get()[rest]).all()
    for t in (dk, dv, ds, ko, vo, do, a, b, d1, ko2):
        t.free()
    kv.close()


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 200])
@pytest.mark.parametrize("start", [0, 1, 64, 100])
def test_write_of_a_run_of_tokens(gpu_ctx, T, start):
    """Tokens in order from any place in a page on: whole chunks, and parts of them at both ends."""
    rng = np.random.default_rng(T)
    for fmt in FORMATS.values():
        H, D, page = 2, 128, 128
        kv = M.KvCache(gpu_ctx, fmt, 4, page, H, D)
        x, y = rng.normal(size=(T, H, D)), rng.normal(size=(T, H, D))
        order = np.array([2, 0, 3, 1])
        t = start + np.arange(T)
        dk, dv, ds = R.Rows(gpu_ctx, x, M.F16), R.Rows(gpu_ctx, y, M.F16), R.i32(gpu_ctx, order[t // page] * page + t % page)
        kv.write(dk.heads, dv.heads, T, ds)
        ko, vo = R.Rows(gpu_ctx, None, M.F32, 4 * page, H, D), R.Rows(gpu_ctx, None, M.F32, 4 * page, H, D)
        every = np.arange(4 * page)
        do = R.i32(gpu_ctx, order[every // page] * page + every % page)
        kv.read(4 * page, do, ko.heads, vo.heads)
        gpu_ctx.sync()
        for got, a in ((ko.get(), x), (vo.get(), y)):
            want = np.zeros((4 * page, H, D))
            want[start:start + T] = R.stored(R.rounded(a, M.F16), fmt)
            assert (got == want).all()
        for b in (dk, dv, ds, ko, vo, do):
            b.free()
        kv.close()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_of_every_length_written_and_read(gpu_ctx, fmt, D):
    """Rows of adjacent slots, of every length and place in a chunk, with gaps and negative slots between them; read
    in the same order, in rows cut elsewhere, and slot by slot."""
    rng = np.random.default_rng(D)
    fmt, H, page, pages = FORMATS[fmt], 2, 128, 24
    kv = M.KvCache(gpu_ctx, fmt, pages, page, H, D)
    rows = []
    for chunk in rng.permutation(pages * page // 64):
        a, b = sorted(rng.choice(65, 2, replace=False))
        rows.append(64 * chunk + np.arange(a, b))
        if chunk % 5 == 0:
            rows.append(np.array([-1]))
    slots = np.concatenate(rows).astype(np.int32)
    T = len(slots)
    x, y = (R.rounded(_values(rng, (T, H, D)), M.BF16) for _ in range(2))
    dk, dv, ds = R.Rows(gpu_ctx, x, M.BF16), R.Rows(gpu_ctx, y, M.BF16), R.i32(gpu_ctx, slots)
    kv.write(dk.heads, dv.heads, T, ds)
    live = slots >= 0
    held = [np.zeros((pages * page, H, D)) for _ in range(2)]
    for h, a in zip(held, (x, y)):
        h[slots[live]] = R.stored(a[live], fmt)
    for order in (slots, np.arange(pages * page)[5:-9], rng.permutation(pages * page)):
        n = len(order)
        ko, vo = (R.Rows(gpu_ctx, None, M.F32, n, H, D, pad=1) for _ in range(2))
        do = R.i32(gpu_ctx, order.astype(np.int32))
        kv.read(n, do, ko.heads, vo.heads)
        gpu_ctx.sync()
        for got, h in ((ko.get(), held[0]), (vo.get(), held[1])):
            want = np.where((order >= 0)[:, None, None], h[np.maximum(order, 0)], 0.0)
            assert (got == want).all()
        for b in (ko, vo, do):
            b.free()
    for b in (dk, dv, ds):
        b.free()
    kv.close()


def test_slots_out_of_range_are_left_out_and_reported(gpu_ctx):
    H, D, page = 2, 64, 64
    kv = M.KvCache(gpu_ctx, M.KV_MXFP4, 2, page, H, D)
    x = np.ones((4, H, D))
    dx, ds = R.Rows(gpu_ctx, x, M.F32), R.i32(gpu_ctx, [128, 3, 2 ** 31 - 1, -2 ** 31])
    kv.write(dx.heads, dx.heads, 4, ds)
    sync_error(gpu_ctx, "slots")
    out = R.Rows(gpu_ctx, None, M.F32, 4, H, D)
    kv.read(4, ds, out.heads, None)
    sync_error(gpu_ctx, "slots")
    got = out.get()
    assert (got[1] == 1).all() and (got[[0, 2, 3]] == 0).all()
    for b in (dx, ds, out):
        b.free()
    kv.close()


# ---- attention of single tokens over the cache -----------------------------------------------------
class Cached:
    """Sequences of given lengths in a cache whose pages lie in any order; rows of the table are garbage
    behind a sequence's pages."""

    def __init__(self, ctx, fmt, lens, H, D, page, seed, spread=1.0):
        rng = np.random.default_rng(seed)
        self.ctx, self.lens, self.page = ctx, lens, page
        counts = [-(-n // page) for n in lens]
        total = sum(counts) + 2
        order = rng.permutation(total)
        self.max_pages = max(1, max(counts)) + 1
        self.table = np.full((len(lens), self.max_pages), -7, np.int32)
        self.kv = M.KvCache(ctx, fmt, total, page, H, D)
        self.k, self.v, at = [], [], 0
        # what earlier requests left in the pages: large values that no row may see
        every = R.i32(ctx, np.arange(total * page))
        old = R.Rows(ctx, np.full((total * page, H, D), 30000.0), M.F16)
        self.kv.write(old.heads, old.heads, total * page, every)
        ctx.sync(), every.free(), old.free()
        for i, (n, c) in enumerate(zip(lens, counts)):
            self.table[i, :c] = order[at:at + c]
            at += c
            k, v = (rng.normal(size=(n, H, D)) * spread).astype(np.float32), rng.normal(size=(n, H, D)).astype(np.float32)
            self.k.append(R.stored(k, fmt)), self.v.append(R.stored(v, fmt))
            if n:
                t = np.arange(n)
                dk, dv, ds = R.Rows(ctx, k, M.F32), R.Rows(ctx, v, M.F32), R.i32(ctx, self.table[i][t // page] * page + t % page)
                self.kv.write(dk.heads, dv.heads, n, ds)
                ctx.sync()
                for b in (dk, dv, ds):
                    b.free()
        self.d_len, self.d_table = R.i32(ctx, lens), R.i32(ctx, self.table)

    def check(self, got, q, dtype, group, scale, window=0, sinks=None, there=None):
        """`there`: tokens of each sequence that can be seen (all, or a list of masks)."""
        for b, n in enumerate(self.lens):
            for h in range(q.shape[1]):
                hk = h // group
                first = max(0, n - window) if window else 0
                k, v = self.k[b][first:, hk], self.v[b][first:, hk]
                if there is not None:
                    k, v = k[there[b][first:]], v[there[b][first:]]
                y, av, ss, cnt = R.attend(q[b, h], k, v, scale, 0, len(k) - 1, None if sinks is None else sinks[h])
                tol = R.attention_bound(y, av, ss, cnt, q.shape[2], dtype, 2.0 ** -11)
                assert (np.abs(got[b, h] - y) <= tol).all(), (b, h, n, float((np.abs(got[b, h] - y) / tol).max()))

    def close(self):
        self.d_len.free(), self.d_table.free(), self.kv.close()


LENS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 511, 512, 513, 1030, 5, 0, 2100]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,hk,group,page", [(64, 2, 8, 64), (128, 3, 4, 128), (256, 1, 16, 256), (128, 1, 1, 64),
                                             (64, 1, 20, 512), (256, 2, 5, 64)])
@pytest.mark.parametrize("dtype,window,sink", [("bf16", 0, False), ("f16", 100, True), ("bf16", 1, True)])
def test_decode(gpu_ctx, fmt, D, hk, group, page, dtype, window, sink):
    dtype = TYPES[dtype]
    c = Cached(gpu_ctx, FORMATS[fmt], LENS, hk, D, page, D + group)
    rng = np.random.default_rng(3)
    H = hk * group
    q = R.rounded(rng.normal(size=(len(LENS), H, D)), dtype)
    sinks = rng.normal(size=H).astype(np.float32) * 3 if sink else None
    if sink:
        sinks[0], sinks[-1] = -np.inf, 40.0
    dq, out = R.Rows(gpu_ctx, q, dtype, pad=1), R.Rows(gpu_ctx, None, dtype, len(LENS), H, D, pad=2, first=1)
    ds = gpu_ctx.to_device(sinks) if sink else None
    c.kv.attend(dq.heads, len(LENS), c.d_len, c.d_table, c.max_pages, out.heads, window=window, sinks=ds)
    gpu_ctx.sync()
    c.check(out.get(), q, dtype, group, D ** -0.5, window, sinks)
    for b in (dq, out):
        b.free()
    if ds:
        ds.free()
    c.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,hk,group", [(64, 8, 8), (128, 4, 8), (256, 2, 8)])
@pytest.mark.parametrize("n,window", [(9000, 0), (20011, 0), (20011, 4097)])
def test_decode_of_one_long_sequence(gpu_ctx, fmt, D, hk, group, n, window):
    c = Cached(gpu_ctx, FORMATS[fmt], [n], hk, D, 256, 9, spread=2.0)
    rng = np.random.default_rng(4)
    q = R.rounded(rng.normal(size=(1, hk * group, D)), M.BF16)
    dq, out = R.Rows(gpu_ctx, q, M.BF16), R.Rows(gpu_ctx, None, M.BF16, 1, hk * group, D)
    first = None
    for _ in range(3):  # the same bits every time
        c.kv.attend(dq.heads, 1, c.d_len, c.d_table, c.max_pages, out.heads, window=window)
        gpu_ctx.sync()
        got = out.get()
        assert first is None or (got == first).all()
        first = got
    c.check(got, q, M.BF16, group, D ** -0.5, window)
    dq.free(), out.free(), c.close()


@pytest.mark.parametrize("n_seqs,long", [(65, 5000), (300, 9000), (1024, 3000), (1100, 2000)])
def test_decode_of_many_sequences(gpu_ctx, n_seqs, long):
    """Short sequences and some long ones among them, which are split or not."""
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(0, 70, n_seqs).tolist()
    lens[1], lens[n_seqs // 2], lens[-1] = long, 1300, long // 2
    c = Cached(gpu_ctx, M.KV_MXFP4, lens, 1, 64, 64, n_seqs)
    q = R.rounded(rng.normal(size=(n_seqs, 3, 64)), M.F16)
    dq, out = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, None, M.F16, n_seqs, 3, 64)
    c.kv.attend(dq.heads, n_seqs, c.d_len, c.d_table, c.max_pages, out.heads)
    gpu_ctx.sync()
    c.check(out.get(), q, M.F16, 3, 0.125)
    dq.free(), out.free(), c.close()


def test_decode_scores_of_any_size(gpu_ctx):
    """Scores far apart, a negative scale, queries near the types' ends: one key takes all the weight."""
    lens = [200, 700]
    for fmt in FORMATS.values():
        c = Cached(gpu_ctx, fmt, lens, 1, 64, 64, 5, spread=8.0)
        rng = np.random.default_rng(6)
        for dtype, size, scale in ((M.BF16, 50.0, 0.0), (M.F16, 50.0, -0.3), (M.BF16, 1e30, 1e-28), (M.BF16, 1e-30, 1e30),
                                   (M.F16, 6e4, 1e-3), (M.F16, 1e-7, 1e5)):
            q = R.rounded(rng.normal(size=(2, 4, 64)).clip(-1, 1) * size, dtype)
            dq, out = R.Rows(gpu_ctx, q, dtype), R.Rows(gpu_ctx, None, dtype, 2, 4, 64)
            c.kv.attend(dq.heads, 2, c.d_len, c.d_table, c.max_pages, out.heads, scale=scale)
            gpu_ctx.sync()
            c.check(out.get(), q, dtype, 4, scale or 0.125)
            dq.free(), out.free()
        c.close()


def test_decode_leaves_out_what_is_not_there(gpu_ctx):
    H, D, page = 2, 128, 64
    lens = [200, 130, 64, 10]
    c = Cached(gpu_ctx, M.KV_MXINT8, lens, H, D, page, 8)
    rng = np.random.default_rng(2)
    q = R.rounded(rng.normal(size=(4, H, D)), M.F16)
    dq, out = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, None, M.F16, 4, H, D)
    table = c.table.copy()
    n_pages = int(c.kv.desc.n_pages)
    table[0, 1], table[1, 2], table[2, 0] = n_pages, -1, 2 ** 31 - 1
    there = [np.arange(n) >= 0 for n in lens]
    there[0][64:128], there[1][128:], there[2][:] = False, False, False
    dt = R.i32(gpu_ctx, table)
    c.kv.attend(dq.heads, 4, c.d_len, dt, c.max_pages, out.heads)
    sync_error(gpu_ctx, "block_table")
    c.check(out.get(), q, M.F16, 1, D ** -0.5, there=there)
    # lengths out of range: the nearest ones (max_pages pages, the last of which is missing; none)
    dl = R.i32(gpu_ctx, [2 ** 31 - 1, 130, -5, 10])
    c.kv.attend(dq.heads, 4, dl, c.d_table, c.max_pages, out.heads)
    sync_error(gpu_ctx, "seq_len block_table")
    got = out.get()
    assert (got[2] == 0).all()
    full = -(-200 // page) * page  # sequence 0 sees all of its pages, what earlier requests left included
    assert full < c.max_pages * page and np.isfinite(got).all()
    c.lens = [10]
    c.k, c.v = c.k[3:], c.v[3:]
    c.check(got[3:], q[3:], M.F16, 1, D ** -0.5)
    for b in (dq, out, dt, dl):
        b.free()
    c.close()


def test_cache_beyond_32_bit_offsets(gpu_ctx):
    """Pages on both sides of 4 GiB."""
    H, D, page = 2, 256, 1024
    n_pages = (5 << 30) // (page * H * D * 4)
    assert M.KvCache.nbytes(M.KV_F16, n_pages, page, H, D) > 5 * 10 ** 9
    kv = M.KvCache(gpu_ctx, M.KV_F16, n_pages, page, H, D)
    rng = np.random.default_rng(0)
    pages, n = [n_pages - 1, 0, n_pages // 2 + 300], 3 * page - 5
    t = np.arange(n)
    k, v = (rng.normal(size=(n, H, D)).astype(np.float32) for _ in range(2))
    dk, dv, ds = R.Rows(gpu_ctx, k, M.F32), R.Rows(gpu_ctx, v, M.F32), R.i32(gpu_ctx, np.array(pages)[t // page] * page + t % page)
    kv.write(dk.heads, dv.heads, n, ds)
    ko = R.Rows(gpu_ctx, None, M.F16, n, H, D)
    kv.read(n, ds, ko.heads, None)
    gpu_ctx.sync()
    assert (ko.get() == R.stored(k, M.KV_F16)).all()
    q = R.rounded(rng.normal(size=(1, 4, D)), M.F16)
    dq, out, dl, dt = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, None, M.F16, 1, 4, D), R.i32(gpu_ctx, [n]), R.i32(gpu_ctx, pages)
    kv.attend(dq.heads, 1, dl, dt, 3, out.heads)
    gpu_ctx.sync()
    for h in range(4):
        y, av, ss, cnt = R.attend(q[0, h], R.stored(k, M.KV_F16)[:, h // 2], R.stored(v, M.KV_F16)[:, h // 2], D ** -0.5, 0, n - 1)
        assert (np.abs(out.get()[0, h] - y) <= R.attention_bound(y, av, ss, cnt, D, M.F16, 2.0 ** -11)).all()
    for b in (dk, dv, ds, ko, dq, out, dl, dt):
        b.free()
    kv.close()


# ---- attention over packed prompts -------------------------------------------------------------------
def prompts(ctx, D, hk, group, dtype, lens_q, lens_k, window=0, sinks=None, behind=3, seed=0, scale=0.0, spread=1.0):
    """Runs packed sequences, rows in none of them in front of and behind the others; checks every row."""
    rng = np.random.default_rng(seed)
    H = hk * group
    cu_q = 2 + np.concatenate([[0], np.cumsum(lens_q)])
    cu_k = 1 + np.concatenate([[0], np.cumsum(lens_k)])
    nq, nk = int(cu_q[-1]) + behind, int(cu_k[-1]) + behind
    q = R.rounded(rng.normal(size=(nq, H, D)) * spread, dtype)
    k, v = (R.rounded(rng.normal(size=(nk, hk, D)) * s, dtype) for s in (spread, 1.0))
    # rows of no sequence hold what must not be looked at
    for a, c in ((k, cu_k), (v, cu_k)):
        a[:c[0]], a[c[-1]:] = np.nan, np.inf
    dq, dk = R.Rows(ctx, q, dtype, pad=1, first=1), R.Rows(ctx, k, dtype, pad=2)
    dv, out = R.Rows(ctx, v, dtype, pad=1, first=1), R.Rows(ctx, None, dtype, nq, H, D, pad=1)
    dcq, dck = R.i32(ctx, cu_q), R.i32(ctx, cu_k)
    ds = None if sinks is None else ctx.to_device(np.asarray(sinks, np.float32))
    M.attn_prefill(ctx, D, dq.heads, dk.heads, dv.heads, nq, nk, len(lens_q), dcq, dck, out.heads, scale=scale, window=window,
                   sinks=ds)
    ctx.sync()
    got = out.get()
    mark = R.from_bits(np.array([out.mark]), dtype)[0]
    assert (got[:cu_q[0]] == mark).all() and (got[cu_q[-1]:] == mark).all(), "rows of no sequence were written"
    worst = 0.0
    for s in range(len(lens_q)):
        rows = np.arange(cu_q[s], cu_q[s + 1])
        if len(rows) > 150:  # the ends, the places around tiles, and some in between
            pick = {0, 1, 31, 32, 63, 64, 127, 128, 129, len(rows) - 1, len(rows) - 2} | set(rng.integers(0, len(rows), 20).tolist())
            rows = rows[sorted(i for i in pick if i < len(rows))]
        for r in rows:
            last = int(cu_k[s + 1] - (cu_q[s + 1] - r))  # the row's own position among the keys
            first = max(int(cu_k[s]), last - window + 1) if window else int(cu_k[s])
            for h in range(H):
                y, av, ss, n = R.attend(q[r, h], k[:, h // group], v[:, h // group], scale or D ** -0.5, first, last,
                                        None if sinks is None else sinks[h])
                # p is rounded to the inputs' type for the second product
                tol = R.attention_bound(y, av, ss, n, D, dtype, R.HALF[dtype])
                d = np.abs(got[r, h] - y) / tol
                worst = max(worst, float(d.max()))
                assert (d <= 1).all(), (s, r, h, n, worst)
    for b in (dq, dk, dv, out, dcq, dck, ds):
        if b is not None:
            b.free()


SHORT = [1, 0, 5, 31, 64, 33, 0, 65, 130]


@pytest.mark.parametrize("D,hk,group", [(64, 2, 8), (128, 3, 2), (256, 1, 3), (128, 1, 1)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window,sink,past", [(0, False, 0), (40, True, 0), (1, False, 0), (0, True, 77), (100, True, 200)])
def test_prefill(gpu_ctx, D, hk, group, dtype, window, sink, past):
    sinks = np.random.default_rng(5).normal(size=hk * group) * 2 if sink else None
    if sink:
        sinks[0] = -np.inf
    prompts(gpu_ctx, D, hk, group, TYPES[dtype], SHORT, [n + past for n in SHORT], window, sinks, seed=D + past)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 200])
def test_prefill_long(gpu_ctx, D, window):
    prompts(gpu_ctx, D, 2, 4, M.BF16, [1000, 257, 3, 511], [1000, 257, 3, 2511], window, seed=D)


@pytest.mark.parametrize("n_seqs", [65, 512, 513, 1500])
def test_prefill_of_many_sequences(gpu_ctx, n_seqs):
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(0, 4, n_seqs)
    lens[[3, n_seqs // 2, n_seqs - 1]] = 140, 257, 129
    prompts(gpu_ctx, 64, 1, 2, M.BF16, lens, lens + rng.integers(0, 3, n_seqs), seed=n_seqs)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_rows_that_see_nothing(gpu_ctx, D):
    """More queries than keys: the first rows are zero, with and without sinks; no keys at all."""
    for sinks in (None, [0.5, -2.0]):
        prompts(gpu_ctx, D, 1, 2, M.F16, [70, 200, 4, 1], [10, 0, 4, 0], 0, sinks, seed=1)


def test_prefill_scores_of_any_size(gpu_ctx):
    for dtype in (M.F16, M.BF16):
        prompts(gpu_ctx, 64, 1, 2, dtype, [150, 90], [150, 90], spread=12.0, seed=2)
        prompts(gpu_ctx, 128, 1, 2, dtype, [150, 90], [150, 90], spread=12.0, scale=-0.5, seed=3)
        prompts(gpu_ctx, 64, 1, 2, dtype, [150], [150], window=20, sinks=[300.0, -300.0], spread=6.0, seed=4)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prefill_infinities_and_nan_where_rows_do_not_look(gpu_ctx, D, dtype):
    """Keys and values that are not finite, at positions before some rows' windows and after others: rows that do not
    see them are as without them, rows that do are NaN, or an infinity where only values of one sign are."""
    dtype, n, window = TYPES[dtype], 200, 50
    rng = np.random.default_rng(D)
    q, k, v = (R.rounded(rng.normal(size=(n, 1, D)), dtype) for _ in range(3))
    clean_k, clean_v = k.copy(), v.copy()
    k[150, 0, 3] = np.nan
    v[20, 0, 5], v[20, 0, 7], v[70, 0, 1], v[71, 0, 1], v[199, 0, :] = np.inf, -np.inf, np.inf, -np.inf, np.nan
    v[45, 0, D - 1] = np.nan
    dq, dk, dv, out = (R.Rows(gpu_ctx, a, dtype, n, 1, D) for a in (q, k, v, None))
    cu = R.i32(gpu_ctx, [0, n])
    M.attn_prefill(gpu_ctx, D, dq.heads, dk.heads, dv.heads, n, n, 1, cu, cu, out.heads, window=window)
    gpu_ctx.sync()
    got = out.get()[:, 0]
    for r in range(n):
        sees = lambda j: max(0, r - window + 1) <= j <= r  # noqa: E731
        y, av, ss, cnt = R.attend(q[r, 0], clean_k[:, 0], clean_v[:, 0], D ** -0.5, max(0, r - window + 1), r)
        y = y.copy()
        if sees(20):
            y[5], y[7] = np.inf, -np.inf
        y[1] = np.nan if sees(70) and sees(71) else np.inf if sees(70) else -np.inf if sees(71) else y[1]
        y[D - 1] = np.nan if sees(45) else y[D - 1]
        if sees(150) or sees(199):
            y[:] = np.nan
        tol = R.attention_bound(np.where(np.isfinite(y), y, 0), av, ss, cnt, D, dtype, R.HALF[dtype])
        fine = np.isfinite(y)
        assert (np.isnan(got[r]) == np.isnan(y)).all(), (r, got[r], y)
        assert (got[r][np.isinf(y)] == y[np.isinf(y)]).all(), r
        assert (np.abs(got[r] - y)[fine] <= tol[fine]).all(), r
    for b in (dq, dk, dv, out, cu):
        b.free()


@pytest.mark.parametrize("hk,group", [(8, 4), (4, 8), (2, 8), (3, 4), (8, 2), (5, 2), (3, 6), (16, 1), (17, 1), (136, 1), (5, 5), (40, 8)])
def test_prefill_heads_in_every_arrangement(gpu_ctx, hk, group):
    """Heads that share keys by 1, 2 and 4, in numbers that are a multiple of 8 and not."""
    lens = [5, 0, 70, 33] if hk * group < 100 else [0, 34, 2]
    prompts(gpu_ctx, 64, hk, group, M.BF16, lens, [n + 40 for n in lens], 50, seed=hk)
    prompts(gpu_ctx, 64, hk, group, M.F16, lens, lens, seed=group)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [2, 4])
def test_prefill_infinities_and_nan_with_shared_keys(gpu_ctx, D, group):
    """All heads of a group: rows that see an infinite value have it, rows that do not are as without it."""
    n, window, hk = 150, 50, 2
    rng = np.random.default_rng(D)
    q, k, v = (R.rounded(rng.normal(size=(n, h, D)), M.BF16) for h in (hk * group, hk, hk))
    clean = v.copy()
    v[20, 0, 5], v[70, 1, 1], v[90, 0, 7] = np.inf, -np.inf, np.nan
    dq, dk, dv, out = (R.Rows(gpu_ctx, a, M.BF16, n, h, D) for a, h in ((q, hk * group), (k, hk), (v, hk), (None, hk * group)))
    cu = R.i32(gpu_ctx, [0, n])
    M.attn_prefill(gpu_ctx, D, dq.heads, dk.heads, dv.heads, n, n, 1, cu, cu, out.heads, window=window)
    gpu_ctx.sync()
    got = out.get()
    for r in range(n):
        for h in range(hk * group):
            first, g = max(0, r - window + 1), h // group
            y, av, ss, cnt = R.attend(q[r, h], k[:, g], clean[:, g], D ** -0.5, first, r)
            y = y.copy()
            for at, head, d, x in ((20, 0, 5, np.inf), (70, 1, 1, -np.inf), (90, 0, 7, np.nan)):
                if g == head and first <= at <= r:
                    y[d] = x
            fine = np.isfinite(y)
            tol = R.attention_bound(np.where(fine, y, 0), av, ss, cnt, D, M.BF16, R.HALF[M.BF16])
            assert np.array_equal(got[r, h][~fine], y[~fine], equal_nan=True), (r, h)
            assert (np.abs(got[r, h] - y)[fine] <= tol[fine]).all(), (r, h)
    for b in (dq, dk, dv, out, cu):
        b.free()


@pytest.mark.parametrize("cu_q,cu_k", [([0, 40, 999], [0, 40, 90]), ([0, 50, 30], [0, 50, 90]), ([-9, 40, 90], [0, 40, 90]),
                                       ([0, 40, 90], [0, 40, 2 ** 31 - 1]), ([0, 40, 90], [0, 60, 50]),
                                       ([0, 40, 90], [-2 ** 31, 40, 90])])
def test_prefill_offsets_out_of_range(gpu_ctx, cu_q, cu_k):
    """Offsets are clamped into the rows, decreasing ones are empty sequences; reported at the next sync."""
    rng = np.random.default_rng(0)
    n, D = 90, 64
    q, k, v = (R.rounded(rng.normal(size=(n, 1, D)), M.F16) for _ in range(3))
    dq, dk, dv, out = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, k, M.F16), R.Rows(gpu_ctx, v, M.F16), R.Rows(gpu_ctx, None, M.F16, n, 1, D)
    dcq, dck = R.i32(gpu_ctx, cu_q), R.i32(gpu_ctx, cu_k)
    M.attn_prefill(gpu_ctx, D, dq.heads, dk.heads, dv.heads, n, n, 2, dcq, dck, out.heads)
    sync_error(gpu_ctx, "cu_q or cu_k")
    got = out.get()
    a, b = np.clip(cu_q, 0, n), np.clip(cu_k, 0, n)
    want = np.full((n, D), -7.5)
    tol = np.zeros((n, D))
    for s in range(2):
        for r in range(a[s], a[s + 1]):
            last = int(b[s + 1] - (a[s + 1] - r))
            y, av, ss, cnt = R.attend(q[r, 0], k[:, 0], v[:, 0], 0.125, int(b[s]), last)
            want[r], tol[r] = y, R.attention_bound(y, av, ss, cnt, D, M.F16, 2.0 ** -11)
    assert (np.abs(got[:, 0] - want) <= tol).all()
    for x in (dq, dk, dv, out, dcq, dck):
        x.free()


# ---- as they are used: a prompt, then tokens one by one ------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("graph", [False, True])
def test_prompt_then_decode(gpu_ctx, fmt, graph):
    """Two sequences: rotation, cache and attention of their prompts, then steps of one token each, eagerly or
    replayed from one captured graph, checked at every step. Keys and values are read back by the oracle."""
    fmt = FORMATS[fmt]
    rng = np.random.default_rng(12)
    D, hq, hk, page, steps = 128, 8, 2, 64, 5
    lens = [61, 130]
    rope = M.Rope(gpu_ctx, D, base=1e6)
    kv = M.KvCache(gpu_ctx, fmt, 8, page, hk, D)
    table = np.array([[5, 2, -1], [0, 7, 3]], np.int32)
    qw, kw = (gpu_ctx.to_device((1 + 0.1 * rng.normal(size=D)).astype(np.float32)) for _ in range(2))
    T = sum(lens)
    qkv = gpu_ctx.to_device(rng.normal(size=(T, hq + 2 * hk, D)).astype(np.float32))
    row = (hq + 2 * hk) * D
    view = lambda buf, first, n: M.Heads(buf.ptr + 4 * first * D, n, M.F32, row, D)  # noqa: E731
    pos = np.concatenate([np.arange(n) for n in lens])
    slots = np.concatenate([table[i][np.arange(n) // page] * page + np.arange(n) % page for i, n in enumerate(lens)])
    dpos, dslots, dcu = R.i32(gpu_ctx, pos), R.i32(gpu_ctx, slots), R.i32(gpu_ctx, [0, lens[0], T])
    q, k, v, out = (R.Rows(gpu_ctx, None, M.F16, T, n, D) for n in (hq, hk, hk, hq))
    M.qk_norm_rope(gpu_ctx, rope, view(qkv, 0, hq), view(qkv, hq, hk), T, dpos, q.heads, k.heads, q_norm=qw, k_norm=kw, eps=1e-6)
    kv.write(k.heads, view(qkv, hq + hk, hk), T, dslots)
    kv.read(T, dslots, k.heads, v.heads)  # the prompt attends over what the cache holds
    M.attn_prefill(gpu_ctx, D, q.heads, k.heads, v.heads, T, T, 2, dcu, dcu, out.heads)
    gpu_ctx.sync()
    qh, kh, vh, oh = q.get(), k.get(), v.get(), out.get()
    hist = [[], []]
    for i, n in enumerate(lens):
        a = sum(lens[:i])
        hist[i] = [kh[a:a + n], vh[a:a + n]]
        for r in range(a, a + n, 9):
            for h in range(hq):
                y, av, size, cnt = R.attend(qh[r, h], kh[:, h // 4], vh[:, h // 4], D ** -0.5, a, r)
                assert (np.abs(oh[r, h] - y) <= R.attention_bound(y, av, size, cnt, D, M.F16, 2.0 ** -11)).all()
    # one token of each sequence a step, in buffers that stay
    x = gpu_ctx.to_device(np.zeros((2, hq + 2 * hk, D), np.float32))
    sp, ss_, sl, dt = (R.i32(gpu_ctx, a) for a in ([0, 0], [0, 0], [0, 0], table))
    q1, k1, o1 = (R.Rows(gpu_ctx, None, M.F16, 2, n, D) for n in (hq, hk, hq))
    kr, vr = (R.Rows(gpu_ctx, None, M.F32, 2, hk, D) for _ in range(2))

    def step():
        M.qk_norm_rope(gpu_ctx, rope, view(x, 0, hq), view(x, hq, hk), 2, sp, q1.heads, k1.heads, q_norm=qw, k_norm=kw, eps=1e-6)
        kv.write(k1.heads, view(x, hq + hk, hk), 2, ss_)
        kv.attend(q1.heads, 2, sl, dt, 3, o1.heads)

    g = None
    if graph:
        sp.upload(np.array(lens, np.int32)), sl.upload(np.array([0, 0], np.int32)), ss_.upload(np.array([-1, -1], np.int32))
        gpu_ctx.graph_begin()
        step()
        g = gpu_ctx.graph_end()
    for t in range(steps):
        n = [a + t for a in lens]
        x.upload(rng.normal(size=(2, hq + 2 * hk, D)).astype(np.float32))
        sp.upload(np.array(n, np.int32)), sl.upload(np.array(n, np.int32) + 1)
        ss_.upload(np.array([table[i][n[i] // page] * page + n[i] % page for i in range(2)], np.int32))
        g.launch() if g else step()
        kv.read(2, ss_, kr.heads, vr.heads)
        gpu_ctx.sync()
        kn, vn, qn, got = kr.get(), vr.get(), q1.get(), o1.get()
        assert (kn == R.stored(k1.get(), fmt)).all()
        for i in range(2):
            hist[i] = [np.concatenate([hist[i][0], kn[i:i + 1]]), np.concatenate([hist[i][1], vn[i:i + 1]])]
            for h in range(hq):
                y, av, s, cnt = R.attend(qn[i, h], hist[i][0][:, h // 4], hist[i][1][:, h // 4], D ** -0.5, 0, n[i])
                assert (np.abs(got[i, h] - y) <= R.attention_bound(y, av, s, cnt, D, M.F16, 2.0 ** -11)).all()
    if g:
        g.close()
    for b in (qw, kw, qkv, dpos, dslots, dcu, q, k, v, out, x, sp, ss_, sl, dt, q1, k1, o1, kr, vr):
        b.free()
    kv.close(), rope.close()


def test_two_graphs_on_one_workspace(gpu_ctx):
    """Graphs of split calls of two caches, replayed in turn with eager calls between: each replay is the eager
    result to the bit, and sees the lengths of its time."""
    caches = [Cached(gpu_ctx, M.KV_MXFP4, [5000, 700], 2, 128, 256, 1), Cached(gpu_ctx, M.KV_F16, [3000], 1, 64, 64, 2)]
    rng = np.random.default_rng(5)
    rows, graphs = [], []
    for c in caches:
        B, H, D = len(c.lens), 4 * c.kv.desc.n_heads, c.kv.desc.head_dim
        rows.append([R.Rows(gpu_ctx, rng.normal(size=(B, H, D)), M.F16)] + [R.Rows(gpu_ctx, None, M.F16, B, H, D) for _ in range(2)])

    def call(i, out):
        c = caches[i]
        c.kv.attend(rows[i][0].heads, len(c.lens), c.d_len, c.d_table, c.max_pages, rows[i][out].heads)

    for i in range(2):
        gpu_ctx.graph_begin()
        call(i, 1)
        graphs.append(gpu_ctx.graph_end())
    for cut in (0, 100, 2500):
        for c in caches:
            c.d_len.upload(np.maximum(np.array(c.lens, np.int32) - cut, 0).astype(np.int32))
        for _ in range(2):
            for i in (0, 1):
                graphs[i].launch()
                call(1 - i, 2)
                call(i, 2)
            gpu_ctx.sync()
            for q, replayed, eager in rows:
                assert (replayed.all() == eager.all()).all()
    for g in graphs:
        g.close()
    for c in caches:
        c.close()
    for r in rows:
        for b in r:
            b.free()


def test_two_contexts_and_a_callers_stream(gpu_ctx):
    """Two contexts at once, one of them on a stream of the caller's, each with its own cache and workspace."""
    lens = [3000, 700]
    owner, other = M.Context(0), M.Context(0)  # `owner` stands for the caller that the stream belongs to
    other.set_stream(M.lib.mr_ctx_stream(owner.h))
    both = [(c, Cached(c, M.KV_MXFP4, lens, 2, 128, 256, seed)) for c, seed in ((gpu_ctx, 1), (other, 2))]
    rng = np.random.default_rng(0)
    q = R.rounded(rng.normal(size=(2, 16, 128)), M.BF16)
    rows = [(R.Rows(c, q, M.BF16), R.Rows(c, None, M.BF16, 2, 16, 128)) for c, _ in both]
    for _ in range(20):
        for (c, cached), (dq, out) in zip(both, rows):
            cached.kv.attend(dq.heads, 2, cached.d_len, cached.d_table, cached.max_pages, out.heads)
    for (c, cached), (dq, out) in zip(both, rows):
        c.sync()
        cached.check(out.get(), q, M.BF16, 8, 128 ** -0.5)
        dq.free(), out.free(), cached.close()
    other.close(), owner.close()
