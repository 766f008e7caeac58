"""Operators over kept states where values and numbers of sequences decide: weights of attention far below the largest; the gated delta rule where numbers
grow, pass 32 bits or are not finite, on each of its paths and types; against plain 64-bit forms (attnref.py, stateref.py)."""
import numpy as np
import pytest

import moe_rocm as M

import attnref as R
import stateref as S
from test_gpu_attn import FORMATS, TYPES, sync_error
from test_gpu_state import Cached, Delta, extend_ref, offsets

pytestmark = pytest.mark.gpu

LARGE = 1e37  # states below it are compared; what 32 bits do not hold may be anything from its token on


def check_what_32_bits_hold(c, compare_states=True):
    """Each row up to the first one at which the 64-bit state, or what makes it, has passed LARGE, column by column; and the last state
    of columns that never do. -> how many rows were compared, how many not."""
    g, beta, g_off, b_off = S.gates(c.a[:, :c.vh], c.b[:, :c.vh], c.a_log, c.dt_bias)
    at, half, seen, unseen = c.start, R.HALF[c.kind], 0, 0
    for s, n in enumerate(c.new):
        for h in range(c.vh):
            hk, i = h // (c.vh // c.kh), slice(at, at + n)
            state = c.states[c.source[s], h] if c.source[s] >= 0 else np.zeros((c.dk, c.dv))
            sizes = np.zeros((n, c.dv))
            x = state.astype(np.float64).copy()
            for t in range(n):  # how large the column is, and its correction
                k = c.k[at + t, hk].astype(np.float64)
                k = k / np.sqrt(k @ k + c.eps) if c.eps else k
                x = x * np.exp(g[at + t, h])
                look = k @ x
                d = beta[at + t, h] * (c.v[at + t, h] - look)
                sizes[t] = np.maximum(np.maximum(np.abs(x).max(0), np.abs(look)), np.maximum(np.abs(d), np.abs(c.v[at + t, h])))
                x = np.clip(x + np.outer(k, d), -1e60, 1e60)
                sizes[t] = np.maximum(sizes[t], np.abs(x).max(0))
            fits = np.maximum.accumulate(sizes, 0) < LARGE
            y, off, last, e = S.delta(c.q[i, hk], c.k[i, hk], c.v[i, h], g[i, h], beta[i, h], state, c.dk ** -0.5, c.eps, g_off[i, h], b_off[i, h])
            tol = off * (1 + half) + half * np.abs(y) * 1.01 + 2.0 ** -25 * (c.kind == M.F16)
            if c.kind == M.F16:
                fits = fits & (np.abs(y) < 65000)
            d = np.abs(c.out[i, h] - y)
            assert (d[fits] <= tol[fits]).all(), (s, h, np.argwhere(fits & ~(d <= tol))[:4])
            seen, unseen = seen + fits.sum(), unseen + (~fits).sum()
            if compare_states and c.target[s] >= 0 and n:
                whole = np.abs(x).max(0) < LARGE
                whole &= sizes.max(0) < LARGE
                d = np.abs(c.kept[c.target[s], h] - last)[:, whole]
                assert (d <= e[whole] + 1e-37).all(), (s, h, float((d / (e[whole] + 1e-37)).max()))
        at += n
    return int(seen), int(unseen)


def grow(c, how, rng):
    """Decays above 0 in c, and what keeps the result within 32 bits."""
    T = c.T
    if how == "until the last token":  # nothing is kept until a sequence's last token
        c.a[:], c.b[:] = 2.0, 0.0
        c.source[:] = -1
        at = 1
        for n in c.new:
            at += n
            c.b[at - 1] = 0.5
    if how == "by steps":  # up and down again, a hundred times and more within a chunk
        c.a[:] = np.where(np.arange(T) // 16 % 2, -0.35, 0.35)[:, None]
    if how == "a little":  # less than a factor of two in 64 tokens
        c.a[:] = 0.01
    if how == "one token":
        c.a[:] = -np.abs(c.a)
        c.a[c.T // 2] = 60.0
        c.a[c.T // 2 + 1] = -58.0
    if how == "beyond":  # out of 32 bits after 40 tokens or so
        c.a[:] = 2.0


@pytest.mark.parametrize("how", ["until the last token", "by steps", "a little", "one token", "beyond"])
@pytest.mark.parametrize("new", [[8], [64], [140], [6, 90, 0, 33]])
@pytest.mark.parametrize("kh,vh,dk,dv,kind", [(1, 2, 64, 64, "bf16"), (1, 1, 64, 128, "f16"), (2, 2, 128, 64, "bf16"), (1, 2, 128, 128, "f16")])
def test_growth(gpu_ctx, how, new, kh, vh, dk, dv, kind):
    """Decays above 0 are taken as they are, whichever path a sequence takes; what leaves 32 bits reaches no earlier token."""
    rng = np.random.default_rng(sum(new) + dk)
    c = Delta(gpu_ctx, kh, vh, dk, dv, new, TYPES[kind], False, rng)
    grow(c, how, rng)
    c.run()
    seen, unseen = check_what_32_bits_hold(c)
    assert seen > 0 and (unseen > 0 or how != "beyond" or max(new) < 60 or kind == "f16")


def test_growth_across_launches(gpu_ctx):
    """256 heads of 128: about seven chunks to a launch; chunks that grow among ones that do not, at the borders too."""
    rng = np.random.default_rng(31)
    new = [40, 700, 3, 500]
    c = Delta(gpu_ctx, 256, 256, 128, 128, new, M.BF16, False, rng, states=np.zeros((9, 256, 128, 128)))
    c.source[:] = -1
    up = np.arange(c.T) // 64 % 3 == 1
    c.a[:] = np.where(up, 0.05, -np.abs(rng.normal(size=c.T)) * 0.3)[:, None]
    c.run()
    at = 1
    for s, n in enumerate(new):
        for h in (0, 255):
            i = slice(at, at + n)
            y, off, last, e = S.delta(c.q[i, h], c.k[i, h], c.v[i, h], c.a[i, h].astype(np.float64), c.b[i, h].astype(np.float64),
                                      np.zeros((128, 128)), 128 ** -0.5, 0.0, np.zeros(n), np.zeros(n))
            assert (np.abs(c.out[i, h] - y) <= off * 1.01 + 2.0 ** -8 * np.abs(y) * 1.01).all(), (s, h)
            assert (np.abs(c.kept[c.target[s], h] - last) <= e + 1e-37).all(), (s, h)
        at += n


@pytest.mark.parametrize("new", [[8], [64], [140], [40, 0, 70]])
@pytest.mark.parametrize("kh,vh,dk,dv,kind", [(1, 2, 64, 64, "bf16"), (1, 1, 64, 128, "f16"), (1, 2, 128, 64, "bf16"), (1, 2, 128, 128, "f16")])
def test_long_keys_without_values(gpu_ctx, new, kh, vh, dk, dv, kind):
    """What tokens would do to each other passes 32 bits, but they do nothing: only a sequence's last one has a value."""
    rng = np.random.default_rng(sum(new) + dv)
    c = Delta(gpu_ctx, kh, vh, dk, dv, new, TYPES[kind], False, rng)
    c.k = R.rounded(rng.normal(size=c.k.shape) * 3, c.kind)
    c.a[:], c.b[:], c.source[:] = 0.0, 1.0, -1
    last = 1 + np.cumsum(new) - 1
    v = np.zeros_like(c.v)
    v[last] = c.v[last]
    c.v = v
    c.run()
    seen, unseen = check_what_32_bits_hold(c)
    assert unseen == 0


@pytest.mark.parametrize("at", [0, 5, 40, 63, 64, 100])
@pytest.mark.parametrize("dk,dv,kind", [(64, 64, "bf16"), (128, 128, "bf16")])
def test_beta_beyond_32_bits_reaches_no_earlier_token(gpu_ctx, at, dk, dv, kind):
    rng = np.random.default_rng(at)
    c = Delta(gpu_ctx, 1, 2, dk, dv, [140], TYPES[kind], False, rng)
    c.k[at + 1] = R.rounded(c.k[at + 1] * 1e10, c.kind)
    c.b[at + 1, 1] = 1e30  # head 0 has only the long key
    c.run()
    seen, unseen = check_what_32_bits_hold(c, compare_states=False)
    assert seen >= at * dv * 2 and unseen > 0


@pytest.mark.parametrize("at", [3, 21, 40, 62, 80, 120])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("how", ["sum", "difference"])
def test_corrections_beyond_32_bits_reach_no_earlier_token(gpu_ctx, at, dk, dv, how):
    """Values near the largest that two tokens add up beyond it, or that a state takes to the last step of 32 bits."""
    rng = np.random.default_rng(at)
    c = Delta(gpu_ctx, 1, 2, dk, dv, [140], M.BF16, False, rng)
    big = R.rounded(np.array([3.38e38]), M.BF16)[0]
    i = at + 1
    c.a[i - 1:i + 2, 1] = 0.0
    if how == "sum":  # the second one's key is the first one's turned round: its correction is twice as large
        c.k[i] = -c.k[i - 1]
        c.v[i - 1, 1, 5] = c.v[i, 1, 5] = big
        c.b[i - 1:i + 1, 1] = 1.0
    else:  # within 32 bits, but not in parts of 8
        c.states[c.source[0], 1, :, 5] = 0.0
        c.k[i - 1] = np.eye(dk)[7]
        c.k[i] = np.eye(dk)[7]
        c.v[i - 1, 1, 5], c.v[i, 1, 5] = R.rounded(np.array([-0.8e36]), M.BF16)[0], R.rounded(np.array([3.3895e38]), M.BF16)[0]
        c.b[i - 1:i + 1, 1] = 1.0
    c.run()
    seen, unseen = check_what_32_bits_hold(c, compare_states=False)
    assert unseen > 0 and seen >= 140 * dv * 2 - 141


@pytest.mark.parametrize("new,deep", [(1, True), (4, True), (5, True), (6, True), (8, True), (9, False), (16, False), (40, False)])
@pytest.mark.parametrize("D,fmt", [(64, "f16"), (64, "mxint8"), (128, "f16"), (128, "mxfp4"), (256, "mxint8")])
def test_extend_weights_keep_the_bits_that_they_are_said_to(gpu_ctx, new, deep, D, fmt):
    """A first key far above the rest that has no value: up to 32 rows on average (4 heads) the rest's weights keep 11 bits down to
    2^-28 of the largest, with more rows down to 2^-25."""
    # Of the rest's weight e^-gap, in steps of 2^-24 below a largest one of 2^11 (2^8), the fraction is near a half: 0.3% of it
    # would be lost with three bits fewer than said.
    gap = 19.34375 if deep else 17.25
    n, group = 500, 4  # not cut into parts
    rng = np.random.default_rng(1)
    cache = Cached(gpu_ctx, FORMATS[fmt], 64, 1, D, [n], rng, scale=0.0)
    k, v = np.zeros((n, 1, D), np.float32), np.full((n, 1, D), 49152.0, np.float32)  # the same in each format
    k[0, 0, 0], v[0] = 16.0, 0.0
    t = np.arange(n)
    bk, bv, slots = R.Rows(gpu_ctx, k, M.F32), R.Rows(gpu_ctx, v, M.F32), R.i32(gpu_ctx, cache.table[0][t // 64] * 64 + t % 64)
    cache.kv.write(bk.heads, bv.heads, n, slots)
    cache.k[0], cache.v[0] = R.stored(k, FORMATS[fmt]), R.stored(v, FORMATS[fmt])
    assert (cache.v[0][1:] == 49152.0).all() and cache.k[0][0, 0, 0] == 16.0
    q = np.zeros((new, group, D))
    q[..., 0] = 1.0
    bq, out = R.Rows(gpu_ctx, q, M.F16), R.Rows(gpu_ctx, None, M.F16, new, group, D)
    dev = [R.i32(gpu_ctx, a) for a in ([0, new], [n], cache.table)]
    cache.kv.extend(bq.heads, new, 1, *dev, cache.table.shape[1], out.heads, scale=gap / 16.0)
    gpu_ctx.sync()
    y, _ = extend_ref(q, cache, [new], [n], gap / 16.0, 0, None, M.F16)
    # half a step of 2^-11 for a weight, the same for the output; what 32 bits add (a score near 28 in powers of two, sums of 500) is
    # less than 2^-17
    assert (np.abs(out.get() - y) <= (2.0 ** -10 + 2.0 ** -17) * np.abs(y)).all()
    for b in (bk, bv, slots, bq, out, *dev):
        b.free()
    cache.kv.close()


@pytest.mark.parametrize("n_seqs", [1024, 1025, 3000])
def test_delta_launches_go_by_rows_not_by_sequences(gpu_ctx, n_seqs):
    """A batch of single tokens has room for few long sequences, however many sequences it has."""
    kh, vh, D = 16, 32, 128
    rng = np.random.default_rng(1)
    q, k = (R.rounded(rng.normal(size=(n_seqs, kh, D)) / D ** 0.5, M.BF16) for _ in range(2))
    v = R.rounded(rng.normal(size=(n_seqs, vh, D)), M.BF16)
    a, b = -np.abs(rng.normal(size=(n_seqs, vh))).astype(np.float32), rng.uniform(0.1, 0.9, (n_seqs, vh)).astype(np.float32)
    rows = [R.Rows(gpu_ctx, x, M.BF16) for x in (q, k, v)] + [R.Rows(gpu_ctx, None, M.BF16, n_seqs, vh, D)]
    dev = [gpu_ctx.to_device(a), gpu_ctx.to_device(b), R.i32(gpu_ctx, np.arange(n_seqs + 1))]
    rule = M.DeltaRule(gpu_ctx, kh, vh, D, D)
    gpu_ctx.set_option(M.OPT_PROFILE, 1)
    gpu_ctx.profile_reset()
    rule.forward(rows[0].heads, rows[1].heads, rows[2].heads, *dev[:2], n_seqs, n_seqs, dev[2], rows[3].heads)
    gpu_ctx.sync()
    launches = {x: gpu_ctx.profile_read(x)[0] for x in ("delta_step", "delta_prepare", "delta_chunks")}
    gpu_ctx.set_option(M.OPT_PROFILE, 0)
    assert launches == {"delta_step": 1, "delta_prepare": 1, "delta_chunks": 1}, launches
    qk = np.repeat((q.astype(np.float64) * k).sum(-1), vh // kh, 1)
    y = D ** -0.5 * (qk * b)[..., None] * v  # from a state of zeros
    size = np.repeat(np.abs(q.astype(np.float64) * k).sum(-1), vh // kh, 1)
    tol = 2.0 ** -8 * np.abs(y) * 1.01 + (D + 8) * S.U * D ** -0.5 * (size * b)[..., None] * np.abs(v)
    assert (np.abs(rows[3].get() - y) <= tol).all()
    rule.close()
    for x in (*rows, *dev):
        x.free()


def test_delta_long_sequences_among_many_across_launches(gpu_ctx):
    """More sequences than each workgroup looks through, some long, with more chunks than the workspace holds at once."""
    n_seqs, kh, vh, D = 1500, 32, 128, 64
    rng = np.random.default_rng(2)
    new = rng.integers(0, 3, n_seqs)
    long = {0: 700, 1: 33, 700: 32, 701: 1500, 1023: 64, 1024: 65, 1300: 1100, n_seqs - 1: 90}
    for s, n in long.items():
        new[s] = n
    new = new.tolist()
    c = Delta(gpu_ctx, kh, vh, D, D, new, M.BF16, False, rng, states=np.zeros((len(long), vh, D, D)))
    c.source[:] = -1
    c.target[:] = -1
    for i, s in enumerate(long):
        c.target[s] = i
    c.run()
    first = 1 + np.concatenate([[0], np.cumsum(new)])
    for s in [*long, 2, 3, 699, 702, 1022, 1299]:
        for h in (0, 77, 127):
            i, n = slice(first[s], first[s] + new[s]), new[s]
            y, off, last, e = S.delta(c.q[i, h // 4], c.k[i, h // 4], c.v[i, h], c.a[i, h].astype(np.float64), c.b[i, h].astype(np.float64),
                                      np.zeros((D, D)), D ** -0.5, 0.0, np.zeros(n), np.zeros(n))
            assert (np.abs(c.out[i, h] - y) <= off * 1.01 + 2.0 ** -8 * np.abs(y) * 1.01).all(), (s, h)
            if c.target[s] >= 0:
                assert (np.abs(c.kept[c.target[s], h] - last) <= e + 1e-37).all(), (s, h)
    assert (c.out[:1] == c.mark).all() and (c.out[first[-1]:] == c.mark).all()


@pytest.mark.parametrize("cu,new", [([0, 60, 400], [60, 83]), ([-3, 4, 143], [4, 139]), ([-9, -2, 100], [0, 100]), ([0, 143, 500], [143, 0]),
                                    ([5, 9, 2 ** 31 - 1], [4, 134])])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_delta_offsets_outside_the_rows(gpu_ctx, cu, new, kind):
    """They are taken as the nearest inside: sequences, states and rows in no sequence as for those."""
    rng = np.random.default_rng(7)
    c = Delta(gpu_ctx, 1, 2, 64, 64, [140, 0], TYPES[kind], False, rng)  # 143 rows
    c.new = new
    c.run(cu=np.array(cu, np.int32), error="cu", start=max(cu[0], 0))
    c.check()


@pytest.mark.parametrize("per", [3, 40])
def test_decreasing_offsets_write_rows_and_targets_only(gpu_ctx, per):
    """All but the last sequence claim the same rows, by turns from the front: an error, and each row of the outputs and each target
    state as it was or with numbers in it; the next call is right."""
    n_seqs, rng = 9, np.random.default_rng(per)
    T = per * n_seqs
    cu = np.array([0, T - per] * 4 + [T - per, T], np.int32)[:n_seqs + 1]
    cu[-2:] = T - per, T
    c = Delta(gpu_ctx, 1, 2, 64, 64, [T - 3] + [0] * (n_seqs - 1), M.BF16, False, rng)
    c.source[:], c.target[:] = -1, np.arange(n_seqs)
    c.run(cu=cu, error="cu")
    assert np.isfinite(c.out).all() and np.isfinite(c.kept).all()
    assert (c.kept[n_seqs:] == c.states[n_seqs:]).all()
    c.new = [per] * n_seqs
    c.run(cu=offsets(c.new), start=0)
    c.check()
    x = R.rounded(rng.normal(size=(T, 1, 64)), M.BF16)
    w, bx, out = gpu_ctx.to_device(np.ones((64, 4), np.float32)), R.Rows(gpu_ctx, x, M.BF16), R.Rows(gpu_ctx, None, M.F32, T, 1, 64)
    states, dev = gpu_ctx.to_device(np.full((n_seqs + 1, 3, 64), 5.0, np.float32)), [R.i32(gpu_ctx, a) for a in (cu, np.arange(n_seqs))]
    for order, error in ((cu, True), (offsets([per] * n_seqs), False)):
        dev[0].upload(order)
        M.causal_conv(gpu_ctx, M.Rows(bx.buf, 64, M.BF16), w, 4, T, n_seqs, dev[0], M.Rows(out.buf, 64), states=states, n_slots=n_seqs + 1,
                      source=None, target=dev[1])
        sync_error(gpu_ctx, "cu") if error else gpu_ctx.sync()
        kept = states.download(np.float32).reshape(-1, 3, 64)
        assert np.isfinite(out.get()).all() and np.isfinite(kept).all() and (kept[n_seqs:] == 5.0).all()
    for s in range(n_seqs):
        y, off, last = S.conv(x[s * per:(s + 1) * per, 0], np.ones((64, 4)), None, False, np.zeros((3, 64)))
        assert (np.abs(out.get()[s * per:(s + 1) * per, 0] - y) <= off).all() and (kept[s] == last).all()
    for b in (w, bx, out, states, *dev):
        b.free()


def test_errors_of_entries_speak_of_their_kind_alone(gpu_ctx):
    """The convolution and the rule are no attention: their errors name the offsets or slots."""
    rng = np.random.default_rng(3)
    c = Delta(gpu_ctx, 1, 1, 64, 64, [3, 2], M.BF16, False, rng)
    c.source[0] = 99
    for change, kind, others in (({}, " source or target", (" cu", "attention", "slots")), ({"cu": np.array([0, 9, 4], np.int32)}, " cu", ("attention", "cu_q"))):
        with pytest.raises(M.MoeRocmError) as e:
            c.run(**change)
        assert kind in e.value.message and not any(x in e.value.message for x in others), e.value.message
        c.source[0] = 0
    gpu_ctx.sync()


@pytest.mark.parametrize("new", [[5], [64], [140], [7, 300, 33]])
@pytest.mark.parametrize("dk,dv,kind", [(64, 64, "bf16"), (64, 128, "f16"), (128, 128, "bf16"), (128, 64, "f16")])
def test_delta_states_to_32_bits(gpu_ctx, new, dk, dv, kind):
    """A head's state is off by a few half steps of 32 bits of its norm: a lost part or product of the matrix instructions' operands is
    twice the bound and more (tests/test_state_precision.py)."""
    c = Delta(gpu_ctx, 1, 2, dk, dv, new, TYPES[kind], False, np.random.default_rng(sum(new) + dk))
    c.a *= np.float32(S.STATE_DECAY / 0.3)
    c.v = R.rounded(c.v * S.STATE_VALUES / 2, c.kind)
    c.run()
    c.check()
    at = 1
    for s, n in enumerate(new):
        for h in range(2):
            i = slice(at, at + n)
            _, _, want, _ = S.delta(c.q[i, 0], c.k[i, 0], c.v[i, h], c.a[i, h].astype(np.float64), c.b[i, h], c.states[c.source[s], h], dk ** -0.5, 0.0, np.zeros(n), np.zeros(n))
            e = S.state_norm_error(c.kept[c.target[s], h], want)
            assert e <= S.STATE_NORM, (s, h, e / S.U)
        at += n


@pytest.mark.parametrize("what,x", [("value", np.inf), ("value", np.nan), ("key", np.inf), ("key", np.nan), ("beta", np.inf), ("beta", np.nan),
                                    ("decay", np.inf), ("decay", np.nan), ("query", np.inf), ("query", np.nan)])
@pytest.mark.parametrize("new,at", [([8], 0), ([8], 5), ([70], 3), ([70], 66), ([5, 140, 2], 6), ([5, 140, 2], 70), ([90, 4], 92)])
@pytest.mark.parametrize("dk,dv,kind,raw", [(64, 64, "f16", False), (128, 128, "bf16", True), (128, 64, "f16", True)])
def test_delta_what_is_not_finite_on_each_path(gpu_ctx, what, x, new, at, dk, dv, kind, raw):
    """It reaches its own sequence from its token on: a value its column, a key all columns, a decay or a beta those of its head, a query its
    own row and no state. Everything else has the bits of the call without it."""
    c = Delta(gpu_ctx, 1, 2, dk, dv, new, TYPES[kind], raw, np.random.default_rng(at + dk))
    row = at + 1
    clean = c.v.copy(), c.k.copy(), c.b.copy(), c.a.copy(), c.q.copy()
    if raw and what in ("beta", "decay"):
        x = np.nan  # raw gates of infinity stand for a beta of one, a decay of minus infinity
    if what == "value":
        c.v[row, 1, 5] = x
    if what == "key":
        c.k[row, 0, 3] = x
    if what == "beta":
        c.b[row, 1] = x
    if what == "decay":
        c.a[row, 1] = x
    if what == "query":
        c.q[row, 0, 9] = x
    c.run()
    out, kept = c.out, c.kept
    c.v, c.k, c.b, c.a, c.q = clean
    c.run()
    c.check()
    ends = 1 + np.cumsum(new)
    s = int((ends > row).argmax())
    heads = [0, 1] if what in ("key", "query") else [1]
    columns = [5] if what == "value" else slice(None)
    hit, lost = np.zeros(out.shape, bool), np.zeros(kept.shape, bool)
    for h in heads:
        hit[row:ends[s] if what != "query" else row + 1, h, columns] = True
        if what != "query":
            lost[c.target[s], h][:, columns] = True
    assert not np.isfinite(out[hit]).any() and (out[~hit] == c.out[~hit]).all()
    # of a state's column that is lost some number is not finite: a zero of a later key keeps a row of it
    assert (kept[~lost] == c.kept[~lost]).all()
    assert not np.isfinite(kept[c.target[s]][heads][..., columns]).all(1).any() if what != "query" else True


def test_delta_graph_of_many_sequences_sees_present_offsets(gpu_ctx):
    """A captured call of 1100 sequences, replayed with other offsets and decays, eager calls of other shapes on the same workspace between:
    the same bits as eager calls."""
    rng, n_seqs, T, D = np.random.default_rng(4), 1100, 1700, 64
    q, k, v = (R.rounded(rng.normal(size=(T, 1, D)) / 8, M.BF16) for _ in range(3))
    rows = [R.Rows(gpu_ctx, x, M.BF16) for x in (q, k, v)] + [R.Rows(gpu_ctx, None, M.BF16, T, 1, D)]
    plans = []
    for at, n, growth in ((3, 500, 0.0), (1099, 300, 0.05), (600, 40, 0.0)):
        new = rng.integers(0, 2, n_seqs)
        new[at], new[at // 2] = n, 70
        a = -np.abs(rng.normal(size=T)).astype(np.float32) * 0.1
        a[offsets(new)[at]:offsets(new)[at] + n // 2] += growth * 4
        plans.append((offsets(new), a))
    states = rng.normal(size=(n_seqs, 1, D, D)).astype(np.float32)
    cu, a, b = R.i32(gpu_ctx, plans[0][0]), gpu_ctx.to_device(plans[0][1]), gpu_ctx.to_device(rng.uniform(0.1, 0.9, T).astype(np.float32))
    ds, slots = gpu_ctx.to_device(states), R.i32(gpu_ctx, np.arange(n_seqs))
    rule = M.DeltaRule(gpu_ctx, 1, 1, D, D)
    mark = rows[3].all().copy()

    def call(n=n_seqs, tokens=T):
        rule.forward(rows[0].heads, rows[1].heads, rows[2].heads, a, b, tokens, n, cu, rows[3].heads, states=ds, n_slots=n_seqs, source=slots, target=slots)

    def start(plan):
        gpu_ctx.sync()
        cu.upload(plan[0]), a.upload(plan[1]), ds.upload(states), rows[3].buf.upload(mark)

    def results():
        gpu_ctx.sync()
        return rows[3].all().copy(), ds.download(np.float32).copy()

    want = []
    for plan in plans:
        start(plan)
        call()
        want.append(results())
    start(plans[0])
    gpu_ctx.graph_begin()
    call()
    graph = gpu_ctx.graph_end()
    for i in (0, 2, 1, 1, 0):
        start(plans[i])
        graph.launch()
        for x, y in zip(results(), want[i]):
            assert np.array_equal(x, y, equal_nan=True)
        start((np.concatenate([[0], np.full(n_seqs, 200)]).astype(np.int32), plans[i][1]))
        call(1, 200)
        gpu_ctx.sync()
    graph.close(), rule.close()
    for x in (*rows, cu, a, b, ds, slots):
        x.free()
