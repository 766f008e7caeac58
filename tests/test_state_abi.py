"""The C ABI over kept states without a GPU: exported symbols, the bindings against the header, and every refusal, on a
host-only context; and the plain forms the GPU tests compare with, at values worked out by hand."""
import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest

import moe_rocm as M
from moe_rocm import state as ST

import stateref as S
import test_attn_abi as AA
from test_attn_abi import hctx, refused  # noqa: F401

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "moe_rocm_state.h"
STATE_RS = ROOT / "moe-stream_amd" / "rust" / "moe-rocm-sys" / "src" / "state.rs"
X = 0x1000  # any non-NULL address: a host-only context never follows it


@pytest.fixture
def header(monkeypatch):
    monkeypatch.setattr(AA, "HEADER", HEADER)


def test_every_function_is_exported_and_bound(header):
    names = AA._functions()
    assert len(names) == 5
    assert set(names) <= set(M.exported_symbols())
    assert all(hasattr(M.lib, n) for n in names)


def test_python_structs_have_the_header_fields(header):
    size = {"u32": 4, "u64": 8, "f32": 4, "f64": 8}
    for name, cls in (("mr_rows", ST.CRows), ("mr_delta_desc", ST.DeltaDesc)):
        fields = AA._structs()[name]
        assert [f[0] for f in cls._fields_] == [f[0] for f in fields], name
        assert [C.sizeof(f[1]) for f in cls._fields_] == [size.get(t, 8) for _, t in fields], name


def test_rust_declarations_match_the_header(header):
    s = STATE_RS.read_text()
    block = s[s.index('extern "C" {'):]
    funcs = {}
    for m in re.finditer(r"pub fn (\w+)\((.*?)\)\s*(->\s*([^;]+))?;", block, flags=re.S):
        params = [" ".join(p.split(":", 1)[1].split()) for p in m.group(2).split(",") if p.strip()]
        funcs[m.group(1)] = (m.group(4).strip() if m.group(4) else None, params)
    assert funcs == AA._functions()
    structs = {m.group(1): re.findall(r"pub (\w+): ([^,\n]+),", m.group(2))
               for m in re.finditer(r"pub struct (\w+) \{(.*?)\n\}", s, flags=re.S)}
    assert {k: v for k, v in structs.items() if v} == AA._structs()
    assert "pub mod state;" in (STATE_RS.parent / "lib.rs").read_text()


def test_extend_refusals(hctx):  # noqa: F811
    kv = M.KvCache(hctx, M.KV_MXFP4, 4, 64, 2, 64)
    q = M.Heads(X, 16, M.BF16)

    def call(q=q, nq=5, n=3, cu=X, lens=X, table=X, pages=2, out=q, **kw):
        kv.extend(q, nq, n, cu, lens, table, pages, out, **kw)

    refused(M.MR_E_NODEV, "host-only", call)
    call(n=0), call(nq=0)
    call_most = (1 << 24) // 8
    refused(M.MR_E_NODEV, "host-only", call, nq=call_most - 1)
    for kw, status, text in (
            (dict(q=M.Heads(X, 16)), M.MR_E_UNSUPPORTED, "F16"), (dict(out=M.Heads(X, 16, M.F16)), M.MR_E_UNSUPPORTED, "F16"),
            (dict(out=M.Heads(X, 8, M.BF16)), M.MR_E_INVAL, "heads"),
            (dict(q=M.Heads(X, 15, M.BF16), out=M.Heads(X, 15, M.BF16)), M.MR_E_INVAL, "evenly"),
            (dict(q=None), M.MR_E_INVAL, "q is NULL"), (dict(out=None), M.MR_E_INVAL, "out is NULL"),
            (dict(cu=None), M.MR_E_INVAL, "cu_q"), (dict(cu=X + 2), M.MR_E_INVAL, "cu_q"),
            (dict(lens=None), M.MR_E_INVAL, "seq_len"), (dict(table=X + 2), M.MR_E_INVAL, "block_table"),
            (dict(pages=0), M.MR_E_INVAL, "max_pages"), (dict(pages=1 << 25), M.MR_E_INVAL, "max_pages"),
            (dict(n=65536), M.MR_E_INVAL, "n_seqs"), (dict(nq=call_most), M.MR_E_INVAL, "2^24"),
            (dict(scale=math.inf), M.MR_E_INVAL, "scale"), (dict(sinks=X + 1), M.MR_E_INVAL, "sinks"),
            (dict(q=M.Heads(X + 2, 16, M.BF16)), M.MR_E_INVAL, "aligned")):
        refused(status, text, call, **kw)
    many = M.KvCache(hctx, M.KV_MXFP4, 4, 64, 64, 64)
    q64 = M.Heads(X, 64, M.BF16)
    for nq, n in ((16 * ((1 << 18) - 2048 - 2), 1), (16, (1 << 16) - 1), (16 * ((1 << 18) - 2048 - 60000 - 1), 60000)):
        refused(M.MR_E_NODEV, "host-only", many.extend, q64, nq, n, X, X, X, 2, q64)
    for nq, n in ((16 * ((1 << 18) - 2048), 1), (16 * ((1 << 18) - 2048 - 60000), 60000)):
        refused(M.MR_E_INVAL, "too many tiles", many.extend, q64, nq, n, X, X, X, 2, q64)
    other = M.Context(M.DEVICE_NONE)
    many.close()
    assert M.lib.mr_attn_extend(other.h, kv.h, C.byref(q.c), 1, 1, X, X, X, 1, None, C.byref(q.c)) == M.MR_E_INVAL
    assert M.lib.mr_attn_extend(None, kv.h, C.byref(q.c), 1, 1, X, X, X, 1, None, C.byref(q.c)) == M.MR_E_INVAL
    other.close(), kv.close()


def test_conv_refusals(hctx):  # noqa: F811
    x = M.Rows(X, 64, M.BF16)

    def call(x=x, w=X, taps=4, n=5, seqs=2, cu=X, out=x, states=X, n_slots=4, source=X, target=X, **kw):
        M.causal_conv(hctx, x, w, taps, n, seqs, cu, out, states=states, n_slots=n_slots, source=source, target=target, **kw)

    refused(M.MR_E_NODEV, "host-only", call)
    refused(M.MR_E_NODEV, "host-only", call, n=0)  # states of sequences without tokens are still carried over
    refused(M.MR_E_NODEV, "host-only", call, states=None, source=None, target=None)
    call(seqs=0)
    for kw, status, text in (
            (dict(x=None), M.MR_E_INVAL, "x is NULL"), (dict(out=None), M.MR_E_INVAL, "out is NULL"),
            (dict(x=M.Rows(X, 60, M.BF16)), M.MR_E_INVAL, "width"), (dict(x=M.Rows(X, 0)), M.MR_E_INVAL, "width"),
            (dict(x=M.Rows(X, (1 << 20) + 8)), M.MR_E_INVAL, "width"), (dict(x=M.Rows(X, 64, 3)), M.MR_E_INVAL, "type"),
            (dict(out=M.Rows(X, 72)), M.MR_E_INVAL, "channels"), (dict(x=M.Rows(X + 8, 64)), M.MR_E_INVAL, "aligned"),
            (dict(x=M.Rows(X, 64, M.F16, 68)), M.MR_E_INVAL, "stride"), (dict(x=M.Rows(X, 64, M.F32, 1 << 40)), M.MR_E_INVAL, "2^40"),
            (dict(taps=1), M.MR_E_UNSUPPORTED, "taps"), (dict(taps=5), M.MR_E_UNSUPPORTED, "taps"),
            (dict(w=None), M.MR_E_INVAL, "w is NULL"), (dict(w=X + 4), M.MR_E_INVAL, "aligned"), (dict(bias=X + 4), M.MR_E_INVAL, "aligned"),
            (dict(cu=None), M.MR_E_INVAL, "cu"), (dict(cu=X + 1), M.MR_E_INVAL, "cu"), (dict(n=1 << 24), M.MR_E_INVAL, "n_tokens"),
            (dict(seqs=65536), M.MR_E_INVAL, "n_seqs"), (dict(states=None), M.MR_E_INVAL, "states"),
            (dict(states=None, source=None), M.MR_E_INVAL, "states"), (dict(states=X + 4), M.MR_E_INVAL, "states"),
            (dict(source=X + 2), M.MR_E_INVAL, "source"), (dict(target=X + 2), M.MR_E_INVAL, "target"),
            (dict(n_slots=1 << 31), M.MR_E_INVAL, "slots")):
        refused(status, text, call, **kw)
    assert M.lib.mr_causal_conv(None, None, None, 4, None, 0, 0, 0, None, None, 0, None, None, None) == M.MR_E_INVAL
    assert M.lib.mr_causal_conv(hctx.h, C.byref(x.c), X, 4, None, 2, 1, 1, X, None, 0, None, None, C.byref(x.c)) == M.MR_E_INVAL


@pytest.mark.parametrize("kw,status,text", [
    (dict(n_key_heads=0), M.MR_E_INVAL, "heads"), (dict(n_value_heads=0), M.MR_E_INVAL, "heads"),
    (dict(n_value_heads=3), M.MR_E_INVAL, "evenly"), (dict(n_value_heads=258), M.MR_E_INVAL, "1..256"),
    (dict(key_dim=96), M.MR_E_UNSUPPORTED, "key_dim"), (dict(value_dim=256), M.MR_E_UNSUPPORTED, "value_dim"),
    (dict(scale=math.nan), M.MR_E_INVAL, "scale"), (dict(unit_eps=-1.0), M.MR_E_INVAL, "unit_eps"),
    (dict(unit_eps=math.nan), M.MR_E_INVAL, "unit_eps"), (dict(gate_stride=3), M.MR_E_INVAL, "gate_stride"),
    (dict(gate_stride=1 << 40), M.MR_E_INVAL, "gate_stride"), (dict(a_log=X), M.MR_E_INVAL, "only one"),
    (dict(dt_bias=X), M.MR_E_INVAL, "only one"), (dict(a_log=X + 1, dt_bias=X), M.MR_E_INVAL, "aligned")])
def test_delta_description_refusals(hctx, kw, status, text):  # noqa: F811
    a = dict(n_key_heads=2, n_value_heads=4, key_dim=128, value_dim=128)
    a.update(kw)
    refused(status, text, M.DeltaRule, hctx, **a)


def test_delta_refusals(hctx):  # noqa: F811
    rule = M.DeltaRule(hctx, 2, 4, 128, 64)
    q, v = M.Heads(X, 2, M.F16), M.Heads(X, 4, M.F16)

    def call(q=q, k=q, v=v, decay=X, beta=X, n=5, seqs=2, cu=X, out=v, states=X, n_slots=4, source=X, target=X):
        rule.forward(q, k, v, decay, beta, n, seqs, cu, out, states=states, n_slots=n_slots, source=source, target=target)

    refused(M.MR_E_NODEV, "host-only", call)
    refused(M.MR_E_NODEV, "host-only", call, states=None, source=None, target=None)
    call(seqs=0)
    for kw, status, text in (
            (dict(q=None), M.MR_E_INVAL, "q is NULL"), (dict(k=None), M.MR_E_INVAL, "k is NULL"), (dict(v=None), M.MR_E_INVAL, "v is NULL"),
            (dict(out=None), M.MR_E_INVAL, "out is NULL"), (dict(q=M.Heads(X, 2)), M.MR_E_UNSUPPORTED, "F16"),
            (dict(k=M.Heads(X, 2, M.BF16)), M.MR_E_UNSUPPORTED, "F16"), (dict(out=M.Heads(X, 4, M.BF16)), M.MR_E_UNSUPPORTED, "F16"),
            (dict(q=M.Heads(X, 4, M.F16)), M.MR_E_INVAL, "heads"), (dict(v=M.Heads(X, 2, M.F16)), M.MR_E_INVAL, "heads"),
            (dict(v=M.Heads(X, 4, M.F16, token_stride=4)), M.MR_E_INVAL, "stride"),
            (dict(k=M.Heads(X, 2, M.F16, token_stride=1 << 24)), M.MR_E_INVAL, "2^24"), (dict(decay=None), M.MR_E_INVAL, "decay"),
            (dict(beta=X + 2), M.MR_E_INVAL, "beta"), (dict(cu=None), M.MR_E_INVAL, "cu"), (dict(n=1 << 24), M.MR_E_INVAL, "n_tokens"),
            (dict(seqs=65536), M.MR_E_INVAL, "n_seqs"), (dict(states=None), M.MR_E_INVAL, "states"),
            (dict(source=X + 2), M.MR_E_INVAL, "source"), (dict(n_slots=1 << 31), M.MR_E_INVAL, "slots")):
        refused(status, text, call, **kw)
    other = M.Context(M.DEVICE_NONE)
    r2 = M.DeltaRule(other, 2, 4, 128, 64)
    assert M.lib.mr_delta_rule(hctx.h, r2.h, *[C.byref(x.c) for x in (q, q, v)], X, X, 1, 1, X, None, 0, None, None,
                               C.byref(v.c)) == M.MR_E_INVAL
    assert M.lib.mr_delta_rule(hctx.h, None, None, None, None, None, None, 0, 0, None, None, 0, None, None, None) == M.MR_E_INVAL
    assert M.lib.mr_delta_create(hctx.h, None, None) == M.MR_E_INVAL
    r2.close(), other.close(), rule.close()


def test_plain_convolution():
    x, w = np.array([[1.0], [2.0], [4.0]]), np.array([[0.5, 0.25, 2.0]])
    y, _, last = S.conv(x, w, np.array([1.0]), False, np.array([[8.0], [16.0]]))
    assert y[:, 0].tolist() == [4 + 4 + 2 + 1, 8 + 0.25 + 4 + 1, 0.5 + 0.5 + 8 + 1] and last[:, 0].tolist() == [2.0, 4.0]
    y, _, last = S.conv(x[:1], w, None, True, np.array([[8.0], [16.0]]))
    assert abs(y[0, 0] - 10 / (1 + math.exp(-10))) < 1e-14 and last[:, 0].tolist() == [16.0, 1.0]


def test_plain_delta_rule():
    # one key element: S' = S / 2, corrected by half of what is missing
    k, q, v = np.array([[1.0], [0.0]]), np.array([[3.0], [1.0]]), np.array([[10.0], [5.0]])
    out, _, state, _ = S.delta(q, k, v, np.log([0.5, 0.25]), np.array([0.5, 1.0]), np.array([[4.0]]), 2.0, 0.0, np.zeros(2), np.zeros(2))
    assert np.allclose(out[:, 0], [2 * 3 * 6.0, 2 * 1.5], rtol=1e-15) and np.allclose(state, 1.5, rtol=1e-15)
    # a key seen with beta one answers with its value
    rng = np.random.default_rng(0)
    k = rng.normal(size=(1, 8))
    out, _, _, _ = S.delta(k, k, v[:1], np.array([-1.0]), np.ones(1), rng.normal(size=(8, 1)), 1.0, 1e-30, np.zeros(1), np.zeros(1))
    assert np.allclose(out, v[:1], rtol=1e-12)
