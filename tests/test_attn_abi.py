"""The attention side's C ABI without a GPU: exported symbols, the bindings against the header, and every
refusal, on a host-only context."""
import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest

import moe_rocm as M
from moe_rocm import attn as A

import attnref as R
import gguf_writer as G
from test_rust_binding import _strip_c_comments, c_to_rust

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "moe_rocm_attn.h"
ATTN_RS = ROOT / "moe-stream_amd" / "rust" / "moe-rocm-sys" / "src" / "attn.rs"
X = 0x1000  # any non-NULL address: a host-only context never follows it


def _functions():
    s = re.sub(r"#.*", "", _strip_c_comments(HEADER.read_text()))
    s = re.sub(r"typedef struct \w+ \{.*?\} \w+;", "", s, flags=re.S)
    out = {}
    for m in re.finditer(r"([\w\s\*]+?)\b(mr_\w+)\s*\(([^)]*)\)\s*;", s):
        params = [c_to_rust(re.match(r"(.*?[\s\*])(\w+)$", p.strip()).group(1)) for p in m.group(3).split(",")]
        ret = " ".join(m.group(1).split())
        out[m.group(2)] = (None if ret == "void" else c_to_rust(ret), params)
    return out


def _structs():
    s = _strip_c_comments(HEADER.read_text())
    out = {}
    for m in re.finditer(r"typedef struct (\w+) \{(.*?)\} \1;", s, flags=re.S):
        out[m.group(1)] = [(p.group(2), c_to_rust(p.group(1)))
                           for p in (re.match(r"(.*?[\s\*])(\w+)$", d.strip()) for d in m.group(2).split(";") if d.strip())]
    return out


def test_every_function_is_exported_and_bound():
    names = _functions()
    assert len(names) == 11
    assert set(names) <= set(M.exported_symbols())
    assert all(hasattr(M.lib, n) for n in names)


def test_python_structs_have_the_header_fields():
    size = {"u32": 4, "u64": 8, "f32": 4, "f64": 8}
    for name, cls in (("mr_heads", A.CHeads), ("mr_rope_desc", A.RopeDesc), ("mr_kv_desc", A.KvDesc),
                      ("mr_attn_opts", A.AttnOpts)):
        fields = _structs()[name]
        assert [f[0] for f in cls._fields_] == [f[0] for f in fields], name
        assert [C.sizeof(f[1]) for f in cls._fields_] == [size.get(t, 8) for _, t in fields], name


def test_rust_declarations_match_the_header():
    s = ATTN_RS.read_text()
    block = s[s.index('extern "C" {'):]
    funcs = {}
    for m in re.finditer(r"pub fn (\w+)\((.*?)\)\s*(->\s*([^;]+))?;", block, flags=re.S):
        params = [" ".join(p.split(":", 1)[1].split()) for p in m.group(2).split(",") if p.strip()]
        funcs[m.group(1)] = (m.group(4).strip() if m.group(4) else None, params)
    assert funcs == _functions()
    structs = {m.group(1): re.findall(r"pub (\w+): ([^,\n]+),", m.group(2))
               for m in re.finditer(r"pub struct (\w+) \{(.*?)\n\}", s, flags=re.S)}
    assert {k: v for k, v in structs.items() if v} == _structs()
    consts = dict(re.findall(r"pub const (MR_\w+): u32 = (\d+);", s))
    assert consts == dict(re.findall(r"#define (MR_\w+) (\d+)", HEADER.read_text()))
    assert "pub mod attn;" in (ATTN_RS.parent / "lib.rs").read_text()


@pytest.fixture
def hctx():
    ctx = M.Context(M.DEVICE_NONE)
    yield ctx
    ctx.close()


def refused(status, text, call, *a, **kw):
    with pytest.raises(M.MoeRocmError) as ei:
        call(*a, **kw)
    assert ei.value.status == status and text in ei.value.message, (ei.value.status, ei.value.message)


@pytest.mark.parametrize("kw,text", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=100), "head_dim"), (dict(head_dim=520), "head_dim"),
    (dict(rotary_dim=12), "rotary_dim"), (dict(rotary_dim=72), "rotary_dim"), (dict(layout=2), "layout"),
    (dict(scaling=4), "scaling"), (dict(base=1.0), "base"), (dict(base=math.nan), "base"), (dict(base=math.inf), "base"),
    (dict(scaling=M.ROPE_LINEAR, factor=0.5), "factor"), (dict(scaling=M.ROPE_YARN, factor=math.nan, orig_context=8), "factor"),
    (dict(scaling=M.ROPE_YARN, factor=2.0), "orig_context"),
    (dict(scaling=M.ROPE_YARN, factor=2.0, orig_context=64, beta_fast=1.0, beta_slow=2.0), "beta"),
    (dict(attn_factor=-1.0), "attn_factor"), (dict(attn_factor=math.inf), "attn_factor")])
def test_rope_refusals(hctx, kw, text):
    a = dict(head_dim=64)
    a.update(kw)
    refused(M.MR_E_INVAL, text, M.Rope, hctx, **a)


@pytest.mark.parametrize("scaling,code", [("plain", M.ROPE_PLAIN), ("linear", M.ROPE_LINEAR), ("yarn", M.ROPE_YARN),
                                          ("yarn_exact", M.ROPE_YARN_EXACT)])
@pytest.mark.parametrize("n,base,factor,orig", [(64, 150000.0, 32.0, 4096), (128, 1e6, 4.0, 32768), (8, 10000.0, 1.0, 64),
                                                (64, 10000.0, 40.0, 1)])
def test_rope_frequencies(hctx, scaling, code, n, base, factor, orig):
    r = M.Rope(hctx, 256, rotary_dim=n, base=base, scaling=code, factor=factor, orig_context=orig)
    f, mul = r.frequencies()
    rf, rmul = R.rope_freqs(n, base, scaling, factor, orig)
    # a power, a quotient and the ramp in 64 bits, the factor in 32
    assert np.allclose(f, rf, rtol=1e-13, atol=0) and abs(mul - rmul) <= 2.0 ** -24 * rmul
    r.close()


def test_qk_norm_rope_refusals(hctx):
    r = M.Rope(hctx, 64)
    q, k = M.Heads(X, 4), M.Heads(X, 2)

    def call(q=q, k=k, n=3, pos=X, q_out=q, k_out=k, rope=r, **kw):
        M.qk_norm_rope(hctx, rope, q, k, n, pos, q_out, k_out, **kw)

    refused(M.MR_E_NODEV, "host-only", call)
    refused(M.MR_E_NODEV, "host-only", call, k=None, k_out=None)
    call(n=0)
    for kw, text in ((dict(q=None), "q is NULL"), (dict(q_out=None), "q_out"), (dict(k=None), "only one"),
                     (dict(k_out=None), "only one"), (dict(q=M.Heads(X + 8, 4)), "aligned"),
                     (dict(q=M.Heads(X, 4, token_stride=258)), "stride"), (dict(q=M.Heads(X, 4, head_stride=66)), "stride"),
                     (dict(q=M.Heads(X, 4, M.F16), k=M.Heads(X, 2, M.BF16)), "one type"),
                     (dict(q_out=M.Heads(X, 4, M.F16)), "one type"),
                     (dict(q=M.Heads(X, 4, 3)), "type"), (dict(q=M.Heads(X, 0)), "heads"), (dict(q=M.Heads(X, 1025)), "heads"),
                     (dict(q_out=M.Heads(X, 5)), "head counts"), (dict(pos=None), "positions"), (dict(pos=X + 2), "positions"),
                     (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(q_norm=X + 4), "aligned"),
                     (dict(k=None, k_out=None, k_norm=X), "k_norm"), (dict(n=1 << 24), "n_tokens"),
                     (dict(q=M.Heads(X, 4, token_stride=1 << 40)), "2^40")):
        refused(M.MR_E_INVAL, text, call, **kw)
    assert M.lib.mr_qk_norm_rope(None, r.h, None, None, None, None, 0.0, None, 0, None, None) == M.MR_E_INVAL
    assert M.lib.mr_qk_norm_rope(hctx.h, None, None, None, None, None, 0.0, None, 0, None, None) == M.MR_E_INVAL
    other = M.Context(M.DEVICE_NONE)
    r2 = M.Rope(other, 64)
    refused(M.MR_E_INVAL, "another context", call, rope=r2)
    r2.close(), other.close(), r.close()


@pytest.mark.parametrize("desc,status,text", [
    ((5, 4, 64, 2, 64), M.MR_E_INVAL, "format"), ((4, 0, 64, 2, 64), M.MR_E_INVAL, "pages"),
    ((4, 4, 32, 2, 64), M.MR_E_INVAL, "page size"), ((4, 4, 96, 2, 64), M.MR_E_INVAL, "page size"),
    ((4, 4, 2048, 2, 64), M.MR_E_INVAL, "page size"), ((4, 4, 64, 0, 64), M.MR_E_INVAL, "heads"),
    ((4, 4, 64, 1025, 64), M.MR_E_INVAL, "heads"), ((4, 4, 64, 2, 80), M.MR_E_UNSUPPORTED, "head_dim"),
    ((4, 1 << 25, 64, 2, 64), M.MR_E_INVAL, "2^31")])
def test_cache_refusals(hctx, desc, status, text):
    refused(status, text, M.KvCache, hctx, *desc)
    assert M.KvCache.nbytes(*desc) == 0


def test_cache_bytes():
    # codes of keys and values, and a byte for each 32 of them
    assert M.KvCache.nbytes(M.KV_MXFP4, 3, 128, 4, 128) == 3 * 128 * 4 * 2 * (64 + 4)
    assert M.KvCache.nbytes(M.KV_MXINT8, 3, 64, 2, 256) == 3 * 64 * 2 * 2 * (256 + 8)
    assert M.KvCache.nbytes(M.KV_F16, 1, 1024, 8, 64) == 1024 * 8 * 2 * 128


def test_tokens_of_a_write_fit_a_launch(hctx):
    kv = M.KvCache(hctx, M.KV_MXFP4, 4, 64, 2, 64)
    h, most = M.Heads(X, 2, M.F16), 2 ** 30 - 64
    refused(M.MR_E_NODEV, "host-only", kv.write, h, h, most, X)
    refused(M.MR_E_NODEV, "host-only", kv.read, most, X, h, h)
    refused(M.MR_E_INVAL, "n_tokens", kv.write, h, h, most + 1, X)
    refused(M.MR_E_INVAL, "n_tokens", kv.read, most + 1, X, h, h)
    kv.close()


def test_write_and_read_refusals(hctx):
    kv = M.KvCache(hctx, M.KV_MXFP4, 4, 64, 2, 64)
    h = M.Heads(X, 2, M.F16)
    refused(M.MR_E_NODEV, "host-only", kv.write, h, M.Heads(X, 2), 3, X)
    refused(M.MR_E_NODEV, "host-only", kv.read, 3, X, h, None)
    kv.write(h, h, 0, X), kv.read(0, X, h, h)
    for a, text in (((None, h, 3, X), "k is NULL"), ((h, None, 3, X), "v is NULL"), ((M.Heads(X, 3), h, 3, X), "heads"),
                    ((h, M.Heads(X, 1), 3, X), "heads"), ((h, h, 3, None), "slots"), ((h, h, 3, X + 1), "slots"),
                    ((M.Heads(X + 4, 2), h, 3, X), "aligned"), ((h, h, 1 << 31, X), "n_tokens")):
        refused(M.MR_E_INVAL, text, kv.write, *a)
    for a, text in (((3, X, None, None), "NULL"), ((3, X, M.Heads(X, 3), None), "head count"), ((3, None, h, h), "slots"),
                    ((3, X, h, M.Heads(X, 2, 7)), "type"), ((1 << 31, X, h, h), "n_tokens")):
        refused(M.MR_E_INVAL, text, kv.read, *a)
    other = M.Context(M.DEVICE_NONE)
    assert M.lib.mr_kv_write(other.h, kv.h, C.byref(h.c), C.byref(h.c), 1, X) == M.MR_E_INVAL
    other.close(), kv.close()


def test_decode_refusals(hctx):
    kv = M.KvCache(hctx, M.KV_MXFP4, 4, 64, 2, 64)
    q = M.Heads(X, 16, M.BF16)

    def call(q=q, n=3, lens=X, table=X, pages=2, out=q, **kw):
        kv.attend(q, n, lens, table, pages, out, **kw)

    refused(M.MR_E_NODEV, "host-only", call)
    call(n=0)
    for kw, status, text in (
            (dict(q=M.Heads(X, 16)), M.MR_E_UNSUPPORTED, "F16"), (dict(out=M.Heads(X, 16, M.F16)), M.MR_E_UNSUPPORTED, "F16"),
            (dict(out=M.Heads(X, 8, M.BF16)), M.MR_E_INVAL, "heads"),
            (dict(q=M.Heads(X, 15, M.BF16), out=M.Heads(X, 15, M.BF16)), M.MR_E_INVAL, "evenly"),
            (dict(q=None), M.MR_E_INVAL, "q is NULL"), (dict(out=None), M.MR_E_INVAL, "out is NULL"),
            (dict(lens=None), M.MR_E_INVAL, "seq_len"), (dict(table=X + 2), M.MR_E_INVAL, "block_table"),
            (dict(pages=0), M.MR_E_INVAL, "max_pages"), (dict(pages=1 << 25), M.MR_E_INVAL, "max_pages"),
            (dict(n=65536), M.MR_E_INVAL, "n_seqs"), (dict(scale=math.inf), M.MR_E_INVAL, "scale"),
            (dict(scale=math.nan), M.MR_E_INVAL, "scale"), (dict(sinks=X + 1), M.MR_E_INVAL, "sinks"),
            (dict(q=M.Heads(X + 2, 16, M.BF16)), M.MR_E_INVAL, "aligned")):
        refused(status, text, call, **kw)
    kv.close()


def test_prefill_refusals(hctx):
    q, k = M.Heads(X, 16, M.F16), M.Heads(X, 2, M.F16)

    def call(D=64, q=q, k=k, v=k, nq=5, nk=5, n=1, cu_q=X, cu_k=X, out=q, **kw):
        M.attn_prefill(hctx, D, q, k, v, nq, nk, n, cu_q, cu_k, out, **kw)

    refused(M.MR_E_NODEV, "host-only", call)
    call(n=0), call(nq=0)
    for kw, status, text in (
            (dict(D=96), M.MR_E_UNSUPPORTED, "head_dim"), (dict(q=M.Heads(X, 16)), M.MR_E_UNSUPPORTED, "F16"),
            (dict(k=M.Heads(X, 2, M.BF16)), M.MR_E_UNSUPPORTED, "type of q"),
            (dict(v=M.Heads(X, 2, M.F32)), M.MR_E_UNSUPPORTED, "type of q"), (dict(v=M.Heads(X, 4, M.F16)), M.MR_E_INVAL, "heads"),
            (dict(k=M.Heads(X, 3, M.F16), v=M.Heads(X, 3, M.F16)), M.MR_E_INVAL, "evenly"),
            (dict(cu_q=None), M.MR_E_INVAL, "cu_q"), (dict(cu_k=X + 2), M.MR_E_INVAL, "cu_k"),
            (dict(nq=1 << 31), M.MR_E_INVAL, "2^31"), (dict(nq=1 << 28), M.MR_E_INVAL, "2^24"), (dict(scale=math.nan), M.MR_E_INVAL, "scale"),
            (dict(k=M.Heads(X, 2, M.F16, token_stride=1 << 24)), M.MR_E_INVAL, "2^24"),
            (dict(k=M.Heads(X, 2, M.F16, token_stride=4)), M.MR_E_INVAL, "stride"), (dict(v=None), M.MR_E_INVAL, "v is NULL")):
        refused(status, text, call, **kw)


def test_shapes_and_frequencies_from_a_model_file(hctx, tmp_path):
    arch = [("general.architecture", G.STR, "gpt-oss"), ("gpt-oss.attention.head_count", G.U32, 64),
            ("gpt-oss.attention.head_count_kv", G.U32, 8), ("gpt-oss.attention.key_length", G.U32, 64),
            ("gpt-oss.attention.sliding_window", G.U32, 128), ("gpt-oss.rope.freq_base", G.F32, 150000.0)]
    yarn = [("gpt-oss.rope.scaling.type", G.STR, "yarn"), ("gpt-oss.rope.scaling.factor", G.F32, 32.0),
            ("gpt-oss.rope.scaling.original_context_length", G.U32, 4096)]
    G.write(tmp_path / "a.gguf", arch + yarn, [])
    with M.GgufFile(tmp_path / "a.gguf") as g:
        assert g.attention() == dict(n_heads=64, n_kv_heads=8, head_dim=64, rotary_dim=64, window=128)
        r, kv = g.rope(hctx), g.kv_cache(hctx, M.KV_MXFP4, 4, 64)
        f, mul = r.frequencies()
        rf, rmul = R.rope_freqs(64, 150000.0, "yarn_exact", 32.0, 4096)
        assert np.allclose(f, rf, rtol=1e-13, atol=0) and abs(mul - rmul) <= 2.0 ** -24 * rmul
        assert (kv.desc.n_heads, kv.desc.head_dim) == (8, 64)
        r.close(), kv.close()
    # defaults: width from the embedding, as many key heads as heads, no scaling; part of a head rotated
    G.write(tmp_path / "b.gguf", [("general.architecture", G.STR, "x"), ("x.attention.head_count", G.U32, 4),
                                  ("x.embedding_length", G.U32, 512), ("x.rope.dimension_count", G.U32, 32)], [])
    with M.GgufFile(tmp_path / "b.gguf") as g:
        assert g.attention() == dict(n_heads=4, n_kv_heads=4, head_dim=128, rotary_dim=32, window=0)
        r = g.rope(hctx, M.ROPE_INTERLEAVED)
        f, mul = r.frequencies()
        assert np.allclose(f, R.rope_freqs(32, 10000.0)[0], rtol=1e-13, atol=0) and mul == 1.0
        r.close()
    G.write(tmp_path / "c.gguf", arch + [("gpt-oss.rope.scaling.type", G.STR, "su")], [])
    with M.GgufFile(tmp_path / "c.gguf") as g:
        refused(M.MR_E_UNSUPPORTED, "su", g.rope, hctx)


# The plain forms the GPU tests compare with, at values worked out by hand.
def test_stored_values_of_the_formats():
    x = np.zeros((1, 32))
    x[0, :9] = [6, 5, 2.5, 3.5, 0.25, 0.75, -1.25, 1.75, -0.2]
    assert (R.stored(x, M.KV_MXFP4)[0, :9] == [6, 4, 2, 4, 0, 1, -1, 2, 0]).all()
    x[0, 0] = 7.0
    assert R.stored(x, M.KV_MXFP4)[0, 0] == 6  # the scale stays
    x[0, 0] = 7.01
    assert (R.stored(x, M.KV_MXFP4)[0, :3] == [8, 4, 2]).all()  # twice the scale: 3.5, 2.5 and 1.25 of it
    x[0, :3] = [127.4, 0.5, 1.5]
    assert (R.stored(x, M.KV_MXINT8)[0, :3] == [127, 0, 2]).all()
    x[0, 0] = 127.5
    assert (R.stored(x, M.KV_MXINT8)[0, :3] == [128, 0, 2]).all()
    x[0, :3] = [np.inf, np.nan, 1e30]
    assert (R.stored(x, M.KV_MXFP4)[0, :3] == [49152, 0, 49152]).all()
    assert (R.stored(x, M.KV_MXINT8)[0, :3] == [65024, 0, 65024]).all()
    assert (R.stored(x, M.KV_F16)[0, :3] == [65504, 0, 65504]).all()
