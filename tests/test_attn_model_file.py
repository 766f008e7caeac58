"""Attention shapes and frequencies from model files whose metadata is not the usual one: arrays with a number for each layer,
keys of another type, further keys that change the rotation. Read right, or refused."""
import numpy as np
import pytest

import moe_rocm as M

import attnref as R
import gguf_writer as G

BASE = [("general.architecture", G.STR, "x"), ("x.attention.head_count", G.U32, 64), ("x.attention.head_count_kv", G.U32, 8),
        ("x.attention.key_length", G.U32, 64)]
YARN = [("x.rope.scaling.type", G.STR, "yarn"), ("x.rope.scaling.factor", G.F32, 32.0),
        ("x.rope.scaling.original_context_length", G.U32, 4096)]


@pytest.fixture
def hctx():
    ctx = M.Context(M.DEVICE_NONE)
    yield ctx
    ctx.close()


@pytest.fixture
def file(tmp_path):
    opened = []

    def make(*more, without=(), tensors=(), arch="x"):
        meta = [(k.replace("x.", arch + ".", 1) if k.startswith("x.") else k, t, arch if k == "general.architecture" else v)
                for k, t, v in [m for m in BASE if m[0] not in without] + list(more)]
        path = tmp_path / f"{len(opened)}.gguf"
        G.write(path, meta, list(tensors))
        opened.append(M.GgufFile(path))
        return opened[-1]

    yield make
    for g in opened:
        g.close()


def refused(status, text, call, *a, **kw):
    with pytest.raises(M.MoeRocmError) as ei:
        call(*a, **kw)
    assert ei.value.status == status and text in ei.value.message, (ei.value.status, ei.value.message)


KV = "x.attention.head_count_kv"


def test_key_heads_for_each_layer(file, hctx):
    g = file((KV, G.ARR, (G.U32, [8, 8, 8, 8])), without=[KV])
    assert g.attention()["n_kv_heads"] == 8
    kv = g.kv_cache(hctx, M.KV_MXFP4, 4, 64)
    assert kv.desc.n_heads == 8
    kv.close()
    g = file((KV, G.ARR, (G.U32, [8, 4, 8, 2])), without=[KV])
    refused(M.MR_E_INVAL, "head_count_kv", g.attention)
    refused(M.MR_E_INVAL, "head_count_kv", g.kv_cache, hctx, M.KV_MXFP4, 4, 64)
    assert [g.attention(i)["n_kv_heads"] for i in range(4)] == [8, 4, 8, 2]
    kv = g.kv_cache(hctx, M.KV_MXFP4, 4, 64, layer=3)
    assert kv.desc.n_heads == 2
    kv.close()
    refused(M.MR_E_INVAL, "4 entries", g.attention, 4)
    refused(M.MR_E_INVAL, "negative", g.attention, -1)
    r = g.rope(hctx)  # one for all layers
    r.close()


def test_query_heads_for_each_layer(file):
    heads = "x.attention.head_count"
    g = file((heads, G.ARR, (G.I32, [64, 32])), without=[heads])
    assert [g.attention(i)["n_heads"] for i in range(2)] == [64, 32]
    refused(M.MR_E_INVAL, "head_count", g.attention)
    refused(M.MR_E_INVAL, "head_count", file(without=[heads]).attention)


def test_windows_for_each_layer(file):
    w = "x.attention.sliding_window"
    g = file((w, G.ARR, (G.U32, [128, 0, 64])))
    assert [g.attention(i)["window"] for i in range(3)] == [128, 0, 64]
    refused(M.MR_E_INVAL, "sliding_window", g.attention)
    # GPT-OSS's one window is that of its even layers, another model's that of all
    g = file((w, G.U32, 128), arch="gpt-oss")
    assert g.attention()["window"] == 128 and [g.attention(i)["window"] for i in range(4)] == [128, 0, 128, 0]
    g = file((w, G.U32, 128))
    assert [g.attention(i)["window"] for i in range(3)] == [128, 128, 128]
    g = file((w, G.ARR, (G.U32, [128, 256, 0, 64])), arch="gpt-oss")  # a number for each layer stands as it is
    assert [g.attention(i)["window"] for i in range(4)] == [128, 256, 0, 64]
    g = file((w, G.U32, 128), ("x.attention.sliding_window_pattern", G.ARR, (G.BOOL, [1, 0])))
    refused(M.MR_E_UNSUPPORTED, "sliding_window_pattern", g.attention, 0)


@pytest.mark.parametrize("key,vtype,value", [("x.attention.sliding_window", G.STR, "128"), (KV, G.STR, "8"), (KV, G.F32, 8.0),
                                             ("x.attention.key_length", G.F32, 64.0), ("x.attention.key_length", G.ARR, (G.U32, [64, 64])),
                                             ("x.rope.dimension_count", G.STR, "64"), (KV, G.ARR, (G.F32, [8.0]))])
def test_shapes_of_another_type_are_refused(file, key, vtype, value):
    refused(M.MR_E_INVAL, key, file((key, vtype, value), without=[key]).attention)


@pytest.mark.parametrize("key,vtype,value", [("x.rope.freq_base", G.U32, 500000), ("x.rope.freq_base", G.STR, "1e6"),
                                             ("x.rope.scaling.type", G.U32, 2), ("x.rope.dimension_count", G.F32, 64.0),
                                             ("x.rope.scaling.original_context_length", G.F32, 4096.0),
                                             ("x.rope.scaling.factor", G.U32, 32), ("x.rope.scaling.yarn_beta_fast", G.U32, 32)])
def test_frequencies_of_another_type_are_refused(file, hctx, key, vtype, value):
    more = [m for m in YARN if m[0] != key] + [(key, vtype, value)]
    refused(M.MR_E_INVAL, key, file(*more).rope, hctx)


def test_yarn_bounds_from_the_file(file, hctx):
    r0 = file(*YARN).rope(hctx)
    r1 = file(*YARN, ("x.rope.scaling.yarn_beta_fast", G.F32, 16.0), ("x.rope.scaling.yarn_beta_slow", G.F32, 2.0)).rope(hctx)
    r2 = M.Rope(hctx, 64, scaling=M.ROPE_YARN, factor=32.0, orig_context=4096, beta_fast=16.0, beta_slow=2.0)
    f0, f1, f2 = (r.frequencies()[0] for r in (r0, r1, r2))
    assert (f1 == f2).all() and (f0 != f1).any()
    for r in (r0, r1, r2):
        r.close()


def test_factor_on_cosine_and_sine(file, hctx):
    factor = ("x.rope.scaling.attn_factor", G.F32, 1.25)
    for more, kw, want in (((factor,), {}, 1.25), ((factor, ("x.rope.scaling.type", G.STR, "linear"), YARN[1]), {}, 1.25),
                           ((factor, *YARN), {"attn_factor": 1.5}, 1.5), (YARN, {}, R.rope_freqs(64, 10000.0, "yarn", 32.0, 4096)[1])):
        r = file(*more).rope(hctx, **kw)
        assert abs(r.frequencies()[1] - want) <= 2.0 ** -24 * want
        r.close()
    refused(M.MR_E_UNSUPPORTED, "attn_factor", file(factor, *YARN).rope, hctx)


@pytest.mark.parametrize("key,vtype,value", [("x.rope.scale_linear", G.F32, 4.0), ("x.rope.dimension_sections", G.ARR, (G.I32, [16, 24, 24, 0])),
                                             ("x.rope.freq_base_swa", G.F32, 10000.0), ("x.rope.scaling.yarn_log_multiplier", G.F32, 0.1),
                                             ("x.rope.scaling.yarn_ext_factor", G.F32, 0.5), ("x.rope.scaling.yarn_attn_factor", G.F32, 1.0)])
def test_other_rules_for_the_rotation_are_refused(file, hctx, key, vtype, value):
    refused(M.MR_E_UNSUPPORTED, key, file((key, vtype, value), *YARN).rope, hctx)


def test_keys_that_change_nothing_are_read_over(file, hctx):
    r0, r1 = file(*YARN).rope(hctx), file(("x.rope.scale_linear", G.F32, 1.0), ("x.rope.scaling.yarn_ext_factor", G.F32, 1.0),
                                          ("x.rope.scaling.yarn_log_multiplier", G.F32, 0.0), *YARN).rope(hctx)
    assert (r0.frequencies()[0] == r1.frequencies()[0]).all() and r0.frequencies()[1] == r1.frequencies()[1]
    r0.close(), r1.close()


def test_a_factor_for_each_frequency_is_refused(file, hctx):
    t = ("rope_freqs.weight", 0, (32,), np.ones(32, np.float32).tobytes())
    refused(M.MR_E_UNSUPPORTED, "rope_freqs", file(tensors=[t]).rope, hctx)


def test_values_of_another_width_are_refused(file, hctx):
    g = file(("x.attention.value_length", G.U32, 128))
    refused(M.MR_E_UNSUPPORTED, "width", g.attention)
    refused(M.MR_E_UNSUPPORTED, "width", g.kv_cache, hctx, M.KV_F16, 4, 64)
    assert file(("x.attention.value_length", G.U32, 64)).attention()["head_dim"] == 64
