"""CPU checks of the argument rules of the 4-bit KV cache's entry points and am_gfx950_qk_norm_rope: a refused call
returns its status before any device work, so none of this needs a GPU (the pointers are never followed)."""

import ctypes as C

import pytest

import aethermind_amd.native as N

P = 1 << 20  # a 16-byte aligned address that nothing follows


def norm_args(**kw):
    v = dict(q=P, k=P, q_out=P, k_out=P, rows=4, hq=8, hkv=2, head_dim=64, q_stride=512, k_stride=128, q_out_stride=512,
             k_out_stride=128, q_norm_w=P, k_norm_w=P, eps=1e-5, pos=P, cos_tab=P, sin_tab=P, max_pos=16, dtype=N.AM_DT_BF16)
    v.update(kw)
    return N.QkNormRopeArgs(**v)


def append_args(**kw):
    v = dict(q=P, k=P, v=P, q_out=P, batch=2, seq=3, hq=8, hkv=2, head_dim=64, q_stride=512, k_stride=128, v_stride=128,
             q_out_stride=512, q_norm_w=P, k_norm_w=None, eps=1e-5, cos_tab=P, sin_tab=P, max_pos=64, start_pos_dev=P, seq_lens=None,
             k_cache=P, v_cache=P, k_scales=P, v_scales=P, capacity=64, cache_batch_stride=2 * 64 * 64, cache_format=N.AM_KV_MXFP4,
             dtype=N.AM_DT_BF16, err_flag=None, pages=None)
    v.update(kw)
    return N.KvAppendArgs(**v)


def read_args(**kw):
    v = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, k_out=P, v_out=P, batch=2, seq=3, hkv=2, head_dim=64, capacity=64,
             cache_batch_stride=2 * 64 * 64, start_pos_dev=P, seq_lens=None, out_dtype=N.AM_DT_BF16, pages=None)
    v.update(kw)
    return N.Kv4ReadArgs(**v)


def attention_args(**kw):
    v = dict(q=P, out=P, k_codes=P, k_scales=P, v_codes=P, v_scales=P, batch=2, seq=3, hq=8, hkv=2, head_dim=64, capacity=64,
             cache_batch_stride=2 * 64 * 64, start_pos_dev=P, seq_lens=None, scale=0.0, dtype=N.AM_DT_BF16, workspace=P,
             workspace_bytes=1 << 40, pages=None)
    v.update(kw)
    return N.Kv4AttentionArgs(**v)


def pages(**kw):
    v = dict(block_table=P, block_size=32, table_stride=2, num_blocks=8, err_flag=None)
    v.update(kw)
    return C.pointer(N.KvPages(**v))


NAN, INF = float("nan"), float("inf")
BAD = {
    "am_gfx950_qk_norm_rope": (norm_args, [
        dict(dtype=N.AM_DT_F16), dict(rows=-1), dict(rows=1 << 31), dict(hq=-1), dict(hkv=-1), dict(hq=0, hkv=0), dict(hq=1 << 40),
        dict(head_dim=63), dict(head_dim=0), dict(head_dim=1026), dict(max_pos=0), dict(q_stride=511), dict(k_stride=127),
        dict(q_out_stride=0), dict(k_out_stride=-5), dict(eps=0.0), dict(eps=NAN), dict(eps=-1.0), dict(eps=INF), dict(q=None),
        dict(k=None), dict(q_out=None), dict(k_out=None), dict(pos=None), dict(cos_tab=None), dict(sin_tab=None),
        dict(rows=1 << 28)]),
    "am_gfx950_kv_append": (append_args, [
        dict(dtype=N.AM_DT_I8), dict(cache_format=2), dict(batch=-1), dict(seq=-1), dict(hq=-1), dict(hkv=0), dict(capacity=0),
        dict(head_dim=32), dict(head_dim=256, q_stride=4096, k_stride=512, v_stride=512, q_out_stride=4096),
        dict(head_dim=96, q_stride=4096, k_stride=512, v_stride=512, q_out_stride=4096, cache_batch_stride=1 << 20),
        dict(head_dim=65, q_stride=4096, k_stride=512, v_stride=512, q_out_stride=4096, cache_format=N.AM_KV_PLAIN),
        dict(max_pos=63), dict(q_stride=500), dict(k_stride=127), dict(v_stride=127), dict(q_out_stride=100), dict(eps=0.0),
        dict(eps=NAN), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(k_cache=None), dict(v_cache=None),
        dict(k_scales=None), dict(v_scales=None), dict(start_pos_dev=None), dict(cos_tab=None), dict(sin_tab=None),
        dict(k_cache=P + 8), dict(v_scales=P + 4), dict(capacity=48), dict(cache_batch_stride=2 * 64 * 64 + 64),
        dict(cache_batch_stride=64 * 64), dict(cache_batch_stride=0), dict(cache_batch_stride=-8192),
        dict(cache_batch_stride=64 * 64, cache_format=N.AM_KV_PLAIN), dict(batch=1 << 20, seq=1 << 20), dict(batch=1 << 60, seq=16),
        dict(capacity=1 << 31, max_pos=1 << 31, cache_batch_stride=1 << 40),
        dict(pages=pages(block_size=16)), dict(pages=pages(block_size=48)), dict(pages=pages(block_table=None)),
        dict(pages=pages(table_stride=1)), dict(pages=pages(num_blocks=0))]),
    "am_gfx950_kv4_read": (read_args, [
        dict(out_dtype=N.AM_DT_I32), dict(batch=-1), dict(seq=-1), dict(hkv=0), dict(capacity=0), dict(capacity=48),
        dict(head_dim=96), dict(head_dim=256), dict(k_codes=None), dict(k_scales=None), dict(v_codes=None), dict(v_scales=None),
        dict(k_out=None), dict(v_out=None), dict(k_out=P + 2), dict(start_pos_dev=None), dict(k_codes=P + 1),
        dict(cache_batch_stride=100), dict(batch=1 << 60, seq=16), dict(seq=1 << 27),
        dict(batch=1 << 24, seq=1, hkv=1, cache_batch_stride=64 * 64), dict(pages=pages(table_stride=1))]),
    "am_gfx950_kv4_attention": (attention_args, [
        dict(dtype=N.AM_DT_F16), dict(hq=0), dict(hkv=0), dict(hq=7), dict(hq=34), dict(batch=-1), dict(seq=-1), dict(capacity=0),
        dict(capacity=1 << 31), dict(capacity=40), dict(head_dim=96), dict(head_dim=32), dict(q=None), dict(out=None),
        dict(q=P + 2), dict(out=P + 8), dict(k_codes=None), dict(v_scales=None), dict(k_scales=P + 2), dict(start_pos_dev=None),
        dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(scale=3e38), dict(workspace=None), dict(workspace=P + 4), dict(workspace_bytes=0),
        dict(workspace_bytes=16384), dict(cache_batch_stride=33 * 64), dict(cache_batch_stride=-8192), dict(batch=1 << 17),
        dict(seq=1 << 25), dict(pages=pages(block_size=24)), dict(pages=pages(table_stride=1))]),
}


@pytest.mark.parametrize("name", sorted(BAD))
def test_refusals(name):
    lib = N.lib()
    make, bad = BAD[name]
    for kw in bad:
        with pytest.raises(N.NativeError) as e:
            lib.call(name, make(**kw), None)
        assert e.value.status == "INVALID_ARGUMENT", kw
        assert lib.last_error(), kw
    assert getattr(lib, name)(None, None) == N.AM_STATUS_INVALID_ARGUMENT


@pytest.mark.parametrize("name,kw", [("am_gfx950_qk_norm_rope", dict(rows=0, q=None)), ("am_gfx950_kv_append", dict(batch=0, k=None)),
                                     ("am_gfx950_kv_append", dict(seq=0)), ("am_gfx950_kv4_read", dict(batch=0, k_codes=None)),
                                     ("am_gfx950_kv4_attention", dict(seq=0, q=None)), ("am_gfx950_kv4_attention", dict(batch=0))])
def test_nothing_to_do(name, kw):
    N.lib().call(name, BAD[name][0](**kw), None)


def test_workspace_bytes():
    """never below the tickets; a workspace of a call's own size is accepted up to its last byte's check"""
    f = N.lib().am_gfx950_kv4_attention_workspace_bytes
    for bad in ((0, 1, 8, 2, 64, 64), (1, 0, 8, 2, 64, 64), (1, 1, 7, 2, 64, 64), (1, 1, 64, 2, 64, 64), (1, 1, 8, 0, 64, 64),
                (1, 1, 8, 2, 64, 0), (1 << 62, 1, 8, 2, 64, 64), (1, 1 << 62, 8, 2, 64, 64), (1, 1, 8, 2, 64, 1 << 62)):
        assert f(*bad) == 16384
    for shape in ((1, 1, 32, 8, 128, 131072), (16, 1, 32, 8, 128, 8192), (1, 1, 16, 1, 128, 1 << 20), (300, 1, 8, 2, 64, 4096),
                  (1, 37, 32, 8, 128, 1024), (1, 2048, 32, 8, 128, 8192)):
        need = f(*shape)
        assert 16384 <= need <= 64 << 20
        b, s, hq, hkv, d, cap = shape
        with pytest.raises(N.NativeError):
            N.lib().call("am_gfx950_kv4_attention", attention_args(batch=b, seq=s, hq=hq, hkv=hkv, head_dim=d, capacity=cap,
                                                                   cache_batch_stride=hkv * cap * d, workspace_bytes=need - 1), None)
