"""Refusals of the q/k norm and E4M3 cache entries: argument checks that answer before
any device is touched (they run without a GPU)."""
import ctypes as C

import pytest

import welvet_b200 as W

P = 1 << 20  # a pointer that is never followed


def _norm(**kw):
    a = dict(tokens=4, heads=8, kv_heads=2, head_dim=64, eps=1e-6, q_gamma=P, k_gamma=P, rope=P, max_pos=8,
             positions=None, pos_mod=0, q=P, ldq=512, k=P, ldk=128, q_out=P, ldqo=512, k_out=P, ldko=128, bf16=1)
    a.update(kw)
    return W.lib().welvet_b200_qk_norm_rope_forward(*a.values(), None)


@pytest.mark.parametrize("bad,code", [
    (dict(tokens=-1), 1), (dict(heads=-1), 1), (dict(heads=0, kv_heads=0), 1), (dict(head_dim=0), 1),
    (dict(head_dim=63), 2), (dict(head_dim=514), 2), (dict(q=None), 1), (dict(k=None), 1), (dict(q_out=None), 1),
    (dict(k_out=None), 1), (dict(ldq=511), 1), (dict(ldk=127), 1), (dict(ldqo=100), 1), (dict(ldko=0), 1),
    (dict(max_pos=0), 1), (dict(eps=float("nan")), 1), (dict(tokens=1 << 31), 1), (dict(tokens=(1 << 31) // 10 + 1), 1),
])
def test_norm_refusals(bad, code):
    st = _norm(**bad)
    assert st.code == code and st.message.startswith(b"qk_norm_rope: ")


def _back(**kw):
    a = dict(tokens=4, heads=8, kv_heads=2, head_dim=64, eps=1e-6, q_gamma=P, k_gamma=P, rope=P, max_pos=8,
             positions=None, pos_mod=0, q=P, ldq=512, k=P, ldk=128, dqo=P, lddqo=512, dko=P, lddko=128, dq=P, lddq=512,
             dk=P, lddk=128, dgq=P, dgk=P, ws=P, bf16=1)
    a.update(kw)
    return W.lib().welvet_b200_qk_norm_rope_backward(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(q=None), dict(lddq=511)])
def test_norm_backward_shares_the_checks(bad):
    assert _back(**bad).code == 1


def test_workspace_size():
    assert W.qk_norm_rope_workspace(128) > 0 and W.qk_norm_rope_workspace(128) % 16 == 0
    assert W.qk_norm_rope_workspace(0) == 0 and W.qk_norm_rope_workspace(514) == 0


def test_rope_table_refusals():
    f = W.lib().welvet_b200_rope_table
    for args in ((0, 64, 1e4, P), (4, 63, 1e4, P), (4, 0, 1e4, P), (4, 64, 0.0, P), (4, 64, float("nan"), P), (4, 64, 1e4, None)):
        assert f(*args, None).code == 1


def _cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, block_table=P, ctx_len=P, batch=2, pages=9, max_pages=4, kv_heads=2, head_dim=64)
    a.update(kw)
    return W._Kv8CacheArgs(*a.values())


BAD_CACHES = [(dict(k=None), 1), (dict(v=None), 1), (dict(k_scale=None), 1), (dict(v_scale=None), 1),
              (dict(block_table=None), 1), (dict(ctx_len=None), 1), (dict(batch=0), 1), (dict(batch=65536), 1),
              (dict(pages=0), 1), (dict(max_pages=0), 1), (dict(max_pages=1 << 26), 1), (dict(kv_heads=0), 1),
              (dict(head_dim=0), 1), (dict(head_dim=65), 2), (dict(head_dim=258), 2)]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_refusals(bad, code):
    c = _cache(**bad)
    st = W.lib().welvet_b200_kv8_append(C.byref(c), 1, None, P, 4096, P, 4096, None, 0, None)
    assert st.code == code and st.message.startswith(b"kv8_append: ")
    cfg = _config()
    st = W.lib().welvet_b200_kv8_attention(C.byref(cfg), C.byref(c), 1, None, 64, P, 4096, P, 4096, None)
    assert st.code == code and st.message.startswith(b"kv8_attention: ")


def test_append_refusals():
    f, c = W.lib().welvet_b200_kv8_append, _cache()
    for seq, k, ldk, v, ldv, rope, max_pos in ((0, P, 128, P, 128, None, 0), (1, None, 128, P, 128, None, 0),
                                               (1, P, 128, None, 128, None, 0), (1, P, 127, P, 128, None, 0),
                                               (1, P, 128, P, 127, None, 0), (1, P, 128, P, 128, P, 0)):
        assert f(C.byref(c), seq, None, k, ldk, v, ldv, rope, max_pos, None).code == 1
    assert f(None, 1, None, P, 128, P, 128, None, 0, None).code == 1


def _config(**kw):
    kv = kw.pop("num_kv_heads", 2)
    return W.MhaConfig.make(512, 8, kv, **{**dict(head_dim=64, precision=1), **kw})


@pytest.mark.parametrize("kw,code", [(dict(precision=0), 2), (dict(softmax=1), 2), (dict(mask=2), 2), (dict(mask=4), 2),
                                     (dict(mask=3, window_causal=0), 2), (dict(head_dim=128), 1),
                                     (dict(num_kv_heads=4), 1), (dict(head_begin=0, head_count=4), 1),
                                     (dict(head_begin=2, head_count=4), 1)])
def test_attention_configurations(kw, code):
    cfg, c = _config(**kw), _cache()
    st = W.lib().welvet_b200_kv8_attention(C.byref(cfg), C.byref(c), 1, None, 64, P, 4096, P, 4096, None)
    assert st.code == code


def test_attention_refusals():
    f, c, cfg = W.lib().welvet_b200_kv8_attention, _cache(), _config()
    for seq, max_ctx, q, ldq, out, ldo in ((0, 64, P, 512, P, 512), (1, 0, P, 512, P, 512), (1, 64, None, 512, P, 512),
                                           (1, 64, P, 512, None, 512), (1, 64, P, 511, P, 512), (1, 64, P, 512, P, 511),
                                           (1 << 29, 64, P, 512, P, 512)):
        assert f(C.byref(cfg), C.byref(c), seq, None, max_ctx, q, ldq, out, ldo, None).code == 1
    assert f(None, C.byref(c), 1, None, 64, P, 512, P, 512, None).code == 1
    assert f(C.byref(cfg), None, 1, None, 64, P, 512, P, 512, None).code == 1
