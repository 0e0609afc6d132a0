"""Pointers of the q/k norm and E4M3 cache entries that no kernel could load from are
refused (code 1) before any device is touched: RoPE tables at 8 bytes, everything else at
its element's size. These run without a GPU, on pointers that are never followed."""
import ctypes as C

import pytest

import welvet_b200 as W
from test_kv8_args import _back, _cache, _config, _norm

P = 1 << 20


def _refused(st):
    assert st.code == 1 and b"misaligned" in st.message


@pytest.mark.parametrize("which", ["q", "k", "q_out", "k_out"])
@pytest.mark.parametrize("bf16,off", [(1, 1), (0, 2)])
def test_norm_rows(which, bf16, off):
    _refused(_norm(**{which: P + off, "bf16": bf16}))


@pytest.mark.parametrize("which", ["q_gamma", "k_gamma", "positions", "rope"])
def test_norm_tables(which):
    _refused(_norm(**{which: P + 2}))


def test_norm_table_between_its_pairs():
    _refused(_norm(rope=P + 4))
    _refused(_back(rope=P + 4))


@pytest.mark.parametrize("which", ["dqo", "dko", "dgq", "dgk"])
def test_norm_gradient(which):
    _refused(_back(**{which: P + 1}))


def test_rope_table():
    _refused(W.lib().welvet_b200_rope_table(4, 64, 1e4, P + 4, None))


@pytest.mark.parametrize("which", ["k_scale", "v_scale", "block_table", "ctx_len"])
def test_caches(which):
    c, cfg = _cache(**{which: P + 2}), _config()
    _refused(W.lib().welvet_b200_kv8_append(C.byref(c), 1, None, P, 128, P, 128, None, 0, None))
    _refused(W.lib().welvet_b200_kv8_attention(C.byref(cfg), C.byref(c), 1, None, 64, P, 512, P, 512, None))


def test_append_and_attention():
    c, cfg = _cache(), _config()
    for lens, k, v, rope in ((P + 2, P, P, P), (None, P + 1, P, P), (None, P, P + 1, P), (None, P, P, P + 4)):
        _refused(W.lib().welvet_b200_kv8_append(C.byref(c), 1, lens, k, 128, v, 128, rope, 8, None))
    for lens, q, out in ((P + 2, P, P), (None, P + 1, P), (None, P, P + 1)):
        _refused(W.lib().welvet_b200_kv8_attention(C.byref(cfg), C.byref(c), 1, lens, 64, q, 512, out, 512, None))
