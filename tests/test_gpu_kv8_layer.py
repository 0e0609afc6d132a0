"""The layer with per-head q/k norms (welvet_b200_mha_set_qk_norm) and an E4M3 KV cache
(welvet_b200_kv_create_e4m3): prefill, decode and extend against a 64-bit layer that
reads the same quantised cache. Tolerances are the layer's: FP32 1e-4, BF16 2e-2 of the
largest output."""
import numpy as np
import pytest

import welvet_b200 as W
from conftest import rel_err

pytestmark = pytest.mark.gpu
BLOCK = 16


class Ref:
    """The layer in 64 bits. Rows of q, k, v are rounded to BF16 where the layer's are."""

    def __init__(self, torch, d, heads, kv, hd, bf16=True, rope=True, norm=None, window=0, seed=0):
        self.t, self.heads, self.kv, self.hd, self.bf16, self.rope, self.window = torch, heads, kv, hd, bf16, rope, window
        self.weights = W.xavier_weights(d, heads * hd, kv * hd, seed)
        self.w = [self.round(torch.from_numpy(x).cuda().double()) for x in self.weights]
        self.norm = norm
        self.k, self.v = [], []  # per sequence: rows [n, kv, hd]

    def round(self, x):
        return x.bfloat16().double() if self.bf16 else x

    def heads_of(self, x, w, heads, pos, gamma):
        t, hd = self.t, self.hd
        y = (x @ w.T).view(len(x), heads, hd)
        if gamma is not None:
            y = self.round(y)
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gamma
        if self.rope and pos is not None:
            e = (t.arange(0, hd, 2, device="cuda", dtype=t.float32) / hd).double()
            ang = (pos[:, None] / 10000.0 ** e)[:, None]
            a, b = y.chunk(2, -1)
            y = t.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
        return self.round(y)

    def held(self, rows):
        """What an E4M3 cache holds of these rows: a power-of-two scale per block and head."""
        t, out = self.t, []
        for p in range(0, len(rows), BLOCK):
            x = rows[p:p + BLOCK]
            amax = x.abs().amax((0, 2))
            s = t.exp2(t.ceil(t.log2(amax / 448)).clamp_min(-64))[None, :, None]
            out.append((x / s).to(t.float8_e4m3fn).double() * s)
        return t.cat(out)

    def step(self, x, b, cached):
        """New rows of sequence b; cached: over the quantised cache, else as a prompt."""
        t = self.t
        first = len(self.k[b]) if b < len(self.k) else 0
        pos = t.arange(first, first + len(x), device="cuda", dtype=t.float64)
        gq, gk = self.norm if self.norm else (None, None)
        q = self.heads_of(x, self.w[0], self.heads, pos, gq)
        k, v = self.heads_of(x, self.w[1], self.kv, pos, gk), self.heads_of(x, self.w[2], self.kv, None, None)
        if b == len(self.k):
            self.k.append(k[:0])
            self.v.append(v[:0])
        self.k[b], self.v[b] = t.cat([self.k[b], k]), t.cat([self.v[b], v])
        k, v = (self.held(r) if cached else r for r in (self.k[b], self.v[b]))
        k, v = (r.repeat_interleave(self.heads // self.kv, 1) for r in (k, v))
        s = t.einsum("qhd,khd->hqk", q, k) / self.hd ** 0.5
        far = pos[:, None] - t.arange(len(k), device="cuda")[None]
        hide = (far < 0) | (far >= self.window) if self.window else far < 0
        a = t.einsum("hqk,khd->qhd", t.softmax(s.masked_fill(hide, float("-inf")), -1), v).reshape(len(x), -1)
        return self.round(a) @ self.w[3].T


def _gammas(torch, hd, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(1 + 0.3 * torch.randn(hd, device="cuda", generator=g)) for _ in range(2)]


@pytest.mark.parametrize("heads,kv,hd,norm,window", [
    (8, 2, 64, True, 0), (8, 2, 64, False, 0), (4, 4, 128, True, 0), (6, 3, 128, False, 24), (8, 4, 32, True, 0),
    (16, 1, 64, True, 40)])
def test_prefill_decode_extend(torch_cuda, heads, kv, hd, norm, window):
    torch = torch_cuda
    d, batch, T = 512, 3, 37
    gam = _gammas(torch, hd) if norm else None
    ref = Ref(torch, d, heads, kv, hd, norm=[g.double() for g in gam] if gam else None, window=window)
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1, max_seq_len=512, mask=3 if window else 1, window=window)
    layer = W.MhaLayer(cfg, *ref.weights)
    if norm:
        layer.set_qk_norm(*gam)
    cache = W.KvCache(layer, 4, 200, e4m3=True)
    g = torch.Generator(device="cuda").manual_seed(1)

    def rows(seq):
        return torch.randn(batch * seq, d, device="cuda", generator=g).bfloat16()

    def check(x, seq, post, cached):
        want = torch.cat([ref.step(x[b * seq:(b + 1) * seq].double(), b, cached) for b in range(batch)])
        assert rel_err(post.float().cpu().numpy(), want.cpu().numpy()) < 2e-2
    x = rows(T)
    post = torch.empty_like(x)
    layer.prefill(cache, batch, T, x, None, post)
    check(x, T, post, False)
    for seq in (1, 1, 5, 1, 70, 1):
        x = rows(seq)
        post, pre = torch.empty_like(x), torch.empty(batch * seq, heads * hd, device="cuda", dtype=torch.bfloat16)
        if seq == 1:
            layer.decode(cache, batch, x, pre, post)
        else:
            layer.extend(cache, batch, seq, x, pre, post)
        check(x, seq, post, True)
        assert bool(torch.isfinite(pre.float()).all())
    layer.check_device()


def test_extend_equals_decode_steps_and_host_buffers(torch_cuda):
    """Five tokens at once and one by one give the same rows up to BF16; host buffers give
    the device's."""
    torch = torch_cuda
    d, heads, kv, hd = 256, 8, 2, 64
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1, max_seq_len=256)
    layer = W.MhaLayer(cfg, *W.xavier_weights(d, heads * hd, kv * hd, 5))
    layer.set_qk_norm(*[t.cpu().numpy() for t in _gammas(torch, hd)])
    caches = [W.KvCache(layer, 2, 128, e4m3=True) for _ in range(3)]
    x0 = torch.randn(2 * 20, d, device="cuda").bfloat16()
    new = torch.randn(2, 5, d, device="cuda").bfloat16()
    post0 = torch.empty_like(x0)
    for c in caches:
        layer.prefill(c, 2, 20, x0, None, post0)
    once = torch.empty(2, 5, d, device="cuda", dtype=torch.bfloat16)
    layer.extend(caches[0], 2, 5, new.view(10, d), None, once.view(10, d))
    steps = torch.empty_like(once)
    for t in range(5):
        x, post = new[:, t].contiguous(), torch.empty(2, d, device="cuda", dtype=torch.bfloat16)
        layer.decode(caches[1], 2, x, None, post)
        steps[:, t] = post
    assert rel_err(once.float().cpu().numpy(), steps.float().cpu().numpy()) < 2e-2
    host = torch.empty(10, d, dtype=torch.bfloat16)
    layer.extend(caches[2], 2, 5, new.view(10, d).cpu(), None, host)
    assert torch.equal(host, once.view(10, d).cpu())


def test_fill_then_decode(torch_cuda):
    """kv_fill stores rows as they are given (position encoding done); a later fill of
    other lengths begins the cache anew."""
    torch = torch_cuda
    d, heads, kv, hd, n = 256, 4, 2, 64, 75
    ref = Ref(torch, d, heads, kv, hd)
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1, max_seq_len=256)
    layer = W.MhaLayer(cfg, *ref.weights)
    cache = W.KvCache(layer, 2, 160, e4m3=True)
    for scale, n in ((30.0, 90), (1.0, 75)):
        k, v = (torch.randn(2, n, kv * hd, device="cuda").bfloat16() * scale for _ in range(2))
        cache.fill(2, n, k, v)
    ref.k, ref.v = ([r[b].double().view(n, kv, hd) for b in range(2)] for r in (k, v))
    x = torch.randn(2, d, device="cuda").bfloat16()
    post = torch.empty_like(x)
    layer.decode(cache, 2, x, None, post)
    want = torch.cat([ref.step(x[b:b + 1].double(), b, True) for b in range(2)])
    assert rel_err(post.float().cpu().numpy(), want.cpu().numpy()) < 2e-2
    kh, vh = (t.cpu().view(torch.int16).numpy().view(np.uint16) for t in (k, v))
    cache.fill(2, n, kh, vh)  # host rows
    post2 = torch.empty_like(x)
    layer.decode(cache, 2, x, None, post2)
    assert torch.equal(post, post2)


@pytest.mark.parametrize("hd,rope", [(64, True), (32, True), (64, False)])
def test_norm_in_the_forward_of_fp32_layers(torch_cuda, hd, rope):
    """FP32 layers (3xTF32 attention for head_dim 64): the norm sits between the projection
    and the attention; taking it away gives the layer's own results back bit for bit."""
    torch = torch_cuda
    d, heads, kv, T = 128, 4, 2, 70
    gam = _gammas(torch, hd)
    ref = Ref(torch, d, heads, kv, hd, bf16=False, rope=rope, norm=[g.double() for g in gam])
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=0, max_seq_len=128, pos=0 if rope else 1)
    layer = W.MhaLayer(cfg, *ref.weights)
    x = torch.randn(2 * T, d, device="cuda")
    plain, post, again = (torch.empty_like(x) for _ in range(3))
    layer.forward(2, T, x, None, plain)
    layer.set_qk_norm(*gam)
    layer.forward(2, T, x, None, post)
    layer.set_qk_norm(None, None)
    layer.forward(2, T, x, None, again)
    want = torch.cat([ref.step(x[b * T:(b + 1) * T].double(), b, False) for b in range(2)])
    assert rel_err(post.cpu().numpy(), want.cpu().numpy()) < 1e-4
    assert torch.equal(plain, again) and not torch.equal(plain, post)


def test_lengths_without_rows_read_zeros(torch_cuda):
    torch = torch_cuda
    cfg = W.MhaConfig.make(128, 4, 2, head_dim=64, precision=1, max_seq_len=256)
    layer = W.MhaLayer(cfg, *W.xavier_weights(128, 256, 128, 0))
    cache = W.KvCache(layer, 2, 200, e4m3=True)
    cache.fill(2, 150)
    x = torch.randn(2, 128, device="cuda").bfloat16()
    pre, post = torch.empty(2, 256, device="cuda", dtype=torch.bfloat16), torch.empty_like(x)
    layer.decode(cache, 2, x, pre, post)
    layer.check_device()
    assert bool(torch.isfinite(pre.float()).all()) and float(pre.abs().max()) < 1.0  # one row in 151 is not zero


def test_refusals(torch_cuda):
    torch = torch_cuda
    d, heads, kv, hd = 128, 4, 2, 32
    weights = W.xavier_weights(d, heads * hd, kv * hd, 0)
    mk = lambda **kw: W.MhaLayer(W.MhaConfig.make(d, heads, kv, head_dim=hd, max_seq_len=64, **kw), *weights)  # noqa: E731
    for kw in (dict(precision=0), dict(precision=1, softmax=1), dict(precision=1, mask=2),
               dict(precision=1, mask=3, window=8, window_causal=0)):
        layer = mk(**kw)
        with pytest.raises(W.WelvetError) as e:
            W.KvCache(layer, 2, 32, e4m3=True)
        assert e.value.code == 2
    layer, other = mk(precision=1), mk(precision=1)
    cache = W.KvCache(layer, 2, 40, e4m3=True)
    plain = W.KvCache(layer, 2, 40)
    x = torch.zeros(2 * 3, d, device="cuda", dtype=torch.bfloat16)
    post = torch.empty_like(x)

    def refused(code, f, *a):
        with pytest.raises(W.WelvetError) as e:
            f(*a)
        assert e.value.code == code
    refused(2, layer.extend, plain, 2, 3, x, None, post)
    refused(1, other.extend, cache, 2, 3, x, None, post)
    refused(1, layer.extend, cache, 3, 2, x, None, post)   # more sequences than the cache has
    refused(1, layer.extend, cache, 2, 0, x, None, post)
    cache.fill(2, 38)
    refused(1, layer.extend, cache, 2, 3, x, None, post)   # 41 tokens in a cache of 40
    layer.extend(cache, 2, 2, x[:4], None, post[:4])
    refused(1, layer.decode, cache, 2, x[:2], None, post[:2])
    lib = W.lib()
    g = torch.ones(hd, device="cuda")
    assert lib.welvet_b200_mha_set_qk_norm(layer.handle, 1e-6, g.data_ptr(), None, 1).code == 1
    assert lib.welvet_b200_mha_set_qk_norm(layer.handle, float("nan"), g.data_ptr(), g.data_ptr(), 1).code == 1
    layer.check_device()
