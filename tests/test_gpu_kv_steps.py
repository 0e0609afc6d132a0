"""KV caches between the steps: a step that is refused leaves the lengths as they were, an
allocation that failed is not reported again by the next call, and every sequence may keep
a length of its own. Tolerances of the layers are those of test_gpu_kv8_layer.py; an E4M3
code is off by a relative 2^-4, or by half of the smallest step, scale * 2^-10."""
import pytest

import welvet_b200 as W
from conftest import rel_err
from test_gpu_kv8 import _cache, _config, _read
from test_gpu_kv8_layer import Ref, _gammas

pytestmark = pytest.mark.gpu


def _layer(d=256, heads=4, kv=2, hd=64, **kw):
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1, max_seq_len=512, **kw)
    return W.MhaLayer(cfg, *W.xavier_weights(d, heads * hd, kv * hd, 2))


@pytest.mark.parametrize("e4m3,seq", [(False, 1), (True, 1), (True, 6)])
def test_a_refused_step_leaves_the_cache(torch_cuda, e4m3, seq):
    """Rows at an odd 16-bit address are refused by the FP8 projection (code 2), after the
    argument checks. The next step gives what it gives on a cache without that call."""
    torch = torch_cuda
    layer = _layer(weight_format=1)
    x0 = torch.randn(2 * 21, 256, device="cuda").bfloat16()
    new = torch.randn(2 * seq, 256, device="cuda").bfloat16()
    odd = torch.zeros(2 * seq * 256 + 8, device="cuda").bfloat16()[1:1 + 2 * seq * 256].view(2 * seq, 256)
    post0, got = torch.empty_like(x0), []
    for refuse in (0, 3):
        cache = W.KvCache(layer, 2, 100, e4m3=e4m3)
        layer.prefill(cache, 2, 21, x0, None, post0)

        def step(x, post, pre=None):
            if seq == 1:
                layer.decode(cache, 2, x, pre, post)
            else:
                layer.extend(cache, 2, seq, x, pre, post)
        for _ in range(refuse):
            with pytest.raises(W.WelvetError) as e:
                step(odd, torch.empty_like(new))
            assert e.value.code == 2
        rows = []
        for _ in range(2):
            pre, post = torch.empty(2 * seq, 256, device="cuda", dtype=torch.bfloat16), torch.empty_like(new)
            step(new, post, pre)
            rows += [pre, post]
        layer.check_device()
        got.append(rows)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_failed_allocation_is_reported_once(torch_cuda):
    torch = torch_cuda
    layer = _layer()
    cache = W.KvCache(layer, 2, 100)
    with pytest.raises(W.WelvetError) as e:
        W.KvCache(layer, 400, 1 << 22)  # 2 x 429 GB
    assert e.value.code == 4 and "memory" in e.value.message
    cache.fill(2, 0)
    x = torch.randn(2, 256, device="cuda").bfloat16()
    layer.decode(cache, 2, x, None, torch.empty_like(x))
    layer.check_device()


@pytest.mark.parametrize("heads,kv,hd,e4m3,seq", [(8, 2, 64, True, 5), (8, 2, 128, True, 5), (8, 4, 32, True, 5), (8, 2, 64, False, 1)])
def test_lengths_of_each_sequence_equal_common_lengths(torch_cuda, heads, kv, hd, e4m3, seq):
    """What a sequence answers at its own length is, bit for bit, what it answers when all
    have that length."""
    torch = torch_cuda
    d, batch, T = 512, 4, 30
    layer = _layer(d, heads, kv, hd)
    x0, x1, x2 = (torch.randn(batch * n, d, device="cuda").bfloat16() for n in (T, seq, 1))

    def run(lengths):
        cache = W.KvCache(layer, batch, 64, e4m3=e4m3)
        layer.prefill(cache, batch, T, x0, None, torch.empty_like(x0))
        if seq > 1:
            layer.extend(cache, batch, seq, x1, None, torch.empty_like(x1))
        else:
            layer.decode(cache, batch, x1, None, torch.empty_like(x1))
        if isinstance(lengths, int):
            cache.fill(batch, lengths)
        else:
            cache.set_lengths(lengths)
        pre, post = torch.empty(batch, heads * hd, device="cuda", dtype=torch.bfloat16), torch.empty_like(x2)
        layer.decode(cache, batch, x2, pre, post)
        layer.check_device()
        return pre, post
    lengths = [T + seq, T, T + seq // 2, 17]
    own = run(lengths)
    for b, n in enumerate(lengths):
        assert all(torch.equal(a[b], c[b]) for a, c in zip(own, run(n)))


# (not head_dim 32: its prompts rotate keys that were rounded to BF16 once before, which
# the reference does not follow, and E4M3 codes of a block amplify that)
@pytest.mark.parametrize("heads,kv,hd,norm", [(8, 2, 64, False), (8, 2, 128, True)])
def test_sequences_keep_different_numbers_of_proposed_tokens(torch_cuda, heads, kv, hd, norm):
    """extend by five, keep some of them in each sequence, continue: the rows of a 64-bit
    layer that never saw the others."""
    torch = torch_cuda
    d, batch, T = 512, 4, 30
    gam = _gammas(torch, hd) if norm else None
    ref = Ref(torch, d, heads, kv, hd, norm=[g.double() for g in gam] if gam else None)
    layer = W.MhaLayer(W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1, max_seq_len=512), *ref.weights)
    if norm:
        layer.set_qk_norm(*gam)
    cache = W.KvCache(layer, batch + 1, 128, e4m3=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = lambda seq: torch.randn(batch * seq, d, device="cuda", generator=g).bfloat16()  # noqa: E731
    x = rows(T)
    post = torch.empty_like(x)
    layer.prefill(cache, batch, T, x, None, post)
    for b in range(batch):
        ref.step(x[b * T:(b + 1) * T].double(), b, False)
    lengths = [T] * batch
    for keep in ([5, 0, 2, 4], [1, 5, 3, 0], [0, 0, 5, 2]):
        x = rows(5)
        post = torch.empty_like(x)
        layer.extend(cache, batch, 5, x, None, post)
        want = torch.cat([ref.step(x[b * 5:(b + 1) * 5].double(), b, True) for b in range(batch)])
        assert rel_err(post.float().cpu().numpy(), want.cpu().numpy()) < 2e-2
        lengths = [n + k for n, k in zip(lengths, keep)]
        cache.set_lengths(lengths)
        for b, n in enumerate(lengths):
            ref.k[b], ref.v[b] = ref.k[b][:n], ref.v[b][:n]
        x = rows(1)
        post = torch.empty_like(x)
        layer.decode(cache, batch, x, None, post)
        want = torch.cat([ref.step(x[b:b + 1].double(), b, True) for b in range(batch)])
        assert rel_err(post.float().cpu().numpy(), want.cpu().numpy()) < 2e-2
        lengths = [n + 1 for n in lengths]
    layer.check_device()


@pytest.mark.parametrize("e4m3", [False, True])
def test_lengths_that_are_refused(torch_cuda, e4m3):
    layer = _layer()
    cache = W.KvCache(layer, 2, 50, e4m3=e4m3)
    for bad in ([], [1, 2, 3], [-1], [51], [3, 51]):
        with pytest.raises(W.WelvetError) as e:
            cache.set_lengths(bad)
        assert e.value.code == 1
    assert W.lib().welvet_b200_kv_set_lengths(cache.handle, 2, None, None).code == 1
    assert W.lib().welvet_b200_kv_set_lengths(None, 2, None, None).code == 1
    cache.set_lengths([50, 0])
    x = torch_cuda.zeros(2, 256, device="cuda", dtype=torch_cuda.bfloat16)
    with pytest.raises(W.WelvetError):  # full
        layer.decode(cache, 2, x, None, torch_cuda.empty_like(x))


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_a_cut_block_keeps_its_scale(torch_cuda, hd):
    """What the header says of dropped tokens: the block that is cut keeps their scale, the
    kept tokens the codes at it; a block cut at its start is begun anew."""
    torch = torch_cuda
    cache = _cache(torch, 1, [64], 1, hd, fill=0)
    rows = torch.randn(40, hd, device="cuda").clamp(-4, 4).bfloat16()
    rows[:, 0] = 4.0                      # the largest of every token: scale 2^-6
    rows[20, 1], rows[33, 1] = 4096.0, float("nan")
    ctx, (page,) = cache.tensors[5], cache.tensors[4][0].tolist()
    kscale = cache.tensors[2][page, 0]

    def append(at, x):
        ctx.fill_(at + len(x))
        W.kv8_append(cache, len(x), x, x)
    append(0, rows)
    assert kscale[0] == 2.0 ** -6 and kscale[1] == 16.0 and bool(torch.isnan(kscale[2]))
    append(20, rows[:1])                  # 20 tokens kept: cut behind the outlier's neighbours
    assert kscale[1] == 16.0
    held = _read(torch, cache, 0, 21, 0)[16:, 0]
    want = torch.cat([rows[16:20], rows[:1]]).double()
    assert bool(((held - want).abs() <= want.abs() * 2.0 ** -4 + 16 * 2.0 ** -10).all())
    append(16, rows[:3])                  # cut at the block's start: begun anew
    assert kscale[1] == 2.0 ** -6
    append(34, rows[:1])                  # behind a value that was not finite
    assert bool(torch.isnan(kscale[2]))
    append(32, rows[:1])
    assert kscale[2] == 2.0 ** -6
    W.device_check()


@pytest.mark.parametrize("hd", [64, 128, 96, 34])
@pytest.mark.parametrize("window", [0, 40])
def test_lengths_far_past_the_table_are_reported(torch_cuda, hd, window):
    """A length that the block table cannot hold, up to the largest there is, ends with
    code 4 and without a walk over its keys; other sequences are not touched by it."""
    torch = torch_cuda
    cache = _cache(torch, 3, [120] * 3, 2, hd)
    cfg = _config(4, 2, hd, **(dict(mask=3, window=window) if window else {}))
    q = torch.randn(3 * 2, 4 * hd, device="cuda").bfloat16()
    good = torch.empty_like(q)
    W.kv8_attention(cfg, cache, 2, q, good, 120)
    W.device_check()
    for wrong in (129, 1 << 20, (1 << 31) - 32, (1 << 31) - 1):
        cache.tensors[5][1] = wrong
        out = torch.empty_like(q)
        W.kv8_attention(cfg, cache, 2, q, out, 120)
        with pytest.raises(W.WelvetError) as e:
            W.device_check()
        assert e.value.code == 4 and "block table" in e.value.message
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])


@pytest.mark.parametrize("e4m3", [False, True])
def test_prefill_refuses_the_cache_of_another_shape(torch_cuda, e4m3):
    """The cache's layer says how its rows lie; decode takes no other layer's cache at all."""
    torch = torch_cuda
    layer = _layer(heads=4, kv=2, hd=64)
    cache = W.KvCache(layer, 2, 64, e4m3=e4m3)
    for other in (_layer(heads=4, kv=4, hd=64), _layer(heads=4, kv=2, hd=128), _layer(heads=4, kv=1, hd=64)):
        x = torch.randn(2 * 8, 256, device="cuda").bfloat16()
        with pytest.raises(W.WelvetError) as e:
            other.prefill(cache, 2, 8, x, None, torch.empty_like(x))
        assert e.value.code == 1
    single = W.MhaLayer(W.MhaConfig.make(256, 4, 2, head_dim=64, precision=0, max_seq_len=512), *W.xavier_weights(256, 256, 128, 2))
    x = torch.randn(2 * 8, 256, device="cuda")
    with pytest.raises(W.WelvetError) as e:
        single.prefill(cache, 2, 8, x, None, torch.empty_like(x))
    assert e.value.code == 1
    x = x.bfloat16()
    layer.prefill(cache, 2, 8, x, None, torch.empty_like(x))
    layer.check_device()


def test_lengths_are_read_before_the_call_returns(torch_cuda):
    """A page-locked array that changes right behind the call, the stream still busy."""
    torch = torch_cuda
    layer = _layer()
    x0, x = torch.randn(2 * 40, 256, device="cuda").bfloat16(), torch.randn(2, 256, device="cuda").bfloat16()
    big = torch.randn(8192, 8192, device="cuda").bfloat16()
    got = []
    for pinned in (False, True):
        cache = W.KvCache(layer, 2, 64)
        layer.prefill(cache, 2, 40, x0, None, torch.empty_like(x0))
        if pinned:
            lengths = torch.tensor([30, 11], dtype=torch.int32).pin_memory()
            for _ in range(20):
                big @ big
            W.check(W.lib().welvet_b200_kv_set_lengths(cache.handle, 2, lengths.data_ptr(), None))
            lengths.fill_(3)
        else:
            cache.set_lengths([30, 11])
        pre, post = torch.empty(2, 256, device="cuda", dtype=torch.bfloat16), torch.empty_like(x)
        layer.decode(cache, 2, x, pre, post)
        layer.check_device()
        got.append(pre)
    assert torch.equal(*got)
