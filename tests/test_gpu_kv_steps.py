"""KV caches between the steps: a step that is refused leaves the lengths as they were, and
an allocation that failed is not reported again by the next call."""
import pytest

import welvet_b200 as W

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
