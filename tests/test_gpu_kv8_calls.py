"""How the q/k norms and the E4M3 cache are called: captured in a CUDA graph, without
allocations, twice with the same bits; the layer with norms over BF16 and FP32 caches."""
import pytest

import welvet_b200 as W
from conftest import rel_err
from test_gpu_kv8 import _cache, _config
from test_gpu_kv8_layer import Ref, _gammas
from test_gpu_threads import bare_calls, bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_captured_in_a_graph(torch_cuda, hd):
    torch = torch_cuda
    calls = bare_calls(torch, hd)
    for _, call, _ in calls:
        call()
    torch.cuda.synchronize()
    want = [bits(torch, outs) for _, _, outs in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _, call, _ in calls:
            call(torch.cuda.current_stream())
    for name, _, outs in calls:
        if name != "append":  # it adds to what the cache holds
            for t in outs:
                t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for (name, _, outs), same in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(bits(torch, outs), same)), name
    W.device_check()


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_nothing_is_allocated_after_the_first_call(torch_cuda, hd):
    torch = torch_cuda
    calls = bare_calls(torch, hd)
    for _, call, _ in calls:
        call()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(20):
        for _, call, _ in calls:
            call()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free


def test_append_token_by_token_holds_the_same_scales(torch_cuda):
    """A running maximum of powers of two: one call and many give the same scales, in
    whole blocks and in the last, partial one."""
    torch = torch_cuda
    for n in (37, 48):
        kv, hd = 2, 64
        g = torch.Generator(device="cuda").manual_seed(3)
        k = (torch.randn(n, kv * hd, device="cuda", generator=g) * torch.randn(n, 1, device="cuda", generator=g).mul(3).exp()).bfloat16()
        v = (torch.randn(n, kv * hd, device="cuda", generator=g) * torch.randn(n, 1, device="cuda", generator=g).exp()).bfloat16()
        once, steps = (_cache(torch, 1, [n], kv, hd, fill=0x7f, seed=1) for _ in range(2))
        W.kv8_append(once, n, k, v)
        for t in range(n):
            steps.tensors[5].fill_(t + 1)
            W.kv8_append(steps, 1, k[t:t + 1], v[t:t + 1])
        W.device_check()
        for which in (2, 3):
            assert torch.equal(once.tensors[which], steps.tensors[which])


@pytest.mark.parametrize("hd", [64, 128, 256, 96])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_norm_gradient_repeats_every_output(torch_cuda, hd, dtype):
    torch = torch_cuda
    tokens, heads, kv = 701, 6, 2
    rows = lambda h: torch.randn(tokens, h * hd, device="cuda").to(getattr(torch, dtype))  # noqa: E731
    q, k, dyq, dyk = rows(heads), rows(kv), rows(heads), rows(kv)
    gam = _gammas(torch, hd)
    ws = torch.empty(W.qk_norm_rope_workspace(hd), dtype=torch.uint8, device="cuda")
    got = []
    for _ in range(4):
        outs = [torch.empty_like(q), torch.empty_like(k), torch.empty(hd, device="cuda"), torch.empty(hd, device="cuda")]
        W.qk_norm_rope_backward(q, k, dyq, dyk, *outs, hd, ws, *gam)
        got.append(outs)
    assert all(torch.equal(a, b) for o in got[1:] for a, b in zip(got[0], o))


@pytest.mark.parametrize("batch,seq,ctx,heads,kv,hd", [(1, 1, 517, 32, 8, 128), (8, 1, 3000, 16, 2, 64), (4, 5, 2100, 32, 8, 128),
                                                       (1, 700, 1500, 8, 2, 128), (2, 1, 900, 6, 2, 96)])
def test_attention_repeats(torch_cuda, batch, seq, ctx, heads, kv, hd):
    torch = torch_cuda
    cache = _cache(torch, batch, [ctx - 3 * b for b in range(batch)], kv, hd)
    q = torch.randn(batch * seq, heads * hd, device="cuda").bfloat16()
    outs = [torch.empty_like(q) for _ in range(20)]
    for o in outs:
        W.kv8_attention(_config(heads, kv, hd), cache, seq, q, o, ctx)
    W.device_check()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("heads,kv,hd,bf16,rope", [(8, 2, 64, True, True), (4, 4, 128, True, True),
                                                   (8, 2, 64, True, False), (8, 2, 64, False, True), (4, 2, 128, False, False)])
def test_layer_norms_over_bf16_and_fp32_caches(torch_cuda, heads, kv, hd, bf16, rope):
    torch = torch_cuda
    d, batch, T = 512, 3, 37
    gam = _gammas(torch, hd)
    ref = Ref(torch, d, heads, kv, hd, bf16=bf16, rope=rope, norm=[g.double() for g in gam])
    cfg = W.MhaConfig.make(d, heads, kv, head_dim=hd, precision=1 if bf16 else 0, max_seq_len=512, pos=0 if rope else 1)
    layer = W.MhaLayer(cfg, *ref.weights)
    layer.set_qk_norm(*gam)
    cache = W.KvCache(layer, 4, 100)
    kind = torch.bfloat16 if bf16 else torch.float32
    for step in range(4):
        seq = 1 if step else T
        x = torch.randn(batch * seq, d, device="cuda").to(kind)
        post = torch.empty_like(x)
        if step:
            layer.decode(cache, batch, x, None, post)
        else:
            layer.prefill(cache, batch, T, x, None, post)
        want = torch.cat([ref.step(x[b * seq:(b + 1) * seq].double(), b, False) for b in range(batch)])
        assert rel_err(post.float().cpu().numpy(), want.cpu().numpy()) < (2e-2 if bf16 else 1e-4)
    layer.check_device()
