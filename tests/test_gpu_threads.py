"""Entries called from a thread that has made no CUDA call yet: it has no context of its
own, and the answers are those of the main thread."""
import threading

import pytest

import welvet_b200 as W
from test_gpu_kv8 import _cache, _config
from test_gpu_kv8_layer import _gammas

pytestmark = pytest.mark.gpu


def in_new_thread(call):
    errors = []

    def body():
        try:
            call()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    t = threading.Thread(target=body)
    t.start()
    t.join()
    if errors:
        raise errors[0]


def bits(torch, ts):
    return [t.clone().view(torch.uint8) for t in ts]


def bare_calls(torch, hd=128):
    """(name, call, outputs) of every bare operator, on buffers of their own."""
    heads, kv, seq, ctx = 8, 2, 3, [130, 77]
    rows = 2 * seq
    g = torch.Generator(device="cuda").manual_seed(hd)
    r = lambda n: torch.randn(rows, n * hd, device="cuda", generator=g).bfloat16()  # noqa: E731
    q, k, v, dq, dk = r(heads), r(kv), r(kv), r(heads), r(kv)
    cache = _cache(torch, 2, ctx, kv, hd)
    table = torch.empty(160, hd // 2, 2, device="cuda")
    gam = _gammas(torch, hd)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    qo, ko, dqo, dko, out = (torch.empty_like(t) for t in (q, k, q, k, q))
    dg = torch.empty(2, hd, device="cuda")
    ws = torch.empty(W.qk_norm_rope_workspace(hd), device="cuda", dtype=torch.uint8)
    cfg = _config(heads, kv, hd)
    return [
        ("rope_table", lambda s=None: W.rope_table(160, hd, table, stream=s), [table]),
        ("norm", lambda s=None: W.qk_norm_rope(q, k, qo, ko, hd, *gam, rope=table, positions=pos, stream=s), [qo, ko]),
        ("norm gradient", lambda s=None: W.qk_norm_rope_backward(q, k, dq, dk, dqo, dko, dg[0], dg[1], hd, ws, *gam, rope=table,
                                                                 positions=pos, stream=s), [dqo, dko, dg]),
        ("append", lambda s=None: W.kv8_append(cache, seq, k, v, rope=table, stream=s), list(cache.tensors[:4])),
        ("attention", lambda s=None: W.kv8_attention(cfg, cache, seq, q, out, max(ctx), stream=s), [out]),
    ]


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_bare_operators(torch_cuda, hd):
    torch = torch_cuda
    calls = bare_calls(torch, hd)
    for _, call, _ in calls:
        call()
    torch.cuda.synchronize()
    want = [bits(torch, outs) for _, _, outs in calls]
    for (name, call, outs), same in zip(calls, want):
        in_new_thread(call)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bits(torch, outs), same)), name
    W.device_check()


def test_gemm_and_prefill_attention(torch_cuda):
    torch = torch_cuda
    a, b = (torch.randn(256, 256, device="cuda").bfloat16() for _ in range(2))
    c = torch.empty(256, 256, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(2 * 128, 4 * 64, device="cuda").bfloat16()
    o = torch.empty_like(q)
    cfg = _config(4, 4, 64, max_seq_len=128)
    for call, out in ((lambda: W.gemm(0, 256, 256, 256, a, b, c, out_bf16=1), c),
                      (lambda: W.attention(cfg, 2, 128, q, q, q, o), o)):
        call()
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        in_new_thread(call)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    W.device_check()
