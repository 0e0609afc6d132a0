"""Per-head q/k RMS norm with the position rotation (welvet_b200_qk_norm_rope_*) against
the formula in 64 bits, and its gradient against the formula's and against differences.

FP32 rows: a sum of hd squares, a reciprocal root, four products and a sum, each
rounded to 2^-24: below 2^-20 of the row's largest value for hd <= 512, and tables of
FP32 (2^-24). BF16 rows: one more rounding of the output, half of a last place, 2^-8 of
each value. The backward has a
second sum; gamma gradients sum tokens * heads FP32 products, whose error stays below
2^-24 sqrt(rows) of the sum of magnitudes' scale: 2^-16 of sum |dz x r| is allowed.
"""
import pytest

import welvet_b200 as W

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _angles(torch, table, pos):
    return torch.complex(*table.double()[pos.long()].unbind(-1))[:, None]


def _forward(torch, x, gamma, z, hd, eps=EPS):
    x = x.double().reshape(x.shape[0], -1, hd)
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    if z is not None:
        y = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * z
        x = torch.cat([y.real, y.imag], -1)
    return x


def _make(torch, tokens, heads, kv, hd, dtype, packed, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + tokens)
    def rows(h):
        if not packed:
            return torch.randn(tokens, h * hd, device="cuda", generator=g).to(dtype) * 3
        wide = (torch.randn(tokens, h * hd + 13, device="cuda", generator=g) * 3).to(dtype)
        return wide[:, 5:5 + h * hd]
    table = torch.empty(512, hd // 2, 2, device="cuda")
    W.rope_table(512, hd, table)
    pos = torch.randint(0, 512, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    gq, gk = (1 + 0.4 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    return rows(heads), rows(kv) if kv else None, table, pos, gq, gk, rows


SHAPES = [(1, 1, 1, 64), (1, 32, 8, 128), (3, 5, 1, 64), (64, 32, 8, 64), (257, 16, 2, 128), (9, 4, 4, 256),
          (31, 6, 2, 96), (5, 3, 1, 2), (7, 2, 1, 34), (4, 1, 1, 512), (1000, 8, 0, 128), (100, 4, 4, 32)]


@pytest.mark.parametrize("tokens,heads,kv,hd", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("packed", [False, True])
def test_forward(torch_cuda, tokens, heads, kv, hd, dtype, packed):
    torch = torch_cuda
    q, k, table, pos, gq, gk, _ = _make(torch, tokens, heads, kv, hd, getattr(torch, dtype), packed)
    z = _angles(torch, table, pos)
    half = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    for use_norm, use_rope in ((True, True), (True, False), (False, True)):
        qo = torch.empty_like(q)
        ko = torch.empty_like(k) if kv else None
        W.qk_norm_rope(q, k, qo, ko, hd, gq if use_norm else None, gk if use_norm and kv else None, EPS,
                       table if use_rope else None, pos)
        for x, y, gamma in ((q, qo, gq), (k, ko, gk)):
            if x is None:
                continue
            ref = _forward(torch, x, gamma if use_norm else None, z if use_rope else None, hd)
            d = (y.double().reshape(ref.shape) - ref).abs()
            assert bool((d <= half * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True)).all())
    W.device_check()


@pytest.mark.parametrize("tokens,heads,kv,hd", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("packed", [False, True])
def test_backward(torch_cuda, tokens, heads, kv, hd, dtype, packed):
    torch = torch_cuda
    q, k, table, pos, gq, gk, rows = _make(torch, tokens, heads, kv, hd, getattr(torch, dtype), packed, 1)
    z = _angles(torch, table, pos)
    dyq, dyk = rows(heads), rows(kv) if kv else None
    dq, dk = torch.empty_like(q), torch.empty_like(k) if kv else None
    dgq, dgk = (torch.full((hd,), 9.0, device="cuda") for _ in range(2))
    ws = torch.empty(W.qk_norm_rope_workspace(hd), dtype=torch.uint8, device="cuda").fill_(255)
    half = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    call = lambda: W.qk_norm_rope_backward(q, k, dyq, dyk, dq, dk, dgq, dgk if kv else None, hd, ws, gq,  # noqa: E731
                                           gk if kv else None, EPS, table, pos)
    call()
    for x, dy, dx, gamma, dg in ((q, dyq, dq, gq, dgq), (k, dyk, dk, gk, dgk)):
        if x is None:
            continue
        xr = x.double().reshape(tokens, -1, hd).requires_grad_(True)
        gr = gamma.double().requires_grad_(True)
        y = _forward(torch, xr, gr, z, hd)
        up = dy.double().reshape(y.shape)
        y.backward(up)
        d = (dx.double().reshape(y.shape) - xr.grad).abs()
        # u - x r mean(u x r) cancels: the error is relative to r |u|
        r = 1 / torch.sqrt((xr.detach() ** 2).mean(-1, keepdim=True) + EPS)
        size = (up.abs().amax(-1, keepdim=True) * gamma.abs().max() * r).detach()
        assert bool((d <= half * xr.grad.abs() + 2.0 ** -19 * (xr.grad.abs().amax(-1, keepdim=True) + size * hd ** 0.5)).all())
        zc = torch.complex(up[..., :hd // 2], up[..., hd // 2:]) * z.conj()
        mag = (torch.cat([zc.real, zc.imag], -1) * xr.detach() * r).abs().sum((0, 1))
        assert bool(((dg.double() - gr.grad).abs() <= 2.0 ** -16 * mag).all())
    first = [t.clone() for t in (dq, dgq, dgk)]
    call()
    assert all(torch.equal(a, b) for a, b in zip(first, (dq, dgq, dgk)))  # the same bits
    W.device_check()


def test_backward_against_differences(torch_cuda):
    """Central differences of the FP32 forward along random directions."""
    torch = torch_cuda
    tokens, heads, kv, hd = 6, 3, 1, 64
    q, k, table, pos, gq, gk, rows = _make(torch, tokens, heads, kv, hd, torch.float32, False)
    dyq, dyk = rows(heads), rows(kv)

    def loss(q, k, gq, gk):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        W.qk_norm_rope(q, k, qo, ko, hd, gq, gk, EPS, table, pos)
        return float((qo.double() * dyq.double()).sum() + (ko.double() * dyk.double()).sum())
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dgq, dgk = torch.empty_like(gq), torch.empty_like(gk)
    ws = torch.empty(W.qk_norm_rope_workspace(hd), dtype=torch.uint8, device="cuda")
    W.qk_norm_rope_backward(q, k, dyq, dyk, dq, dk, dgq, dgk, hd, ws, gq, gk, EPS, table, pos)
    for i, (x, dx) in enumerate(((q, dq), (k, dk), (gq, dgq), (gk, dgk))):
        way = torch.randn_like(x)
        step = 2.0 ** -7
        a, b = ([t.clone() for t in (q, k, gq, gk)] for _ in range(2))
        a[i] += step * way
        b[i] -= step * way
        slope = (loss(*a) - loss(*b)) / (2 * step)
        want = float((dx.double() * way.double()).sum())
        # third-order term ~ step^2, and the FP32 rounding of two sums over 2 * step
        assert abs(slope - want) <= 2e-3 * float((dx.double() * way.double()).abs().sum())


def test_in_place_positions_and_rows_of_zeros(torch_cuda):
    torch = torch_cuda
    for hd in (64, 128, 20):
        q, k, table, pos, gq, gk, _ = _make(torch, 40, 4, 2, hd, torch.bfloat16, False)
        q[3] = 0
        q[5] = 1e-20
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        index = (torch.arange(40, device="cuda") % 17).to(torch.int32)
        W.qk_norm_rope(q, k, qo, ko, hd, gq, gk, EPS, table, index)
        q2, k2 = q.clone(), k.clone()
        W.qk_norm_rope(q2, k2, q2, k2, hd, gq, gk, EPS, table, None, pos_mod=17)
        assert torch.equal(qo, q2) and torch.equal(ko, k2)
        assert float(qo[3].abs().sum()) == 0 and bool(torch.isfinite(qo.float()).all())
        W.qk_norm_rope(q[:0], k[:0], qo[:0], ko[:0], hd, gq, gk, EPS, table, index)  # no tokens
        W.device_check()


def test_backward_without_tokens_and_without_a_side(torch_cuda):
    torch = torch_cuda
    hd = 128
    q, k, table, pos, gq, gk, rows = _make(torch, 12, 4, 2, hd, torch.bfloat16, False)
    dy = rows(4)
    ws = torch.empty(W.qk_norm_rope_workspace(hd), dtype=torch.uint8, device="cuda")
    dg, dg2 = torch.full((hd,), 9.0, device="cuda"), torch.full((hd,), 9.0, device="cuda")
    W.qk_norm_rope_backward(q[:0], k[:0], dy[:0], k[:0], q[:0], k[:0], dg, dg2, hd, ws, gq, gk, EPS, table, pos)
    assert float(dg.abs().sum()) == 0 and float(dg2.abs().sum()) == 0
    # rotation alone: the gradient is the rotation back, and gamma has none
    dq = torch.empty_like(q)
    W.qk_norm_rope_backward(q, None, dy, None, dq, None, None, None, hd, ws, None, None, EPS, table, pos)
    back = torch.empty_like(q)
    W.qk_norm_rope(dq, None, back, None, hd, rope=table, positions=pos)
    assert float((back.float() - dy.float()).abs().max()) <= 3 * 2.0 ** -8 * float(dy.abs().max())
    W.device_check()


def test_a_position_outside_the_table_is_reported(torch_cuda):
    torch = torch_cuda
    for hd in (64, 20):
        q, k, table, pos, gq, gk, _ = _make(torch, 4, 2, 1, hd, torch.float32, False)
        pos[2] = 512
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        W.qk_norm_rope(q, k, qo, ko, hd, rope=table, positions=pos)
        with pytest.raises(W.WelvetError) as e:
            W.device_check()
        assert e.value.code == 4 and "RoPE" in e.value.message
        assert torch.equal(qo[2], q[2])  # left unrotated
    W.device_check()
