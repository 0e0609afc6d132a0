"""The E4M3 paged KV cache (welvet_b200_kv8_append, welvet_b200_kv8_attention) against
plain 64-bit implementations.

Append: a code is right when no E4M3 value is nearer to the 64-bit x / scale, up to the
FP32 rounding of the rotation (two products and a sum: 3 x 2^-24 of |x|, here 2^-21);
scales are exact.

Attention: the kernels hold queries to 2^-14 or better of the row's largest value,
probabilities to a relative 2^-10 (each by its own rounding) and sums in FP32, and
round the output to BF16 (half of a last place: 2^-8 |o|). The tests allow that, twice
the probabilities' part of sum p |v|, and 2^-13 of it for the scores.
"""
import pytest

import welvet_b200 as W

pytestmark = pytest.mark.gpu
PAGE, BLOCK, FLOOR = 64, 16, 2.0 ** -64


def _e4m3_values(torch):
    return torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).double().cuda()


def _pow2_scale(amax):
    """Smallest power of two s >= FLOOR with amax <= 448 s, by trial."""
    s = FLOOR
    while amax > 448 * s:
        s *= 2
    return s


def _cache(torch, batch, ctx, kv, hd, extra=3, fill=None, seed=0):
    """A cache for up to max(ctx) tokens: shuffled pages, codes and scales of random
    tokens, or `fill` in every code byte and scale 1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = (max(ctx) + PAGE - 1) // PAGE
    pages = batch * per + extra
    if fill is None:
        x = torch.randn(2, pages, kv, 4, BLOCK, hd, device="cuda", generator=g)
        x *= torch.exp(torch.randn(2, pages, kv, 4, 1, 1, device="cuda", generator=g))
        s = torch.tensor([_pow2_scale(float(a)) for a in x.abs().amax((4, 5)).flatten()], device="cuda")
        s = s.view(2, pages, kv, 4)
        c = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(2, pages, kv, PAGE, hd)
    else:
        c = torch.full((2, pages, kv, PAGE, hd), fill, dtype=torch.uint8, device="cuda")
        s = torch.ones(2, pages, kv, 4, device="cuda")
    bt = torch.randperm(pages, device="cuda", generator=g)[:batch * per].to(torch.int32).view(batch, per).contiguous()
    return W.Kv8Cache(c[0].contiguous(), c[1].contiguous(), s[0].contiguous(), s[1].contiguous(), bt,
                      torch.tensor(ctx, dtype=torch.int32, device="cuda"))


def _read(torch, cache, b, n, which):
    """Tokens [0, n) of sequence b in 64 bits: [n, kv, hd]."""
    codes, scales = cache.tensors[which], cache.tensors[2 + which]
    pages = cache.tensors[4][b].long()
    x = codes[pages].view(torch.float8_e4m3fn).double() * scales[pages].double().repeat_interleave(BLOCK, 2)[..., None]
    return x.transpose(1, 2).reshape(-1, *x.shape[1:2], x.shape[3])[:n]


def _rotate(torch, x, cs):
    """Pairs (i, i + hd/2) of x [n, heads, hd] by the (cos, sin) of cs [n, hd/2, 2]."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(*cs.double().unbind(-1))[:, None]
    return torch.cat([z.real, z.imag], -1)


@pytest.mark.parametrize("hd,theta", [(64, 10000.0), (128, 500000.0), (34, 10000.0), (2, 10.0)])
def test_rope_table(torch_cuda, hd, theta):
    """(cos, sin) of pos / theta^e with the layer's FP32 exponent e = 2i/hd, rounded once."""
    torch = torch_cuda
    table = torch.empty(700, hd // 2, 2, device="cuda")
    W.rope_table(700, hd, table, theta)
    e = (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd).double()
    ang = torch.arange(700, device="cuda", dtype=torch.float64)[:, None] / theta ** e
    want = torch.stack([ang.cos(), ang.sin()], -1)
    assert float((table.double() - want).abs().max()) <= 2.0 ** -24  # half a last place below 1 is 2^-25


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("batch,seq,ctx,lens,kv,hd,rope", [
    (1, 1, [1], None, 1, 64, True),                    # the first token of a sequence
    (3, 1, [16, 17, 64], None, 2, 128, True),          # the last of a block, the first, the end of a page
    (2, 5, [5, 133], None, 3, 64, False),
    (4, 77, [77, 100, 141, 300], [77, 0, 13, 40], 2, 128, True),  # unequal, one without new tokens
    (2, 300, [300, 811], [300, 299], 1, 64, True),
    (2, 33, [40, 33], None, 2, 96, True),              # other head sizes
    (1, 18, [30], None, 2, 34, True),
    (1, 40, [129], None, 1, 256, False),
])
@pytest.mark.parametrize("packed", [False, True])
def test_append(torch_cuda, batch, seq, ctx, lens, kv, hd, rope, packed):
    torch = torch_cuda
    cache = _cache(torch, batch, ctx, kv, hd, seed=hd + seq)
    before = [t.clone() for t in cache.tensors[:4]]
    g = torch.Generator(device="cuda").manual_seed(7)
    if packed:  # views of wider rows at an odd offset: no 16-byte alignment
        wide = torch.randn(batch * seq, 2 * kv * hd + 5, device="cuda", generator=g).bfloat16()
        k, v = wide[:, 3:3 + kv * hd], wide[:, 3 + kv * hd:3 + 2 * kv * hd]
    else:
        k = torch.randn(batch * seq, kv * hd, device="cuda", generator=g).bfloat16() * 5
        v = torch.randn(batch * seq, kv * hd, device="cuda", generator=g).bfloat16()
    table = None
    if rope:
        table = torch.empty(max(ctx), hd // 2, 2, device="cuda")
        W.rope_table(max(ctx), hd, table)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    W.kv8_append(cache, seq, k, v, rope=table, seq_lens=sl)
    W.device_check()
    values = _e4m3_values(torch)
    finite = values[torch.isfinite(values)]
    touched = torch.zeros_like(before[0], dtype=torch.bool)
    for which, x in ((0, k), (1, v)):
        codes, scales = cache.tensors[which], cache.tensors[2 + which]
        want_s = before[2 + which].clone()
        for b in range(batch):
            n = lens[b] if lens else seq
            rows = x[b * seq:b * seq + n].double().view(n, kv, hd)
            start = ctx[b] - n
            if rope and which == 0 and n:
                rows = _rotate(torch, rows, table[start:ctx[b]])
            for p0 in range(start // BLOCK * BLOCK, ctx[b], BLOCK):
                lo, hi = max(start, p0), min(ctx[b], p0 + BLOCK)
                if lo >= hi:
                    continue
                page, sub = int(cache.tensors[4][b, p0 // PAGE]), p0 % PAGE // BLOCK
                at = slice(sub * BLOCK, sub * BLOCK + hi - p0)
                for h in range(kv):
                    want = rows[lo - start:hi - start, h]
                    s = _pow2_scale(float(want.abs().max()) * (1 - 2 ** -20))
                    s2 = _pow2_scale(float(want.abs().max()) * (1 + 2 ** -20))
                    if lo > p0:
                        old_s = float(before[2 + which][page, h, sub])
                        s, s2 = max(s, old_s), max(s2, old_s)
                        held = before[which][page, h, sub * BLOCK:sub * BLOCK + lo - p0].view(torch.float8_e4m3fn)
                        want = torch.cat([held.double() * old_s, want])
                    got_s = float(scales[page, h, sub])
                    assert got_s in (s, s2)
                    want_s[page, h, sub] = got_s
                    y = want / got_s
                    got = values[codes[page, h, at].long()]
                    best = (finite[:, None, None] - y).abs().amin(0)
                    assert bool(((got - y).abs() <= best + 2.0 ** -21 * y.abs()).all())
                    touched[page, h, at] = True
        assert torch.equal(scales, want_s)
        assert torch.equal(codes[~touched], before[which][~touched])  # nothing else is written


def test_append_token_by_token_holds_the_same_values(torch_cuda):
    """Scales are powers of two: codes that stay normal keep their value when a later
    token raises the scale, so one call and many give the same cache."""
    torch = torch_cuda
    n, kv, hd = 37, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    grow = torch.linspace(-1, 1, n, device="cuda").mul(3).exp()[:, None]  # later tokens are larger
    k = ((torch.rand(n, kv * hd, device="cuda", generator=g) + 0.5) * grow).bfloat16()
    v = -k
    once, steps = (_cache(torch, 1, [n], kv, hd, fill=0x7f, seed=1) for _ in range(2))
    W.kv8_append(once, n, k, v)
    for t in range(n):
        steps.tensors[5].fill_(t + 1)
        W.kv8_append(steps, 1, k[t:t + 1], v[t:t + 1])
    W.device_check()
    for which in (0, 1):
        assert torch.equal(once.tensors[2 + which], steps.tensors[2 + which]) or n % BLOCK
        assert torch.equal(_read(torch, once, 0, n, which), _read(torch, steps, 0, n, which))


def test_append_twice_is_the_same(torch_cuda):
    torch = torch_cuda
    ctx = [50, 90]
    cache = _cache(torch, 2, ctx, 2, 128)
    k = torch.randn(2 * 21, 256, device="cuda").bfloat16()
    W.kv8_append(cache, 21, k, k)
    first = [t.clone() for t in cache.tensors[:4]]
    W.kv8_append(cache, 21, k, k)
    assert all(torch.equal(a, b) for a, b in zip(first, cache.tensors[:4]))


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_values_that_are_not_finite(torch_cuda, hd, bad):
    """Their block reads as NaN, its codes stay finite, others are untouched; the next
    sequence in the page begins it anew."""
    torch = torch_cuda
    cache = _cache(torch, 1, [64], 2, hd, fill=0)
    k = torch.ones(40, 2 * hd, device="cuda").bfloat16()
    v = k.clone()
    k[20, hd + 3] = bad  # block 1 of KV head 1
    cache.tensors[5].fill_(40)
    W.kv8_append(cache, 40, k, v)
    page = int(cache.tensors[4][0, 0])
    ks = cache.tensors[2][page]
    assert bool(torch.isnan(ks[1, 1])) and int(torch.isnan(cache.tensors[2]).sum()) == 1
    assert not bool(torch.isnan(cache.tensors[3]).any())
    assert not bool(torch.isnan(cache.tensors[0].view(torch.float8_e4m3fn).float()).any())
    cache.tensors[5].fill_(41)  # block 2 gains a token, block 1 does not
    W.kv8_append(cache, 1, v[:1], v[:1])
    assert bool(torch.isnan(ks[1, 1])) and float(ks[1, 2]) == _pow2_scale(1.0)
    cache.tensors[5].fill_(32)
    W.kv8_append(cache, 32, v[:32], v[:32])
    assert not bool(torch.isnan(cache.tensors[2]).any())
    W.device_check()


def test_append_zeros_and_extremes(torch_cuda):
    torch = torch_cuda
    for hd in (64, 128, 32):
        cache = _cache(torch, 1, [64], 1, hd, fill=0)
        k = torch.zeros(64, hd, device="cuda").bfloat16()
        k[16:32] = 3e38   # near the largest BF16
        k[32:48] = 1e-30  # below the smallest scale's range
        W.kv8_append(cache, 64, k, k)
        page = int(cache.tensors[4][0, 0])
        assert cache.tensors[2][page, 0].tolist() == [FLOOR, _pow2_scale(float(k[16, 0])), FLOOR, FLOOR]
        got = _read(torch, cache, 0, 64, 0)[:, 0, 0]
        assert float(got[0]) == 0 and float(got[32]) == 0 and abs(float(got[16]) / float(k[16, 0]) - 1) < 2 ** -4


# ---------------------------------------------------------------- attention
def _reference(torch, cache, cfg, seq, q, lens=None):
    """(o, sum p |v|) in 64 bits, [batch * seq, heads, hd], and the rows that see keys."""
    heads, kv, hd = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
    ctx = cache.tensors[5].tolist()
    o = torch.zeros(len(ctx) * seq, heads, hd, dtype=torch.float64, device="cuda")
    a = o.clone()
    scale = cfg.scale_override or hd ** -0.5
    for b, n in enumerate(ctx):
        new = seq if lens is None else max(0, min(lens[b], seq))
        k, v = (_read(torch, cache, b, n, w) for w in (0, 1))
        for t in range(new):
            p = n - new + t
            if p < 0:
                continue
            lo = max(0, p + 1 - cfg.window) if cfg.mask == 3 else 0
            kk = k[lo:p + 1].repeat_interleave(heads // kv, 1)
            vv = v[lo:p + 1].repeat_interleave(heads // kv, 1)
            qq = q[b * seq + t].double().view(heads, hd)
            x = torch.einsum("hd,nhd->hn", qq, kk) * scale
            if cfg.pos in (2, 3):
                slope = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float64) / heads)
                x = x - slope[:, None] * (p - torch.arange(lo, p + 1, device="cuda"))
            pr = torch.softmax(x, -1)
            o[b * seq + t] = torch.einsum("hn,nhd->hd", pr, vv)
            a[b * seq + t] = torch.einsum("hn,nhd->hd", pr, vv.abs())
    return o, a


def _close(got, o, a):
    d = (got.double().view(o.shape) - o).abs()
    return bool((d <= 2.0 ** -8 * o.abs() + (2.0 ** -9 + 2.0 ** -13) * a).all())


def _config(heads, kv, hd, **kw):
    return W.MhaConfig.make(heads * hd, heads, kv, head_dim=hd, precision=1, **kw)


SHAPES = [
    # batch, seq, ctx, heads, kv, hd
    (1, 1, [1], 1, 1, 64),
    (1, 1, [1], 8, 1, 128),
    (3, 1, [16, 17, 129], 8, 2, 64),
    (2, 1, [63, 65], 4, 4, 128),
    (5, 1, [1, 700, 64, 1000, 128], 32, 8, 128),
    (2, 1, [2500, 1], 32, 8, 64),
    (1, 1, [9001], 16, 2, 128),       # split over the context
    (2, 3, [3, 300], 6, 2, 64),       # groups of three heads
    (2, 5, [700, 133], 32, 8, 128),
    (1, 17, [200], 16, 2, 64),
    (2, 64, [64, 400], 8, 2, 128),
    (1, 150, [611], 12, 4, 64),
    (1, 333, [333], 10, 2, 128),      # a whole prompt
    (2, 2, [140, 9], 4, 2, 96),       # head sizes of the general kernel
    (1, 3, [90], 3, 1, 256),
    (1, 1, [77], 2, 1, 34),
]


@pytest.mark.parametrize("batch,seq,ctx,heads,kv,hd", SHAPES)
@pytest.mark.parametrize("kind", ["causal", "window", "alibi"])
def test_attention(torch_cuda, batch, seq, ctx, heads, kv, hd, kind):
    torch = torch_cuda
    cache = _cache(torch, batch, ctx, kv, hd, seed=sum(ctx) + heads)
    extra = {"causal": {}, "window": dict(mask=3, window=37), "alibi": dict(pos=2)}[kind]
    cfg = _config(heads, kv, hd, **extra)
    g = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn(batch * seq, heads * hd, device="cuda", generator=g) * 2).bfloat16()
    out = torch.full_like(q, 7.0)
    W.kv8_attention(cfg, cache, seq, q, out, max(ctx))
    W.device_check()
    assert _close(out, *_reference(torch, cache, cfg, seq, q))


@pytest.mark.parametrize("hd,kv,seq", [(64, 8, 1), (64, 8, 5), (64, 4, 16), (128, 8, 1), (128, 8, 3), (128, 4, 12)])
def test_attention_full_gpu(torch_cuda, hd, kv, seq):
    """More sequences than fit the GPU at once, lengths that end anywhere in a tile, NaN
    codes behind their ends, five times over. Keys of zeros make every probability the
    same power of two and small integers make every sum exact, so a row is the mean of
    its values up to the quotient's and the output's rounding."""
    torch = torch_cuda
    batch, heads, most = 96, 4 * kv, 3700
    ctx = [most - (b * 389) % 700 for b in range(batch)]
    cache = _cache(torch, batch, ctx, kv, hd, seed=1)
    keys, values, ks, vs, table, lens = cache.tensors
    table, lens = table.long(), lens.long()
    for x in (ks, vs):
        x.fill_(1.0)
    at = torch.arange(table.shape[1] * PAGE, device="cuda")
    val = 1 + (at[:, None] // 48 + torch.arange(hd, device="cuda")) % 7      # [token][hd]
    code = val.float().to(torch.float8_e4m3fn).view(torch.uint8)
    for b in range(batch):
        past = (at >= ctx[b])[:, None]
        for c, x in ((keys, torch.zeros_like(code)), (values, code)):
            x = torch.where(past, 0x7f, x).view(-1, 1, PAGE, hd)
            used = (ctx[b] + PAGE - 1) // PAGE
            c[table[b, :used]] = x[:used].expand(-1, kv, -1, -1)
    pos = lens[:, None] - seq + torch.arange(seq, device="cuda")              # [batch][seq]
    sums = torch.cumsum(val.double(), 0)
    o = (sums[pos] / (pos + 1)[..., None]).view(batch * seq, 1, hd)
    q = torch.randn(batch * seq, heads * hd, device="cuda").bfloat16()
    out = torch.empty_like(q)
    for _ in range(5):
        out.fill_(7)
        W.kv8_attention(_config(heads, kv, hd), cache, seq, q, out, most)
        W.device_check()
        d = (out.double().view(batch * seq, heads, hd) - o).abs()
        assert bool((d <= (2.0 ** -8 + 2.0 ** -20) * o).all())


@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("seq", [1, 4, 70])
def test_attention_unequal_lengths_and_empty_rows(torch_cuda, hd, seq):
    """Sequences without tokens, without new tokens, with fewer than seq: their missing
    rows are zero. What lies past a sequence's end in its page is NaN codes."""
    torch = torch_cuda
    ctx, lens = [0, 5, 130, 1, 300], [0, 0, min(seq, 3), 1, seq]
    cache = _cache(torch, 5, [max(ctx)] * 5, 2, hd, seed=2)
    cache.tensors[5].copy_(torch.tensor(ctx, dtype=torch.int32))
    for b, n in enumerate(ctx):
        per = cache.tensors[4].shape[1]
        for j in range(n // PAGE, per):
            page = int(cache.tensors[4][b, j])
            first = max(0, n - j * PAGE)
            for w in (0, 1):
                cache.tensors[w][page, :, first:] = 0x7f
                cache.tensors[2 + w][page, :, (first + BLOCK - 1) // BLOCK:] = float("nan")
    cfg = _config(8, 2, hd)
    q = torch.randn(5 * seq, 8 * hd, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    W.kv8_attention(cfg, cache, seq, q, out, max(ctx), seq_lens=sl)
    W.device_check()
    o, a = _reference(torch, cache, cfg, seq, q, lens)
    assert _close(out, o, a)
    for b in range(5):
        assert float(out[b * seq + lens[b]:(b + 1) * seq].abs().sum()) == 0


@pytest.mark.parametrize("hd", [64, 128, 48])
def test_attention_poisoned_block_reaches_only_rows_that_see_it(torch_cuda, hd):
    torch = torch_cuda
    for which in (0, 1):
        cache = _cache(torch, 1, [200], 2, hd, seed=9)
        page = int(cache.tensors[4][0, 2])
        cache.tensors[2 + which][page, 1, 1] = float("nan")  # tokens 144..159 of KV head 1
        cfg = _config(4, 2, hd, mask=3, window=20)
        q = torch.randn(100, 4 * hd, device="cuda").bfloat16()
        out = torch.empty_like(q)
        W.kv8_attention(cfg, cache, 100, q, out, 200)  # rows at positions 100..199
        nan = torch.isnan(out.float()).view(100, 4, hd)
        sees = torch.tensor([p >= 144 and p - 20 < 159 for p in range(100, 200)], device="cuda")
        assert not bool(nan[:, :2].any())
        assert bool(nan[sees][:, 2:].all()) and not bool(nan[~sees][:, 2:].any())


@pytest.mark.parametrize("hd", [64, 128, 48])
def test_attention_ranges(torch_cuda, hd):
    """Blocks whose scales differ by 2^40, scores in the thousands, a query of zeros, a
    query that is not finite."""
    torch = torch_cuda
    cache = _cache(torch, 1, [500], 1, hd, seed=4)
    pages = cache.tensors[4][0].long()
    cache.tensors[3][pages[0]] *= 2.0 ** 20
    cache.tensors[3][pages[3]] *= 2.0 ** -20
    cache.tensors[2][pages[5]] *= 2.0 ** 6
    cfg = _config(6, 1, hd)
    q = torch.randn(2, 6 * hd, device="cuda").bfloat16()
    q[0, :hd] = 0
    q[1, hd:2 * hd] *= 300
    out = torch.empty_like(q)
    W.kv8_attention(cfg, cache, 2, q, out, 500)
    W.device_check()
    assert _close(out, *_reference(torch, cache, cfg, 2, q))
    q[0, 2 * hd + 1] = float("nan")
    W.kv8_attention(cfg, cache, 2, q, out, 500)
    nan = torch.isnan(out.float()).view(2, 6, hd)
    assert bool(nan[0, 2].all()) and int(nan.sum()) == hd


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_one_far_key(torch_cuda, hd):
    """One key holds almost all of the weight and thousands share the rest: the small
    probabilities add up."""
    torch = torch_cuda
    n = 20000
    cache = _cache(torch, 1, [n], 1, hd, fill=0x38)  # every code is 1.0
    q = torch.zeros(1, hd, device="cuda").bfloat16()
    q[0, 0] = 1.0
    pages = cache.tensors[4][0].long()
    cache.tensors[0][pages[0], 0, 5, 0] = 0x60  # 32: 31 above the others before the scale
    cache.tensors[1][pages[0], 0, 5] = 0        # ... and its value is 0
    for gap in (6.0, 11.0, 16.0):
        cfg = _config(1, 1, hd, scale_override=gap / 31)
        out = torch.empty_like(q)
        W.kv8_attention(cfg, cache, 1, q, out, n)
        o, a = _reference(torch, cache, cfg, 1, q)
        assert _close(out, o, a)


def test_attention_strides_streams_and_repeatability(torch_cuda):
    """Query and output rows inside wider rows, a stream of its own, the same bits twice;
    what lies between the rows is left alone."""
    torch = torch_cuda
    heads, kv, hd, seq = 8, 2, 128, 3
    ctx = [700, 90]
    cache = _cache(torch, 2, ctx, kv, hd, seed=8)
    cfg = _config(heads, kv, hd)
    for off in (0, 8, 3):  # 16-byte aligned rows, and rows that are not
        wide = torch.randn(2 * seq, heads * hd + 24, device="cuda").bfloat16()
        outw = torch.full_like(wide, 5.0)
        q, out = wide[:, off:off + heads * hd], outw[:, off:off + heads * hd]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        W.kv8_attention(cfg, cache, seq, q, out, max(ctx), stream=st)
        st.synchronize()
        first = outw.clone()
        assert _close(out, *_reference(torch, cache, cfg, seq, q.contiguous()))
        assert bool((outw[:, :off] == 5).all()) and bool((outw[:, off + heads * hd:] == 5).all())
        W.kv8_attention(cfg, cache, seq, q, out, max(ctx))
        torch.cuda.synchronize()
        assert torch.equal(first, outw)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,kv", [(1, 2), (160, 2), (7, 3)])
@pytest.mark.parametrize("seq", [1, 9, 40])
def test_attention_alignment_changes_nothing(torch_cuda, hd, batch, kv, seq):
    """Rows at any 2-byte address give the bits of aligned ones, with a split context
    and with more sequences than fit at once."""
    torch = torch_cuda
    heads = 2 * kv
    ctx = [40 + (b * 97) % 461 for b in range(batch)]
    cache = _cache(torch, batch, ctx, kv, hd, seed=9)
    cfg = _config(heads, kv, hd)
    q = torch.randn(batch * seq, heads * hd, device="cuda").bfloat16()
    out = torch.empty_like(q)
    W.kv8_attention(cfg, cache, seq, q, out, max(ctx))
    for off, extra in ((1, 3), (2, 2), (4, 8)):
        wide = torch.zeros(batch * seq, heads * hd + off + extra, device="cuda", dtype=torch.bfloat16)
        outw = torch.full_like(wide, 5.0)
        wide[:, off:off + heads * hd] = q
        W.kv8_attention(cfg, cache, seq, wide[:, off:off + heads * hd], outw[:, off:off + heads * hd], max(ctx))
        W.device_check()
        assert torch.equal(outw[:, off:off + heads * hd], out)
        assert bool((outw[:, :off] == 5).all()) and bool((outw[:, off + heads * hd:] == 5).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv", [1, 3, 5, 6])
@pytest.mark.parametrize("rope", [False, True])
def test_append_alignment_changes_nothing(torch_cuda, hd, kv, rope):
    """Rows that are not aligned take another kernel and give the same codes and scales,
    for any number of heads, whether a block is begun, continued or left partial."""
    torch = torch_cuda
    batch, seq = 3, 70
    ctx, lens = [70, 203, 131], [70, 9, 33]
    table = torch.empty(max(ctx), hd // 2, 2, device="cuda")
    W.rope_table(max(ctx), hd, table)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = (torch.randn(2, batch * seq, kv * hd + 1, device="cuda") * 3).bfloat16()
    got = []
    for k, v in ((wide[0, :, 1:], wide[1, :, 1:]), (wide[0, :, 1:].contiguous(), wide[1, :, 1:].contiguous())):
        cache = _cache(torch, batch, ctx, kv, hd, seed=4)
        W.kv8_append(cache, seq, k, v, rope=table if rope else None, seq_lens=sl)
        W.device_check()
        got.append(cache.tensors[:4])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_attention_head_shard(torch_cuda):
    """A shard of the heads over its own KV heads equals those heads of the whole,
    ALiBi slopes included."""
    torch = torch_cuda
    heads, kv, hd = 8, 4, 64
    cache = _cache(torch, 2, [300, 77], kv, hd, seed=6)
    q = torch.randn(2, heads * hd, device="cuda").bfloat16()
    whole = torch.empty_like(q)
    W.kv8_attention(_config(heads, kv, hd, pos=2), cache, 1, q, whole, 300)
    k, v, ks, vs, bt, ctx = cache.tensors
    part = W.Kv8Cache(k[:, 2:].contiguous(), v[:, 2:].contiguous(), ks[:, 2:].contiguous(), vs[:, 2:].contiguous(), bt, ctx)
    qs = q[:, 4 * hd:].contiguous()
    out = torch.empty_like(qs)
    W.kv8_attention(_config(heads, kv, hd, pos=2, head_begin=4, head_count=4), part, 1, qs, out, 300)
    assert torch.equal(out, whole[:, 4 * hd:])


def test_faults_of_the_data_are_reported(torch_cuda):
    """A page outside the pool, a table that ends before the context, a position past the
    RoPE table: code 4 from the device check, nothing out of range is touched."""
    torch = torch_cuda
    for hd in (64, 128, 48):
        cfg = _config(2, 1, hd)
        k = torch.ones(1, hd, device="cuda").bfloat16()
        q = torch.ones(1, 2 * hd, device="cuda").bfloat16()
        out = torch.empty_like(q)
        for page, ctx in ((1 << 20, 10), (-1, 10), (0, 65)):
            cache = _cache(torch, 1, [64], 1, hd)
            cache.tensors[4].fill_(page)
            cache.tensors[5].fill_(ctx)
            before = [t.clone() for t in cache.tensors[:4]]
            W.kv8_append(cache, 1, k, k)
            with pytest.raises(W.WelvetError) as e:
                W.device_check()
            assert e.value.code == 4 and "block table" in e.value.message
            assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors[:4]))
            W.kv8_attention(cfg, cache, 1, q, out, 128)
            with pytest.raises(W.WelvetError) as e:
                W.device_check()
            assert e.value.code == 4 and "block table" in e.value.message
        cache = _cache(torch, 1, [64], 1, hd)
        table = torch.empty(32, hd // 2, 2, device="cuda")
        W.rope_table(32, hd, table)
        W.kv8_append(cache, 1, k, k, rope=table)  # position 63
        with pytest.raises(W.WelvetError) as e:
            W.device_check()
        assert e.value.code == 4 and "RoPE" in e.value.message
    W.device_check()
