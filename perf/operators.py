"""The serving and training operators around the 8-bit paged KV cache: what they
compute in plain torch, the cases they are measured on, and their 64-bit values.

  norm    per-head RMS norm of queries and keys with the position rotation in the
          same pass, forward and backward
  append  new keys and values into a paged cache of E4M3 codes with one power-of-two
          scale for each 16 tokens of a KV head, keys rotated on the way
  attend  attention of new tokens over that cache

A cache holds pages of 64 tokens, codes [page, kv_head, 64, head_dim] and scales
[page, kv_head, 4]; block_table [batch, max_pages] names each sequence's pages and
ctx_len [batch] counts its tokens, the new ones included. The last page of a pool
belongs to no sequence.
"""
import math
import os
import sys

import torch

own = False

PAGE, BLOCK = 64, 16
FLOOR = 2.0 ** -64  # smallest scale of a block
EPS = 1e-6


def _framework():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "welvet.metal_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import welvet_b200
    return welvet_b200


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 64 sequences, 32 query heads over 8 KV heads of 64
        dict(name="norm step", op="norm", grad=False, bf16=True, tokens=64, heads=32, kv=8, hd=64),
        # the prompts of a small batch: 4 x 4096 tokens, 32 heads of 128
        dict(name="norm prompt", op="norm", grad=False, bf16=True, tokens=16384, heads=32, kv=32, hd=128),
        # a training micro-batch of grouped-query heads
        dict(name="norm train", op="norm", grad=True, bf16=True, tokens=16384, heads=32, kv=8, hd=128),
        # an FP32 training batch cut at an odd place, 16 heads of 64
        dict(name="norm train f32", op="norm", grad=True, bf16=False, tokens=4099, heads=16, kv=16, hd=64),
        # one token for each of 64 sequences in the middle of their blocks
        dict(name="append step", op="append", batch=64, seq=1, ctx=4096, spread=777, kv=8, hd=64, cut=0),
        # whole prompts, the sequences of unequal length
        dict(name="append prompt", op="append", batch=4, seq=4096, ctx=4096, spread=0, kv=32, hd=128, cut=611),
        # a chunk of a few dozen tokens that begins and ends inside blocks
        dict(name="append chunk", op="append", batch=3, seq=77, ctx=1001, spread=313, kv=8, hd=128, cut=9),
        # a single sequence answering its first tokens: latency alone
        dict(name="attend one", op="attend", batch=1, seq=1, ctx=517, spread=0, heads=32, kv=8, hd=128, window=0),
        # 64 sequences of 4096 tokens, 32 heads over 8 KV heads of 64
        dict(name="attend step gqa", op="attend", batch=64, seq=1, ctx=4096, spread=777, heads=32, kv=8, hd=64, window=0),
        # 32 sequences of 8192 tokens, 32 heads of 128 with KV heads of their own
        dict(name="attend step", op="attend", batch=32, seq=1, ctx=8192, spread=0, heads=32, kv=32, hd=128, window=0),
        # five proposed tokens verified for each sequence, a sliding window over a long cache
        dict(name="attend verify", op="attend", batch=8, seq=5, ctx=20011, spread=9001, heads=32, kv=8, hd=128, window=8192),
        # a later piece of a prompt read against the tokens cached before it
        dict(name="attend chunk", op="attend", batch=1, seq=2048, ctx=10001, spread=0, heads=32, kv=8, hd=128, window=0),
    ]


def _size(rng, lo, hi):
    """A whole number from [lo, hi], spread over its logarithm, every other one odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n | 1 if rng.random() < 0.5 else n))
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["norm", "append", "attend", "attend"])
    heads, kv = rng.choice([(32, 32), (32, 8), (16, 16), (16, 2), (64, 8), (8, 1)])
    if op == "norm":
        return dict(op="norm", grad=rng.random() < 0.5, bf16=rng.random() < 0.6, tokens=_size(rng, 1, 8192), heads=heads, kv=kv,
                    hd=rng.choice([64, 128, 256]) if heads < 64 else 64)
    hd = rng.choice([64, 128])
    if op == "append":
        seq = _size(rng, 1, 4096)
        batch = _size(rng, 1, max(1, min(64, 16384 // seq)))
        ctx = seq + _size(rng, 1, 4096)
        return dict(op="append", batch=batch, seq=seq, ctx=ctx, spread=rng.randrange(0, ctx - seq + 1), kv=kv, hd=hd, cut=rng.randrange(0, max(1, seq // 2)))
    if rng.random() < 0.6:  # single tokens, and few
        seq = rng.choice([1, 1, 1, 2, 3, 5, 8])
        batch = _size(rng, 1, 64)
    else:
        seq = _size(rng, 16, 1024)
        batch = _size(rng, 1, 2)
    most = min(32768, (32 * 8192 * 32 * 128) // (batch * kv * hd))  # cached values of the largest listed case
    most = min(most, (32 * 2048 * 10001) // (batch * heads * seq))  # and its scores
    ctx = seq + _size(rng, 1, max(2, most - seq))
    window = _size(rng, 16, 8192) if rng.random() < 0.25 else 0
    return dict(op="attend", batch=batch, seq=seq, ctx=ctx, spread=rng.randrange(0, ctx - seq + 1), heads=heads, kv=kv, hd=hd, window=window)


def _ctx(case):
    """Tokens of each sequence, the new ones included: between ctx - spread and ctx."""
    return [case["ctx"] - (b * 7919) % (case["spread"] + 1) for b in range(case["batch"])]


def _new(case):
    """New tokens of each sequence: seq, or up to `cut` fewer."""
    return [max(1, case["seq"] - (b * 97) % (case.get("cut", 0) + 1)) for b in range(case["batch"])]


def _seen(case):
    """(query, key) pairs, and keys that some query sees, of each sequence."""
    got = []
    for n in _ctx(case):
        w = case["window"] or n
        first = n - case["seq"]
        got.append((sum(min(p + 1, w) for p in range(first, n)), n - max(0, first + 1 - w)))
    return got


def work(case):
    if case["op"] == "norm":
        size = 2 if case["bf16"] else 4
        values = case["tokens"] * (case["heads"] + case["kv"]) * case["hd"]
        table = case["tokens"] * case["hd"] * 4
        if case["grad"]:  # reads x and dy, writes dx
            return {"bytes": 3 * values * size + table, "flops": 16 * values}
        return {"bytes": 2 * values * size + table, "flops": 8 * values}
    row = case["kv"] * case["hd"]
    if case["op"] == "append":
        rows = sum(_new(case))
        return {"bytes": rows * row * (2 * 2 + 2 * 1) + 2 * rows / BLOCK * case["kv"] * 4 + rows * case["hd"] * 4, "flops": 8 * rows * row}
    pairs = sum(p for p, _ in _seen(case))
    keys = sum(k for _, k in _seen(case))
    io = 2 * 2 * case["batch"] * case["seq"] * case["heads"] * case["hd"]
    return {"bytes": 2 * keys * row + 2 * keys / BLOCK * case["kv"] * 4 + io, "flops": 4 * case["hd"] * case["heads"] * pairs}


# ----------------------------------------------------------------- their inputs
def _table(positions, hd):
    """(cos, sin) of position / 10000^(2 i / hd), [positions, hd / 2, 2]."""
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] / torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), 2 * i / hd)
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _scale(amax):
    """The smallest power of two s, not below FLOOR, with amax / s <= 448."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1), and 448 = 7/8 2^9
    return torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8)).clamp_min(FLOOR)


def _pool(pages, case, g):
    """Codes and scales of a pool whose every token is there."""
    x = torch.randn(pages, case["kv"], PAGE // BLOCK, BLOCK, case["hd"], device="cuda", generator=g, dtype=torch.bfloat16)
    x *= torch.rand(1, case["kv"], 1, 1, case["hd"], device="cuda", generator=g).mul_(1.5).add_(0.25).bfloat16()  # channels differ
    s = _scale(x.abs().amax((3, 4)).float())
    x /= s[..., None, None].bfloat16()
    return x.to(torch.float8_e4m3fn).view(torch.uint8).view(pages, case["kv"], PAGE, case["hd"]), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    hd = case["hd"]
    rand = lambda rows, heads: torch.randn(rows, heads * hd, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "norm":
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        n = case["tokens"]
        s = dict(case=case, table=_table(max(4096, min(n, 8192)), hd), q=(rand(n, case["heads"]) * 3).to(kind), k=(rand(n, case["kv"]) * 2).to(kind),
                 q_gamma=1 + 0.3 * rand(1, 1)[0], k_gamma=1 + 0.3 * rand(1, 1)[0],
                 pos=torch.randint(0, 4096, (n,), device="cuda", generator=g, dtype=torch.int32))
        outs = ("q_out", "k_out")
        if case["grad"]:
            s.update(dyq=rand(n, case["heads"]).to(kind), dyk=rand(n, case["kv"]).to(kind))
            s.update(dg_q=torch.empty(hd, device="cuda"), dg_k=torch.empty(hd, device="cuda"))
            outs = ("dq", "dk")
        s.update({outs[0]: torch.empty_like(s["q"]), outs[1]: torch.empty_like(s["k"])})
        if own:  # the scratch that a program keeps
            s["ws"] = torch.empty(_framework().qk_norm_rope_workspace(hd), device="cuda", dtype=torch.uint8)
        return s
    batch, seq = case["batch"], case["seq"]
    per = (case["ctx"] + PAGE - 1) // PAGE
    pages = batch * per + 1
    kc, ks = _pool(pages, case, g)
    vc, vs = _pool(pages, case, g)
    bt = torch.randperm(pages - 1, device="cuda", generator=g).to(torch.int32).view(batch, per)
    ctx = torch.tensor(_ctx(case), device="cuda", dtype=torch.int32)
    s = dict(case=case, kc=kc, vc=vc, ks=ks, vs=vs, bt=bt, ctx=ctx)
    if case["op"] == "append":
        s.update(k=rand(batch * seq, case["kv"]).bfloat16(), v=rand(batch * seq, case["kv"]).bfloat16(), table=_table(case["ctx"], hd),
                 new=torch.tensor(_new(case), device="cuda", dtype=torch.int32))
    else:
        s.update(q=(2 * rand(batch * seq, case["heads"])).bfloat16(), out=torch.empty(batch * seq, case["heads"] * hd, device="cuda", dtype=torch.bfloat16))
    if own:  # the views that a program keeps of its cache and its configuration
        W = _framework()
        s["cache"] = W.Kv8Cache(kc, vc, ks, vs, bt, ctx)
        if case["op"] == "attend":
            s["cfg"] = W.MhaConfig.make(case["heads"] * hd, case["heads"], case["kv"], head_dim=hd, precision=1, mask=3 if case["window"] else 1, window=case["window"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _heads(x, hd):
    return x.float().view(x.shape[0], -1, hd)


def _turn(x, cs, back=False):
    """Rotates the pairs (i, i + hd / 2) of x [rows, heads, hd] by the angles of cs [rows, hd / 2, 2]."""
    a, b = x.chunk(2, -1)
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c + b * n, b * c - a * n] if back else [a * c - b * n, a * n + b * c], -1)


def _norm_plain(s):
    hd, got = s["case"]["hd"], []
    cs = s["table"][s["pos"].long()]
    if not s["case"]["grad"]:
        def forward(x, gamma):
            h = _heads(x, hd)
            h = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma
            return _turn(h, cs).to(x.dtype).view_as(x)
        return [forward(s["q"], s["q_gamma"]), forward(s["k"], s["k_gamma"])]

    def backward(x, dy, gamma):
        h = _heads(x, hd)
        r = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
        h, dz = h * r, _turn(_heads(dy, hd), cs, back=True)
        got.append((dz * h).sum((0, 1)))
        dz = dz * gamma
        return (r * (dz - h * (dz * h).mean(-1, keepdim=True))).to(x.dtype).view_as(x)
    return [backward(s["q"], s["dyq"], s["q_gamma"]), backward(s["k"], s["dyk"], s["k_gamma"])] + got


def _norm_own(s):
    W = _framework()
    if not s["case"]["grad"]:
        W.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], s["case"]["hd"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS, rope=s["table"], positions=s["pos"])
        return [s["q_out"], s["k_out"]]
    W.qk_norm_rope_backward(s["q"], s["k"], s["dyq"], s["dyk"], s["dq"], s["dk"], s["dg_q"], s["dg_k"], s["case"]["hd"], s["ws"],
                            q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS, rope=s["table"], positions=s["pos"])
    return [s["dq"], s["dk"], s["dg_q"], s["dg_k"]]


def _append_plain(s):
    case = s["case"]
    batch, seq, kv, hd = case["batch"], case["seq"], case["kv"], case["hd"]
    start = (s["ctx"] - s["new"]).long()
    # the blocks that the new tokens of a sequence touch, and each of their places
    blocks = (seq + BLOCK - 2) // BLOCK + 1
    blk = start[:, None] // BLOCK + torch.arange(blocks, device="cuda")
    at = blk[..., None] * BLOCK + torch.arange(BLOCK, device="cuda") - start[:, None, None]  # row among the new tokens
    is_new = (at >= 0) & (at < s["new"][:, None, None])
    is_old = at < 0
    live = is_new.any(-1)
    page = torch.where(live, s["bt"].gather(1, (blk // 4).clamp(max=s["bt"].shape[1] - 1)).long(), s["kc"].shape[0] - 1)
    sub = torch.where(live, blk % 4, 0)
    row = (torch.arange(batch, device="cuda")[:, None, None] * seq + at.clamp(0, seq - 1))
    turned = _turn(_heads(s["k"], hd), s["table"][(start[:, None] + torch.arange(seq, device="cuda")).clamp(max=case["ctx"] - 1).view(-1)])

    def put(x, codes, scales):
        codes = codes.view(-1, kv, PAGE // BLOCK, BLOCK, hd)
        x = x[row].transpose(2, 3)  # [batch, blocks, kv, 16, hd]
        m, o = is_new[:, :, None, :, None], is_old[:, :, None, :, None]
        held = codes[page, :, sub]
        s_old = scales[page, :, sub]
        had = (is_old.any(-1) & live)[:, :, None]
        scale = _scale(torch.where(m, x, 0).abs().amax((3, 4)))
        scale = torch.where(had, torch.maximum(scale, s_old), scale)
        scale = torch.where(live[:, :, None], scale, s_old)
        old = held.view(torch.float8_e4m3fn).float() * (s_old / scale)[..., None, None]
        new = (torch.where(m, x, old) / torch.where(m, scale[..., None, None], 1)).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[page, :, sub] = torch.where(m | (o & had[..., None, None]), new, held)
        scales[page, :, sub] = scale
    put(turned, s["kc"], s["ks"])
    put(_heads(s["v"], hd), s["vc"], s["vs"])
    return [s["kc"].view(torch.float8_e4m3fn), s["vc"].view(torch.float8_e4m3fn), s["ks"], s["vs"]]


def _append_own(s):
    _framework().kv8_append(s["cache"], s["case"]["seq"], s["k"], s["v"], rope=s["table"], seq_lens=s["new"])
    return [s["kc"].view(torch.float8_e4m3fn), s["vc"].view(torch.float8_e4m3fn), s["ks"], s["vs"]]


def _attend_plain(s):
    case = s["case"]
    batch, seq, kv, hd = case["batch"], case["seq"], case["kv"], case["hd"]
    group = case["heads"] // kv
    at = torch.arange(s["bt"].shape[1] * PAGE, device="cuda")
    pos = s["ctx"][:, None] - seq + torch.arange(seq, device="cuda")
    seen = at <= pos[..., None]
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]

    def held(codes, scales):
        x = codes[s["bt"].long()].view(torch.float8_e4m3fn).float().view(batch, -1, kv, PAGE // BLOCK, BLOCK, hd)
        x *= scales[s["bt"].long()][..., None, None]
        return x.transpose(1, 2).reshape(batch, kv, -1, hd)
    q = s["q"].float().view(batch, seq, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * seq, hd)
    x = (q @ held(s["kc"], s["ks"]).transpose(2, 3)).view(batch, kv, group, seq, -1) / math.sqrt(hd)
    x = torch.where(seen[:, None, None], x, float("-inf"))
    x = (x - x.amax(-1, keepdim=True)).exp()
    total = x.sum(-1, keepdim=True)
    y = (x.view(batch, kv, group * seq, -1) @ held(s["vc"], s["vs"])).view(batch, kv, group, seq, hd) / total
    return y.permute(0, 3, 1, 2, 4).reshape(batch * seq, -1).bfloat16()


def _attend_own(s):
    _framework().kv8_attention(s["cfg"], s["cache"], s["case"]["seq"], s["q"], s["out"], s["case"]["ctx"])
    return s["out"]


_plain = {"norm": _norm_plain, "append": _append_plain, "attend": _attend_plain}
_own = {"norm": _norm_own, "append": _append_own, "attend": _attend_own}


# ------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    hd = case["hd"]
    half = hd // 2
    if case["op"] == "norm":
        if case["tokens"] * (case["heads"] + case["kv"]) * hd > 1 << 28:
            return None
        cos, sin = s["table"][s["pos"].long()].double().unsqueeze(1).unbind(-1)
        z = torch.complex(cos, sin)
        got, sums = [], []
        for x, gamma, dy in ((s["q"], s["q_gamma"], s.get("dyq")), (s["k"], s["k_gamma"], s.get("dyk"))):
            x = x.double().view(x.shape[0], -1, hd)
            gamma = gamma.double()
            inv = torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + EPS)
            if dy is None:
                y = x * inv * gamma
                y = torch.complex(y[..., :half], y[..., half:]) * z
                got.append(torch.cat([y.real, y.imag], -1).view(x.shape[0], -1))
                continue
            dy = dy.double().view(x.shape)
            u = torch.complex(dy[..., :half], dy[..., half:]) * z.conj()
            u = torch.cat([u.real, u.imag], -1)
            sums.append(torch.einsum("thd,thd->d", u, x * inv))
            u = u * gamma
            got.append((u * inv - x * inv ** 3 * (u * x).sum(-1, keepdim=True) / hd).view(x.shape[0], -1))
        return got + sums
    if case["op"] == "append":
        if sum(_new(case)) * case["kv"] * hd > 1 << 27:
            return None
        angle = s["table"].double()
        z = torch.complex(angle[..., 0], angle[..., 1])
        for codes, scales, x, turn in ((s["kc"], s["ks"], s["k"], True), (s["vc"], s["vs"], s["v"], False)):
            for b, (n, new) in enumerate(zip(_ctx(case), _new(case))):
                y = x[b * case["seq"]: b * case["seq"] + new].double().view(new, case["kv"], hd)
                if turn:
                    y = torch.complex(y[..., :half], y[..., half:]) * z[n - new: n, None]
                    y = torch.cat([y.real, y.imag], -1)
                p = n - new
                while p < n:
                    end = min(n, (p // BLOCK + 1) * BLOCK)
                    page, sub, lo = int(s["bt"][b, p // PAGE]), p % PAGE // BLOCK, p % BLOCK
                    piece = y[p - (n - new): end - (n - new)].transpose(0, 1)  # [kv, tokens, hd]
                    scale = torch.exp2(torch.ceil(torch.log2(piece.abs().amax((1, 2)) / 448))).clamp_min(FLOOR)
                    block = codes[page, :, sub * BLOCK: (sub + 1) * BLOCK].view(torch.float8_e4m3fn)
                    if lo:
                        was = scales[page, :, sub].double()
                        scale = torch.maximum(scale, was)
                        held = block[:, :lo].double() * (was / scale)[:, None, None]
                        block[:, :lo] = held.to(torch.float8_e4m3fn)
                    block[:, lo: lo + end - p] = (piece / scale[:, None, None]).to(torch.float8_e4m3fn)
                    scales[page, :, sub] = scale.float()
                    p = end
        return [s["kc"].view(torch.float8_e4m3fn), s["vc"].view(torch.float8_e4m3fn), s["ks"], s["vs"]]
    if sum(p for p, _ in _seen(case)) * case["heads"] * hd > 1 << 37:
        return None
    group, out = case["heads"] // case["kv"], []
    for b, n in enumerate(_ctx(case)):
        pages = s["bt"][b, : (n + PAGE - 1) // PAGE].long()
        first = n - case["seq"]
        pos = torch.arange(first, n, device="cuda")
        far = torch.arange(n, device="cuda")[None] - pos[:, None]
        hidden = (far > 0) | (far <= -(case["window"] or n + 1))
        q = s["q"][b * case["seq"]: (b + 1) * case["seq"]].double().view(case["seq"], case["heads"], hd)
        rows = []
        for h in range(case["kv"]):
            k, v = ((c[pages, h].view(torch.float8_e4m3fn).double() * r[pages, h].double().repeat_interleave(BLOCK, 1)[..., None]).reshape(-1, hd)[:n]
                    for c, r in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            x = torch.einsum("thd,nd->thn", q[:, h * group: (h + 1) * group], k) / hd ** 0.5
            rows.append(torch.softmax(x.masked_fill(hidden[:, None], float("-inf")), -1) @ v)
        out.append(torch.cat(rows, 1).reshape(case["seq"], -1))
    return torch.cat(out)
