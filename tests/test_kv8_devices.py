"""The bare q/k norm and E4M3 cache entries take tensors of the device that they run on:
a host tensor or one of another GPU is refused before its pointer reaches the library.
Tensors are stand-ins with a torch tensor's attributes, so this runs without a GPU."""
import pytest

import welvet_b200 as W

torch = pytest.importorskip("torch")
HERE, HD, ROWS, HEADS, KV = 1, 64, 6, 4, 2
SIZES = {torch.float32: 4, torch.bfloat16: 2, torch.int32: 4, torch.uint8: 1}


class Fake:
    def __init__(self, shape, dtype, device=HERE):
        self.shape, self.dtype, self._device = shape, dtype, device

    device = property(lambda self: f"cuda:{self._device}" if self._device >= 0 else "cpu")

    def get_device(self):
        return self._device

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def stride(self):
        return tuple(torch.Size(self.shape[i + 1:]).numel() for i in range(len(self.shape)))

    def element_size(self):
        return SIZES[self.dtype]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20


def rows(heads):
    return Fake((ROWS, heads * HD), torch.bfloat16)


def f32(*shape):
    return Fake(shape, torch.float32)


def cache_tensors():
    codes = lambda: Fake((5, KV, 64, HD), torch.uint8)  # noqa: E731
    return dict(ck=codes(), cv=codes(), ks=f32(5, KV, 4), vs=f32(5, KV, 4), table=Fake((2, 2), torch.int32),
                ctx=Fake((2,), torch.int32))


def cache(t):
    return W.Kv8Cache(t.pop("ck"), t.pop("cv"), t.pop("ks"), t.pop("vs"), t.pop("table"), t.pop("ctx"))


def call_rope_table(t):
    W.rope_table(8, HD, t["out"])


def call_norm(t):
    W.qk_norm_rope(t["q"], t["k"], t["qo"], t["ko"], HD, t["gq"], t["gk"], rope=t["rope"], positions=t["pos"])


def call_backward(t):
    W.qk_norm_rope_backward(t["q"], t["k"], t["dqo"], t["dko"], t["qo"], t["ko"], t["dgq"], t["dgk"], HD, t["ws"], t["gq"], t["gk"],
                            rope=t["rope"], positions=t["pos"])


def call_append(t):
    W.kv8_append(cache(t), 3, t["k"], t["v"], rope=t["rope"], seq_lens=t["lens"])


def call_attention(t, device=-1):
    c = cache(t)
    cfg = W.MhaConfig()
    cfg.d_model, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.device = HEADS * HD, HEADS, KV, HD, device
    W.kv8_attention(cfg, c, 3, t["q"], t["out"], 64, seq_lens=t["lens"])


def norm_tensors(**more):
    return dict(q=rows(HEADS), k=rows(KV), qo=rows(HEADS), ko=rows(KV), gq=f32(HD), gk=f32(HD), rope=f32(8, HD // 2, 2),
                pos=Fake((ROWS,), torch.int32), **more)


CALLS = {
    "rope_table": (call_rope_table, lambda: dict(out=f32(8, HD // 2, 2))),
    "norm": (call_norm, norm_tensors),
    "backward": (call_backward, lambda: norm_tensors(dqo=rows(HEADS), dko=rows(KV), dgq=f32(HD), dgk=f32(HD),
                                                     ws=Fake((1 << 24,), torch.uint8))),
    "append": (call_append, lambda: dict(cache_tensors(), k=rows(KV), v=rows(KV), rope=f32(8, HD // 2, 2),
                                         lens=Fake((2,), torch.int32))),
    "attention": (call_attention, lambda: dict(cache_tensors(), q=rows(HEADS), out=rows(HEADS), lens=Fake((2,), torch.int32))),
}


class Reached(Exception):
    pass


@pytest.fixture
def library(monkeypatch):
    """The library's entries replaced by one that says that it was reached; the process on
    device HERE."""
    class Entries:
        def __getattr__(self, name):
            if name == "welvet_b200_qk_norm_rope_workspace":
                return lambda hd: 592 * hd * 4

            def entry(*a):
                raise Reached(name)
            return entry
    monkeypatch.setattr(W, "lib", lambda: Entries())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: HERE)


@pytest.mark.parametrize("name", CALLS)
def test_tensors_of_the_device_reach_the_library(library, name):
    call, make = CALLS[name]
    with pytest.raises(Reached):
        call(make())


@pytest.mark.parametrize("name,which", [(n, w) for n, (_, make) in CALLS.items() for w in make()])
@pytest.mark.parametrize("device", [-1, 0])
def test_a_tensor_of_another_place_is_refused(library, name, which, device):
    call, make = CALLS[name]
    t = make()
    t[which]._device = device
    with pytest.raises(ValueError):
        call(t)


@pytest.mark.parametrize("name", CALLS)
def test_tensors_of_a_device_that_is_not_current_are_refused(library, monkeypatch, name):
    call, make = CALLS[name]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError):
        call(make())


def test_attention_runs_on_the_device_of_its_configuration(library, monkeypatch):
    make = CALLS["attention"][1]
    with pytest.raises(ValueError):
        call_attention(make(), device=0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(Reached):
        call_attention(make(), device=HERE)


def test_host_tensors_are_refused():
    t = torch.zeros(ROWS, HEADS * HD, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        W.qk_norm_rope(t, None, t, None, HD)
    with pytest.raises(ValueError):
        W.rope_table(8, HD, torch.zeros(8, HD // 2, 2))
    codes, scales = torch.zeros(5, KV, 64, HD, dtype=torch.uint8), torch.zeros(5, KV, 4)
    with pytest.raises(ValueError):
        W.Kv8Cache(codes, codes, scales, scales, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
