"""Host-side checks of the shared-prefix attention, sampling, top-logit and distillation entry points: arguments that
are refused before anything is launched, and the workspace query. Pointers are small aligned numbers that nothing
reads."""
import pytest
import torch

A = 256  # a non-NULL, 16-byte aligned pointer


def _call(name, *args):
    from midstream_llm_b200 import _lib
    _lib.call(name, *args)


def _prefix(**kw):
    a = dict(qkv=A, ld_qkv=768, kp=A, vp=A, ld_p=256, P=100, kc=A, vc=A, ld_c=256, bs=25600, lens=A, max_len=100, B=2, H=4,
             kv=4, D=64, scale=0.125, ws=A, out=A, ld_out=256, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(D=128), "head_dim must be 64"), (dict(qkv=None), "NULL"), (dict(lens=None), "NULL"), (dict(kp=None), "NULL"),
    (dict(B=0), "bad shape"), (dict(H=5, kv=2), "bad shape"), (dict(H=130, kv=1), "bad shape"), (dict(P=-1), "bad shape"),
    (dict(max_len=0), "bad shape"), (dict(P=1 << 40), "bad shape"), (dict(qkv=A + 8), "16-byte"), (dict(ws=A + 4), "16-byte"),
    (dict(ld_qkv=764), "strides"), (dict(ld_qkv=760), "strides"), (dict(ld_c=248), "strides"), (dict(ld_p=260), "strides"),
    (dict(bs=12), "strides"), (dict(ld_out=255), "strides"),
])
def test_prefix_attention_refuses(kw, text):
    from midstream_llm_b200 import _lib
    with pytest.raises(_lib.JxError, match=text):
        _call("jx_attn_decode_prefix", *_prefix(**kw))


def test_prefix_workspace_query():
    from midstream_llm_b200 import _lib, ops
    need = lambda *a: _lib.query("jx_attn_decode_prefix_workspace_bytes", *a)  # noqa: E731
    assert need(0, 4, 4, 10, 10) == need(1, 4, 3, 10, 10) == need(1, 4, 4, -1, 10) == need(1, 4, 4, 10, 0) == -1
    # every row has room for at least one part: (m, l) and 64 sums
    for B, H, kv, P, S in ((1, 4, 4, 1, 1), (16, 16, 16, 1791, 257), (64, 16, 4, 40000, 1000), (300, 2, 1, 129, 5)):
        assert need(B, H, kv, P, S) >= B * H * (8 + 256)
        assert need(B, H, kv, 0, S) >= B * H * (8 + 256)
    with pytest.raises(ValueError, match="unsupported shape"):
        ops.attn_decode_prefix_workspace_bytes(2, 130, 1, 10, 10)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "NULL"), (dict(u=None), "NULL"), (dict(tok=None), "NULL"), (dict(rows=0), "bad shape"),
    (dict(V=0), "bad shape"), (dict(V=(1 << 20) + 1, ld=(1 << 20) + 8), "bad shape"), (dict(ld=992), "bad shape"),
    (dict(ld=1004), "ld%8"), (dict(x=A + 2), "16B"),
])
def test_sample_refuses(kw, text):
    from midstream_llm_b200 import _lib
    a = dict(x=A, rows=3, V=1000, ld=1000, u=A, T=None, Ts=1.0, k=None, ks=0, p=None, ps=1.0, m=None, ms=0.0, tok=A, lp=None,
             stream=None)
    a.update(kw)
    with pytest.raises(_lib.JxError, match=text):
        _call("jx_sample", *a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(k=0), "k must be"), (dict(k=1001), "k must be"), (dict(V=4000, ld=4000, k=1025), "k must be"), (dict(v=None), "NULL"),
    (dict(rows=-1), "bad shape"), (dict(ld=1004), "ld%8"),
])
def test_top_logits_refuses(kw, text):
    from midstream_llm_b200 import _lib
    a = dict(x=A, rows=3, V=1000, ld=1000, k=5, v=A, i=A, stream=None)
    a.update(kw)
    with pytest.raises(_lib.JxError, match=text):
        _call("jx_top_logits", *a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "NULL"), (dict(ids=None), "NULL"), (dict(stats=None), "NULL"), (dict(K=0), "teacher slots"),
    (dict(K=1025), "teacher slots"), (dict(tau=0.0), "temperature"), (dict(tau=float("nan")), "temperature"),
    (dict(alpha=-0.1), "alpha"), (dict(alpha=float("nan")), "alpha"), (dict(rows=0), "bad shape"), (dict(ld=1004), "ld%8"),
])
def test_distill_refuses(kw, text):
    from midstream_llm_b200 import _lib
    a = dict(x=A, rows=3, V=1000, ld=1000, ids=A, t=A, f16=1, K=4, y=A, ignore=-100, tau=1.0, alpha=1.0)
    a.update({k: v for k, v in kw.items() if k in a})
    s = kw.get("stats", A)
    with pytest.raises(_lib.JxError, match=text):
        _call("jx_distill_fwd", *a.values(), None, s, A, None)
    with pytest.raises(_lib.JxError, match=text):
        _call("jx_distill_bwd", *a.values(), s, A, A, A, 1000, None)


def test_distill_backward_refuses_other_strides_in_place():
    from midstream_llm_b200 import _lib
    with pytest.raises(_lib.JxError, match="in place"):
        _call("jx_distill_bwd", A, 3, 1000, 1008, A, A, 1, 4, A, -100, 1.0, 1.0, A, A, A, A, 1000, None)


def test_wrappers_refuse_cpu_tensors():
    from midstream_llm_b200 import ops
    x, u = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(2)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ops.sample(x, u), lambda: ops.top_logits(x, 2), lambda: ops.distill_fwd(x, ids, x[:, :3], ids[:, 0]),
                 lambda: ops.attn_decode_prefix(x, x, x, 1, x, x, u.int(), 4, 64)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_prefix_schedule_gives_every_tile_to_one_block():
    """The rule that cuts the prefix tiles among blocks, restated: runs that cover the line, at least one tile each,
    and no more blocks on a unit than the workspace has parts for."""
    import random
    r = random.Random(0)
    for _ in range(2000):
        NT, units, blocks = r.randint(1, 300), r.randint(1, 70), r.choice([2, 20, 296])
        T = NT * units
        gp = min(T, blocks)
        per, more = T // gp, T % gp
        starts = [c * per + min(c, more) for c in range(gp + 1)]
        assert starts[0] == 0 and starts[-1] == T and all(b > a for a, b in zip(starts, starts[1:]))
        big = more * (per + 1)
        block_of = lambda x: x // (per + 1) if x < big else more + (x - big) // per  # noqa: E731
        for x in {0, T - 1, *(r.randrange(T) for _ in range(5))}:
            c = block_of(x)
            assert starts[c] <= x < starts[c + 1]
        room = min(NT, -(-(NT - 1) // per) + 1)
        for u in range(units):
            assert block_of(u * NT + NT - 1) - block_of(u * NT) + 1 <= room


@pytest.mark.parametrize("what", ["generate", "next_token_logits"])
def test_decoding_state_follows_the_model_to_another_device(monkeypatch, what):
    """What is kept on the model between calls belongs to a device: on another one it is built anew."""
    from midstream_llm_b200 import decode
    made = []

    class Kept:
        def __init__(self, model, n=0, max_new=0):
            self.n, self.max_new, self.device = n, max_new, next(model.parameters()).device
            made.append(self.device.type)

        def generate(self, prompt, **settings):
            return self

        def next_token_logits(self, context):
            return self

    monkeypatch.setattr(decode, "PromptSampler", Kept)
    monkeypatch.setattr(decode, "KVCacheDecoder", Kept)
    model = torch.nn.Linear(2, 2)
    run = {"generate": lambda: decode.generate(model, [1], n=2, max_new_tokens=4),
           "next_token_logits": lambda: decode.next_token_logits(model, [1])}[what]
    first = run()
    assert run() is first
    model.to("meta")
    second = run()
    assert second is not first and second.device.type == "meta" and run() is second
    assert made == ["cpu", "meta"]


def test_decoding_state_refuses_a_model_that_has_moved():
    from types import SimpleNamespace

    from midstream_llm_b200 import decode
    fl = SimpleNamespace(device=torch.device("cpu"))
    model = SimpleNamespace(flat=lambda: fl)
    assert decode._flat_on(model, torch.device("cpu")) is fl
    sampler = object.__new__(decode.PromptSampler)
    sampler.model, sampler.device = SimpleNamespace(flat=lambda: fl, config=None), torch.device("cuda:1")
    with pytest.raises(RuntimeError, match="moved to cpu"):
        sampler._start([1], -1)


@pytest.mark.parametrize("scale", [-0.125, float("nan"), float("inf"), -float("inf")])
def test_prefix_attention_refuses_a_scale_without_order(scale):
    from midstream_llm_b200 import _lib
    with pytest.raises(_lib.JxError, match="scale"):
        _call("jx_attn_decode_prefix", *_prefix(scale=scale))


@pytest.mark.parametrize("H", [1 << 22, 1 << 23, 1 << 24])
def test_prefix_attention_counts_the_columns_of_many_heads(H):
    """Rows of 2^30 elements and more, whose count does not fit 32 bits: too short a stride is seen, more heads are refused."""
    from midstream_llm_b200 import _lib
    with pytest.raises(_lib.JxError, match="strides|bad shape"):
        _call("jx_attn_decode_prefix", *_prefix(B=1, H=H, kv=H, ld_qkv=64, ld_p=H * 64, ld_c=H * 64, ld_out=H * 64, P=4, max_len=4))


@pytest.mark.parametrize("B,bs,ld_c", [(2, 0, 256), (2, 8, 256), (2, 248, 512), (2, 256, 256), (3, 256, 512), (2, 25592, 256),
                                       (2, 12800, 256)])
def test_prefix_attention_refuses_caches_that_overlap(B, bs, ld_c):
    from midstream_llm_b200 import _lib
    with pytest.raises(_lib.JxError, match="overlap"):
        _call("jx_attn_decode_prefix", *_prefix(B=B, bs=bs, ld_c=ld_c))


def test_a_captured_step_goes_with_the_weight_storage_it_reads():
    """A storage that takes the place (and may take the address) of the one that a step was captured with ends that step's use."""
    from types import SimpleNamespace

    from midstream_llm_b200 import decode
    new = lambda: SimpleNamespace(device=torch.device("cpu"), generation=0, refresh_f16=lambda: None)  # noqa: E731
    model = SimpleNamespace(_flat=None)
    model.flat = lambda: model._flat
    dec = object.__new__(decode.KVCacheDecoder)
    dec.model, dec.device, dec.max_len, dec.logits = model, torch.device("cpu"), 8, torch.zeros(1, 4)
    dec.context, dec._fl, dec._generation, dec._graph = [], None, -1, None
    dec._prefill = lambda ctx: None
    model._flat = new()
    dec.next_token_logits([1, 2])
    dec._graph = object()
    kept = dec._graph
    dec.next_token_logits([3])  # another prompt, the same storage
    assert dec._graph is kept
    model._flat = new()
    dec.next_token_logits([3])
    assert dec._graph is None and dec._fl is model._flat
