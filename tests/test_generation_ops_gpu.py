"""Shared-prefix decode attention, sampling and top logits on the GPU, each against its definition in 64 bits.

Tolerances, before any run. Attention: probabilities are rounded to fp16 before the product with V (half a step,
2^-11 of each), the output once more, and fp32 arithmetic (scores up to about 40 in the exponent, 2^-24 each)
stays below 2^-17 of the weighted magnitudes; with A = sum p |v| an element may be off by
2^-11 |o| + (2^-11 + 2^-17) A + 2^-25 (half the finest fp16 step). Tokens, ids and values are exact. A log
probability is rounded to fp32 once: 2^-24 of it, plus 1e-9 for the weights' units of 2^-42."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    from midstream_llm_b200 import ops as _ops
    return _ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- shared-prefix attention
def _prefix_state(B, H, kv, P, S, lens, seed=0, ld_extra=0, junk=NAN):
    """Inputs whose caches hold `junk` wherever nothing may be read."""
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    qkv = r(B, (H + 2 * kv) * 64 + ld_extra)[:, :(H + 2 * kv) * 64]
    kp, vp = r(P + 9, kv * 64), r(P + 9, kv * 64)
    kp[P:], vp[P:] = junk, junk
    kc, vc = r(B, S + 3, kv * 64), r(B, S + 3, kv * 64)
    for b, n in enumerate(lens):
        kc[b, max(n - 1, 0):], vc[b, max(n - 1, 0):] = junk, junk
    return qkv, kp, vp, kc, vc, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _prefix_check(out, qkv, kp, vp, kc, vc, P, lens, H, kv, bad=()):
    """Output and caches after the call against the definition."""
    G = H // kv
    for b, n in enumerate(lens):
        if n <= 0 or b in bad:
            assert bool((out[b] == 0).all())
            continue
        newk, newv = qkv[b, H * 64:(H + kv) * 64], qkv[b, (H + kv) * 64:]
        assert torch.equal(kc[b, n - 1], newk) and torch.equal(vc[b, n - 1], newv)
        assert bool(kc[b, n:].isnan().all()) and bool(vc[b, n:].isnan().all())
        k = torch.cat([kp[:P], kc[b, :n]]).double().view(P + n, kv, 1, 64).expand(-1, -1, G, -1).reshape(P + n, H, 64)
        v = torch.cat([vp[:P], vc[b, :n]]).double().view(P + n, kv, 1, 64).expand(-1, -1, G, -1).reshape(P + n, H, 64)
        q = qkv[b, :H * 64].double().view(H, 64)
        w = torch.softmax(torch.einsum("hd,phd->hp", q, k) / 8.0, dim=-1)
        o, a = torch.einsum("hp,phd->hd", w, v), torch.einsum("hp,phd->hd", w, v.abs())
        tol = 2 ** -11 * o.abs() + (2 ** -11 + 2 ** -17) * a + 2 ** -25
        err = (out[b].double().view(H, 64) - o).abs()
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))


@pytest.mark.parametrize("B,H,kv,P,lens", [
    (1, 4, 4, 0, [1]),                                    # nothing but the new token
    (1, 4, 4, 1, [1]),
    (2, 1, 1, 127, [0, 3]),
    (3, 4, 4, 128, [1, 128, 129]),
    (4, 11, 11, 129, [127, 0, 256, 1]),
    (5, 4, 4, 0, [1, 130, 64, 0, 257]),
    (16, 16, 16, 1000, [(37 * i) % 200 for i in range(16)]),
    (7, 8, 2, 515, [1, 2, 0, 40, 300, 128, 5]),           # four heads a key head
    (50, 6, 2, 260, [1 + (i * 11) % 70 for i in range(50)]),  # three: 42 sequences a row tile
    (130, 4, 4, 200, [(i * 7) % 33 for i in range(130)]),  # two row tiles
    (3, 64, 1, 300, [5, 0, 131]),                         # 64 heads on one key head
    (1030, 2, 2, 70, [i % 4 for i in range(1030)]),       # more sequences than lengths kept on chip
    (2, 2, 2, 20000, [2000, 1]),                          # long enough to split both
    (1, 2, 2, 3, [9000]),
])
def test_prefix_attention(ops, B, H, kv, P, lens):
    S = max(max(lens), 1)
    st = _prefix_state(B, H, kv, P, S, lens, seed=B + P)
    before = [t.clone() for t in st[:3]]
    out = ops.attn_decode_prefix(*st[:3], P, *st[3:], H, 64, kv_heads=kv, max_len=S)
    _prefix_check(out, *st[:5], P, lens, H, kv)
    for t, u in zip(st[:3], before):
        assert torch.equal(t.view(torch.int16), u.view(torch.int16))


@pytest.mark.parametrize("kv,P,S", [(8, 0, 512), (8, 40, 130), (1, 0, 512), (1, 300, 257)])
@pytest.mark.parametrize("G", [1, 2, 3, 4])
def test_prefix_attention_own_keys(ops, G, kv, P, S):
    """Own keys up to every border of the steps they are read in, with few and with many (sequence, head) pairs."""
    lens = [0, 1, 15, 16, 17, 31, 33, 48, 63, 64, 65, 80, 96, 112, 127, 128, 129, 130]
    lens += [n for n in (143, 144, 145, 192, 255, 256, 257, 384, 500, 511, 512) if n <= S]
    lens = lens * (2 if kv > 1 else 1)
    st = _prefix_state(len(lens), G * kv, kv, P, S, lens, seed=G + P)
    out = ops.attn_decode_prefix(*st[:3], P, *st[3:], G * kv, 64, kv_heads=kv, max_len=S)
    _prefix_check(out, *st[:5], P, lens, G * kv, kv)


@pytest.mark.parametrize("H,kv", [(2, 2), (8, 1)])
def test_prefix_attention_scores_of_minus_infinity(ops, H, kv):
    """Keys with an infinite score below weigh nothing, a whole tile of them included; with such keys alone the result is
    NaN, as the formula's."""
    P, S, lens = 300, 200, [1, 40, 200, 3]
    qkv, kp, vp, kc, vc, n = _prefix_state(4, H, kv, P, S, lens, seed=9)
    q = qkv[:, :H * 64].view(4, H, 64)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    kp.view(-1, kv, 64)[:256, :, 0] = -INF
    kc[1:, :2].view(3, 2, kv, 64)[:, :, :, 0] = -INF  # (the first sequence has no keys before its new one)
    out = ops.attn_decode_prefix(qkv, kp, vp, P, kc, vc, n, H, 64, kv_heads=kv, max_len=S)
    _prefix_check(out, qkv, kp, vp, kc, vc, P, lens, H, kv)
    kp.view(-1, kv, 64)[:, :, 0] = -INF
    qkv[:, H * 64:(H + kv) * 64].view(4, kv, 64)[:, :, 0] = -INF
    out = ops.attn_decode_prefix(qkv, kp, vp, P, kc, vc, n, H, 64, kv_heads=kv, max_len=S)
    assert bool(out[0].isnan().all())


@pytest.mark.parametrize("B", [1, 3])
def test_prefix_attention_single_rows(ops, B):
    """A prefix of no rows or one, caches of one row: dimensions whose stride says nothing."""
    H, kv = 4, 2
    qkv, kp, vp, kc, vc, n = _prefix_state(B, H, kv, 1, 1, [1] * B, seed=B)
    for P in (0, 1):
        k, v = kp[:P], vp[:P]
        kb, vb = kc[:, :1].clone(), vc[:, :1].clone()
        out = ops.attn_decode_prefix(qkv, k, v, P, kb, vb, n, H, 64, kv_heads=kv)
        _prefix_check(out, qkv, k, v, kb, vb, P, [1] * B, H, kv)
    empty = torch.empty(0, kv * 64, device="cuda", dtype=torch.float16)
    assert torch.equal(ops.attn_decode_prefix(qkv, empty, empty, 0, kb, vb, n, H, 64, kv_heads=kv),
                       ops.attn_decode_prefix(qkv, kp, vp, 0, kb, vb, n, H, 64, kv_heads=kv))


def test_prefix_attention_views_and_repeats(ops):
    """Keys and values as columns of one fused buffer, padded rows of the queries and the output, the caches'
    sequences in another order than their rows; the same call twice gives the same bits."""
    B, H, P, lens = 6, 4, 333, [5, 0, 77, 128, 1, 200]
    d, S = H * 64, 200
    qkv, kp, vp, kc, vc, n = _prefix_state(B, H, H, P, S, lens, seed=3, ld_extra=40)
    fused = torch.full((P + 9, 3 * d), NAN, device="cuda", dtype=torch.float16)
    fused[:, d:2 * d], fused[:, 2 * d:] = kp, vp
    caches = torch.full((2, S + 3, B, d), NAN, device="cuda", dtype=torch.float16)  # position-major
    caches[0], caches[1] = kc.transpose(0, 1), vc.transpose(0, 1)
    kct, vct = caches[0].transpose(0, 1), caches[1].transpose(0, 1)
    o = torch.full((B + 1, d + 24), 7.0, device="cuda", dtype=torch.float16)
    ops.attn_decode_prefix(qkv, fused[:, d:2 * d], fused[:, 2 * d:], P, kct, vct, n, H, 64, max_len=S, out=o[:B, :d])
    _prefix_check(o[:B, :d], qkv, kp, vp, kct, vct, P, lens, H, H)
    assert bool((o[B] == 7).all()) and bool((o[:, d:] == 7).all())
    first = o[:B, :d].clone()
    for _ in range(3):
        again = ops.attn_decode_prefix(qkv, kp, vp, P, kct, vct, n, H, 64, max_len=S)
        assert torch.equal(again, first)


def test_prefix_attention_graph_replay_and_bad_length(ops):
    """One captured step replayed while the lengths grow; a sequence past the bound is left out and reported."""
    from midstream_llm_b200 import _lib
    B, H, P, S = 3, 4, 150, 140
    lens = [120, 1, 0]
    qkv, kp, vp, kc, vc, n = _prefix_state(B, H, H, P, S, lens, seed=5)
    ws = torch.empty(ops.attn_decode_prefix_workspace_bytes(B, H, H, P, S) // 4 + 4, device="cuda")
    out = torch.empty(B, H * 64, device="cuda", dtype=torch.float16)
    run = lambda: ops.attn_decode_prefix(qkv, kp, vp, P, kc, vc, n, H, 64, max_len=S, workspace=ws, out=out)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    _lib.device_status()
    for step in range(22):
        if step:
            n += (n > 0).int()
            lens = [x + (x > 0) for x in lens]
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=_gen(step)))
        graph.replay()
        torch.cuda.synchronize()
        bad = [b for b in range(B) if lens[b] > S]
        _prefix_check(out, qkv, kp, vp, kc, vc, P, lens, H, H, bad=bad)
        assert _lib.device_status() == (204 if bad else 0)
    assert lens[0] > S


def test_prefix_attention_on_two_streams(ops):
    cases = []
    for i, (B, P) in enumerate([(4, 700), (9, 90)]):
        lens = [(k * 17) % 90 for k in range(B)]
        cases.append((B, P, lens, _prefix_state(B, 4, 4, P, 90, lens, seed=20 + i), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for B, P, lens, st, stream in cases:
        with torch.cuda.stream(stream):
            for _ in range(5):
                o = ops.attn_decode_prefix(*st[:3], P, *st[3:], 4, 64, max_len=90)
            outs.append(o)
    torch.cuda.synchronize()
    for (B, P, lens, st, _), o in zip(cases, outs):
        _prefix_check(o, *st[:5], P, lens, 4, 4)


def test_prefix_attention_refusals(ops):
    B, H, P, S = 2, 4, 20, 10
    st = _prefix_state(B, H, H, P, S, [1, 2])
    call = lambda *a, **k: ops.attn_decode_prefix(*a, **k)  # noqa: E731
    qkv, kp, vp, kc, vc, n = st
    with pytest.raises(ValueError, match="prefix_len"):
        call(qkv, kp, vp, P + 10, kc, vc, n, H, 64)
    with pytest.raises(ValueError, match="max_len"):
        call(qkv, kp, vp, P, kc, vc, n, H, 64, max_len=S + 4)
    with pytest.raises(TypeError, match="lengths"):
        call(qkv, kp, vp, P, kc, vc, n.long(), H, 64)
    with pytest.raises(ValueError, match="qkv"):
        call(qkv[:, :-64], kp, vp, P, kc, vc, n, H, 64)
    with pytest.raises(ValueError, match="layout"):
        call(qkv, kp, vp[:-1], P, kc, vc, n, H, 64)
    with pytest.raises(ValueError, match="overlap"):
        call(qkv, kp, vp, P, kc[:1].expand(2, -1, -1), vc[:1].expand(2, -1, -1), n, H, 64)
    with pytest.raises(ValueError, match="workspace"):
        call(qkv, kp, vp, P, kc, vc, n, H, 64, workspace=torch.empty(4, device="cuda"))
    with pytest.raises(RuntimeError, match="16-byte"):
        call(torch.empty(B, H * 192 + 8, device="cuda", dtype=torch.float16)[:, 4:-4], kp, vp, P, kc, vc, n, H, 64)


# ---------------------------------------------------------------- sampling
def _draw(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """The definition for one row, in 64 bits: (token, log probability)."""
    x, V = x.astype(np.float64), len(x)
    T, p, m = (float(np.float32(v)) for v in (T, p, m))
    if np.isnan(x).any() or (x == -np.inf).all():
        return -1, NAN
    best = int(x.argmax())
    if T <= 0:
        return best, 0.0
    with np.errstate(invalid="ignore"):
        e = np.where(x == x[best], 1.0, np.exp((x - x[best]) / T))
    order = np.lexsort((np.arange(V), -x))
    if 0 < k < V:
        order = order[:k]
    if p < 1:
        c = np.cumsum(e[order])
        order = order[:max(1, int((c - e[order] < p * c[-1]).sum()))]
    order = order[:max(1, int((e[order] >= m).sum()))]
    ids = np.sort(order)
    ids = ids[e[ids] > 0]
    c = np.cumsum(e[ids])
    at = min(int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right")), len(ids) - 1)
    return int(ids[at]), math.log(e[ids[at]] / c[-1])


def _check_draws(ops, x, u, settings, tokens=None):
    """`settings`: one dict per row. Once with tensors; once with numbers if all rows agree."""
    R = x.shape[0]
    name = {"T": ("temperature", 1.0, torch.float32), "k": ("top_k", 0, torch.int32), "p": ("top_p", 1.0, torch.float32),
            "m": ("min_p", 0.0, torch.float32)}
    calls = [{n: torch.tensor([s.get(a, d) for s in settings], device="cuda", dtype=t) for a, (n, d, t) in name.items()}]
    if all(s == settings[0] for s in settings):
        calls.append({n: settings[0].get(a, d) for a, (n, d, t) in name.items()})
    host = x.cpu().numpy()
    want = [_draw(host[r], float(u[r]), **settings[r]) for r in range(R)]
    for kw in calls:
        tok, lp = ops.sample(x, u, **kw)
        got = tok.tolist()
        assert got == [w[0] for w in want], [(r, settings[r], got[r], want[r]) for r in range(R) if got[r] != want[r][0]][:3]
        for r in range(R):
            if math.isnan(want[r][1]):
                assert math.isnan(float(lp[r]))
            else:
                assert abs(float(lp[r]) - want[r][1]) <= 2 ** -24 * abs(want[r][1]) + 1e-9, (r, settings[r])


FILTERS = [dict(), dict(T=0.0), dict(T=0.7), dict(k=1), dict(k=5), dict(k=300), dict(k=5000), dict(p=0.9), dict(p=0.3, T=1.5),
           dict(p=0.0), dict(m=0.1), dict(m=1.0), dict(m=2.0), dict(k=40, p=0.95), dict(k=40, p=0.95, m=0.05, T=0.8),
           dict(p=0.9, m=0.3), dict(k=700, p=0.5, T=2.0), dict(T=100.0), dict(T=0.01), dict(T=1e-6), dict(T=1e30)]


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 255, 256, 257, 1000, 8193, 24000, 32000, 32768, 32769, 50257])
@pytest.mark.parametrize("kind", ["model", "ties", "flat"])
def test_sample_matches_the_definition(ops, V, kind):
    R = len(FILTERS)
    g = _gen(V)
    ld = (V + 7) // 8 * 8 + 8
    x = torch.randn(R, ld, device="cuda", generator=g) * {"model": 3.0, "ties": 3.0, "flat": 0.05}[kind]
    if kind == "ties":
        x = (x * 2).round() / 2  # a few dozen values, -0 among them
        x[:, ::3] *= -1.0
    x = x.half()[:, :V]
    u = torch.rand(R, device="cuda", generator=g)
    _check_draws(ops, x, u, FILTERS)


@pytest.mark.parametrize("V,R", [(1, 1300), (257, 1300), (2049, 1400), (8192, 1300), (8193, 1200), (24000, 300)])
@pytest.mark.parametrize("kind", ["model", "ties", "flat"])
def test_sample_many_rows(ops, V, R, kind):
    """Rows drawn many at a time, where they get smaller blocks: the definition for some, and for all the bits of the same
    rows in small calls."""
    x = torch.randn(R, (V + 7) // 8 * 8, device="cuda", generator=_gen(V + 1)) * {"model": 3.0, "ties": 3.0, "flat": 0.05}[kind]
    if kind == "ties":
        x = (x * 2).round() / 2
    x = x.half()[:, :V]
    u = torch.rand(R, device="cuda", generator=_gen(R))
    rows = [FILTERS[r % len(FILTERS)] for r in range(R)]
    kw = {n: torch.tensor([s.get(a, d) for s in rows], device="cuda", dtype=t)
          for n, a, d, t in (("temperature", "T", 1.0, torch.float32), ("top_k", "k", 0, torch.int32),
                             ("top_p", "p", 1.0, torch.float32), ("min_p", "m", 0.0, torch.float32))}
    tok, lp = ops.sample(x, u, **kw)
    host = x[:63].cpu().numpy()
    assert tok[:63].tolist() == [_draw(host[r], float(u[r]), **rows[r])[0] for r in range(63)]
    for i in range(0, R, 100):
        t, l = ops.sample(x[i:i + 100], u[i:i + 100], **{n: v[i:i + 100] for n, v in kw.items()})
        assert torch.equal(t, tok[i:i + 100]) and torch.equal(l.view(torch.int32), lp[i:i + 100].view(torch.int32))


@pytest.mark.parametrize("V,kind", [(40, "model"), (300, "ties"), (4000, "model"), (4000, "ties"), (24000, "model"), (24000, "flat")])
def test_sample_short_lists(ops, V, kind):
    """Every number of kept elements up to and past what the way for short lists takes, with the other filters on top."""
    ks = [2, 3, 4, 5, 8, 31, 32, 33, 63, 64, 100, 127, 128, 129, 200, 251, 252, 253, 254, 255, 256, 257, 300]
    rows = [dict(k=k, **more) for k in ks for more in (dict(), dict(p=0.8), dict(m=0.2, T=0.9), dict(p=0.6, m=0.05, T=3.0))]
    rows += [dict(m=m, T=T) for m in (1e-6, 1e-3, 0.05, 0.5) for T in (0.3, 1.0, 4.0)]
    x = torch.randn(len(rows), (V + 7) // 8 * 8, device="cuda", generator=_gen(V)) * (0.05 if kind == "flat" else 3.0)
    if kind == "ties":
        x = (x * 4).round() / 4
    u = torch.rand(len(rows), device="cuda", generator=_gen(3))
    u[::9], u[1::9] = 0.0, 1.0 - 2 ** -24
    _check_draws(ops, x.half()[:, :V], u, rows)


def test_sample_a_large_vocabulary(ops):
    V = 200_001
    x = (torch.randn(6, 200_008, device="cuda", generator=_gen(1)) * 2).half()[:, :V]
    u = torch.rand(6, device="cuda", generator=_gen(2))
    _check_draws(ops, x, u, [dict(), dict(k=100), dict(p=0.9), dict(m=0.2), dict(k=50000, p=0.99), dict(T=0.0)])


def test_sample_same_settings_as_numbers_and_tensors(ops):
    x = (torch.randn(40, 32000, device="cuda", generator=_gen(4)) * 3).half()
    u = torch.rand(40, device="cuda", generator=_gen(5))
    for s in (dict(T=0.8, k=50, p=0.95, m=0.02), dict(p=0.9), dict(), dict(T=0.0)):
        _check_draws(ops, x, u, [s] * 40)


def test_sample_masks_infinities_and_bad_rows(ops):
    V = 3000
    base = (torch.randn(V, device="cuda", generator=_gen(6)) * 2).half()
    rows, settings = [], []
    for s in (dict(), dict(k=20), dict(p=0.9), dict(m=0.1), dict(T=0.0), dict(k=3, p=0.5)):
        masked = base.clone()
        masked[torch.rand(V, device="cuda", generator=_gen(7)) < 0.9] = -INF
        one = torch.full_like(base, -INF)
        one[1234] = -3.0
        none = torch.full_like(base, -INF)
        lowest = torch.full_like(base, torch.finfo(torch.float16).min)
        inf = base.clone()
        inf[[17, 99, 2000]] = INF
        nan = base.clone()
        nan[V - 1] = NAN
        few = torch.full_like(base, -INF)
        few[[5, 2999]] = torch.tensor([1.0, 1.0], device="cuda", dtype=torch.float16)
        for t in (masked, one, none, lowest, inf, nan, few):
            rows.append(t)
            settings.append(s)
    x = torch.stack(rows)
    for u0 in (0.0, 0.4, 1.0 - 2 ** -24):
        _check_draws(ops, x, torch.full((x.shape[0],), u0, device="cuda"), settings)


def test_sample_uniforms_outside_their_range_still_give_kept_tokens(ops):
    x = (torch.randn(4, 500, device="cuda", generator=_gen(8)) * 2).half()[:, :500]
    x = torch.nn.functional.pad(x, (0, 4))[:, :500]
    u = torch.tensor([1.0, 2.0, -1.0, NAN], device="cuda")
    tok, lp = ops.sample(x, u, top_k=3)
    for r in range(4):
        kept = sorted(np.lexsort((np.arange(500), -x[r].cpu().numpy().astype(np.float64)))[:3].tolist())
        assert int(tok[r]) == (kept[-1] if r < 2 else kept[0])


def test_sample_frequencies_follow_the_probabilities(ops):
    """Evenly spaced numbers draw each token as often as its probability says, to within one draw at each end."""
    x = (torch.randn(300, device="cuda", generator=_gen(9)) * 2).half()
    n = 20000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    rows = torch.nn.functional.pad(x, (0, 4))[None].expand(1, -1).repeat(n, 1)[:, :300]
    tok, _ = ops.sample(rows, u, temperature=1.2)
    got = torch.bincount(tok, minlength=300).double() / n
    want = torch.softmax(x.double() / float(np.float32(1.2)), 0)
    assert float((got - want).abs().max()) <= 1.0 / n + 2 ** -23  # u itself is rounded to fp32


def test_sample_in_a_graph_and_refusals(ops):
    x = (torch.randn(5, 4096, device="cuda", generator=_gen(10)) * 2).half()
    u = torch.rand(5, device="cuda", generator=_gen(11))
    tok = torch.empty(5, device="cuda", dtype=torch.int64)
    lp = torch.empty(5, device="cuda")
    ops.sample(x, u, top_p=0.9, tokens=tok, logprobs=lp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, u, top_p=0.9, tokens=tok, logprobs=lp)
    for seed in (12, 13):
        x.copy_(torch.randn(x.shape, device="cuda", generator=_gen(seed)))
        u.copy_(torch.rand(5, device="cuda", generator=_gen(seed + 50)))
        graph.replay()
        host = x.cpu().numpy()
        assert tok.tolist() == [_draw(host[r], float(u[r]), p=0.9)[0] for r in range(5)]
    with pytest.raises(ValueError, match="16-byte"):
        ops.sample(torch.zeros(4, 1001, device="cuda", dtype=torch.float16), u[:4])
    with pytest.raises(ValueError, match="uniforms"):
        ops.sample(x, u[:4])
    with pytest.raises(TypeError, match="top_k"):
        ops.sample(x, u, top_k=torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError, match="temperature"):
        ops.sample(x, u, temperature=-1.0)
    with pytest.raises(TypeError, match="logits16"):
        ops.sample(x.float(), u)


# ---------------------------------------------------------------- top logits
def _top(x, k):
    x = x.astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -np.where(np.isnan(x), -np.inf, x), np.isnan(x)))[:k]
    return x[order], order


@pytest.mark.parametrize("V,k", [(1, 1), (9, 9), (300, 1), (300, 256), (1000, 64), (2048, 1024), (2049, 1024), (24000, 16),
                                 (32000, 64), (32000, 128), (32000, 129), (32000, 1000), (40001, 64), (100_000, 700)])
@pytest.mark.parametrize("kind", ["model", "ties", "equal", "nan", "rising"])
def test_top_logits(ops, V, k, kind):
    _top_logits_case(ops, V, k, kind)


# A limit by threads and by vectors (above 3/8 of the threads), blocks of 128, 256 and 512 threads, rows that need a second
# reading, and k past half of the vectors.
@pytest.mark.parametrize("V,k", [(8000, 48), (8000, 49), (8192, 500), (8192, 513), (8193, 96), (16384, 97), (16377, 1024),
                                 (16385, 192), (32768, 193), (32000, 256), (32776, 400), (65536, 1024), (65537, 193)])
@pytest.mark.parametrize("kind", ["model", "ties", "equal", "nan", "rising"])
def test_top_logits_limits(ops, V, k, kind):
    _top_logits_case(ops, V, k, kind)


def _top_logits_case(ops, V, k, kind):
    R = 3
    x = torch.randn(R, (V + 7) // 8 * 8, device="cuda", generator=_gen(V + k)) * 3
    if kind == "ties":
        x = (x * 2).round() / 2
        x[:, ::3] *= -1.0
    elif kind == "equal":
        x = torch.full_like(x, -1.5)
    elif kind == "rising":
        x = torch.arange(x.shape[1], device="cuda")[None].expand(R, -1) / 64.0
    x = x.half()[:, :V].clone(memory_format=torch.preserve_format)
    x = torch.nn.functional.pad(x, (0, -V % 8), value=9.0)[:, :V]
    if kind == "nan":
        x[:, torch.rand(V, device="cuda", generator=_gen(1)) < 0.5] = NAN
        x[1] = NAN
        x[2, ::5] = -INF
        x[2, V // 2] = INF
    v, i = ops.top_logits(x, k)
    for r in range(R):
        wv, wi = _top(x[r].cpu().numpy(), k)
        assert i[r].tolist() == wi.tolist(), (kind, r)
        assert np.array_equal(v[r].cpu().numpy().astype(np.float64), wv, equal_nan=True)


def test_top_logits_refusals(ops):
    x = torch.zeros(2, 64, device="cuda", dtype=torch.float16)
    for k in (0, 65):
        with pytest.raises(RuntimeError, match="k must be"):
            ops.top_logits(x, k)
    with pytest.raises(RuntimeError, match="k must be"):
        ops.top_logits(torch.zeros(1, 4096, device="cuda", dtype=torch.float16), 1025)
    v, i = ops.top_logits(x[:0], 4)
    assert v.shape == (0, 4) and i.shape == (0, 4)


# ---------------------------------------------------------------- top-p alone
# Smooth rows: most of the weight lies below the limit that a row's list of tokens starts at. (spread, temperature)
SMOOTH = [(0.36, 1.0), (0.4, 1.0), (0.45, 1.0), (0.5, 1.0), (0.55, 1.0), (1.0, 3.0)]


def _check_alike(ops, x, u, tokens, logprobs, times, **kw):
    """The rows again, `times` over in one call: the same draws (more rows get smaller blocks)."""
    tok, lp = ops.sample(x.repeat(times, 1), u.repeat(times), **kw)
    assert torch.equal(tok, tokens.repeat(times)) and torch.equal(lp.view(torch.int32), logprobs.view(torch.int32).repeat(times))


@pytest.mark.parametrize("V", [8192, 24000, 32000, 32768, 50256])
@pytest.mark.parametrize("p", [0.3, 0.5, 0.7, 0.8, 0.9, 0.95])
def test_sample_nucleus_of_smooth_rows(ops, V, p):
    n = len(SMOOTH)
    x = torch.randn(n, V, device="cuda", generator=_gen(V))
    x = (x * torch.tensor([s for s, _ in SMOOTH], device="cuda")[:, None] + 0.3).half()
    u = torch.rand(n, device="cuda", generator=_gen(int(100 * p)))
    _check_draws(ops, x, u, [dict(p=p, T=T) for _, T in SMOOTH])
    same = slice(0, n - 1)
    _check_draws(ops, x[same], u[same], [dict(p=p)] * (n - 1))
    tok, lp = ops.sample(x[same], u[same], top_p=p)
    for times in (40, 240):
        _check_alike(ops, x[same], u[same], tok, lp, times, top_p=p)


@pytest.mark.parametrize("V,first", [(32000, 8192), (50256, 8192), (50256, 50000), (32000, 4096)])
@pytest.mark.parametrize("p", [0.5, 0.9])
def test_sample_nucleus_of_rows_that_begin_unlike_the_rest(ops, V, first, p):
    """The first tokens masked, or far below or above all others: what they say about the row is wrong."""
    x = (torch.randn(6, V, device="cuda", generator=_gen(V + first)) * 0.4).half()
    x[0, :first] = -INF
    x[1, :first] -= 4.0
    x[2, :first] -= 20.0
    x[3, :first] += 4.0
    x[4, :first] += 2.0
    x[5, first:] = -INF
    u = torch.rand(6, device="cuda", generator=_gen(first))
    _check_draws(ops, x, u, [dict(p=p)] * 6)
    tok, lp = ops.sample(x, u, top_p=p)
    _check_alike(ops, x, u, tok, lp, 30, top_p=p)


def _rows_cut_near_a_border(V, n, seed):
    """Rows of two values whose nucleus ends within 1e-4 of a token's weight of a border between two tokens, just before
    it and just behind it in turn: (logits, uniforms, settings). The tokens of the lower value lie below the list of
    the larger ones, so the sum of their weights, all equal, sets the place of the cut. The definition's running sum
    of up to V / 2 equal terms is off by at most V / 2 half steps of a number below V: 3e-5 for V of a million (the border
    is 1e-4 to 1e-3 away there), below 1e-7 for 50256."""
    rng, near = np.random.default_rng(seed), max(1e-5, 1e-10 * V)
    x, settings = np.empty((n, V), np.float16), []
    for r in range(n):
        while True:
            m, d = np.float16(rng.uniform(-9, 9)), np.float16(rng.uniform(2.1, 3.9))
            low = np.float16(m - d)
            e = math.exp(float(low) - float(m))
            high = rng.integers(int(0.5 * V), int(0.8 * V), 20000)
            p = rng.uniform(0.3, 0.75, 20000).astype(np.float32)
            q = p.astype(np.float64) * (high + (V - high) * e)
            off = q - np.rint(q)
            want = (off < 0) if r % 2 else (off > 0)
            fits = np.flatnonzero(want & (np.abs(off) > near) & (np.abs(off) < 10 * near))
            if len(fits):
                break
        i = fits[0]
        x[r] = np.where(rng.permutation(V) < high[i], m, low)
        settings.append(dict(p=float(p[i])))
    return torch.from_numpy(x).cuda(), torch.full((n,), 1.0 - 2 ** -24, device="cuda"), settings


@pytest.mark.parametrize("V,n", [(8192, 12), (50256, 24), (1_000_000, 6)])
def test_sample_nucleus_that_ends_at_a_border(ops, V, n):
    """Which tokens are kept is decided in 64 bits, however many equal weights the sum below the list has. (With the last
    kept token drawn, its place and probability both tell how many there are.)"""
    x, u, settings = _rows_cut_near_a_border(V, n, V)
    _check_draws(ops, x, u, settings)
    p = torch.tensor([s["p"] for s in settings], device="cuda")
    tok, lp = ops.sample(x, u, top_p=p)
    for times in (200 // n, 1200 // n) if V < 10 ** 6 else ():
        _check_alike(ops, x, u, tok, lp, times, top_p=p.repeat(times))


def test_sample_nucleus_of_smooth_rows_of_a_large_vocabulary(ops):
    V, n = 200_000, len(SMOOTH)
    x = torch.randn(n, V, device="cuda", generator=_gen(V))
    x = (x * torch.tensor([s for s, _ in SMOOTH], device="cuda")[:, None]).half()
    u = torch.rand(n, device="cuda", generator=_gen(1))
    for p in (0.3, 0.5, 0.8, 0.95):
        _check_draws(ops, x, u, [dict(p=p, T=T) for _, T in SMOOTH])
        tok, lp = ops.sample(x[:5], u[:5], top_p=p)
        _check_alike(ops, x[:5], u[:5], tok, lp, 32, top_p=p)
