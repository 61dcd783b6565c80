"""Shared-prefix attention on the GPU where scores rise from tile to tile and blocks have many tiles, against its definition
in 64 bits.

Tolerance, before any run, in terms of A = sum p |v|: the output's rounding, 2^-11 of it and half of fp16's finest step,
and what fp32 scores and exponents leave, stated with the test."""
import math

import pytest
import torch

from test_generation_ops_gpu import _gen, _prefix_state, ops  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def _check(out, qkv, kp, vp, kc, vc, P, lens, H, kv, part):
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k = torch.cat([kp[:P], kc[b, :n]]).double().view(P + n, kv, 64)
        v = torch.cat([vp[:P], vc[b, :n]]).double().view(P + n, kv, 64)
        q = qkv[b, :H * 64].double().view(kv, H // kv, 64)
        w = torch.softmax(torch.einsum("hgd,phd->hgp", q, k) / 8.0, dim=-1)
        o, a = torch.einsum("hgp,phd->hgd", w, v), torch.einsum("hgp,phd->hgd", w, v.abs())
        err = (out[b].double().view(kv, H // kv, 64) - o).abs()
        tol = 2 ** -11 * o.abs() + part * a + 2 ** -25
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))


@pytest.mark.parametrize("B,H,kv,P,lens", [
    (70, 16, 16, 6000, [3] * 70),                       # 64 and 6 rows a tile, five tiles a block
    (8, 64, 8, 20000, [2500, 1, 0, 129, 1300, 640, 2, 2000]),  # 64 rows; own keys as products, two tiles an item
    (6, 16, 4, 30000, [1, 300, 5, 0, 129, 64]),         # 24 rows
    (3, 40, 8, 20000, [5, 129, 0]),                     # 15
])
@pytest.mark.parametrize("top", [4.0, 15.0, 40.0, -40.0, 150.0])
def test_scores_that_rise_and_fall(ops, B, H, kv, P, lens, top):  # noqa: F811
    """Scores that rise over five tiles and fall back, by less than what may pass the reference, by more, and by so much
    that all before is lost. Scores reach 1200, which leaves 4 2^-23 1200 / 8 = 2^-13.8 of an exponential."""
    S, period = max(lens), 640
    qkv, kp, vp, kc, vc, n = _prefix_state(B, H, kv, P, S, lens, seed=41 + B)
    q = qkv[:, :H * 64].view(B, H, 64)
    q[:, :, 0] = (4.0 + q[:, :, 0].abs()).clamp(max=8.0)
    saw = lambda m: (torch.arange(m, device="cuda") % period).half()[:, None] * (top / period)  # noqa: E731
    kp[:P].view(P, kv, 64)[:, :, 0] = saw(P)
    for b, m in enumerate(lens):
        if m > 1:
            kc[b, :m - 1].view(m - 1, kv, 64)[:, :, 0] = saw(m - 1)
    qkv[:, H * 64:(H + kv) * 64].view(B, kv, 64)[:, :, 0] = top / 2
    out = ops.attn_decode_prefix(qkv, kp, vp, P, kc, vc, n, H, 64, kv_heads=kv, max_len=S)
    _check(out, qkv, kp, vp, kc, vc, P, lens, H, kv, 2 ** -13)


# Scores and exponents in fp32, and what two fp16 numbers leave of a probability (2^-22 of it, and 2^-43 of the row's largest
# where it is far below that). A score of q.k = 40, the sum of whose 64 products may lose 2^-23 of it in each of four
# steps, is off by 2^-17 relative in its exponential (40 2^-21 / 8); the rest adds less than as much again.
@pytest.mark.parametrize("B,H,kv,P,lens", [
    (4, 4, 4, 200, [64, 3, 0, 20]), (16, 16, 16, 1791, [1 + 16 * i for i in range(16)]), (9, 32, 8, 2000, [300] * 9),
    (21, 6, 2, 1500, [7] * 21), (2, 16, 1, 700, [500, 90]), (3, 64, 1, 300, [5, 0, 131]), (2, 2, 2, 0, [2000, 1])])
def test_probabilities_are_held_in_32_bits(ops, B, H, kv, P, lens):  # noqa: F811
    S = max(lens)
    st = _prefix_state(B, H, kv, P, S, lens, seed=31 + B)
    out = ops.attn_decode_prefix(*st[:3], P, *st[3:], H, 64, kv_heads=kv, max_len=S)
    _check(out, *st[:5], P, lens, H, kv, 2 ** -16)


@pytest.mark.parametrize("B,H,kv,P", [(4, 4, 4, 300), (20, 16, 16, 128), (3, 16, 2, 500), (1, 64, 1, 129), (5, 6, 2, 1000)])
def test_one_key_far_above_the_rest(ops, B, H, kv, P):  # noqa: F811
    """A key that outweighs every other by 2^16 to 2^20, but whose value is zero: the output is made of the others. Of each of
    those two fp16 numbers leave 2^-22, and 2^-43 of the largest (half of fp16's finest step, 2^-25, 2^-11 times as
    fine, against 2^7)."""
    lens = [1 + b % 3 for b in range(B)]
    qkv, kp, vp, kc, vc, n = _prefix_state(B, H, kv, P, 3, lens, seed=51 + B)
    q = qkv[:, :H * 64].view(B, H, 64)
    q[:] = 0.0
    q[:, :, 0] = 8.0
    kp[:P].view(P, kv, 64)[:, :, 0] = torch.rand(P, kv, device="cuda", generator=_gen(P)).half() / 4
    kp[P // 2].view(kv, 64)[:, 0] = torch.linspace(16, 20, kv, device="cuda") * math.log(2)
    vp[:P] = 500 + 500 * torch.rand(P, kv * 64, device="cuda", generator=_gen(52)).half()
    vp[P // 2] = 0.0
    out = ops.attn_decode_prefix(qkv, kp, vp, P, kc, vc, n, H, 64, kv_heads=kv, max_len=3)
    _check(out, qkv, kp, vp, kc, vc, P, lens, H, kv, 2 ** -16)
