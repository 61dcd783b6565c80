"""Shared-prefix attention on the GPU where scores rise from tile to tile and blocks have many tiles, against its definition
in 64 bits.

Tolerance, before any run, in terms of A = sum p |v|: the output's rounding, 2^-11 of it and half of fp16's finest step,
and what fp32 scores and exponents leave, stated with the test."""
import pytest
import torch

from test_generation_ops_gpu import _prefix_state, ops  # noqa: F401 (a fixture)

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
