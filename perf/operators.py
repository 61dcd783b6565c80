"""Workloads of the generation and distillation operators, each in a plain form and through the framework.

Four operators that a distillation run strings together: completions are drawn from a model by decoding many
sequences that share one prompt (`attn_decode_prefix`) and sampling their next tokens (`sample`), the teacher's
top logits at every position are recorded (`top_logits`), and a student learns from them (`distill_fwd`,
`distill_bwd`).

`own` selects what `run` calls: elementary torch operations, or midstream_llm_b200.ops. Every size is one
of this repository's configurations (vocabularies 24000, 32000, 32768; 4, 11 or 16 heads of 64; 16 x 1024 tokens
a step) or a generic one.
"""
import math
import random

import torch

own = False

F16, F32, F64, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
D = 64  # head width of every configuration
IGNORE = -100


def listed():
    return [
        # One decode step of four completions of a short prompt on the tiny model: all latency.
        dict(name="prefix_tiny", op="prefix", B=4, H=4, kv=4, P=200, S=64, idle=0),
        # Sixteen completions of one prompt on the 200M model, near the end of its 2048-token context.
        dict(name="prefix_samples", op="prefix", B=16, H=16, kv=16, P=1791, S=257, idle=0),
        # A serving batch behind a long common document, a few of its slots idle.
        dict(name="prefix_long", op="prefix", B=64, H=16, kv=16, P=32749, S=1000, idle=3),
        # The same with four query heads on each key / value head.
        dict(name="prefix_grouped", op="prefix", B=96, H=32, kv=8, P=8191, S=500, idle=0),
        # The next token of a single generation, with the usual filters.
        dict(name="sample_one", op="sample", R=1, V=32000, filters="all"),
        # A serving batch whose requests each bring their own settings.
        dict(name="sample_batch", op="sample", R=64, V=32768, filters="mixed"),
        # Many completions at once under nucleus sampling, a vocabulary that is no multiple of anything.
        dict(name="sample_nucleus", op="sample", R=1024, V=50257, filters="p"),
        # The teacher's top logits of one short text.
        dict(name="top_text", op="top", R=200, V=24000, K=16),
        # The teacher's top logits of one training micro-batch (16 x 1024 tokens).
        dict(name="top_batch", op="top", R=16384, V=32000, K=64),
        # Loss and logit gradient of a short batch at temperature 1, soft targets only.
        dict(name="distill_short", op="distill", R=1000, V=24000, K=16, tau=1.0, alpha=1.0, grad=True),
        # A validation pass: the loss alone over one micro-batch, soft and hard targets mixed.
        dict(name="distill_loss", op="distill", R=16384, V=32000, K=64, tau=2.0, alpha=0.7, grad=False),
        # A training step's loss and logit gradient over one micro-batch.
        dict(name="distill_step", op="distill", R=16384, V=32000, K=64, tau=2.0, alpha=0.7, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefix", "sample", "top", "distill"])
    if op == "prefix":
        while True:
            kv = rng.choice([1, 2, 4, 8, 11, 16])
            G = rng.choice([1, 1, 2, 4, 8])
            c = dict(op=op, B=_log_int(rng, 1, 200), H=kv * G, kv=kv, P=_log_int(rng, 1, 40000), S=_log_int(rng, 1, 1500),
                     idle=0)
            c["idle"] = rng.choice([0, 0, c["B"] // 4])
            if c["H"] <= 32 and c["B"] * c["H"] * (c["P"] + c["S"]) <= 64 * 16 * 33000 and c["B"] * kv * c["S"] <= 64 * 16 * 1000:
                return c
    V = rng.choice([24000, 32000, 32768, _log_int(rng, 300, 70000)])
    if op == "sample":
        R = _log_int(rng, 1, 1024 * 50257 // V)
        return dict(op=op, R=R, V=V, filters=rng.choice(["all", "mixed", "k", "p", "min_p", "none", "greedy"]))
    if op == "top":
        return dict(op=op, R=_log_int(rng, 1, 16384 * 32000 // max(V, 32000)), V=V, K=_log_int(rng, 1, 256))
    return dict(op=op, R=_log_int(rng, 1, 16384 * 32000 // max(V, 32000)), V=V, K=_log_int(rng, 1, 128),
                tau=rng.choice([1.0, 1.5, 2.0, 4.0]), alpha=rng.choice([1.0, 0.7, 0.5]), grad=rng.choice([True, True, False]))


def _lengths(case):
    """Tokens each sequence has of its own, the new one included: ragged, 0 for an idle slot."""
    r = random.Random(case["B"] * 7919 + case["S"])
    n = [r.randint(1, case["S"]) for _ in range(case["B"])]
    n[r.randrange(case["B"])] = case["S"]
    for b in r.sample(range(case["B"]), case["idle"]):
        n[b] = 0
    return n


def _logits(R, V, g):
    """fp16 logits as a trained decoder gives them: a spread of a few units and some tokens that stand out. The row
    stride is a multiple of 8, as the head's output has it."""
    x = torch.randn(R, -(-V // 8) * 8, device="cuda", generator=g) * 2.2
    hot = torch.randint(0, V, (R, 12), device="cuda", generator=g)
    x.scatter_add_(1, hot, torch.rand(R, 12, device="cuda", generator=g) * 9.0)
    return x.half()[:, :V]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "prefix":
        B, H, kv, P, S = (case[k] for k in ("B", "H", "kv", "P", "S"))
        s["qkv"] = torch.randn(B, (H + 2 * kv) * D, device="cuda", generator=g).half()
        # The caches are longer than what is filled of them.
        s["kp"] = torch.randn(P + 21, kv * D, device="cuda", generator=g).half()
        s["vp"] = torch.randn(P + 21, kv * D, device="cuda", generator=g).half()
        s["kc"] = torch.randn(B, S + 5, kv * D, device="cuda", generator=g).half()
        s["vc"] = torch.randn(B, S + 5, kv * D, device="cuda", generator=g).half()
        s["lens"] = torch.tensor(_lengths(case), dtype=I32, device="cuda")
        if own:
            from midstream_llm_b200 import ops
            n = ops.attn_decode_prefix_workspace_bytes(B, H, kv, P, S)
            s["ws"] = torch.empty(n // 4 + 4, device="cuda", dtype=F32)
        return s
    R, V = case["R"], case["V"]
    s["x"] = _logits(R, V, g)
    if case["op"] == "sample":
        s["u"] = torch.rand(R, device="cuda", generator=g)
        f = case["filters"]
        s["set"] = dict(temperature=0.8, top_k=50 if f in ("all", "k") else 0, top_p=0.95 if f in ("all", "p") else 1.0,
                        min_p=0.02 if f in ("all", "min_p") else 0.0)
        if f == "greedy":
            s["set"]["temperature"] = 0.0
        if f == "mixed":
            pick = lambda v, t: torch.tensor(v, device="cuda", dtype=t)[  # noqa: E731
                torch.randint(0, len(v), (R,), device="cuda", generator=g)]
            s["set"] = dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.3], F32), top_k=pick([0, 1, 20, 50, 400], I32),
                            top_p=pick([1.0, 0.8, 0.9, 0.95], F32), min_p=pick([0.0, 0.0, 0.05, 0.1], F32))
    elif case["op"] == "distill":
        K = case["K"]
        teacher = _logits(R, V, g)
        # The teacher's logits at distinct tokens, most likely first; every seventh position has fewer of them.
        n = max(1, min(K, V))
        top = torch.cat([t.float().topk(n, dim=1)[1] for t in teacher.split(4096)])
        s["ids"] = torch.full((R, K), -1, device="cuda", dtype=I64)
        s["ids"][:, :n] = top
        s["t"] = torch.zeros(R, K, device="cuda", dtype=F16)
        s["t"][:, :n] = teacher.gather(1, top)
        s["ids"][::7, (K + 1) // 2:] = -1
        s["y"] = torch.randint(0, V, (R,), device="cuda", generator=g)
        s["y"][3::50] = IGNORE  # padding
        s["g"] = torch.full((1,), 65536.0, device="cuda")  # the loss scale
        if case["grad"]:
            s["dx"] = torch.empty(R, s["x"].stride(0), device="cuda", dtype=F16)[:, :V]
    return s


# ---------------------------------------------------------------- the passes
def run(s):
    return {"prefix": _run_prefix, "sample": _run_sample, "top": _run_top, "distill": _run_distill}[s["op"]](s)


def _run_prefix(s):
    B, H, kv, P = s["B"], s["H"], s["kv"], s["P"]
    if own:
        from midstream_llm_b200 import ops
        o = ops.attn_decode_prefix(s["qkv"], s["kp"], s["vp"], P, s["kc"], s["vc"], s["lens"], H, D, kv_heads=kv,
                                   max_len=s["S"], workspace=s["ws"])
        return {"out": o, "k": s["kc"], "v": s["vc"]}
    G, lens = H // kv, s["lens"].long()
    live = lens > 0
    rows = torch.arange(B, device="cuda")[live]
    at = (lens - 1)[live]
    s["kc"][rows, at] = s["qkv"][rows, H * D:(H + kv) * D]
    s["vc"][rows, at] = s["qkv"][rows, (H + kv) * D:]
    q = s["qkv"][:, :H * D].float().view(B, kv, G, D) / math.sqrt(D)
    S = s["S"]
    kp, vp = (s[n][:P].float().view(P, kv, D) for n in ("kp", "vp"))
    kc, vc = (s[n][:, :S].float().view(B, S, kv, D) for n in ("kc", "vc"))
    a = torch.einsum("bhgd,phd->bhgp", q, kp)
    b = torch.einsum("bhgd,bshd->bhgs", q, kc)
    b.masked_fill_((torch.arange(S, device="cuda")[None] >= lens[:, None])[:, None, None], float("-inf"))
    w = torch.cat([a, b], dim=-1)
    w = (w - w.amax(-1, keepdim=True)).exp_()
    w /= w.sum(-1, keepdim=True)
    o = torch.einsum("bhgp,phd->bhgd", w[..., :P], vp) + torch.einsum("bhgs,bshd->bhgd", w[..., P:], vc)
    o = o.reshape(B, H * D) * live[:, None]
    return {"out": o.half(), "k": s["kc"], "v": s["vc"]}


def _columns(s, R, dtype):
    return [torch.as_tensor(s["set"][k], device="cuda").to(dtype).expand(R)[:, None]
            for k in ("temperature", "top_k", "top_p", "min_p")]


def _run_sample(s):
    if own:
        from midstream_llm_b200 import ops
        tokens, logp = ops.sample(s["x"], s["u"], **s["set"])
        return {"tokens": tokens, "logp": logp}
    # Near a border one more bit decides which token is drawn: probabilities in 64 bits.
    R, V = s["R"], s["V"]
    T, k, p, m = _columns(s, R, F64)
    x, order = s["x"].double().sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    e = ((x - x[:, :1]) / torch.where(T > 0, T, torch.ones_like(T))).exp()
    rank = torch.arange(V, device="cuda")[None]
    keep = rank < torch.where(T > 0, torch.where(k > 0, k, torch.full_like(k, V)), torch.ones_like(T))
    c = (e * keep).cumsum(1)
    keep &= (c - e < p * c[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= (e >= m) | (rank == 0)
    w = torch.zeros_like(e).scatter_(1, order, e * keep)
    c = w.cumsum(1)
    hit = (c > s["u"].double()[:, None] * c[:, -1:]) & (w > 0)
    tokens = hit.int().argmax(1)
    logp = (w.gather(1, tokens[:, None]) / c[:, -1:]).log()[:, 0]
    return {"tokens": tokens, "logp": logp.float()}


def _run_top(s):
    if own:
        from midstream_llm_b200 import ops
        values, ids = ops.top_logits(s["x"], min(s["K"], s["V"]))
        return {"values": values, "ids": ids}
    vs, ids = [], []
    for x in s["x"].split(2048):
        v, i = x.float().sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
        vs.append(v[:, :s["K"]].half())
        ids.append(i[:, :s["K"]].clone())
    return {"values": torch.cat(vs), "ids": torch.cat(ids)}


def _run_distill(s):
    R, V, tau, alpha = s["R"], s["V"], s["tau"], s["alpha"]
    if own:
        from midstream_llm_b200 import ops
        stats, row_loss = ops.distill_fwd(s["x"], s["ids"], s["t"], s["y"], temperature=tau, alpha=alpha, ignore_index=IGNORE)
        loss = ops.ce_loss(row_loss, s["y"], IGNORE)
        out = {"loss": loss[2], "rows": row_loss}
        if s["grad"]:
            out["dx"] = ops.distill_bwd(s["x"], s["ids"], s["t"], s["y"], stats, s["g"], loss[1:2], temperature=tau,
                                        alpha=alpha, ignore_index=IGNORE, out=s["dx"])
        return out
    count = (s["y"] != IGNORE).sum()
    rows, grads = [], []
    for x16, ids, t, y in zip(*(s[n].split(4096) for n in ("x", "ids", "t", "y"))):
        x = x16.float()
        real = y != IGNORE
        y0 = y.clamp(min=0)[:, None]
        used = ids >= 0
        i0 = ids.clamp(min=0)
        lp = torch.where(used, t.float() / tau, torch.full_like(t, float("-inf"), dtype=F32))
        lp = lp - lp.logsumexp(1, keepdim=True)
        pt = lp.exp()
        lq = x / tau
        lq -= lq.logsumexp(1, keepdim=True)
        kl = torch.where(used, pt * (lp - lq.gather(1, i0)), torch.zeros_like(pt)).sum(1)
        l1 = x - x.logsumexp(1, keepdim=True)
        rows.append((alpha * tau * tau * kl - (1 - alpha) * l1.gather(1, y0)[:, 0]) * real)
        if s["grad"]:
            d = alpha * tau * lq.exp_()
            d.scatter_add_(1, i0, -alpha * tau * pt)
            if alpha < 1:
                d += (1 - alpha) * l1.exp_()
                d.scatter_add_(1, y0, torch.full_like(y0, alpha - 1, dtype=F32))
            grads.append((d * (s["g"] / count) * real[:, None]).half())
    rows = torch.cat(rows)
    out = {"loss": rows.sum() / count, "rows": rows}
    if s["grad"]:
        out["dx"] = torch.cat(grads)
    return out


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"prefix": _exact_prefix, "sample": _exact_sample, "top": _exact_top, "distill": _exact_distill}[case["op"]](s)


def _exact_prefix(s):
    B, H, kv, P = s["B"], s["H"], s["kv"], s["P"]
    G = H // kv
    out = torch.zeros(B, H, D, device="cuda", dtype=F64)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        s["kc"][b, n - 1] = s["qkv"][b, H * D:(H + kv) * D]
        s["vc"][b, n - 1] = s["qkv"][b, (H + kv) * D:]
        for h in range(kv):
            c = slice(h * D, (h + 1) * D)
            k = torch.cat([s["kp"][:P, c], s["kc"][b, :n, c]]).double()
            v = torch.cat([s["vp"][:P, c], s["vc"][b, :n, c]]).double()
            q = s["qkv"][b, h * G * D:(h + 1) * G * D].double().view(G, D)
            out[b, h * G:(h + 1) * G] = torch.softmax(q @ k.T * D ** -0.5, dim=-1) @ v
    return {"out": out.view(B, H * D), "k": s["kc"].double(), "v": s["vc"].double()}


def _exact_sample(s):
    import numpy as np
    R, V = s["R"], s["V"]
    T, k, p, m = (c[:, 0].tolist() for c in _columns(s, R, F64))
    u, x = s["u"].double().cpu().numpy(), s["x"].cpu().numpy().astype(np.float64)
    tokens, logp = [], []
    for r in range(R):
        best = int(x[r].argmax())
        if T[r] <= 0:
            tokens.append(best)
            logp.append(0.0)
            continue
        prob = np.exp((x[r] - x[r, best]) / T[r])
        ranked = np.lexsort((np.arange(V), -x[r]))
        if k[r] > 0:
            ranked = ranked[:int(k[r])]
        if p[r] < 1:  # the fewest tokens that reach p of what top-k left
            above = np.concatenate([[0.0], np.cumsum(prob[ranked])])
            ranked = ranked[:max(1, int(np.searchsorted(above[:-1], p[r] * above[-1], side="left")))]
        ranked = ranked[:max(1, int((prob[ranked] >= m[r]).sum()))]
        ids = np.sort(ranked)
        mass = np.cumsum(prob[ids])
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(ids) - 1)
        tokens.append(int(ids[at]))
        logp.append(math.log(prob[ids[at]] / mass[-1]))
    return {"tokens": torch.tensor(tokens, device="cuda"), "logp": torch.tensor(logp, device="cuda", dtype=F64)}


def _exact_top(s):
    V, K = s["V"], min(s["K"], s["V"])
    ids = []
    back = torch.arange(V - 1, -1, -1, device="cuda")
    for x in s["x"].split(2048):  # one key of value (in units of 2^-24, the finest fp16 step) and place
        key = (x.double() * 2.0 ** 24).long() * (1 << 17) + back
        ids.append(V - 1 - key.topk(K, dim=1)[0].remainder(1 << 17))
    ids = torch.cat(ids)
    return {"values": s["x"].gather(1, ids).double(), "ids": ids}


def _exact_distill(s):
    tau, alpha, n = s["tau"], s["alpha"], int((s["y"] != IGNORE).sum())
    rows, grads = [], []
    for i in range(0, s["R"], 2048):
        x, ids, t, y = (s[k][i:i + 2048] for k in ("x", "ids", "t", "y"))
        r = torch.arange(x.shape[0], device="cuda")
        weight = torch.exp((t.double() - t[:, :1].double()) / tau) * (ids >= 0)
        weight /= weight.sum(1, keepdim=True)
        p = torch.zeros(x.shape[0], s["V"] + 1, device="cuda", dtype=F64).scatter_add_(1, ids % (s["V"] + 1), weight)
        p = p[:, :s["V"]]
        q, q1 = (torch.softmax(x.double() / c, dim=1) for c in (tau, 1.0))
        keep = (y != IGNORE).double()
        kl = torch.where(p > 0, p * (p / q).log(), torch.zeros_like(p)).sum(1)
        hot = y.clamp(min=0)
        rows.append(keep * (alpha * tau ** 2 * kl - (1 - alpha) * q1[r, hot].log()))
        if s["grad"]:
            q1[r, hot] -= 1
            grads.append((alpha * tau * (q - p) + (1 - alpha) * q1) * keep[:, None] * (65536.0 / n))
    rows = torch.cat(rows)
    out = {"loss": rows.sum() / n, "rows": rows}
    if s["grad"]:
        out["dx"] = torch.cat(grads)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "prefix":
        B, H, kv, P = (case[k] for k in ("B", "H", "kv", "P"))
        lens = _lengths(case)
        live = sum(n > 0 for n in lens)
        keys = P + sum(n - 1 for n in lens if n)  # read from the caches
        return {"bytes": 4 * D * kv * keys + 2 * D * (2 * H + 4 * kv) * live + 4 * B,
                "flops": 4 * D * H * (P * live + sum(lens))}
    R, V = case["R"], case["V"]
    if case["op"] == "sample":
        return {"bytes": 2 * R * V + (4 + 8 + 4) * R, "flops": 3 * R * V}
    K = case["K"]
    if case["op"] == "top":
        return {"bytes": 2 * R * V + 10 * R * min(K, V), "flops": R * V}
    b = 2 * R * V + R * (10 * K + 8 + 4)
    if case["grad"]:
        b += 2 * R * V
    return {"bytes": b, "flops": R * V * (12 if case["grad"] else 6)}
