"""Generation from one prompt and distillation of a student, run as a user strings them together: completions drawn from
a teacher, its top logits over them, a student's loss and gradients, one optimizer update. Against the oracle (the
reference decoder restated, fp16 autocast) where numbers are compared, with the whole-model tolerances of the other
tests: logits 5e-3 (as incremental decoding), loss 1e-3 relative, gradients 1e-2."""
from functools import partial

import numpy as np
import pytest
import torch

from conftest import rel_err
from oracle import jishui_ref as oracle
from test_model_gpu import SMALL, _batch, _pair

pytestmark = pytest.mark.gpu


def _pairs(**kw):
    from midstream_llm_b200.config import ModelConfig
    return _pair(ModelConfig(**dict(SMALL, **kw)))


def _ref_logits(ref, seqs):
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        return torch.stack([ref(torch.tensor([s], device="cuda"))[0, -1].float() for s in seqs])


@pytest.mark.parametrize("kw,n,P", [
    (dict(), 1, 1), (dict(), 5, 300), (dict(), 20, 257),
    (dict(norm_type="layernorm", norm_bias=True, hidden_size=192, num_attention_heads=3, num_key_value_heads=3,
          intermediate_size=320), 9, 40)])
def test_every_step_has_the_logits_of_the_whole_context(kw, n, P):
    """The logits of each completion at each step are those of its whole context, eager and replayed steps alike."""
    from midstream_llm_b200.decode import PromptSampler
    ref, mine = _pairs(**kw)
    rng = np.random.default_rng(0)
    prompt = rng.integers(3, mine.config.vocab_size, size=P).tolist()
    s = PromptSampler(mine, n, 6)
    s.uniforms.uniform_(generator=torch.Generator(device="cuda").manual_seed(1))
    for (_, buf), v in zip(s.settings.items(), (1.0, 0, 1.0, 0.0)):
        buf.fill_(v)
    with torch.no_grad():
        s._start(prompt, -1)
        seqs = [list(prompt) for _ in range(n)]
        for step in range(5):
            want = _ref_logits(ref, seqs)
            assert rel_err(s.logits, want) < 5e-3, (step, rel_err(s.logits, want))
            if step == 0:
                s._draw()
            drawn = s.tokens[step].tolist()
            for q, t in zip(seqs, drawn):
                q.append(t)
            s._advance()
    assert s._graph is not None


def test_completions_repeat_and_follow_the_settings():
    from midstream_llm_b200 import generate
    _, mine = _pairs()
    prompt = list(range(10, 60))
    u = torch.rand(12, 7, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    a = generate(mine, prompt, n=7, max_new_tokens=12, top_p=0.9, uniforms=u)
    b = generate(mine, prompt, n=7, max_new_tokens=12, top_p=0.9, uniforms=u)  # all steps replayed
    assert a.tokens.shape == (7, 12) and a.lengths == [12] * 7
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.logprobs, b.logprobs)
    assert bool((a.logprobs <= 0).all()) and len({tuple(s) for s in a.sequences()}) > 1
    greedy = generate(mine, prompt, n=7, max_new_tokens=12, temperature=0.0)
    assert len({tuple(s) for s in greedy.sequences()}) == 1 and bool((greedy.logprobs == 0).all())
    # settings of their own for every completion, in the same captured step
    mixed = generate(mine, prompt, n=7, max_new_tokens=12, temperature=[0, 1, 0, 1, 0, 1, 0], top_k=[0, 5, 0, 1, 0, 0, 0],
                     uniforms=u)
    for r in (0, 2, 3, 4, 6):
        assert torch.equal(mixed.tokens[r], greedy.tokens[r])
    seeded = [generate(mine, prompt, n=7, max_new_tokens=12, generator=torch.Generator(device="cuda").manual_seed(3)).tokens
              for _ in range(2)]
    assert torch.equal(*seeded)


def test_another_prompt_weights_and_the_end_token():
    from midstream_llm_b200 import generate
    ref, mine = _pairs()
    u = torch.rand(40, 6, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    first = generate(mine, range(5, 50), n=6, max_new_tokens=40, uniforms=u)
    other = generate(mine, range(5, 90), n=6, max_new_tokens=40, uniforms=u)
    assert not torch.equal(first.tokens, other.tokens)
    assert torch.equal(generate(mine, range(5, 50), n=6, max_new_tokens=40, uniforms=u).tokens, first.tokens)
    # a token that some completion drew in the middle ends that one and no other
    end = int(first.tokens[2, 7])
    cut = generate(mine, range(5, 50), n=6, max_new_tokens=40, uniforms=u, eos_token_id=end)
    for r, (row, full) in enumerate(zip(cut.sequences(), first.tokens.tolist())):
        want = full[:full.index(end) + 1] if end in full else full
        assert row == want, r
    n = cut.lengths[2]
    assert bool((cut.tokens[2, n:] == end).all()) and bool((cut.logprobs[2, n:] == 0).all())
    # changed weights take effect in replayed steps too
    with torch.no_grad():
        mine.layers[0].mlp.down_proj.weight.mul_(1.5)
    assert not torch.equal(generate(mine, range(5, 50), n=6, max_new_tokens=40, uniforms=u).tokens, first.tokens)


def test_generation_refusals():
    from midstream_llm_b200 import generate
    from midstream_llm_b200.decode import PromptSampler
    _, mine = _pairs()
    with pytest.raises(ValueError, match="empty prompt"):
        generate(mine, [], n=2, max_new_tokens=4)
    with pytest.raises(ValueError, match="exceed"):
        generate(mine, [5] * 1021, n=2, max_new_tokens=4)
    with pytest.raises(ValueError, match="uniforms"):
        generate(mine, [5], n=2, max_new_tokens=4, uniforms=torch.zeros(3, 2, device="cuda"))
    with pytest.raises(ValueError, match="positive"):
        PromptSampler(mine, 0, 4)
    with pytest.raises(ValueError, match="context"):
        PromptSampler(mine, 1, 4, max_len=4096)
    with torch.no_grad():
        mine.norm.weight[0] = float("nan")
    with pytest.raises(FloatingPointError, match="non-finite"):
        generate(mine, [5, 6], n=2, max_new_tokens=4)


def _ref_distill(ref, x, y, ids, t, tau, alpha):
    with torch.autocast("cuda", dtype=torch.float16):
        z = ref(x).float()
    keep = (y != -100).float()
    used = ids >= 0
    lp = torch.where(used, t.float() / tau, torch.full_like(t, -torch.inf, dtype=torch.float32)).log_softmax(-1)
    lq = (z / tau).log_softmax(-1).gather(-1, ids.clamp(min=0))
    kl = torch.where(used, lp.exp() * (lp - lq), torch.zeros_like(lq)).sum(-1)
    ce = -z.log_softmax(-1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
    return ((alpha * tau ** 2 * kl + (1 - alpha) * ce) * keep).sum() / keep.sum()


@pytest.mark.parametrize("B,T,K,tau,alpha", [(2, 256, 16, 1.0, 1.0), (2, 256, 8, 2.0, 0.5), (3, 100, 32, 1.0, 0.3),
                                             (1, 300, 4, 1.7, 0.9)])
def test_distillation_loss_and_gradients(B, T, K, tau, alpha):
    ref, mine = _pairs()
    _, teacher = _pairs(num_hidden_layers=1, hidden_size=192, num_attention_heads=3, num_key_value_heads=3, intermediate_size=320)
    with torch.no_grad():  # a teacher with preferences
        teacher.embed_tokens.weight.mul_(8)
    x, y = _batch(mine.config, B, T, 1)
    y = y.clone()  # with one row, x and y are views of the same tokens
    y[:, -3:] = -100
    t, ids = teacher.top_logits(x, K)
    assert t.shape == ids.shape == (B, T, K)
    with torch.no_grad():
        full = teacher(x)
    assert torch.equal(t, full.gather(-1, ids)) and torch.equal(t[..., 0], full.amax(-1))
    ids[0, 5:20, K // 2:] = -1
    loss = mine.distill_loss(x, y, ids, t, temperature=tau, alpha=alpha)
    want = _ref_distill(ref, x, y, ids, t, tau, alpha)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-3 * abs(float(want.detach()))
    with torch.no_grad():
        again = mine.distill_loss(x, y, ids, t, temperature=tau, alpha=alpha)
    assert abs(float(again) - float(loss.detach())) < 1e-6 * abs(float(again))
    (loss * 1024).backward()
    (want * 1024).backward()
    for (name, a), (_, b) in zip(mine.named_parameters(), ref.named_parameters()):
        assert rel_err(a.grad, b.grad) < 1e-2, (name, rel_err(a.grad, b.grad))


def test_from_completions_to_a_students_update():
    """The whole run: completions of the teacher, its top logits over prompt and completion, two updates of a student."""
    from midstream_llm_b200 import AdamW, GradScaler, distillation_loss, generate, train_update
    _, teacher = _pairs()
    _, student = _pairs(num_hidden_layers=1)
    prompt = list(range(100, 140))
    c = generate(teacher, prompt, n=8, max_new_tokens=30, temperature=0.9, top_p=0.95, eos_token_id=7,
                 generator=torch.Generator(device="cuda").manual_seed(5))
    rows = torch.tensor([prompt + s + [7] * (31 - len(s)) for s in c.sequences()], device="cuda")
    x, y = rows[:, :-1].contiguous(), rows[:, 1:].clone()
    for r, n in enumerate(c.lengths):
        y[r, len(prompt) + n - 1:] = -100
    t, ids = teacher.top_logits(x, 20)
    opt = AdamW(student.parameters(), lr=1e-3, betas=(0.9, 0.95), eps=1e-5, weight_decay=0.1, fused=True)
    scaler = GradScaler("cuda", init_scale=1024.0)
    before = student.embed_tokens.weight.detach().clone()
    loss_fn = partial(distillation_loss, temperature=2.0, alpha=0.7)
    with torch.no_grad():
        start = float(loss_fn(student, x, y, ids, t))
    for _ in range(2):
        r = train_update(student, opt, scaler, lambda: [(x, y, ids, t)], 1, 1.0, 1e-3, loss_fn=loss_fn)
        assert r["attempts"] == 1 and np.isfinite(r["loss"])
    assert not torch.equal(before, student.embed_tokens.weight)
    assert abs(start - float(loss_fn(student, x, y, ids, t).detach())) > 0
    # the plain loss still runs through the same function
    r = train_update(student, opt, scaler, lambda: [(x, y)], 1, 1.0, 1e-3)
    assert np.isfinite(r["loss"])


def test_distill_loss_refusals():
    _, mine = _pairs()
    x, y = _batch(mine.config, 1, 64, 1)
    t, ids = mine.top_logits(x, 4)
    with pytest.raises(ValueError, match="must be"):
        mine.distill_loss(x, y, ids[:, :32], t)
    with pytest.raises(ValueError, match="differ in shape"):
        mine.distill_loss(x, y[:, :32], ids, t)
    with pytest.raises(ValueError, match="k must be"):
        mine.top_logits(x, 0)
    with pytest.raises(ValueError, match="context"):
        mine.top_logits(torch.zeros(1, 2000, device="cuda", dtype=torch.long), 4)


def test_generate_refuses_settings_without_a_meaning():
    from midstream_llm_b200 import generate
    _, mine = _pairs()
    for bad in (dict(temperature=-1.0), dict(temperature=[1.0, -0.5]), dict(top_p=float("nan")), dict(min_p=[0.0, float("nan")])):
        with pytest.raises(ValueError, match="bad"):
            generate(mine, [1, 2, 3], n=2, max_new_tokens=4, **bad)


@pytest.mark.parametrize("distill", [False, True])
def test_a_second_backward_of_the_same_loss_is_refused(distill):
    """The first one leaves the logits' gradient in their place."""
    _, mine = _pairs()
    x, y = _batch(mine.config, 1, 256, 1)
    t, ids = mine.top_logits(x, 8)
    loss = mine.distill_loss(x, y, ids, t, temperature=2.0) if distill else mine.loss(x, y)
    loss.backward(retain_graph=True)
    first = mine.embed_tokens.weight.grad.clone()
    with pytest.raises(RuntimeError, match="backward"):
        loss.backward()
    assert torch.equal(mine.embed_tokens.weight.grad, first)


@pytest.mark.parametrize("bad", [[5, -1], [5, 1 << 30]])
def test_generate_refuses_tokens_outside_the_vocabulary(bad):
    from midstream_llm_b200 import _lib, generate
    _, mine = _pairs()
    _lib.device_status()
    with pytest.raises(ValueError, match="vocabulary"):
        generate(mine, bad, n=2, max_new_tokens=4)
    with pytest.raises(ValueError, match="vocabulary"):
        generate(mine, [5, mine.config.vocab_size], n=2, max_new_tokens=4)
    assert _lib.device_status() == 0


def test_non_finite_logits_leave_no_status_behind():
    """Rows without a token to draw end the call with an error; what is fed meanwhile is a token of the vocabulary."""
    from midstream_llm_b200 import _lib, generate
    _, mine = _pairs()
    with torch.no_grad():
        mine.norm.weight[0] = float("nan")
    for end in (None, 0, 7):
        _lib.device_status()
        with pytest.raises(FloatingPointError, match="non-finite"):
            generate(mine, [5, 6], n=2, max_new_tokens=6, eos_token_id=end)
        assert _lib.device_status() == 0
