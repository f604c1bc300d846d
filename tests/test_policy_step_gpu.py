"""The embedding, the log probabilities and the clipping together, as a training step and a decode
loop use them: a policy-gradient step of the drop-in model (UnifiedLM.token_logprobs with
fused_embedding, an entropy bonus, clip_grad_norm_) against the float64 oracle, and
BatchedDecoder.logprobs against the logits that it holds."""
import math

import pytest
import torch

import unifiedlm_c_b200._lib as L
from oracle import memory as O
from unifiedlm_c_b200.clip import clip_grad_norm_
from unifiedlm_c_b200.decode import BatchedDecoder
from unifiedlm_c_b200.model import ModelArgs, UnifiedLM

pytestmark = pytest.mark.gpu
TOL = {"bf16": 1e-2, "fp32": 1e-5}  # the model tests' tolerances


def tiny(seed=0):
    torch.manual_seed(seed)
    model = UnifiedLM(ModelArgs(dim=64, n_layers=2, hidden_dim=140, vocab_size=512, max_seq_len=200))
    with torch.no_grad():
        for layer in model.layers:
            layer.conv.weight.normal_(std=0.5)
            layer.key.bias.normal_(std=0.5)
            layer.val.weight.normal_(std=0.2)
            layer.log_rate.fill_(math.log(0.05))
    return model


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_policy_gradient_step(precision):
    model = tiny()
    sd = {k: v.detach().clone().double() for k, v in model.state_dict().items()}
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 512, (2, 200), generator=gen)
    targets = torch.randint(0, 512, (2, 200), generator=gen)
    targets[1, 150:] = -1  # a shorter sequence
    adv = torch.randn(2, 200, generator=gen)
    model = model.cuda().train().set_precision(precision)
    model.fused_embedding = True
    r = model.token_logprobs(tokens.cuda(), targets.cuda(), top_k=3)
    keep = (targets >= 0).float().cuda()
    loss = -((r.logprobs * adv.cuda() + 0.1 * r.entropy) * keep).sum() / keep.sum()
    loss.backward()

    leaves = {k: v.clone().requires_grad_() for k, v in sd.items() if k != "tok_embeddings.weight"}
    logits, _ = O.lm_forward({**leaves, "tok_embeddings.weight": leaves["output.weight"]}, tokens, form="dense")
    logp = torch.log_softmax(logits, -1)
    ent = -(logp.exp() * logp).sum(-1)
    given = logp.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    k64 = keep.double().cpu()
    want = -((given * adv.double() + 0.1 * ent) * k64).sum() / k64.sum()
    want.backward()
    assert abs(float(loss) - float(want)) <= TOL[precision] * float((given.abs() * adv.abs()).mean())
    grads = {k: p.grad for k, p in model.named_parameters()}
    errs = {k: rel(g, leaves["output.weight" if k == "tok_embeddings.weight" else k].grad) for k, g in grads.items()
            if not k.endswith("log_rate")}  # (the decay's gradient is held to its own bound in the model tests)
    assert max(errs.values()) < TOL[precision], errs

    n = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    before = {k: g.clone() for k, g in grads.items()}
    got = clip_grad_norm_(model.parameters(), 0.5 * n)
    assert abs(float(got) - n) <= 1e-6 * n
    for k, p in model.named_parameters():
        assert torch.allclose(p.grad, before[k] * 0.5, rtol=1e-5, atol=0)
    torch.optim.SGD(model.parameters(), lr=0.1).step()
    assert all(bool(p.isfinite().all()) for p in model.parameters()) and L.device_error() == 0


def test_fused_embedding_gives_the_same_forward():
    model = tiny(3).cuda()
    tokens = torch.randint(0, 512, (2, 50)).cuda()
    plain = model(tokens, tokens)
    loss = model.last_loss
    model.fused_embedding = True
    assert torch.equal(model(tokens, tokens), plain) and torch.equal(model.last_loss, loss)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_decode_logprobs(temperature):
    model = tiny(5)
    dec = BatchedDecoder(model.state_dict(), batch=3, precision="fp32", temperature=temperature, seed=4)
    dec.prepare_graph()
    token = torch.tensor([1, 7, 9])
    for _ in range(4):
        token = dec.feed(token, sample=temperature > 0)
        logp = torch.log_softmax(dec.logits.double(), -1)
        r = dec.logprobs(top_k=5)
        want = logp.gather(1, token.long()[:, None])[:, 0]
        assert r.logprobs.shape == (3,) and bool((r.logprobs - want).abs().max() < 1e-5)
        assert bool((r.entropy - -(logp.exp() * logp).sum(-1)).abs().max() < 1e-5)
        assert torch.equal(r.top_ids, torch.sort(dec.logits, dim=-1, descending=True, stable=True).indices[:, :5])
        other = torch.tensor([0, 5, 511])
        assert torch.allclose(dec.logprobs(other).logprobs.double(), logp.gather(1, other.cuda()[:, None])[:, 0], atol=1e-5)
        if temperature == 0:
            assert torch.equal(r.top_ids[:, 0], token.long())
