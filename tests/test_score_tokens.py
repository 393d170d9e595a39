"""score_tokens on the CPU: the product and the log probabilities are stood in for by torch's."""
import copy

import pytest
import torch

from promoe_b200 import hf_fused


class StandIn:
    def __init__(self, weight, bias=None, activation=None, out_dtype=None):
        self.weight, self.bias, self.out_dtype, (self.N, self.K) = weight.detach(), bias, out_dtype, weight.shape

    def __call__(self, x, residual=None, out=None):
        y = x.float() @ self.weight.float().T
        y = y if self.bias is None else y + self.bias.float()
        if out is None:
            return y.to(self.out_dtype)
        return out.copy_(y)


def logprobs(logits, targets, top_n=0, out=None):
    lp = torch.log_softmax(logits.double(), -1)
    logp, entropy, ids, best = out
    logp.copy_(torch.where(targets < 0, 0.0, lp.gather(1, targets.clamp_min(0)[:, None])[:, 0]))
    entropy.copy_(-(lp.exp() * lp).sum(-1))
    v, i = lp.topk(top_n, -1)
    ids.copy_(i)
    best.copy_(v)
    return out


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(hf_fused.ops, "Linear", StandIn)
    monkeypatch.setattr(hf_fused.ops, "token_logprobs", logprobs)


def qwen(**kw):
    from transformers.models.qwen2.configuration_qwen2 import Qwen2Config
    from transformers.models.qwen2.modeling_qwen2 import Qwen2ForCausalLM
    torch.manual_seed(0)
    return Qwen2ForCausalLM(Qwen2Config(vocab_size=97, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4,
                                        num_key_value_heads=2, max_position_embeddings=64, tie_word_embeddings=False, **kw)).eval()


def gpt2():
    """Positions are learned here: they have to be counted from a text's own start."""
    from transformers.models.gpt2.configuration_gpt2 import GPT2Config
    from transformers.models.gpt2.modeling_gpt2 import GPT2LMHeadModel
    torch.manual_seed(1)
    return GPT2LMHeadModel(GPT2Config(vocab_size=97, n_embd=32, n_layer=2, n_head=4, n_positions=64)).eval()


@pytest.mark.parametrize("make", [qwen, gpt2])
@pytest.mark.parametrize("side", ["left", "right", "both"])
def test_padding_changes_nothing(stand_ins, make, side):
    model = make()
    texts = [torch.randint(0, 97, (n,), generator=torch.Generator().manual_seed(n)) for n in (9, 6, 1, 2)]
    S = 12
    ids, mask = torch.full((4, S), 5), torch.zeros(4, S, dtype=torch.long)
    first = [S - len(t) if side == "left" else 0 if side == "right" else (S - len(t)) // 2 for t in texts]
    for b, (t, f) in enumerate(zip(texts, first)):
        ids[b, f:f + len(t)], mask[b, f:f + len(t)] = t, 1
    got = hf_fused.score_tokens(model, ids, mask, top_n=2)
    for b, (t, f) in enumerate(zip(texts, first)):
        alone = hf_fused.score_tokens(model, t[None], top_n=2)
        here = slice(f, f + len(t) - 1)
        for k in ("logp", "entropy", "top_logp"):
            torch.testing.assert_close(got[k][b, here], alone[k][0], rtol=1e-4, atol=1e-5)
        outside = torch.ones(S - 1, dtype=torch.bool)
        outside[here] = False
        assert bool((got["logp"][b, outside] == 0).all())  # nothing is scored from or to a padding position
    with pytest.raises(ValueError):
        hf_fused.score_tokens(model, ids, mask[:, :-1])


@pytest.mark.parametrize("make", [qwen, gpt2])
def test_no_keys_and_values_are_kept(stand_ins, make):
    model = make()
    out = []
    model.base_model.register_forward_hook(lambda m, args, kwargs, o: out.append((kwargs.get("use_cache"), o.past_key_values)), with_kwargs=True)
    hf_fused.score_tokens(model, torch.arange(8)[None])
    assert out and all(o == (False, None) for o in out)


def change(model, f):
    """The model with f between its vocabulary projection and its logits."""
    own = type(model).forward

    class Changed(type(model)):
        def forward(self, input_ids=None, attention_mask=None, position_ids=None, use_cache=None, logits_to_keep=0, **kw):
            out = own(self, input_ids=input_ids, attention_mask=attention_mask, position_ids=position_ids, use_cache=use_cache,
                      logits_to_keep=logits_to_keep, **kw)
            out.logits = f(out.logits)
            return out
    model.__class__ = Changed
    return model


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_models_that_change_their_logits_are_refused(stand_ins, dtype):
    ids = torch.arange(10)[None]
    mask = torch.ones_like(ids)
    mask[:, :3] = 0
    hf_fused.score_tokens(change(qwen().to(dtype), lambda l: l), ids, mask)
    for f in (lambda l: l * 0.97, lambda l: l / 1.5, lambda l: 0.5 * torch.tanh(l / 0.5), lambda l: torch.log_softmax(l, -1), lambda l: l + 0.1,
              lambda l: l[..., :-1], lambda l: l.masked_fill(torch.arange(97) > 90, -float("inf"))):
        with pytest.raises(ValueError):
            hf_fused.score_tokens(change(qwen().to(dtype), f), ids, mask)


def test_an_adapter_on_the_vocabulary_projection_is_refused(stand_ins):
    class Adapter(torch.nn.Module):
        def __init__(self, base):
            super().__init__()
            self.base = base
            self.a, self.b = torch.randn(2, 32), torch.randn(97, 2) * 0.1
        weight, bias = property(lambda self: self.base.weight), None

        def forward(self, x):
            return self.base(x) + x @ self.a.T @ self.b.T
    model = qwen()
    model.lm_head = Adapter(model.lm_head)
    with pytest.raises(ValueError):
        hf_fused.score_tokens(model, torch.arange(8)[None])


def test_a_model_that_gives_all_its_logits_or_has_another_trunk(stand_ins):
    model, ids = qwen(), torch.randint(0, 97, (2, 9))
    want = hf_fused.score_tokens(model, ids, top_n=2)
    own = type(model).forward

    class All(type(model)):
        def forward(self, input_ids=None, attention_mask=None, use_cache=None):
            out = own(self, input_ids=input_ids, attention_mask=attention_mask, use_cache=use_cache)
            out.logits = out.logits * self.factor
            return out
    model.__class__, model.factor = All, 1.0
    got = hf_fused.score_tokens(model, ids, top_n=2)
    for k in want:
        torch.testing.assert_close(got[k], want[k])
    model.factor = 0.9
    with pytest.raises(ValueError):
        hf_fused.score_tokens(model, ids)

    class Twice(type(model)):
        def forward(self, input_ids=None, attention_mask=None, use_cache=None):
            self.model(input_ids)
            return own(self, input_ids=input_ids)
    model.__class__ = Twice
    with pytest.raises(ValueError):
        hf_fused.score_tokens(model, ids)
    assert not model.model._forward_hooks


def test_a_model_that_counts_its_kept_logits(stand_ins):
    """logits_to_keep as a number of last positions, as all models know it."""
    model, ids = qwen(), torch.randint(0, 97, (2, 9))
    want = hf_fused.score_tokens(model, ids)
    own = type(model).forward

    class Counts(type(model)):
        def forward(self, input_ids=None, attention_mask=None, use_cache=None, logits_to_keep=0):
            assert isinstance(logits_to_keep, int)
            out = own(self, input_ids=input_ids, attention_mask=attention_mask, use_cache=use_cache)
            out.logits = out.logits[:, -logits_to_keep:]
            return out
    model.__class__ = Counts
    for k, v in hf_fused.score_tokens(model, ids).items():
        torch.testing.assert_close(v, want[k])
    assert hf_fused.score_tokens(model, ids[:, :1])["logp"].shape == (2, 0)
