"""score_tokens of an injected model."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def injected():
    from promoe_b200.hf_fused import inject_hf_fused_model
    from tests.test_hf_fused_gpu import tiny_qwen
    model = tiny_qwen()
    cache = inject_hf_fused_model(model, cache_rate=1.0, num_predict_expert_per_layer=0)
    return model.cuda(), cache


def test_a_left_padded_text_scores_as_the_text_alone(lib):
    from promoe_b200.hf_fused import score_tokens
    model, cache = injected()
    g = torch.Generator().manual_seed(3)
    S, lengths = 14, (14, 9, 2, 1)
    ids, mask = torch.full((4, S), 7), torch.zeros(4, S, dtype=torch.long)
    for b, n in enumerate(lengths):
        ids[b, S - n:], mask[b, S - n:] = torch.randint(0, 128, (n,), generator=g), 1
    ids, mask = ids.cuda(), mask.cuda()
    got = score_tokens(model, ids, mask, top_n=2)
    for b, n in enumerate(lengths):
        alone = score_tokens(model, ids[b:b + 1, S - n:], top_n=2)
        # hidden rows in bf16, summed in another order: logits of up to 4 that are off by a few half steps of 2^-8
        assert n == 1 or float((got["logp"][b, S - n:] - alone["logp"][0]).abs().max()) < 8 * 4 * 2.0 ** -8
        assert bool((got["logp"][b, :S - n] == 0).all())
    cache.close()


def test_the_models_own_logits_are_compared(lib):
    from promoe_b200.hf_fused import score_tokens
    model, cache = injected()
    ids = torch.randint(0, 128, (2, 9), device="cuda")
    score_tokens(model, ids)
    own = model.lm_head.forward
    model.lm_head.forward = lambda x: own(x) * 0.95
    with pytest.raises(ValueError):
        score_tokens(model, ids)
    cache.close()
