"""What the entry points of the operators around the experts refuse, without a GPU: pm_k_route, pm_k_linear and
pm_k_token_logprobs check their arguments before they touch a device."""
import ctypes as C

import pytest

from promoe_b200 import _lib, ops

PTR = 1 << 20  # a 16-byte boundary; never dereferenced


def route(n=0, logits=None, dtype=0, ld=None, ids=None, w=None, **over):
    r = dict(num_expert=64, top_k=6, scoring=0, n_group=1, topk_group=1, group_score=0, norm_topk=0, routed_scale=1.0)
    r.update(over)
    rule = _lib.pm_router(**r)
    _lib.call("pm_k_route", C.byref(rule), logits, dtype, r["num_expert"] if ld is None else ld, n, ids, w, None)


@pytest.mark.parametrize("over", [dict(num_expert=0), dict(num_expert=1025), dict(top_k=0), dict(top_k=33), dict(num_expert=4, top_k=5),
                                  dict(n_group=0), dict(n_group=33, num_expert=66), dict(n_group=5), dict(topk_group=0),
                                  dict(n_group=4, topk_group=5), dict(n_group=16, topk_group=1), dict(scoring=2), dict(scoring=-1),
                                  dict(group_score=2), dict(n=-1), dict(dtype=3), dict(ld=63), dict(n=1), dict(n=1, logits=PTR),
                                  dict(n=1, logits=PTR + 2, ids=PTR, w=PTR), dict(n=1, logits=PTR, ids=PTR + 1, w=PTR),
                                  dict(n=1, logits=PTR, ids=PTR, w=PTR, choice_bias=PTR + 2)])
def test_route_refuses(lib, over):
    with pytest.raises(_lib.PromoeError) as e:
        route(**over)
    assert e.value.code == 1 and "route" in str(e.value)


def test_route_of_no_tokens_is_nothing(lib):
    route()
    with pytest.raises(_lib.PromoeError):
        _lib.call("pm_k_route", None, None, 0, 64, 0, None, None, None)


def linear(**over):
    a = dict(x=PTR, w=PTR, y=PTR, ld_x=64, ld_w=64, ld_residual=32, ld_y=32, M=4, N=32, K=64, dtype=1, out_dtype=1, bias_dtype=0, act=0)
    a.update(over)
    _lib.call("pm_k_linear", C.byref(_lib.pm_linear(**a)), None)


@pytest.mark.parametrize("over", [dict(M=-1), dict(N=0), dict(K=0), dict(dtype=0), dict(dtype=3), dict(out_dtype=2), dict(dtype=2, out_dtype=1),
                                  dict(bias=PTR, bias_dtype=2), dict(act=-1), dict(act=5), dict(ld_x=63), dict(ld_w=63), dict(ld_y=31),
                                  dict(residual=PTR, ld_residual=31), dict(x=None), dict(w=None), dict(y=None), dict(x=PTR + 1),
                                  dict(w=PTR + 1), dict(y=PTR + 1), dict(out_dtype=0, y=PTR + 2), dict(residual=PTR + 1),
                                  dict(bias=PTR + 2, bias_dtype=0), dict(err_flag=PTR + 2), dict(residual=PTR, ld_residual=40),
                                  dict(M=(1 << 30) + 1)])
def test_linear_refuses(lib, over):
    with pytest.raises(_lib.PromoeError) as e:
        linear(**over)
    assert e.value.code == 1 and "linear" in str(e.value)


def test_linear_of_no_rows_is_nothing(lib):
    linear(M=0)
    linear(M=0, x=None, y=None)
    with pytest.raises(_lib.PromoeError):
        _lib.call("pm_k_linear", None, None)


def logprobs(**over):
    a = dict(logits=PTR, dtype=0, ld=1000, rows=4, vocab=1000, targets=PTR, top_n=5, logp=PTR, entropy=PTR, ids=PTR, top=PTR)
    a.update(over)
    _lib.call("pm_k_token_logprobs", *a.values(), None)


@pytest.mark.parametrize("over", [dict(rows=-1), dict(vocab=0), dict(dtype=7), dict(ld=999), dict(top_n=-1), dict(top_n=33),
                                  dict(vocab=4, top_n=5), dict(logits=None), dict(targets=None), dict(ids=None), dict(top=None),
                                  dict(logits=PTR + 2), dict(dtype=1, logits=PTR + 1), dict(targets=PTR + 4), dict(logp=PTR + 2),
                                  dict(entropy=PTR + 1), dict(ids=PTR + 2), dict(top=PTR + 2), dict(rows=(1 << 28) + 1)])
def test_logprobs_refuse(lib, over):
    with pytest.raises(_lib.PromoeError) as e:
        logprobs(**over)
    assert e.value.code == 1 and "token_logprobs" in str(e.value)


def test_logprobs_of_no_rows_is_nothing(lib):
    logprobs(rows=0)


def test_the_python_handles_check_before_a_device_is_needed(lib):
    import torch
    with pytest.raises(ValueError):
        ops.Router(64, 6, scoring="tanh")
    with pytest.raises(ValueError):
        ops.Router(64, 6, group_score="mean")
    with pytest.raises(ValueError):
        ops.Router(64, 6, bias=torch.zeros(64))  # not on a device
    with pytest.raises(_lib.PromoeError):
        ops.Router(64, 65)
    with pytest.raises(ValueError):
        ops.Linear(torch.zeros((4, 4), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.Router(64, 6)(torch.zeros((3, 64)))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros((3, 64)), torch.zeros(3, dtype=torch.int64))


def test_a_layer_refuses_a_router_that_does_not_fit(lib):
    ctx = C.c_void_p()
    _lib.call("pm_ctx_create", C.byref(ctx), 2, 16, b"num_expert_per_token=4")

    def set_router(layer=0, **over):
        r = dict(num_expert=16, top_k=4, scoring=1, n_group=4, topk_group=2, group_score=1, norm_topk=1, routed_scale=2.5)
        r.update(over)
        _lib.call("pm_layer_set_router", ctx, layer, C.byref(_lib.pm_router(**r)))

    with pytest.raises(_lib.PromoeError) as e:
        set_router()
    assert e.value.code == 3  # the weights come first
    w = _lib.pm_layer_weights()
    w.hidden, w.inter, w.top_k = 128, 64, 4
    _lib.call("pm_layer_set_weights", ctx, 0, C.byref(w))
    set_router()
    for bad in (dict(layer=-1), dict(layer=2), dict(num_expert=32), dict(top_k=3), dict(n_group=3), dict(topk_group=5), dict(scoring=7),
                dict(choice_bias=PTR + 2), dict(n_group=8, topk_group=1)):
        with pytest.raises(_lib.PromoeError) as e:
            set_router(**bad)
        assert e.value.code == 1
    _lib.call("pm_layer_set_router", ctx, 0, None)
    _lib.call("pm_ctx_destroy", ctx)
