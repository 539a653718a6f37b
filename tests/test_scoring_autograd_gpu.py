"""What autograd sees of the scoring calls: blocks written in place, outputs, derivatives that they do not have."""
import pytest

pytestmark = pytest.mark.gpu


def _teacher(s, B, V, n=8):
    import torch

    o = s.logprobs(torch.randn(B, V, device="cuda"), top_n=n)
    return o.top_ids, o.top_logprobs


@pytest.mark.parametrize("forward", ["logprobs", "distill_loss"])
@pytest.mark.parametrize("over", ["logprobs_backward", "distill_grad"])
def test_a_gradient_written_over_saved_logits_is_noticed(sampler, forward, over):
    """Autograd raises, as for any block that is modified in place, where it would use the overwritten logits."""
    import torch

    x = torch.randn(5, 301, device="cuda", requires_grad=True)
    tok = torch.randint(0, 301, (5,), device="cuda", dtype=torch.int32)
    ids, v = _teacher(sampler, 5, 301)
    y = (sampler.logprobs(x, tok).logprobs if forward == "logprobs" else sampler.distill_loss(x, ids, v)).sum()
    before = x._version
    with torch.no_grad():
        if over == "logprobs_backward":
            o = sampler.logprobs(x, tok, stats=True)
            sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, torch.ones(5, device="cuda"), out=x)
        else:
            sampler.distill_grad(x, ids, v, out=x)
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_ids_drawn_over_saved_tokens_are_noticed(sampler):
    import torch

    from minisample import SampleParams

    x = torch.randn(5, 301, device="cuda", requires_grad=True)
    u = torch.rand(5, dtype=torch.float64, device="cuda")
    ids = sampler.sample(x.detach(), SampleParams(), u=u, sync=False)
    y = sampler.logprobs(x, ids).logprobs.sum()
    sampler.sample(x.detach(), SampleParams(), u=u, out=ids, sync=False)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradients_written_to_a_block_of_inference_mode(sampler):
    """Blocks without a version counter are taken as they were."""
    import torch

    from minisample import SampleParams

    with torch.inference_mode():
        x = torch.randn(5, 301, device="cuda")
        ids, v = _teacher(sampler, 5, 301)
        loss, dx = sampler.distill_grad(x, ids, v)
        l2, d2 = sampler.distill_grad(x.clone(), ids, v, out=torch.empty_like(x))
        assert torch.equal(loss, l2) and torch.equal(dx, d2)
        drawn = torch.empty(5, dtype=torch.int32, device="cuda")
        u = torch.rand(5, dtype=torch.float64, device="cuda")
        assert torch.equal(sampler.sample(x, SampleParams(), u=u, out=drawn), sampler.sample(x, SampleParams(), u=u))


@pytest.mark.parametrize("grad", [False, True])
def test_outputs_that_were_not_asked_for_are_none(sampler, grad):
    import torch

    x = torch.randn(3, 301, device="cuda", requires_grad=grad)
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    o = sampler.logprobs(x, tok)
    assert [v is None for v in o] == [False, True, True, True, True, True]
    o = sampler.logprobs(x, top_n=2, stats=True)
    assert [v is None for v in o] == [True, True, False, False, False, False]
    o = sampler.logprobs(x, entropy=True)
    assert [v is None for v in o] == [True, False, True, True, True, True]
    if grad:
        (g,) = torch.autograd.grad(o.entropy.sum(), x)
        assert g.shape == x.shape
    assert all(v is None for v in sampler.logprobs(x))


def test_forward_mode_is_refused(sampler):
    """The calls have no forward derivatives: a tangent is not dropped without a word."""
    import torch
    import torch.autograd.forward_ad as fwad

    x, t = torch.randn(3, 301, device="cuda"), torch.randn(3, 301, device="cuda")
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    ids, v = _teacher(sampler, 3, 301)
    o = sampler.logprobs(x, tok, stats=True)
    g = torch.ones(3, device="cuda")
    with fwad.dual_level():
        for z in (fwad.make_dual(x, t), fwad.make_dual(x.clone().requires_grad_(), t)):
            for call in (lambda: sampler.logprobs(z, tok), lambda: sampler.distill_loss(z, ids, v),
                         lambda: sampler.logprobs_backward(z, tok, o.row_max, o.row_sum, g),
                         lambda: sampler.distill_grad(z, ids, v)):
                with pytest.raises(ValueError, match="forward-mode"):
                    call()
        assert torch.equal(sampler.logprobs(x, tok).logprobs, o.logprobs)  # no tangent: as ever
    for call in (lambda z: sampler.logprobs(z, tok).logprobs, lambda z: sampler.distill_loss(z, ids, v)):
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (x,), (t,))
