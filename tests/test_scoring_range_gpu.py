"""Scoring operators over the whole range of finite logits and of temperatures, against the 64-bit oracle within
the bounds that it derives, and over offsets beyond 32 bits."""
import numpy as np
import pytest

import scoring_oracle as O
from test_scoring_gpu import _block, _check_distill, _check_grad, _check_score, _near, _np, _torch

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]
# masks that callers write instead of -Inf, and large logits
LARGE = [-1e9, -1e10, -1e20, -1e30, "lowest", 1e10, 1e30]
LOWEST = {"float32": 3.4028234663852886e38, "bfloat16": 3.3895313892515355e38, "float16": 65504.0}  # but for the sign
LARGE_OF = [(d, v) for d in DTYPES for v in LARGE if v == "lowest" or abs(v) <= LOWEST[d]]


def _large(dtype, value):
    """The value as the type holds it."""
    import torch

    return -LOWEST[dtype] if value == "lowest" else torch.tensor(value).to(_torch(dtype)).item()


def _large_rows(dtype, value, V, seed=5):
    """All of one value; all but the last tenth, but the first tenth, but every second id, but one id."""
    x = _block(np.random.default_rng(seed), 5, V, dtype, 1, 3)
    x[0] = value
    x[1, : V - V // 10] = value
    x[2, V // 10:] = value
    x[3, ::2] = value
    x[4, : V // 2] = value
    x[4, V // 2 + 1:] = value
    return x


@pytest.mark.parametrize("T,dtype,value", [(T, d, v) for T in (0.001, 0.5, 1.0, 1.5, 2.0, 4.0, 10.0, 10000.0)
                                           for d, v in LARGE_OF
                                           if abs(LOWEST[d] if v == "lowest" else v) / T <= LOWEST["float32"]])
def test_score_of_large_logits(sampler, T, dtype, value):
    """Rows and parts of rows of one large value, in long rows too, where a thread has several steps of it; where
    the log-probability of a mask is an fp32 number."""
    v = _large(dtype, value)
    for V in (5003, 150011):
        x = _large_rows(dtype, v, V)
        o = _check_score(sampler, x, T, [[0, V // 2, V - 1]] * 5, 5)
        assert np.isfinite(_np(o.entropy)).all()


@pytest.mark.parametrize("T", [0.25, 1.0, 3.0])
@pytest.mark.parametrize("middle", [2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 30])
def test_score_of_close_large_logits(sampler, T, middle):
    """Logits some steps of fp32 around a number whose reference in the exponents' unit is near 2^24, below or above."""
    import torch

    rng = np.random.default_rng(int(middle))
    c = np.float32(middle * T / 1.4426950408889634)
    for sign in (-1, 1):
        n = rng.integers(-12, 13, (4, 30011))
        x = torch.from_numpy((sign * c * (1 + n * 2.0 ** -23)).astype(np.float32)).cuda()
        _check_score(sampler, x, T, [[1, 30010]] * 4, 9)
        _check_grad(sampler, x, T, [[1, 30010]] * 4, [[0.5, -0.25]] * 4, None)


@pytest.mark.parametrize("dtype,value", LARGE_OF)
def test_score_gradient_of_large_logits(sampler, dtype, value):
    v = _large(dtype, value)
    V = 5003
    x = _large_rows(dtype, v, V)
    for T in (0.7, 2.0, 10.0):
        _check_grad(sampler, x, T, [[0, V // 2, V - 1]] * 5, [[0.5, -1.0, 0.25]] * 5, None)


@pytest.mark.parametrize("dtype,value", LARGE_OF)
@pytest.mark.parametrize("kind", ["logits", "logprobs"])
def test_distill_of_large_logits(sampler, dtype, value, kind):
    """One large value everywhere, in most of a row, at listed ids, and at every id that is not listed."""
    import torch

    v = _large(dtype, value)
    for V in (2003, 150011):
        x = torch.cat([_large_rows(dtype, v, V), _block(np.random.default_rng(6), 2, V, dtype)])
        ids = [[5, 9, V // 2, V - 1]] * 7
        x[5] = v
        x[5, ids[5]] = torch.tensor([1.0, 2.0, 0.5, -1.0], dtype=x.dtype, device="cuda")
        x[6, [9, V - 1]] = v
        q = np.log(np.array([[0.4, 0.3, 0.2, 0.05]] * 7))
        for T in (1.0, 1.5, 2.0, 4.0, 10.0):
            _check_distill(sampler, x, T, ids, q.tolist(), kind, [1.0, 0.5, 1.0, 2.0, 1.0, 1.0, 0.25])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [0.00011, 0.001, 0.01, 0.1, 1.0, 30.0, 10000.0])
def test_score_gradient_of_masked_rows_at_any_temperature(sampler, dtype, T):
    """Masks of -Inf and of the type's lowest value, masked tokens, entropy gradients as a loss scale leaves them.
    fp16: such that the gradient of an id that is not masked stays finite."""
    import torch

    V = 2051
    low = torch.finfo(_torch(dtype)).min
    x = _block(np.random.default_rng(8), 6, V, dtype, 1, 1)
    x[0, ::2] = -float("inf")
    x[1, ::2] = low
    x[2, : V - 3] = -float("inf")
    x[3, 3:] = low
    x[4] = -float("inf")
    x[4, 77] = 2.0
    tokens = [[0, 1], [2, 2000], [5, V - 1], [1, 100], [77, 3], [7, 8]]
    most = 1e4 if dtype != "float16" else min(1e4, 1e3 * T)
    for g in (1e-3, 1.0, 5.0, 655.0, 1e4):
        g = min(g, most)
        _check_grad(sampler, x, T, tokens, [[0.5 * g, -0.25 * g]] * 6, [g, -g, g, g, g, -g])
        _check_grad(sampler, x, T, None, None, [g, -g, g, g, g, -g])


@pytest.mark.parametrize("dtype", DTYPES)
def test_score_gradients_that_cancel_in_rows_without_a_distribution(sampler, dtype):
    """Token gradients that add up to 0: NaN for a NaN or +Inf logit (0 times a NaN probability), 0 for padding and
    for -Inf alone; all gradients 0: 0."""
    import torch

    V = 1501
    x = _block(np.random.default_rng(4), 6, V, dtype, 1, 1)
    x[0, 17] = float("nan")
    x[1, 9] = float("inf")
    x[2] = -float("inf")
    x[3, 3] = float("nan")
    x[5, 17] = float("nan")
    tok = torch.tensor([[3, 4]] * 3 + [[-1, V]] + [[3, 4]] * 2, dtype=torch.int32, device="cuda")
    g = torch.tensor([[0.5, -0.5]] * 5 + [[0.0, 0.0]], device="cuda")
    o = sampler.logprobs(x, tok, entropy=True, stats=True)
    for g_ent in (None, torch.zeros(6, device="cuda")):
        dx = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, g, g_ent, o.entropy if g_ent is not None else None)
        assert bool(dx[:2].isnan().all())
        assert bool((dx[[2, 3, 5]] == 0).all())
        want = torch.zeros(V, dtype=x.dtype, device="cuda")
        want[3], want[4] = 0.5, -0.5
        assert torch.equal(dx[4], want)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [0.00011, 0.01, 0.3, 30.0, 10000.0])
def test_distill_of_masked_rows_at_any_temperature(sampler, kind, dtype, T):
    import torch

    V, K = 2051, 6
    low = torch.finfo(_torch(dtype)).min
    x = _block(np.random.default_rng(8), 5, V, dtype, 1, 1)
    ids = [[1, 3, 501, 77, V - 2, -1]] * 5
    x[0, ::2] = -float("inf")
    if dtype == "float16" or T >= 1:  # elsewhere (lowest - largest) / T is no fp32 number
        x[1, ::2] = low
        x[2, 600:] = low
    x[3, 600:V - 3] = -float("inf")
    v = np.log(np.array([[0.3, 0.25, 0.2, 0.1, 0.05, 0.9]] * 5))
    _check_distill(sampler, x, T, ids, v.tolist(), kind, [T, 0.5 * T, -T, T, 0.0])


def test_gradients_beyond_32_bit_offsets(sampler):
    """Rows 2^27 elements apart, the last ones beyond 2^31 elements: gradients written over the logits and beside
    them equal those of the same rows packed."""
    import torch

    B, V, ld = 20, 1003, (1 << 27) + 1
    packed = torch.randn(B, V, device="cuda").bfloat16()
    buf = torch.empty((B - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((B, V), (ld, 1))
    tok = torch.randint(0, V, (B,), dtype=torch.int32, device="cuda")
    g, ge = torch.randn(B, device="cuda"), torch.randn(B, device="cuda")
    o = sampler.logprobs(packed, tok, entropy=True, stats=True, top_n=9)
    want = sampler.logprobs_backward(packed, tok, o.row_max, o.row_sum, g, ge, o.entropy)
    x.copy_(packed)
    over = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, g, ge, o.entropy, out=x)
    assert over.data_ptr() == x.data_ptr() and torch.equal(over, want)
    beside = sampler.logprobs_backward(packed, tok, o.row_max, o.row_sum, g, ge, o.entropy, out=x.zero_())
    assert torch.equal(beside, want)
    x.copy_(torch.randn(B, V, device="cuda"))
    ids, v = o.top_ids, o.top_logprobs
    X, loss = _np(x), sampler.distill_loss(x, ids, v)
    l1, d1 = sampler.distill_grad(x, ids, v, g)
    l2, d2 = sampler.distill_grad(x, ids, v, g, out=x)
    assert d2.data_ptr() == x.data_ptr() and torch.equal(d2, d1)
    assert torch.equal(l1, loss) and torch.equal(l2, loss)
    for r in range(B):
        wl, bl, wd, bd = O.distill(X[r], 1.0, ids[r].tolist(), _np(v[r]), "logprobs", float(g[r]), "bfloat16")
        _near([_np(loss)[r]], [wl], bl, ("loss", r))
        _near(_np(d1[r]), wd, bd, ("dlogits", r))
    # the scores' gradient against the definition
    lp = torch.log_softmax(packed.double(), 1)
    h = -(lp.exp() * lp).sum(1, keepdim=True)
    d = -lp.exp() * (g[:, None].double() + ge[:, None].double() * (lp + h))
    d.scatter_add_(1, tok[:, None].long(), g[:, None].double())
    # one rounding to bf16, and some hundred fp32 roundings of terms of at most |g| + |g_H| (|log p| + H)
    near = 2.0 ** -8 * d.abs() + 2.0 ** -16 * (g.abs() + 20 * ge.abs())[:, None]
    assert bool(((want.double() - d).abs() <= near).all())


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
def test_distill_of_an_id_listed_twice(sampler, kind):
    """Against the same teacher with the id listed once with both masses: the gradient is the same, the loss less by
    sum_j q_j log(q_id / q_j)."""
    import torch

    V, T = 1203, 1.5
    x = _block(np.random.default_rng(3), 2, V, "float32")
    q = np.array([0.3, 0.2, 0.15, 0.1])                         # 7 twice, in one row next to one another
    ids = torch.tensor([[7, 40, 7, 1200], [40, 7, 7, 3]], dtype=torch.int32, device="cuda")
    both = [0.45, 0.35]
    less = [0.3 * np.log(0.45 / 0.3) + 0.15 * np.log(0.45 / 0.15), 0.2 * np.log(0.35 / 0.2) + 0.15 * np.log(0.35 / 0.15)]
    if kind == "logits":
        less = [v / q.sum() for v in less]
    scale = T if kind == "logits" else 1.0                      # the logits' softmax is taken at T
    v = torch.tensor(np.log(np.array([q, q])) * scale, dtype=torch.float32, device="cuda")
    one, w = ids.clone(), v.clone()
    one[0, 2] = one[1, 2] = -1
    w[0, 0], w[1, 1] = np.log(both[0]) * scale, np.log(both[1]) * scale
    loss, dx = sampler.distill_grad(x, ids, v, temperature=T, kind=kind)
    l1, d1 = sampler.distill_grad(x, one, w, temperature=T, kind=kind)
    # the masses differ by the rounding of their logarithms (of at most 3, half a step 2^-24 of it), the loss by that
    # of its terms (of at most 16 here), the gradient by a mass's
    np.testing.assert_allclose(_np(l1) - _np(loss), less, atol=2.0 ** -24 * 3 * 2 * 16)
    np.testing.assert_allclose(_np(dx), _np(d1), atol=2.0 ** -24 * 3 * 2)
    # a row's own distribution with an id's mass in two halves: no divergence but that of the halves
    z = torch.log(torch.tensor([[0.5, 0.25, 0.25]], device="cuda"))
    halves = torch.log(torch.tensor([[0.25, 0.25, 0.25, 0.25]], device="cuda"))
    own = sampler.distill_loss(z, torch.tensor([[0, 0, 1, 2]], dtype=torch.int32, device="cuda"), halves, kind=kind)
    np.testing.assert_allclose(_np(own), [0.5 * np.log(0.5)], atol=2.0 ** -20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["logits", "logprobs"])
def test_distill_of_a_bad_logit_in_the_list_and_masks_outside(sampler, dtype, kind):
    """A NaN or +Inf logit at a listed id makes the whole row NaN where every other id is masked, too."""
    V = 1201
    x = _block(np.random.default_rng(2), 4, V, dtype, 1, 1)
    x[:] = -float("inf")
    x[0, 40] = float("nan")
    x[1, 40] = float("inf")
    x[2, [40, 41]] = 1.0
    x[3, 700] = float("nan")
    ids, v = [[40, 41, V - 1]] * 3 + [[700, -1, -1]], np.log([[0.5, 0.25, 0.2]] * 4)
    _check_distill(sampler, x, 1.0, ids, v.tolist(), kind, [1.0, -2.0, 0.5, 1.0])


def test_largest_vocabulary(sampler):
    """One row of the largest accepted V: the last id drawn, listed and at the end of the gradient."""
    import torch

    V = 65535 * 16384
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, V, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    best = [V - 1, 7, V // 2 + 3, V - 12345, 1 << 29]
    x[0, best] = torch.tensor([16.0, 15.5, 15.0, 14.5, 14.0], dtype=x.dtype, device="cuda")
    s = q = 0.0
    for part in x[0].split(1 << 26):
        z = part.double() - 16.0
        e = z.exp()
        s, q = s + float(e.sum()), q + float((e * z).sum())
    log_s, h = np.log(s), np.log(s) - q / s
    # roundings of the sums if one CTA took the row: 32 terms a step, V / (256 * 32) steps, and those of RowDist
    eps = (32 + V / (256 * 32) + 117 + 3 * h) * 2.0 ** -24
    tok = torch.tensor([V - 1], dtype=torch.int32, device="cuda")
    o = sampler.logprobs(x, tok, top_n=5, entropy=True, stats=True)
    assert o.top_ids.tolist() == [best]
    np.testing.assert_allclose(_np(o.top_logprobs)[0], np.array([16.0, 15.5, 15.0, 14.5, 14.0]) - 16.0 - log_s,
                               rtol=2.0 ** -24, atol=eps)
    assert float(o.logprobs) == float(o.top_logprobs[0, 0])
    # an entropy's terms are weighed by their distance from the maximum, of about 16 here
    np.testing.assert_allclose(float(o.entropy), h, atol=eps * (1 + 20 + h))
    p = np.exp(_np(x[0, best]) - 16.0 - log_s)
    one = torch.ones(1, device="cuda")
    dx = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, one)
    want = np.array([1.0, 0, 0, 0, 0]) - p
    np.testing.assert_allclose(_np(dx[0, best]), want, rtol=2.0 ** -8, atol=eps)
    del dx
    ids = torch.tensor([best], dtype=torch.int32, device="cuda")
    t = np.array([0.5, 0.2, 0.1, 0.1, 0.05])
    v = torch.tensor(np.log(t)[None], dtype=torch.float32, device="cuda")
    loss, dd = sampler.distill_grad(x, ids, v, out=x)
    rest = 1.0 - np.exp(_np(v)).sum()
    want = (t * (np.log(t) - np.log(p))).sum() + rest * (np.log(rest) - np.log1p(-p.sum()))
    np.testing.assert_allclose(float(loss), want, rtol=2.0 ** -23, atol=3 * eps)
    np.testing.assert_allclose(_np(dd[0, best]), p - t, rtol=2.0 ** -8, atol=2 * eps)
    assert all(bool(part.isfinite().all()) for part in dd[0].split(1 << 26))


def test_hundreds_of_thousands_of_short_rows(sampler):
    """All rows of a batch that every cluster goes through hundreds of times, against torch in 64 bits."""
    import torch

    B, V, K = 300_007, 5, 2
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(B, V, device="cuda", generator=g)
    tok = torch.randint(-1, V, (B,), device="cuda", generator=g, dtype=torch.int32)
    ids = torch.rand(B, V, device="cuda", generator=g).argsort(1)[:, :K].to(torch.int32)
    ids[::3, 0] = -1
    ids[::9] = -1
    v = torch.log_softmax(torch.randn(B, V, device="cuda", generator=g), 1)[:, :K].contiguous()
    o = sampler.logprobs(x, tok, top_n=3, entropy=True, stats=True)
    dx = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, torch.ones(B, device="cuda"))
    loss, dd = sampler.distill_grad(x, ids, v)
    lp = torch.log_softmax(x.double(), 1)
    p, live, at = lp.exp(), tok >= 0, tok.clamp(min=0).long()[:, None]
    near = 2.0 ** -24 * 140  # the roundings of a row of few ids, over values of order 1 to 10
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    got = [(o.logprobs, torch.where(live, lp.gather(1, at)[:, 0], zero)),
           (o.entropy, torch.where(live, -(p * lp).sum(1), zero)),
           (dx, torch.where(live[:, None], torch.zeros_like(p).scatter_(1, at, 1.0) - p, zero))]
    top = torch.sort(x, dim=1, descending=True, stable=True)
    assert torch.equal(o.top_ids[live], top.indices[live, :3].int()) and bool((o.top_ids[~live] == -1).all())
    got.append((o.top_logprobs[live], lp.gather(1, top.indices)[live, :3]))
    there = ids >= 0
    q = torch.where(there, v.double().exp(), zero)
    mass = torch.zeros(B, V + 1, dtype=torch.float64, device="cuda").scatter_(1, torch.where(there, ids, V).long(), q)
    on = torch.zeros(B, V + 1, dtype=torch.bool, device="cuda").scatter_(1, torch.where(there, ids, V).long(), True)
    mass, on, rest = mass[:, :V], on[:, :V], 1.0 - q.sum(1)
    left = torch.where(on, zero, p).sum(1)
    want = torch.where(there, q * (v.double() - lp.gather(1, ids.clamp(min=0).long())), zero).sum(1)
    want = want + rest * (rest.log() - left.log())
    some = there.any(1)
    got.append((loss, torch.where(some, want, zero)))
    got.append((dd, torch.where(some[:, None], p - torch.where(on, mass, p * (rest / left)[:, None]), zero)))
    for i, (a, b) in enumerate(got):
        off = (a.double() - b).abs()
        assert bool((off <= near * (1 + b.abs()) + 3 * near).all()), (i, float(off.max()))
