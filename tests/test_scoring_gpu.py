"""Scoring operators on the GPU against the 64-bit oracle (scoring_oracle.py),
within the bounds that it derives, at the sizes, strides and masks where they
can go wrong; autograd, streams, graphs; and the operators together, as a
generation loop and a training step use them."""
import numpy as np
import pytest

import scoring_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]


def _torch(name):
    import torch

    return getattr(torch, name)


def _block(rng, B, V, dtype, shift=0, pad=0, scale=2.5):
    """A [B, V] block whose rows start `shift` elements into a buffer and lie
    V + pad elements apart, and the values it holds as float64."""
    import torch

    x = torch.from_numpy(rng.normal(0.0, scale, (B, V)).astype(np.float32)).to(_torch(dtype)).cuda()
    return _placed(x, shift, pad)


def _placed(x, shift=0, pad=0):
    import torch

    B, V = x.shape
    buf = torch.full((B * (V + pad) + shift,), 77.0, dtype=x.dtype, device="cuda")
    v = buf[shift:].view(B, V + pad)[:, :V]
    v.copy_(x)
    return v


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _near(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=str(what))
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)], err_msg=str(what))
    off = np.abs(got[fine] - want[fine])
    lim = np.broadcast_to(bound, want.shape)[fine]
    bad = np.nonzero(off > lim)[0]
    assert bad.size == 0, (what, off[bad[:4]], lim[bad[:4]], want[fine][bad[:4]])


def _check_score(s, x, T=1.0, tokens=None, top_n=0):
    import torch

    B = x.shape[0]
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device="cuda")
    o = s.logprobs(x, tok, temperature=T, top_n=top_n, entropy=True, stats=True)
    torch.cuda.synchronize()
    X = _np(x)
    for r in range(B):
        row = None if tokens is None else np.atleast_1d(tokens[r])
        want, bound = O.score(X[r], T, row, top_n)
        for k, v in want.items():
            got = _np(getattr(o, k))
            if got is None:
                continue
            _near(np.atleast_1d(got[r]), np.atleast_1d(v), bound[k], (k, r))
    return o


# ---------------------------------------------------------------- forward
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 5, 8, 9, 31, 64, 255, 513, 1000, 4099, 20011])
def test_score_sizes(sampler, dtype, V):
    rng = np.random.default_rng(V)
    B = 5
    tokens = rng.integers(0, V, (B, 3))
    for shift, pad in ((0, 0), (1, 0), (3, 5), (7, 1)):
        x = _block(rng, B, V, dtype, shift, pad)
        _check_score(sampler, x, 1.0, tokens.tolist(), 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", [(1, 50257), (2, 128256), (1, 262144), (3, 131077), (1, 1000003)])
def test_score_long_rows(sampler, dtype, B, V):
    rng = np.random.default_rng(B + V)
    x = _block(rng, B, V, dtype, 1, 3)
    _check_score(sampler, x, 0.8, rng.integers(0, V, B).tolist(), 20)


@pytest.mark.parametrize("B,V", [(17, 5003), (150, 777), (700, 130), (5000, 33), (3, 0x8000)])
def test_score_many_rows(sampler, B, V):
    rng = np.random.default_rng(B)
    x = _block(rng, B, V, "float32", 0, 1)
    _check_score(sampler, x, 1.3, rng.integers(0, V, B).tolist(), 3)


@pytest.mark.parametrize("T", [0.00011, 0.05, 0.7, 3.0, 10000.0])
def test_score_temperatures(sampler, T):
    x = _block(np.random.default_rng(8), 3, 3001, "float32")
    _check_score(sampler, x, T, [[0, 3000], [5, 5], [17, 9]], 5)


@pytest.mark.parametrize("top_n", [1, 2, 31, 32, 33, 64, 100, 255, 256])
@pytest.mark.parametrize("V", [7, 300, 1030, 1500, 2049, 5000, 40000])
def test_top_alternatives(sampler, top_n, V):
    """Continuous values, and a few distinct values only (ties by ascending id)."""
    rng = np.random.default_rng(top_n)
    for dtype in ("float32", "bfloat16"):
        x = _block(rng, 3, V, dtype, 1, 2)
        x[1] = (x[1] * 2).round() / 2
        x[2] = x[2].sign()
        _check_score(sampler, x, 1.0, None, top_n)


@pytest.mark.parametrize("B,V,dtype,top_n", [(512, 262144, "float32", 64), (512, 262144, "bfloat16", 200),
                                             (1100, 65537, "float16", 0), (460, 131075, "float32", 3)])
def test_rows_over_several_rounds(sampler, B, V, dtype, top_n):
    """More rows than the GPU takes at once, padding among them, rows of one and of several CTAs: rows of
    every round against the oracle, all of them against a call of their own few rows."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(B + top_n)
    x = _placed((torch.randn(B, V, device="cuda", generator=g) * 2.5).to(_torch(dtype)), 1, 2)
    tok = torch.randint(0, V, (B, 1), device="cuda", generator=g, dtype=torch.int32)
    tok[::7] = -1
    o = sampler.logprobs(x, tok, top_n=top_n, entropy=True, stats=True)
    torch.cuda.synchronize()
    for r in [0, 1, 7, 147, 148, 295, 296, 443, 444, B - 2, B - 1]:
        if r >= B:
            continue
        want, bound = O.score(_np(x[r]), 1.0, tok[r].tolist(), top_n)
        for k, v in want.items():
            got = _np(getattr(o, k))
            if got is not None:
                _near(np.atleast_1d(got[r]), np.atleast_1d(v), bound[k], (k, r))
    if top_n:
        live = (tok >= 0).flatten()
        xf = x.float()
        got = torch.gather(xf, 1, o.top_ids.clamp(min=0).long())[live]
        assert torch.equal(got, torch.topk(xf, top_n, dim=1).values[live])
        assert bool((o.top_ids[~live] == -1).all())
    few = [sampler.logprobs(x[r:r + 50], tok[r:r + 50], entropy=True) for r in range(0, B, 50)]
    # both within the sums' bound of the truth, which is some hundred 2^-24 of a value near 10
    assert torch.allclose(o.entropy, torch.cat([f.entropy for f in few]), rtol=2.0 ** -15, atol=0)
    assert torch.allclose(o.logprobs, torch.cat([f.logprobs for f in few]), rtol=2.0 ** -15, atol=2.0 ** -15)


@pytest.mark.parametrize("B,V,dtype,K", [(300, 262144, "float32", 40), (700, 50259, "bfloat16", 256)])
def test_distill_rows_over_several_rounds(sampler, B, V, dtype, K):
    import torch

    g = torch.Generator(device="cuda").manual_seed(K)
    x = _placed((torch.randn(B, V, device="cuda", generator=g) * 2.5).to(_torch(dtype)), 1, 2)
    v, ids = torch.topk(x.float() + 0.7 * torch.randn(B, V, device="cuda", generator=g), K, dim=1)
    v, ids = torch.log_softmax(v, 1) - 0.05, ids.to(torch.int32)
    ids[::5] = -1
    w = torch.rand(B, device="cuda", generator=g)
    w[3::11] = 0.0
    loss, dx = sampler.distill_grad(x, ids, v, w)
    assert torch.equal(loss, sampler.distill_loss(x, ids, v))
    torch.cuda.synchronize()
    for r in [0, 1, 3, 14, 147, 148, 295, 296, 297, B - 2, B - 1]:
        if r >= B:
            continue
        wl, bl, wd, bd = O.distill(_np(x[r]), 1.0, ids[r].tolist(), _np(v[r]), "logprobs", float(w[r]), dtype)
        _near([_np(loss)[r]], [wl], bl, ("loss", r))
        _near(_np(dx[r]), wd, bd, ("dlogits", r))
    # the gradient of a row of weight sums to 0, the softmax's, up to its elements' rounding
    live = (ids >= 0).any(1) & (w != 0)
    assert bool((dx[~live] == 0).all())
    big = dx.double().abs().sum(1)
    assert bool((dx.double().sum(1).abs()[live] <= big[live] * (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -18)).all())


def _shaped(kind, V, rng):
    i = np.arange(V)
    if kind == "constant":
        return np.zeros(V)
    if kind == "zeros of both signs":
        return np.where(i % 3 == 0, -0.0, 0.0)
    if kind == "ascending":
        return i / 1024.0 - 7
    if kind == "descending":
        return 7 - i / 1024.0
    if kind == "front":  # the largest ids side by side
        return np.where(i < 700, 20 + rng.random(V), rng.random(V))
    if kind == "back":
        return np.where(i >= V - 700, 20 + rng.random(V), rng.random(V))
    if kind.startswith("every"):  # the largest at a fixed distance: in a few threads' hands
        n = int(kind.split()[1])
        return np.where(i % n < 4, 20 + rng.random(V), rng.random(V))
    if kind == "one":
        return np.where(i == V // 2, 60.0, 0.0)
    if kind == "few left":
        return np.where(i % 5003 == 11, rng.random(V), -np.inf)
    if kind == "few left, lowest":
        return np.where(i % 5003 == 11, rng.random(V), np.finfo(np.float32).min)
    raise KeyError(kind)


SHAPES = ["constant", "zeros of both signs", "ascending", "descending", "front", "back", "every 1024", "every 2048",
          "every 4096", "every 8192", "one", "few left", "few left, lowest"]


@pytest.mark.parametrize("kind", SHAPES)
@pytest.mark.parametrize("top_n", [5, 64, 256])
def test_top_alternatives_of_shaped_rows(sampler, kind, top_n):
    import torch

    V = 30011
    rng = np.random.default_rng(3)
    for rows in (1, 40):  # few rows and many: a row is split or not
        x = torch.from_numpy(np.stack([_shaped(kind, V, rng) for _ in range(2)]).astype(np.float32)).cuda()
        x = x.repeat(rows, 1)[: max(rows, 1)]
        o = sampler.logprobs(x, top_n=top_n)
        X = _np(x)
        for r in (0, rows - 1):
            want, bound = O.score(X[r], 1.0, None, top_n)
            _near(_np(o.top_ids)[r], want["top_ids"], 0, (kind, r))
            _near(_np(o.top_logprobs)[r], want["top_logprobs"], bound["top_logprobs"], (kind, r))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_distribution(sampler, dtype):
    """NaN, +Inf, all -Inf, lowest values, a NaN among -Inf, one id left; with and without padding."""
    import torch

    V = 3003
    t = _torch(dtype)
    low = torch.finfo(t).min
    x = _block(np.random.default_rng(4), 10, V, dtype, 1, 1)
    x[0, 17] = float("nan")
    x[1, V - 1] = float("inf")
    x[2] = -float("inf")
    x[3] = low
    x[4] = -float("inf")
    x[4, 5] = float("nan")
    x[5] = -float("inf")
    x[5, V - 2] = 3.0
    x[6, ::2] = low
    x[7, : V - 9] = -float("inf")
    x[8] = float("inf")
    x[9] = -float("inf")
    x[9, 1000] = low
    tokens = [[5, 17]] * 10
    _check_score(sampler, x, 1.0, tokens, 12)
    _check_score(sampler, x, 0.7, None, 12)
    bad = [[-1, V], [2**31 - 1, -2**31], [3, -1]] + [[-5, V + 1]] * 7  # all padding but row 2
    o = _check_score(sampler, x, 1.0, bad, 12)
    assert _np(o.logprobs)[0].tolist() == [0.0, 0.0] and _np(o.entropy)[0] == 0.0


def test_score_offsets_beyond_32_bits(sampler):
    """Rows 2^27 elements apart: the last one starts beyond 2^31 elements."""
    import torch

    B, V, ld = 20, 1003, (1 << 27) + 1
    buf = torch.empty((B - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((B, V), (ld, 1))
    x.copy_(torch.randn(B, V, device="cuda"))
    _check_score(sampler, x, 1.0, [[3]] * B, 4)
    tok = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    o = sampler.logprobs(x, tok, stats=True)
    g = torch.ones(B, device="cuda")
    dx = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, g, out=x)
    small = sampler.logprobs_backward(x.contiguous(), tok, o.row_max, o.row_sum, g)
    assert dx.data_ptr() == x.data_ptr()
    del small, buf


def test_score_empty_batch_and_no_outputs(sampler):
    import torch

    x = torch.zeros((0, 10), device="cuda")
    o = sampler.logprobs(x, torch.zeros(0, dtype=torch.int32, device="cuda"), top_n=3, entropy=True, stats=True)
    assert o.logprobs.shape == (0,) and o.top_ids.shape == (0, 3) and o.row_max.shape == (0,)
    o = sampler.logprobs(torch.zeros((2, 10), device="cuda"))
    assert all(v is None for v in o)
    loss, dx = sampler.distill_grad(x, torch.zeros((0, 2), dtype=torch.int32, device="cuda"),
                                    torch.zeros((0, 2), device="cuda"))
    assert loss.shape == (0,) and dx.shape == (0, 10)


def test_score_of_one_row_with_any_row_stride(sampler):
    import torch

    x = torch.randn(1, 999, device="cuda").as_strided((1, 999), (1, 1))
    _check_score(sampler, x, 1.0, [[5]], 3)
    col = torch.randn(7, 3, device="cuda")[:, :1]  # V = 1: any column stride
    _check_score(sampler, col, 1.0, [[0]] * 7, 3)


# ---------------------------------------------------------------- backward
def _check_grad(s, x, T, tokens, g_lp, g_H, out=None):
    import torch

    X, dtype = _np(x), str(x.dtype).split(".")[1]
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device="cuda")
    gl = None if g_lp is None else torch.tensor(g_lp, dtype=torch.float32, device="cuda")
    gh = None if g_H is None else torch.tensor(g_H, dtype=torch.float32, device="cuda")
    o = s.logprobs(x, tok, temperature=T, entropy=True, stats=True)
    dx = s.logprobs_backward(x, tok, o.row_max, o.row_sum, gl, gh, o.entropy if g_H is not None else None,
                             temperature=T, out=out)
    torch.cuda.synchronize()
    got = _np(dx)
    for r in range(X.shape[0]):
        want, bound = O.score_grad(X[r], T, None if tokens is None else np.atleast_1d(tokens[r]),
                                   None if gl is None else np.atleast_1d(_np(gl)[r]),
                                   None if gh is None else _np(gh)[r], dtype)
        _near(got[r], want, bound, ("dlogits", r))
    return dx


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 9, 250, 4099, 50257])
def test_score_gradient_sizes(sampler, dtype, V):
    rng = np.random.default_rng(V)
    B = 4
    tokens = rng.integers(0, V, (B, 3))
    tokens[1, 1] = tokens[1, 0]          # the same token twice
    tokens[2] = [-1, V, -7]              # padding
    tokens[3, 2] = 2**31 - 1
    g, gH = rng.normal(0, 1, (B, 3)), rng.normal(0, 0.3, B)
    for shift, pad in ((0, 0), (1, 0), (5, 3)):
        x = _block(rng, B, V, dtype, shift, pad)
        _check_grad(sampler, x, 0.9, tokens.tolist(), g.tolist(), gH.tolist())
        _check_grad(sampler, x, 1.0, tokens.tolist(), g.tolist(), None)
        _check_grad(sampler, x, 1.0, None, None, gH.tolist())


def test_score_gradient_of_many_tokens(sampler):
    rng = np.random.default_rng(9)
    B, V = 3, 600
    tokens = rng.integers(-5, V + 5, (B, 256))
    x = _block(rng, B, V, "float32", 1, 1)
    _check_grad(sampler, x, 1.0, tokens.tolist(), rng.normal(0, 1, (B, 256)).tolist(), [0.1, 0.0, -2.0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_score_gradient_of_rows_without_a_distribution(sampler, dtype):
    import torch

    V = 1501
    t = _torch(dtype)
    x = _block(np.random.default_rng(4), 8, V, dtype, 1, 1)
    x[0, 17] = float("nan")
    x[1] = -float("inf")
    x[2] = torch.finfo(t).min
    x[3, ::2] = -float("inf")
    x[4, ::2] = torch.finfo(t).min
    x[5, 9] = float("inf")
    x[6, 3] = float("nan")               # a padded row that holds anything
    x[7] = -float("inf")
    x[7, 4] = 1.0                        # one id left: gradient 0 but for rounding
    tokens = [[3, 4]] * 6 + [[-1, -1], [4, 4]]
    _check_grad(sampler, x, 1.0, tokens, [[0.5, 0.25]] * 8, [0.125] * 8)
    _check_grad(sampler, x, 1.0, tokens, [[0.0, 0.0]] * 8, [0.0] * 8)


def test_score_gradients_that_cancel(sampler):
    x = _block(np.random.default_rng(5), 3, 777, "float32")
    _check_grad(sampler, x, 1.0, [[3, 4], [3, 3], [5, 700]], [[0.5, -0.5], [0.5, -0.5], [1.0, -1.0]], None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_score_gradient_written_in_place_and_beside(sampler, dtype):
    """Over the logits, and into rows that start at another offset from 16 bytes; the room
    between the rows and after the last stays as it was."""
    import torch

    rng = np.random.default_rng(6)
    B, V = 3, 2051
    tokens, g = rng.integers(0, V, (B, 2)).tolist(), rng.normal(0, 1, (B, 2)).tolist()
    for shift, pad in ((0, 0), (3, 2)):
        for oshift, opad in ((0, 0), (1, 0), (3, 2), (5, 7)):
            x = _block(rng, B, V, dtype, shift, pad)
            base = torch.full((B * (V + opad) + oshift + 64,), 5.0, dtype=x.dtype, device="cuda")
            out = base[oshift:].as_strided((B, V), (V + opad, 1), base.storage_offset() + oshift)
            keep = torch.ones_like(base, dtype=torch.bool)
            keep.as_strided((B, V), (V + opad, 1), oshift).fill_(False)
            beside = _check_grad(sampler, x, 1.0, tokens, g, [0.2] * B, out=out).clone()
            assert bool((base[keep] == 5.0).all())
            over = _check_grad(sampler, x, 1.0, tokens, g, [0.2] * B, out=x)
            assert over.data_ptr() == x.data_ptr()
            assert torch.equal(over, beside)


# ---------------------------------------------------------------- distillation
def _check_distill(s, x, T, ids, values, kind, weight=None, out=None):
    import torch

    X, dtype = _np(x), str(x.dtype).split(".")[1]
    it = torch.tensor(ids, dtype=torch.int32, device="cuda")
    vt = torch.tensor(values, dtype=torch.float32, device="cuda")
    wt = None if weight is None else torch.tensor(weight, dtype=torch.float32, device="cuda")
    alone = s.distill_loss(x, it, vt, temperature=T, kind=kind)
    loss, dx = s.distill_grad(x, it, vt, wt, temperature=T, kind=kind, out=out)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(_np(alone), _np(loss))
    L, D, Vt = _np(loss), _np(dx), _np(vt)
    for r in range(X.shape[0]):
        wl, bl, wd, bd = O.distill(X[r], T, ids[r], Vt[r], kind, 1.0 if weight is None else float(np.float32(weight[r])),
                                   dtype)
        _near([L[r]], [wl], bl, ("loss", r))
        _near(D[r], wd, bd, ("dlogits", r))
    return loss, dx


def _teacher(rng, X, K, T, kind, noise=0.7):
    """The K largest ids of the logits with noise, and their values, row by row."""
    t = X + rng.normal(0, noise, X.shape)
    K = min(K, X.shape[1])
    ids = np.argsort(-t, axis=1)[:, :K]
    v = np.take_along_axis(t, ids, 1)
    if kind == "logprobs":
        z = t / T
        m = z.max(1, keepdims=True)
        v = v / T - m - np.log(np.exp(z - m).sum(1, keepdims=True))
    return ids.tolist(), v.astype(np.float32).tolist()


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,K", [(1, 1), (2, 1), (7, 3), (9, 8), (300, 256), (513, 64), (4099, 20), (50257, 100)])
def test_distill_sizes(sampler, dtype, kind, V, K):
    rng = np.random.default_rng(V + K)
    B, T = 4, 1.5
    for shift, pad in ((0, 0), (3, 1)):
        x = _block(rng, B, V, dtype, shift, pad)
        ids, v = _teacher(rng, _np(x), K, T, kind)
        _check_distill(sampler, x, T, ids, v, kind, rng.uniform(-1, 2, B).tolist())


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("B,V,K", [(1, 262144, 50), (3, 131077, 256), (1, 1000003, 7)])
def test_distill_long_rows(sampler, kind, B, V, K):
    rng = np.random.default_rng(V)
    for dtype in ("float32", "bfloat16"):
        x = _block(rng, B, V, dtype, 1, 1)
        ids, v = _teacher(rng, _np(x), K, 1.0, kind)
        _check_distill(sampler, x, 1.0, ids, v, kind)


@pytest.mark.parametrize("B,V,K", [(150, 777, 9), (700, 130, 130), (3000, 17, 5)])
def test_distill_many_rows(sampler, B, V, K):
    rng = np.random.default_rng(B)
    x = _block(rng, B, V, "float32", 0, 1)
    ids, v = _teacher(rng, _np(x), K, 1.0, "logprobs")
    _check_distill(sampler, x, 1.0, ids, v, "logprobs", rng.uniform(0, 1, B).tolist())


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
def test_distill_lists(sampler, kind):
    """Absent entries anywhere, the same id several times, neighbouring ids (one
    vector, one thread), ids a block's threads apart (one thread), the row's
    ends, a list without mass, padding, weight 0."""
    rng = np.random.default_rng(7)
    V, K = 9001, 12
    lists = [
        [-1] * 11 + [5],
        [5, -1, 7, V, -2**31, 2**31 - 1, 0, V - 1, -1, 3, 4, 6],
        [8, 8, 8, 9, 9, 1000, 8, 1000, 7, 7, 7, 7],
        list(range(100, 112)),
        [3 + 2048 * i for i in range(4)] + [4 + 4096 * i for i in range(2)] + [1024 * i for i in range(1, 7)],
        [-1] * 12,
        list(range(12)),
        [0, V - 1] + [-1] * 10,
        list(range(0, 96, 8)),
    ]
    B = len(lists)
    v = rng.normal(-3, 1, (B, K)).astype(np.float32)
    v[7, 0] = -np.inf  # a listed id without mass
    v[6, 3:] = -np.inf
    v[8] = -0.001 + np.log(1.0 / K)      # next to no mass left: 1 - sum q = 0.001
    weight = [1.0, 0.5, 2.0, 1.0, -1.0, 1.0, 0.0, 1.0, 0.25]
    for dtype in ("float32", "bfloat16"):
        x = _block(rng, B, V, dtype, 1, 1)
        _check_distill(sampler, x, 1.0, lists, v.tolist(), kind, weight)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_rows_without_a_distribution(sampler, kind, dtype):
    """Students with NaN, +Inf, -Inf alone, -Inf at listed ids, everything but
    the list masked, lowest values, next to no mass outside the list."""
    import torch

    V, K = 2003, 4
    t = _torch(dtype)
    x = _block(np.random.default_rng(4), 11, V, dtype, 1, 1)
    ids = [[5, 9, 700, V - 1]] * 11
    x[0, 17] = float("nan")
    x[1, 9] = float("nan")               # a listed one
    x[2, 40] = float("inf")
    x[3] = -float("inf")
    x[4, 9] = -float("inf")              # the teacher has mass where the student has none
    x[5] = -float("inf")
    x[5, [5, 9, 700, V - 1]] = torch.tensor([1.0, 2.0, 0.5, -1.0], dtype=t, device="cuda")
    x[6] = torch.finfo(t).min
    x[6, 5] = 1.0
    x[7, ::2] = torch.finfo(t).min
    x[8] = -100.0
    x[8, [5, 9, 700, V - 1]] = torch.tensor([8.0, 9.0, 7.5, 6.0], dtype=t, device="cuda")
    x[9, 17] = float("nan")              # padded below
    x[10, 17] = float("nan")             # weight 0 below
    ids[9] = [-1, V, -1, -1]
    v = np.log(np.array([[0.4, 0.3, 0.2, 0.05]] * 11))
    weight = [1.0] * 10 + [0.0]
    _check_distill(sampler, x, 1.0, ids, v.tolist(), kind, weight)


def test_distill_whole_vocabulary_listed(sampler):
    """No id outside the list: the mass that rounding leaves is none."""
    rng = np.random.default_rng(3)
    x = _block(rng, 5, 200, "float32")
    ids, v = _teacher(rng, _np(x), 200, 1.0, "logprobs")
    _check_distill(sampler, x, 1.0, ids, v, "logprobs")


def test_distill_from_itself_is_zero(sampler):
    """The teacher's lists of the student itself: loss and gradient 0 up to the bounds."""
    import torch

    x = torch.randn(6, 5003, device="cuda") * 2
    o = sampler.logprobs(x, top_n=40, temperature=2.0)
    loss, dx = sampler.distill_grad(x, o.top_ids, o.top_logprobs, temperature=2.0)
    # q is off by the log-probabilities' rounding, p by its sum's: some 2^-20 of a probability each
    assert float(loss.abs().max()) < 2.0 ** -18
    assert float(dx.abs().max()) < 2.0 ** -18
    _check_distill(sampler, x, 2.0, o.top_ids.cpu().tolist(), o.top_logprobs.cpu().tolist(), "logprobs")


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_gradient_written_in_place_and_beside(sampler, dtype):
    import torch

    rng = np.random.default_rng(6)
    B, V = 3, 2051
    for shift, pad in ((0, 0), (3, 2)):
        for oshift, opad in ((0, 0), (1, 0), (5, 7)):
            x = _block(rng, B, V, dtype, shift, pad)
            ids, v = _teacher(rng, _np(x), 33, 1.0, "logprobs")
            base = torch.full((B * (V + opad) + oshift + 64,), 5.0, dtype=x.dtype, device="cuda")
            out = base.as_strided((B, V), (V + opad, 1), oshift)
            keep = torch.ones_like(base, dtype=torch.bool)
            keep.as_strided((B, V), (V + opad, 1), oshift).fill_(False)
            beside = _check_distill(sampler, x, 1.0, ids, v, "logprobs", out=out)[1].clone()
            assert bool((base[keep] == 5.0).all())
            it = torch.tensor(ids, dtype=torch.int32, device="cuda")
            vt = torch.tensor(v, dtype=torch.float32, device="cuda")
            over = sampler.distill_grad(x, it, vt, out=x)[1]
            assert over.data_ptr() == x.data_ptr() and torch.equal(over, beside)


# ---------------------------------------------------------------- autograd
def test_autograd_of_logprobs_and_entropy(sampler):
    """The gradient through torch's graph equals the formula's; broadcast and
    missing gradients, a block used twice, 1-D and 2-D tokens."""
    import torch

    x = (torch.randn(6, 1201, device="cuda") * 2).requires_grad_()
    tok = torch.randint(0, 1201, (6, 2), device="cuda", dtype=torch.int32)
    adv = torch.randn(6, 2, device="cuda")

    def plain(z):
        lp = torch.log_softmax(z / 0.8, 1)
        h = -(lp.exp() * lp).sum(1)
        return (lp.gather(1, tok.long()) * adv).sum() + 0.3 * h.sum() + lp.gather(1, tok[:, :1].long()).mean()

    o = sampler.logprobs(x, tok, temperature=0.8, entropy=True, top_n=3)
    one = sampler.logprobs(x, tok[:, 0].contiguous(), temperature=0.8)
    assert not o.top_logprobs.requires_grad and o.logprobs.requires_grad and one.entropy is None
    (got,) = torch.autograd.grad((o.logprobs * adv).sum() + 0.3 * o.entropy.sum() + one.logprobs.mean(), x)
    z = x.detach().double().requires_grad_()
    (want,) = torch.autograd.grad(plain(z), z)
    # sums of three fp32 gradients of at most ~4 each
    np.testing.assert_allclose(_np(got), _np(want), atol=16 * 2.0 ** -20)
    # no gradient asked for: no graph
    with torch.no_grad():
        assert not sampler.logprobs(x, tok).logprobs.requires_grad
    # entropy alone, tokens without a gradient
    o = sampler.logprobs(x, tok, entropy=True)
    (got,) = torch.autograd.grad(o.entropy.sum(), x)
    lp = torch.log_softmax(z, 1)
    (want,) = torch.autograd.grad(-(lp.exp() * lp).sum(), z)
    np.testing.assert_allclose(_np(got), _np(want), atol=2.0 ** -20)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
def test_autograd_of_distillation(sampler, kind):
    import torch

    rng = np.random.default_rng(2)
    x = (torch.randn(5, 901, device="cuda") * 2).requires_grad_()
    ids, v = _teacher(rng, _np(x), 16, 2.0, kind)
    it, vt = torch.tensor(ids, dtype=torch.int32, device="cuda"), torch.tensor(v, device="cuda")
    loss = sampler.distill_loss(x, it, vt, temperature=2.0, kind=kind)
    (mean,) = torch.autograd.grad(loss.mean(), x, retain_graph=True)   # a broadcast gradient
    w = torch.rand(5, device="cuda")
    (some,) = torch.autograd.grad(loss, x, grad_outputs=w)
    fused = sampler.distill_grad(x.detach(), it, vt, w, temperature=2.0, kind=kind)
    assert torch.equal(some, fused[1]) and torch.equal(loss.detach(), fused[0])
    even = sampler.distill_grad(x.detach(), it, vt, torch.full((5,), 0.2, device="cuda"), temperature=2.0, kind=kind)
    assert torch.equal(mean, even[1])


def test_kernel_gradients_against_differences(sampler):
    """Central differences of the kernels' own values along random directions.
    With |f''| of order 1 and values off by a few 2^-22, a step of 2^-5 leaves
    2^-10 of curvature and 2^-15 of rounding."""
    import torch

    torch.manual_seed(3)
    x = torch.randn(4, 300, device="cuda")
    tok = torch.randint(0, 300, (4,), device="cuda", dtype=torch.int32)
    it = torch.randint(0, 300, (4, 6), device="cuda", dtype=torch.int32)
    vt = torch.log_softmax(torch.randn(4, 8, device="cuda"), 1)[:, :6].contiguous()

    def f(z):
        o = sampler.logprobs(z, tok, entropy=True)
        return (o.logprobs + 0.5 * o.entropy + sampler.distill_loss(z, it, vt)).double()

    z = x.clone().requires_grad_()
    o = sampler.logprobs(z, tok, entropy=True)
    (g,) = torch.autograd.grad((o.logprobs + 0.5 * o.entropy + sampler.distill_loss(z, it, vt)).sum(), z)
    h = 2.0 ** -5
    for _ in range(4):
        u = torch.randn_like(x)
        u /= u.norm(dim=1, keepdim=True)
        diff = (f(x + h * u) - f(x - h * u)) / (2 * h)
        np.testing.assert_allclose(_np((g * u).sum(1)), _np(diff), atol=2.0 ** -9)


# ---------------------------------------------------------------- refusals
def test_refusals(sampler):
    import torch

    x = torch.randn(4, 100, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    ids, v = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    mx = torch.zeros(4, dtype=torch.float64, device="cuda")
    g = torch.zeros(4, device="cuda")
    from minisample import MiniSampleError

    bad = [
        lambda: sampler.logprobs(x.cpu().numpy()), lambda: sampler.logprobs(x.double()), lambda: sampler.logprobs(x.cpu()), lambda: sampler.logprobs(x[0]),
        lambda: sampler.logprobs(x.t()), lambda: sampler.logprobs(x[:1].expand(4, 100)),
        lambda: sampler.logprobs(x[:, ::2]), lambda: sampler.logprobs(x, tok.long()),
        lambda: sampler.logprobs(x, tok[:3]), lambda: sampler.logprobs(x, tok.cpu()),
        lambda: sampler.logprobs(x, tok.view(4, 1)[:, :0]), lambda: sampler.logprobs(x, tok.view(4, 1, 1)),
        lambda: sampler.logprobs(x, top_n=257), lambda: sampler.logprobs(x, top_n=-1),
        lambda: sampler.logprobs_backward(x, tok, mx.float(), mx, g),
        lambda: sampler.logprobs_backward(x, tok, mx, mx[:3], g),
        lambda: sampler.logprobs_backward(x, tok, mx, mx, g.double()),
        lambda: sampler.logprobs_backward(x, tok, mx, mx, g.view(4, 1)),
        lambda: sampler.logprobs_backward(x, None, mx, mx, g),
        lambda: sampler.logprobs_backward(x, tok, mx, mx, g, g),
        lambda: sampler.logprobs_backward(x, tok, mx, mx, g, out=x[:3]),
        lambda: sampler.logprobs_backward(x, tok, mx, mx, g, out=x.half()),
        lambda: sampler.distill_loss(x, ids.long(), v), lambda: sampler.distill_loss(x, ids, v.double()),
        lambda: sampler.distill_loss(x, ids, v[:, :1]), lambda: sampler.distill_loss(x, ids[:3], v[:3]),
        lambda: sampler.distill_loss(x, ids, v, kind="probs"), lambda: sampler.distill_grad(x, ids, v, g[:2]),
        lambda: sampler.distill_grad(x, ids, v, g, out=x.t()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: sampler.logprobs(x, temperature=0.0), lambda: sampler.logprobs(x, temperature=float("nan")),
                 lambda: sampler.distill_loss(x, ids, v, temperature=-1.0),
                 lambda: sampler.distill_loss(x, ids[:, :0], v[:, :0]),
                 lambda: sampler.distill_grad(x, torch.zeros(4, 257, dtype=torch.int32, device="cuda"),
                                              torch.zeros(4, 257, device="cuda")),
                 lambda: sampler.logprobs(x, torch.zeros(4, 257, dtype=torch.int32, device="cuda")),
                 lambda: sampler.logprobs(torch.zeros(2, 0, device="cuda"))):
        with pytest.raises(MiniSampleError) as e:
            call()
        assert "MS_ERR_ARG" in str(e.value)
    # the logits shifted by one column: an overlap that is not the logits themselves
    wide = torch.randn(4, 101, device="cuda")
    with pytest.raises(MiniSampleError, match="overlaps"):
        sampler.distill_grad(wide[:, :100], ids, v, out=wide[:, 1:])


# ---------------------------------------------------------------- streams and graphs
def test_calls_on_other_streams(sampler):
    """Two streams at once, on the sampler's one handle, and the stream argument."""
    import torch

    xs = [torch.randn(64, 30011, device="cuda") for _ in range(2)]
    tok = torch.randint(0, 30011, (64,), device="cuda", dtype=torch.int32)
    want = [sampler.logprobs(x, tok, top_n=9, entropy=True) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for rep in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(sampler.logprobs(x, tok, top_n=9, entropy=True))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)
    o = sampler.logprobs(xs[0], tok, top_n=9, entropy=True, stream=streams[0])
    ids, v = want[0].top_ids, want[0].top_logprobs
    l0, d0 = sampler.distill_grad(xs[1], ids, v)
    l1, d1 = sampler.distill_grad(xs[1], ids, v, stream=streams[1])
    l2 = sampler.distill_loss(xs[1], ids, v, stream=streams[0])
    torch.cuda.synchronize()
    assert torch.equal(o.entropy, want[0].entropy)
    assert torch.equal(l0, l1) and torch.equal(d0, d1) and torch.equal(l0, l2)


def test_captured_and_replayed(sampler):
    """Two graphs captured on the sampler's one handle, replayed in turn and at
    once on two streams, with inputs that change between the replays."""
    import torch

    V = 20011
    xs = [torch.randn(8, V, device="cuda") for _ in range(2)]
    tok = torch.randint(0, V, (8,), device="cuda", dtype=torch.int32)
    g = torch.randn(8, device="cuda")

    def step(x):
        o = sampler.logprobs(x, tok, top_n=5, entropy=True, stats=True)
        dx = sampler.logprobs_backward(x, tok, o.row_max, o.row_sum, g, g, o.entropy)
        loss, dd = sampler.distill_grad(x, o.top_ids, o.top_logprobs, g)
        return [*o, dx, loss, dd]

    for x in xs:
        step(x)
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(x))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        for x in xs:
            x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            for a, b in zip(out, step(x)):
                assert torch.equal(a, b)


def test_first_calls_captured():
    """A fresh process whose first scoring calls are captured ones."""
    code = """
import sys
sys.path.insert(0, %r)
import torch
from minisample import Sampler
s = Sampler()
x = torch.randn(5, 3001, device="cuda")
tok = torch.full((5,), 7, dtype=torch.int32, device="cuda")
g = torch.ones(5, device="cuda")
def step():
    o = s.logprobs(x, tok, top_n=5, entropy=True, stats=True)
    dx = s.logprobs_backward(x, tok, o.row_max, o.row_sum, g, g, o.entropy)
    plain = s.logprobs(x, tok)
    return [*o, dx, plain.logprobs, *s.distill_grad(x, o.top_ids, o.top_logprobs, g),
            s.distill_loss(x, o.top_ids, o.top_logprobs)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
print("captured")
"""
    import os
    import subprocess
    import sys

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omni.js_b200")
    r = subprocess.run([sys.executable, "-c", code % pkg], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_results_are_the_same_every_time(sampler):
    import torch

    x = (torch.randn(33, 50257, device="cuda") * 2).bfloat16()
    first = sampler.logprobs(x, top_n=100, entropy=True)
    l0, d0 = sampler.distill_grad(x, first.top_ids, first.top_logprobs)
    for _ in range(5):
        o = sampler.logprobs(x, top_n=100, entropy=True)
        l1, d1 = sampler.distill_grad(x, first.top_ids, first.top_logprobs)
        assert torch.equal(o.top_ids, first.top_ids) and torch.equal(o.entropy, first.entropy)
        assert torch.equal(l0, l1) and torch.equal(d0, d1)
    # a row's results do not depend on the batch around it where the split is the same
    part = sampler.logprobs(x[:32], top_n=100)
    assert torch.equal(part.top_ids, first.top_ids[:32])


def test_launches_are_counted(sampler):
    import torch

    x = torch.randn(4, 1000, device="cuda")
    n0 = sampler.launch_count()
    o = sampler.logprobs(x, top_n=4, stats=True, entropy=True)
    sampler.logprobs_backward(x, None, o.row_max, o.row_sum, None, torch.ones(4, device="cuda"), o.entropy)
    sampler.distill_grad(x, o.top_ids, o.top_logprobs)
    assert sampler.launch_count() - n0 == 3


# ---------------------------------------------------------------- together
def test_sampling_scoring_and_training_together(sampler):
    """The sampler draws ids; they are scored; a policy-gradient step and a
    distillation step from the scorer's own lists update the logits that they
    came from; all on one stream without a synchronisation between."""
    import torch

    from minisample import SampleParams

    B, V = 12, 30011
    torch.manual_seed(1)
    logits = torch.randn(B, V, device="cuda") * 2
    u = torch.rand(B, dtype=torch.float64, device="cuda")
    ids = sampler.sample(logits, SampleParams(True, 0.8, 50, 0.95, 1.0), u=u, sync=False)
    o = sampler.logprobs(logits, ids, temperature=0.8, top_n=50, entropy=True, stats=True)
    adv = torch.randn(B, device="cuda")
    dx = sampler.logprobs_backward(logits, ids, o.row_max, o.row_sum, adv, temperature=0.8)
    student = torch.randn(B, V, device="cuda")
    loss, dd = sampler.distill_grad(student, o.top_ids, o.top_logprobs, temperature=0.8)
    after = sampler.logprobs(logits + 0.05 * dx, ids, temperature=0.8)
    nearer = sampler.distill_loss(student - 0.5 * dd, o.top_ids, o.top_logprobs, temperature=0.8)
    torch.cuda.synchronize()
    # every drawn id is one of the 50 largest, where the lists agree
    hit = o.top_ids == ids[:, None]
    assert bool(hit.any(1).all())
    assert torch.equal(o.top_logprobs[hit], o.logprobs)
    # a small step along the gradient moves each log-probability by its advantage's sign
    assert bool((((after.logprobs - o.logprobs) * adv) > 0).all())
    assert bool((nearer < loss).all())


class _TableModel:
    """forward_batch gives each row logits that depend on its last id; what it gave is kept."""

    V = 5003

    def __init__(self, B):
        self.B, self.given = B, []

    def make_cache(self):
        return {}

    def dispose_cache(self, cache):
        pass

    def forward_batch(self, last_ids, caches):
        import torch

        last = last_ids if last_ids is not None else list(range(self.B))
        rows = [np.random.default_rng(1000 * len(self.given) + int(i)).normal(0, 2, self.V) for i in last]
        self.given.append(np.stack(rows).astype(np.float32))
        return torch.from_numpy(self.given[-1]).cuda()


@pytest.mark.parametrize("n", [0, 4])
def test_generation_loop_returns_log_probabilities(n):
    """The device loop's `logprobs` option: the ids are those without it, and every generated id's scores
    are the oracle's on the logits that the model gave."""
    from minisample.generation import generate_tokens_device, set_backend

    set_backend("cuda")
    B = 3
    opts = {"maxNewTokens": 5, "temperature": 0.9, "topK": 20, "topP": 0.9, "repetitionPenalty": 1.2}

    def rands():
        return [iter(np.random.default_rng(i).random(50)).__next__ for i in range(B)]

    prompts = [[1, 2], [3], [4, 5, 6]]
    plain = generate_tokens_device(_TableModel(B), prompts, opts, rands=rands())
    eos = plain[1][2]
    opts = dict(opts, eosTokenId=eos)
    plain = generate_tokens_device(_TableModel(B), prompts, opts, rands=rands())
    model = _TableModel(B)
    ids, scores = generate_tokens_device(model, prompts, dict(opts, logprobs=n), rands=rands())
    assert ids == plain and [len(x) for x in scores] == [len(x) for x in ids]
    for i in range(B):
        for step, (tok, sc) in enumerate(zip(ids[i], scores[i])):
            want, bound = O.score(model.given[step][i], 1.0, [tok], n)
            _near([sc["logprob"]], want["logprobs"], bound["logprobs"], (i, step))
            _near([sc["entropy"]], [want["entropy"]], bound["entropy"], (i, step))
            assert sc["top_ids"] == want["top_ids"].tolist()
            _near(sc["top_logprobs"], want["top_logprobs"], bound["top_logprobs"], (i, step))
