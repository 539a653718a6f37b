"""The scoring operators over a [rows, vocab] block of logits: what is measured of them.

  score       log-probabilities of given tokens, the entropy of each row and its top alternatives
  score_grad  their backward pass: the gradient of the logits
  distill     the loss against a teacher's top values and the gradient of the logits, or the loss alone

`run` computes them in plain torch operations, or with `own` through the framework's Sampler.
"""
import math
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}
_LARGEST = 4096 * 151936 * 2  # bytes of the largest listed case's logits
# The teacher's mass outside its list counts as none below this: fp32 log-probabilities do not resolve it.
_NO_TAIL = 2.0 ** -20


def _score(name, rows, vocab, dtype, temperature, tokens, top, entropy, padded=0, banned=0.0):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "tokens": tokens, "top": top, "entropy": entropy, "padded": padded, "banned": banned}


def _score_grad(name, rows, vocab, dtype, temperature, tokens, entropy, padded=0):
    return {"name": name, "op": "score_grad", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "tokens": tokens, "entropy": entropy, "padded": padded}


def _distill(name, rows, vocab, dtype, temperature, teacher, kind, grad, padded=0, ragged=False):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "teacher": teacher, "kind": kind, "grad": grad, "padded": padded, "ragged": ragged}


def listed():
    return [
        # one sequence being decoded: the sampled id's log-probability and five alternatives
        _score("score one row", 1, 50257, "f32", 1.0, 1, 5, True),
        # a decoding batch under a grammar that bans 40% of the vocabulary, twenty alternatives
        _score("score decoding batch", 64, 128256, "f32", 0.7, 1, 20, True, banned=0.4),
        # every position of long prompts scored: the next id's log-probability and the entropy
        _score("score prompts", 2048, 151936, "bf16", 1.0, 1, 0, True),
        # the teacher's lists for distillation: the top 64 of every position
        _score("score teacher lists", 512, 262144, "f32", 2.0, 0, 64, False),
        # eight answer labels ranked at odd sizes, a quarter of the positions padding
        _score("score answer labels", 333, 50257, "f16", 1.0, 8, 3, False, padded=83),
        # a policy-gradient step with an entropy bonus over sampled continuations, a fifth padding
        _score_grad("score_grad policy step", 2048, 151936, "bf16", 1.0, 1, True, padded=409),
        # the likelihood gradient of one short sequence
        _score_grad("score_grad short", 61, 50257, "f32", 1.0, 1, False),
        # a training step against teacher log-probabilities, the mass outside the list included
        _distill("distill step", 4096, 151936, "bf16", 1.0, 64, "logprobs", True, padded=512),
        # teacher logits at a high temperature, half-precision logits
        _distill("distill warm logits", 1024, 128256, "f16", 4.0, 100, "logits", True),
        # ragged lists at odd sizes
        _distill("distill ragged", 509, 50257, "f32", 2.0, 20, "logits", True, padded=101, ragged=True),
        # a few positions of the largest vocabulary
        _distill("distill few rows", 8, 262144, "f32", 1.0, 50, "logprobs", True),
        # the loss alone over a held-out batch, with the longest lists
        _distill("distill held-out loss", 1024, 151936, "bf16", 1.0, 256, "logprobs", False),
    ]


def draw(rng):
    op = rng.choice(["score", "score", "score_grad", "distill", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    vocab = int(math.exp(rng.uniform(math.log(1024), math.log(262144))))
    most = max(1, min(4096, _LARGEST // 2 // (vocab * _SIZES[dtype])))
    rows = int(math.exp(rng.uniform(0.0, math.log(most + 0.999))))
    temperature = rng.choice([0.7, 1.0, 1.0, 2.0])
    padded = rng.choice([0, rows // 5])
    if op == "score":
        tokens = rng.choice([0, 1, 1, 1, 5])
        top = rng.choice([0, 1, 5, 20, rng.randint(1, 256)])
        if tokens == 0 and top == 0:
            top = 10
        c = _score("", rows, vocab, dtype, temperature, tokens, top, rng.choice([True, False]),
                   padded if tokens else 0, rng.choice([0.0, 0.0, 0.5]))
    elif op == "score_grad":
        c = _score_grad("", rows, vocab, dtype, temperature, rng.choice([1, 1, 3]), rng.choice([True, False]), padded)
    else:
        c = _distill("", rows, vocab, dtype, temperature, rng.choice([1, 20, 64, rng.randint(1, 256)]),
                     rng.choice(["logits", "logprobs"]), rng.choice([True, True, False]), padded,
                     rng.choice([True, False]))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _pieces(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def prepare(case, seed):
    """Logits as a language model gives them: a power law over the ids with noise, so that a few ids hold most of a
    row's mass and the rest a long tail; the teacher's are the student's with noise."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B, V, T = case["rows"], case["vocab"], case["temperature"]
    x = torch.empty((B, V), dtype=_DTYPES[case["dtype"]], device="cuda")
    st = {"case": case, "x": x}
    if case["op"] == "distill":
        K = min(case["teacher"], V)
        ids = torch.empty((B, K), dtype=torch.int32, device="cuda")
        values = torch.empty((B, K), dtype=torch.float32, device="cuda")
    for r0, r1 in _pieces(B, V):
        u = 1.0 - torch.rand((r1 - r0, V), generator=g, device="cuda")
        u = torch.log_(u.mul_(V)).mul_(-1.1)
        u += torch.randn((r1 - r0, V), generator=g, device="cuda").mul_(0.5)
        if case.get("banned"):
            u[torch.rand((r1 - r0, V), generator=g, device="cuda") < case["banned"]] = -math.inf
        x[r0:r1] = u
        if case["op"] == "distill":
            t = (u + torch.randn((r1 - r0, V), generator=g, device="cuda").mul_(0.7)).clamp_(-50, 50)
            v, i = torch.topk(t, K, dim=1)
            if case["kind"] == "logprobs":
                v = v.double() / T - torch.logsumexp(t.double() / T, 1, keepdim=True)
            ids[r0:r1], values[r0:r1] = i, v
    pad = torch.randperm(B, generator=g, device="cuda")[: case["padded"]]
    if case["op"] == "distill":
        if case["ragged"]:  # lists of different lengths: the rest of a list is absent
            n = torch.randint(1, K + 1, (B, 1), generator=g, device="cuda")
            ids[torch.arange(K, device="cuda") >= n] = -1
        ids[pad] = -1
        live = max(1, B - case["padded"])
        # the mean over the positions that count; half precision scales its loss
        st["weight"] = torch.full((B,), (4096.0 if case["dtype"] == "f16" else 1.0) / live, device="cuda")
        st["weight"][pad] = 0.0
        st["ids"], st["values"] = ids, values
        return st
    if case["tokens"]:
        y = torch.randint(0, V, (B, case["tokens"]), generator=g, device="cuda", dtype=torch.int32)
        best = torch.cat([x[r0:r1].argmax(1) for r0, r1 in _pieces(B, V)]).to(torch.int32)
        often = torch.rand(B, generator=g, device="cuda") < 0.5  # half the positions hold the likeliest id
        y[:, 0] = torch.where(often, best, y[:, 0])
        y[pad] = -1
        st["tokens"] = y
    if case["op"] == "score_grad":
        # what the forward pass left: the row's maximum and sum at its temperature, and the entropy
        st["row_max"] = torch.empty(B, dtype=torch.float64, device="cuda")
        st["row_sum"] = torch.empty(B, dtype=torch.float64, device="cuda")
        st["entropy"] = torch.empty(B, device="cuda")
        for r0, r1 in _pieces(B, V):
            z = x[r0:r1].double() / T
            m = z.amax(1, keepdim=True)
            e = torch.exp(z - m)
            s = e.sum(1)
            st["row_max"][r0:r1], st["row_sum"][r0:r1] = m[:, 0], s
            st["entropy"][r0:r1] = torch.log(s) - (e * (z - m)).sum(1) / s
        scale = (4096.0 if case["dtype"] == "f16" else 1.0) / max(1, B - case["padded"])
        st["g_logprobs"] = torch.randn((B, case["tokens"]), generator=g, device="cuda") * scale
        st["g_logprobs"][pad] = 0.0
        if case["entropy"]:
            st["g_entropy"] = torch.full((B,), 0.01 * scale, device="cuda")
            st["g_entropy"][pad] = 0.0
    return st


# ---------------------------------------------------------------- one pass
_handle = None


def _sampler():
    """The framework's handle, made once as a user's program makes it."""
    global _handle
    if _handle is None:
        if "omni.js_b200" not in sys.path:
            sys.path.insert(0, "omni.js_b200")
        from minisample import Sampler

        _handle = Sampler()
    return _handle


def run(st):
    c = st["case"]
    if c["op"] == "score":
        if own:
            o = _sampler().logprobs(st["x"], st.get("tokens"), temperature=c["temperature"], top_n=c["top"],
                                    entropy=c["entropy"])
            return {k: v for k, v in (("logprobs", o.logprobs), ("entropy", o.entropy), ("top_ids", o.top_ids),
                                      ("top_logprobs", o.top_logprobs)) if v is not None}
        return _plain_score(st["x"], st.get("tokens"), c["temperature"], c["top"], c["entropy"])
    if c["op"] == "score_grad":
        if own:
            return _sampler().logprobs_backward(st["x"], st["tokens"], st["row_max"], st["row_sum"],
                                                st["g_logprobs"], st.get("g_entropy"),
                                                st["entropy"] if c["entropy"] else None,
                                                temperature=c["temperature"])
        return _plain_score_grad(st, c["temperature"], c["entropy"])
    if own:
        if c["grad"]:
            loss, dx = _sampler().distill_grad(st["x"], st["ids"], st["values"], st["weight"],
                                               temperature=c["temperature"], kind=c["kind"])
            return {"loss": loss, "dlogits": dx}
        return {"loss": _sampler().distill_loss(st["x"], st["ids"], st["values"], temperature=c["temperature"],
                                                kind=c["kind"])}
    return _plain_distill(st, c["temperature"], c["kind"], c["grad"])


def _plain_score(x, tokens, T, top, entropy):
    V = x.shape[1]
    z = x.float() / T
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    lp = d - torch.log(s)
    out = {}
    live = None
    if tokens is not None:
        valid = (tokens >= 0) & (tokens < V)
        live = valid.any(1)
        got = torch.gather(lp, 1, torch.where(valid, tokens, 0).long())
        out["logprobs"] = torch.where(valid, got, 0.0)
    if entropy:
        h = -torch.where(e > 0, e * lp, 0.0).sum(1) / s[:, 0]
        out["entropy"] = h if live is None else torch.where(live, h, 0.0)
    if top:
        # one whole number for each logit, in the logits' order and then the lowest id first: no two are alike
        bits = (x.float() + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        key |= 0xFFFFFFFF - torch.arange(V, device=x.device)
        ids = 0xFFFFFFFF - (torch.topk(key, min(top, V), dim=1).values & 0xFFFFFFFF)
        best = torch.gather(lp, 1, ids)
        gone = best == -math.inf
        if live is not None:
            gone |= ~live[:, None]
        ids, best = torch.where(gone, -1, ids).int(), torch.where(gone, -math.inf, best)
        out["top_ids"] = torch.nn.functional.pad(ids, (0, top - ids.shape[1]), value=-1)
        out["top_logprobs"] = torch.nn.functional.pad(best, (0, top - best.shape[1]), value=-math.inf)
    return out


def _plain_score_grad(st, T, entropy):
    x, y, g = st["x"], st["tokens"], st["g_logprobs"]
    valid = (y >= 0) & (y < x.shape[1])
    g = torch.where(valid, g, 0.0)
    lp = x.float() / T - st["row_max"].float()[:, None] - torch.log(st["row_sum"]).float()[:, None]
    p = torch.exp(lp)
    c = g.sum(1, keepdim=True)
    if entropy:
        c = c + st["g_entropy"][:, None] * torch.where(p > 0, lp + st["entropy"][:, None], 0.0)
    dx = -p * c
    dx.scatter_add_(1, torch.where(valid, y, 0).long(), g)
    dx = torch.where(valid.any(1, keepdim=True), dx / T, 0.0)
    return dx.to(x.dtype)


def _plain_distill(st, T, kind, grad):
    x, ids = st["x"], st["ids"]
    present = (ids >= 0) & (ids < x.shape[1])
    live = present.any(1, keepdim=True)
    # an absent entry stands on the row's first present id with no mass
    first = torch.gather(ids, 1, present.int().argmax(1, keepdim=True))
    at = torch.where(present, ids, torch.where(live, first, 0)).long()
    v = torch.where(present, st["values"], -math.inf).double()
    if kind == "logits":
        v = v / T
        v = v - torch.where(live, torch.logsumexp(v, 1, keepdim=True), 0.0)
    q = torch.exp(v)
    r = (1.0 - q.sum(1, keepdim=True)) if kind == "logprobs" else torch.zeros_like(q[:, :1])
    r = torch.where(r < _NO_TAIL, 0.0, r)
    z = x.float() / T
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    log_s = torch.log(e.sum(1, keepdim=True).double())
    tail = e.scatter(1, at, 0.0).sum(1, keepdim=True).double() / torch.exp(log_s)
    log_p = torch.gather(d, 1, at).double() - log_s
    loss = torch.where(q > 0, q * (v - log_p), 0.0).sum(1, keepdim=True)
    loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(tail)), 0.0)
    out = {"loss": torch.where(live, loss, 0.0)[:, 0].float()}
    if grad:
        p = e * torch.exp(-log_s).float()
        every = q.sum(1, keepdim=True) + r
        c = (every - torch.where(tail > 0, r / tail, 0.0)).float()
        dx = p * c
        dx.scatter_(1, at, torch.gather(p, 1, at) * every.float())
        dx.scatter_add_(1, at, -q.float())
        dx *= (st["weight"] / T)[:, None]
        out["dlogits"] = torch.where(live, dx, 0.0).to(x.dtype)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    B, V, es = case["rows"], case["vocab"], _SIZES[case["dtype"]]
    read = (B - case["padded"]) * V * es
    if case["op"] == "score":
        small = B * (case["tokens"] * 8 + case["top"] * 8 + (4 if case["entropy"] else 0))
        return {"bytes": read + small, "flops": (B - case["padded"]) * V * 5}
    if case["op"] == "score_grad":
        return {"bytes": read + B * V * es + B * (case["tokens"] * 8 + 24), "flops": (B - case["padded"]) * V * 6}
    small = B * (min(case["teacher"], V) * 8 + 8)
    write = B * V * es if case["grad"] else 0
    return {"bytes": read + write + small, "flops": (B - case["padded"]) * V * (7 if case["grad"] else 4)}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    """Row by row pieces in 64 bits, straight from the definitions."""
    st = prepare(case, seed)
    V, T = case["vocab"], case["temperature"]
    got = [_exact_piece(case, st, r0, r1, V, T) for r0, r1 in _pieces(case["rows"], V)]
    if not isinstance(got[0], dict):
        return torch.cat(got)
    return {k: None if got[0][k] is None else torch.cat([g[k] for g in got]) for k in got[0]}


def _exact_piece(case, st, r0, r1, V, T):
    z = st["x"][r0:r1].double().div_(T)
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    zero = torch.zeros((), dtype=torch.float64, device=z.device)
    out = {}
    if case["op"] != "distill":
        y = st["tokens"][r0:r1].long() if "tokens" in st else None
        keep = torch.ones(r1 - r0, dtype=torch.bool, device=z.device) if y is None else (y >= 0).any(1)
        minus = torch.where(p > 0, p * logp, zero).sum(1).neg()
    if case["op"] == "score":
        if y is not None:
            out["logprobs"] = torch.where(y >= 0, logp.gather(1, y.clamp(min=0)), zero)
        if case["entropy"]:
            out["entropy"] = torch.where(keep, minus, zero)
        if case["top"]:
            n = min(case["top"], V)
            best = logp.topk(n, 1).values
            best = torch.cat([best, best.new_full((r1 - r0, case["top"] - n), -math.inf)], 1)
            out["top_ids"] = None
            out["top_logprobs"] = torch.where(keep[:, None], best, -math.inf)
        return out
    if case["op"] == "score_grad":
        g = torch.where(y >= 0, st["g_logprobs"][r0:r1].double(), zero)
        dz = torch.zeros_like(z).scatter_add_(1, y.clamp(min=0), g) - p * g.sum(1, keepdim=True)
        if case["entropy"]:
            dz -= st["g_entropy"][r0:r1, None].double() * torch.where(p > 0, p * (logp + minus[:, None]), zero)
        return dz.div_(T) * keep[:, None]
    ids, val = st["ids"][r0:r1].long(), st["values"][r0:r1].double()
    there = ids >= 0
    teacher = torch.zeros((r1 - r0, V + 1), dtype=torch.float64, device=z.device)  # one column for absent entries
    mass = torch.where(there, torch.exp(val / (T if case["kind"] == "logits" else 1.0)), zero)
    if case["kind"] == "logits":
        mass = mass / mass.sum(1, keepdim=True).clamp(min=1e-300)
    teacher.scatter_add_(1, torch.where(there, ids, V), mass)
    teacher = teacher[:, :V]
    on = torch.zeros((r1 - r0, V + 1), dtype=torch.bool, device=z.device).scatter_(1, torch.where(there, ids, V), True)
    on = on[:, :V]
    rest = 1.0 - mass.sum(1) if case["kind"] == "logprobs" else torch.zeros(r1 - r0, dtype=torch.float64, device=z.device)
    rest = rest.where(rest >= _NO_TAIL, zero)
    left = torch.where(on, zero, p).sum(1)
    keep = there.any(1)
    kl = torch.where(teacher > 0, teacher * (torch.log(teacher) - logp), zero).sum(1)
    kl += torch.where(rest > 0, rest * (torch.log(rest) - torch.log(left)), zero)
    out["loss"] = torch.where(keep, kl, zero)
    if case["grad"]:
        # the teacher's rest is spread over the ids outside its list as the student spreads its own
        spread = torch.where(on, teacher, p * (rest / left.clamp(min=1e-300))[:, None])
        total = (mass.sum(1) + rest)[:, None]
        dx = (p * total - spread) * (st["weight"][r0:r1].double() / T)[:, None]
        out["dlogits"] = torch.where(keep[:, None], dx, zero)
    return out
