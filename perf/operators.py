"""The work that the scores and losses over a vocabulary are measured on: log probabilities of given tokens with entropy and top
alternatives, and distillation from a teacher's top logits.

    listed()           the cases that are always measured
    draw(rng)          one more case of the same ranges
    prepare(case, s)   what a program holds before the call: seeded logits, tokens, teacher entries, weights, output buffers
    run(state)         one pass; in plain torch operations, or through the library's entry points where `own` is true
    work(case)         bytes and floating-point operations the pass cannot do without
    exact(case, s)     what run returns, from the definition in 64 bits

kinds:  score          token_logprobs_: log probability of the token (targets), entropy, `top` alternatives
        policy         token_logprobs_ with entropy, then grad_token_logprobs_: the weights depend on the forward's result
        nll            token_logprobs_with_grad_: weights known in advance, value and gradient in one call
        distill        distill_: the loss alone
        distill_grad   distill_, then grad_distill_
        distill_train  distill_with_grad_: value and gradient in one call
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
DEV = "cuda"
LARGEST = 4096 * 131072          # logits of the largest case


def _library():
    """The package directory's name holds a dot, so it is loaded by path."""
    if "tylo_b200" not in sys.modules:
        pkg = ROOT / "tylo.jl_b200"
        spec = importlib.util.spec_from_file_location("tylo_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["tylo_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["tylo_b200"]


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def _case(name, kind, dtype, rows, vocab, *, top=0, targets=True, entropy=False, temperature=1.0, masked=False, pad=0, renormalize=True):
    return dict(name=name, kind=kind, dtype=dtype, rows=rows, vocab=vocab, top=top, targets=targets, entropy=entropy,
                temperature=temperature, masked=masked, pad=pad, renormalize=renormalize)


def listed():
    return [
        # one decoded token: its log probability, the entropy and twenty alternatives; launch and host latency
        _case("token_answer", "score", "bf16", 1, 32768, top=20, entropy=True),
        # a full batch of decoded tokens over a large vocabulary
        _case("batch_answer", "score", "bf16", 64, 131072, top=20, entropy=True, temperature=0.8),
        # grammar-constrained decoding: almost every logit is -Inf, fewer are left than alternatives asked for
        _case("constrained", "score", "f16", 256, 32000, top=64, masked=True),
        # the log probabilities of a prompt, nothing else
        _case("prompt_score", "score", "bf16", 2048, 131072),
        # a teacher writes down its top logits for distillation: an odd vocabulary in a padded buffer
        _case("teacher_top", "score", "bf16", 2048, 100003, top=128, targets=False, pad=5),
        # policy gradient with an entropy bonus: the weights are computed from the log probabilities, so two calls
        _case("policy_train", "policy", "bf16", 4096, 65536, entropy=True),
        # the same for a small Float32 model with an odd vocabulary
        _case("policy_fp32", "policy", "f32", 777, 50001, entropy=True, temperature=0.7),
        # next-token training: value and gradient in one call
        _case("nll_train", "nll", "bf16", 4096, 32768),
        # distillation loss of a held-out batch
        _case("distill_eval", "distill", "bf16", 512, 131072, top=64),
        # distillation with the teacher's own mass kept, half precision, an odd vocabulary, two calls
        _case("distill_small", "distill_grad", "f16", 96, 32001, top=17, temperature=2.0, renormalize=False),
        # distillation training over a large vocabulary
        _case("distill_train", "distill_train", "bf16", 4096, 131072, top=128, temperature=1.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "score", "policy", "nll", "distill", "distill_grad", "distill_train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _log_int(rng, 1000, 262144) if rng.random() < 0.5 else _log_int(rng, 125, 32768) * 8
    rows = min(_log_int(rng, 1, 8192), max(1, LARGEST // vocab // (SIZE[dtype] // 2)))
    top = _log_int(rng, 1, 256)
    c = dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, top=0, targets=True, entropy=False,
             temperature=rng.choice([1.0, 1.0, 0.6, 2.0]), masked=False, pad=rng.choice([0, 0, 0, 7, 64]), renormalize=True)
    if kind == "score":
        c.update(top=rng.choice([0, top, top]), entropy=rng.random() < 0.5, masked=rng.random() < 0.2)
        c["targets"] = c["top"] == 0 or rng.random() < 0.7
        if c["top"]:      # the top alternatives' plain form holds a 64-bit key per logit
            c["rows"] = min(c["rows"], max(1, LARGEST // 2 // vocab))
    elif kind == "policy":
        c["entropy"] = True
    elif kind != "nll":
        c.update(top=top, renormalize=rng.random() < 0.7)
    return c


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    N, M, K, dt = c["rows"], c["vocab"], c["top"], TYPES[c["dtype"]]
    g = torch.Generator(DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    rows = torch.arange(N, device=DEV)
    # logits: tokens with low ids are more frequent; some rows are sure of their token and others are not
    x = normal(N, M).mul_(2.5).sub_(torch.arange(M, device=DEV, dtype=torch.float32).mul_(8.0 / M).add_(1.0).log_().mul_(2.0))
    target = torch.randint(0, M, (N,), generator=g, device=DEV)
    x[rows, target] += normal(N).mul_(6.0).add_(4.0)
    s = dict(case=c, target=target.to(torch.int32))
    if c["masked"]:         # what a grammar allows at a place: a few dozen tokens, the token among them
        live = torch.rand(N, M, generator=g, device=DEV) < 40.0 / M
        live[rows, target] = True
        x.masked_fill_(~live, -math.inf)
    distill = c["kind"].startswith("distill")
    if distill:             # K different entries per row, the teacher's values falling; every eighth row has fewer than K
        step = 1 + torch.randint(0, max(1, M // K), (N, 1), generator=g, device=DEV)
        index = (target[:, None] + torch.arange(K, device=DEV) * step) % M
        index = torch.where(torch.arange(K, device=DEV) * step < M, index, -1)
        value = normal(N, K).mul_(3.0).sort(dim=1, descending=True).values
        if not c["renormalize"]:       # log probabilities that leave a tenth of the mass to the rest
            value = torch.log_softmax(value, 1) + math.log(0.9)
        x.scatter_add_(1, index.clamp(min=0), value * 0.5)
        if K > 2:
            index[::8, -2:] = -1
        s["index"], s["value"] = index.to(torch.int32), value
    if c["pad"]:            # rows of a wider buffer
        buf = torch.zeros(N, M + c["pad"], dtype=dt, device=DEV)
        buf[:, :M] = x
        s["X"] = buf[:, :M]
        s["dX"] = torch.zeros(N, M + c["pad"], dtype=dt, device=DEV)[:, :M]
    else:
        s["X"] = x.to(dt)
        s["dX"] = torch.empty_like(s["X"])
    del x
    s["weight"] = normal(N)
    s["entropy_weight"] = torch.full((N,), 0.1, device=DEV)
    f32 = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=DEV)
    s["out"], s["entropy"], s["M"], s["L"] = f32(N), f32(N), f32(N), f32(N)
    if c["kind"] == "score" and K:
        s["top_logp"], s["top_index"] = f32(N, K), torch.empty(N, K, dtype=torch.int32, device=DEV)
    if c["kind"] in ("score", "distill"):
        del s["dX"]
    return s


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def _softmax_parts(X, temperature):
    """(z - max z, sum of its exponentials), z = X / temperature in 32 bits."""
    y = X.float()
    y = (y - y.amax(1, keepdim=True)) / temperature
    return y, y.exp().sum(1, keepdim=True)


def _entropy(y, total):
    """-sum p log p with p = exp(y) / total; entries without probability leave nothing."""
    return total.log()[:, 0] - torch.where(y > -200.0, y.exp() * y, 0.0).sum(1) / total[:, 0]


def _top(X, K):
    """Indices of the K largest entries of each row, the lowest index first among equals: keys of value and index, all different."""
    bits = (X.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -2147483648 - bits - 1)
    return torch.topk(order * (1 << 32) + ((1 << 31) - torch.arange(X.shape[1], device=X.device)), K, dim=1).indices


def _plain_logprobs(s, c):
    y, total = _softmax_parts(s["X"], c["temperature"])
    logsum = total.log()
    out = {}
    if c["targets"]:
        out["logp"] = y.gather(1, s["target"].long()[:, None])[:, 0] - logsum[:, 0]
    if c["entropy"]:
        out["entropy"] = _entropy(y, total)
    if c["kind"] == "score" and c["top"]:
        index = _top(s["X"], c["top"])
        out["top_logp"], out["top_index"] = y.gather(1, index) - logsum, index.to(torch.int32)
    if c["kind"] in ("policy", "nll"):
        logp = y - logsum
        p = logp.exp()
        d = p * -s["weight"][:, None]
        if c["entropy"]:
            d -= s["entropy_weight"][:, None] * p * (logp + out["entropy"][:, None])
        d.scatter_add_(1, s["target"].long()[:, None], s["weight"][:, None])
        out["dX"] = (d / c["temperature"]).to(s["X"].dtype)
    return out


def _plain_distill(s, c):
    y, total = _softmax_parts(s["X"], c["temperature"])
    live = s["index"] >= 0
    at = s["index"].long().clamp(min=0)
    v = torch.where(live, s["value"] / c["temperature"] if c["renormalize"] else s["value"], -math.inf)
    if c["renormalize"]:
        v = v - v.amax(1, keepdim=True)
        v = v - v.exp().sum(1, keepdim=True).log()
    p = v.exp()
    logq = y.gather(1, at) - total.log()
    out = {"loss": torch.where(live, p * (v - logq), 0.0).sum(1)}
    if c["kind"] != "distill":
        w = s["weight"][:, None] / c["temperature"]
        d = y.exp() * (p.sum(1, keepdim=True) / total * w)
        d.scatter_add_(1, at, -p * w)
        out["dX"] = d.to(s["X"].dtype)
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return (_plain_distill if c["kind"].startswith("distill") else _plain_logprobs)(s, c)
    t = _library()
    kind, dup, tau = c["kind"], t.Duplicated, c["temperature"]
    if kind == "score":
        top = t.TopAlternatives(s["top_logp"], s["top_index"]) if c["top"] else None
        t.token_logprobs_(s["out"] if c["targets"] else None, s["X"], s["target"] if c["targets"] else None, temperature=tau,
                          entropy=s["entropy"] if c["entropy"] else None, top=top)
        out = {"logp": s["out"]} if c["targets"] else {}
        if c["entropy"]:
            out["entropy"] = s["entropy"]
        if top is not None:
            out.update(top_logp=top.logp, top_index=top.index)
        return out
    if kind == "policy":
        cp = t.LogprobCheckpoints(s["M"], s["L"])
        t.token_logprobs_(s["out"], s["X"], s["target"], temperature=tau, entropy=s["entropy"], checkpoints=cp)
        t.grad_token_logprobs_(dup(s["out"], s["weight"]), dup(s["X"], s["dX"]), s["target"], temperature=tau, checkpoints=cp,
                               entropy=dup(s["entropy"], s["entropy_weight"]))
        return {"logp": s["out"], "entropy": s["entropy"], "dX": s["dX"]}
    if kind == "nll":
        t.token_logprobs_with_grad_(dup(s["out"], s["weight"]), dup(s["X"], s["dX"]), s["target"], temperature=tau)
        return {"logp": s["out"], "dX": s["dX"]}
    how = dict(temperature=tau, renormalize=c["renormalize"], teacher_temperature=None if c["renormalize"] else 1.0)
    if kind == "distill":
        t.distill_(s["out"], s["X"], s["value"], s["index"], **how)
        return {"loss": s["out"]}
    if kind == "distill_grad":
        cp = t.LogprobCheckpoints(s["M"], s["L"])
        t.distill_(s["out"], s["X"], s["value"], s["index"], checkpoints=cp, **how)
        t.grad_distill_(dup(s["out"], s["weight"]), dup(s["X"], s["dX"]), s["value"], s["index"], checkpoints=cp, **how)
    else:
        t.distill_with_grad_(dup(s["out"], s["weight"]), dup(s["X"], s["dX"]), s["value"], s["index"], **how)
    return {"loss": s["out"], "dX": s["dX"]}


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    N, M, K = c["rows"], c["vocab"], c["top"]
    x = N * M * SIZE[c["dtype"]]
    gradient = c["kind"] not in ("score", "distill")
    nbytes = x * (2 if gradient else 1) + 8 * N * c["targets"] + 4 * N * c["entropy"] + 8 * N * K + 4 * N * gradient
    return dict(bytes=nbytes, flops=N * M * (4 + 2 * c["entropy"] + 4 * gradient))


# ---------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    N, M, K, tau = case["rows"], case["vocab"], case["top"], float(case["temperature"])
    out = {}
    add = lambda name, value: out.setdefault(name, []).append(value)
    some = max(1, (1 << 26) // M)
    for at in range(0, N, some):
        cut = slice(at, at + some)
        x = s["X"][cut].double()
        logq = torch.log_softmax(x / tau, dim=1)
        q = logq.exp()
        n = x.shape[0]
        w = s["weight"][cut].double()[:, None]
        if case["kind"].startswith("distill"):
            index, value = s["index"][cut].long(), s["value"][cut].double()
            if case["renormalize"]:
                value = value / tau
            p = torch.where(index < 0, 0.0, value.exp())
            if case["renormalize"]:
                p = p / p.sum(dim=1, keepdim=True)
            teacher = torch.zeros(n, M + 1, dtype=torch.float64, device=DEV)        # entries that are left out go to column M
            teacher.scatter_add_(1, torch.where(index < 0, M, index), p)
            teacher = teacher[:, :M]
            add("loss", torch.where(teacher > 0, teacher * (teacher.log() - logq), 0.0).sum(dim=1))
            if case["kind"] != "distill":
                add("dX", (q * teacher.sum(dim=1, keepdim=True) - teacher) * w / tau)
            continue
        token = torch.zeros(n, M, dtype=torch.bool, device=DEV)
        token[torch.arange(n, device=DEV), s["target"][cut].long()] = True
        H = torch.where(q > 0, -q * logq, 0.0).sum(dim=1)
        if case["targets"]:
            add("logp", logq[token])
        if case["entropy"]:
            add("entropy", H)
        if case["kind"] == "score" and K:
            index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :K]
            add("top_logp", torch.take_along_dim(logq, index, dim=1))
            add("top_index", index.int())
        if case["kind"] in ("policy", "nll"):
            d = w * (token.double() - q)
            if case["entropy"]:
                d = d - s["entropy_weight"][cut].double()[:, None] * torch.where(q > 0, q * (logq + H[:, None]), 0.0)
            add("dX", d / tau)
    return {name: torch.cat(parts) for name, parts in out.items()}
