"""Performance cases of the token-score and top-k distillation operators: what
is timed, on which inputs, and what it must compute.

The operators are the device-pointer entry points of the C-ABI
(`include/seeml_hip.h`) that score given tokens under a model's logits and
train a student on what such a score reports of its teacher:

  score      `seeml_hip_token_logprobs_fwd`: the log probability of each row's
             token, the row's entropy and its k likeliest classes. What a
             teacher's pass stores, what an evaluation reports.
  policy     the same, then `seeml_hip_token_logprobs_bwd`: the gradient of
             any function of the log probabilities and entropies.
  distill    `seeml_hip_topk_distill_fwd_bwd`: the KL divergence of the student
             from the teacher's k likeliest classes (renormalised, or with
             the rest of the classes as one more), with its gradient.
  validate   `seeml_hip_topk_distill_fwd`: that loss alone.
  replay     `seeml_hip_topk_distill_fwd`, then `seeml_hip_topk_distill_bwd`
             for a gradient that arrives later.

Sizes are those of the repository's own workloads (vocabularies of 256 to 32000
classes, batches of 32 to 8192 rows), the wider vocabularies of current
tokenizers up to 131072 classes, and ragged sizes between them.
"""
import math
import os
import sys

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One row of one sequence: latency of a single token's score.
        dict(name="score_1x32000", kind="score", rows=1, classes=32000, type="f32", k=20, T=1.0,
             pad=0, masked=False, padded=False),
        # One decoding step of 24 sequences over a wide vocabulary whose last
        # classes no token uses.
        dict(name="score_24x131072_bf16", kind="score", rows=24, classes=131072, type="bf16", k=8,
             T=0.7, pad=0, masked=True, padded=False),
        # A teacher's pass over the d_model-2048 decoder's own batch, 8 x 1024.
        dict(name="score_8192x32000", kind="score", rows=8192, classes=32000, type="f32", k=32,
             T=1.0, pad=0, masked=False, padded=True),
        # Sizes that divide by nothing, rows of a wider buffer.
        dict(name="score_777x10007_f16", kind="score", rows=777, classes=10007, type="f16", k=64,
             T=1.3, pad=5, masked=False, padded=True),
        # A policy update on sampled tokens with an entropy bonus.
        dict(name="policy_4096x32000", kind="policy", rows=4096, classes=32000, type="f32", k=0,
             T=1.0, pad=0, masked=False, padded=True),
        dict(name="policy_333x8191_bf16", kind="policy", rows=333, classes=8191, type="bf16", k=4,
             T=0.9, pad=1, masked=True, padded=True),
        # A distillation step at the d_model-2048 decoder's own batch: the largest.
        dict(name="distill_8192x32000", kind="distill", rows=8192, classes=32000, type="f32", k=64,
             T=2.0, tail=True, pad=0, masked=False, padded=True),
        # The small decoder's vocabulary, renormalised; the gradient in its own call.
        dict(name="replay_2048x8192", kind="replay", rows=2048, classes=8192, type="f32", k=16,
             T=1.0, tail=False, pad=0, masked=False, padded=False),
        # Ragged sizes and short lists, 16-bit logits.
        dict(name="distill_600x1999_bf16", kind="distill", rows=600, classes=1999, type="bf16",
             k=50, T=1.5, tail=True, pad=0, masked=False, padded=True),
        # Few rows of a wide vocabulary.
        dict(name="distill_40x131072_bf16", kind="distill", rows=40, classes=131072, type="bf16",
             k=100, T=1.0, tail=True, pad=0, masked=True, padded=False),
        # The loss of a validation batch.
        dict(name="validate_2048x32000", kind="validate", rows=2048, classes=32000, type="f32",
             k=32, T=1.0, tail=True, pad=0, masked=False, padded=True),
        # A loss that is one term of several, its gradient scaled for 16 bits.
        dict(name="replay_1024x50001_f16", kind="replay", rows=1024, classes=50001, type="f16",
             k=8, T=1.0, tail=False, pad=7, masked=False, padded=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "policy", "distill", "distill", "validate", "replay"])
    classes = rng.choice([_log(rng, 100, 131072), _log(rng, 1000, 131072), 8192, 32000])
    rows = _log(rng, 1, max(2, min(8192, 131072000 // classes)))
    case = dict(kind=kind, rows=rows, classes=classes,
                type=rng.choice(["f32", "f32", "bf16", "f16"]),
                k=min(_log(rng, 1, 128), classes // 2), T=round(rng.uniform(0.5, 3.0), 2),
                pad=rng.choice([0, 0, 1, 8, 13]), masked=rng.random() < 0.3,
                padded=rng.random() < 0.5)
    if kind in ("score", "policy"):
        case["k"] = rng.choice([0, case["k"], case["k"]])
    else:
        case["tail"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(1000003 * int(seed) + 29)
    N, C, k, T = case["rows"], case["classes"], case["k"], case["T"]
    randn = lambda *s: torch.randn(*s, generator=g, device=_DEV)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device=_DEV)  # noqa: E731
    # Logits of a language model: a broad floor and a few likely classes.
    x = randn(N, C).mul_(2.0)
    likely = torch.randint(0, C, (N, 8), generator=g, device=_DEV)
    x.scatter_add_(1, likely, rand(N, 8) * 9.0)
    if case["masked"]:  # the last classes are no tokens
        x[:, C - C // 16:] = -math.inf
    buf = torch.zeros(N, C + case["pad"], device=_DEV, dtype=_TYPES[case["type"]])
    buf[:, :C] = x
    s = dict(case=case, logits=buf[:, :C])
    # Half-precision gradients are kept in range by a scaled loss.
    up = 256.0 * N if case["type"] == "f16" else 1.0
    real = torch.ones(N, device=_DEV, dtype=torch.bool)
    if case["padded"]:  # rows behind a sequence's end, the first row never
        real[1:] = rand(N)[1:] >= 0.125
    if case["kind"] in ("score", "policy"):
        named = torch.where(rand(N) < 0.7, likely[:, 0],
                            torch.randint(0, max(1, C - C // 16), (N,), generator=g, device=_DEV))
        if case["masked"]:
            named = named.clamp(max=C - C // 16 - 1)
        s["targets"] = torch.where(real, named, -1).int()
        if case["kind"] == "policy":
            s["dlogp"] = randn(N) * (up / N)
            s["dentropy"] = torch.full((N,), -0.01 * up / N, device=_DEV)
        return s
    # The teacher's likeliest classes at the same temperature, some lists short.
    t = x.add_(randn(N, C).mul_(0.7)).div_(T)
    lse = torch.logsumexp(t, -1, keepdim=True)
    top, ids = torch.topk(t, k, -1)
    kept = torch.isfinite(top)
    short = torch.where(rand(N) < 0.125, (rand(N) * k).long() + 1, k)
    kept &= torch.arange(k, device=_DEV)[None, :] < short[:, None]
    s["t_ids"] = torch.where(kept, ids, -1).int()
    s["t_logp"] = torch.where(kept, top - lse, 0.0)
    s["weight"] = torch.where(real, 1.0 / real.sum(), 0.0).float()
    s["seed"] = torch.full((1,), up * (0.7 if case["kind"] == "replay" else 1.0), device=_DEV)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    """The calls of a user's program: outputs and scratch from torch's
    allocator, the current stream."""
    path = os.path.join(os.getcwd(), "see-ml_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from seeml_amd import lib
    L, c, x = lib(), s["case"], s["logits"]
    N, C, k, T, stride = c["rows"], c["classes"], c["k"], c["T"], x.stride(0)
    dtype = {"f32": 0, "bf16": 1, "f16": 2}[c["type"]]
    new = lambda *shape: torch.empty(*shape, device=_DEV)  # noqa: E731
    at = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream

    def call(name, *args):
        args = [at(a) if a is None or isinstance(a, torch.Tensor) else a for a in args]
        if getattr(L, "seeml_hip_" + name)(*args, stream) != 0:
            raise RuntimeError("%s: %s" % (name, L.seeml_hip_kernel_error().decode()))

    if c["kind"] in ("score", "policy"):
        logp, entropy = new(N), new(N)
        top_ids = torch.empty(N, k, device=_DEV, dtype=torch.int32) if k else None
        top_logp = new(N, k) if k else None
        stats = new(N, 4) if c["kind"] == "policy" else None
        nbytes = L.seeml_hip_token_logprobs_scratch(N, C, dtype, k)
        scratch = torch.empty(nbytes, device=_DEV, dtype=torch.uint8) if nbytes else None
        call("token_logprobs_fwd", x, dtype, stride, s["targets"], T, k, logp, entropy, stats,
             top_ids, top_logp, N, C, scratch, nbytes)
        out = dict(logp=logp, entropy=entropy)
        if k:
            out.update(top_ids=top_ids, top_logp=top_logp)
        if c["kind"] == "policy":
            dx = torch.empty(N, C, device=_DEV, dtype=x.dtype)
            call("token_logprobs_bwd", x, dtype, stride, s["targets"], T, stats, s["dlogp"],
                 s["dentropy"], dx, C, N, C)
            out["dlogits"] = dx
        return out
    loss, row_loss = new(1), new(N)
    tail = 1 if c["tail"] else 0
    nbytes = L.seeml_hip_topk_distill_scratch(N, C, dtype, k)
    scratch = torch.empty(nbytes, device=_DEV, dtype=torch.uint8) if nbytes else None
    head = (x, dtype, stride, s["t_ids"], s["t_logp"], k, s["weight"])
    if c["kind"] == "validate":
        call("topk_distill_fwd", *head, T, tail, loss, row_loss, None, N, C, scratch, nbytes)
        return dict(loss=loss, row_loss=row_loss)
    dx = torch.empty(N, C, device=_DEV, dtype=x.dtype)
    if c["kind"] == "distill":
        call("topk_distill_fwd_bwd", *head, s["seed"], T, tail, loss, row_loss, dx, C, N, C,
             scratch, nbytes)
    else:
        stats = new(N, 8)
        call("topk_distill_fwd", *head, T, tail, loss, row_loss, stats, N, C, scratch, nbytes)
        call("topk_distill_bwd", *head, s["seed"], T, tail, stats, dx, C, N, C)
    return dict(loss=loss, row_loss=row_loss, dlogits=dx)


def _softmax_parts(x, T):
    """max, (x - max) / T, its exponential and the exponentials' sum, 32 bits."""
    m = x.amax(-1, keepdim=True)
    d = (x - m) / T
    e = torch.exp(d)
    return d, e, e.sum(-1, keepdim=True)


def _plain(s):
    c = s["case"]
    x = s["logits"].float()
    C, k, T = c["classes"], c["k"], c["T"]
    d, e, total = _softmax_parts(x, T)
    log_total = torch.log(total)
    if c["kind"] in ("score", "policy"):
        tgt = s["targets"].long()
        scored = tgt >= 0
        at = tgt.clamp(min=0)[:, None]
        logp = torch.where(scored, (d.gather(1, at) - log_total)[:, 0], 0.0)
        mean = (e * torch.where(e > 0, d, 0.0)).sum(-1, keepdim=True) / total
        entropy = log_total - mean
        out = dict(logp=logp, entropy=entropy[:, 0])
        if k:  # by value, ties by the lowest class: one whole number orders both
            bits = (x + 0.0).view(torch.int32)
            bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
            key = (bits << 32) + (C - 1 - torch.arange(C, device=x.device))
            ids = C - 1 - (torch.topk(key, k, -1).values & 0xFFFFFFFF)
            live = torch.isfinite(x.gather(1, ids))
            out["top_ids"] = torch.where(live, ids, -1).int()
            out["top_logp"] = d.gather(1, ids) - log_total
        if c["kind"] == "policy":
            p = e / total
            lp = torch.where(p > 0, d - log_total, 0.0)
            a = torch.where(scored, s["dlogp"], 0.0)[:, None]
            g = -p * (a + s["dentropy"][:, None] * (lp + entropy))
            g.scatter_add_(1, at, a)
            out["dlogits"] = (g / T).to(s["logits"].dtype)
        return out
    ids, v, w = s["t_ids"].long(), s["t_logp"], s["weight"]
    kept = ids >= 0
    at = ids.clamp(min=0)
    # The lists are short and their terms cancel: 64 bits.
    log_q = torch.where(kept, v, 0.0).double()
    q = torch.where(kept, torch.exp(log_q), 0.0)
    if not c["tail"]:
        mass = q.sum(-1, keepdim=True)
        q, log_q = q / mass, log_q - torch.log(mass)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    lp = (x.gather(1, at).double() - x.amax(-1, keepdim=True)) / T - torch.log(total)
    row = torch.where(kept, q * (log_q - lp), 0.0).sum(-1)
    p = e / total.float()
    if c["tail"]:
        listed_ = torch.zeros(x.shape[0], C + 1, device=x.device, dtype=torch.bool)
        listed_ = listed_.scatter_(1, torch.where(kept, ids, C), True)[:, :C]
        qt = (1.0 - q.sum(-1, keepdim=True)).clamp(min=0)
        pt = torch.where(listed_, 0.0, e).sum(-1, keepdim=True, dtype=torch.float64) / total
        row = row + torch.where(qt > 0, qt * (torch.log(qt) - torch.log(pt)), 0.0)[:, 0]
        g = torch.where(listed_, p, p * (1.0 - qt / pt).float())
    else:
        g = p
    row = torch.where(w != 0, row.float(), 0.0)
    loss = (w * row).sum().reshape(1)
    if c["kind"] == "validate":
        return dict(loss=loss, row_loss=row)
    g.scatter_add_(1, at, -q.float())
    g = g * (w * s["seed"] / T)[:, None]
    return dict(loss=loss, row_loss=row, dlogits=g.to(s["logits"].dtype))


# ------------------------------------------------- the work of one pass

def work(case):
    """The logits read once, the gradient written once, the rows' short inputs
    and outputs. Per logit: scaled difference, exponential, sum, and the
    entropy's or the gradient's product."""
    N, C, k = case["rows"], case["classes"], case["k"]
    size = 4 if case["type"] == "f32" else 2
    grad = case["kind"] in ("policy", "distill", "replay")
    return dict(bytes=N * (C * size * (2 if grad else 1) + 8 * k + 24),
                flops=N * C * (8.0 if grad else 5.0))


# -------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    z = s["logits"].double() / case["T"]
    log_p = torch.log_softmax(z, -1)
    del z
    rows = torch.arange(case["rows"], device=_DEV)
    if case["kind"] in ("score", "policy"):
        ask = s["targets"].long()
        some = (ask >= 0).double()
        p = log_p.exp()
        h = -torch.special.xlogy(p, p).sum(-1)
        out = dict(logp=log_p[rows, ask.clamp(min=0)].masked_fill(ask < 0, 0.0), entropy=h)
        if case["k"]:
            out["top_ids"] = None
            out["top_logp"] = torch.topk(log_p, case["k"], -1).values
        if case["kind"] == "policy":
            up, bonus = s["dlogp"].double() * some, s["dentropy"].double()
            g = -up[:, None] * p - bonus[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            g[rows, ask.clamp(min=0)] += up
            out["dlogits"] = g / case["T"]
        return out
    ids, v, w = s["t_ids"].long(), s["t_logp"].double(), s["weight"].double()
    empty = ids < 0
    v = v.masked_fill(empty, -math.inf)
    if not case["tail"]:
        v = torch.log_softmax(v, -1)
    q = v.exp()
    spot = ids.masked_fill(empty, 0)
    row = (torch.special.xlogy(q, q) - q * log_p.gather(1, spot).masked_fill(empty, 0.0)).sum(-1)
    aim = torch.zeros_like(log_p).scatter_add_(1, spot, q)  # the teacher over all classes
    if case["tail"]:
        rest = torch.ones_like(log_p, dtype=torch.bool)
        keep = torch.zeros_like(log_p).scatter_add_(1, spot, (~empty).double())
        rest &= keep == 0
        del keep
        left = (1.0 - q.sum(-1)).clamp(min=0)
        inside = log_p.masked_fill(~rest, -math.inf)
        log_left = torch.logsumexp(inside, -1)
        row = row + torch.special.xlogy(left, left) - left * log_left.masked_fill(left == 0, 0.0)
        aim += left[:, None] * (inside - log_left[:, None]).exp()
    row = row.masked_fill(w == 0, 0.0)
    out = dict(loss=(w * row).sum().reshape(1), row_loss=row)
    if case["kind"] != "validate":
        g = log_p.exp() - aim
        out["dlogits"] = g * (w * s["seed"].double() / case["T"])[:, None]
    return out
