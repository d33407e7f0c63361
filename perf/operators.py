"""Cases of the teacher / student operators: the 8-bit linear head, the selection of a row's largest logits, and the
distillation loss over a teacher's kept logits with its gradient.

`own = False` computes each in its plain form (elementary torch operations in 32 bits, rounded once at the end);
`own = True` makes the calls a user makes of `subreg_hip.functional`.
"""
import functools
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
SPARSE = 0.1                     # share of the rows of a padded batch that hold neither teacher entries nor a label
IGNORE = -100


@functools.lru_cache(maxsize=None)
def _functional():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "subspace-reg_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from subreg_hip import functional
    return functional


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the frozen head of a teacher, 640 features to 351 classes, for a training batch of 64 images (fp32 features)
        dict(name="linear_features", op="linear", rows=64, dim=640, out=351, dtype="f32", bias=True),
        # one token against a large vocabulary: the weights' stream is all there is
        dict(name="linear_token", op="linear", rows=1, dim=4096, out=32768, dtype="bf16", bias=False),
        # a serving batch of tokens: still bound by the weights, but 48 rows share them
        dict(name="linear_batch", op="linear", rows=48, dim=4096, out=16384, dtype="bf16", bias=True),
        # odd everything: rows, features (rows of the weights start at any byte) and classes
        dict(name="linear_ragged", op="linear", rows=333, dim=1111, out=5003, dtype="f16", bias=True),
        # a prompt's tokens: bound by the matrix units
        dict(name="linear_prompt", op="linear", rows=8192, dim=4096, out=8192, dtype="bf16", bias=False),
        # a teacher's five best of 351 classes for a training batch
        dict(name="top_classes", op="top", rows=64, vocab=351, top=5, dtype="f32", wide=False),
        # the best of one token's logits: one row has to be spread over the chip
        dict(name="top_token", op="top", rows=1, vocab=128000, top=64, dtype="bf16", wide=False),
        # a teacher's best of a batch of 2048 tokens
        dict(name="top_batch", op="top", rows=2048, vocab=32000, top=32, dtype="bf16", wide=False),
        # the pretraining step of this repository: 64 images, 60 base classes, fp32 logits, labels beside the teacher
        dict(name="distill_pretrain", op="distill", rows=64, vocab=60, top=10, dtype="f32", temperature=4.0, labels=True, train=True,
             wide=False),
        # a training batch of tokens with padded rows and labels
        dict(name="distill_batch", op="distill", rows=4096, vocab=32000, top=64, dtype="bf16", temperature=2.0, labels=True, train=True,
             wide=False),
        # the longest rows: a large vocabulary, many kept entries, no labels
        dict(name="distill_long", op="distill", rows=1024, vocab=131072, top=128, dtype="bf16", temperature=1.0, labels=False, train=True,
             wide=False),
        # a validation pass: the loss alone, an odd vocabulary in rows of a wider buffer
        dict(name="distill_eval", op="distill", rows=517, vocab=50021, top=50, dtype="f16", temperature=2.0, labels=True, train=False,
             wide=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "top", "distill", "distill"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if op == "linear":
        dim = _log(rng, 64, 8192)
        dim = max(16, dim // 16 * 16) if rng.random() < 0.7 else dim
        out = _log(rng, 40, 65536)
        rows = _log(rng, 1, max(2, min(8192, 8192 * 8192 * 4096 // (dim * out))))
        return dict(op=op, rows=rows, dim=dim, out=out, dtype=dtype, bias=rng.random() < 0.5)
    vocab = _log(rng, 50, 131072)
    rows = _log(rng, 1, min(8192, 2 ** 26 // vocab))
    top = min(vocab, _log(rng, 1, 256))
    wide = rng.random() < 0.25
    if op == "top":
        return dict(op=op, rows=rows, vocab=vocab, top=top, dtype=dtype, wide=wide)
    return dict(op=op, rows=rows, vocab=vocab, top=top, dtype=dtype, temperature=rng.choice((1.0, 2.0, 3.0, 4.0)),
                labels=rng.random() < 0.6, train=rng.random() < 0.75, wide=wide)


def _logits(rows, vocab, dtype, wide, gen):
    """Rows of logits; `wide`: the first `vocab` columns of a buffer padded to a wider vocabulary."""
    cols = vocab + 27 if wide else vocab
    z = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.float32).mul_(2.5).to(TYPES[dtype])
    return z[:, :vocab]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "linear":
        m, k, n = case["rows"], case["dim"], case["out"]
        x = torch.randn(m, k, generator=gen, device="cuda", dtype=torch.float32)
        state["x"] = x.mul_(0.5 + torch.rand(m, 1, generator=gen, device="cuda")).to(TYPES[case["dtype"]])
        w = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float32).mul_(k ** -0.5)
        amax = w.abs().amax(1, keepdim=True)
        state["weight"] = torch.round(w * (127.0 / amax)).clamp_(-127, 127).to(torch.int8)
        state["scale"] = (amax / 127.0).reshape(n)
        state["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        return state
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    state["logits"] = _logits(rows, vocab, case["dtype"], case["wide"], gen)
    if case["op"] == "top":
        return state
    # the teacher agrees with the student in part; some rows keep fewer entries, some rows are padding
    noise = torch.randn(rows, vocab, generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    values, indices = torch.topk(noise.add_(state["logits"], alpha=0.7), top, dim=1)
    kept = 1 + (torch.rand(rows, 1, generator=gen, device="cuda") * 2 * top).long().clamp_(max=top - 1)
    empty = torch.rand(rows, 1, generator=gen, device="cuda") < SPARSE
    drop = (torch.arange(top, device="cuda")[None] >= kept) | empty
    state["top_values"] = values.to(TYPES[case["dtype"]])
    state["top_indices"] = indices.masked_fill(drop, -1)
    state["target"] = None
    if case["labels"]:
        state["target"] = indices[:, 0].masked_fill(empty[:, 0], IGNORE)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
    HF = _functional()
    if s["op"] == "linear":
        return HF.linear_int8(s["x"], s["weight"], s["scale"], bias=s["bias"])
    if s["op"] == "top":
        return HF.top_logits(s["logits"], s["top"])
    z = s["logits"].detach()
    args = dict(target=s["target"], temperature=s["temperature"], ce_weight=0.5 if s["labels"] else 0.0, ignore_index=IGNORE)
    if not s["train"]:
        with torch.no_grad():
            return HF.distill_loss(z, s["top_values"], s["top_indices"], **args)
    z.requires_grad_()
    loss = HF.distill_loss(z, s["top_values"], s["top_indices"], **args)
    loss.backward()
    return loss.detach(), z.grad


def _plain_linear(s):
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    full = torch.full_like(amax, 127.0)                      # (tensor by tensor: both quotients rounded once)
    codes = torch.round(x * torch.div(full, amax)).clamp_(-127, 127)
    y = (codes @ s["weight"].float().t()) * torch.div(amax, full) * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_top(s):
    z, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    return z[:, :s["top"]].to(s["logits"].dtype), order[:, :s["top"]]


def _log_probs(z):
    z = z - z.amax(1, keepdim=True)
    return z - z.exp().sum(1, keepdim=True).log()


def _plain_distill(s):
    z, t, idx, temp = s["logits"].float(), s["top_values"].float(), s["top_indices"], s["temperature"]
    keep = (idx >= 0) & (t > -math.inf)
    row = keep.any(1)
    n_kd = row.sum().clamp_min(1)
    t = torch.where(keep, t / temp, -math.inf)
    t = t - torch.where(row, t.amax(1), 0.0)[:, None]
    p = t.exp()
    total = torch.where(row, p.sum(1), 1.0)[:, None]
    p = p / total
    logq = _log_probs(z / temp)
    at = idx.clamp_min(0)
    kl = torch.where(keep, p * (t - total.log() - logq.gather(1, at)), 0.0).sum(1)
    loss = temp * temp * kl.sum() / n_kd
    dz = None
    if s["train"]:
        w = temp / n_kd
        dz = logq.exp_().mul_(row[:, None] * w).scatter_add_(1, at, -p * w)
    del logq
    if s["labels"]:
        y = s["target"]
        has = y != IGNORE
        n_ce = has.sum().clamp_min(1)
        logp = _log_probs(z)
        y = y.clamp_min(0)[:, None]
        loss = loss - 0.5 * torch.where(has, logp.gather(1, y)[:, 0], 0.0).sum() / n_ce
        if s["train"]:
            w = (has * 0.5 / n_ce)[:, None]
            dz = dz.add_(logp.exp_().mul_(w)).scatter_add_(1, y, -w)
    return (loss, dz.to(s["logits"].dtype)) if s["train"] else loss


def run(state):
    if own:
        return _run_own(state)
    return {"linear": _plain_linear, "top": _plain_top, "distill": _plain_distill}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e, rows = SIZE[case["dtype"]], case["rows"]
    if case["op"] == "linear":
        k, n = case["dim"], case["out"]
        return {"bytes": rows * k * e + n * k + 4 * n * (2 if case["bias"] else 1) + rows * n * e, "flops": 2 * rows * n * k}
    v, top = case["vocab"], case["top"]
    if case["op"] == "top":
        return {"bytes": rows * v * e + rows * top * (e + 8), "flops": rows * v}
    exps = 2 if case["labels"] and case["temperature"] != 1.0 else 1
    read, write = (1.0 - SPARSE) * rows * v * e, rows * v * e if case["train"] else 0
    return {"bytes": read + write + rows * top * (e + 8) + (8 * rows if case["labels"] else 0), "flops": rows * v * (3 + 3 * exps)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_linear(s):
    x, w = s["x"].double(), s["weight"].double()
    top = torch.maximum(x.abs().max(dim=1).values, torch.tensor(2.0 ** -100, device=x.device, dtype=torch.float64))
    inverse = (127.0 / top).float().double()                 # the definition holds 127 / max, max / 127 and the product in 32 bits
    step = (top / 127.0).float().double()
    codes = (x * inverse[:, None]).float().double().round()
    y = torch.mm(codes, w.t().contiguous()) * torch.outer(step, s["scale"].double())
    return y if s["bias"] is None else y + s["bias"].double()[None]


def _exact_rows(z, t, idx, y, temp):
    """KL and CE of some rows and d KL / dz, d CE / dz, in 64 bits."""
    z, t = z.double(), t.double()
    kept = (idx >= 0).double()
    weight = torch.exp((t - t.max(dim=1, keepdim=True).values) / temp) * kept
    mass = weight.sum(dim=1, keepdim=True)
    weight = weight / torch.where(mass > 0, mass, torch.ones_like(mass))
    q = torch.softmax(z / temp, dim=1)
    at = idx.clamp(min=0)
    ratio = torch.where(weight > 0, weight / q.gather(1, at), torch.ones_like(weight))
    kl = (weight * torch.log(ratio)).sum(dim=1)
    some = (mass > 0).double()
    dkl = (q * some).scatter_add(1, at, -weight) / temp
    ce, dce = torch.zeros_like(kl), 0.0
    if y is not None:
        has = (y != IGNORE).double()
        s = torch.softmax(z, dim=1)
        label = y.clamp(min=0)[:, None]
        ce = -torch.log(s.gather(1, label))[:, 0] * has
        dce = (s.scatter_add(1, label, -torch.ones_like(label, dtype=torch.float64))) * has[:, None]
    return kl, ce, dkl, dce


def _exact_distill(s):
    z, t, idx, y, temp = s["logits"], s["top_values"], s["top_indices"], s["target"], s["temperature"]
    n_kd = max(1, int((idx >= 0).any(dim=1).sum()))
    n_ce = 1 if y is None else max(1, int((y != IGNORE).sum()))
    kls, ces, grads = [], [], []
    step = max(1, 2 ** 25 // z.shape[1])
    for lo in range(0, z.shape[0], step):
        cut = slice(lo, lo + step)
        kl, ce, dkl, dce = _exact_rows(z[cut], t[cut], idx[cut], None if y is None else y[cut], temp)
        kls.append(kl)
        ces.append(ce)
        if s["train"]:
            grads.append(temp * temp * dkl / n_kd + 0.5 * dce / n_ce)
    loss = temp * temp * torch.cat(kls).sum() / n_kd + 0.5 * torch.cat(ces).sum() / n_ce
    return (loss, torch.cat(grads)) if s["train"] else loss


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(state)
    if case["op"] == "top":
        return torch.topk(state["logits"].double(), case["top"], dim=1, sorted=True).values, None
    return _exact_distill(state)
