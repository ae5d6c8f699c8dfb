"""The vocabulary operators of raft_b200.linalg as they are measured: their cases, inputs and plain forms.

Four operators around the vocabulary axis of a language model, each next to a reduction the library has:

  lookup   rows of an embedding table by token, scaled                    (gather; the inverse of keyed row sums)
  grad     its gradient: keyed row sums over tens of thousands of keys    (reduce_rows_by_key)
  distill  distillation from a teacher's top logits: the loss of each row of student logits, its gradient,
           or both in one call                                            (log-sum-exp row reductions)
  sample   one token per row of logits by temperature, top-k, top-p and min-p from given uniform numbers
                                                                          (row argmax)

`run` computes a case in elementary torch operations, or through raft_b200.linalg where `own` is set.
"""
import math

import numpy as np
import torch

own = False  # set from outside: run() then calls the library

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a small batch: latency
        {"name": "lookup_decode_64", "op": "lookup", "tokens": 64, "cols": 2048, "vocab": 32000, "dtype": "bf16",
         "pad": False},
        # the token rows of a long training batch
        {"name": "lookup_train_65536", "op": "lookup", "tokens": 65536, "cols": 4096, "vocab": 131072,
         "dtype": "bf16", "pad": False},
        # rows off 16-byte boundaries, padded sequences
        {"name": "lookup_odd_10007", "op": "lookup", "tokens": 10007, "cols": 1001, "vocab": 50001, "dtype": "f16",
         "pad": True},
        # fine-tuning on a few short sequences: the table is mostly zero rows
        {"name": "grad_small_512", "op": "grad", "tokens": 512, "cols": 1024, "vocab": 32000, "dtype": "bf16",
         "out": "bf16", "pad": True},
        # a long training batch, table and gradient in 16 bits
        {"name": "grad_train_65536", "op": "grad", "tokens": 65536, "cols": 4096, "vocab": 131072, "dtype": "bf16",
         "out": "bf16", "pad": False},
        # odd sizes, 16-bit activations with a 32-bit gradient
        {"name": "grad_odd_20011", "op": "grad", "tokens": 20011, "cols": 777, "vocab": 50001, "dtype": "f16",
         "out": "f32", "pad": True},
        # loss alone, as in evaluation
        {"name": "distill_loss_2048", "op": "distill", "mode": "loss", "rows": 2048, "vocab": 131072, "k": 64,
         "dtype": "bf16", "pad": False},
        # one training step's share: loss and gradient of every position in one call
        {"name": "distill_step_4096", "op": "distill", "mode": "step", "rows": 4096, "vocab": 131072, "k": 64,
         "dtype": "bf16", "pad": True},
        # the backward pass by itself, odd vocabulary, 32-bit logits
        {"name": "distill_grad_333", "op": "distill", "mode": "grad", "rows": 333, "vocab": 50001, "k": 17,
         "dtype": "f32", "pad": True},
        # interactive decoding: a few rows, every filter in use
        {"name": "sample_decode_4", "op": "sample", "rows": 4, "vocab": 131072, "filters": "mixed", "dtype": "f32"},
        # a serving batch with every mix of filters
        {"name": "sample_batch_256", "op": "sample", "rows": 256, "vocab": 131072, "filters": "mixed",
         "dtype": "bf16"},
        # roll-outs: plain temperature sampling with a nucleus over a wide distribution
        {"name": "sample_nucleus_512", "op": "sample", "rows": 512, "vocab": 50001, "filters": "nucleus",
         "dtype": "f32"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges that the listed ones stand for, no larger than the largest of its operator."""
    while True:
        op = rng.choice(["lookup", "grad", "distill", "sample"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        if op in ("lookup", "grad"):
            case = {"op": op, "tokens": _log_uniform(rng, 1, 65536), "cols": _log_uniform(rng, 64, 4096),
                    "vocab": _log_uniform(rng, 1000, 131072), "dtype": dtype, "pad": rng.random() < 0.5}
            if rng.random() < 0.5:
                case["cols"] = max(64, case["cols"] // 64 * 64)
            if op == "grad":
                case["out"] = rng.choice([dtype, "f32"])
        elif op == "distill":
            case = {"op": op, "mode": rng.choice(["loss", "step", "grad"]), "rows": _log_uniform(rng, 1, 4096),
                    "vocab": _log_uniform(rng, 1000, 131072), "k": _log_uniform(rng, 1, 128), "dtype": dtype,
                    "pad": rng.random() < 0.5}
            if rng.random() < 0.5:
                case["vocab"] = max(1000, case["vocab"] // 64 * 64)
        else:
            case = {"op": op, "rows": _log_uniform(rng, 1, 512), "vocab": _log_uniform(rng, 1000, 131072),
                    "filters": rng.choice(["none", "topk", "nucleus", "minp", "mixed"]), "dtype": dtype}
            if rng.random() < 0.5:
                case["vocab"] = max(1000, case["vocab"] // 64 * 64)
        most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
        cells = case.get("rows", 0) * case.get("vocab", 0)
        if work(case)["bytes"] <= most and (op != "sample" or cells <= 256 * 131072):
            return case


def work(case):
    """Bytes each input is read for once and each output written for once; operations on each element."""
    op = case["op"]
    s = SIZE[case["dtype"]]
    if op == "lookup":  # the distinct rows of the tokens, counted as min(tokens, vocab), and every output row
        n, c = case["tokens"], case["cols"]
        return {"bytes": n * 8 + _distinct(n, case["vocab"]) * c * s + n * c * s, "flops": n * c}
    if op == "grad":  # every gradient row, the whole table
        n, c = case["tokens"], case["cols"]
        return {"bytes": n * 8 + n * c * s + case["vocab"] * c * SIZE[case["out"]], "flops": n * c}
    r, v = case["rows"], case["vocab"]
    if op == "distill":
        once = r * v * s + r * case["k"] * (8 + 4) + 8 * r
        more = {"loss": 0, "grad": r * v * s, "step": r * v * s}[case["mode"]]
        return {"bytes": once + more, "flops": r * v * {"loss": 4, "grad": 4, "step": 8}[case["mode"]]}
    return {"bytes": r * v * s + r * (4 * 5 + 8), "flops": r * v * 4}


def _distinct(n, vocab):
    """Expected number of distinct tokens among n of _tokens."""
    share = np.diff(np.log(np.arange(1, vocab + 2))) / math.log(vocab + 1)
    return max(1, int(-np.expm1(n * np.log1p(-share)).sum()))


# -------------------------------------------------------------------------------------------- inputs
def _tokens(gen, n, vocab, pad):
    """Tokens as text has them: the share of a token falls with its number as 1 / number."""
    u = torch.rand(n, generator=gen, device=DEVICE, dtype=torch.float64)
    t = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)
    if pad:  # one token in twenty is padding
        t = torch.where(torch.rand(n, generator=gen, device=DEVICE) < 0.05, -1, t)
    return t


def _normal(gen, shape, dtype, scale):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)


def _places(gen, rows, k, vocab):
    """k different tokens for each row."""
    step = vocab // k
    first = torch.randint(0, vocab, (rows, 1), generator=gen, device=DEVICE)
    return (first + torch.arange(k, device=DEVICE) * step
            + torch.randint(0, step, (rows, k), generator=gen, device=DEVICE)) % vocab


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "lookup":
        s["table"] = _normal(gen, (case["vocab"], case["cols"]), dtype, 0.02)
        s["tokens"] = _tokens(gen, case["tokens"], case["vocab"], case["pad"])
        s["scale"] = math.sqrt(case["cols"])
    elif case["op"] == "grad":
        s["grad_out"] = _normal(gen, (case["tokens"], case["cols"]), dtype, 1.0)
        s["tokens"] = _tokens(gen, case["tokens"], case["vocab"], case["pad"])
        s["scale"] = math.sqrt(case["cols"])
        s["vocab"], s["out"] = case["vocab"], DTYPES[case["out"]]
    elif case["op"] == "distill":
        r, v, k = case["rows"], case["vocab"], case["k"]
        logits = _normal(gen, (r, v), dtype, 2.5)
        ids = _places(gen, r, k, v)
        teacher = torch.randn((r, k), generator=gen, device=DEVICE).mul_(2.0).add_(8.0)
        teacher = teacher.sort(dim=1, descending=True).values
        # where the teacher is sure the student mostly is too
        noise = torch.randn((r, k), generator=gen, device=DEVICE)
        logits.scatter_(1, ids, (teacher + noise).to(dtype))
        if case["pad"]:  # lists shorter than k, and rows (prompt, padding) that carry no list at all
            length = torch.randint(1, k + 1, (r, 1), generator=gen, device=DEVICE)
            length = torch.where(torch.rand((r, 1), generator=gen, device=DEVICE) < 0.1, 0, length)
            ids = torch.where(torch.arange(k, device=DEVICE) < length, ids, -1)
        s.update(logits=logits, ids=ids, teacher=teacher, temperature=2.0)
        s["grad_loss"] = torch.rand(r, generator=gen, device=DEVICE).add_(0.5).div_(r)
        if case["mode"] == "grad":  # what the forward pass left behind
            s["lse"] = torch.logsumexp(logits.double() / s["temperature"], 1).float()
    else:
        r, v = case["rows"], case["vocab"]
        logits = _normal(gen, (r, v), dtype, 2.5)
        peaks = _places(gen, r, 64, v)
        logits.scatter_(1, peaks, (torch.randn((r, 64), generator=gen, device=DEVICE) * 2.5 + 10.0).to(dtype))
        s["logits"] = logits
        s["uniform"] = torch.rand(r, generator=gen, device=DEVICE)

        def some(values, kind):
            pick = torch.randint(0, len(values), (r,), generator=gen, device=DEVICE)
            return torch.tensor(values, device=DEVICE, dtype=kind)[pick]
        f = case["filters"]
        s["temperature"] = some([0.0, 0.6, 0.8, 1.0, 1.3] if f == "mixed" else [0.7, 0.8, 1.0], torch.float32)
        s["top_k"] = some({"topk": [20, 50, 100], "mixed": [0, 20, 50, 1000]}.get(f, [0]), torch.int32)
        s["top_p"] = some({"nucleus": [0.8, 0.9, 0.95], "mixed": [1.0, 0.9, 0.95]}.get(f, [1.0]), torch.float32)
        s["min_p"] = some({"minp": [0.02, 0.05, 0.1], "mixed": [0.0, 0.0, 0.05]}.get(f, [0.0]), torch.float32)
    return s


# ------------------------------------------------------------------------------------ the operators
def run(s):
    return {"lookup": _lookup, "grad": _grad, "distill": _distill, "sample": _sample}[s["case"]["op"]](s)


def _lookup(s):
    if own:
        from raft_b200 import linalg
        return linalg.embedding_lookup(s["table"], s["tokens"], scale=s["scale"])
    table, tokens = s["table"], s["tokens"]
    valid = (tokens >= 0) & (tokens < table.shape[0])
    rows = table[torch.where(valid, tokens, 0)].float() * s["scale"]
    return torch.where(valid[:, None], rows, 0.0).to(table.dtype)


def _grad(s):
    if own:
        from raft_b200 import linalg
        return linalg.embedding_grad(s["grad_out"], s["tokens"], s["vocab"], scale=s["scale"], out_dtype=s["out"])
    tokens, vocab, g = s["tokens"], s["vocab"], s["grad_out"]
    valid = (tokens >= 0) & (tokens < vocab)
    table = torch.zeros((vocab + 1, g.shape[1]), dtype=torch.float32, device=g.device)
    table.index_add_(0, torch.where(valid, tokens, vocab), g.float())
    return (table[:vocab] * s["scale"]).to(s["out"])


def _distill(s):
    mode, t = s["case"]["mode"], s["temperature"]
    if own:
        from raft_b200 import linalg
        if mode == "loss":
            return linalg.topk_distill(s["logits"], s["ids"], s["teacher"], temperature=t)
        if mode == "grad":
            return linalg.topk_distill_grad(s["logits"], s["ids"], s["teacher"], s["lse"], s["grad_loss"],
                                            temperature=t)
        return linalg.topk_distill_step(s["logits"], s["ids"], s["teacher"], s["grad_loss"], temperature=t)
    logits, ids = s["logits"], s["ids"]
    z = logits.float() / t
    valid = (ids >= 0) & (ids < logits.shape[1])
    at = torch.where(valid, ids, 0)
    y = torch.where(valid, s["teacher"].float() / t, -math.inf)
    some = y.max(dim=1, keepdim=True).values > -math.inf
    w = torch.where(valid & some, torch.exp(y - torch.where(some, y.max(dim=1, keepdim=True).values, 0.0)), 0.0)
    total = torch.where(some, w.sum(dim=1, keepdim=True), 1.0)
    p = w / total
    if mode == "grad":
        lse = s["lse"][:, None]
    else:
        top = z.max(dim=1, keepdim=True).values
        lse = top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))
        log_ratio = torch.log(torch.where(p > 0, p, 1.0)) - (z.gather(1, at) - lse)
        loss = t * t * torch.where(p > 0, p * log_ratio, 0.0).sum(dim=1)
        if mode == "loss":
            return loss, lse[:, 0]
    factor = torch.where(some, s["grad_loss"].float()[:, None] * t, 0.0)
    grad = torch.exp(z - lse) * factor
    grad.scatter_add_(1, at, -p * factor)
    grad = grad.to(logits.dtype)
    return grad if mode == "grad" else (loss, lse[:, 0], grad)


def _sample(s):
    if own:
        from raft_b200 import linalg
        return linalg.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                    top_p=s["top_p"], min_p=s["min_p"])
    # 64 bits: which side of a border a token falls on is decided by sums over the whole vocabulary
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    n = x.shape[1]
    by_value, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = by_value[:, :1]
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    weight = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, t)))
    weight = torch.where(x > -math.inf, weight, 0.0)
    sorted_weight = weight.gather(1, order)
    rank = torch.arange(n, device=x.device)
    k = s["top_k"].long()[:, None]
    keep = (rank < torch.where(k > 0, k, n)) & (sorted_weight >= s["min_p"].double()[:, None].clamp(max=1.0))
    sorted_weight = torch.where(keep, sorted_weight, 0.0)
    upto = torch.cumsum(sorted_weight, dim=1)
    top_p = s["top_p"].double()[:, None]
    keep &= (upto - sorted_weight < top_p * upto[:, -1:]) | (top_p >= 1.0) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    weight = torch.where(kept, weight, 0.0)
    upto = torch.cumsum(weight, dim=1)
    total = upto[:, -1:]
    token = (upto <= s["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True)
    last = n - 1 - torch.argmax(kept.flip(1).to(torch.int8), dim=1, keepdim=True)
    token = torch.minimum(token, last)
    token = torch.where(greedy, order[:, :1], token)
    logprob = torch.where(greedy, 0.0, torch.log(weight.gather(1, token) / total))
    alive = top > -math.inf
    token = torch.where(alive, token, -1)
    logprob = torch.where(alive, logprob, -math.inf)
    return token[:, 0].to(torch.int32), logprob[:, 0].float()


# ----------------------------------------------------------------- the same by definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        table = torch.cat([s["table"].double(), torch.zeros((1, case["cols"]), dtype=torch.float64, device=DEVICE)])
        return table.index_select(0, torch.where(s["tokens"] < 0, case["vocab"], s["tokens"])) * s["scale"]
    if case["op"] == "grad":
        # rows in the order of their tokens; the sum of a token's rows is a difference of running sums
        order = torch.argsort(s["tokens"], stable=True)
        sums = torch.zeros((len(order) + 1, case["cols"]), dtype=torch.float64, device=DEVICE)
        torch.cumsum(s["grad_out"].index_select(0, order).double(), 0, out=sums[1:])
        edges = torch.searchsorted(s["tokens"][order], torch.arange(case["vocab"] + 1, device=DEVICE))
        return (sums[edges[1:]] - sums[edges[:-1]]) * s["scale"]
    if case["op"] == "distill":
        t = s["temperature"]
        parts = [_exact_distill(case["mode"], t, s["logits"][i:i + 512], s["ids"][i:i + 512],
                                s["teacher"][i:i + 512], s["grad_loss"][i:i + 512],
                                s["lse"][i:i + 512] if "lse" in s else None) for i in range(0, case["rows"], 512)]
        out = tuple(torch.cat(p) for p in zip(*parts))
        return out[0] if case["mode"] == "grad" else out
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        tok, lp = _exact_sample(s["logits"][r].double().cpu().numpy(), float(s["uniform"][r]),
                                float(s["temperature"][r]), int(s["top_k"][r]), float(s["top_p"][r]),
                                float(s["min_p"][r]))
        tokens.append(tok)
        logprobs.append(lp)
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)


def _exact_distill(mode, t, logits, ids, teacher, grad_loss, lse):
    """The teacher's distribution laid out over the vocabulary; cross entropy less its own entropy."""
    z = logits.double().mul_(1.0 / t)
    v = z.shape[1]
    ids = torch.where((ids >= 0) & (ids < v), ids, v)
    target = torch.where(ids < v, teacher.double() / t, -math.inf).softmax(1).nan_to_num_(0.0)
    spread = torch.zeros((z.shape[0], v + 1), dtype=torch.float64, device=z.device)
    spread = spread.scatter_add_(1, ids, target)[:, :v]
    lse = z.logsumexp(1) if lse is None else lse.double()
    out = []
    if mode != "grad":
        entropy = torch.special.entr(target).sum(1)
        cross = lse * target.sum(1) - (spread * z).sum(1)
        out += [(cross - entropy) * t * t, lse]
    if mode != "loss":
        some = (ids < v).any(1)
        out.append(((z - lse[:, None]).exp_() - spread) * (grad_loss.double() * t * some)[:, None])
    return out


def _exact_sample(x, u, t, k, top_p, min_p):
    x = np.where(np.isnan(x), -np.inf, x)
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1, -math.inf
    if not t > 0:
        return best, 0.0
    with np.errstate(invalid="ignore"):
        p = np.where(x == x[best], 1.0, np.exp((x - x[best]) / t))
    order = np.lexsort((np.arange(x.size), -x))
    order = order[: k if k > 0 else x.size]
    order = order[(p[order] >= min(min_p, 1.0)) & (p[order] > 0)]
    if top_p < 1:
        upto = np.cumsum(p[order])
        order = order[: max(1, int(np.searchsorted(upto, top_p * upto[-1], side="left")) + 1)]
    order = np.sort(order)
    upto = np.cumsum(p[order])
    at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), order.size - 1)
    return int(order[at]), float(np.log(p[order[at]] / upto[-1]))
