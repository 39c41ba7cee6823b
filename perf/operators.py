"""The operators at the two ends of a token model, as cases that can be timed and compared.

    embed         table rows by token id, scaled                                (embeddingForward)
    embed_grad    their gradient, summed per token                              (embeddingBackward)
    scores        log-probability of a given token, entropy, top alternatives   (tokenLogProbs)
    scores_grad   the gradient of the first two with respect to the logits      (tokenLogProbsBackward)
    distill       distillation from a teacher's top logits: loss and gradient   (distillLoss)
    head4         product with 4-bit weights in scaled groups                   (matMul4BiasAct)

`run` computes an operator in its plain form (elementary torch operations in 32 bits) or, with `own` set, by the
calls a user makes of this package.  `exact` gives the definition's value in 64 bits.
"""
import math

import torch

own = False

EMBED, EMBED_GRAD, SCORES, SCORES_GRAD, DISTILL, HEAD4 = "embed", "embed_grad", "scores", "scores_grad", "distill", "head4"


def listed():
    return [
        # one token's row while generating: nothing but latency
        {"name": "embed_one", "op": EMBED, "rows": 1, "vocab": 32768, "dim": 1024},
        # the lookup of a long prompt or of a training batch
        {"name": "embed_batch", "op": EMBED, "rows": 32768, "vocab": 131072, "dim": 2048},
        # the table's whole gradient in a training step (rows without a token become zero), word-like frequencies
        {"name": "embed_grad_step", "op": EMBED_GRAD, "rows": 16384, "vocab": 50001, "dim": 1024, "accumulate": False},
        # a short fine-tuning batch added into a gradient that is there already, odd width
        {"name": "embed_grad_into", "op": EMBED_GRAD, "rows": 777, "vocab": 131072, "dim": 1003, "accumulate": True},
        # a few sequences that generate: one token each, twenty alternatives, sampled at a temperature
        {"name": "scores_step", "op": SCORES, "rows": 4, "vocab": 131072, "pitch": 131072, "top": 20, "temperature": 0.8},
        # scoring whole prompts: many rows of an odd vocabulary
        {"name": "scores_batch", "op": SCORES, "rows": 4096, "vocab": 50001, "pitch": 50001, "top": 5, "temperature": 1.0},
        # the policy and entropy gradient over a batch of generated tokens
        {"name": "scores_grad_batch", "op": SCORES_GRAD, "rows": 2048, "vocab": 131072, "pitch": 131072, "temperature": 1.0},
        # a small distillation step
        {"name": "distill_small", "op": DISTILL, "rows": 48, "vocab": 32000, "pitch": 32000, "top": 16, "temperature": 2.0},
        # odd vocabulary in padded rows, short teacher lists, rows of padding tokens
        {"name": "distill_ragged", "op": DISTILL, "rows": 1111, "vocab": 50001, "pitch": 50023, "top": 20, "temperature": 1.5},
        # a full distillation batch over a large vocabulary
        {"name": "distill_large", "op": DISTILL, "rows": 4096, "vocab": 131072, "pitch": 131072, "top": 64, "temperature": 2.0},
        # one token through a square 4-bit layer
        {"name": "head4_one", "op": HEAD4, "rows": 1, "k": 4096, "n": 4096, "group": 64},
        # a batch of generating sequences through a 4-bit output layer
        {"name": "head4_batch", "op": HEAD4, "rows": 8, "k": 8192, "n": 65536, "group": 128},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice([EMBED, EMBED_GRAD, SCORES, SCORES_GRAD, DISTILL, HEAD4])
    if op == EMBED:
        dim = _log_uniform(rng, 16, 4096)
        return {"op": op, "rows": _log_uniform(rng, 1, min(65536, (1 << 26) // dim)), "vocab": _log_uniform(rng, 100, 131072), "dim": dim}
    if op == EMBED_GRAD:
        dim = _log_uniform(rng, 16, 2048)
        return {"op": op, "rows": _log_uniform(rng, 1, min(65536, (1 << 26) // dim)), "vocab": _log_uniform(rng, 100, 131072), "dim": dim,
                "accumulate": rng.random() < 0.5}
    if op == HEAD4:
        return {"op": op, "rows": rng.randint(1, 16), "k": _log_uniform(rng, 64, 8192), "n": _log_uniform(rng, 64, 32768),
                "group": rng.choice([32, 64, 128])}
    vocab = _log_uniform(rng, 100, 200000)
    case = {"op": op, "rows": _log_uniform(rng, 1, min(8192, (1 << 28) // vocab)), "vocab": vocab,
            "pitch": vocab + rng.choice([0, 0, 1, 7, 64]), "temperature": rng.choice([0.5, 0.8, 1.0, 1.0, 2.0, 4.0])}
    if op == SCORES:
        case["top"] = rng.randint(0, 64)
    if op == DISTILL:
        case["top"] = rng.randint(1, 100)
    return case


def _tokens(gen, rows, vocab):
    """Token ids with a frequency that falls as one over the rank, as words have; one in a hundred is padding (-1)."""
    u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    ids = (ids * 7919 + 13) % vocab if math.gcd(7919, vocab) == 1 else ids      # frequent words stand anywhere in the table
    pad = torch.rand(rows, generator=gen, device="cuda") < 0.01
    return torch.where(pad, torch.full_like(ids, -1), ids).to(torch.int32)


def _logits(gen, rows, vocab, pitch):
    """Rows as a model gives them: spread-out values, a few likely tokens, an offset of the row's own; the last
    columns of a vocabulary that fills a multiple of 64 are masked out by minus infinity."""
    x = torch.randn(rows, pitch, generator=gen, device="cuda") * 2.0
    hot = torch.randint(0, vocab, (rows, 4), generator=gen, device="cuda")
    x.scatter_add_(1, hot, 6.0 + 4.0 * torch.rand(rows, 4, generator=gen, device="cuda"))
    x += 3.0 * torch.randn(rows, 1, generator=gen, device="cuda")
    if vocab % 64 == 0 and vocab > 64:
        x[:, vocab - 17:vocab] = -math.inf
    return x


def _uniform_ids(gen, rows, vocab):
    live = vocab - 17 if vocab % 64 == 0 and vocab > 64 else vocab
    ids = torch.randint(0, live, (rows,), generator=gen, device="cuda")
    pad = torch.rand(rows, generator=gen, device="cuda") < 0.02
    return torch.where(pad, torch.full_like(ids, -1), ids).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows = case["op"], case["rows"]
    s = dict(case)
    f32 = {"dtype": torch.float32, "device": "cuda"}
    if op == EMBED:
        s["table"] = torch.randn(case["vocab"], case["dim"], generator=gen, device="cuda") * 0.02
        s["tokens"] = _tokens(gen, rows, case["vocab"])
        s["scale"] = math.sqrt(case["dim"])
        s["out"] = torch.zeros(rows, case["dim"], **f32)
    elif op == EMBED_GRAD:
        s["tokens"] = _tokens(gen, rows, case["vocab"])
        s["grad_out"] = torch.randn(rows, case["dim"], generator=gen, device="cuda") * 1e-3
        s["scale"] = math.sqrt(case["dim"])
        s["grad_table"] = torch.randn(case["vocab"], case["dim"], generator=gen, device="cuda") * 1e-3
    elif op in (SCORES, SCORES_GRAD, DISTILL):
        vocab, pitch = case["vocab"], case["pitch"]
        s["buffer"] = _logits(gen, rows, vocab, pitch)
        s["logits"] = s["buffer"][:, :vocab]
        if op != DISTILL:
            s["tokens"] = _uniform_ids(gen, rows, vocab)
        if op == SCORES:
            s["logprob"], s["entropy"], s["stats"] = torch.zeros(rows, **f32), torch.zeros(rows, **f32), torch.zeros(rows, 2, **f32)
            s["top_tokens"] = torch.zeros(rows, case["top"], dtype=torch.int32, device="cuda")
            s["top_logprobs"] = torch.zeros(rows, case["top"], **f32)
        elif op == SCORES_GRAD:
            # what the forward call left: statistics and entropy of every row
            x = s["logits"].double() / case["temperature"]
            m = x.amax(1, keepdim=True)
            e = torch.exp(x - m)
            total = e.sum(1)
            s["stats"] = torch.stack((s["logits"].amax(1), torch.log(total).float()), 1).contiguous()
            s["entropy"] = (torch.log(total) - torch.where(e > 0, e * (x - m), 0.0).sum(1) / total).float()
            del x, m, e
            s["grad_logprob"] = torch.randn(rows, generator=gen, device="cuda")
            s["grad_entropy"] = 0.01 * torch.randn(rows, generator=gen, device="cuda")
            s["grad"] = torch.zeros(rows, pitch, **f32)
        else:
            k = case["top"]
            order = torch.rand(rows, k, generator=gen, device="cuda")
            span = max(1, vocab // k)
            base = torch.arange(k, device="cuda") * span        # k tokens of every row, all different
            ids = (base + (order * min(span, vocab - int(base[-1]))).long()).clamp_(max=vocab - 1)
            if vocab < k:
                ids = torch.arange(k, device="cuda").expand(rows, k) % vocab
            if vocab % 64 == 0 and vocab > 64:
                ids = torch.where(ids >= vocab - 17, torch.full_like(ids, -1), ids)
            short = torch.rand(rows, k, generator=gen, device="cuda") < 0.05      # lists with fewer tokens
            s["teacher_tokens"] = torch.where(short, torch.full_like(ids, -1), ids).to(torch.int32).contiguous()
            s["teacher_logits"] = torch.randn(rows, k, generator=gen, device="cuda") * 3.0 + 10.0
            w = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.1, 0.0, 1.0)     # padding counts for nothing
            s["weights"] = (w / max(1, rows)).contiguous()
            s["loss"] = torch.zeros(rows, **f32)
            s["grad"] = torch.zeros(rows, pitch, **f32)
    else:
        n, k, g = case["n"], case["k"], case["group"]
        blocks = -(-k // 128)
        s["packed"] = torch.randint(-(1 << 31), 1 << 31, (n, blocks * 16), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        s["scales"] = (0.5 + torch.rand(n, -(-k // g), generator=gen, device="cuda")) * (0.2 / math.sqrt(k))
        s["x"] = torch.randn(rows, k, generator=gen, device="cuda")
        s["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.1
        s["y"] = torch.zeros(rows, n, **f32)
    return s


# ---- the framework's calls ---------------------------------------------------------------------

_backend = None


def _be():
    global _backend
    if _backend is None:
        import zigneuron_b200 as zn
        _backend = zn.Backend(torch.cuda.current_device())
    return _backend


def _own(s):
    be, op = _be(), s["op"]
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if op == EMBED:
        be.embeddingForward(p("table"), p("tokens"), p("out"), s["rows"], s["vocab"], s["dim"], s["scale"])
        return s["out"]
    if op == EMBED_GRAD:
        be.embeddingBackward(p("grad_out"), p("tokens"), p("grad_table"), s["rows"], s["vocab"], s["dim"], s["scale"], s["accumulate"])
        return s["grad_table"]
    if op == SCORES:
        top = s["top"]
        be.tokenLogProbs(p("buffer"), p("tokens"), s["rows"], s["vocab"], logprob=p("logprob"), entropy=p("entropy"), row_stats=p("stats"),
                         top_k=top, top_tokens=p("top_tokens") if top else None, top_logprobs=p("top_logprobs") if top else None,
                         temperature=s["temperature"], ld=s["pitch"])
        return s["logprob"], s["entropy"], s["stats"], s["top_tokens"], s["top_logprobs"]
    if op == SCORES_GRAD:
        be.tokenLogProbsBackward(p("buffer"), p("tokens"), p("stats"), p("entropy"), p("grad_logprob"), p("grad_entropy"), p("grad"),
                                 s["rows"], s["vocab"], temperature=s["temperature"], ld=s["pitch"], ld_grad=s["pitch"])
        return s["grad"][:, :s["vocab"]]
    if op == DISTILL:
        be.distillLoss(p("buffer"), p("teacher_tokens"), p("teacher_logits"), s["rows"], s["vocab"], s["top"], s["temperature"],
                       row_weights=p("weights"), row_loss=p("loss"), grad_logits=p("grad"), ld=s["pitch"], ld_grad=s["pitch"])
        return s["loss"], s["grad"][:, :s["vocab"]]
    be.matMul4BiasAct(p("x"), p("packed"), p("scales"), p("bias"), p("y"), s["rows"], s["n"], s["k"], s["group"], 0)      # relu
    return s["y"]


# ---- the plain forms ----------------------------------------------------------------------------

def _top(x, k):
    """The k largest of every row, the lowest index first among equals: values and indices."""
    bits = x.view(torch.int32).long()
    rank = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))        # orders as the values do, with -0 and 0 equal
    key = rank * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
    index = torch.topk(key, k, dim=1).indices
    return torch.gather(x, 1, index), index


def _codes(packed, n, k):
    """Weight codes [n, k] less 8: word 4 i + t of every 16 stands at 4 t + i, eight codes to a word, the lowest bits first."""
    words = packed.view(n, -1, 4, 4).transpose(2, 3).reshape(n, -1, 1)
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=packed.device)
    return ((words >> shifts) & 15).reshape(n, -1)[:, :k] - 8


def _plain(s):
    op = s["op"]
    if op == EMBED:
        ids = s["tokens"].long()
        return torch.where(ids[:, None] >= 0, s["table"][ids.clamp(min=0)] * s["scale"], 0.0)
    if op == EMBED_GRAD:
        live = s["tokens"] >= 0
        ids = torch.where(live, s["tokens"], 0).long()
        rows = torch.where(live[:, None], s["grad_out"], 0.0) * s["scale"]
        grad = s["grad_table"]
        if not s["accumulate"]:
            grad.zero_()
        return grad.index_add_(0, ids, rows)
    if op == SCORES:
        raw, t = s["logits"], s["temperature"]
        top = raw.amax(1, keepdim=True)
        z = (raw - top) / t
        e = torch.exp(z)
        total = e.sum(1)
        log_total = torch.log(total)
        ids = s["tokens"].long()
        given = torch.gather(z, 1, ids.clamp(min=0)[:, None])[:, 0] - log_total
        entropy = log_total - torch.where(e > 0, e * z, 0.0).sum(1) / total
        values, index = _top(raw.contiguous(), s["top"])
        lp = (values - top) / t - log_total[:, None]
        masked = values == -math.inf
        return (torch.where(ids >= 0, given, 0.0), entropy, torch.stack((top[:, 0], log_total), 1),
                torch.where(masked, -1, index).to(torch.int32), lp)
    if op == SCORES_GRAD:
        t = s["temperature"]
        logp = (s["logits"] - s["stats"][:, :1]) / t - s["stats"][:, 1:]
        p = torch.exp(logp)
        ids = s["tokens"].long()
        gl = torch.where(ids >= 0, s["grad_logprob"], 0.0)[:, None]
        gh = s["grad_entropy"][:, None]
        grad = -p * gl - torch.where(p > 0, p * (logp + s["entropy"][:, None]), 0.0) * gh
        grad = grad.scatter_add(1, ids.clamp(min=0)[:, None], gl)
        return grad / t
    if op == DISTILL:
        t, ids = s["temperature"], s["teacher_tokens"].long()
        z = s["logits"] / t
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        there = ids >= 0
        u = torch.where(there, s["teacher_logits"] / t, -math.inf)
        peak = u.amax(1, keepdim=True)
        peak = torch.where(peak == -math.inf, 0.0, peak)
        qe = torch.exp(u - peak)
        mass = qe.sum(1, keepdim=True)
        some = mass > 0
        q = torch.where(some, qe / torch.where(some, mass, 1.0), 0.0)
        logq = u - peak - torch.log(torch.where(some, mass, 1.0))
        logp = torch.gather(z, 1, ids.clamp(min=0)) - top - torch.log(total)
        w = s["weights"]
        loss = torch.where(q > 0, q * (logq - logp), 0.0).sum(1) * (t * t) * w
        grad = torch.where(some, e / total, 0.0)
        grad = grad.scatter_add(1, ids.clamp(min=0), -q)
        return loss, grad * (t * w[:, None])
    weights = _codes(s["packed"], s["n"], s["k"]).float()
    scales = s["scales"].repeat_interleave(s["group"], 1)[:, :s["k"]]
    return torch.clamp(s["x"] @ (weights * scales).T + s["bias"], min=0.0)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def _distinct(rows, vocab):
    """How many different table rows a batch of tokens is expected to name."""
    rank = torch.arange(1, vocab + 1, dtype=torch.float64)
    share = torch.log1p(1.0 / rank) / math.log(vocab + 1.0)
    return float(-torch.expm1(0.99 * rows * torch.log1p(-share)).sum())


def work(case):
    op, rows = case["op"], case["rows"]
    if op == EMBED:
        read = _distinct(rows, case["vocab"])
        return {"bytes": 4.0 * case["dim"] * (rows + read) + 4.0 * rows, "flops": float(rows * case["dim"])}
    if op == EMBED_GRAD:
        table = 2.0 * _distinct(rows, case["vocab"]) if case["accumulate"] else float(case["vocab"])
        return {"bytes": 4.0 * case["dim"] * (rows + table) + 4.0 * rows, "flops": 2.0 * rows * case["dim"]}
    if op == HEAD4:
        n, k = case["n"], case["k"]
        return {"bytes": n * k / 2.0 + 4.0 * n * -(-k // case["group"]) + 4.0 * rows * (n + k) + 4.0 * n, "flops": 2.0 * rows * n * k}
    cells = float(rows * case["vocab"])
    if op == SCORES:
        return {"bytes": 4.0 * cells + rows * (20.0 + 8.0 * case["top"]), "flops": 5.0 * cells}
    if op == SCORES_GRAD:
        return {"bytes": 8.0 * cells + 24.0 * rows, "flops": 7.0 * cells}
    return {"bytes": 8.0 * cells + rows * (8.0 + 8.0 * case["top"]), "flops": 6.0 * cells}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op, rows = case["op"], case["rows"]
    if op == EMBED:
        out = torch.zeros(rows, case["dim"], dtype=torch.float64, device="cuda")
        live = (s["tokens"] >= 0).nonzero()[:, 0]
        out[live] = s["table"].double()[s["tokens"][live].long()] * s["scale"]
        return out
    if op == EMBED_GRAD:
        out = s["grad_table"].double() if case["accumulate"] else torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        live = (s["tokens"] >= 0).nonzero()[:, 0]
        return out.index_put_((s["tokens"][live].long(),), s["grad_out"][live].double() * s["scale"], accumulate=True)
    if op == HEAD4:
        out = torch.empty(rows, case["n"], dtype=torch.float64, device="cuda")
        k = case["k"]
        column = torch.arange(k, device="cuda")
        word, nibble = column // 8, column % 8
        place = word // 16 * 16 + (word % 4) * 4 + word % 16 // 4
        for lo in range(0, case["n"], 8192):
            packed, scales = s["packed"][lo:lo + 8192].long(), s["scales"][lo:lo + 8192].double()
            code = torch.bitwise_and(torch.bitwise_right_shift(packed[:, place], 4 * nibble), 15).double() - 8.0
            out[:, lo:lo + 8192] = s["x"].double() @ (code * scales[:, column // case["group"]]).T
        return torch.relu(out + s["bias"].double())
    parts = []
    step = max(1, (1 << 27) // case["vocab"])
    t = case["temperature"]
    for lo in range(0, rows, step):
        cut = slice(lo, lo + step)
        x = s["logits"][cut].double()
        logp = torch.log_softmax(x / t, 1)
        p = torch.exp(logp)
        row = torch.arange(x.shape[0], device="cuda")
        if op == DISTILL:
            ids = s["teacher_tokens"][cut].long()
            grad, loss = torch.zeros_like(p), torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
            has = (ids >= 0).any(1)
            q = torch.softmax(s["teacher_logits"][cut].double().masked_fill(ids < 0, -math.inf) / t, 1).nan_to_num_(0.0)
            grad[has] = p[has]
            for j in range(ids.shape[1]):
                use = (ids[:, j] >= 0).nonzero()[:, 0]
                at = ids[use, j]
                qj = q[use, j]
                loss[use] += torch.xlogy(qj, qj) - qj * logp[use, at]
                grad[use, at] -= qj
            w = s["weights"][cut].double()
            parts.append((loss * t * t * w, grad * t * w[:, None]))
            continue
        ids = s["tokens"][cut].long()
        live = ids >= 0
        if op == SCORES:
            given = torch.where(live, logp[row, ids.clamp(min=0)], 0.0)
            entropy = -torch.nan_to_num(p * logp, nan=0.0).sum(1)
            peak = x.max(1).values
            stats = torch.stack((peak, torch.logsumexp(x / t, 1) - peak / t), 1)
            parts.append((given, entropy, stats, torch.sort(logp, 1, descending=True).values[:, :case["top"]]))
        else:
            # d logprob / d x_c = (1[c = token] - p_c) / t;  d entropy / d x_c = -p_c (log p_c + entropy) / t
            entropy = -torch.nan_to_num(p * logp, nan=0.0).sum(1, keepdim=True)
            g = torch.where(live, s["grad_logprob"][cut].double(), 0.0)
            out = -p * g[:, None]
            out[row[live], ids[live]] += g[live]
            out -= s["grad_entropy"][cut].double()[:, None] * torch.nan_to_num(p * (logp + entropy), nan=0.0)
            parts.append((out / t,))
    columns = [torch.cat(c) for c in zip(*parts)]
    if op == SCORES_GRAD:
        return columns[0]
    if op == DISTILL:
        return tuple(columns)
    return columns[0], columns[1], columns[2], None, columns[3]
