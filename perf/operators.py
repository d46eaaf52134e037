"""What the operators on class scores are measured on: `thundergbm_amd.scores`, on data that lies on the GPU.

A model with one tree per class and round gives every row a score for each class. `adjust` applies what is known besides the
model before it answers: biases, classes that are not allowed, penalties on classes that a row was shown before. `top` lists
the best classes of every row with the logarithm of the sum that turns scores into probabilities: an answer, or what a teacher
hands on. `distill` is the loss of class scores against a teacher's top scores, with the gradient pairs that the trees of the
next round are built from.

Scores are [classes, rows], with the rows of a class side by side (as trainers and predictors hold them) or the classes of a
row side by side (as other models leave them).
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def distill_case(name, rows, classes, entries, **more):
    c = dict(name=name, call="distill", rows=rows, classes=classes, entries=entries, teacher="float32", rest=False, temperature=1.0,
             weight=1.0, gradient=True)
    c.update(more)
    return c


def score_case(name, call, rows, classes, **more):
    """order: "class" (the rows of a class side by side) or "row"; sets: allowed sets, 0 for none; shown: classes shown to a
    row on average, 0 for none; k: of top."""
    c = dict(name=name, call=call, rows=rows, classes=classes, order="class", type="float32", bias=False, sets=0, shown=0)
    if call == "top":
        c.update(k=1, temperature=1.0)
    c.update(more)
    return c


def listed():
    return [
        # one row that arrives while a service keeps learning, eight classes as in the multi-class benchmark configuration
        distill_case("distill_one_row", 1, 8, 8),
        # a boosting round on that configuration's table: few classes, a teacher's five best, true labels beside it
        distill_case("distill_few_classes", 500_000, 8, 5, teacher="float16", temperature=2.0, weight=0.7),
        # a boosting round with many classes: half precision teacher, what it left out is known
        distill_case("distill_many_classes", 120_011, 1000, 32, teacher="bfloat16", rest=True, temperature=2.0, weight=0.5),
        # few rows, very many classes: the classes have to be shared out
        distill_case("distill_few_rows", 24, 50_021, 100, rest=True),
        # the loss alone, on held-out rows
        distill_case("distill_loss", 200_000, 100, 10, gradient=False, temperature=4.0),
        # one request of a service: the best allowed class, with a history
        score_case("top_one_row", "top", 1, 32_000, order="row", k=1, bias=True, sets=1, shown=200),
        # a teacher's top scores, written down for a student
        score_case("top_teacher", "top", 2048, 65_537, order="row", type="bfloat16", k=64, temperature=2.0),
        # the three best of eight classes for a whole table
        score_case("top_few_classes", "top", 500_000, 8, k=3, bias=True),
        # recommendations: the ten best of what is allowed to a row, what it was shown counting less
        score_case("top_many_classes", "top", 50_021, 1000, k=10, bias=True, sets=64, shown=20),
        # a small batch of a service
        score_case("adjust_small", "adjust", 16, 100, bias=True, sets=16),
        # a table's scores before they become probabilities
        score_case("adjust_table", "adjust", 100_003, 500, bias=True, sets=64, shown=20),
        # a batch over a large vocabulary, every row in a state of its own, with long histories
        score_case("adjust_long_rows", "adjust", 512, 65_537, order="row", type="bfloat16", bias=True, sets=512, shown=1500),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    call = rng.choice(("distill", "top", "adjust"))
    few = rng.random() < 0.4
    if call == "distill":
        classes = rng.randint(3, 32) if few else spread(rng, 33, 50_000)
        rows = spread(rng, 1, min(500_000, 80_000_000 // classes))
        entries = min(classes, rng.randint(1, 8) if few else rng.randint(4, 128))
        c = distill_case("", rows, classes, entries, teacher=rng.choice(tuple(TYPES)), rest=rng.random() < 0.5,
                         temperature=rng.choice((1.0, 1.0, 2.0, 3.0, 0.7)), weight=rng.choice((1.0, 0.9, 0.5, 0.2)), gradient=rng.random() < 0.8)
    else:
        classes = rng.randint(3, 32) if few else spread(rng, 33, 65_537)
        rows = spread(rng, 1, min(500_000, 100_000_000 // classes))
        order = "class" if few else rng.choice(("class", "row"))
        c = score_case("", call, rows, classes, order=order, type=rng.choice(tuple(TYPES)) if order == "row" else "float32", bias=rng.random() < 0.6,
                       sets=rng.choice((0, 1, 7, 64, rows)), shown=rng.choice((0, 0, 5, 40, 300)) if rows <= 100_000 else rng.choice((0, 3)))
        if call == "top":
            c.update(k=min(classes, rng.choice((1, 2, 5, 10, 40, 64, 128))), temperature=rng.choice((1.0, 1.0, 2.0, 0.5)))
        elif not (c["bias"] or c["sets"] or c["shown"]):
            c["bias"] = True
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------- the inputs


def prepare_distill(c, gen):
    n, C, K, T = c["rows"], c["classes"], c["entries"], c["temperature"]
    label = torch.randint(0, C, (n,), device="cuda", generator=gen)
    scores = torch.randn(C, n, device="cuda", generator=gen)
    scores *= 1.5
    scores.scatter_add_(0, label[None], torch.full((1, n), 2.0, device="cuda"))
    # the teacher: surer of the label than the student, and of the student's opinion in part
    full = torch.randn(n, C, device="cuda", generator=gen)
    full += scores.t()
    full.scatter_add_(1, label[:, None], torch.full((n, 1), 3.0, device="cuda"))
    full = full.to(TYPES[c["teacher"]]).float()
    lse = torch.empty(n, device="cuda")
    top = torch.empty(n, K, device="cuda")
    at = torch.empty(n, K, dtype=torch.int64, device="cuda")
    for a in range(0, n, 16_384):
        lse[a:a + 16_384] = torch.logsumexp(full[a:a + 16_384].double() / T, 1).float()
        top[a:a + 16_384], at[a:a + 16_384] = torch.topk(full[a:a + 16_384], K, dim=1)
    # one row in ten has a shorter list
    if n > 1 and K > 1:
        short = torch.rand(n, device="cuda", generator=gen) < 0.1
        keep = torch.randint(1, K, (n, 1), device="cuda", generator=gen)
        at.masked_fill_(short[:, None] & (torch.arange(K, device="cuda")[None] >= keep), -1)
    return dict(scores=scores, classes=at.int(), teacher=top.to(TYPES[c["teacher"]]), teacher_lse=lse if c["rest"] else None,
                labels=label.float() if c["weight"] < 1 else None, temperature=T, weight=c["weight"], gradient=c["gradient"])


def prepare_scores(c, gen):
    n, C = c["rows"], c["classes"]
    s = dict(bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None)
    if c["order"] == "row":
        s["scores"] = (torch.randn(n, C, device="cuda", generator=gen) * 2.5).to(TYPES[c["type"]]).t()
    else:
        s["scores"] = (torch.randn(C, n, device="cuda", generator=gen) * 2.5).to(TYPES[c["type"]])
    if c["bias"]:  # log-odds of rare and frequent classes, as they are set by hand: in steps of a sixteenth
        s["bias"] = torch.round(torch.randn(C, device="cuda", generator=gen) * 16) / 16
    if c["sets"]:  # some states allow most classes, some few
        S, words = c["sets"], (C + 31) // 32
        dense = torch.rand(S, 1, device="cuda", generator=gen) < 0.5
        bits = torch.randint(-2**31, 2**31, (2, S, words), dtype=torch.int64, device="cuda", generator=gen)
        s["allowed"] = torch.where(dense, bits[0] | bits[1], bits[0] & bits[1]).int()
        if S != n and S != 1:
            s["allowed_set"] = torch.randint(0, S, (n,), dtype=torch.int32, device="cuda", generator=gen)
    if c["shown"]:  # between none and twice the average, popular classes more often
        count = torch.randint(0, 2 * c["shown"] + 1, (n,), device="cuda", generator=gen)
        begin = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
        torch.cumsum(count, 0, out=begin[1:])
        u = torch.rand(int(begin[-1]), device="cuda", generator=gen)
        s["shown"] = (u * u * C).int().clamp_(max=C - 1)
        s["shown_begin"] = begin
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = prepare_distill(case, gen) if case["call"] == "distill" else prepare_scores(case, gen)
    s["call"] = case["call"]
    if case["call"] == "top":
        s.update(k=case["k"], temperature=case["temperature"])
    if case["call"] != "distill":
        # how strongly repeated answers are held back
        s.update(repetition=1.25, frequency=0.125, presence=0.5)
    return s


# -------------------------------------------------------------------------------------------------- the plain forms


def log_sum_exp(x, dim):
    """log(sum(exp(x))) with the largest value taken out; of nothing it is -inf."""
    m = x.amax(dim, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    return (torch.exp(x - m).sum(dim, keepdim=True).log() + m).squeeze(dim)


def plain_adjusted(s):
    """The adjusted scores in 32 bits, [classes, rows]."""
    x = s["scores"].float()
    C, n = x.shape
    if s["bias"] is not None:
        x = x + s["bias"][:, None]
    if s["shown"] is not None:
        begin = s["shown_begin"]
        row = torch.repeat_interleave(torch.arange(n, device=x.device), begin[1:] - begin[:-1], output_size=s["shown"].numel())
        count = torch.zeros(C * n, device=x.device).index_add_(0, s["shown"].long() * n + row, torch.ones(row.numel(), device=x.device)).view(C, n)
        by = torch.full((), s["repetition"], device=x.device)  # (a tensor, so that it is divided by, not multiplied by its inverse)
        less = torch.where(x > 0, x / by, x * by) - s["frequency"] * count - s["presence"]
        x = torch.where(count > 0, less, x)
    if s["allowed"] is not None:
        cls = torch.arange(C, device=x.device)
        bit = (s["allowed"][:, cls // 32] >> (cls % 32).int()) & 1  # [sets, classes]
        if s["allowed_set"] is not None:
            bit = bit[s["allowed_set"].long()]
        x = torch.where(bit.t() != 0, x, -math.inf)
    return x


def plain_top(s):
    x = plain_adjusted(s).t()
    n, C = x.shape
    lse = log_sum_exp(x / s["temperature"], 1)
    # keys that order by score, then by the lower class: all of them distinct
    bits = (x + 0.0).contiguous().view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * 2**32 + (2**32 - 1 - torch.arange(C, device=x.device))
    key = torch.where(x > -math.inf, key, -2**63)
    classes = 2**32 - 1 - (torch.topk(key, s["k"], dim=1).values & (2**32 - 1))
    listed_ = classes < C
    values = torch.where(listed_, x.gather(1, torch.where(listed_, classes, 0)), -math.inf)
    return dict(values=values, classes=torch.where(listed_, classes, -1).int(), lse=lse)


def plain_distill(s):
    z, T = s["scores"].float(), s["temperature"]
    C, n = z.shape
    cls, t = s["classes"].long(), s["teacher"].float() / T
    valid = (cls >= 0) & (cls < C) & (t > -math.inf)
    t = torch.where(valid, t, -math.inf)
    some = valid.any(1)
    total = s["teacher_lse"] if s["teacher_lse"] is not None else log_sum_exp(t, 1)
    q_entry = torch.where(valid, torch.exp(t - torch.where(some, total, torch.zeros_like(total))[:, None]), torch.zeros_like(t))
    at = torch.where(valid, cls, 0).t()
    q = torch.zeros(C, n, device=z.device).scatter_add_(0, at, q_entry.t())
    member = torch.zeros(C, n, device=z.device).scatter_add_(0, at, valid.t().float()) > 0
    zt = z / T
    lse = log_sum_exp(zt, 0)
    logp = zt - lse
    terms = torch.where(q > 0, q * (torch.log(q) - logp), torch.zeros_like(q))
    soft = terms.sum(0)
    other = torch.zeros_like(z)
    if s["teacher_lse"] is not None:
        lse_rest = log_sum_exp(torch.where(member, -math.inf, zt), 0)
        r = torch.where(some & (lse_rest > -math.inf), (1 - q_entry.sum(1)).clamp(min=0), torch.zeros_like(lse))
        soft = soft + torch.where(r > 0, r * (torch.log(r) - (lse_rest - lse)), torch.zeros_like(r))
        other = torch.where(member | (r == 0), other, r * torch.exp(zt - lse_rest))
    a = s["weight"] * some.float()
    loss = a * T * T * soft
    p = torch.exp(logp)
    g = a * T * (p - torch.where(member, q, other))
    h = a * p * (1 - p)
    if s["labels"] is not None:
        y = s["labels"]
        labelled = (y >= 0) & (y < C) & (y == torch.floor(y))
        at = torch.where(labelled, y, 0).long()
        b = (1 - s["weight"]) * labelled.float()
        log1 = z - log_sum_exp(z, 0)
        loss = loss + torch.where(labelled, -b * log1.gather(0, at[None])[0], torch.zeros_like(b))
        p1 = torch.exp(log1)
        g = g + b * (p1 - (torch.arange(C, device=z.device)[:, None] == at).float())
        h = h + b * p1 * (1 - p1)
    if not s["gradient"]:
        return dict(loss=loss)
    return dict(loss=loss, pairs=torch.stack((g, (2 * h).clamp(min=1e-16)), -1))


# ----------------------------------------------------------------------------------------------------- what is timed


def run(s):
    if own:
        from thundergbm_amd import scores
        if s["call"] == "distill":
            loss, pairs = scores.distill(s["scores"], s["classes"], s["teacher"], labels=s["labels"], teacher_lse=s["teacher_lse"],
                                         temperature=s["temperature"], weight=s["weight"], gradient=s["gradient"])
            return dict(loss=loss, pairs=pairs) if s["gradient"] else dict(loss=loss)
        known = dict(bias=s["bias"], allowed=s["allowed"], allowed_set=s["allowed_set"], shown=s["shown"], shown_begin=s["shown_begin"],
                     repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"])
        if s["call"] == "adjust":
            return scores.adjust(s["scores"], **known)
        values, classes, lse = scores.top(s["scores"], s["k"], temperature=s["temperature"], **known)
        return dict(values=values, classes=classes, lse=lse)
    if s["call"] == "distill":
        return plain_distill(s)
    if s["call"] == "adjust":
        return plain_adjusted(s).to(s["scores"].dtype)
    return plain_top(s)


def work(case):
    c = case
    n, C = c["rows"], c["classes"]
    if c["call"] == "distill":
        entry = 4 + (4 if c["teacher"] == "float32" else 2)
        per_row = c["entries"] * entry + 4 + (4 if c["rest"] else 0) + (4 if c["weight"] < 1 else 0)
        # an exponential, its sum and the largest value; then the pair. Twice where two temperatures meet
        twice = 2 if c["weight"] < 1 and c["temperature"] != 1 else 1
        return {"bytes": n * C * (12 if c["gradient"] else 4) + n * per_row, "flops": n * C * (4 * twice + (7 * twice if c["gradient"] else 0))}
    size = 4 if c["type"] == "float32" else 2
    nbytes = n * C * size * (2 if c["call"] == "adjust" else 1)
    nbytes += C * 4 if c["bias"] else 0
    nbytes += c["sets"] * ((C + 31) // 32) * 4 + (n * 4 if c["sets"] not in (0, 1, n) else 0)
    nbytes += n * (c["shown"] * 4 + 8) if c["shown"] else 0
    flops = n * C * ((1 if c["bias"] else 0) + (1 if c["sets"] else 0)) + n * c["shown"] * 4
    if c["call"] == "top":
        nbytes += n * (c["k"] * 8 + 4)
        flops += n * C * 5  # an exponential, its sum, the largest value, the comparison with the k-th
    return {"bytes": nbytes, "flops": flops}


# -------------------------------------------------------------------------------------------------- the definition


def exact_adjusted(s):
    """[rows, classes]. A score is a 32-bit number after every step, by definition: the order of the classes hangs on it."""
    x = s["scores"].t().to(torch.float32).contiguous()
    n, C = x.shape
    if s["bias"] is not None:
        x += s["bias"]
    if s["shown"] is not None:
        first, last = s["shown_begin"][:-1], s["shown_begin"][1:]
        row = torch.searchsorted(s["shown_begin"], torch.arange(s["shown"].numel(), device=x.device), right=True) - 1
        assert bool(((last - first) >= 0).all())
        pair, times = torch.unique(row * C + s["shown"].long(), return_counts=True)
        old = x.view(-1)[pair]
        strength = torch.tensor(s["repetition"], device=x.device)
        new = torch.where(old > 0, torch.div(old, strength), old * strength)
        new = new - s["frequency"] * times.to(torch.float32)
        x.view(-1)[pair] = new - s["presence"]
    if s["allowed"] is not None:
        words = s["allowed"].long() & 0xFFFFFFFF
        bits = ((words[:, :, None] >> torch.arange(32, device=x.device)) & 1).reshape(words.shape[0], -1)[:, :C].bool()
        which = s["allowed_set"].long() if s["allowed_set"] is not None else torch.arange(n, device=x.device) % words.shape[0]
        for a in range(0, n, 65_536):
            x[a:a + 65_536].masked_fill_(~bits[which[a:a + 65_536]], -math.inf)
    return x


def exact_top(s):
    x = exact_adjusted(s)
    k = s["k"]
    value, cls, lse = [], [], []
    for part in x.split(max(1, 50_000_000 // x.shape[1])):
        v, i = torch.sort(part, dim=1, descending=True, stable=True)
        v, i = v[:, :k], i[:, :k]
        value.append(v.double())
        cls.append(torch.where(v > -math.inf, i, -1).int())
        lse.append(torch.logsumexp(part.double() / s["temperature"], 1))
    return dict(values=torch.cat(value), classes=torch.cat(cls), lse=torch.cat(lse))


def exact_distill(s):
    T, w = s["temperature"], s["weight"]
    C, n = s["scores"].shape
    loss, pairs = [], []
    step = max(1, 60_000_000 // C)
    for a in range(0, n, step):
        part = slice(a, min(n, a + step))
        z = s["scores"][:, part].double()
        cls, t = s["classes"][part].long(), s["teacher"][part].double() / T
        there = cls >= 0
        t = t.masked_fill(~there, -math.inf)
        norm = s["teacher_lse"][part].double() if s["teacher_lse"] is not None else torch.logsumexp(t, 1)
        qe = torch.exp(t - norm[:, None])
        # one more class that takes the padding and is cut off again
        slot = torch.where(there, cls, C)
        q = torch.zeros(cls.shape[0], C + 1, dtype=torch.float64, device=z.device).scatter_add_(1, slot, qe)[:, :C].t()
        named = torch.zeros(cls.shape[0], C + 1, dtype=torch.bool, device=z.device).scatter_(1, slot, True)[:, :C].t()
        logp = torch.log_softmax(z / T, 0)
        p = logp.exp()
        soft = (torch.special.xlogy(q, q) - q * logp).sum(0)
        target = q
        if s["teacher_lse"] is not None:
            outside = logp.masked_fill(named, -math.inf)
            logR = torch.logsumexp(outside, 0)
            r = (1 - qe.sum(1)).clamp(min=0)
            r = torch.where(torch.isinf(logR), 0.0, r)
            soft = soft + torch.special.xlogy(r, r) - torch.where(r > 0, r * logR, 0.0)
            target = torch.where(named | torch.isinf(logR), q, r * torch.exp(outside - logR))
        total = w * T * T * soft
        g, h = w * T * (p - target), w * p * (1 - p)
        if s["labels"] is not None:
            y = s["labels"][part].long()
            log1 = torch.log_softmax(z, 0)
            total = total - (1 - w) * log1.gather(0, y[None])[0]
            p1 = log1.exp()
            h = h + (1 - w) * p1 * (1 - p1)
            g = g + (1 - w) * p1
            g.scatter_add_(0, y[None], torch.full((1, y.numel()), -(1 - w), dtype=torch.float64, device=z.device))
        loss.append(total)
        if s["gradient"]:
            pairs.append(torch.stack((g, (2 * h).clamp(min=1e-16)), -1).float() if C * n > 60_000_000 else torch.stack((g, (2 * h).clamp(min=1e-16)), -1))
    out = dict(loss=torch.cat(loss))
    if s["gradient"]:
        out["pairs"] = torch.cat(pairs, 1).double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["call"] == "distill":
        return exact_distill(s)
    if case["call"] == "adjust":
        return exact_adjusted(s).t().double()
    return exact_top(s)
