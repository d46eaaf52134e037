"""What more operators on class scores are measured on: `thundergbm_amd.scores`, on data that lies on the GPU.

`quantise` holds rows of numbers in 8 bits with a scale each, `linear` multiplies rows of features in 8 bits by a row of weights for every class - the
last layer of a larger model, which a student's trees are trained against or which answers beside them - and `sample` draws a class
of every row from its scores, under temperature and cuts, by random numbers that are given.

Scores are [classes, rows], with the rows of a class side by side ("class") or the classes of a row side by side ("row").
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def quantise_case(name, rows, features, **more):
    c = dict(name=name, call="quantise", rows=rows, features=features, type="bfloat16")
    c.update(more)
    return c


def linear_case(name, rows, features, classes, **more):
    """type: of the features ("int8": they are held so already); order and out: of the scores."""
    c = dict(name=name, call="linear", rows=rows, features=features, classes=classes, type="bfloat16", order="row", out="bfloat16", bias=False)
    c.update(more)
    return c


def sample_case(name, rows, classes, **more):
    """sets: allowed sets, 0 for none; shown: classes shown to a row on average, 0 for none; k: 0 for all; each: every row has cuts and a
    temperature of its own."""
    c = dict(name=name, call="sample", rows=rows, classes=classes, order="row", type="float32", bias=False, sets=0, shown=0, k=0, p=1.0, min_p=0.0,
             temperature=1.0, each=False)
    c.update(more)
    return c


def listed():
    return [
        # one request's features
        quantise_case("quantise_one_row", 1, 4096),
        # a teacher's weights, laid out once
        quantise_case("quantise_weights", 65_537, 1024),
        # one request of a service: the weights go by once
        linear_case("linear_one_row", 1, 4096, 32_000, out="float32", bias=True),
        # a small batch, very many classes
        linear_case("linear_small_batch", 24, 1000, 50_021, type="float16", out="float16"),
        # a table's scores for the trainer: few features, its order and type
        linear_case("linear_table", 100_003, 200, 500, type="float32", order="class", out="float32", bias=True),
        # a teacher's scores, from which the top ones are written down for a student
        linear_case("linear_teacher", 2048, 4096, 65_537, bias=True),
        # a teacher's scores for a large batch
        linear_case("linear_large", 8192, 8192, 32_000, type="int8"),
        # one request of a service, with a history
        sample_case("sample_one_row", 1, 32_000, bias=True, sets=1, shown=200, k=50, p=0.9, temperature=0.7),
        # drawn labels for a whole table of eight classes
        sample_case("sample_few_classes", 500_000, 8, order="class"),
        # recommendations with variety: drawn from the best of what is allowed to a row
        sample_case("sample_many_classes", 50_021, 1000, order="class", bias=True, sets=64, shown=20, k=40, p=0.95),
        # a batch of requests over a large vocabulary, each with its own settings
        sample_case("sample_requests", 256, 128_003, type="bfloat16", bias=True, each=True),
        # a large batch cut by its mass alone
        sample_case("sample_nucleus", 2048, 65_537, type="bfloat16", p=0.9, temperature=0.8),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    call = rng.choice(("quantise", "linear", "linear", "sample", "sample"))
    if call == "quantise":
        features = spread(rng, 8, 16_384)
        c = quantise_case("", spread(rng, 1, min(100_000, 67_000_000 // features)), features, type=rng.choice(tuple(TYPES)))
    elif call == "linear":
        features = spread(rng, 8, 8192)
        classes = spread(rng, 2, min(65_537, 500_000_000 // features))
        rows = spread(rng, 1, min(100_000, 130_000_000 // classes, 500_000_000 // features, 1_000_000_000_000 // (features * classes)))
        c = linear_case("", rows, features, classes, type=rng.choice((*TYPES, "int8")), order=rng.choice(("class", "row")), out=rng.choice(tuple(TYPES)),
                        bias=rng.random() < 0.5)
    else:
        few = rng.random() < 0.3
        classes = rng.randint(2, 32) if few else spread(rng, 33, 131_073)
        rows = spread(rng, 1, min(500_000, 100_000_000 // classes))
        order = "class" if few else rng.choice(("class", "row"))
        c = sample_case("", rows, classes, order=order, type=rng.choice(tuple(TYPES)) if order == "row" else "float32", bias=rng.random() < 0.4,
                        sets=rng.choice((0, 0, 1, 7, rows)), shown=rng.choice((0, 0, 0, 5, 40, 300)) if rows <= 50_000 else 0, each=rng.random() < 0.2,
                        temperature=rng.choice((1.0, 0.7, 2.0, 0.2)), k=rng.choice((0, 0, 1, 20, 50, 120, 500)), p=rng.choice((1.0, 1.0, 0.95, 0.8, 0.3)),
                        min_p=rng.choice((0.0, 0.0, 0.0, 0.05, 0.2)))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------- the inputs


def features_of(rows, features, dtype, gen):
    """Hidden features: some columns are much larger than the others, as they are in practice."""
    x = torch.randn(rows, features, device="cuda", generator=gen)
    large = torch.rand(features, device="cuda", generator=gen) < 0.01
    x *= torch.where(large, 8.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n = c["rows"]
    if c["call"] == "quantise":
        return dict(call="quantise", x=features_of(n, c["features"], TYPES[c["type"]], gen))
    C = c["classes"]
    if c["call"] == "linear":
        F, pitch = c["features"], (c["features"] + 127) // 128 * 128
        s = dict(call="linear", order=c["order"], out=TYPES[c["out"]], x_scale=None, bias=None)
        # weights in 8 bits, rows at multiples of 128 bytes, as a program that keeps them lays them out
        s["weight"] = torch.zeros(C, pitch, dtype=torch.int8, device="cuda")[:, :F]
        s["weight"].copy_(torch.randn(C, F, device="cuda", generator=gen).mul_(40).round_().clamp_(-127, 127))
        s["weight_scale"] = (0.75 + 0.5 * torch.rand(C, device="cuda", generator=gen)) / (40 * math.sqrt(F))
        if c["bias"]:
            s["bias"] = torch.randn(C, device="cuda", generator=gen)
        if c["type"] == "int8":
            s["x"] = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")[:, :F]
            s["x"].copy_(features_of(n, F, torch.float32, gen).mul_(12).round_().clamp_(-127, 127))
            s["x_scale"] = (0.5 + torch.rand(n, device="cuda", generator=gen)) / 12
        else:
            s["x"] = features_of(n, F, TYPES[c["type"]], gen)
        return s
    s = dict(call="sample", bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None, k=c["k"], p=c["p"], min_p=c["min_p"],
             temperature=c["temperature"], repetition=1.25, frequency=0.125, presence=0.5)
    if c["order"] == "row":
        s["scores"] = (torch.randn(n, C, device="cuda", generator=gen) * 2.5).to(TYPES[c["type"]]).t()
    else:
        s["scores"] = (torch.randn(C, n, device="cuda", generator=gen) * 2.5).to(TYPES[c["type"]])
    s["u"] = torch.rand(n, device="cuda", generator=gen)
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
    if c["each"]:  # one request in eight wants the best class, some have no cut, some have one or several

        def one_of(*values):
            return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (n,), device="cuda", generator=gen)]

        s["temperature"] = one_of(0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.0, 1.3)
        s["k"] = one_of(0, 0, 0, 20, 50, 400).int()
        s["p"] = one_of(1.0, 1.0, 0.9, 0.95, 0.5)
        s["min_p"] = one_of(0.0, 0.0, 0.05, 0.1)
    return s


# -------------------------------------------------------------------------------------------------- the plain forms


def plain_quantised(x):
    """The whole numbers of rows, as 32-bit floating numbers, and their scales."""
    x = x.float()
    by = torch.full((), 127.0, device=x.device)  # (a tensor, so that it is divided by, not multiplied by its inverse)
    scale = x.abs().amax(1) / by
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    return torch.where(scale[:, None] > 0, q, torch.zeros_like(q)), scale


def plain_linear(s):
    q, scale = (s["x"].float(), s["x_scale"]) if s["x_scale"] is not None else plain_quantised(s["x"])
    z = q @ s["weight"].float().t()
    z = z * scale[:, None] * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"]
    z = z.to(s["out"]).t()
    return z if s["order"] == "row" else z.contiguous()


def plain_adjusted(s):
    """The scores of the rows under the rules, in 32 bits, [rows, classes]."""
    x = s["scores"].float().t()
    n, C = x.shape
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["shown"] is not None:
        begin = s["shown_begin"]
        row = torch.repeat_interleave(torch.arange(n, device=x.device), begin[1:] - begin[:-1], output_size=s["shown"].numel())
        count = torch.zeros(n * C, device=x.device).index_add_(0, row * C + s["shown"].long(), torch.ones(row.numel(), device=x.device)).view(n, C)
        by = torch.full((), s["repetition"], device=x.device)
        less = torch.where(x > 0, x / by, x * by) - s["frequency"] * count - s["presence"]
        x = torch.where(count > 0, less, x)
    if s["allowed"] is not None:
        cls = torch.arange(C, device=x.device)
        bit = (s["allowed"][:, cls // 32] >> (cls % 32).int()) & 1  # [sets, classes]
        if s["allowed_set"] is not None:
            bit = bit[s["allowed_set"].long()]
        x = torch.where(bit != 0, x, -math.inf)
    return x


def a_row(v, x, dtype):
    """A setting as a number for each row, [rows or 1, 1], of the 32-bit value that it is."""
    v = v if isinstance(v, torch.Tensor) else torch.full((1,), v, device=x.device, dtype=torch.float32 if dtype.is_floating_point else dtype)
    return v.to(dtype)[:, None]


def plain_sample(s):
    x, cls = torch.sort(plain_adjusted(s), dim=1, descending=True, stable=True)
    T, p, min_p, k = a_row(s["temperature"], x, torch.float64), a_row(s["p"], x, torch.float64), a_row(s["min_p"], x, torch.float64), a_row(s["k"], x, torch.int64)
    place = torch.arange(x.shape[1], device=x.device)
    # 64 bits: a drawn class hangs on sums of all the others
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(T > 0, T, 1.0))
    w = torch.where(((place < k) | (k <= 0)) & (w >= min_p) & ((T > 0) | (place < 1)), w, 0.0)
    upto = torch.cumsum(w, 1)
    before = torch.cat((torch.zeros_like(upto[:, :1]), upto[:, :-1]), 1)
    kept = torch.where((before < p * upto[:, -1:]) & (w > 0), w, 0.0)
    total = kept.sum(1, keepdim=True)
    at = torch.minimum((upto <= s["u"].double()[:, None] * total).sum(1, keepdim=True), (kept > 0).sum(1, keepdim=True) - 1).clamp(min=0)
    some = total > 0  # (nothing is drawn where nothing is allowed)
    logp = torch.where(some, torch.log(kept.gather(1, at) / torch.where(some, total, 1.0)), -math.inf)
    return dict(classes=torch.where(some, cls.gather(1, at), -1)[:, 0].int(), logp=logp[:, 0].float())


# ----------------------------------------------------------------------------------------------------- what is timed


def run(s):
    if own:
        from thundergbm_amd import scores
        if s["call"] == "quantise":
            q, scale = scores.quantise(s["x"])
            return dict(values=q * scale[:, None], scale=scale)
        if s["call"] == "linear":
            return scores.linear(s["x"], s["weight"], s["weight_scale"], bias=s["bias"], x_scale=s["x_scale"], order=s["order"], dtype=s["out"])
        classes, logp = scores.sample(s["scores"], s["u"], k=s["k"], p=s["p"], min_p=s["min_p"], temperature=s["temperature"], bias=s["bias"],
                                      allowed=s["allowed"], allowed_set=s["allowed_set"], shown=s["shown"], shown_begin=s["shown_begin"],
                                      repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"])
        return dict(classes=classes, logp=logp)
    if s["call"] == "quantise":
        q, scale = plain_quantised(s["x"])
        return dict(values=q * scale[:, None], scale=scale)
    return plain_linear(s) if s["call"] == "linear" else plain_sample(s)


def work(case):
    c, n = case, case["rows"]
    if c["call"] == "sample":
        C = c["classes"]
        nbytes = n * C * (4 if c["type"] == "float32" else 2) + n * 12
        nbytes += C * 4 if c["bias"] else 0
        nbytes += c["sets"] * ((C + 31) // 32) * 4 + (n * 4 if c["sets"] not in (0, 1, n) else 0)
        nbytes += n * (c["shown"] * 4 + 8) if c["shown"] else 0
        nbytes += n * 16 if c["each"] else 0
        # the largest score; a comparison where the count cuts, else an exponential and its sum
        flops = n * C * (2 if c["k"] else 4) + n * C * ((1 if c["bias"] else 0) + (1 if c["sets"] else 0)) + n * c["shown"] * 4
        return {"bytes": nbytes, "flops": flops}
    F, size = c["features"], {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1}
    if c["call"] == "quantise":
        # (the values that the whole numbers stand for are written beside them)
        return {"bytes": n * F * (size[c["type"]] + 1 + 4) + n * 4, "flops": n * F * 4}
    C = c["classes"]
    nbytes = n * F * size[c["type"]] + C * F + n * C * size[c["out"]] + C * (8 if c["bias"] else 4) + (n * 4 if c["type"] == "int8" else 0)
    return {"bytes": nbytes, "flops": 2 * n * C * F}


# -------------------------------------------------------------------------------------------------- the definition


def exact_quantised(x):
    """The scale is a 32-bit number by definition, and so is what is rounded to a whole number: which one it becomes hangs on it."""
    x = x.to(torch.float32)
    scale = torch.div(x.abs().max(dim=1).values, torch.tensor(127.0, device=x.device))
    q = torch.div(x, torch.where(scale == 0, 1.0, scale).unsqueeze(1)).round()
    return q.double().clamp(-127, 127), scale


def exact_linear(s):
    q, scale = (s["x"].double(), s["x_scale"]) if s["x_scale"] is not None else exact_quantised(s["x"])
    z = torch.mm(s["weight"].double(), q.t().contiguous())
    z *= s["weight_scale"].double().unsqueeze(1)
    z *= scale.double().unsqueeze(0)
    if s["bias"] is not None:
        z += s["bias"].double().unsqueeze(1)
    return z


def exact_adjusted(s):
    """[rows, classes]. A score is a 32-bit number after every step, by definition: the order of the classes hangs on it."""
    x = s["scores"].t().to(torch.float32).contiguous()
    n, C = x.shape
    if s["bias"] is not None:
        x += s["bias"]
    if s["shown"] is not None:
        row = torch.searchsorted(s["shown_begin"], torch.arange(s["shown"].numel(), device=x.device), right=True) - 1
        pair, times = torch.unique(row * C + s["shown"].long(), return_counts=True)
        old = x.view(-1)[pair]
        strength = torch.tensor(s["repetition"], device=x.device)
        new = torch.where(old > 0, torch.div(old, strength), old * strength)
        x.view(-1)[pair] = (new - s["frequency"] * times.to(torch.float32)) - s["presence"]
    if s["allowed"] is not None:
        words = s["allowed"].long() & 0xFFFFFFFF
        bits = ((words[:, :, None] >> torch.arange(32, device=x.device)) & 1).reshape(words.shape[0], -1)[:, :C].bool()
        which = s["allowed_set"].long() if s["allowed_set"] is not None else torch.arange(n, device=x.device) % words.shape[0]
        for a in range(0, n, 65_536):
            x[a:a + 65_536].masked_fill_(~bits[which[a:a + 65_536]], -math.inf)
    return x


def exact_sample(s):
    x = exact_adjusted(s)
    n, C = x.shape
    setting = {}
    for name in ("temperature", "k", "p", "min_p"):
        v = s[name]
        setting[name] = (v.float() if isinstance(v, torch.Tensor) else torch.full((n,), float(v), device=x.device)).double()
    classes, logp = [], []
    step = max(1, 30_000_000 // C)
    for a in range(0, n, step):
        part = x[a:a + step]
        T, k, p, min_p = (setting[name][a:a + step, None] for name in ("temperature", "k", "p", "min_p"))
        order = torch.argsort(part, dim=1, descending=True, stable=True)
        z = part.gather(1, order).double()
        z = (z - z[:, :1]) / torch.where(T == 0, 1.0, T)
        rank = torch.arange(C, device=x.device).expand_as(z)
        z = z.masked_fill((T == 0) & (rank > 0), -math.inf)
        z = z.masked_fill((k > 0) & (rank >= k), -math.inf)
        z = z.masked_fill(z < torch.log(min_p), -math.inf)
        prob = torch.softmax(z, 1)
        front = torch.cumsum(prob, 1).roll(1, 1)
        front[:, 0] = 0
        z = z.masked_fill((front >= p) & (rank > 0) & (p < 1), -math.inf)
        prob = torch.softmax(z, 1)
        drawn = torch.searchsorted(torch.cumsum(prob, 1), s["u"][a:a + step].double()[:, None], right=True)
        drawn = torch.minimum(drawn, (prob > 0).sum(1, keepdim=True) - 1).clamp(min=0)
        nothing = ~(part > -math.inf).any(1)
        classes.append(order.gather(1, drawn)[:, 0].int().masked_fill(nothing, -1))
        logp.append(torch.log_softmax(z, 1).gather(1, drawn)[:, 0].masked_fill(nothing, -math.inf))
    return dict(classes=torch.cat(classes), logp=torch.cat(logp))


def exact(case, seed):
    s = prepare(case, seed)
    if case["call"] == "quantise":
        q, scale = exact_quantised(s["x"])
        return dict(values=q * scale.double()[:, None], scale=scale.double())
    return exact_linear(s) if case["call"] == "linear" else exact_sample(s)
