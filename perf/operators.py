"""The operators of training by distillation from a teacher's stored answers, and of the feature cache: the loss and gradient over a
teacher's top logits, and the 8-bit paged cache that features are written to and read back from.

`own` false computes them with elementary torch operations, true through the framework's entry points.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # distillation: loss and gradient (training), the loss alone (evaluation), the gradient alone (a backward pass of its own)
        # characters of transcripts for the frames of 32 clips, as a speech model answers them
        dict(name="characters", op="step", rows=16000, vocab=29, row=29, k=5, type="f32", t=2.0, padded=0.2),
        # one position of an ordinary vocabulary: the smallest call
        dict(name="one position", op="step", rows=1, vocab=32000, row=32000, k=20, type="bf16", t=1.0, padded=0.0),
        # a micro-batch; an odd vocabulary in rows that are a little longer
        dict(name="odd vocabulary", op="step", rows=2048, vocab=50257, row=50304, k=20, type="bf16", t=2.0, padded=0.1),
        # the largest training step
        dict(name="large vocabulary", op="step", rows=8192, vocab=131072, row=131072, k=64, type="bf16", t=1.5, padded=0.0),
        # evaluation in 32 bits, rows one element off every alignment
        dict(name="evaluation", op="loss", rows=1024, vocab=32001, row=32001, k=32, type="f32", t=1.0, padded=0.1),
        # the gradient by itself, with an upstream factor for each row
        dict(name="backward", op="grad", rows=4096, vocab=32000, row=32000, k=20, type="f16", t=2.0, padded=0.1),
        # cache: write (returns the values that the codes stand for, which the first epoch trains on) and read
        # streams that each append one frame
        dict(name="append", op="write", seqs=16, tokens=1, heads=8, dim=64, page=16, type="bf16", code="int8", ragged=False, start=True),
        # a loader's batch of log-mel spectrograms: 256 clips of up to 200 frames of 40 bands
        dict(name="spectrograms in", op="write", seqs=256, tokens=200, heads=1, dim=40, page=64, type="f32", code="int8", ragged=True, start=False),
        # long sequences with heads
        dict(name="long in", op="write", seqs=64, tokens=4096, heads=8, dim=128, page=64, type="bf16", code="e4m3", ragged=False, start=False),
        # the loader's batch in the epochs after the first
        dict(name="spectrograms out", op="read", seqs=256, tokens=200, heads=1, dim=40, page=64, type="f32", code="int8", ragged=True, start=False),
        # cepstra: rows of 13, pages that end inside every vector
        dict(name="cepstra out", op="read", seqs=512, tokens=333, heads=1, dim=13, page=7, type="f32", code="e4m3", ragged=True, start=True),
        dict(name="long out", op="read", seqs=64, tokens=4096, heads=8, dim=128, page=64, type="bf16", code="int8", ragged=True, start=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        op = rng.choice(["step", "step", "loss", "grad"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        vocab = _spread(rng, 20, 131072)
        rows = _spread(rng, 1, max(2, min(60000, int(1.0e9 * 2 / _SIZE[dtype]) // vocab)))
        row = vocab + rng.choice([0, 0, 1, (-vocab) % 64])
        k = min(vocab, rng.choice([1, 4, 5, 10, 20, 33, 64, 100]))
        return dict(op=op, rows=rows, vocab=vocab, row=row, k=k, type=dtype, t=rng.choice([0.7, 1.0, 2.0, 4.0]),
                    padded=rng.choice([0.0, 0.1, 0.4]) if rows > 1 else 0.0)
    op = rng.choice(["write", "read"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([13, 40, 64, 80, 96, 128, 161, 256, 512])
    heads = rng.choice([1, 1, 2, 8, 16])
    page = rng.choice([1, 7, 16, 64, 128, 256])
    seqs = _spread(rng, 1, 256)
    tokens = rng.choice([1, _spread(rng, 1, max(2, min(8192, 200_000_000 // (seqs * heads * dim))))])
    return dict(op=op, seqs=seqs, tokens=tokens, heads=heads, dim=dim, page=page, type=dtype, code=rng.choice(["int8", "e4m3"]),
                ragged=tokens > 1 and rng.random() < 0.6, start=rng.random() < 0.5)


def work(case):
    e = _SIZE[case["type"]]
    if case["op"] in ("step", "loss", "grad"):
        full = case["rows"] - int(case["rows"] * case["padded"])
        v = case["vocab"]
        read = full * (v * e + case["k"] * 8) + case["rows"] * 8
        wrote = case["rows"] * (v * e if case["op"] != "loss" else 0) + case["rows"] * 8
        return {"bytes": read + wrote, "flops": full * v * (4 if case["op"] == "loss" else 8)}
    groups = case["seqs"] * case["tokens"] * case["heads"] * (0.5 if case["ragged"] else 1.0)
    n = groups * case["dim"]
    out = n * e if case["op"] == "write" else case["seqs"] * case["tokens"] * case["heads"] * case["dim"] * e
    return {"bytes": n * 1 + groups * 4 + out + (n * e if case["op"] == "write" else 0), "flops": 4 * n}


# ---- what a program has before the call


def _prepare_distill(case, g):
    dev = "cuda"
    rows, v, k, dtype = case["rows"], case["vocab"], case["k"], _DTYPE[case["type"]]
    held = torch.empty(rows, case["row"], dtype=dtype, device=dev)
    # the teacher's ids: distinct, one out of each of k runs of the vocabulary
    width = v // k
    ids = torch.randint(0, width, (rows, k), generator=g, device=dev) + torch.arange(k, device=dev) * width
    ids = ids.gather(1, torch.rand(rows, k, generator=g, device=dev).argsort(1)).to(torch.int32)
    teacher = (14.0 - torch.rand(rows, k, generator=g, device=dev).mul_(12.0)).sort(1, descending=True).values
    full = rows - int(rows * case["padded"])
    ids[full:] = -1
    weights = torch.ones(rows, device=dev)
    weights[full:] = 0.0
    step = max(1, (1 << 27) // v)
    for r in range(0, rows, step):  # the student is about as sure as the teacher, of mostly the same ids
        part = torch.randn(min(step, rows - r), v, generator=g, device=dev).mul_(2.0)
        near = teacher[r:r + step] + torch.randn(part.shape[0], k, generator=g, device=dev)
        part.scatter_(1, ids[r:r + step].clamp_min(0).long(), near)
        held[r:r + step, :v] = part
    held[:, v:] = 0
    state = dict(case=case, logits=held[:, :v], ids=ids, teacher=teacher, weights=weights, scale=(1024.0 if case["type"] == "f16" else 1.0) / max(1, full))  # 16-bit gradients are scaled up
    if case["op"] == "grad":
        state["upstream"] = torch.rand(rows, generator=g, device=dev).add_(0.5)
        state["lse"] = torch.empty(rows, device=dev)
        for r in range(0, rows, step):
            state["lse"][r:r + step] = torch.logsumexp(state["logits"][r:r + step].double() / case["t"], 1).float()
        state["lse"][full:] = 0.0
    return state


def _prepare_cache(case, g):
    dev = "cuda"
    n, tokens, h, d, page, dtype = case["seqs"], case["tokens"], case["heads"], case["dim"], case["page"], _DTYPE[case["type"]]
    start = torch.randint(0, 3 * page, (n,), generator=g, device=dev, dtype=torch.int32) if case["start"] else None
    length = torch.randint(0, tokens + 1, (n,), generator=g, device=dev, dtype=torch.int32) if case["ragged"] else None
    pages = (tokens + (3 * page if case["start"] else 0) + page - 1) // page
    table = torch.randperm(n * pages, generator=g, device=dev).to(torch.int32).reshape(n, pages)
    held = torch.int8 if case["code"] == "int8" else torch.float8_e4m3fn
    state = dict(case=case, table=table, start=start, length=length)
    if case["op"] == "write":
        # features of a few loud and many quiet frames
        x = torch.randn(n, tokens, h, d, generator=g, device=dev)
        x *= torch.exp(torch.randn(n, tokens, h, 1, generator=g, device=dev))
        state["x"] = x.to(dtype)
        state["values"] = torch.zeros(n, tokens, h, d, dtype=dtype, device=dev)
        state["codes"] = torch.zeros(n * pages, page, h, d, dtype=torch.int8, device=dev).view(held)
        state["scales"] = torch.zeros(n * pages, page, h, device=dev)
    else:
        q = torch.randint(-127, 128, (n * pages, page, h, d), generator=g, device=dev, dtype=torch.int8)
        if case["code"] == "e4m3":  # every pattern but the two that are no numbers
            q = torch.where((q & 0x7F) == 0x7F, torch.zeros_like(q), q).view(held)
        state["codes"] = q
        state["scales"] = torch.exp(torch.randn(n * pages, page, h, generator=g, device=dev)) / _LARGEST[case["code"]]
    return state


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return _prepare_distill(case, g) if case["op"] in ("step", "loss", "grad") else _prepare_cache(case, g)


# ---- the framework's calls

_context = []


def _ctx():
    """The program's context, made at the first call."""
    if not _context:
        from aeon_b200.kernels import Context
        _context.append(Context(torch.cuda.current_device()))
    return _context[0]


def _own(state):
    from aeon_b200 import kernels as K
    case = state["case"]
    ctx = _ctx()
    if case["op"] == "step":
        loss, lse, grad = K.distill_loss(ctx, state["logits"], state["ids"], state["teacher"], temperature=case["t"],
                                         weights=state["weights"], grad_scale=state["scale"])
        return {"loss": loss, "lse": lse, "grad": grad}
    if case["op"] == "loss":
        loss, lse, _ = K.distill_loss(ctx, state["logits"], state["ids"], state["teacher"], temperature=case["t"],
                                      weights=state["weights"], want_grad=False)
        return {"loss": loss, "lse": lse}
    if case["op"] == "grad":
        grad = K.distill_grad(ctx, state["logits"], state["ids"], state["teacher"], state["lse"], temperature=case["t"],
                              weights=state["weights"], upstream=state["upstream"], grad_scale=state["scale"])
        return {"grad": grad}
    if "cache" not in state:
        state["cache"] = K.FeatureCache(ctx, state["codes"], state["scales"])
    if case["op"] == "write":
        state["cache"].write(state["x"], state["table"], start=state["start"], length=state["length"], values=state["values"])
        return {"values": state["values"], "scales": state["scales"]}
    out = state["cache"].read(state["table"], case["tokens"], start=state["start"], length=state["length"], dtype=_DTYPE[case["type"]])
    return {"values": out}


# ---- the plain forms


def _teacher(ids, teacher, weights, t):
    """p and log p of the valid entries (0 elsewhere), and which rows count."""
    valid = ids >= 0
    y = torch.where(valid, teacher / t, torch.full_like(teacher, -math.inf))
    top = y.amax(1, keepdim=True)
    rows = (top > -math.inf).squeeze(1) & (weights != 0)
    y = y - torch.where(top > -math.inf, top, torch.zeros_like(top))
    e = torch.exp(y)
    total = e.sum(1, keepdim=True).clamp_min(1e-30)
    p = e / total
    return p, torch.where(p > 0, y - torch.log(total), torch.zeros_like(y)), rows


def _gradient(x, ids, p, rows, lse, factor, dtype):
    """factor (exp(x - lse) - p at the ids), in place of x (the scaled logits)."""
    x.sub_(lse[:, None]).exp_()
    x.scatter_add_(1, ids.clamp_min(0).long(), -p)
    x.mul_(torch.where(rows, factor, torch.zeros_like(factor))[:, None])
    return x.to(dtype)


def _plain_distill(state):
    case = state["case"]
    t = case["t"]
    x = state["logits"].float() / t
    ids, weights = state["ids"], state["weights"]
    p, logp, rows = _teacher(ids, state["teacher"], weights, t)
    if case["op"] == "grad":
        factor = state["upstream"] * weights * (t * state["scale"])
        return {"grad": _gradient(x, ids, p, rows, state["lse"], factor, state["logits"].dtype)}
    top = x.amax(1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(1)) + top[:, 0]
    at = x.gather(1, ids.clamp_min(0).long())
    loss = (p * (logp - at + lse[:, None])).sum(1) * weights * (t * t)
    zero = torch.zeros_like(loss)
    out = {"loss": torch.where(rows, loss, zero), "lse": torch.where(rows, lse, zero)}
    if case["op"] == "step":
        out["grad"] = _gradient(x, ids, p, rows, lse, weights * (t * state["scale"]), state["logits"].dtype)
    return out


def _places(state):
    """Page, place in it, and whether there is a token at all, for each sequence and token."""
    case, table = state["case"], state["table"]
    at = torch.arange(case["tokens"], device=table.device)[None, :].expand(case["seqs"], -1)
    there = at < state["length"][:, None] if state["length"] is not None else torch.ones_like(at, dtype=torch.bool)
    if state["start"] is not None:
        at = at + state["start"][:, None]
    return table.long().gather(1, at // case["page"]), at % case["page"], there


def _grid(y, code):
    """y to the nearest number of the code, ties to even (in the type of y, which holds them all)."""
    if code == "int8":
        return torch.round(y)
    e = torch.frexp(y).exponent - 1  # |y| is in [2^e, 2^(e+1))
    step = torch.ldexp(torch.ones_like(y), e.clamp_min(-6) - 3)
    return (torch.round(y / step) * step).clamp_(-448.0, 448.0)


def _plain_write(state):
    case = state["case"]
    x, codes, scales, values = state["x"], state["codes"], state["scales"], state["values"]
    page, place, there = _places(state)
    x = x.float()[there]  # tokens x heads x dim
    # the quotients in 64 bits: in 32 those next to the middle between two codes would fall to either side
    scale = (x.abs().amax(-1).double() / _LARGEST[case["code"]]).float().clamp_min(2.0 ** -126)
    q = _grid(x.double() / scale.double()[..., None], case["code"])
    page, place = page[there], place[there]
    q = q.float()
    codes.view(torch.int8)[page, place] = q.to(codes.dtype).view(torch.int8)
    scales[page, place] = scale
    values[there] = (q * scale[..., None]).to(values.dtype)
    return {"values": values, "scales": scales}


def _plain_read(state):
    case = state["case"]
    page, place, there = _places(state)
    page = torch.where(there, page, torch.zeros_like(page))
    x = state["codes"].view(torch.int8)[page, place].view(state["codes"].dtype).float() * state["scales"][page, place][..., None]
    return {"values": torch.where(there[..., None, None], x, torch.zeros_like(x)).to(_DTYPE[case["type"]])}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_write(state) if op == "write" else _plain_read(state) if op == "read" else _plain_distill(state)


# ---- the definitions in 64 bits


def _exact_distill(case, s):
    rows, v, k, t = case["rows"], case["vocab"], case["k"], case["t"]
    full = rows - int(rows * case["padded"])  # the rows behind are padding
    logits, ids, teacher = s["logits"], s["ids"].long(), s["teacher"].double()
    loss, lse = torch.zeros(2, rows, dtype=torch.float64, device="cuda").unbind(0)
    grad = torch.zeros(rows, v, dtype=torch.float64, device="cuda") if case["op"] != "loss" else None
    p = torch.softmax(teacher / t, 1)
    step = max(1, (1 << 27) // v)
    for r in range(0, full, step):
        part = slice(r, min(full, r + step))
        x = logits[part].double() / t
        z = torch.logsumexp(x, 1) if case["op"] != "grad" else s["lse"][part].double()
        lse[part] = z
        loss[part] = t * t * (torch.special.xlogy(p[part], p[part]) + p[part] * (z[:, None] - x.gather(1, ids[part]))).sum(1)
        if grad is not None:
            x = torch.exp(x - z[:, None])
            x.scatter_add_(1, ids[part], -p[part])
            f = t * s["scale"] * (s["upstream"][part].double() if case["op"] == "grad" else torch.ones_like(z))
            grad[part] = x * f[:, None]
    if case["op"] == "grad":
        return {"grad": grad}
    return {"loss": loss, "lse": lse} if grad is None else {"loss": loss, "lse": lse, "grad": grad}


def _numbers(code):
    """The non-negative numbers of a code, ascending."""
    if code == "int8":
        return torch.arange(128, dtype=torch.float64)
    return torch.tensor([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64)


def _exact_cache(case, s):
    n, tokens, h, d, page = case["seqs"], case["tokens"], case["heads"], case["dim"], case["page"]
    begin = s["start"].tolist() if s["start"] is not None else [0] * n
    count = s["length"].tolist() if s["length"] is not None else [tokens] * n
    table = s["table"].long()
    out = torch.zeros(n, tokens, h, d, dtype=torch.float64, device="cuda")
    scales = s["scales"].double()
    numbers = _numbers(case["code"]).cuda()
    middle = (numbers[1:] + numbers[:-1]) / 2
    for i in range(n):
        at = torch.arange(begin[i], begin[i] + count[i], device="cuda")
        pages, places = table[i][at // page], at % page
        if case["op"] == "read":
            q = s["codes"][pages, places].float().double()
            out[i, :count[i]] = q * scales[pages, places][..., None]
            continue
        x = s["x"][i, :count[i]].double()
        scale = (x.abs().amax(-1) / _LARGEST[case["code"]]).float().double().clamp_min(2.0 ** -126)  # held in 32 bits
        y = (x.abs() / scale[..., None])
        low, high = torch.searchsorted(middle, y), torch.searchsorted(middle, y, right=True)
        q = numbers[torch.where(low % 2 == 0, low, high)]  # in the middle of two: the even one
        out[i, :count[i]] = torch.copysign(q, x) * scale[..., None]
        scales[pages, places] = scale
    return {"values": out, "scales": scales} if case["op"] == "write" else {"values": out}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_distill(case, s) if case["op"] in ("step", "loss", "grad") else _exact_cache(case, s)
