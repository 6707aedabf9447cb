"""The distillation loss and its gradient against the 64-bit oracle.

Tolerances, from the operations (u = 2^-24, one float32 rounding; all logarithms to the base 2 in the kernel):
* an exponential: its argument (x - m) log2(e) / T carries three roundings of at most R = the row's range of x / T each, 3 R u
  absolute, and the function 2 ulp: relative error E = (3 R + 4) u.  The sum over the vocabulary adds one rounding per addition
  of the longest chain of additions, at most V / 32 + 64 (a warp's lanes, the finest split): lse is off by
  (E + (V / 32 + 64) u) + 2 |lse| u.
* loss: w T^2 sum p (log p - s / T + lse): each of the terms is off by 4 u times its size (R + log k + |log V|) and by what lse is.
* gradient: g (q - P): q relative E plus lse's error, P relative (E + (k + 8) u); then half a step of the type, relative to the
  result, and half its smallest subnormal.  Exponentials against the row's largest value (or lse) that are below 2^-126 count as 0:
  the sum is at least 1, so each is off by 2^-126 at most, and the product with g carries that on as |g| 2^-126.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import distill as odistill

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def make(rng, rows, vocab, k, dtype, pad=0, spread=3.0):
    """Logits in a buffer `pad` elements longer per row, ids with repeats, teacher's logits."""
    held = torch.from_numpy(rng.normal(0, spread, (rows, vocab + pad)).astype(np.float32)).cuda().to(TYPES[dtype])
    ids = torch.from_numpy(rng.integers(0, vocab, (rows, k)).astype(np.int32)).cuda()
    teacher = torch.from_numpy(rng.normal(0, 4, (rows, k)).astype(np.float32)).cuda()
    return held[:, :vocab], ids, teacher


def bounds(x, want, dtype, t, w, factor, k):
    """Tolerances of loss, lse and gradient (finite rows), by the rules above."""
    rows, vocab = x.shape
    y = x / t
    finite = np.where(np.isfinite(y), y, y.max(1, keepdims=True))
    reach = finite.max(1) - finite.min(1) + np.abs(finite).max(1)
    e = (3 * reach + 4) * U
    lse_tol = e + (vocab / 32 + 64) * U + 2 * np.abs(want[1]) * U
    loss_tol = np.abs(w) * t * t * (lse_tol + 4 * U * (reach + np.log(k) + np.log(vocab) + 40))
    q = np.exp(y - want[1][:, None])
    grad_tol = np.abs(factor)[:, None] * (q * (lse_tol + e + 4 * U)[:, None] * 1.1 + (np.abs(want[2]) / np.maximum(np.abs(factor)[:, None], 1e-300) + q)
                                          * (e[:, None] + (k + 8) * U)) \
        + np.abs(want[2]) * torch.finfo(TYPES[dtype]).eps / 2 * 1.01 + TINY[dtype] / 2 + np.abs(factor)[:, None] * 2.0 ** -126
    # rows with a NaN among the logits have no tolerance: they are NaN, or exactly 0 where they do not count
    return tuple(np.where(np.isnan(v), 0.0, v) for v in (loss_tol, lse_tol, grad_tol))


def compare(got, want, tol, what):
    got = got.double().cpu().numpy() if torch.is_tensor(got) else got
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(np.isinf(got), np.isinf(want)), what
    ok = np.isfinite(want)
    with np.errstate(invalid="ignore"):
        bad = ok & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


def check(ctx, logits, ids, teacher, t=1.0, weights=None, upstream=None, scale=1.0, dtype="f32"):
    """Every form of the call against the oracle; returns the fused call's results."""
    from aeon_b200 import kernels as K
    rows, vocab = logits.shape
    x = logits.double().cpu().numpy()
    w = None if weights is None else torch.tensor(weights, dtype=torch.float32, device="cuda")
    up = None if upstream is None else torch.tensor(upstream, dtype=torch.float32, device="cuda")
    wn = np.ones(rows) if w is None else w.double().cpu().numpy()
    un = np.ones(rows) if up is None else up.double().cpu().numpy()
    tn = np.float64(np.float32(t))
    want = odistill.distill(x, ids.cpu().numpy(), teacher.double().cpu().numpy(), tn, wn, un, np.float32(scale))
    factor = wn * un * tn * float(np.float32(scale))
    with np.errstate(invalid="ignore", over="ignore"):
        tol = bounds(x, want, dtype, tn, wn, factor, ids.shape[1])
    loss, lse, grad = K.distill_loss(ctx, logits, ids, teacher, t, w, up, scale)
    compare(loss, want[0], tol[0], "loss")
    compare(lse, want[1], tol[1], "lse")
    compare(grad, want[2], tol[2], "gradient")
    loss2, lse2, none = K.distill_loss(ctx, logits, ids, teacher, t, w, want_grad=False)
    assert none is None
    compare(loss2, want[0], tol[0], "loss alone")
    compare(lse2, want[1], tol[1], "lse alone")
    grad2 = K.distill_grad(ctx, logits, ids, teacher, lse2, t, w, up, scale)
    compare(grad2, want[2], tol[2], "gradient alone")
    return loss, lse, grad


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k,pad", [
    (1, 1, 1, 0), (3, 2, 3, 0), (7, 29, 5, 0), (33, 29, 5, 3), (5, 31, 2, 1), (4, 32, 32, 0), (9, 33, 7, 0), (2, 64, 256, 0),
    (3, 127, 8, 1), (6, 256, 10, 0), (2, 511, 100, 1), (5, 1000, 20, 24), (3, 1023, 9, 0), (4, 1025, 9, 2), (2, 2047, 33, 1),
    (3, 4096, 20, 0), (2, 4099, 255, 5), (2, 8191, 17, 1), (3, 8200, 64, 0), (2, 16385, 20, 0),
])
def test_sizes_types_and_strides(ctx, dtype, rows, vocab, k, pad):
    rng = np.random.default_rng(rows * 1000003 + vocab * 31 + k)
    logits, ids, teacher = make(rng, rows, vocab, k, dtype, pad)
    check(ctx, logits, ids, teacher, t=1.0 if k % 2 else 2.5, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,pad", [(32000, 0), (32001, 0), (50257, 47), (65536, 0), (100003, 1), (131072, 0), (131077, 3), (300007, 0)])
def test_long_rows(ctx, dtype, vocab, pad):
    rng = np.random.default_rng(vocab)
    logits, ids, teacher = make(rng, 3, vocab, 20, dtype, pad)
    check(ctx, logits, ids, teacher, t=2.0, weights=[1.0, 0.25, 3.0], dtype=dtype)


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (17, 4096), (149, 1000), (300, 33), (2000, 29), (1200, 8191), (700, 32000)])
def test_many_rows(ctx, rows, vocab):
    """Row counts around those at which the launch changes; the oracle on a sample of rows."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(rows + vocab)
    g = torch.Generator("cuda")
    g.manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=g, device="cuda").mul_(3).bfloat16()
    ids = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda", dtype=torch.int32)
    teacher = torch.randn(rows, 6, generator=g, device="cuda")
    loss, lse, grad = K.distill_loss(ctx, logits, ids, teacher, 1.5)
    at = torch.from_numpy(np.unique(rng.integers(0, rows, 24)))
    x = logits[at.cuda()].double().cpu().numpy()
    want = odistill.distill(x, ids.cpu()[at].numpy(), teacher.cpu()[at].double().numpy(), 1.5)
    n = len(at)
    tol = bounds(x, want, "bf16", 1.5, np.ones(n), np.full(n, 1.5), 6)
    compare(loss.cpu()[at], want[0], tol[0], "loss")
    compare(lse.cpu()[at], want[1], tol[1], "lse")
    compare(grad.cpu()[at], want[2], tol[2], "gradient")
    grad2 = K.distill_grad(ctx, logits, ids, teacher, lse, 1.5)
    compare(grad2.cpu()[at], want[2], tol[2], "gradient alone")
    # a row's result does not depend on the rows beside it, nor on the run
    again = K.distill_loss(ctx, logits, ids, teacher, 1.5)
    for a, b in zip((loss, lse, grad), again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("vocab", [29, 1000, 32001, 140001])
def test_weights_upstream_temperature(ctx, vocab):
    rng = np.random.default_rng(vocab + 1)
    for t, scale in ((0.25, 1.0), (1.0, 1e-3), (7.0, -2.0)):
        logits, ids, teacher = make(rng, 5, vocab, 11, "f32", 1)
        check(ctx, logits, ids, teacher, t, [1.0, 0.0, -1.5, 0.5, 2.0], [0.5, 1.0, 0.0, -2.0, 1.0], scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 5000, 40000, 150000])
def test_rows_without_entries_and_numbers(ctx, dtype, vocab):
    """Rows whose mask leaves nothing are zero whatever their logits hold; infinities and NaN stay in their rows."""
    rng = np.random.default_rng(vocab + 2)
    inf, nan = float("inf"), float("nan")
    logits, ids, teacher = make(rng, 16, vocab, 4, dtype, 1)
    ids[0] = -1                                     # no entry
    logits[0] = nan
    logits[1] = nan                                 # weight 0
    teacher[2] = -inf                               # no entry again
    ids[3, 1:] = -1                                 # one entry: cross entropy
    teacher[4, 2] = -inf                            # an entry that does not count, at a valid id
    teacher[5, 0] = nan                             # -> NaN
    teacher[6, 0] = inf                             # -> NaN
    ids[7, 3] = vocab                               # -> NaN, nothing read there
    ids[8, 0] = 2 ** 31 - 1                         # -> NaN
    teacher[8, 0] = -inf                            # ... but this entry does not count
    logits[9, vocab // 2] = nan                     # -> NaN
    logits[10, vocab - 1] = inf                     # -> NaN
    logits[11] = -inf                               # -> NaN
    logits[12, : vocab - 1] = -inf                  # one value left
    ids[12] = vocab - 1
    ids[13] = 3                                     # the same id four times
    logits[14, 1] = -inf                            # the teacher wants what the student rules out: loss +inf, gradient finite
    ids[14, 0] = 1
    ids[14, 1:] = 2
    teacher[14] = 0.0
    logits[15] = -3.0e38 if dtype == "f32" else -3.0e38  # the type's lowest values, all alike
    ids[15] = torch.arange(4, dtype=torch.int32)
    weights = [1.0] * 16
    weights[1] = 0.0
    loss, lse, grad = check(ctx, logits, ids, teacher, 1.0, weights, dtype=dtype)
    for r in (0, 1, 2):
        assert loss[r] == 0 and lse[r] == 0 and not grad[r].any()
    for r in (5, 6, 7, 9, 10, 11):
        assert loss[r].isnan() and lse[r].isnan() and grad[r].isnan().all()
    assert loss[14] == inf and grad[14].isfinite().all()


def test_a_mask_of_the_lowest_value(ctx):
    """Logits masked with the type's lowest value have no probability and no gradient."""
    rng = np.random.default_rng(12)
    for dtype in TYPES:
        logits, ids, teacher = make(rng, 4, 3001, 6, dtype)
        logits[:, 1500:] = torch.finfo(TYPES[dtype]).min
        ids %= 1500
        _, _, grad = check(ctx, logits, ids, teacher, 1.0, dtype=dtype)
        assert not grad[:, 1500:].any()


def test_three_dimensions_and_refusals(ctx):
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(13)
    logits, ids, teacher = make(rng, 12, 100, 5, "bf16", 28)
    flat = K.distill_loss(ctx, logits, ids, teacher, 2.0)
    cube = K.distill_loss(ctx, logits.unflatten(0, (3, 4)), ids.view(3, 4, 5), teacher.view(3, 4, 5), 2.0)
    for a, b in zip(flat, cube):
        assert torch.equal(a.reshape(b.shape), b)
    for bad in (lambda: K.distill_loss(ctx, logits.cpu(), ids, teacher),
                lambda: K.distill_loss(ctx, logits, ids.long(), teacher),
                lambda: K.distill_loss(ctx, logits, ids, teacher.half()),
                lambda: K.distill_loss(ctx, logits, ids[:, :4], teacher),
                lambda: K.distill_loss(ctx, logits[:6], ids, teacher),
                lambda: K.distill_loss(ctx, logits.double(), ids, teacher),
                lambda: K.distill_loss(ctx, logits.t(), torch.zeros(100, 5, dtype=torch.int32, device="cuda"), torch.zeros(100, 5, device="cuda")),
                lambda: K.distill_loss(ctx, logits.unflatten(0, (3, 4)).transpose(0, 1), ids.view(4, 3, 5), teacher.view(4, 3, 5)),
                lambda: K.distill_loss(ctx, logits, ids, teacher, weights=torch.ones(11, device="cuda")),
                lambda: K.distill_loss(ctx, logits, ids, teacher, grad=torch.empty(12, 99, dtype=logits.dtype, device="cuda")),
                lambda: K.distill_loss(ctx, logits, ids, teacher, grad=torch.empty(12, 100, device="cuda")),
                lambda: K.distill_grad(ctx, logits, ids, teacher, torch.ones(3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for t in (0.0, -1.0, float("nan")):
        with pytest.raises(RuntimeError):
            K.distill_loss(ctx, logits, ids, teacher, t)
    with pytest.raises(RuntimeError):
        K.distill_loss(ctx, logits, torch.zeros(12, 257, dtype=torch.int32, device="cuda"), torch.zeros(12, 257, device="cuda"))
    empty = K.distill_loss(ctx, logits[:0], ids[:0], teacher[:0])
    assert [tuple(x.shape) for x in empty] == [(0,), (0,), (0, 100)]


@pytest.mark.parametrize("vocab,pad", [(29, 0), (1001, 3), (32000, 0), (150001, 1)])
def test_gradient_in_place(ctx, vocab, pad):
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(vocab + 3)
    logits, ids, teacher = make(rng, 40, vocab, 7, "bf16", pad)
    ids[3] = ids[3, 0]
    want = K.distill_loss(ctx, logits, ids, teacher, 2.0)
    held = torch.full((40, vocab + pad), 5.0, dtype=torch.bfloat16, device="cuda")
    a, b = held[:, :vocab], held.clone()[:, :vocab]
    a.copy_(logits)
    b.copy_(logits)
    loss, lse, grad = K.distill_loss(ctx, a, ids, teacher, 2.0, grad=a)
    assert grad is a and torch.equal(a, want[2]) and torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    assert (held[:, vocab:] == 5.0).all()  # what lies between the rows stays
    alone = K.distill_grad(ctx, logits, ids, teacher, lse, 2.0)
    K.distill_grad(ctx, b, ids, teacher, lse, 2.0, grad=b)
    assert torch.equal(b, alone)


def test_gradients_lie_as_the_logits_do(ctx):
    """Views into the middle of a tensor, padded and broadcast rows: the gradient has the logits' strides and place in 16 bytes where it
    can, and the same values wherever it is written."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(22)
    for dtype in TYPES:
        for vocab in (29, 501, 9001):
            whole, ids, teacher = make(rng, 9, vocab, 5, dtype)
            whole = whole.contiguous()
            padded = torch.zeros(9, vocab + 7, dtype=TYPES[dtype], device="cuda")[:, 3:vocab + 3]
            padded.copy_(whole)
            for x, i, t in ((whole[1:], ids[1:], teacher[1:]), (whole[2:7], ids[2:7], teacher[2:7]), (padded, ids, teacher), (padded[4:], ids[4:], teacher[4:])):
                loss, lse, grad = K.distill_loss(ctx, x, i, t, 2.0)
                assert grad.shape == x.shape and grad.stride() == x.stride() and (grad.data_ptr() - x.data_ptr()) % 16 == 0
                elsewhere = torch.empty(x.shape[0], vocab + 1, dtype=x.dtype, device="cuda")[:, 1:]
                K.distill_loss(ctx, x, i, t, 2.0, grad=elsewhere)
                assert torch.equal(elsewhere, grad)
                assert torch.equal(K.distill_grad(ctx, x, i, t, lse, 2.0), K.distill_grad(ctx, x, i, t, lse, 2.0, grad=elsewhere))
            same = K.distill_loss(ctx, whole[:1].expand(4, vocab), ids[:4], teacher[:4], 2.0)
            assert same[2].is_contiguous()
            one = [K.distill_loss(ctx, whole[:1], ids[j:j + 1], teacher[j:j + 1], 2.0) for j in range(4)]
            assert torch.equal(same[0], torch.cat([o[0] for o in one])) and torch.equal(same[2], torch.cat([o[2] for o in one]))


def test_what_lies_around_the_outputs_stays(ctx):
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(14)
    for vocab in (29, 500, 33333):
        for dtype in TYPES:
            logits, ids, teacher = make(rng, 21, vocab, 5, dtype, 1)
            held = torch.full((23 * (vocab + 5),), 7.0, dtype=TYPES[dtype], device="cuda")
            grad = held[vocab + 5 + 3:][: 21 * (vocab + 5)].view(21, vocab + 5)[:, :vocab]
            K.distill_loss(ctx, logits, ids, teacher, grad=grad)
            mask = torch.ones_like(held, dtype=torch.bool)
            mask[vocab + 5 + 3:][: 21 * (vocab + 5)].view(21, vocab + 5)[:, :vocab] = False
            assert (held[mask] == 7.0).all()


def test_gradient_against_differences_of_the_loss(ctx):
    """Central differences with h = 2^-5 of the kernel's own float32 loss: h^2 / 6 times the third derivative (at most 1 / T here)
    plus twice the loss's error over 2 h."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(15)
    vocab, h, t = 23, 2.0 ** -5, 2.0
    logits, ids, teacher = make(rng, 1, vocab, 4, "f32")
    _, _, grad = K.distill_loss(ctx, logits, ids, teacher, t)
    step = torch.eye(vocab, device="cuda") * h
    many = lambda x: K.distill_loss(ctx, x, ids.expand(vocab, 4), teacher.expand(vocab, 4), t, want_grad=False)[0]  # noqa: E731
    diff = (many(logits + step) - many(logits - step)) / (2 * h)
    x = logits.double().cpu().numpy()
    want = odistill.distill(x, ids.cpu().numpy(), teacher.double().cpu().numpy(), t)
    loss_tol = bounds(x, want, "f32", t, np.ones(1), np.full(1, t), 4)[0][0]
    assert (diff - grad[0]).abs().max().item() <= h * h / 6 / t + loss_tol / h * 1.5


def test_another_stream_and_device_of_the_caller(ctx):
    """Inputs made and results read on the caller's stream without a wait of the caller's."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(16)
    logits, ids, teacher = make(rng, 64, 32000, 20, "bf16")
    want = [x.clone() for x in K.distill_loss(ctx, logits, ids, teacher)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            late = torch.empty_like(logits)
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(20):
                big = big @ big * 1e-3  # keeps the stream busy
            late.copy_(logits)
            got = K.distill_loss(ctx, late, ids, teacher)
            late.fill_(0)
            same = [torch.equal(a, b) for a, b in zip(got, want)]
            assert all(same)
    with torch.cuda.stream(ctx.torch_stream):
        got = K.distill_loss(ctx, logits, ids, teacher)
    ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("vocab", [29, 4000, 150000])
def test_two_captured_graphs(ctx, vocab):
    """Two graphs of the same context replayed after their inputs have changed, in turn and one behind the other."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(17)
    sets, graphs = [], []
    for i in range(2):
        logits, ids, teacher = make(rng, 9, vocab, 6, "bf16")
        logits = logits.contiguous()
        K.distill_loss(ctx, logits, ids, teacher, 2.0)  # first launches outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = K.distill_loss(ctx, logits, ids, teacher, 2.0)
            alone = K.distill_grad(ctx, logits, ids, teacher, out[1], 2.0)
        sets.append((logits, ids, teacher, out, alone))
        graphs.append(g)
    for turn in range(2):
        for logits, ids, teacher, _, _ in sets:
            fresh = make(rng, 9, vocab, 6, "bf16")
            for a, b in zip((logits, ids, teacher), fresh):
                a.copy_(b)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for logits, ids, teacher, out, alone in sets:
            want = K.distill_loss(ctx, logits, ids, teacher, 2.0)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert torch.equal(alone, K.distill_grad(ctx, logits, ids, teacher, want[1], 2.0))


def test_a_first_call_inside_a_capture(ctx):
    """Sizes and entries that no other test uses: what the library asks the driver for at their first call is allowed there."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(20)
    for vocab, k in ((9001, 70), (70003, 129)):
        logits, ids, teacher = make(rng, 300, vocab, k, "f16")
        logits = logits.contiguous()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = K.distill_loss(ctx, logits, ids, teacher, 2.0)
        g.replay()
        torch.cuda.synchronize()
        again = K.distill_loss(ctx, logits, ids, teacher, 2.0)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("k", [31, 33, 64, 65, 200])
@pytest.mark.parametrize("vocab", [100, 700, 3000, 9000, 40000, 140000])
def test_many_entries_with_repeats(ctx, k, vocab):
    """Entry counts around those at which the kernels change, ids that occur often, all at one end of the row or spread."""
    rng = np.random.default_rng(k * 7 + vocab)
    logits, ids, teacher = make(rng, 4, vocab, k, "f32", 3)
    ids[0] = ids[0] % 7 + vocab - 7
    ids[1] = torch.arange(k, dtype=torch.int32) % vocab
    ids[2, ::2] = ids[2, 0]
    ids[2, 1::3] = -1
    check(ctx, logits, ids, teacher, 1.5, [1.0, -0.5, 2.0, 1.0], [1.0, 2.0, 0.5, -1.0])


def test_temperatures_at_the_ends(ctx):
    """The coldest and the hottest temperature: all on the largest value, all alike."""
    rng = np.random.default_rng(21)
    for vocab in (50, 5000, 50000):
        for t in (2.0 ** -40, 2.0 ** 40):
            logits, ids, teacher = make(rng, 3, vocab, 5, "f32")
            from aeon_b200 import kernels as K
            loss, lse, grad = K.distill_loss(ctx, logits, ids, teacher, t)
            assert lse.isfinite().all() and grad.isfinite().all()
            top = logits.max(1).values.double()
            if t < 1:  # q is 1 at the largest value and 0 elsewhere, p too
                want = torch.zeros(3, vocab, dtype=torch.float64, device="cuda")
                want.scatter_add_(1, logits.argmax(1, keepdim=True), torch.full((3, 1), t, dtype=torch.float64, device="cuda"))
                want.scatter_add_(1, ids.gather(1, teacher.argmax(1, keepdim=True)).long(), torch.full((3, 1), -t, dtype=torch.float64, device="cuda"))
                assert (grad.double() - want).abs().max().item() <= t * 2.0 ** -20
                assert ((lse.double() * t - top).abs() <= top.abs() * 2.0 ** -22).all()
            else:
                want = torch.full((3, vocab), t / vocab, dtype=torch.float64, device="cuda")
                want.scatter_add_(1, ids.long(), torch.full((3, 5), -t / 5, dtype=torch.float64, device="cuda"))
                assert (grad.double() - want).abs().max().item() <= t * 2.0 ** -20


def test_offsets_past_32_bits(ctx):
    """Rows so far apart that byte and element offsets pass 2^32."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(18)
    for vocab in (29, 32000):
        logits, ids, teacher = make(rng, 3, vocab, 6, "bf16")
        far = 2 ** 31 + 24
        held = torch.empty(2 * far + vocab, dtype=torch.bfloat16, device="cuda")
        rows = held.as_strided((3, vocab), (far, 1))
        rows.copy_(logits)
        want = K.distill_loss(ctx, logits, ids, teacher, 2.0)
        got = K.distill_loss(ctx, rows, ids, teacher, 2.0, grad=rows)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del held, rows, got


def test_profile_counts_the_launches(ctx):
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(19)
    logits, ids, teacher = make(rng, 8, 1000, 6, "bf16")
    ctx.profile(True)
    _, lse, _ = K.distill_loss(ctx, logits, ids, teacher)
    K.distill_grad(ctx, logits, ids, teacher, lse)
    got = ctx.profile_read()["other"]
    ctx.profile(False)
    assert got["launches"] == 2 and got["algorithmic_bytes"] == 2 * 8 * (1000 * 2 * 2 + 6 * 8 + 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(7001, 2100, 20), (4201, 7001, 64), (6001, 6000, 20), (4500, 6100, 20), (3200, 12000, 30), (4100, 8192, 20), (2303, 16384, 20), (2200, 12001, 70), (1201, 32001, 20),
                                          (1100, 50257, 129), (301, 131077, 64)])
def test_rounds_of_rows(ctx, dtype, rows, vocab, k):
    """Several rows for each block, one after the other, some of them without weight or entries: every row's result is the one that
    it has in any other place, and that of the oracle on a sample."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(rows)
    g = torch.Generator("cuda")
    g.manual_seed(rows)
    wide = (vocab + 15) // 8 * 8  # whole multiples of 16 bytes: a row may change its place
    logits = torch.randn(rows, wide, generator=g, device="cuda").mul_(3).to(TYPES[dtype])[:, 3:3 + vocab]
    ids = torch.randint(0, vocab, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    ids[:, k // 2] = ids[:, 0]
    teacher = torch.randn(rows, k, generator=g, device="cuda")
    weights = torch.rand(rows, generator=g, device="cuda") + 0.5
    none = torch.rand(rows, generator=g, device="cuda")
    none[rows // 2:rows // 2 + rows // 3] = 0.9  # a run of whole rounds
    weights[none > 0.7] = 0.0
    ids[(none > 0.5) & (none < 0.6)] = -1
    counts = (weights != 0) & (ids >= 0).any(1)
    up = torch.randn(rows, generator=g, device="cuda")
    loss, lse, grad = K.distill_loss(ctx, logits, ids, teacher, 1.5, weights, up)
    alone = K.distill_loss(ctx, logits, ids, teacher, 1.5, weights, want_grad=False)
    grad2 = K.distill_grad(ctx, logits, ids, teacher, alone[1], 1.5, weights, up)
    assert not loss[~counts].any() and not alone[0][~counts].any() and not grad[~counts].any() and not grad2[~counts].any()

    order = torch.randperm(rows, generator=g, device="cuda")
    other = torch.empty_strided(logits.shape, logits.stride(), dtype=logits.dtype, device="cuda")  # on 16 bytes
    moved = torch.zeros(rows, wide, dtype=logits.dtype, device="cuda")[:, 3:3 + vocab]
    moved.copy_(logits[order])
    there = K.distill_loss(ctx, moved, ids[order], teacher[order], 1.5, weights[order], up[order])
    for a, b in zip((loss, lse, grad), there):
        assert torch.equal(a[order], b)
    there = K.distill_loss(ctx, moved, ids[order], teacher[order], 1.5, weights[order], want_grad=False)
    for a, b in zip(alone[:2], there[:2]):
        assert torch.equal(a[order], b)
    assert torch.equal(grad2[order], K.distill_grad(ctx, moved, ids[order], teacher[order], alone[1][order], 1.5, weights[order], up[order], grad=other))

    at = np.unique(np.concatenate([rng.integers(0, rows, 16), [0, rows - 1]]))
    to = torch.from_numpy(at).cuda()
    w, u = weights[to].double().cpu().numpy(), up[to].double().cpu().numpy()
    want = odistill.distill(logits[to].double().cpu().numpy(), ids[to].cpu().numpy(), teacher[to].double().cpu().numpy(), 1.5, w, u)
    tol = bounds(logits[to].double().cpu().numpy(), want, dtype, 1.5, w, w * u * 1.5, k)
    for got, i in ((loss, 0), (lse, 1), (grad, 2), (alone[0], 0), (alone[1], 1), (grad2, 2)):
        compare(got[to], want[i], tol[i], ("loss", "lse", "gradient")[i])
