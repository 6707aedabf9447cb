"""The feature cache and the distillation loss at the ends of what they take: reads under way when their loader closes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_read_under_way_when_the_passes_close(ctx):
    """The consumer's stream is busy when the loader goes: its last read still finds the pages, which the allocator then gives away."""
    from aeon_b200 import _lib as L
    from aeon_b200.dataloader import _CachedPasses
    shape, size = (640, 64), 256
    g = torch.Generator("cuda")
    g.manual_seed(5)
    x = torch.randn((size,) + shape, generator=g, device="cuda")
    torch.cuda.synchronize()
    passes = _CachedPasses(0, "int8", [("audio", shape, L.F32)], size, 1)
    passes.add((("audio", x),))
    assert passes.restart()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(40):
            big = big @ big * 1e-3
        (_, got), = passes.next()
    codes = passes.caches["audio"].codes.numel()
    passes.close()
    del passes
    taken = [torch.full((codes,), 77, dtype=torch.uint8, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(got, x)  # add() has put the kept values into x
    del taken


U = 2.0 ** -24


@pytest.mark.parametrize("dtype,vocab,kind", [
    (torch.bfloat16, 2 ** 24 + 3, "alike"), (torch.bfloat16, 2 ** 26, "alike"), (torch.float32, 2 ** 25 + 1, "alike"), (torch.float16, 2 ** 25, "alike"),
    (torch.float32, 2 ** 24 + 1, "rising"), (torch.bfloat16, 2 ** 24, "rising"), (torch.float32, 600001, "holes"), (torch.float16, 2 ** 24 + 5, "holes"),
])
def test_sums_over_millions_of_values(ctx, dtype, vocab, kind):
    """The log-sum-exp of rows that no cluster holds does not lose more with every value.  Its error, with u = 2^-24 and R the range of
    the exponents: an exponential (3 R + 4) u, the additions of sixteen of them 16 u (those in 64 bits nothing), four more roundings,
    and four of the lse itself; a sum that is rescaled (when the largest value has grown by 2^4; after six times nothing is left of
    what 2^24 terms made) takes an exponential's error each time, (3 5 + 4) u.  The gradient takes the lse's error and an exponential's."""
    from aeon_b200 import kernels as K
    g = torch.Generator("cuda")
    g.manual_seed(vocab)
    if kind == "alike":
        x = torch.full((1, vocab), -0.6, device="cuda")
        x[0, 7] = 0.0
    elif kind == "rising":
        x = torch.linspace(-9.0, 9.0, vocab, device="cuda")[None]
    else:
        x = torch.randn(1, vocab, generator=g, device="cuda") * 2
        x[0, ::3] = float("-inf")
        x[0, :5000] = float("-inf")
    x = x.to(dtype)
    ids = torch.tensor([[7, vocab - 1, vocab // 2]], dtype=torch.int32, device="cuda")
    teacher = torch.tensor([[1.0, 0.5, -1.0]], device="cuda")
    x[0, ids[0].long()] = torch.tensor([0.0, 0.25, 0.5], dtype=dtype, device="cuda")
    loss, lse, grad = K.distill_loss(ctx, x, ids, teacher)
    loss2, lse2, _ = K.distill_loss(ctx, x, ids, teacher, want_grad=False)
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2)
    y = x[0].double()
    want = torch.logsumexp(y, 0)
    p = torch.softmax(teacher[0].double(), 0)
    finite = y[y > -float("inf")]
    reach = (finite.max() - finite.min()).item()
    e = (3 * reach + 4) * U
    lse_tol = e + (16 + 4 + (0 if kind == "alike" else 7 * 19) + 4 * abs(want.item())) * U
    assert abs(lse.item() - want.item()) <= lse_tol
    want_loss = (p * (p.log() - y[ids[0].long()] + want)).sum().item()
    assert abs(loss.item() - want_loss) <= lse_tol + 4 * U * (reach + 40)
    q = torch.exp(y - want)
    tol = q * ((lse_tol + e + 4 * U) * 1.1 + torch.finfo(dtype).eps / 2 * 1.01) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 + 2.0 ** -126
    q.scatter_add_(0, ids[0].long(), -p)
    tol.scatter_add_(0, ids[0].long(), p * (e + 11 * U + torch.finfo(dtype).eps / 2))
    assert ((grad[0].double() - q).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("vocab,pad", [(151936, 0), (262144, 0), (262151, 1)])
@pytest.mark.parametrize("k", [33, 100, 256])
def test_repeated_ids_in_long_parts(ctx, dtype, vocab, pad, k):
    """Rows whose blocks look for repeated ids in half of their part at a time: repeats in either half only, at the ends of both, in
    all blocks, and none."""
    from tests.test_gpu_distill import check, make
    rng = np.random.default_rng(vocab + k)
    logits, ids, teacher = make(rng, 6, vocab, k, dtype, pad)
    distinct = np.stack([rng.choice(vocab, k, replace=False) for _ in range(6)]).astype(np.int32)
    distinct[1, 1] = distinct[1, 0] = 16391
    distinct[2, -1] = distinct[2, 3] = 16392
    part = (vocab // 8 // 8 + 7) // 8 * 8 * 8  # values of a block, but for those in front of the first whole vector
    for j in range(8):
        distinct[3, 4 * j:4 * j + 4] = [part * j + 16390, part * j + 16392, part * j + 16390, part * j + 16392]
    distinct[3] = np.minimum(distinct[3], vocab - 1)
    distinct[4, :32] = np.repeat(np.arange(8) * part, 4)
    ids.copy_(torch.from_numpy(distinct))
    check(ctx, logits, ids, teacher, 1.5, dtype=dtype)


def test_the_profile_of_a_context_whose_calls_are_captured(ctx):
    """A captured call has no time of its own: it is left out, and the launches beside it are read as ever."""
    from aeon_b200 import kernels as K
    g = torch.Generator("cuda")
    g.manual_seed(6)
    logits = torch.randn(8, 1000, generator=g, device="cuda")
    ids = torch.randint(0, 1000, (8, 3), generator=g, device="cuda", dtype=torch.int32)
    teacher = torch.randn(8, 3, generator=g, device="cuda")
    rows, table = torch.randn(4, 9, 1, 40, generator=g, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")[:, None]
    cache = K.FeatureCache.allocate(ctx, 4, 16, 1, 40)
    torch.cuda.synchronize()
    ctx.profile(True)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = K.distill_loss(ctx, logits, ids, teacher)
            cache.write(rows, table)
            read = cache.read(table, 9)
        graph.replay()
        torch.cuda.synchronize()
        assert ctx.profile_read()["other"]["launches"] == 0
        want = K.distill_loss(ctx, logits, ids, teacher)
        again = cache.read(table, 9)
        got = ctx.profile_read()["other"]
        assert got["launches"] == 2 and got["ms"] > 0
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(read, again)
    finally:
        ctx.profile(False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,row,at", [(29, 5001, 3), (300, 9000, 8), (5000, 65537, 1)])
def test_columns_of_far_longer_rows(ctx, dtype, vocab, row, at):
    """A student whose answers are some columns of a wide tensor: the gradient's rows lie closer, and hold the same."""
    from aeon_b200 import kernels as K
    from tests.test_gpu_distill import check, make
    rng = np.random.default_rng(vocab)
    wide, ids, teacher = make(rng, 12, row, 5, dtype)
    logits, ids = wide[:, at:at + vocab], ids % vocab
    before = wide.clone()
    loss, lse, grad = check(ctx, logits, ids, teacher, 2.0, dtype=dtype)
    assert grad.stride(0) < vocab + 8 and torch.equal(wide, before)
    cube = K.distill_loss(ctx, logits.unflatten(0, (3, 4)), ids.view(3, 4, 5), teacher.view(3, 4, 5), 2.0)
    assert torch.equal(cube[2].reshape(12, vocab), grad) and torch.equal(cube[0].view(-1), loss) and torch.equal(cube[1].view(-1), lse)
    given = K.distill_loss(ctx, logits, ids, teacher, 2.0, grad=logits)[2]
    assert given is logits and torch.equal(logits, grad)
    wide[:, at:at + vocab] = before[:, at:at + vocab]
    assert torch.equal(wide, before)  # nothing but the columns


@pytest.mark.parametrize("batch_major", [True, False])
def test_teacher_entries_behind_a_short_batch(ctx, batch_major):
    """Two records where five may be: no entries behind them in buffers made by the call, which the loss counts as nothing; a caller's own
    keep what they held, but for the layout whose rows are the batch."""
    from aeon_b200 import kernels as K
    from aeon_b200.provider import Provider, top_logits_record
    P, k, n = 3, 2, 5
    prov = Provider(ctx, {"batch_size": n, "batch_major": batch_major, "etl": [{"type": "top_logits", "max_positions": P, "k": k, "name": "big"}]})
    ids, logits = np.array([[[1, 2], [3, 0], [4, 5]], [[6, 7], [8, 9], [0, 1]]]), np.arange(12.0).reshape(2, P, k)
    records = [(top_logits_record(i, t),) for i, t in zip(ids, logits)]

    def rows(out, name, shape):
        a = out["big.teacher_" + name]
        a = a.cpu().numpy() if torch.is_tensor(a) else a
        return a if batch_major else a.T.reshape((n,) + shape)

    for out in (prov.run_host(records), prov.run_device(records)):
        assert np.array_equal(rows(out, "ids", (P, k))[:2], ids) and (rows(out, "ids", (P, k))[2:] == -1).all()
        assert np.array_equal(rows(out, "logits", (P, k))[:2], logits) and not rows(out, "logits", (P, k))[2:].any()
        assert rows(out, "count", (1,)).ravel().tolist() == [3, 3, 0, 0, 0]
    if batch_major:
        student = torch.randn(n, P, 10, device="cuda")
        loss, _, grad = K.distill_loss(ctx, student, out["big.teacher_ids"], out["big.teacher_logits"])
        assert loss[:2].all() and not loss[2:].any() and not grad[2:].any()
    for make in (lambda s, t: np.full(s, 77, t), lambda s, t: torch.full(s, 77, dtype={np.int32: torch.int32, np.float32: torch.float32}[t], device="cuda")):
        own = {name: make(prov._shape(dims), np.float32 if name.endswith("logits") else np.int32) for name, dims, _, _ in prov.outputs}
        torch.cuda.synchronize()
        (prov.run_device if torch.is_tensor(own["big.teacher_ids"]) else prov.run_host)(records, own)
        assert np.array_equal(rows(own, "ids", (P, k))[:2], ids)
        assert (rows(own, "ids", (P, k))[2:] == (77 if batch_major else -1)).all()
        assert (rows(own, "count", (1,))[2:] == (77 if batch_major else 0)).all()
