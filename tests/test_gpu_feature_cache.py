"""The feature cache against the 64-bit oracle: codes and scales bit for bit; values off by one rounding of code * scale to float32
and one to the rows' type, 2^-24 + eps / 2 of the value, or half the type's smallest subnormal."""
import numpy as np
import pytest
import torch

from oracle import feature_cache as ocache

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}
HELD = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def cache(ctx, pages, page, heads, dim, code, fill=0x55):
    from aeon_b200 import kernels as K
    c = K.FeatureCache.allocate(ctx, pages, page, heads, dim, code)
    c.codes.view(torch.uint8).fill_(fill)
    c.scales.fill_(-1.0)
    return c


def features(rng, shape, dtype):
    x = rng.normal(0, 1, shape) * np.exp(rng.normal(0, 2, shape[:-1] + (1,)))
    return torch.from_numpy(x.astype(np.float32)).cuda().to(TYPES[dtype])


def tables(rng, seqs, n, pages):
    return torch.from_numpy(rng.permutation(pages)[: seqs * n].reshape(seqs, n).astype(np.int32)).cuda()


def expected(c, rows, table, start, length, code, before):
    """Codes, scales after a write, and the (seq, token) pairs written with their places."""
    q, s = ocache.encode(rows.double().cpu().numpy(), code)
    codes, scales = before[0].copy(), before[1].copy()
    tb = table.cpu().numpy()
    where = []
    for i in range(rows.shape[0]):
        n = rows.shape[1] if length is None else min(max(int(length[i]), 0), rows.shape[1])
        for j in range(n):
            at = j + (0 if start is None else int(start[i]))
            if at < 0 or at // c.page_tokens >= tb.shape[1]:
                continue
            page = tb[i, at // c.page_tokens]
            if page < 0 or page >= c.pages:
                continue
            codes[page, at % c.page_tokens], scales[page, at % c.page_tokens] = q[i, j], s[i, j]
            where.append((i, j, page, at % c.page_tokens))
    return codes, scales, where


def held(c):
    return c.codes.view(torch.uint8).cpu().numpy(), c.scales.cpu().numpy()


def close(got, want, dtype):
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert np.array_equal(g[np.isinf(want)], want[np.isinf(want)])
    ok = np.isfinite(want)
    tol = np.abs(want[ok]) * (2.0 ** -24 + torch.finfo(TYPES[dtype]).eps / 2) * 1.001 + TINY[dtype] / 2
    assert (np.abs(g[ok] - want[ok]) <= tol).all()


def round_trip(ctx, c, rows, table, start, length, code, dtype):
    before = held(c)
    values = torch.full_like(rows, 3.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.write(rows, table, start, length, values, status)
    codes, scales, where = expected(c, rows, table, start, length, code, before)
    got = held(c)
    assert np.array_equal(got[1], scales, equal_nan=True)
    assert np.array_equal(got[0], codes)
    out = c.read(table, rows.shape[1], start, length, dtype=TYPES[dtype])
    want = np.zeros(tuple(rows.shape))
    kept = np.full(tuple(rows.shape), 3.0)
    for i, j, page, place in where:
        want[i, j] = kept[i, j] = ocache.decode(codes[page, place], scales[page, place], code)
    n = [rows.shape[1] if length is None else min(max(int(length[i]), 0), rows.shape[1]) for i in range(rows.shape[0])]
    placed = {(i, j) for i, j, _, _ in where}
    missing = False
    for i in range(rows.shape[0]):
        for j in range(n[i]):
            if (i, j) not in placed:
                want[i, j] = np.nan
                missing = True
    close(out, want, dtype)
    close(values, kept, dtype)
    assert bool(status.item()) == missing
    return out


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,tokens,heads,dim,page", [
    (1, 1, 1, 1, 1), (2, 3, 1, 2, 2), (3, 5, 2, 7, 4), (2, 9, 1, 13, 7), (2, 17, 3, 16, 16), (3, 33, 1, 40, 16), (1, 5, 2, 64, 3),
    (2, 4, 1, 80, 64), (2, 7, 8, 128, 4), (3, 6, 1, 161, 5), (2, 3, 5, 256, 2), (1, 4, 2, 512, 1), (2, 3, 1, 1000, 2), (1, 2, 2, 1027, 3),
    (1, 2, 1, 4100, 1), (2, 300, 1, 24, 32), (40, 11, 4, 32, 8),
])
def test_sizes_types_and_codes(ctx, code, dtype, seqs, tokens, heads, dim, page):
    rng = np.random.default_rng(seqs * 7 + tokens * 1001 + heads * 17 + dim * 131 + page)
    n = (tokens + 2 * page) // page + 1
    c = cache(ctx, seqs * n + 3, page, heads, dim, code)
    rows, table = features(rng, (seqs, tokens, heads, dim), dtype), tables(rng, seqs, n, c.pages)
    start = torch.from_numpy(rng.integers(0, 2 * page + 1, seqs).astype(np.int32)).cuda()
    length = torch.from_numpy(rng.integers(0, tokens + 1, seqs).astype(np.int32)).cuda()
    round_trip(ctx, c, rows, table, None, None, code, dtype)
    round_trip(ctx, c, rows, table, start, length, code, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quotients_next_to_the_middle(ctx, code, dtype):
    """Every group has values in the middle between two codes, one float on either side of it, and the numbers themselves."""
    rng = np.random.default_rng(41)
    numbers = np.arange(128.0) if code == "int8" else ocache.e4m3_numbers()[:127]
    middle = (numbers[1:] + numbers[:-1]) / 2
    rows = []
    for i in range(64):
        largest = np.float32(numbers[-1] * 2.0 ** rng.integers(-20, 20)) if i % 2 == 0 else np.float32(np.exp(rng.normal(0, 5)))
        if dtype == "bf16":
            largest = np.float32(torch.tensor(float(largest)).bfloat16().float())
        s = np.float64(np.float32(largest / numbers[-1]))
        near = (middle * s).astype(np.float32)
        v = np.concatenate([near, np.nextafter(near, np.float32(0)), np.nextafter(near, np.float32(np.inf)), (numbers * s).astype(np.float32)])
        v = np.minimum(v, largest) * np.where(rng.random(len(v)) < 0.5, -1, 1)
        v[-1] = largest
        rows.append(v)
    rows = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda().to(TYPES[dtype])[:, None, None, :]
    c = cache(ctx, 64, 1, 1, rows.shape[3], code)
    round_trip(ctx, c, rows, tables(rng, 64, 1, 64), None, None, code, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [5, 40, 128])
def test_infinities_nan_zeros_and_the_ends_of_the_range(ctx, code, dtype, dim):
    rng = np.random.default_rng(42)
    rows = features(rng, (14, 1, 1, dim), dtype)
    big, small = torch.finfo(TYPES[dtype]).max, TINY[dtype]
    rows[0] = 0.0
    rows[1, ..., 1] = float("-inf")       # an empty mel filter
    rows[2] = float("-inf")
    rows[3, ..., 2] = float("inf")        # the whole group reads back as NaN
    rows[4, ..., 3] = float("nan")
    rows[5, ..., 0], rows[5, ..., 1] = float("-inf"), float("nan")
    rows[6] = small                       # scale at its floor
    rows[6, ..., 0] = 0.0
    rows[7, ..., 0] = big
    rows[8] = -big
    rows[9] = rows[9] * 0 + 2.0 ** -24
    rows[10] = -0.0
    rows[11, ..., 1:] = 1e-3 * rows[11, ..., :1].abs()
    rows[12] = torch.finfo(TYPES[dtype]).smallest_normal
    c = cache(ctx, 14, 1, 1, dim, code)
    table = tables(rng, 14, 1, 14)
    out = round_trip(ctx, c, rows, table, None, None, code, dtype)
    assert out[1, 0, 0, 1] == float("-inf") and out[1, 0, 0, 2:].isfinite().all() and (out[2] == float("-inf")).all()
    assert out[3].isnan().all() and out[4].isnan().all() and out[5].isnan().all()
    assert out[7].isfinite().all() and out[8].isfinite().all() and not out[0].any()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_lengths_starts_and_pages_that_do_not_fit(ctx, code):
    """Lengths of zero, below zero and above the rows; negative positions, positions behind the table, pages that do not exist.
    (What has no place is not written and reads as NaN; the bounds are the kernel's own.)"""
    rng = np.random.default_rng(43)
    for dim, dtype in ((40, "f32"), (13, "f32"), (128, "bf16")):
        c = cache(ctx, 40, 4, 2, dim, code)
        rows, table = features(rng, (8, 9, 2, dim), dtype), tables(rng, 8, 4, 40)
        table[3, 1] = -1
        table[4, 2] = 40
        table[5, 0] = 2 ** 31 - 1
        table[6, 0] = -2 ** 31
        start = torch.tensor([0, 3, 0, 2, 0, 0, 1, 12], dtype=torch.int32, device="cuda")
        length = torch.tensor([0, 1, -5, 9, 100, 3, 9, 9], dtype=torch.int32, device="cuda")
        round_trip(ctx, c, rows, table, start, length, code, dtype)
        start = torch.tensor([-1, -9, 2 ** 31 - 1, -2 ** 31, 15, 16, 7, 8], dtype=torch.int32, device="cuda")
        round_trip(ctx, c, rows, table, start, None, code, dtype)
        none = torch.zeros(8, 0, dtype=torch.int32, device="cuda")
        round_trip(ctx, c, rows, none, None, None, code, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_orders_and_alignment(ctx, code, dtype):
    rng = np.random.default_rng(44)
    seqs, tokens, heads, dim, page = 3, 10, 4, 40, 4
    base = features(rng, (seqs, tokens, heads, dim), dtype)
    table = tables(rng, seqs, 3, 12)
    c = cache(ctx, 12, page, heads, dim, code)
    c.write(base, table)
    want = held(c)
    read = c.read(table, tokens, dtype=TYPES[dtype])
    shapes = []
    a = torch.empty(heads, seqs, tokens, dim, dtype=TYPES[dtype], device="cuda").permute(1, 2, 0, 3)     # heads outermost
    b = torch.empty(tokens, heads, seqs, dim, dtype=TYPES[dtype], device="cuda").permute(2, 0, 1, 3)     # tokens outermost
    d = torch.empty(seqs, tokens, heads, dim + 3, dtype=TYPES[dtype], device="cuda")[..., 3:]            # rows off every alignment
    e = torch.empty(seqs, tokens, heads, 2 * dim, dtype=TYPES[dtype], device="cuda")[..., dim:]
    f = torch.empty(seqs * tokens * heads * dim + 1, dtype=TYPES[dtype], device="cuda")[1:].view(seqs, tokens, heads, dim)
    shapes += [a, b, d, e, f]
    for x in shapes:
        c2 = cache(ctx, 12, page, heads, dim, code)
        x.copy_(base)
        c2.write(x, table, values=x)  # in place: the values replace the rows
        got = held(c2)
        used = want[1] >= 0
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0][used], want[0][used])
        assert torch.equal(x, read)
        x.fill_(9.0)
        c2.read(table, tokens, out=x)
        assert torch.equal(x, read)
    wide = torch.zeros(seqs, 5, dtype=torch.int32, device="cuda")
    wide[:, 1:4] = table
    assert torch.equal(c.read(wide[:, 1:4], tokens, dtype=TYPES[dtype]), read)
    # one row for all sequences, as a broadcast input
    c2 = cache(ctx, 12, page, heads, dim, code)
    c2.write(base[:1].expand(seqs, -1, -1, -1), table)
    assert torch.equal(c2.read(table, tokens, dtype=TYPES[dtype]), read[:1].expand(seqs, -1, -1, -1))
    if heads == 4:  # three dimensions for one head
        c3 = cache(ctx, 12, page, 1, dim, code)
        c3.write(base[:, :, 0], table)
        assert torch.equal(c3.read(table, tokens, dtype=TYPES[dtype])[:, :, 0], read[:, :, 0])


def test_frames_one_at_a_time_equal_the_whole(ctx):
    rng = np.random.default_rng(45)
    for heads, dim, dtype, code in ((1, 40, "f32", "int8"), (8, 64, "bf16", "e4m3")):
        rows, table = features(rng, (5, 23, heads, dim), dtype), tables(rng, 5, 4, 20)
        whole, one = cache(ctx, 20, 7, heads, dim, code), cache(ctx, 20, 7, heads, dim, code)
        whole.write(rows, table)
        for j in range(23):
            one.write(rows[:, j:j + 1], table, start=torch.full((5,), j, dtype=torch.int32, device="cuda"))
        assert np.array_equal(held(whole)[0], held(one)[0]) and np.array_equal(held(whole)[1], held(one)[1])
        all_rows = whole.read(table, 23)
        for j in (0, 6, 7, 22):
            got = one.read(table, 1, start=torch.full((5,), j, dtype=torch.int32, device="cuda"))
            assert torch.equal(got[:, 0], all_rows[:, j])


def test_read_into_every_type(ctx):
    rng = np.random.default_rng(46)
    for code in HELD:
        c = cache(ctx, 256, 1, 1, 256, code)
        q = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
        c.codes.view(torch.uint8).copy_(torch.from_numpy(q).cuda()[:, None, None, :])
        s = np.exp(rng.normal(0, 4, 256)).astype(np.float32)
        s[0], s[1], s[2] = 0.0, 2.0 ** -126, np.nan
        c.scales.copy_(torch.from_numpy(s).cuda()[:, None, None])
        table = torch.arange(256, dtype=torch.int32, device="cuda")[:, None]
        want = ocache.decode(q, s, code)
        for dtype in ("f32", "bf16"):
            close(c.read(table, 1, dtype=TYPES[dtype])[:, 0, 0], want, dtype)
        got = c.read(table, 1, dtype=torch.float16)[:, 0, 0].double().cpu().numpy()
        with np.errstate(over="ignore", invalid="ignore"):
            half = want.astype(np.float32).astype(np.float16).astype(np.float64)  # both roundings, large values to infinity
        assert np.array_equal(got, half, equal_nan=True)


def test_other_streams_graphs_and_refusals(ctx):
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(47)
    rows, table = features(rng, (64, 200, 1, 40), "f32"), tables(rng, 64, 4, 256)
    c = cache(ctx, 256, 64, 1, 40, "int8")
    c.write(rows, table)
    want = c.read(table, 200)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        late = rows.clone()
        c2 = K.FeatureCache.allocate(ctx, 256, 64, 1, 40)
        c2.write(late, table)
        late.fill_(0)
        got = c2.read(table, 200)
        assert torch.equal(got, want)
    # a graph follows what its table, start, length and rows hold at each replay
    start, length = torch.zeros(64, dtype=torch.int32, device="cuda"), torch.full((64,), 200, dtype=torch.int32, device="cuda")
    c3 = K.FeatureCache.allocate(ctx, 256, 64, 1, 40)
    c3.write(rows, table, start, length)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    held_rows, values = rows.clone(), torch.zeros_like(rows)
    with torch.cuda.graph(g):
        c3.write(held_rows, table, start, length, values)
        out = c3.read(table, 200, start, length)
    for turn in range(2):
        held_rows.copy_(features(rng, (64, 200, 1, 40), "f32"))
        start.copy_(torch.from_numpy(rng.integers(0, 56, 64).astype(np.int32)))
        length.copy_(torch.from_numpy(rng.integers(0, 201, 64).astype(np.int32)))
        table.copy_(tables(rng, 64, 4, 256))
        values.zero_()
        g.replay()
        torch.cuda.synchronize()
        c2.write(held_rows, table, start, length)
        assert torch.equal(out, c2.read(table, 200, start, length)) and torch.equal(out, values)
    for bad in (lambda: c.write(rows.cpu(), table), lambda: c.write(rows.double(), table), lambda: c.write(rows, table.long()),
                lambda: c.write(rows[:3], table), lambda: c.write(rows[..., :39], table), lambda: c.write(rows, table, start=start[:3]),
                lambda: c.write(rows, table, length=length.long()), lambda: c.write(rows, table, values=rows[:, :3]),
                lambda: c.write(rows, table, values=rows.half()), lambda: c.write(rows.transpose(1, 3), table),
                lambda: c.read(table, 200, dtype=torch.float64), lambda: c.read(table, 200, out=rows[:3]),
                lambda: c.read(table.t(), 200), lambda: c.read(table, 200, status=torch.zeros(1, device="cuda")),
                lambda: K.FeatureCache(ctx, c.codes.view(torch.uint8), c.scales), lambda: K.FeatureCache(ctx, c.codes, c.scales[:1]),
                lambda: K.FeatureCache(ctx, c.codes[:, ::2], c.scales[:, ::2]), lambda: K.FeatureCache.allocate(ctx, 1, 1, 1, 1, "int4")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        c.read(table, 200, out=torch.zeros(64, 1, 1, 40, device="cuda").expand(-1, 200, -1, -1))
    assert c.read(table[:0], 200).shape == (0, 200, 1, 40) and c.read(table, 0).shape == (64, 0, 1, 40)


def test_pages_past_32_bits(ctx):
    """Codes, rows and values whose offsets pass 2^32."""
    rng = np.random.default_rng(48)
    from aeon_b200 import kernels as K
    pages, page, dim = 66000, 64, 1024  # 4.3 GB of codes
    dev = torch.device("cuda")
    for code, dtype in (("int8", "f32"), ("e4m3", "bf16")):
        c = K.FeatureCache(ctx, torch.empty(pages, page, 1, dim, dtype=torch.int8, device=dev).view(HELD[code]),
                           torch.empty(pages, page, 1, device=dev))
        table = torch.tensor([[0, 65999], [65998, 1]], dtype=torch.int32, device=dev)
        rows = features(rng, (2, 100, 1, dim), dtype)
        c.write(rows, table)
        q, s = ocache.encode(rows.double().cpu().numpy(), code)
        far = 2 ** 31 + 16
        out = torch.empty(far + 100 * dim, dtype=TYPES[dtype], device=dev).as_strided((2, 100, 1, dim), (far, dim, dim, 1))
        c.read(table, 100, out=out)
        close(out, ocache.decode(q, s, code), dtype)
        del out, c


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_million_quotients(ctx, code, dtype):
    """Codes of many groups of many sizes, in vectors and value by value: bit for bit those of the exact quotient."""
    rng = np.random.default_rng(50)
    for dim in (512, 77):
        rows = features(rng, (2000, 1, 1, dim), dtype)
        rows[::5] = (rows[::5] * 64 / rows[::5].abs().amax(-1, keepdim=True)).round()  # small whole numbers: many middles
        c = cache(ctx, 2000, 1, 1, dim, code)
        c.write(rows, torch.arange(2000, dtype=torch.int32, device="cuda")[:, None])
        q, s = ocache.encode(rows.double().cpu().numpy(), code)
        got = held(c)
        assert np.array_equal(got[1][:, 0, 0], s[:, 0, 0])
        assert np.array_equal(got[0][:, 0, 0], q[:, 0, 0])


def test_more_sequences_than_a_grid_is_high(ctx):
    rng = np.random.default_rng(51)
    seqs = 70001
    for dim, dtype in ((4, "f32"), (16, "bf16")):
        rows = features(rng, (seqs, 1, 1, dim), dtype)
        c = cache(ctx, seqs, 1, 1, dim, "int8")
        table = torch.randperm(seqs, device="cuda").to(torch.int32)[:, None]
        values = torch.empty_like(rows)
        c.write(rows, table, values=values)
        assert torch.equal(c.read(table, 1, dtype=TYPES[dtype]), values)
        q, s = ocache.encode(rows.double().cpu().numpy(), "int8")
        assert np.array_equal(held(c)[1][table[:, 0].cpu().numpy(), 0, 0], s[:, 0, 0])


def test_positions_past_31_bits(ctx):
    """Pages so long that a token's position passes 2^31."""
    from aeon_b200 import kernels as K
    rng = np.random.default_rng(52)
    page = 2 ** 30
    c = K.FeatureCache(ctx, torch.empty(3, page, 1, 1, dtype=torch.int8, device="cuda"), torch.empty(3, page, 1, device="cuda"))
    table = torch.tensor([[1, 0, 2]], dtype=torch.int32, device="cuda")
    rows = features(rng, (1, 6, 1, 1), "f32")
    start = torch.tensor([2 ** 31 - 3], dtype=torch.int32, device="cuda")
    values = torch.empty_like(rows)
    c.write(rows, table, start=start, values=values)
    assert torch.equal(c.read(table, 6, start=start), values)
    q, s = ocache.encode(rows.double().cpu().numpy(), "int8")
    assert np.array_equal(c.scales[0, page - 3:, 0].cpu().numpy(), s[0, :3, 0]) and np.array_equal(c.scales[2, :3, 0].cpu().numpy(), s[0, 3:, 0])


def test_random_cases_round_trip(ctx):
    rng = np.random.default_rng(49)
    for _ in range(30):
        code, dtype = ("int8", "e4m3")[rng.integers(2)], ("f32", "f16", "bf16")[rng.integers(3)]
        seqs, tokens, heads = (int(rng.integers(1, 6)) for _ in range(3))
        dim, page = int(np.exp(rng.uniform(0, 6.5))), int(rng.integers(1, 9))
        n = (tokens + 5) // page + 1
        c = cache(ctx, seqs * n, page, heads, dim, code)
        rows, table = features(rng, (seqs, tokens, heads, dim), dtype), tables(rng, seqs, n, c.pages)
        start = torch.from_numpy(rng.integers(0, 5, seqs).astype(np.int32)).cuda()
        round_trip(ctx, c, rows, table, start, None, code, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("chunks", [4, 5, 8, 16, 24, 32])
@pytest.mark.parametrize("shift", [0, 16])
def test_large_calls_equal_small_ones(ctx, code, dtype, chunks, shift):
    """Calls of so many groups that a lane takes four chunks of each, on 32 and on 16 bytes: the same bits as in small calls, and the
    oracle's where groups hold infinities, NaN, nothing but zeros or the smallest numbers."""
    rng = np.random.default_rng(chunks * 2 + shift)
    t = TYPES[dtype]
    size = torch.finfo(t).bits // 8
    dim = chunks * (32 - shift) // size
    seqs, heads, page = 37, 2, 24
    tokens = 148 * 1024 * 4 // (chunks * seqs * heads) + 9  # lanes in all: above a thousand for each of 148 SMs

    def room():
        all_of = torch.full((seqs * tokens * heads * dim + shift,), 7.0, dtype=t, device="cuda")
        return all_of[shift // size:][:seqs * tokens * heads * dim].view(seqs, tokens, heads, dim)

    rows = room()
    torch.manual_seed(chunks)
    rows.copy_(torch.randn(rows.shape, device="cuda") * torch.exp2(torch.randint(-12, 12, rows.shape[:3] + (1,), device="cuda").float()))
    special = rows[5]  # one sequence's groups
    kinds = torch.arange(tokens, device="cuda") % 9
    special[kinds == 0, :, 1] = float("-inf")
    special[kinds == 1] = 0.0
    special[kinds == 2, 0, dim - 1] = float("nan")
    special[kinds == 3, 1, dim // 2] = float("inf")
    special[kinds == 4] = TINY[dtype]
    special[kinds == 5, 0] = torch.finfo(t).max
    special[kinds == 6, 1] = float("-inf")
    special[kinds == 7] *= torch.finfo(t).smallest_normal
    n = (tokens + 30) // page + 1
    big, small = cache(ctx, seqs * n, page, heads, dim, code), cache(ctx, seqs * n, page, heads, dim, code)
    table = tables(rng, seqs, n, big.pages)
    start = torch.from_numpy(rng.integers(0, 30, seqs).astype(np.int32)).cuda()
    lengths = rng.integers(0, tokens + 1, seqs).astype(np.int32)
    lengths[:7] = [0, 1, tokens, tokens, tokens, tokens, 2]
    length = torch.from_numpy(lengths).cuda()
    bits = {4: torch.int32, 2: torch.int16}[size]
    values, apart = room(), room()
    big.write(rows, table, start, length, values)
    for s in range(seqs):
        one = slice(s, s + 1)
        small.write(rows[one], table[one], start[one], length[one], apart[one])
    assert torch.equal(big.codes.view(torch.uint8), small.codes.view(torch.uint8))
    assert torch.equal(big.scales.view(torch.int32), small.scales.view(torch.int32))
    assert torch.equal(values.isnan(), apart.isnan())
    assert torch.equal(values.nan_to_num(0.5).view(bits), apart.nan_to_num(0.5).view(bits))
    out = big.read(table, tokens, start, length, out=room())
    pieces = torch.cat([small.read(table[s:s + 1], tokens, start[s:s + 1], length[s:s + 1], dtype=t) for s in range(seqs)])
    assert torch.equal(out.isnan(), pieces.isnan())
    assert torch.equal(out.nan_to_num(0.5).view(bits), pieces.nan_to_num(0.5).view(bits))
    q, s = ocache.encode(special.double().cpu().numpy(), code)
    close(out[5], ocache.decode(q, s, code), dtype)
    close(values[5], ocache.decode(q, s, code), dtype)
    big.write(rows, table, start, length, rows)  # in place
    assert torch.equal(rows[5].isnan(), out[5].isnan()) and torch.equal(rows[5].nan_to_num(0.5), out[5].nan_to_num(0.5))
