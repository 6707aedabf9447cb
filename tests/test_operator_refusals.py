"""What the feature cache and the distillation loss refuse, on a machine without a GPU: every refusal comes before the context
or any device memory is touched, so a block of zeros stands in for the context and numbers for the device pointers."""
import ctypes as C

import numpy as np
import pytest

from aeon_b200 import _lib as L
from oracle import distill as odistill
from oracle import feature_cache as ocache


def fake_context():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def cache_desc(**changes):
    d = L.CacheDesc()
    d.codes, d.scales, d.pages, d.page_tokens, d.heads, d.dim, d.code = 4096, 8192, 4, 16, 2, 8, L.CODE_INT8
    d.table, d.table_stride, d.table_pages, d.seqs, d.tokens, d.dtype = 16384, 2, 2, 2, 5, L.F32
    d.rows, d.row_stride_seq, d.row_stride_token, d.row_stride_head = 65536, 80, 16, 8
    d.values, d.value_stride_seq, d.value_stride_token, d.value_stride_head = 131072, 80, 16, 8
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def distill_desc(**changes):
    d = L.DistillDesc()
    d.logits, d.logits_stride, d.rows, d.vocab, d.dtype = 65536, 32, 4, 32, L.BF16
    d.ids, d.teacher, d.entry_stride, d.k, d.temperature = 4096, 8192, 5, 5, 2.0
    d.loss, d.lse, d.grad, d.grad_stride, d.grad_scale = 16384, 20480, 131072, 32, 1.0
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def test_descriptor_sizes():
    # natural alignment on x86-64: computed by hand from the header
    assert C.sizeof(L.CacheDesc) == 168
    assert C.sizeof(L.DistillDesc) == 128


BAD_CACHE = [
    (dict(dtype=L.F64), "type of the rows"), (dict(dtype=99), "type of the rows"), (dict(code=2), "code of a cache"),
    (dict(page_tokens=0), "page_tokens"), (dict(heads=0), "heads"), (dict(dim=-1), "dim"), (dict(pages=-1), "cache needs"),
    (dict(seqs=-1), "negative"), (dict(tokens=-2), "negative"), (dict(table_pages=-1), "negative"),
    (dict(pages=1 << 60, page_tokens=1 << 20), "64-bit"),
    (dict(rows=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(table=None), "NULL"),
    (dict(rows=65538), "aligned"), (dict(scales=8193), "aligned"), (dict(table=16386), "aligned"), (dict(start=2), "aligned"),
    (dict(length=6), "aligned"), (dict(status=1), "aligned"),
]


@pytest.mark.parametrize("changes,words", BAD_CACHE)
@pytest.mark.parametrize("name", ["aeonb_cache_write", "aeonb_cache_read"])
def test_cache_refusals(name, changes, words):
    lib = L.load()
    assert getattr(lib, name)(fake_context(), C.byref(cache_desc(**changes))) == L.ERR_INVALID
    assert words in lib.aeonb_last_error().decode()


@pytest.mark.parametrize("name,changes", [
    ("aeonb_cache_read", dict(row_stride_token=15)), ("aeonb_cache_read", dict(row_stride_seq=0)),
    ("aeonb_cache_read", dict(row_stride_seq=79)), ("aeonb_cache_read", dict(row_stride_head=7)),
    ("aeonb_cache_write", dict(value_stride_head=0)), ("aeonb_cache_write", dict(value_stride_seq=79)),
    ("aeonb_cache_write", dict(values=65536, value_stride_seq=160)), ("aeonb_cache_write", dict(values=131074)),
    ("aeonb_cache_write", dict(row_stride_token=-16)),
])
def test_cache_destinations_that_overlap(name, changes):
    assert getattr(L.load(), name)(fake_context(), C.byref(cache_desc(**changes))) == L.ERR_INVALID


def test_cache_null_and_empty():
    lib = L.load()
    for f in (lib.aeonb_cache_write, lib.aeonb_cache_read):
        assert f(None, C.byref(cache_desc())) == L.ERR_INVALID
        assert f(fake_context(), None) == L.ERR_INVALID
        for empty in (dict(seqs=0), dict(tokens=0), dict(seqs=0, rows=None, codes=None, table=None)):
            assert f(fake_context(), C.byref(cache_desc(**empty))) == L.OK


BAD_DISTILL = [
    (dict(dtype=L.U8), "type of the rows"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(vocab=0), "rows"), (dict(vocab=(1 << 30) + 1), "rows"),
    (dict(k=0), "entries"), (dict(k=257), "entries"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-13), "temperature"), (dict(temperature=2e12), "temperature"),
    (dict(logits=None), "NULL"), (dict(ids=None), "NULL"), (dict(teacher=None), "NULL"),
    (dict(logits=65537), "aligned"), (dict(grad=131073), "aligned"), (dict(ids=4098), "aligned"), (dict(teacher=8194), "aligned"),
    (dict(weights=2), "aligned"), (dict(upstream=1), "aligned"), (dict(loss=16386), "aligned"), (dict(lse=20482), "aligned"),
    (dict(logits_stride=-1), "stride"), (dict(entry_stride=-5), "stride"), (dict(grad_stride=31), "overlap"),
    (dict(grad=65536, grad_stride=64), "in place"),
]


@pytest.mark.parametrize("changes,words", BAD_DISTILL)
@pytest.mark.parametrize("name", ["aeonb_distill_loss", "aeonb_distill_grad"])
def test_distill_refusals(name, changes, words):
    lib = L.load()
    assert getattr(lib, name)(fake_context(), C.byref(distill_desc(**changes))) == L.ERR_INVALID
    assert words in lib.aeonb_last_error().decode()


def test_distill_nothing_to_do():
    lib = L.load()
    assert lib.aeonb_distill_loss(fake_context(), C.byref(distill_desc(loss=None, lse=None, grad=None))) == L.ERR_INVALID
    assert lib.aeonb_distill_grad(fake_context(), C.byref(distill_desc(lse=None))) == L.ERR_INVALID
    assert lib.aeonb_distill_grad(fake_context(), C.byref(distill_desc(grad=None))) == L.ERR_INVALID
    for f in (lib.aeonb_distill_loss, lib.aeonb_distill_grad):
        assert f(None, C.byref(distill_desc())) == L.ERR_INVALID
        assert f(fake_context(), None) == L.ERR_INVALID
        assert f(fake_context(), C.byref(distill_desc(rows=0))) == L.OK


def test_oracle_gradient_against_differences():
    """The oracle's gradient against central differences of its loss, in 64 bits: the error is h^2 / 6 times a third derivative
    (below T^2 / T^3 here) plus the loss's own 2^-52 over h."""
    rng = np.random.default_rng(5)
    rows, vocab, k, t, h = 3, 17, 4, 1.7, 1e-4
    s = rng.normal(0, 2, (rows, vocab))
    ids = rng.integers(0, vocab, (rows, k))  # ids that occur twice among them
    ids[1, 2] = ids[1, 0]
    ids[2] = [-1, 5, -1, 3]
    teacher = rng.normal(0, 3, (rows, k))
    w, up = np.array([0.5, 1.0, 2.0]), np.array([1.0, -2.0, 3.0])
    _, _, grad = odistill.distill(s, ids, teacher, t, w, up, 0.25)
    for v in range(vocab):
        a, b = s.copy(), s.copy()
        a[:, v] += h
        b[:, v] -= h
        diff = (odistill.distill(a, ids, teacher, t, w)[0] - odistill.distill(b, ids, teacher, t, w)[0]) / (2 * h) * up * 0.25
        assert np.abs(diff - grad[:, v]).max() < 1e-7


def test_oracle_codes_are_the_nearest():
    """Each code of the oracle is the nearest number, and torch's own conversion agrees where float32 holds the quotient."""
    import torch
    rng = np.random.default_rng(6)
    x = np.concatenate([rng.normal(0, 1, 4000) * np.exp(rng.normal(0, 3, 4000)), [0.0, -0.0, 448.0, 2.0 ** -9, 2.0 ** -10]])
    x[x > 448] = 448
    x[x < -448] = -448
    x = x.astype(np.float32)[None]
    q, s = ocache.encode(x, "e4m3")
    assert s[0] == 1.0
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(q, want)
    y = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5, -127.0, -np.inf]])
    q, s = ocache.encode(y, "int8")
    assert s[0] == 1.0
    assert q.view(np.int8).tolist() == [[127, 0, 2, 2, 0, -2, 126, -126, -127, -128]]
    assert ocache.decode(q, s, "int8").tolist() == [[127.0, 0.0, 2.0, 2.0, 0.0, -2.0, 126.0, -126.0, -127.0, -np.inf]]


def loader_config(**changes):
    cfg = {"manifest_filename": "m.tsv", "batch_size": 4, "device_output": True, "feature_cache": "int8",
           "etl": [{"type": "audio", "max_samples": 3200}, {"type": "label"}, {"type": "top_logits", "max_positions": 4, "k": 2}]}
    cfg.update(changes)
    return cfg


def test_feature_cache_configurations():
    from aeon_b200 import DataLoader
    from aeon_b200.dataloader import check_feature_cache
    assert check_feature_cache(loader_config()) == "int8"
    assert check_feature_cache(loader_config(feature_cache="e4m3", iteration_mode="ONCE")) == "e4m3"
    assert check_feature_cache({"etl": [{"type": "image"}], "shuffle_enable": True}) is None
    for changes, words in [
            (dict(feature_cache="int4"), "int8"), (dict(feature_cache=True), "int8"), (dict(device_output=False), "device_output"),
            (dict(batch_major=False), "batch_major"), (dict(iteration_mode="INFINITE"), "ONCE"),
            (dict(iteration_mode="COUNT", iteration_mode_count=3), "ONCE"), (dict(shuffle_enable=True), "shuffle"),
            (dict(etl=[{"type": "label"}]), "audio"), (dict(etl=[{"type": "audio"}, {"type": "image"}]), "image"), (dict(etl=[]), "audio")]:
        with pytest.raises(ValueError, match=words):
            DataLoader(loader_config(**changes))


def test_top_logits_record_bytes():
    from aeon_b200.provider import top_logits_record
    got = top_logits_record([[3, -1], [7, 2], [0, 1]], [[0.5, 0], [2, 1], [-1, -2]])
    assert np.frombuffer(got[:8], "<i4").tolist() == [3, 2]
    assert np.frombuffer(got[8:32], "<i4").tolist() == [3, -1, 7, 2, 0, 1]
    assert np.frombuffer(got[32:], "<f4").tolist() == [0.5, 0, 2, 1, -1, -2]
    assert top_logits_record(np.zeros((0, 3)), np.zeros((0, 3))) == np.array([0, 3], "<i4").tobytes()
    for ids, logits in (([1, 2], [1, 2]), ([[1, 2]], [[1, 2, 3]]), (np.zeros((2, 0)), np.zeros((2, 0)))):
        with pytest.raises(ValueError):
            top_logits_record(ids, logits)
