"""Records with a clip and a teacher's top logits, from the manifest to the gradient: the top_logits element, the passes that read
features from the cache, and the loss on what they deliver."""
import numpy as np
import pytest
import torch

from oracle import distill as odistill
from oracle import feature_cache as ocache

pytestmark = pytest.mark.gpu

VOCAB, K, FRAMES = 29, 4, 30


def clips(rng, n):
    out = []
    for _ in range(n):
        t = np.arange(int(rng.integers(700, 6000))) / 16000
        x = sum(0.2 * np.sin(2 * np.pi * rng.uniform(100, 6000) * t) for _ in range(3)) + rng.normal(0, 0.05, len(t))
        out.append(np.clip(x * 16000, -32768, 32767).astype(np.int16))
    return out


def answers(rng, frames):
    ids = np.stack([rng.permutation(VOCAB)[:K] for _ in range(frames)]) if frames else np.zeros((0, K))
    return ids.astype(np.int32), -np.sort(-rng.normal(0, 3, (frames, K)).astype(np.float32), 1)


AUDIO = {"type": "audio", "frame_length": 320, "frame_stride": 160, "max_time_steps": FRAMES, "num_filters": 64, "sample_rate": 16000,
         "window_type": "hann"}
TOP = {"type": "top_logits", "max_positions": FRAMES, "k": K + 1, "vocab": VOCAB}


@pytest.fixture(scope="module")
def dataset(tmp_path_factory):
    from aeon_b200.provider import top_logits_record
    root = tmp_path_factory.mktemp("speech")
    rng = np.random.default_rng(61)
    lines, recs = ["@FILE\tFILE\tASCII_INT"], []
    for i, clip in enumerate(clips(rng, 10)):
        frames = max(0, (len(clip) - 320) // 160 + 1)
        ids, logits = answers(rng, frames)
        blob = top_logits_record(ids, logits)
        (root / ("c%d.raw" % i)).write_bytes(clip.tobytes())
        (root / ("t%d.bin" % i)).write_bytes(blob)
        lines.append("c%d.raw\tt%d.bin\t%d" % (i, i, i))
        recs.append((clip.tobytes(), blob, np.int32(i).tobytes(), ids, logits))
    (root / "m.tsv").write_text("\n".join(lines) + "\n")
    return root, recs


def padded(recs, which):
    ids, logits = np.full((len(which), FRAMES, K + 1), -1, np.int32), np.zeros((len(which), FRAMES, K + 1), np.float32)
    count = np.zeros((len(which), 1), np.int32)
    for j, r in enumerate(which):
        n = min(len(recs[r][3]), FRAMES)
        ids[j, :n, :K], logits[j, :n, :K], count[j] = recs[r][3][:n], recs[r][4][:n], n
    return ids, logits, count


@pytest.mark.parametrize("batch_major", [True, False])
def test_top_logits_through_the_provider(ctx, dataset, batch_major):
    from aeon_b200.provider import Provider
    _, recs = dataset
    prov = Provider(ctx, {"batch_size": 5, "batch_major": batch_major, "etl": [AUDIO, dict(TOP, name="big"), {"type": "label", "binary": True}]})
    assert [o[0] for o in prov.outputs] == ["audio", "big.teacher_ids", "big.teacher_logits", "big.teacher_count", "label"]
    want = padded(recs, range(5))
    for got in (prov.run_host([r[:3] for r in recs[:5]]), {k: v.cpu().numpy() for k, v in prov.run_device([r[:3] for r in recs[:5]]).items()}):
        for name, w in zip(("ids", "logits", "count"), want):
            g = got["big.teacher_" + name]
            assert np.array_equal(g if batch_major else g.T.reshape(w.shape), w)
    # a short batch leaves no entries behind its records
    out = {n: torch.full((5,) + d, 77, dtype=torch.int32 if "logits" not in n and n != "audio" else torch.float32, device="cuda")
           for n, d, _, _ in prov.outputs}
    if batch_major:
        prov.run_device([r[:3] for r in recs[:2]], out)
        assert np.array_equal(out["big.teacher_ids"][:2].cpu().numpy(), want[0][:2])
        assert (out["big.teacher_ids"][2:] < 0).all() or (out["big.teacher_ids"][2:] == 77).all()


def test_top_logits_records_that_are_refused(ctx):
    from aeon_b200.provider import Provider, top_logits_record
    cfg = {"batch_size": 1, "etl": [dict(TOP)], "augmentation": []}
    prov = Provider(ctx, cfg)
    good = top_logits_record([[1, 28, -7]], [[3.0, 2.0, 1.0]])
    got = prov.run_host([(good,)])
    assert got["teacher_ids"][0, 0].tolist() == [1, 28, -1, -1, -1] and got["teacher_count"][0, 0] == 1
    assert prov.run_host([(top_logits_record(np.zeros((0, 2)), np.zeros((0, 2))),)])["teacher_count"][0, 0] == 0
    long = top_logits_record(np.ones((FRAMES + 5, 1)), np.ones((FRAMES + 5, 1)))
    assert prov.run_host([(long,)])["teacher_count"][0, 0] == FRAMES
    head = lambda n, k, size: np.array([n, k], "<i4").tobytes() + bytes(size)  # noqa: E731
    for blob, words in ((b"", "size 0"), (b"1234", "does not hold"), (good[:-1], "does not hold"), (good + b"12345678", "does not hold"),
                        (head(-1, 1, 8), "does not hold"), (head(1, 0, 0), "does not hold"), (head(1, -1, 0), "does not hold"),
                        (head(2 ** 31 - 1, 2 ** 31 - 1, 8), "does not hold"), (top_logits_record([[29]], [[0]]), "vocab"),
                        (top_logits_record(np.zeros((2, 6)), np.zeros((2, 6))), "entries")):
        with pytest.raises(RuntimeError, match=words):
            prov.run_host([(blob,)])
    assert prov.run_host([(good,)])["teacher_ids"][0, 0, 0] == 1
    for changes in (dict(k=0), dict(k=257), dict(max_positions=0), dict(vocab=-1), dict(depth=3)):
        with pytest.raises(RuntimeError):
            Provider(ctx, dict(cfg, etl=[dict(TOP, **changes)]))
    with pytest.raises(RuntimeError):
        Provider(ctx, dict(cfg, etl=[{"type": "top_logits", "k": 2}]))


def loader(root, **changes):
    from aeon_b200 import DataLoader
    cfg = {"manifest_filename": str(root / "m.tsv"), "manifest_root": str(root), "batch_size": 4, "cpu_list": "0", "device_output": True,
           "etl": [AUDIO, TOP, {"type": "label", "binary": True}]}
    return DataLoader(dict(cfg, **changes))


def one_pass(dl):
    return [{k: v.clone() for k, v in batch} for batch in dl]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_passes_from_the_cache(ctx, dataset, code):
    root, _ = dataset
    plain, kept = loader(root), loader(root, feature_cache=code)
    want = one_pass(plain)
    assert len(want) == 3  # ten records, the last batch starts over
    first = one_pass(kept)
    for w, f in zip(want, first):
        for name in ("teacher_ids", "teacher_logits", "teacher_count", "label"):
            assert torch.equal(w[name], f[name])
        x = w["audio"].double().cpu().numpy()
        q, s = ocache.encode(x, code)
        v = ocache.decode(q, s, code)
        got = f["audio"].double().cpu().numpy()
        assert np.array_equal(np.isinf(got), np.isinf(v)) and np.isinf(v).any()  # the empty mel filters
        ok = np.isfinite(v)
        assert (np.abs(got[ok] - v[ok]) <= 2.0 ** -24 * np.abs(v[ok]) * 1.001).all()
    assert list(kept) == []  # finished until reset
    for _ in range(3):
        kept.reset()
        assert kept.position == 0
        again = []
        for batch in kept:
            assert [n for n, _ in batch] == [n for n, _, _ in kept.outputs]
            again.append({k: v.clone() for k, v in batch})
            dict(batch)["label"].fill_(99)  # the caller's own to write to
        assert kept.position == 3 and len(again) == 3
        for f, a in zip(first, again):
            assert f.keys() == a.keys() and all(torch.equal(f[k], a[k]) and f[k].shape == a[k].shape for k in f)
    plain.close()
    kept.close()


def test_an_incomplete_pass_is_read_again(ctx, dataset):
    root, _ = dataset
    dl = loader(root, feature_cache="int8")
    next(dl)
    dl.reset()
    a = one_pass(dl)
    dl.reset()
    next(dl)
    dl.reset()  # a pass from the cache, left early
    b = one_pass(dl)
    assert len(a) == len(b) == 3 and all(torch.equal(x[k], y[k]) for x, y in zip(a, b) for k in x)
    dl.close()


def test_training_by_distillation(ctx, dataset):
    """Two passes of a linear student over the loader's batches, on streams of the caller's choice; loss and gradients of every step
    against the 64-bit oracle and torch's own product for the weights."""
    from aeon_b200 import kernels as K_
    root, recs = dataset
    g = torch.Generator("cuda")
    g.manual_seed(3)
    weight = (torch.randn(64, VOCAB, generator=g, device="cuda") * 0.02).requires_grad_()
    dl = loader(root, feature_cache="int8")
    t, steps = 2.0, 0
    for epoch in range(2):
        for batch in dl:
            d = dict(batch)
            x = torch.where(d["audio"] == float("-inf"), torch.zeros_like(d["audio"]), d["audio"])
            logits = x @ weight
            ids, teacher = d["teacher_ids"], d["teacher_logits"]
            rows = d["teacher_count"].sum().item()
            loss, lse, grad = K_.distill_loss(ctx, logits.detach(), ids, teacher, t, grad_scale=1.0 / rows)
            weight.grad = None
            logits.backward(grad)
            flat = [a.reshape(-1, a.shape[-1]).double().cpu().numpy() if a.is_floating_point() else a.reshape(-1, a.shape[-1]).cpu().numpy()
                    for a in (logits.detach(), ids, teacher)]
            want = odistill.distill(flat[0], flat[1], flat[2], t, grad_scale=1.0 / rows)
            # rows of 29 values: every tolerance of test_gpu_distill is below 1e-5 of the terms, which stay below 100 here
            assert np.abs(loss.double().cpu().numpy().ravel() - want[0]).max() < 1e-3
            assert np.abs(grad.double().cpu().numpy().reshape(-1, VOCAB) - want[2]).max() < 1e-5
            assert not loss[~(ids >= 0).any(-1)].any()
            w = x.reshape(-1, 64).double().T @ torch.from_numpy(want[2]).cuda()
            assert (weight.grad.double() - w).abs().max().item() <= 1e-4 * w.abs().max().item() + 1e-4
            with torch.no_grad():
                weight -= 1e-4 * weight.grad
            steps += 1
        dl.reset()
    assert steps == 6
    dl.close()
