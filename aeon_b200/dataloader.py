"""Python iterator with the surface of aeon's ``aeon.DataLoader`` (aeon src/api.cpp:104-425).

    dl = DataLoader(config={...})        # aeon's loader JSON as a dict
    for batch in dl:                     # tuple of (name, array) pairs, one per output buffer
        ...
    len(dl); dl.ndata; dl.batch_size; dl.axes_info; dl.config; dl.reset()

Arrays are numpy views of the loader's pinned host buffers (valid until the next batch, as in
aeon), or torch CUDA tensors when the config sets ``"device_output": true``.  With
``"batch_major": false`` they are 2-D ``(elements, batch)`` views, as in aeon.

``"feature_cache": "int8"`` (or ``"e4m3"``) keeps the features of audio elements on the GPU in 8 bits, with a scale for each frame,
while they are first delivered, and the other outputs as they are; the passes after the first complete one (each started by
``reset()``) read them from there, with no file, upload or transform.  Every pass delivers the same values: the first one those that
its codes stand for.  It needs ``"device_output": true``, elements that are the same in every pass (audio, label, blob, top_logits)
in the same order (no ``shuffle_enable``, no ``shuffle_manifest``), and the iteration mode ONCE.
"""
import ctypes as C
import json

import numpy as np

from . import _lib as L
from .provider import NP_DTYPE


def dict2json(config):
    """aeon.dict2json: the JSON text aeon builds from a python dict."""
    return json.dumps(config)


PAGE_FRAMES = 64  # frames in a page of the feature cache


def check_feature_cache(config):
    """The code of the feature cache a configuration asks for, None without one; ValueError where it cannot have one."""
    code = config.get("feature_cache")
    if code is None:
        return None
    if code not in ("int8", "e4m3"):
        raise ValueError("feature_cache must be 'int8' or 'e4m3', not %r" % (code,))
    if not config.get("device_output", False) or not config.get("batch_major", True):
        raise ValueError("feature_cache needs device_output and batch_major")
    if config.get("iteration_mode", "ONCE") != "ONCE":
        raise ValueError("feature_cache needs the iteration mode ONCE")
    if config.get("shuffle_enable", False):
        raise ValueError("feature_cache keeps the order of the first pass: shuffle_enable must be off")
    if config.get("shuffle_manifest", False):
        # every pass has another order of the blocks, and with several nodes other records
        raise ValueError("feature_cache keeps the records and order of the first pass: shuffle_manifest must be off")
    types = [e.get("type") for e in config.get("etl", [])]
    if "audio" not in types or set(types) - {"audio", "label", "blob", "top_logits"}:
        raise ValueError("feature_cache takes audio elements, with label, blob and top_logits beside them, not %s" % ", ".join(map(str, types)))
    return code


class _CachedPasses:
    """The batches of a complete pass: audio outputs in 8-bit pages, one sequence for each record of a batch, the others as they are."""

    def __init__(self, device, code, outputs, batch_size, batches):
        import torch
        from .kernels import Context, FeatureCache
        self.ctx = Context(device)
        self.batches, self.batch_size = batches, batch_size
        self.filled = self.position = 0
        self.serving = False  # whether the pass under way is read from here
        self.outputs, self.caches, self.tables, self.kept = outputs, {}, {}, {}
        for name, shape, dt in outputs:
            if name != "audio" and not name.endswith(".audio"):
                self.kept[name] = []
                continue
            frames, bands = shape
            pages = -(-frames // PAGE_FRAMES)
            with torch.cuda.device(device):
                self.tables[name] = torch.arange(batches * batch_size * pages, dtype=torch.int32, device="cuda").view(batches, batch_size, pages)
                self.caches[name] = FeatureCache.allocate(self.ctx, batches * batch_size * pages, PAGE_FRAMES, 1, bands, code)
        torch.cuda.synchronize(device)

    def add(self, batch):
        """Keeps a batch of the first pass; its audio is replaced by the values that are kept.  Complete on return: the loader
        may write the next batch over it."""
        import torch
        with torch.cuda.stream(self.ctx.torch_stream):
            for name, array in batch:
                if name in self.caches:
                    self.caches[name].write(array, self.tables[name][self.filled], values=array)
                else:
                    self.kept[name].append(array.clone())
        self.ctx.synchronize()
        self.filled += 1

    def next(self):
        if self.position >= self.batches:
            raise StopIteration
        b, self.position = self.position, self.position + 1
        out = []
        for name, shape, _ in self.outputs:
            if name in self.caches:
                out.append((name, self.caches[name].read(self.tables[name][b], shape[0]).squeeze(2)))
            else:
                out.append((name, self.kept[name][b].clone()))  # the caller may write to what it is given
        return tuple(out)

    def restart(self):
        """Whether the next pass is read from here; an incomplete first pass is dropped."""
        self.position = 0
        self.serving = self.filled == self.batches
        if not self.serving:
            self.filled = 0
            for kept in self.kept.values():
                kept.clear()
        return self.serving

    def close(self):
        # reads run on the streams that were current at their calls; the pages may not go to another user of the memory before
        # the last of them
        import torch
        torch.cuda.synchronize(self.ctx.device)
        self.caches.clear()
        self.tables.clear()
        self.kept.clear()
        self.ctx.close()


class DataLoader:
    def __init__(self, config, device=0):
        if not isinstance(config, dict):
            raise TypeError("config must be a dict")
        self.handle = None
        code = check_feature_cache(config)
        self.lib = L.load()
        self.config = dict(config)
        own = {k: v for k, v in config.items() if k != "feature_cache"}
        h = C.c_void_p()
        L.check(self.lib.aeonb_loader_create(dict2json(own).encode(), int(device), C.byref(h)))
        self.handle = h
        self.device = int(device)
        self.batch_size = self.lib.aeonb_loader_batch_size(h)
        self.ndata = self.lib.aeonb_loader_record_count(h)
        self.batch_major = bool(self.config.get("batch_major", True))
        self.device_output = bool(self.config.get("device_output", False))
        self.outputs = []
        self.axes_info = {}
        for i in range(self.lib.aeonb_loader_output_count(h)):
            dims = (C.c_int64 * 8)()
            dt = C.c_int32()
            rank = self.lib.aeonb_loader_output_shape(h, i, dims, C.byref(dt))
            name = self.lib.aeonb_loader_output_name(h, i).decode()
            shape = tuple(int(dims[k]) for k in range(rank))
            axes = self.lib.aeonb_loader_axis_names(h, i).decode()
            self.outputs.append((name, shape, int(dt.value)))
            if axes:
                self.axes_info[name] = dict(zip(axes.split(","), shape))
        self._passes = None
        if code:
            self._passes = _CachedPasses(self.device, code, self.outputs, self.batch_size, self.lib.aeonb_loader_batch_count(h))

    def __len__(self):
        return self.ndata

    def __iter__(self):
        return self

    def _wrap(self, ptr, shape, dt):
        full = (self.batch_size,) + shape if self.batch_major else (int(np.prod(shape)), self.batch_size)
        count = int(np.prod(full))
        if self.device_output:
            import torch
            from .kernels import _TORCH_DTYPE, DTYPE_SIZE

            class _Mem:  # minimal __cuda_array_interface__ holder
                pass
            m = _Mem()
            m.__cuda_array_interface__ = {"shape": full, "typestr": np.dtype(NP_DTYPE[dt]).str, "data": (ptr, False),
                                          "version": 2}
            return torch.as_tensor(m, device="cuda:%d" % self.device)
        buf = (C.c_char * (count * np.dtype(NP_DTYPE[dt]).itemsize)).from_address(ptr)
        return np.frombuffer(buf, NP_DTYPE[dt]).reshape(full)

    def __next__(self):
        passes = self._passes
        if passes is not None and passes.serving:
            return passes.next()
        ptrs = (C.c_void_p * len(self.outputs))()
        status = L.check(self.lib.aeonb_loader_next(self.handle, ptrs))
        if status == L.END:
            raise StopIteration
        batch = tuple((name, self._wrap(ptrs[i], shape, dt)) for i, (name, shape, dt) in enumerate(self.outputs))
        if passes is not None:
            passes.add(batch)
        return batch

    next = __next__

    def reset(self):
        if self._passes is not None and self._passes.restart():
            return
        L.check(self.lib.aeonb_loader_reset(self.handle))

    @property
    def position(self):
        if self._passes is not None and self._passes.serving:
            return self._passes.position
        return self.lib.aeonb_loader_position(self.handle)

    def close(self):
        if getattr(self, "handle", None):
            self.lib.aeonb_loader_destroy(self.handle)
            self.handle = None
        if getattr(self, "_passes", None):
            self._passes.close()
            self._passes = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
