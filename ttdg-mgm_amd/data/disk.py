"""A test stream on disk + the reference's loader topology (data/build.py:122-154: torch DataLoader, NUM_WORKERS worker
PROCESSES, batch sampler of TEST.BATCH, trivial collate).

``prerender`` writes a registered synthetic dataset to a directory once (one uncompressed .npz per image: the uint8 image, the
bit-packed ground-truth masks, boxes, classes) - standing for a dataset of decoded images on local storage; ``DiskStream``
reads it back through worker processes that never touch the GPU.  The main process then only pins, uploads and (on the
device) resizes: TestLoader(resident=False) on a ``kind == "disk"`` dataset."""
import os

import numpy as np
import torch


def prerender(name, root):
    """Materialise dataset ``name`` (any registered kind) under ``root``; returns the number of images written."""
    from . import dataset_dicts, dataset_size
    os.makedirs(root, exist_ok=True)
    n = dataset_size(name)
    for i in range(n):
        path = os.path.join(root, "%07d.npz" % i)
        if os.path.exists(path):
            continue
        d = dataset_dicts(name, i, i + 1)[0]
        anns = d["annotations"]
        masks = np.stack([a["mask"].numpy() for a in anns]) if anns else np.zeros((0, d["height"], d["width"]), bool)
        tmp = path + ".tmp.npz"
        np.savez(tmp, image=d["image"].numpy(), masks=np.packbits(masks, axis=-1), mask_w=np.int64(d["width"]),
                 boxes=np.stack([a["bbox"].numpy() for a in anns]).astype(np.float32) if anns else np.zeros((0, 4), np.float32),
                 classes=np.array([a["category_id"] for a in anns], np.int64), image_id=np.int64(d["image_id"]), seed=np.int64(d.get("seed", -1)))
        os.replace(tmp, path)
    return n


class DiskDataset(torch.utils.data.Dataset):
    """Map-style dataset over a pre-rendered directory: __getitem__ returns the same dict ``data.dataset_dicts`` yields."""

    def __init__(self, root, n):
        self.root, self.n = root, int(n)

    def __len__(self):
        return self.n

    def __getitem__(self, i):
        with np.load(os.path.join(self.root, "%07d.npz" % i)) as z:
            img = torch.from_numpy(z["image"])
            w = int(z["mask_w"])
            masks = torch.from_numpy(np.unpackbits(z["masks"], axis=-1, count=w).astype(bool))
            boxes, classes = torch.from_numpy(z["boxes"]), z["classes"]
            image_id, seed = int(z["image_id"]), int(z["seed"])
        anns = []
        for k in range(len(classes)):
            m = masks[k]
            rows, cols = m.sum(1, dtype=torch.int64), m.sum(0, dtype=torch.int64)          # centroid as DiceEvaluator._centroid (exact integer sums)
            cnt = int(rows.sum())
            cen = (float("nan"), float("nan")) if cnt == 0 else (float((rows * torch.arange(m.shape[0])).sum()) / cnt,
                                                                  float((cols * torch.arange(m.shape[1])).sum()) / cnt)
            anns.append(dict(bbox=boxes[k], category_id=int(classes[k]), mask=m, centroid=cen))
        d = dict(image=img, height=int(img.shape[1]), width=int(img.shape[2]), image_id=image_id, annotations=anns)
        if seed >= 0:
            d["seed"] = seed
        return d


def _copy(to, of):
    """Host memory to host memory on the calling thread alone: 0.1 ms for 3 MB.  torch's copy_ wakes a thread
    per CPU, which beside the busy workers took 1.2 ms a tensor in the loader and more in the adaptation loop: with it the streamed input ran at
    84 of 112.6 images/s, with this at 104.6 (20 batches of four 512 x 512 images, two runs each in turn)."""
    np.copyto(to.numpy(), of.numpy())
    return to


class _Ring:
    """A ring of batch slots in SHARED memory: worker processes write a decoded batch straight into its slot - no per-batch
    shared-memory segment.  For the GPU every slot has a page-locked twin of the main process (allocated as such: registering the
    shared memory itself is refused on some hosts): ``expand`` copies an arrived slot there once and the DMA starts from it.
    Where page-locked memory is refused the slots themselves are handed out (``pinned`` False) and uploaded through staging buffers.
    Allocated before the workers are forked, so they inherit the mapping.  Slot s is handed to a worker again only after the
    upload that read it or its twin has completed (``wait``)."""

    def __init__(self, slots, batch, image_shape, masks_per_image, mask_shape, register):
        self.slots, self.batch, self.mpi = slots, batch, masks_per_image
        self.images = torch.empty((slots, batch) + tuple(image_shape), dtype=torch.uint8).share_memory_()
        self.masks = torch.empty((slots, batch * max(1, masks_per_image)) + tuple(mask_shape), dtype=torch.bool).share_memory_()
        self.events = [None] * slots
        self.pinned = False
        if register and torch.cuda.is_available():
            try:
                self.pin_images = torch.empty(self.images.shape, dtype=self.images.dtype, pin_memory=True)
                self.pin_masks = torch.empty(self.masks.shape, dtype=self.masks.dtype, pin_memory=True)
                self.pinned = True
            except RuntimeError:
                self.pin_images = self.pin_masks = None          # both or none

    def batch_views(self, slot, nb):
        """Images and masks (None without any) of the ``nb`` items that have arrived in a slot."""
        images, masks = self.images[slot, :nb], self.masks[slot, :nb * self.mpi] if self.mpi else None
        if self.pinned:
            images = _copy(self.pin_images[slot, :nb], images)
            masks = None if masks is None else _copy(self.pin_masks[slot, :nb * self.mpi], masks)
        return images, masks

    def wait(self, slot):
        if self.events[slot] is not None:
            self.events[slot].synchronize()
            self.events[slot] = None


class _Batches(torch.utils.data.Sampler):
    """Batch sampler whose index range is set per pass (the workers are persistent: they outlive a pass).  With a ring every
    index travels as (image index, slot, position in the batch): the worker-side collate knows where to write."""

    def __init__(self, batch, ring=None):
        self.batch, self.lo, self.hi, self.ring, self.count = batch, 0, 0, ring, 0

    def __iter__(self):
        for s in range(self.lo, self.hi, self.batch):
            idx = list(range(s, min(s + self.batch, self.hi)))
            if self.ring is None:
                yield idx
            else:
                slot = self.count % self.ring.slots
                self.count += 1
                self.ring.wait(slot)                 # main process: the slot's previous upload must have completed
                yield [(i, slot, k) for k, i in enumerate(idx)]

    def __len__(self):
        return (self.hi - self.lo + self.batch - 1) // self.batch


class _RingDataset(DiskDataset):
    """DiskDataset whose items land in a ring slot (worker side)."""

    def __init__(self, root, n, ring):
        super().__init__(root, n)
        self.ring = ring

    def __getitem__(self, key):
        i, slot, k = key
        d = super().__getitem__(i)
        r = self.ring
        fits = tuple(d["image"].shape) == tuple(r.images.shape[2:]) and len(d["annotations"]) == r.mpi and \
            all(tuple(a["mask"].shape) == tuple(r.masks.shape[2:]) for a in d["annotations"])
        if fits:
            r.images[slot, k].copy_(d["image"])
            for j, a in enumerate(d["annotations"]):
                r.masks[slot, k * r.mpi + j].copy_(a["mask"])
        d["_ring"] = (slot, k, fits)
        return d


def _collate(items):
    """Runs in the WORKER process.  A batch crosses the process boundary as plain Python metadata plus EITHER a ring slot
    number (the pixels are already in shared memory) OR two shared-memory tensors - the stacked uint8 images and the
    stacked ground-truth masks: every tensor costs the receiving process a connection to the worker's resource sharer (~1 ms with
    its authentication handshake; 14 tensors per batch were 15 ms), Python numbers cost nothing.  ``expand`` rebuilds the
    per-image dicts as views.  Images of different sizes travel as they are."""
    ring = [d.pop("_ring", None) for d in items]
    if len({tuple(d["image"].shape) for d in items}) != 1 or len({tuple(a["mask"].shape) for d in items for a in d["annotations"]}) > 1:
        return dict(items=items, images=None, masks=None, slot=None)
    ms = [a["mask"] for d in items for a in d["annotations"]]
    meta = [dict(height=d["height"], width=d["width"], image_id=d["image_id"], seed=d.get("seed"),
                 anns=[(a["bbox"].tolist(), a["category_id"], a.get("centroid")) for a in d["annotations"]]) for d in items]
    if all(x is not None and x[2] for x in ring):
        return dict(items=None, images=None, masks=None, meta=meta, slot=ring[0][0])
    return dict(items=None, images=torch.stack([d["image"] for d in items]), masks=torch.stack(ms) if ms else None, meta=meta, slot=None)


def expand(batch, ring=None):
    """Main process: the list of dataset dicts of a collated batch (tensors are views of the two stacked ones / of the ring slot)."""
    if batch["items"] is not None:
        return batch["items"]
    if batch.get("slot") is not None and batch["images"] is None:
        nb = len(batch["meta"])
        batch["images"], batch["masks"] = ring.batch_views(batch["slot"], nb)
    out, k = [], 0
    for i, m in enumerate(batch["meta"]):
        anns = []
        for box, cat, cen in m["anns"]:
            a = dict(bbox=torch.tensor(box, dtype=torch.float32), category_id=cat, mask=batch["masks"][k])
            if cen is not None:
                a["centroid"] = cen
            anns.append(a)
            k += 1
        d = dict(image=batch["images"][i], height=m["height"], width=m["width"], image_id=m["image_id"], annotations=anns)
        if m["seed"] is not None:
            d["seed"] = m["seed"]
        out.append(d)
    return out


class DiskStream:
    """Persistent worker processes over a DiskDataset; ``epoch(lo, hi)`` iterates collated batches (``_collate``): pass them to
    ``expand(batch, stream.ring)`` for the list of dataset dicts; ``images`` / ``masks`` are then the stacked tensors (None for
    ragged batches).  ``ring=True``: batches of the dataset's common shape travel through a shared ring."""

    def __init__(self, root, n, batch, workers=4, prefetch=2, ring=False, register=True):
        self.ring = None
        if ring and workers > 0 and n > 0:
            d0 = DiskDataset(root, n)[0]
            if d0["annotations"]:
                self.ring = _Ring(workers * prefetch + 4, batch, d0["image"].shape, len(d0["annotations"]), d0["annotations"][0]["mask"].shape, register)
        self.sampler = _Batches(batch, self.ring)
        kw = dict(persistent_workers=True, prefetch_factor=prefetch) if workers > 0 else {}
        ds = _RingDataset(root, n, self.ring) if self.ring is not None else DiskDataset(root, n)
        self.loader = torch.utils.data.DataLoader(ds, batch_sampler=self.sampler, num_workers=workers, collate_fn=_collate, **kw)

    def epoch(self, lo, hi):
        self.sampler.lo, self.sampler.hi = int(lo), int(hi)
        return iter(self.loader)

    def start(self):
        """Spawn the workers (a one-batch pass that is thrown away): loader construction, outside any timed region."""
        for _ in self.epoch(0, min(self.sampler.batch, len(self.loader.dataset))):
            pass
