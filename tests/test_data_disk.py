"""The ring that batches of a disk stream travel through (data/disk.py), without a GPU."""
import torch

from ttdg_mgm_amd.data import disk


def ring_of(monkeypatch, **kw):
    """A ring as a process with a GPU makes it."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    real = torch.empty

    def empty(*a, pin_memory=False, **k):
        if pin_memory and "refuse" in kw:
            raise RuntimeError("no page-locked memory")
        t = real(*a, **k)
        made.append((t, pin_memory))
        return t

    made = []
    monkeypatch.setattr(torch, "empty", empty)
    r = disk._Ring(3, 2, (3, 4, 5), 2, (4, 5), kw.get("register", True))
    return r, made


def test_a_ring_without_page_locked_memory_still_carries_batches(monkeypatch):
    """Where page-locked memory is refused the slots themselves are handed out, as with register=False."""
    for kw in (dict(refuse=True), dict(register=False)):
        r, _ = ring_of(monkeypatch, **kw)
        assert not r.pinned
        r.images[1].fill_(7)
        r.masks[1].fill_(True)
        images, masks = r.batch_views(1, 1)
        assert images.data_ptr() == r.images[1].data_ptr() and images.shape == (1, 3, 4, 5) and int(images.min()) == 7
        assert masks.data_ptr() == r.masks[1].data_ptr() and masks.shape == (2, 4, 5) and bool(masks.all())


def test_a_batch_is_copied_to_the_twin_of_its_slot(monkeypatch):
    """With page-locked memory a batch is read from the slot's twin: a worker's next batch in the slot does not reach it."""
    r, made = ring_of(monkeypatch)
    assert r.pinned and sum(p for _, p in made) == 2
    r.images[2].fill_(7)
    r.masks[2].fill_(True)
    images, masks = r.batch_views(2, 2)
    r.images[2].fill_(9)
    r.masks[2].fill_(False)
    assert int(images.min()) == int(images.max()) == 7 and bool(masks.all())


def test_a_slot_is_copied_without_waking_other_threads(monkeypatch):
    """torch's copy_ shares 3 MB out to a thread per CPU; beside busy workers that took milliseconds a batch, and the streamed rate a quarter."""
    r, _ = ring_of(monkeypatch)

    def refused(*a, **k):
        raise AssertionError("a copy over several threads")

    monkeypatch.setattr(torch.Tensor, "copy_", refused)
    assert r.batch_views(0, 2)[0].shape == (2, 3, 4, 5)
