"""A disk stream whose ring got no page-locked memory delivers the same items (data/disk.py, data/__init__.py)."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.multiprocess]


@pytest.mark.parametrize("refused", [False, True])
def test_streaming_disk_loader_with_and_without_page_locked_slots(tmp_path, monkeypatch, refused):
    """More batches than ring slots; every item is kept and looked at after the pass, when its slot has taken other batches: images, the masks
    on the device and the masks the annotations hold are the resident loader's."""
    from ttdg_mgm_amd import data
    from ttdg_mgm_amd.config import get_cfg
    cfg = get_cfg()
    cfg.TEST.BATCH = 2
    cfg.INPUT.MIN_SIZE_TEST = 200
    tag = "gtwin%d" % refused
    data.register_synthetic(tag + "_src", 31, size=128, id_offset=900)
    data.register_disk(tag, str(tmp_path / "s"), source=tag + "_src", workers=2)
    ref = [it for b in data.build_detection_test_loader(cfg, tag + "_src", 0, 1, None, resident=True) for it in b]
    real = torch.empty

    def empty(*a, pin_memory=False, **k):
        if pin_memory and refused:
            raise RuntimeError("no page-locked memory")
        return real(*a, pin_memory=pin_memory, **k)

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        stm = data.build_detection_test_loader(cfg, tag, 0, 1, torch.device("cuda:0"), resident=False)
    stm.start_workers()
    assert stm._disk.ring.pinned == (not refused)
    got = [it for batch in stm for it in batch]
    torch.cuda.synchronize()
    assert len(got) == len(ref) == 31 and (len(ref) + 1) // 2 > stm._disk.ring.slots
    for it, r in zip(got, ref):
        want = torch.stack([a["mask"] for a in r["dataset_dict"]["annotations"]])
        assert it["image_id"] == r["image_id"]
        assert int((it["image"].cpu().int() - r["image"].int()).abs().max()) <= 1
        assert torch.equal(it["dataset_dict"]["device_masks"].cpu(), want)
        assert torch.equal(torch.stack([a["mask"] for a in it["dataset_dict"]["annotations"]]).cpu(), want)
