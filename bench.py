"""bench.py — adapted images/sec of the multi-graph-matching TTA hot path on MI355X.

    python bench.py --gpus N --steps K --warmup W          (N > 1 launches its own N ranks, one per GPU, over RCCL;
                                                            under torch.distributed.run the environment decides instead)

Workload: synthetic 512x512 2-class fundus stream, ResNet-50-FPN Mask R-CNN stand-in,
TEST.BATCH = 4 (-> 800x800 after the test mapper's resize), 20-sweep Sinkhorn, one TTA step per batch, then the eval-mode
Dice pass over the same batches (reference order, engine/trainer.py:469-485).  One "step" = one adapted batch (its TTA step
+ its share of the Dice pass).  Each rank adapts its own contiguous shard (InferenceSampler semantics, no data-path
collective); at N > 1 the one collective of the path is the all-gather of the per-rank Dice score lists (RCCL).

Weights: by default a deterministic TRAINED-REGIME checkpoint fitted before the timed region by tools/synth_checkpoint.py
on a disjoint synthetic source stream (no real checkpoint is obtainable offline): detections are the detector's own
(free-running), Dice is numeric, the solver runs in its converging regime.  `--weights random` / `--teacher-forced`
select the round-1 configuration; at N = 1 both are also run as labelled A/B lines (`ab`) next to the headline.

Prints ONE JSON line on rank 0: the contract fields, `roofline` (dominant hand-written kernel, timed live with HIP events on
the launch stream) + `roofline_other_kernels`, and at N = 1 `cpu_baseline` (the oracle "port" on the host cores: 1 warm-up +
median of `--cpu-reps`) and `dice_parity` (GPU vs CPU port on the same checkpoint and images).
"""
import argparse
import json
import os
import socket
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

FP32_PEAK_TFLOPS = 157.3      # MI355X fp32 vector == fp32 MFMA peak (MI355X_MICROARCH.md)
HBM_PEAK_GBS = 8000.0


def parse(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--size", type=int, default=0, help="image side (0 = the workload's: 512 for cfg2, 384 for cfg5)")
    ap.add_argument("--workload", choices=("cfg2", "cfg5"), default="cfg2",
                    help="cfg2: 512x512 2-class fundus stream, fp32 (the headline); cfg5: 384x384 3-class polyp stream with the bf16 "
                         "backbone / fp32 matching split (BASELINE configs[4], here per GPU)")
    ap.add_argument("--images", type=int, default=0,
                    help="strong-scaling mode (cfg-4): a FIXED stream of this many images is sharded over the ranks "
                         "(steps per rank = images / (gpus * batch)); 0 = weak scaling with --steps per rank")
    ap.add_argument("--weights", choices=("trained", "random"), default="trained")
    ap.add_argument("--random-init", action="store_true", help="alias of --weights random")
    ap.add_argument("--teacher-forced", action="store_true", help="replace the detector's boxes by jittered GT boxes (SURVEY.md §8d)")
    ap.add_argument("--free-running", action="store_true", help="(default; kept for round-1 command lines)")
    ap.add_argument("--no-ab", action="store_true", help="skip the A/B variants (teacher-forced, random-init, loader-inclusive)")
    ap.add_argument("--ckpt-steps", type=int, default=-1, help="stage-1 steps of the synthetic checkpoint (-1 = the tool's default)")
    ap.add_argument("--ckpt-tta-steps", type=int, default=-1)
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--cpu-reps", type=int, default=3, help="timed CPU repetitions after 1 warm-up (median reported)")
    ap.add_argument("--cpu-threads", type=int, default=0, help="0 = min(os.cpu_count(), 64)")
    ap.add_argument("--cpu-1thread", action="store_true", help="also time ONE repetition with 1 thread (minutes)")
    ap.add_argument("--cpu-allcores", action="store_true",
                    help="also time ONE repetition with os.cpu_count() threads, under a 10-minute limit (recorded once per round in profiles/)")
    ap.add_argument("--strong-images", type=int, default=512,
                    help="with --gpus N > 1 and no --images: size of the fixed stream of the additional strong-scaling pass (0 = skip it)")
    ap.add_argument("--eval-streams", type=int, default=1, help="concurrent eval batches (HIP streams) in the Dice pass; 1 = sequential")
    ap.add_argument("--no-overlap-detector", action="store_true", help="A/B: keep the teacher-forced RPN + box head on the main stream")
    ap.add_argument("--eval-coalesce", type=int, default=1, help="loader batches merged into one inference call in the Dice pass; 1 = none")
    ap.add_argument("--bf16-backbone", action="store_true", help="cfg-5 style: bf16 autocast for the backbone only")
    ap.add_argument("--dist-backend", default="nccl", help="nccl (= RCCL, default) or gloo (validation on a 1-GPU box / CPU plumbing test)")
    ap.add_argument("--share-device", action="store_true", help="validation only: every rank uses cuda:0")
    ap.add_argument("--sync-universe", action="store_true",
                    help="Mode S (SURVEY.md 8e): all ranks adapt on ONE multi-graph (RCCL all-gather of the node embeddings, gradient "
                         "all-reduce) = the single-GPU algorithm at batch N*B; default is Mode R (independent shards, as the reference)")
    ap.add_argument("--gagm-threads", type=int, default=0, help="A/B: workgroup size of the single-workgroup solver (256 / 512; 0 = automatic)")
    ap.add_argument("--roi-align-mode", type=int, default=3, help="A/B: 3 = channels-last ROIPooler kernel (default), 2 = separable table kernel on NCHW, "
                                                                  "1 = direct kernel, XCD-sliced, 0 = direct, flat (round 1)")
    ap.add_argument("--roi-xcd-chunks", action="store_true", help="A/B: channels-last ROIPooler with one contiguous eighth of the ROI list per XCD instead of ROI r on workgroup r")
    ap.add_argument("--roi-one-channel-per-lane", action="store_true", help="A/B: the round 2-5 channels-last ROIPooler (one channel per lane, dword taps) instead of four channels per lane (16-byte taps)")
    ap.add_argument("--roi-chunk", type=int, default=0, help="A/B: bins the channels-last ROIPooler stages per output flush: 49 (round 2), 25 (default) or 13")
    ap.add_argument("--graphs", action="store_true", help="A/B: hipGraph replay of the backbone's no-grad forward in the Dice pass (modeling/graphed.py; default: eager - measured equal)")
    ap.add_argument("--timer-every", type=int, default=7, help="HIP-event pairs around every N-th launch of the kernels launched dozens of times per batch "
                    "(ops.KERNEL_TIMER_SAMPLED; 1 = every launch, the round 1-5 protocol, which costs ~4 %% of the timed region)")
    ap.add_argument("--vendor-rpn-heads", action="store_true", help="A/B: the RPN's two 1 x 1 heads as vendor convolutions behind a bias + ReLU pass (round 5) instead of one streaming product per level")
    ap.add_argument("--own-pointwise-backward", action="store_true", help="A/B: dX / dW of the 1 x 1 convolutions on the streaming product's backward layouts instead of MIOpen")
    ap.add_argument("--cfg3-only", action="store_true", help="run only the cfg-3 operator-level block and print it (the command rocprofv3 profiles for profiles/rNN_cfg3_block_*)")
    ap.add_argument("--no-cfg3", action="store_true", help="skip the cfg-3 operator-level block and the whole-step FLOP count")
    ap.add_argument("--stamp-all", action="store_true", help="rounds 1-5 protocol: the headline pass itself stamps every hand-written kernel (no separate instrumented pass)")
    ap.add_argument("--no-kernel-timers", action="store_true", help="debug A/B: no HIP events around the hand-written kernels in the timed pass (the rooflines are then empty): what the event pairs themselves cost")
    ap.add_argument("--vendor-pointwise", action="store_true", help="A/B: the backbone's 1 x 1 convolutions on MIOpen + the one-pass epilogue kernel (round 5) instead of the fused streaming product (csrc/pointwise.hip)")
    ap.add_argument("--no-miopen-db", action="store_true", help="A/B: ignore the tuned MIOpen find-db shipped in ttdg-mgm_amd/miopen_db (MIOpen's heuristic picks the solvers)")
    ap.add_argument("--miopen-search", action="store_true", help="tuning run: torch.backends.cudnn.benchmark = True, i.e. MIOpen times its solvers for every "
                    "convolution shape it meets (minutes) and records the winners in its user find-db (MIOPEN_USER_DB_PATH)")
    ap.add_argument("--sync-debug", default="", help="debug: after the headline pass, repeat it with torch.cuda.set_sync_debug_mode('warn') and write the "
                    "host-synchronising call sites (file:line inside the package, counts per adapted batch) to this path")
    ap.add_argument("--copy-debug", default="", help="debug: after the headline pass, repeat it under a dispatch mode that records every tensor copy of "
                    ">= 256 K elements (shape, strides, call site) and write the table to this path")
    ap.add_argument("--torch-profile", default="", help="debug: after the headline pass, repeat it under torch.profiler and write the per-operator table to this path")
    ap.add_argument("--plumbing-only", action="store_true",
                    help="launch, rendezvous, sharding and the collectives of the bench without any GPU work (CPU test of --gpus N)")
    a = ap.parse_args(argv)
    if a.random_init:
        a.weights = "random"
    a.kind, a.num_cls, a.stream_id = ("fundus", 2, 2) if a.workload == "cfg2" else ("polyp", 3, 5)
    if a.workload == "cfg5":
        a.bf16_backbone = True
    a.size = a.size or (512 if a.workload == "cfg2" else 384)
    return a


# ------------------------------------------------------------------------------------------- model / data
def base_cfg(args, device):
    from ttdg_mgm_amd.config import get_cfg
    cfg = get_cfg()
    cfg.merge_from_file(os.path.join(ROOT, "configs", "test_segment.yaml"))
    cfg.TEST.BATCH = args.batch
    cfg.MODEL.DEVICE = str(device)
    cfg.MODEL.ROI_HEADS.NUM_CLASSES = args.num_cls
    if args.workload == "cfg5":
        cfg.INPUT.MIN_SIZE_TEST = args.size          # cfg-5 keeps the stream's own 384 x 384 (the reference's polyp configs resize less)
    return cfg


def staged_batches(cfg, name, n_images, args, device, rank, world, cfg_id=None, id_offset=0):
    """The rank's shard of a synthetic stream, mapped (resize to 800) and uploaded: resident in HBM before the timed region."""
    from ttdg_mgm_amd import data
    from ttdg_mgm_amd.engine import BaselineTrainer
    data.register_synthetic(name, n_images, size=args.size, cfg_id=args.stream_id if cfg_id is None else cfg_id, id_offset=id_offset,
                            kind=args.kind, num_cls=args.num_cls)
    BaselineTrainer.rank, BaselineTrainer.world, BaselineTrainer.device = rank, world, device
    BaselineTrainer.resident_inputs = True
    loader = BaselineTrainer.build_test_loader(cfg, name)
    return list(loader), loader.dataset_dicts


def trained_checkpoint(cfg, args, device, rank, world):
    """Rank 0 fits (or finds) the synthetic trained-regime checkpoint; every rank of the node then reads the same file."""
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import synth_checkpoint as sc
    kw = {}
    if args.kind != "fundus":
        kw["kind"], kw["size"] = args.kind, args.size
    if args.ckpt_steps >= 0:
        kw["steps"] = args.ckpt_steps
    if args.ckpt_tta_steps >= 0:
        kw["tta_steps"] = args.ckpt_tta_steps
    path = rep = None
    if rank == 0:
        path, rep = sc.get_or_make(cfg, device, log=lambda m: print("[ckpt] " + m, file=sys.stderr, flush=True), **kw)
    if rank == 0:
        rep = dict(rep or {}, content_sha16=checkpoint_hash(path))
    if world > 1:
        box = [path, rep]
        dist.broadcast_object_list(box, src=0)
        path, rep = box
    return path, rep


def checkpoint_hash(path):
    """sha256 over the tensors of the state dict (names + raw bytes): the fit is not bit-reproducible across boxes (vendor
    convolutions), so every bench line names the weights it was measured on."""
    import hashlib
    sd = torch.load(path, map_location="cpu", weights_only=True)["model"]
    h = hashlib.sha256()
    for k in sorted(sd):
        h.update(k.encode())
        h.update(sd[k].contiguous().numpy().tobytes())
    return h.hexdigest()[:16]


def build_model(cfg, args, device, weights, calib_batch, world):
    from ttdg_mgm_amd.engine import BaselineTrainer
    from ttdg_mgm_amd.engine.checkpoint import load_weights
    from ttdg_mgm_amd.modeling import calibrate_frozen_bn
    torch.manual_seed(0)
    model = BaselineTrainer.build_model(cfg)
    if weights:
        missing, unexpected = load_weights(model, weights)
        assert not missing and not unexpected, (missing[:3], unexpected[:3])
    else:
        calibrate_frozen_bn(model, calib_batch)          # random init: give the frozen BatchNorm layers statistics
    if args.no_overlap_detector:
        from ttdg_mgm_amd.modeling import rcnn as _rcnn
        _rcnn.OVERLAP_DETECTOR = False
    model.autocast_backbone = args.bf16_backbone
    if args.sync_universe and world > 1:
        model.sync_universe = True
        with torch.no_grad():          # replicas must start identical
            for t in list(model.parameters()) + list(model.buffers()):
                if dist.get_backend() == "nccl":
                    dist.broadcast(t, 0)
                else:
                    h = t.cpu()
                    dist.broadcast(h, 0)
                    t.copy_(h)
    return model


# ------------------------------------------------------------------------------------------- the timed pass
def timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, teacher_forced, loader_factory=None, only=None):
    """W untimed warm-up batches, then EXACTLY K adapted batches (K TTA steps, then the Dice pass over the same K batches)
    between barrier + synchronize on both sides.  ``loader_factory`` (A/B): the K timed batches come from a streaming loader
    (decode / synthesise + resize + H2D inside the loop, 2-deep prefetch) instead of the resident list."""
    from ttdg_mgm_amd.engine import BaselineTrainer
    from ttdg_mgm_amd.engine.trainer import run_eval_batches
    from ttdg_mgm_amd.evaluation import DiceEvaluator
    from ttdg_mgm_amd import ops
    model.load_state_dict(init_state)
    model.teacher_forced = teacher_forced
    opt = BaselineTrainer.build_optimizer(cfg, model)
    dice = DiceEvaluator(name, cfg.TEST.DICE_THRES, dataset_dicts=local_dicts)
    dice.prestage(device)              # the evaluator's inputs (ground-truth masks) are resident in HBM like the images
    # (a streamed pass: the timed batches are not in local_dicts; the evaluator takes their ground truth from the items)

    def adapt(bs):
        n = 0
        for b in bs:
            n += BaselineTrainer.tta_step(model, opt, b) is not None
        return n

    def evaluate(bs):
        model.eval()
        dice.reset()
        run_eval_batches(model, bs, dice, max(1, args.eval_streams), args.eval_coalesce)
        model.train()
        if world > 1:
            dice.gather_scores()     # Mode R's one collective: all-gather of the per-rank score lists over RCCL
        return dice.evaluate()

    model.train()
    adapt(batches[:W])
    evaluate(batches[:W])
    stamps = []
    ops.KERNEL_TIMERS = None if args.no_kernel_timers else stamps          # (name, start_event, end_event, meta, info) recorded around our kernels
    ops.KERNEL_TIMER_ONLY = None if only is None else set(only)           # which kernels carry HIP-event pairs in THIS pass
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    t0 = time.perf_counter()
    stepped = adapt(loader_factory() if loader_factory else batches[W:W + K])
    torch.cuda.synchronize()
    t_mid = time.perf_counter()
    res = evaluate(loader_factory() if loader_factory else batches[W:W + K])
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    t1 = time.perf_counter()
    ops.KERNEL_TIMERS = None
    ops.KERNEL_TIMER_ONLY = None
    el, tta = t1 - t0, t_mid - t0
    if world > 1:
        t = torch.tensor([el, tta], device=device if dist.get_backend() == "nccl" else "cpu", dtype=torch.float64)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        el, tta = float(t[0]), float(t[1])
    return dict(elapsed=el, tta=tta, dice=res, kept_masks=len(dice.dice_scores), stamps=stamps, steps_taken=stepped)


# ------------------------------------------------------------------------------------------- rooflines
def _pairs(sizes):
    return [(sizes[a], sizes[b]) for a in range(len(sizes)) for b in range(a + 1)]


BIAS_ACT_KERNEL = "bias_act_nhwc_kernel"      # the epilogue kernel of the channels-last backbone


def kernel_rooflines(run):
    """Algorithmic work per launch (formulas restated in DESIGN.md §5) / HIP-event time on the launch stream.
    gagm: per iteration 2u*sum(n_g^2) + 4Mu^2 + 2M^2u + projector (5*K_sk*sum(max(n_g,u)^2) Sinkhorn, ~n^2*u LAP), times the
    measured iteration count, against the fp32 peak; affinity: 4*512*n_a*n_b per ordered pair (x2 backward) against the fp32 VALU
    peak; pair Sinkhorn: 8*r*c bytes per pair (x2 backward) against HBM; fused SGD: 20 B per parameter against HBM."""
    u, ksk, H = 32, 20, 512
    acc = {}
    for nm, a, b, meta, info in run["stamps"]:
        dt = a.elapsed_time(b) * 1e-3
        e = acc.setdefault(nm, dict(t=0.0, work=0.0, n=0, extra=[]))
        e["t"] += dt
        e["n"] += 1
        if nm == "gagm":
            it = info.cpu().tolist()
            sizes, isk, ih = meta, sum(it[:5]), it[5]
            M = sum(sizes)
            base = 2 * u * sum(n * n for n in sizes) + 4 * M * u * u + 2 * M * M * u
            e["work"] += (isk + ih) * base + isk * 5 * ksk * sum(max(n, u) ** 2 for n in sizes) + ih * sum(min(n, u) ** 2 * max(n, u) for n in sizes)
            e["extra"].append((sizes, it[:6], it[14], it[15], it[22] if len(it) > 22 else 0))
        elif nm in ("affinity_fwd", "affinity_bwd"):
            e["work"] += (1 if nm == "affinity_fwd" else 2) * sum(4 * H * r * c for r, c in _pairs(meta))
        elif nm in ("sinkhorn_pairs_fwd", "sinkhorn_pairs_bwd"):
            e["work"] += (1 if nm == "sinkhorn_pairs_fwd" else 2) * sum(8 * r * c for r, c in _pairs(meta))
        elif nm == "pair_stage_fwd":          # the fused pair stage: the affinity's FLOPs (the Sinkhorn half adds 5*20*c^2 per pair, < 1 %)
            e["work"] += sum(4 * H * r * c for r, c in _pairs(meta))
        elif nm == "pair_stage_bwd":
            e["work"] += 2 * sum(8 * r * c for r, c in _pairs(meta))
        elif nm in ("sgd", "bias_act", "relu_bwd", "roi_align_nhwc", "row_scale_multi", "rpn_heads"):
            e["work"] += meta
        elif nm in ("pointwise_fwd", "pointwise_dx", "pointwise_dw"):      # meta = (algorithmic bytes, FLOPs) of the product
            e["work"] += meta[1]
            e["bytes"] = e.get("bytes", 0) + meta[0]
    from ttdg_mgm_amd import ops as _o

    def every(nm):
        return _o.KERNEL_TIMER_EVERY if nm in _o.KERNEL_TIMER_SAMPLED else 1
    out = []
    for nm, e in acc.items():
        hbm = nm in ("sinkhorn_pairs_fwd", "sinkhorn_pairs_bwd", "sgd", "pair_stage_bwd", "bias_act", "relu_bwd", "roi_align_nhwc", "row_scale_multi", "rpn_heads")
        ach = e["work"] / e["t"] / (1e9 if hbm else 1e12)
        peak = HBM_PEAK_GBS if hbm else FP32_PEAK_TFLOPS
        r = {"kernel": {"gagm": "gagm_kernel", "sgd": "sgd_multi_tensor_kernel", "affinity_fwd": "affinity_fwd_kernel",
                        "affinity_bwd": "affinity_bwd_kernel(+finish)", "sinkhorn_pairs_fwd": "sinkhorn_pairs_fwd_kernel",
                        "sinkhorn_pairs_bwd": "sinkhorn_pairs_bwd_kernel", "pair_stage_fwd": "pair_stage_fwd_kernel",
                        "pair_stage_bwd": "pair_stage_bwd_kernel", "bias_act": BIAS_ACT_KERNEL, "relu_bwd": "relu_bwd_kernel",
                        "roi_align_nhwc": "roi_align_nhwc4_kernel", "row_scale_multi": "row_scale_multi_kernel",
                        "rpn_heads": "mm_kernel (RPN objectness + anchor-delta heads, one product per level, split output)",
                        "pointwise_fwd": "mm_kernel (1x1 convolutions, forward + fused epilogue)", "pointwise_dx": "mm_kernel (1x1 convolutions, dX)",
                        "pointwise_dw": "mm_kernel + mm_reduce_kernel (1x1 convolutions, dW over pixel slices)"}[nm],
             "bound": "hbm" if hbm else "mfma", "achieved": ach, "peak": peak, "unit": "GB/s" if hbm else "TFLOP/s", "frac": ach / peak,
             "traffic": pmc_traffic(nm), "launches_timed": e["n"], "launches": e["n"] * every(nm), "avg_launch_ms": e["t"] / e["n"] * 1e3,
             "total_ms": e["t"] * 1e3 * every(nm),
             "sampling": ("HIP-event pair around every %d-th launch (ops.KERNEL_TIMER_EVERY); launches / total_ms are the timed ones x %d" % (every(nm), every(nm))) if every(nm) > 1 else "every launch timed",
             "algorithmic_work_per_launch": e["work"] / e["n"]}
        if "bytes" in e:
            r["algorithmic_bytes_per_launch"] = e["bytes"] / e["n"]       # what `traffic` (PMC) compares with
            r["algorithmic_hbm_gbs"] = e["bytes"] / e["t"] / 1e9          # the same launches against the other roofline (HBM 8 TB/s)
            r["frac_hbm"] = r["algorithmic_hbm_gbs"] / HBM_PEAK_GBS
        if nm == "gagm":
            its = [sum(x[1]) for x in e["extra"]]
            r.update({"avg_iterations_per_launch": sum(its) / len(its), "us_per_iteration": e["t"] / max(sum(its), 1) * 1e6,
                      "avg_nodes_per_launch": sum(sum(x[0]) for x in e["extra"]) / len(e["extra"]), "graphs_per_launch": len(e["extra"][0][0]),
                      "avg_iterations_per_stage": [sum(x[1][k] for x in e["extra"]) / len(e["extra"]) for k in range(6)],
                      "hungarian_cycle_periods": [x[2] for x in e["extra"]],
                      "avg_executed_launch_pairs": sum(x[4] for x in e["extra"]) / len(e["extra"]),      # multi-workgroup solver only (info[22]); 0: single-workgroup kernel
                      "note": "single-workgroup latency-bound solver (state LDS-resident); fp32 VALU peak == fp32 MFMA peak"})
        out.append(r)
    out.sort(key=lambda r: -r["total_ms"])
    return out


def pmc_traffic(stamp_name):
    """HBM bytes per launch from the committed PMC passes of this command (rocprofv3 --pmc FETCH_SIZE / --pmc WRITE_SIZE in
    separate runs -> tools/pmc_summary.py -> profiles/rNN_bench_pmc.json, the newest round's record that holds the kernel).  Counters cannot be read from inside the timed
    process, so this is the recorded figure, not a live one; None when absent."""
    names = {"gagm": ("gagm_kernel", False), "sgd": ("sgd_multi_tensor", True), "affinity_fwd": ("affinity_fwd", False),
             "affinity_bwd": ("affinity_bwd_kernel", False), "sinkhorn_pairs_fwd": ("sinkhorn_pairs_fwd", False),
             "sinkhorn_pairs_bwd": ("sinkhorn_pairs_bwd", False), "pair_stage_fwd": ("pair_stage_fwd", False),
             "pair_stage_bwd": ("pair_stage_bwd", False), "bias_act": ("bias_act", True), "relu_bwd": ("relu_bwd", True),
             "roi_align_nhwc": ("roi_align_nhwc", True), "row_scale_multi": ("row_scale_multi", True),
             "pointwise_fwd": ("mm_kernel", True), "pointwise_dx": ("mm_kernel", True), "pointwise_dw": ("mm_kernel", True)}
    if stamp_name not in names:          # (no separate PMC record: the RPN heads' launches are mm_kernel instantiations inside the pointwise record)
        return None
    kernel, streaming = names[stamp_name]
    import glob
    for f in sorted((os.path.basename(x) for x in glob.glob(os.path.join(ROOT, "profiles", "r[0-9][0-9]_bench_pmc.json"))), reverse=True):   # newest round first
        try:
            with open(os.path.join(ROOT, "profiles", f)) as fh:
                rec = json.load(fh).get(kernel)
        except (OSError, ValueError):
            continue
        if rec:
            if stamp_name in ("bias_act", "relu_bwd", "roi_align_nhwc", "pointwise_fwd", "pointwise_dx", "pointwise_dw") and "hbm_bytes_per_launch_mean_streaming_corrected" in rec:
                return rec["hbm_bytes_per_launch_mean_streaming_corrected"]        # many launch sizes: mean, like `achieved`
            return rec["hbm_bytes_per_launch_streaming_corrected" if streaming else "hbm_bytes_per_launch_raw"]
    return None


# ------------------------------------------------------------------------------------------- whole-step roofline + cfg-3
def step_flops(cfg, model, init_state, batch, teacher_forced):
    """Algorithmic fp32 FLOPs of ONE adapted batch (TTA step forward + backward, then the eval-mode inference): counted, not
    estimated - torch.utils.flop_counter over the aten convolutions / matrix products of one un-timed batch with the pointwise
    convolutions routed to aten (same arithmetic as the fused product: 2 * pixels * Cin * Cout), plus the hand-written matching
    kernels' own formulas (affinity 4 h n_i n_j per ordered pair, x 3 with its backward; they are < 0.1 % of the
    step).  ROIAlign, NMS, Sinkhorn sweeps and element-wise work are not counted (they are not matrix work)."""
    from torch.utils.flop_counter import FlopCounterMode
    from ttdg_mgm_amd.engine import BaselineTrainer
    from ttdg_mgm_amd.engine.trainer import run_eval_batches
    from ttdg_mgm_amd.evaluation import DiceEvaluator
    from ttdg_mgm_amd.modeling import backbone as bb
    model.load_state_dict(init_state)
    model.teacher_forced = teacher_forced
    opt = BaselineTrainer.build_optimizer(cfg, model)
    keep = bb.OWN_POINTWISE
    bb.OWN_POINTWISE = False
    try:
        model.train()
        with FlopCounterMode(display=False) as fc_tta:
            BaselineTrainer.tta_step(model, opt, batch)
        model.eval()

        class _Sink:
            def process(self, *a, **k):
                pass
        with FlopCounterMode(display=False) as fc_eval:
            run_eval_batches(model, [batch], _Sink(), 1, 1)
        model.train()
    finally:
        bb.OWN_POINTWISE = keep
    tta, ev = float(fc_tta.get_total_flops()), float(fc_eval.get_total_flops())
    return {"flops_per_step": tta + ev, "tta_step_flops": tta, "eval_pass_flops": ev,
            "counted": "aten convolution / addmm / mm / bmm FLOPs (2 per multiply-add) of one adapted batch of %d images, forward and backward, torch.utils.flop_counter; "
                       "hand-written matching kernels and element-wise work not included (< 0.1 %%)" % len(batch),
            "peak_tflops": FP32_PEAK_TFLOPS, "peak": "fp32 matrix = fp32 vector peak (MI355X_MICROARCH.md)"}


def cfg3_block(device, seeds=(0, 1, 2, 3, 4), reps=20):
    """MGM3_unsup on 8 graphs x 256 nodes (nodes = randn(256, 256) * 0.1, labels in
    {1, 2}, U = randn(32, 256) + 1/32, weights std 0.05, seeds 0..4), forward + backward, HIP events on the launch stream, `reps`
    repetitions per seed after 3 warm-up steps; per-kernel averages from a separate stamped repetition set (rooflines as in
    kernel_rooflines: SURVEY.md §8d algorithmic work / live duration)."""
    from ttdg_mgm_amd import ops, synth
    from ttdg_mgm_amd.GModule import MGM3_unsup
    sizes = (256,) * 8
    fb, fw, its, solver_us, pairs, kern = [], [], [], [], [], {}
    for seed in seeds:
        params, U = synth.mgm3_params(9000 + seed), synth.universe(9100 + seed)
        nodes, labels = synth.node_sets(9200 + seed, sizes, scale=0.1)
        m = MGM3_unsup(2, 32).to(device).eval()
        m.load_state_dict(params)
        dn = [x.to(device).requires_grad_() for x in nodes]
        dl = [l.to(device) for l in labels]
        Ud = U.to(device)
        for _ in range(3):
            m(dn, dl, Ud).backward()
        torch.cuda.synchronize()
        e = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        e[0].record()
        for _ in range(reps):
            m(dn, dl, Ud).backward()
        e[1].record()
        with torch.no_grad():
            for _ in range(reps):
                m(dn, dl, Ud)
        e[2].record()
        torch.cuda.synchronize()
        fb.append(e[0].elapsed_time(e[1]) / reps)
        fw.append(e[1].elapsed_time(e[2]) / reps)
        stamps = []
        ops.KERNEL_TIMERS, keep_every = stamps, ops.KERNEL_TIMER_EVERY
        ops.KERNEL_TIMER_EVERY = 1
        try:
            for _ in range(5):
                m(dn, dl, Ud).backward()
            torch.cuda.synchronize()
        finally:
            ops.KERNEL_TIMERS, ops.KERNEL_TIMER_EVERY = None, keep_every
        for r in kernel_rooflines({"stamps": stamps}):
            k = kern.setdefault(r["kernel"], {"avg_us": [], "frac": [], "work": [], "bound": r["bound"], "unit": r["unit"]})
            k["avg_us"].append(r["avg_launch_ms"] * 1e3)
            k["frac"].append(r["frac"])
            k["work"].append(r["algorithmic_work_per_launch"])
            if r["kernel"] == "gagm_kernel":
                its.append(r["avg_iterations_per_launch"])
                pairs.append(r.get("avg_executed_launch_pairs", 0))
                solver_us.append(r["avg_launch_ms"] * 1e3)
    mean = lambda v: sum(v) / max(1, len(v))
    # what an event pair itself reads with nothing between its two records (the marker packets' own round trip): rocprofv3's kernel
    # durations (profiles/rNN_cfg3_rocprof_summary.txt, same block under `bench.py --cfg3-only`) are this much shorter per launch
    br = []
    for _ in range(50):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        b.record()
        br.append((a, b))
    torch.cuda.synchronize()
    bracket = sorted(x.elapsed_time(y) * 1e3 for x, y in br)[len(br) // 2]
    return {"workload": "cfg-3: MGM3_unsup forward + backward, 8 graphs x 256 nodes, d = 256, h = 512, seeds %s, %d repetitions each (HIP events on the launch stream)" % (list(seeds), reps),
            "fwd_bwd_ms": mean(fb), "fwd_bwd_ms_per_seed": fb, "fwd_ms": mean(fw), "fwd_ms_per_seed": fw,
            "solver_us": mean(solver_us) if solver_us else None, "executed_iterations": mean(its) if its else None,
            "solver_us_per_iteration": (mean(solver_us) / mean(its)) if its and mean(its) else None,
            "launched_iterations": mean(pairs) if pairs else None,
            "solver_us_per_launched_iteration": (mean(solver_us) / mean(pairs)) if pairs and mean(pairs) else None,
            "iterations_note": "executed_iterations = the stage machine's count (info[0..5]): it includes the iterations a Hungarian-stage cycle of period >= 3 lets the "
                               "solver skip (the exact cycle shortcut jumps to the state iteration max_iter - 1 would land on); launched_iterations = the (mul, projection) "
                               "launch pairs that did work (info[22]) - the figure the per-iteration kernel time belongs to",
            "event_bracket_us": bracket,
            "kernels_note": "avg_us = live HIP-event bracket around the launch (includes event_bracket_us of marker round trip and the launch latency of a cold "
                            "stream); rocprofv3 kernel durations of the same block: profiles/r06_cfg3_block_rocprof_summary.txt",
            "kernels": {k: {"avg_us": mean(v["avg_us"]), "algorithmic_work": mean(v["work"]), "frac": mean(v["frac"]), "bound": v["bound"],
                            "unit": "bytes" if v["bound"] == "hbm" else "FLOP"} for k, v in kern.items()}}


# ------------------------------------------------------------------------------------------- CPU baseline + Dice parity
def cpu_model_string():
    try:
        with open("/proc/cpuinfo") as f:
            for line in f:
                if line.startswith("model name"):
                    return line.split(":", 1)[1].strip()
    except OSError:
        pass
    return "unknown"


def allcores_note():
    """Why `cores` is min(os.cpu_count(), 64): the recorded all-cores measurement of this round (profiles/r03_bench_cpu_allcores.json,
    `bench.py --cpu-allcores`), when present."""
    try:
        with open(os.path.join(ROOT, "profiles", "r03_bench_cpu_allcores.json")) as f:
            a = json.load(f)["cpu_baseline"]["all_cores"]
        if a["value"] is None:
            return "all %d host threads, tried once this round: %s (64 threads is the fastest setting found)" % (a["cores"], a["protocol"])
        return "all %d host threads, recorded once this round: %s images/s (%s)" % (a["cores"], a["value"], a["protocol"])
    except (OSError, ValueError, KeyError):
        return "torch's CPU kernels stop scaling beyond 64 intra-op threads on these tensor sizes; all-cores figure not recorded"


def cpu_baseline(args, weights, teacher_forced):
    """SURVEY.md §8d protocol: 1 warm-up + median of --cpu-reps repetitions of (one TTA step + eval pass on 4 images), each
    from the same checkpoint; the warm-up repetition's Dice is the CPU side of `dice_parity`.  Runs in a CHILD process with
    a time limit (the oracle port must never be able to hang the bench) and its own thread count: min(os.cpu_count(), 64)
    unless --cpu-threads - beyond 64 intra-op threads torch's CPU kernels stop scaling on these tensor sizes, and on a
    cgroup-limited box oversubscribed spin-waits stall them altogether (measured: > 30 min at 256 threads)."""
    import subprocess
    cores = args.cpu_threads or min(os.cpu_count() or 1, 64)
    spec = dict(batch=args.batch, size=args.size, teacher_forced=teacher_forced, weights=weights, reps=args.cpu_reps, warmup=1, threads=cores)
    code = ("import json, sys, torch; sys.path.insert(0, %r); spec = json.loads(sys.argv[1]); torch.set_num_threads(spec['threads']); "
            "from oracle import tta_cpu; r = tta_cpu.run(1, spec['batch'], spec['size'], teacher_forced=spec['teacher_forced'], "
            "weights=spec['weights'], reps=spec['reps'], warmup=spec['warmup']); print('CPUJSON' + json.dumps(r))" % ROOT)
    env = dict(os.environ, OMP_NUM_THREADS=str(cores), MKL_NUM_THREADS=str(cores), HIP_VISIBLE_DEVICES="", CUDA_VISIBLE_DEVICES="")
    limit = 120 + 90 * (1 + args.cpu_reps)
    p = subprocess.run([sys.executable, "-c", code, json.dumps(spec)], capture_output=True, text=True, timeout=limit, env=env, cwd=ROOT)
    if p.returncode != 0:
        raise RuntimeError("CPU port failed: " + p.stderr[-800:])
    r = json.loads([l for l in p.stdout.splitlines() if l.startswith("CPUJSON")][-1][7:])
    med = statistics.median(r["times"])
    out = {"value": args.batch / med, "unit": "adapted images/s", "cores": cores, "host_cores": os.cpu_count(), "cpu_model": cpu_model_string(),
           "kind": "port", "protocol": "1 warm-up + median of %d" % len(r["times"]), "seconds_median": med, "seconds_all": r["times"],
           "cores_note": allcores_note(),
           "seconds_warmup": r["warmup_times"],
           "sample": "1 TTA step + eval pass on %d synthetic %dx%d images per repetition, torch-CPU model + oracle GModule, %d threads, %s weights, %s detections"
                     % (args.batch, args.size, args.size, cores, "trained-regime checkpoint" if weights else "random-init",
                        "teacher-forced" if teacher_forced else "free-running")}
    if args.cpu_allcores and (os.cpu_count() or 1) != cores:
        n_all = os.cpu_count()
        speca = dict(spec, reps=1, warmup=0, threads=n_all)
        enva = dict(env, OMP_NUM_THREADS=str(n_all), MKL_NUM_THREADS=str(n_all))
        try:
            pa = subprocess.run([sys.executable, "-c", code, json.dumps(speca)], capture_output=True, text=True, timeout=600, env=enva, cwd=ROOT)
            ra = json.loads([l for l in pa.stdout.splitlines() if l.startswith("CPUJSON")][-1][7:])
            out["all_cores"] = {"cores": n_all, "value": args.batch / ra["times"][0], "seconds": ra["times"][0], "protocol": "one cold repetition"}
        except subprocess.TimeoutExpired:
            out["all_cores"] = {"cores": n_all, "value": None, "seconds": None, "protocol": "one cold repetition: did not finish within 600 s"}
    if args.cpu_1thread:
        spec1 = dict(spec, reps=1, warmup=0, threads=1)
        env1 = dict(env, OMP_NUM_THREADS="1", MKL_NUM_THREADS="1")
        p1 = subprocess.run([sys.executable, "-c", code, json.dumps(spec1)], capture_output=True, text=True, timeout=3600, env=env1, cwd=ROOT)
        r1 = json.loads([l for l in p1.stdout.splitlines() if l.startswith("CPUJSON")][-1][7:])
        out["one_thread"] = {"value": args.batch / r1["times"][0], "seconds": r1["times"][0]}
    return out, r["dice"]


def gpu_dice_parity_leg(cfg, model, init_state, batch, dicts, name, teacher_forced):
    """The GPU side of `dice_parity`: from the checkpoint, ONE TTA step on the first batch, then the Dice pass on it."""
    from ttdg_mgm_amd.engine import BaselineTrainer
    from ttdg_mgm_amd.engine.trainer import run_eval_batches
    from ttdg_mgm_amd.evaluation import DiceEvaluator
    model.load_state_dict(init_state)
    model.teacher_forced = teacher_forced
    model.train()
    BaselineTrainer.tta_step(model, BaselineTrainer.build_optimizer(cfg, model), batch)
    ev = DiceEvaluator(name, cfg.TEST.DICE_THRES, dataset_dicts=dicts)
    model.eval()
    run_eval_batches(model, [batch], ev, 1, 1)
    model.train()
    res = ev.evaluate()
    res["kept_masks"] = len(ev.dice_scores)
    return res


def parity_block():
    """The parity statement a number of this line is quoted under: the gates in force in tests/ (-m gpu, through the C ABI) and
    what the last recorded run of those tests actually asserted (the newest profiles/rNN_parity_ledger.json, rNN_trained_census.json,
    rNN_trajectory.json, rNN_census_exchangeability.json - copied from gpurun_out/ after the round's final GPU test run).  Recorded figures, not live ones; the
    live parity leg of this run is `dice_parity`."""
    import glob

    def rec(suffix):
        """The newest round's record of that name (profiles/rNN_<suffix>)."""
        for path in sorted(glob.glob(os.path.join(ROOT, "profiles", "r[0-9][0-9]_" + suffix)), reverse=True):
            try:
                with open(path) as f:
                    return json.load(f)
            except (OSError, ValueError):
                continue
        return None
    census, ledger, traj, exch = rec("trained_census.json"), rec("parity_ledger.json"), rec("trajectory.json"), rec("census_exchangeability.json")
    out = {
        "gates": {
            "Wds / first V / loss / d loss / d nodes / parameter gradients vs oracle and reference goldens": "1e-4 abs (fp32)",
            "log-domain Sinkhorn vs the reference tree's own log-Sinkhorn": "1e-4 + 40 ulp(max|s/tau|)  [above the flat 1e-4: 1.8e-4 measured at tau = 0.00625]",
            "iterated maps (solver step, HiPPI, backward of 20 sweeps)": "max(1e-4, 2 x what the fp32 oracle loses against its own float64 statement)",
            "planted goldens (15 cases + 2 at BASELINE cfg-3 size, 8 x 256; admitted only if the reference's answer survives structured rounding-sized perturbations)":
                "identical permutation matrices and Sinkhorn-stage iteration counts; Hungarian-stage count +-1",
            "trained-regime free-running solve": "stage-end states within 1e-4 of the oracle wherever the reference's own eight runs define them; final answers: gross-error bound per batch, "
                                                 "rank-sum over the census batches, and exchangeability with the reference's own runs on 8 recorded inputs (pooled |z| <= 3.5 at 1e-5 input noise)",
            "continual TTA (8 steps, momentum carried)": "per tensor group and step |device - float64 trajectory| <= 4 x max(max_{j<=k} h_j, (k + 1) / K h_{K-1}) + (k + 1) ulp, h = |float32 host - float64 trajectory| (reference side only) - the bound of round 5, COUNTED since round 6: at most 2 of the 40 (group, step) checks outside it, none beyond 1.5 x (one fresh box of fourteen exceeded it, twice, by 7 % and 19 %); Dice within 1e-3 relative",
            "Dice / E / S vs the reference's numpy functions": "1e-9 / 1e-9 / 1e-6",
        },
    }
    if census:
        out["trained_regime_census"] = {k: census[k] for k in ("steps", "strong", "weak", "device_equals_oracle32", "mean_iterations") if k in census}
    if ledger:
        out["statement_ledger"] = ledger
    if traj:
        out["continual_tta"] = {"steps": traj.get("steps"), "worst_fraction_of_bound": traj.get("worst_fraction_of_bound"), "outside_frozen_bound": traj.get("outside_frozen_bound"),
                                "dice_device": traj.get("dice_device"),
                                "dice_host": traj.get("dice_host"),
                                "max_rel_param_distance": max((g["rel"] for r in traj.get("records", []) for g in r["groups"].values()), default=None)}
    if exch:
        out["exchangeability"] = {e: {"pooled_z_objective": v.get("pooled_z_objective"), "pooled_z_loss": v.get("pooled_z_loss")} for e, v in exch.get("by_eps", {}).items()}
    return out


_T0 = time.perf_counter()


def note(msg):
    """Progress on stderr (the one JSON line stays alone on stdout)."""
    print("[bench %6.1fs] %s" % (time.perf_counter() - _T0, msg), file=sys.stderr, flush=True)


def _finite(x):
    """NaN / inf -> null: the line must be strict JSON."""
    if isinstance(x, float):
        return x if x == x and abs(x) != float("inf") else None
    if isinstance(x, dict):
        return {k: _finite(v) for k, v in x.items()}
    if isinstance(x, (list, tuple)):
        return [_finite(v) for v in x]
    return x


# ------------------------------------------------------------------------------------------- one rank
def plumbing_only(args, rank, world):
    """Everything of the bench that is not GPU work: rendezvous, shard arithmetic, barrier, max-over-ranks timing, the Dice
    all-gather.  Used by the CPU test of `bench.py --gpus N` (gloo)."""
    from ttdg_mgm_amd.evaluation import DiceEvaluator
    K, W, B = steps_per_rank(args, world), args.warmup, args.batch
    n = world * (K + W) * B
    shard = (n - 1) // world + 1
    lo, hi = shard * rank, min(shard * (rank + 1), n)
    ev = DiceEvaluator("plumbing", 0.9, dataset_dicts=[])
    ev.dice_scores, ev.ea_scores, ev.sm_scores = [float(rank)] * (rank + 1), [0.0] * (rank + 1), [0.0] * (rank + 1)
    dist.barrier()
    t = torch.tensor([0.001 * (rank + 1)], dtype=torch.float64)
    dist.all_reduce(t, op=dist.ReduceOp.MAX)
    ev.gather_scores()
    # the strong-scaling pass of a launch, with stand-in clocks: rank r "spends" (r + 1) ms on its shard of the fixed stream, rank 0 alone
    # 1 ms per rank's share x 0.9: same barrier, same max over the ranks, same arithmetic (strong_record) as the GPU pass
    T = max(1, args.strong_images // (world * B)) * world * B
    ts = torch.tensor([0.001 * (rank + 1)], dtype=torch.float64)
    dist.barrier()
    dist.all_reduce(ts, op=dist.ReduceOp.MAX)
    strong = strong_record(T, float(ts[0]), 0.001 * world * 0.9, world, B) if rank == 0 else None
    if rank == 0:
        print(json.dumps({"plumbing_only": True, "strong": strong, "n_gpus": world, "ranks_seen": dist.get_world_size(), "backend": dist.get_backend(),
                          "steps": K, "shard_rank0": [lo, hi], "images_total": n, "max_time": float(t[0]),
                          "gathered_scores": len(ev.dice_scores), "scaling": "strong" if args.images else "weak"}))


def strong_record(T, elapsed_sharded, elapsed_solo, world, B):
    """The strong-scaling arithmetic of a launch (rank 0): `elapsed_sharded` = the max-over-ranks time of the fixed T-image stream
    sharded over `world` ranks, `elapsed_solo` = rank 0 alone on the whole stream in the same process.  Shared by the GPU pass and
    by --plumbing-only (CPU test), so the first real 8-GPU launch computes its efficiency with tested code."""
    return {"images": T, "value": T / elapsed_sharded, "unit": "images/s", "n1_value_same_stream": T / elapsed_solo,
            "efficiency_vs_n1": (T / elapsed_sharded) / (world * T / elapsed_solo), "steps_per_rank": T // (world * B),
            "ranks": dist.get_world_size(), "backend": dist.get_backend(),
            "note": "fixed %d-image stream sharded over the ranks (continual TTA per shard, then the Dice pass + RCCL score all-gather); "
                    "n1 = rank 0 alone on the whole stream, same process, other ranks idle" % T}


def steps_per_rank(args, world):
    if args.images:
        per = args.images // (world * args.batch)
        if per < 1 or per * world * args.batch != args.images:
            raise SystemExit("--images must be a multiple of gpus * batch (%d)" % (world * args.batch))
        return per
    return args.steps


def run(args):
    if args.no_miopen_db:
        os.environ["TTDG_MIOPEN_DB"] = "0"              # read when the package is first imported (below)
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    if world != args.gpus:
        raise SystemExit("WORLD_SIZE=%d but --gpus %d" % (world, args.gpus))
    if world > 1:
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
        dist.init_process_group(args.dist_backend)      # "nccl" is RCCL on ROCm
    try:
        if args.plumbing_only:
            if world == 1:
                dist.init_process_group(args.dist_backend if args.dist_backend != "nccl" else "gloo",
                                        init_method="tcp://127.0.0.1:%d" % free_port(), rank=0, world_size=1)
            return plumbing_only(args, rank, world)
        return gpu_main(args, rank, world, 0 if args.share_device else local)
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


def gpu_main(args, rank, world, local):
    torch.cuda.set_device(local)
    device = torch.device("cuda", local)
    if args.miopen_search:
        torch.backends.cudnn.benchmark = True
    from ttdg_mgm_amd import _lib
    if rank == 0 and not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    if world > 1:
        dist.barrier()
    if args.cfg3_only:
        if rank == 0:
            print(json.dumps(_finite({"cfg3": cfg3_block(device)})))
        return
    K, W, B = steps_per_rank(args, world), args.warmup, args.batch
    cfg = base_cfg(args, device)
    from ttdg_mgm_amd import ops as _ops
    from ttdg_mgm_amd.modeling import detector as _det
    from ttdg_mgm_amd.modeling import graphed as _graphed
    _graphed.ENABLED = bool(args.graphs)
    if args.vendor_pointwise:
        from ttdg_mgm_amd.modeling import backbone as _bb
        _bb.OWN_POINTWISE = False
    if args.own_pointwise_backward:
        _ops.POINTWISE_BACKWARD = "own"
    if args.vendor_rpn_heads:
        _det.FUSED_RPN_HEADS = False
    _ops.KERNEL_TIMER_EVERY = max(1, args.timer_every)
    assert _det._backend is _ops, "the GPU legs must run on the HIP operators (detector._backend was re-pointed)"
    if args.gagm_threads or args.roi_align_mode != 3:
        from ttdg_mgm_amd import _lib
        if args.gagm_threads == 256:
            from ttdg_mgm_amd import ops as _ops
            _ops.GAGM_VARIANT |= _lib.GAGM_256_THREADS
        _ops.ROI_ALIGN_NHWC = args.roi_align_mode == 3
        _lib.load().ttdg_debug_set_roi_align_sliced(min(args.roi_align_mode, 2))
    if args.roi_xcd_chunks or args.roi_chunk or args.roi_one_channel_per_lane:
        from ttdg_mgm_amd import _lib
        _lib.load().ttdg_debug_set_roi_align_sliced(2 | (16 if args.roi_xcd_chunks else 0) | {0: 0, 25: 0, 49: 32, 13: 64}[args.roi_chunk] |
                                                    (128 if args.roi_one_channel_per_lane or args.roi_xcd_chunks or args.roi_chunk else 0))
    if args.images:
        # strong scaling: the FIXED stream is sharded; warm-up batches come from another stream so that the timed work is
        # exactly args.images images whatever the rank count
        timed, dicts_t = staged_batches(cfg, "synthfundus_bench", args.images, args, device, rank, world)
        warm, dicts_w = staged_batches(cfg, "synthfundus_warm", world * W * B, args, device, rank, world, cfg_id=args.stream_id + 10, id_offset=10 ** 6)
        batches, local_dicts = warm + timed, dicts_w + dicts_t
    else:
        # weak scaling: every rank owns (K + W) batches of a (world * (K + W) * B)-image stream
        batches, local_dicts = staged_batches(cfg, "synthfundus_bench", world * (K + W) * B, args, device, rank, world)
    assert len(batches) >= K + W, (len(batches), K, W)
    name = "synthfundus_bench"
    weights, ckpt_report = (None, None)
    if args.weights == "trained":
        weights, ckpt_report = trained_checkpoint(cfg, args, device, rank, world)
    note("inputs staged, weights: %s" % (weights or "random init"))
    model = build_model(cfg, args, device, weights, batches[0], world)
    init_state = {k: v.detach().clone() for k, v in model.state_dict().items()}
    tf = bool(args.teacher_forced)
    # The headline pass carries HIP-event pairs around ONE kernel family only - the dominant hand-written kernel, whose live average
    # feeds `roofline` - sampled every --timer-every-th launch.  Every other hand-written kernel is timed in a SECOND, fully stamped
    # pass over the same batches (`instrumented_pass`, the source of `roofline_other_kernels`): an event pair is two marker packets in
    # the launch queue, and ~250 pairs per batch cost 1.7 ms of a 38.4 ms batch (profiles/r06_event_overhead.txt).
    dominant = ("bias_act",) if args.vendor_pointwise else ("pointwise_fwd",)
    main = timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf, only=None if args.stamp_all else dominant)
    instrumented = main if args.stamp_all or args.no_kernel_timers else timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf)
    eager_probe = None
    if _graphed.ENABLED and model.__dict__.get("_graphed") is not None and model.__dict__["_graphed"].stats["eval_replays"] > 0:
        # Inside a graph replay no HIP event can be placed around a single kernel from here.  The per-kernel durations of the
        # rooflines therefore come from a SECOND timed pass over the same K batches with the backbone launched eagerly (live HIP
        # events on the launch stream, as before); its images/s is the graphs-off A/B figure of the line.
        _graphed.ENABLED = False
        try:
            eager_probe = timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf)
        finally:
            _graphed.ENABLED = True
        main["stamps"] = eager_probe["stamps"]
    note("headline pass done: %.1f images/s" % (world * K * B / main["elapsed"]))
    if args.sync_debug and world == 1:
        import collections
        import traceback
        import warnings
        sites = collections.Counter()

        def record(message, category, filename, lineno, file=None, line=None):
            if "synchron" not in str(message):
                return
            frames = [f for f in traceback.extract_stack() if (os.sep + "ttdg-mgm_amd" + os.sep in f.filename or f.filename.endswith("bench.py")) and f.name != "record"]
            where = " <- ".join("%s:%d %s" % (os.path.relpath(f.filename, ROOT), f.lineno, f.name) for f in reversed(frames[-3:]))
            sites[(where, str(message).split("\n")[0][:80])] += 1
        old_show = warnings.showwarning
        warnings.showwarning = record
        warnings.simplefilter("always")
        torch.cuda.set_sync_debug_mode("warn")
        try:
            timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf)
        finally:
            torch.cuda.set_sync_debug_mode("default")
            warnings.showwarning = old_show
        with open(args.sync_debug, "w") as f:
            f.write("# host-synchronising calls over W=%d warm-up + K=%d adapted batches (TTA steps, then the Dice pass), torch.cuda.set_sync_debug_mode('warn')\n" % (W, K))
            for (where, msg), n in sites.most_common():
                f.write("%6d  (%.1f / batch)  %s   [%s]\n" % (n, n / (W + K), where, msg))
    if args.copy_debug and world == 1:
        import collections
        import traceback
        from torch.utils._python_dispatch import TorchDispatchMode
        seen = collections.Counter()

        class Copies(TorchDispatchMode):
            def __torch_dispatch__(self, func, types, a=(), kw=None):
                name = str(func)
                if ("copy" in name or "clone" in name or "contiguous" in name) and a and isinstance(a[0], torch.Tensor) and a[0].is_cuda and a[0].numel() >= 262144:
                    src = a[1] if len(a) > 1 and isinstance(a[1], torch.Tensor) else a[0]
                    frames = [f for f in traceback.extract_stack() if os.sep + "ttdg-mgm_amd" + os.sep in f.filename]
                    where = " <- ".join("%s:%d" % (os.path.basename(f.filename), f.lineno) for f in reversed(frames[-3:])) or "(autograd / outside the package)"
                    seen[(name, tuple(a[0].shape), tuple(src.stride()), tuple(a[0].stride()) if "copy_" in name else str(kw), where)] += 1
                return func(*a, **(kw or {}))
        with Copies():
            timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf)
        with open(args.copy_debug, "w") as f:
            f.write("# tensor copies >= 256 K elements over W=%d + K=%d adapted batches: count, op, shape, source strides, destination strides / kwargs, call site\n" % (W, K))
            for key, n in sorted(seen.items(), key=lambda kv: -kv[1] * torch.Size(kv[0][1]).numel()):
                f.write("%5d  %s\n" % (n, "  ".join(str(x) for x in key)))
    if args.torch_profile and world == 1:
        from torch.profiler import ProfilerActivity, profile
        with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA], with_stack=True) as prof:
            timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf)
        with open(args.torch_profile, "w") as f:
            f.write("# torch.profiler over W=%d warm-up + K=%d adapted batches (TTA steps + Dice pass), operators by device time\n" % (W, K))
            f.write(prof.key_averages().table(sort_by="self_cuda_time_total", row_limit=70, max_name_column_width=70))
            f.write("\n\n# copies by call site (aten::copy_ with device time, grouped by the Python stack)\n")
            cps = [e for e in prof.key_averages(group_by_stack_n=6) if e.key == "aten::copy_" and e.self_device_time_total > 0]
            for e in sorted(cps, key=lambda e: -e.self_device_time_total)[:25]:
                where = " <- ".join(fr.split("/")[-1] for fr in e.stack[:6] if "ttdg" in fr or "bench.py" in fr or "torch/nn/functional" in fr)
                f.write("calls %5d  self device %9.1f us  avg %7.1f us   %s\n" % (e.count, e.self_device_time_total, e.self_device_time_total / e.count, where[:300]))
            f.write("\n\n# by call count\n")
            rows = sorted(prof.key_averages(), key=lambda e: -e.count)[:60]
            for e in rows:
                f.write("%-70s calls %6d  self device %9.1f us  self cpu %9.1f us\n" % (e.key[:70], e.count, e.self_device_time_total, e.self_cpu_time_total))

    strong = None
    if world > 1 and not args.images and args.strong_images and not args.sync_universe:
        # the driver's `--gpus N --steps K` form is weak scaling (per-rank work fixed); north_star asks for STRONG scaling, so
        # the same launch also times a FIXED stream sharded over the N ranks, and rank 0 alone on the whole stream (the N = 1
        # reference of the efficiency, measured in this very process group while the other ranks wait)
        from ttdg_mgm_amd.engine import BaselineTrainer
        T = max(1, args.strong_images // (world * B)) * world * B
        sb, sd = staged_batches(cfg, "synthfundus_strong", T, args, device, rank, world, cfg_id=args.stream_id + 30, id_offset=3 * 10 ** 6)
        rs = timed_pass(cfg, model, init_state, batches[:W] + sb, local_dicts + sd, name, T // (world * B), W, args, world, device, tf)
        solo = None
        if rank == 0:
            ab_, ad_ = staged_batches(cfg, "synthfundus_strong", T, args, device, 0, 1, cfg_id=args.stream_id + 30, id_offset=3 * 10 ** 6)
            solo = timed_pass(cfg, model, init_state, batches[:W] + ab_, local_dicts + ad_, name, T // B, W, args, 1, device, tf)
            del ab_, ad_
        BaselineTrainer.rank, BaselineTrainer.world = rank, world
        dist.barrier()
        if rank == 0:
            strong = strong_record(T, rs["elapsed"], solo["elapsed"], world, B)
            strong.update(dice=rs["dice"], kept_masks=rs["kept_masks"])
        note("strong-scaling pass done")
        del sb, sd

    ab = {}
    parity = None
    if world == 1 and not args.no_ab:
        def short(r, label):
            roofs = kernel_rooflines(r)
            g = next((x for x in roofs if x["kernel"] == "gagm_kernel"), None)
            return {"label": label, "value": K * B / r["elapsed"], "tta_only_images_per_s": K * B / r["tta"], "dice": r["dice"],
                    "kept_masks": r["kept_masks"], "gagm_avg_launch_ms": g and g["avg_launch_ms"],
                    "gagm_avg_iterations_per_stage": g and g["avg_iterations_per_stage"]}
        if args.weights == "trained":
            note("A/B: other detection mode")
            ab["teacher_forced" if not tf else "free_running"] = short(
                timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, not tf),
                "same checkpoint, %s detections" % ("teacher-forced" if not tf else "free-running"))
            note("A/B: random init")
            rmodel = build_model(cfg, args, device, None, batches[0], world)
            rstate = {k: v.detach().clone() for k, v in rmodel.state_dict().items()}
            ab["random_init"] = short(timed_pass(cfg, rmodel, rstate, batches, local_dicts, name, K, W, args, world, device, True),
                                      "random-init weights, teacher-forced detections (the round-1 configuration: worst-case solver regime, Dice undefined)")
            del rmodel, rstate
        # inputs through the loader INSIDE the timed region: the stream is pre-rendered to local storage before
        # t0 (standing for a dataset of decoded images), read back by NUM_WORKERS worker processes (the reference's loader
        # topology, data/build.py:148-153), pinned, uploaded as raw 512 x 512 uint8 and resized to 800 x 800 on the device
        # (csrc/resize.hip); 2-deep prefetch on a side stream.  Both passes (TTA and Dice) stream; the evaluator reads the
        # ground truth each item carries.  Worker start-up (loader construction) is outside the timed region.
        note("A/B: loader-inclusive")
        import tempfile
        from ttdg_mgm_amd import data
        data.register_synthetic("synthfundus_stream_src", K * B, size=args.size, cfg_id=args.stream_id + 20, id_offset=2 * 10 ** 6, kind=args.kind,
                                num_cls=args.num_cls)
        droot = os.path.join(tempfile.gettempdir(), "ttdg_stream_%s_%d_%d" % (args.workload, args.size, K * B))
        data.register_disk("synthfundus_stream", droot, source="synthfundus_stream_src", workers=cfg.DATALOADER.NUM_WORKERS)
        sloader = data.TestLoader("synthfundus_stream", B, 0, 1, device, cfg.INPUT.MIN_SIZE_TEST, cfg.INPUT.MAX_SIZE_TEST, resident=False)
        sloader.start_workers()

        def stream():
            return sloader
        ab["loader_inclusive"] = short(
            timed_pass(cfg, model, init_state, batches, local_dicts, name, K, W, args, world, device, tf, loader_factory=stream),
            "timed batches stream from local storage through %d worker processes that write each batch into a shared ring; one host copy into the "
            "slot's page-locked twin, DMA of the raw %dx%d uint8 batch and its ground-truth masks from there, resize to the test size ON THE DEVICE, staged one batch ahead; "
            "in both passes (rendering the stream to disk and starting the workers are outside the timed region)"
            % (cfg.DATALOADER.NUM_WORKERS, args.size, args.size))
        ab["loader_inclusive"]["fraction_of_resident"] = ab["loader_inclusive"]["value"] / (K * B / main["elapsed"])
    if args.workload != "cfg2":
        args.no_cpu_baseline = True           # the CPU port is set up for the headline workload only
    if world == 1 and args.weights == "trained" and not args.no_cpu_baseline:
        note("Dice parity leg (GPU)")
        parity = {"gpu": gpu_dice_parity_leg(cfg, model, init_state, batches[0], local_dicts, name, tf)}

    step_roof = cfg3 = None
    if world == 1 and not args.no_cfg3:
        try:
            note("whole-step FLOP count")
            step_roof = step_flops(cfg, model, init_state, batches[W], tf)
            note("cfg-3 operator-level block (8 graphs x 256 nodes)")
            cfg3 = cfg3_block(device)
        except Exception as e:          # reports, never a reason to lose the headline
            note("cfg-3 / step-roofline block failed: %r" % (e,))
            cfg3 = {"error": repr(e)}
    if rank != 0:
        return
    images = world * K * B
    roofs_head = kernel_rooflines(main)
    roofs_all = roofs_head if instrumented is main else kernel_rooflines(instrumented)
    roofs = roofs_head[:1] + [r for r in roofs_all if not roofs_head or r["kernel"] != roofs_head[0]["kernel"]]
    out = {
        "metric": "adapted images/sec (%dx%d, %d-class)" % (args.size, args.size, args.num_cls), "value": images / main["elapsed"], "unit": "images/s",
        "n_gpus": world, "steps": K, "warmup": W, "ms_per_step": main["elapsed"] / K * 1e3,
        "higher_is_better": True, "scaling": "strong" if args.images else "weak", "vs_baseline": None,
        "dtype": "f32" if not args.bf16_backbone else "bf16 backbone / f32 matching", "data": "synthetic",
        "config": {"workload": "%s: %d-image synthetic %dx%d %d-class %s stream%s, TEST.BATCH=%d (%dx%d after the test mapper), "
                               "ResNet-50-FPN stand-in + 20-sweep Sinkhorn, 1 TTA step per batch + Dice pass"
                               % ("cfg-2" if args.workload == "cfg2" else "cfg-5 (per GPU)", args.images or K * B, args.size, args.size, args.num_cls, args.kind,
                                  " in total" if args.images else " per GPU", B, cfg.INPUT.MIN_SIZE_TEST if args.workload == "cfg5" else 800,
                                  cfg.INPUT.MIN_SIZE_TEST if args.workload == "cfg5" else 800),
                   "global_batch": world * B,
                   "parallelism": ("dp%d (independent shards, no data-path collective; Dice scores all-gathered)" % world) if not (args.sync_universe and world > 1)
                   else "dp%d synchronous universe graph (all-gather of node embeddings + gradient all-reduce)" % world,
                   "ranks_seen_by_%s" % (dist.get_backend() if world > 1 else "single_process"): world},
        "weights": ("trained-regime synthetic checkpoint (tools/synth_checkpoint.py: %s)" % json.dumps(ckpt_report, default=str)) if weights else "random init + FrozenBN calibration",
        "detections": "teacher-forced (GT boxes jittered +-2 px)" if tf else "free-running (the detector's own boxes)",
        "inputs": "pre-staged in HBM (uint8, already resized to 800x800 by the test mapper); loader-inclusive rate under ab.loader_inclusive",
        "tta_only_images_per_s": images / main["tta"], "dice": main["dice"], "kept_masks": main["kept_masks"],
        "tta_steps_taken": main["steps_taken"],
        "eager_pass": (None if eager_probe is None else {"value": images / eager_probe["elapsed"], "unit": "images/s", "dice": eager_probe["dice"],
                                                          "note": "same K batches, backbone launched kernel by kernel (graphs off): the pass the per-kernel HIP-event durations of `roofline` come from"}),
        "backbone_launches": ("hipGraph replay of the backbone's no-grad forward (Dice pass); the TTA step's forward + backward eagerly (modeling/graphed.py): %s (A/B: --graphs)" % (model.__dict__["_graphed"].stats,)
                              if model.__dict__.get("_graphed") is not None and model.__dict__["_graphed"].stats["eval_replays"] > 0 else "eager, kernel by kernel (A/B: --graphs replays the Dice pass's backbone forward from a hipGraph)"),
        "vendor_convolutions": ("MIOpen immediate mode, solvers from the find-db shipped in ttdg-mgm_amd/miopen_db (tools/tune_miopen.sh; A/B: --no-miopen-db)"
                                if os.path.basename(os.environ.get("MIOPEN_USER_DB_PATH", "").rstrip("/")).startswith(("miopen_db", "ttdg_miopen_db")) and not args.miopen_search else
                                "MIOpen timing its solvers in this process (--miopen-search)" if args.miopen_search else "MIOpen immediate mode, heuristic solver choice"),
    }
    if roofs:
        out["roofline"] = roofs[0]          # the hand-written kernel with the largest total time in the timed region (live HIP events)
        out["roofline"]["traffic_note"] = "HBM bytes per launch from the committed PMC passes of this command (profiles/), null when not collected"
        out["roofline_other_kernels"] = roofs[1:]
        if instrumented is not main:
            dom_all = roofs_all[0]["kernel"] if roofs_all else None
            out["instrumented_pass"] = {"value": images / instrumented["elapsed"], "unit": "images/s", "ms_per_step": instrumented["elapsed"] / K * 1e3,
                                        "dominant_kernel_by_total_time": dom_all,
                                        "note": "same K batches with HIP-event pairs around EVERY hand-written kernel family (the per-layer ones every %d-th launch): the source of "
                                                "roofline_other_kernels; the headline pass stamps %s only" % (args.timer_every, "/".join(dominant))}
    if world == 1 and step_roof is not None:
        step_roof.update(achieved_tflops=step_roof["flops_per_step"] / (main["elapsed"] / K) / 1e12)
        step_roof["frac_fp32_mfma"] = step_roof["achieved_tflops"] / FP32_PEAK_TFLOPS
        out["roofline_step"] = step_roof
    if cfg3 is not None:
        out["cfg3"] = cfg3
    if strong is not None:
        out["strong"] = strong
    if ab:
        out["ab"] = ab
    out["parity"] = parity_block()
    if world == 1 and not args.no_cpu_baseline:
        try:
            note("CPU baseline (1 warm-up + %d repetitions)" % args.cpu_reps)
            out["cpu_baseline"], cpu_dice = cpu_baseline(args, weights, tf)
            note("CPU baseline done: %s s per repetition" % out["cpu_baseline"]["seconds_all"])
            out["speedup_vs_cpu_baseline"] = out["value"] / out["cpu_baseline"]["value"]
            if parity is not None:
                parity["cpu_port"] = cpu_dice
                parity["abs_diff"] = {k: abs(parity["gpu"][k] - cpu_dice[k]) for k in cpu_dice if k in parity["gpu"] and k != "kept_masks"}
                parity["sample"] = "same checkpoint; 1 TTA step on the first %d-image batch, then the Dice pass on it; 0-100 scale" % B
        except Exception as e:  # the baseline is a report, never a reason to lose the GPU number
            out["cpu_baseline"] = {"error": repr(e)}
    if parity is not None:
        out["dice_parity"] = parity
    print(json.dumps(_finite(out)))


# ------------------------------------------------------------------------------------------- launcher
def free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _spawned(rank, world, port, argv):
    os.environ.update(RANK=str(rank), LOCAL_RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                      HSA_ENABLE_IPC_MODE_LEGACY="0")
    run(parse(argv))


def main(argv=None):
    args = parse(argv)
    if "WORLD_SIZE" in os.environ or args.gpus <= 1:       # launched by torch.distributed.run, or a single rank
        return run(args)
    # `python bench.py --gpus N`: spawn one rank per GPU on 127.0.0.1, as the reference's launch(main, num_gpus) does
    # (train_net.py:94-101)
    import torch.multiprocessing as mp
    mp.spawn(_spawned, args=(args.gpus, free_port(), list(sys.argv[1:] if argv is None else argv)), nprocs=args.gpus, join=True)


if __name__ == "__main__":
    main()
