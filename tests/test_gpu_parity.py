"""-m gpu: parity of the HIP path (through the C ABI) against the oracle on a real MI355X."""
import os

import pytest
import torch

import deft_oracle as O
import parity_checks as pc
from parity_checks import T

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("args", [
    (1, 8, 12, 16, 16, 3, 1, 1, T(128, 32)),
    (2, 9, 7, 3, 16, 7, 1, 3, T(128, 32)),
    (1, 10, 12, 32, 64, 3, 2, 1, T(64, 64)),
    (1, 10, 12, 64, 64, 3, 1, 1, T(128, 64)),
    (1, 6, 10, 448, 128, 1, 1, 0, T(128, 128)),
    (1, 6, 10, 64, 200, 1, 1, 0, T(64, 128)),
    (2, 38, 68, 256, 256, 3, 1, 1, 0),
    (1, 152, 272, 64, 64, 3, 1, 1, 0),
    (3, 4, 4, 128, 27, 3, 1, 1, 0),
    (1, 10, 12, 64, 64, 3, 1, 1, T(128, 64) | (1 << 29)),
    (1, 10, 12, 64, 64, 3, 1, 1, T(64, 64) | (1 << 29)),
    (1, 5, 9, 32, 48, 1, 1, 0, T(64, 64)),
    (1, 5, 9, 64, 48, 1, 1, 0, T(64, 64)),
    (2, 7, 9, 64, 27, 3, 1, 1, T(64, 32)),                   # intra-workgroup split-K, 2 waves per output tile
    (2, 7, 9, 64, 27, 3, 1, 1, T(32, 32)),                   # 4 waves per output tile
    (1, 6, 5, 16, 20, 3, 1, 1, T(32, 32) | (1 << 29)),       # split-K + 2-stage loop + Cin < 32
    (1, 11, 13, 128, 27, 3, 1, 1, 0),                        # auto tile -> split-K (few rows, Cout <= 32)
])
def test_conv(gpu_lib, args):
    pc.check_conv(gpu_lib, "cuda", *args, res=(args[4] % 3 == 1), relu=(args[3] != 448))


@pytest.mark.parametrize("Ci,k", [(3, 7), (16, 3), (8, 5)])
def test_conv_pixel_pair(gpu_lib, Ci, k):
    pc.check_conv_pair(gpu_lib, "cuda", Ci, k)


@pytest.mark.parametrize("Ci,k,kw", [(3, 7, {}), (16, 3, {}), (16, 3, {"N": 1, "H": 8, "W": 32, "Co": 12, "relu": False}), (3, 7, {"N": 1, "H": 19, "W": 70, "wide": True}),
                                     (16, 3, {"wide": True, "seed": 3}), (16, 3, {"stride": 2, "Co": 32}), (16, 3, {"stride": 2, "Co": 24, "H": 16, "W": 66, "N": 1, "relu": False}), (16, 3, {"stride": 2, "Co": 32, "H": 9, "W": 130, "wide": True}), (16, 3, {"N": 3, "H": 152, "W": 272}), (3, 7, {"N": 2, "H": 152, "W": 272, "seed": 5})])
def test_conv_direct(gpu_lib, Ci, k, kw):
    pc.check_conv_direct(gpu_lib, "cuda", Ci, k, **kw)


def test_conv_direct_reads_the_image_planes(gpu_lib):
    pc.check_conv_direct_planar(gpu_lib, "cuda")
    pc.check_conv_direct_planar(gpu_lib, "cuda", N=3, H=64, W=96, seed=6)


@pytest.mark.parametrize("args", [(1, 9, 37, 64, 256, 1, "halo", 0), (2, 5, 33, 64, 256, 3, "halo", T(4, 128)), (1, 6, 40, 64, 128, 10, "halo", T(8, 64)),
                                  (1, 7, 19, 64, 256, 2, "im2col", T(64, 128) | (1 << 30)), (1, 6, 21, 64, 72, 1, "im2col", T(128, 64) | (1 << 30)),
                                  (2, 152, 272, 64, 256, 1, "halo", 0), (1, 152, 272, 64, 256, 10, "halo", 0)])
def test_conv_fold(gpu_lib, args):
    pc.check_conv_fold(gpu_lib, "cuda", *args)


def test_concat_conv(gpu_lib):
    pc.check_concat_conv(gpu_lib, "cuda")


@pytest.mark.parametrize("args", [(1, 7, 9, 64, 64, 0), (2, 5, 6, 128, 64, 0), (1, 6, 6, 64, 160, T(64, 128)),
                                  (1, 38, 68, 256, 128, 0), (1, 76, 136, 64, 64, 0),
                                  (1, 9, 9, 64, 64, T(128, 64)), (1, 4, 5, 256, 128, T(128, 128)),
                                  (1, 7, 9, 64, 64, T(64, 64) | (1 << 29)), (1, 5, 5, 128, 64, T(128, 64) | (1 << 29))])
def test_dcn(gpu_lib, args):
    pc.check_dcn(gpu_lib, "cuda", *args[:5], tile=args[5])


@pytest.mark.parametrize("args", [(1, 7, 9, 64, 64, 0), (2, 5, 6, 128, 64, 0), (1, 6, 6, 64, 160, 0), (1, 9, 19, 64, 64, 0), (1, 17, 35, 32, 128, 0),
                                  (2, 3, 2, 64, 8, 0), (1, 8, 16, 64, 128, 64), (1, 11, 20, 32, 40, 128), (2, 38, 68, 256, 128, 0), (1, 19, 34, 512, 256, 0)])
def test_dcn_patch(gpu_lib, args):
    for big in (False, True):
        pc.check_dcn(gpu_lib, "cuda", *args[:5], tile=args[5], seed=3, big_offsets=big, patch=True)


@pytest.mark.parametrize("patch", [False, True])
@pytest.mark.parametrize("name", ["small", "borders", "wide"])
def test_dcn_golden_vectors(gpu_lib, name, patch):
    """Both DCN kernel forms against the vectors of the scalar restatement of upstream DCNv2 (tests/golden/dcn_v2_*.npz)."""
    pc.check_dcn_golden(gpu_lib, "cuda", name, patch)


@pytest.mark.parametrize("shape", [(152, 272, 64, 64, 16), (76, 136, 128, 128, 32), (76, 136, 128, 64, 32), (38, 68, 256, 128, 64)])
def test_dcn_patch_batch_invariance(gpu_lib, shape):
    """Several generations of workgroups per CU (5168 / 2880 / 2880 / 1600 workgroups on 256 CUs): a frame alone, inside the batch, run
    after run -- the same bits (this is where round 2's weight-DMA form of the DCN failed)."""
    H, W, Ci, Co, N = shape
    pc.check_dcn_patch_batch_invariance(gpu_lib, "cuda", H, W, Ci, Co, N=N, reps=5)


@pytest.mark.parametrize("args", [(1, 7, 9, 64), (2, 19, 34, 128), (16, 152, 272, 64), (32, 76, 136, 128), (64, 38, 68, 256)])
def test_dcn_producer_consumer_identical(gpu_lib, args):
    """Round 6: the producer / consumer form of the 64-column DCN tile (dcn_pc_kernel: eight waves, A fragments handed over through LDS,
    one barrier per chunk) against the one-role kernel (dcn_patch_kernel<2>, tile bit 27) -- bit for bit, small and at the bench's launch
    sizes (several generations of workgroups per CU), small and large offsets (the far lanes' global loads)."""
    for big in (False, True):
        pc.check_dcn_pc_identical(gpu_lib, "cuda", *args, big_offsets=big, seed=5)


def test_dcn_big_offsets(gpu_lib):
    pc.check_dcn(gpu_lib, "cuda", 1, 6, 8, 64, 64, big_offsets=True, seed=3)
    pc.check_dcn(gpu_lib, "cuda", 1, 19, 34, 128, 64, big_offsets=True, seed=4)


def test_pool_upsample(gpu_lib):
    pc.check_pool_upsample(gpu_lib, "cuda")


def test_layout(gpu_lib):
    pc.check_layout(gpu_lib, "cuda")


@pytest.mark.parametrize("C,Co", [(16, 32), (64, 48), (128, 64), (512, 32)])
def test_embed_map(gpu_lib, C, Co):
    pc.check_embed_map(gpu_lib, "cuda", C, Co)


def test_embed_fused(gpu_lib):
    pc.check_embed_fused(gpu_lib, "cuda")


@pytest.mark.parametrize("tile", [0, T(128, 32), T(64, 32), T(32, 32), T(64, 64)])
def test_sparse_row_conv(gpu_lib, tile):
    pc.check_sparse_conv(gpu_lib, "cuda", tile)


def test_heads_at_peaks(gpu_lib):
    pc.check_heads_at_peaks(gpu_lib, "cuda")


def test_topk_edge_cases(gpu_lib):
    pc.check_topk_edge_cases(gpu_lib, "cuda")


@pytest.mark.parametrize("dataset", ["mot", "nuscenes"])
def test_lstm(gpu_lib, dataset):
    pc.check_lstm(gpu_lib, "cuda", dataset)


@pytest.mark.parametrize("dataset", ["mot", "nuscenes"])
def test_motion_step(gpu_lib, dataset):
    pc.check_motion(gpu_lib, "cuda", dataset)


def test_track_similarity(gpu_lib):
    pc.check_track_similarity(gpu_lib, "cuda")


@pytest.mark.parametrize("tag,dataset,H,W", [("mot_128x160", "mot", 128, 160), ("mot_224x384", "mot", 224, 384),
                                              ("nuscenes_96x128", "nuscenes", 96, 128),
                                              ("kitti_96x320", "kitti_tracking", 96, 320)])
def test_forward_embed_affinity_golden(gpu_lib, tag, dataset, H, W):
    """Whole path vs the oracle AND the golden fixture written from the reference modules."""
    sd = O.synth_state_dict(dataset)
    plan, rep, (ora_out, ora_maps) = pc.check_forward(gpu_lib, "cuda", dataset, H, W, golden_tag=tag, sd=sd)
    afe, emb = pc.check_embed(gpu_lib, "cuda", plan, ora_maps, sd, golden_tag=tag)
    pc.check_affinity(gpu_lib, "cuda", sd, golden_tag=tag, afe=afe)


def test_forward_batched(gpu_lib):
    """N=3 frames in one pass (frames are independent: detector.py:153,162)."""
    sd = O.synth_state_dict("mot")
    plan, rep, (ora_out, ora_maps) = pc.check_forward(gpu_lib, "cuda", "mot", 96, 160, N=3, sd=sd)
    pc.check_embed(gpu_lib, "cuda", plan, ora_maps, sd)


def test_affinity_config_sizes(gpu_lib):
    """BASELINE configs A (32x128 = 4x32) and B (100x500 = 5x100) against the oracle."""
    sd = O.synth_state_dict("mot")
    from deft_amd import engine
    afe = engine.AfePlan(sd, 100, "cuda", gpu_lib)
    g = torch.Generator().manual_seed(11)
    for F_, P, Q in ((4, 32, 32), (5, 100, 100)):
        hist = [torch.randn(P, afe.D, generator=g).abs() * 2 for _ in range(F_)]
        cur = torch.randn(Q, afe.D, generator=g).abs() * 2
        out, starts = afe.affinity(hist, cur)
        for f in (0, F_ - 1):
            ref = torch.from_numpy(O.afe_affinity(hist[f].unsqueeze(0), cur.unsqueeze(0), sd, 100))
            assert pc.maxabs(out[starts[f]:starts[f + 1]], ref) <= 1e-4
        # size-independent property: every row of [P, Q+1] is bounded by softmax mass
        assert float(out.min()) >= 0.0 and float(out.max()) <= 1.0


def test_full_size_properties(gpu_lib):
    """BASELINE config B shape (1088x608): too big for a full oracle diff inside the suite's
    time budget on every run, so check size-independent properties + a sampled oracle diff:
    decode ordering, NMS property, and equality with the same frame run inside a batch of 2."""
    from deft_amd import engine
    sd = O.synth_state_dict("mot")
    H, W = 608, 1088
    seed, x0, out, maps, od = pc.stable_frame(sd, "mot", H, W, K=100, seed0=0)      # chosen from the oracle alone
    x = torch.cat([x0, torch.randn(1, 3, H, W, generator=torch.Generator().manual_seed(50))], 0)
    p1 = engine.DlaSegPlan(sd, 1, H, W, "mot", K=100, device="cuda", lib=gpu_lib)     # one frame: deep layers use the cross-workgroup split-K
    assert any(d.splitk > 1 for _, _, d in p1._gemms)
    p1.forward(x[:1].cuda())
    torch.cuda.synchronize()
    s = p1.scores[0].cpu()
    assert bool((s[:-1] >= s[1:]).all()) and float(s[-1]) > 0       # sorted, all real peaks
    # batch invariance: with one summation order (no cross-workgroup split) a frame gives the same bits alone and
    # inside a batch; the split only changes the order (round-off level) and keeps the decode
    # (same kernel for both batch sizes: which kernel a layer runs on normally depends on how many tiles the launch has,
    #  engine.p3_choice -- the pre-split kernels only when they fill the chip)
    engine.SPLITK = False
    saved_min, engine.P3_MIN_TILES = engine.P3_MIN_TILES, 0
    saved_dmin, engine.DCN_PATCH_MIN_TILES = engine.DCN_PATCH_MIN_TILES, 0
    try:
        q1 = engine.DlaSegPlan(sd, 1, H, W, "mot", K=100, device="cuda", lib=gpu_lib)
        q2 = engine.DlaSegPlan(sd, 2, H, W, "mot", K=100, device="cuda", lib=gpu_lib)
    finally:
        engine.SPLITK = True
        engine.P3_MIN_TILES = saved_min
        engine.DCN_PATCH_MIN_TILES = saved_dmin
    assert not any(d.splitk > 1 for _, _, d in q1._gemms)
    q1.forward(x[:1].cuda()); q2.forward(x.cuda())
    torch.cuda.synchronize()
    assert torch.equal(q1.inds[0].cpu(), q2.inds[0].cpu())          # batch-invariant, bit-exact
    assert torch.equal(q1.scores[0].cpu(), q2.scores[0].cpu())
    assert torch.equal(q1.bboxes[0].cpu(), q2.bboxes[0].cpu())
    assert torch.equal(p1.inds[0].cpu(), q1.inds[0].cpu())
    assert pc.maxabs(p1.scores.cpu(), q1.scores.cpu()) <= 1e-5 and pc.maxabs(p1.bboxes.cpu(), q1.bboxes.cpu()) <= pc.TOL
    # every reported index is a 3x3 local maximum of the dense hm map
    hm = torch.sigmoid(p1.dense["hm"].to_nchw().cpu())
    keep = torch.nn.functional.max_pool2d(hm, 3, 1, 1) == hm
    assert bool(keep.view(-1)[p1.inds[0].cpu().long()].all())
    # the oracle on the same frame
    assert torch.equal(p1.inds[0].cpu().long(), od["inds"][0]), "top-100 indices differ at 1088x608 (seed %d)" % seed
    assert pc.maxabs(p1.bboxes.cpu(), od["bboxes"]) <= pc.TOL
    assert pc.maxabs(p1.scores.cpu(), od["scores"]) <= pc.TOL


@pytest.mark.parametrize("seed", [100, 101, 102])
def test_full_size_index_differences_are_ties(gpu_lib, seed):
    """How far ordered top-K equality can hold between two fp32 implementations with different summation
    orders: on arbitrary random frames at 1088x608 either the indices are identical, or every
    difference is a tie at round-off level -- the oracle's own heat map puts the device's extra peak within
    1e-4 (logit) of its 3x3 neighbourhood maximum or of the K-th score -- and the float outputs still agree
    within 1e-3.  (Seed 101 is a frame where one NMS near-tie resolves to the neighbouring pixel.)"""
    from deft_amd import engine
    sd = O.synth_state_dict("mot")
    H, W, K = 608, 1088, 100
    x = torch.randn(1, 3, H, W, generator=torch.Generator().manual_seed(seed))
    plan = engine.DlaSegPlan(sd, 1, H, W, "mot", K=K, device="cuda", lib=gpu_lib)
    plan.forward(x.cuda())
    with torch.no_grad():
        out, _ = O.dlaseg_forward(x, sd, "mot")
    pc.compare_topk_with_oracle(plan, out, K)


@pytest.mark.parametrize("dataset,H,W,nseeds", [("mot", 608, 1088, 64), ("kitti_tracking", 384, 1280, 16), ("nuscenes", 448, 800, 16)])
def test_topk_seed_sweep_both_arithmetics(gpu_lib, dataset, H, W, nseeds):
    """the top-K index claim as a measured property of BOTH contraction arithmetics (prec 0 = fp32 MFMA,
    prec 1 = split bf16, the default) on ARBITRARY frames (no stable_frame selection): every frame either reproduces the
    oracle's ordered top-100 indices or differs only at <= 1e-4 logit ties (compare_topk_with_oracle), and the default
    arithmetic does not mismatch more often than the fp32 MFMA beyond counting noise.  The rates go to
    gpurun_out/topk_sweep_<dataset>.json (copied to profiles/)."""
    import json
    from deft_amd import engine
    sd = O.synth_state_dict(dataset)
    plans = {}
    saved = engine.PREC
    try:
        for prec in (0, 1):
            engine.PREC = prec
            plans[prec] = engine.DlaSegPlan(sd, 1, H, W, dataset, K=100, device="cuda", lib=gpu_lib)
            assert all(d.prec == prec for _, _, d in plans[prec]._gemms)
    finally:
        engine.PREC = saved
    torch.set_num_threads(max(1, min(32, os.cpu_count() or 8)))      # ATen's CPU convs thrash far below the box's 256 hardware threads
    # heat-map logits agree to <= 2e-4 and every index difference is a <= 1e-4 tie, for every dataset (round 2 needed 3e-3 for the KITTI /
    # nuScenes nets: their trunks were a worse-conditioned random draw, see deft_amd.synth.synth_state_dict)
    logit_tol, tie = 2e-4, 1e-4          # ONE tolerance set for all datasets: the synthetic nets share a trunk now (deft_amd.synth.synth_state_dict)
    diff = {0: [], 1: []}
    worst = {0: 0.0, 1: 0.0}
    events = {0: [], 1: []}
    # what the tracker keeps of a frame's detections: score > out_thresh = max(track_thresh, out_thresh) (opts.py:438; detector.py:577-583),
    # 0.4 for MOT17 (experiments/mot17_tracking.sh), the 0.3 default otherwise; nuScenes adds its 0.3 / 0.35 class thresholds (detector.py:222-225)
    out_thresh = 0.4 if dataset == "mot" else 0.3
    # the SAME seeds also through the plans the bench number is measured on -- 32 frames per step as two 16-frame
    # sub-batch plans on two HIP streams (halo / patch / pre-split kernels at their batched tile counts, the two plans co-resident), key "timed".
    # Fewer than 32 seeds: the step's second half repeats them, so every seed is checked in both sub-batch plans.
    from deft_amd.pipeline import HipCompute
    TB = 32
    comp = HipCompute(sd, TB, H, W, dataset, K=100, device="cuda", lib=gpu_lib, streams=2, ndet=30)
    assert all(d.prec == 1 for p_ in comp.plans for _, _, d in p_._gemms)
    frames = [torch.randn(1, 3, H, W, generator=torch.Generator().manual_seed(seed)) for seed in range(1000, 1000 + nseeds)]
    timed = {}                                                       # seed index -> [(class ids, indices, scores, boxes, hm logits)] per slot it ran in

    class _Slot:                                                     # what compare_topk_with_oracle reads of a plan, for one frame
        def __init__(self, p_, j):
            self.inds, self.clses, self.scores, self.bboxes = [p_.inds[j].cpu()], [p_.clses[j].cpu()], [p_.scores[j].cpu()], [p_.bboxes[j].cpu()]
            hm = p_.dense["hm"].to_nchw()[j:j + 1].cpu()
            self.dense = {"hm": type("V", (), {"to_nchw": staticmethod(lambda hm=hm: hm)})}
    for s0 in range(0, max(nseeds, TB), TB):
        ids = [(s0 + b) % nseeds for b in range(TB)]
        comp.detect_embed(torch.cat([frames[i] for i in ids], 0).cuda())
        torch.cuda.synchronize()
        for b, i in enumerate(ids):
            timed.setdefault(i, []).append(_Slot(comp.plans[b // comp.sub], b % comp.sub))
    diff["timed"], worst["timed"], events["timed"] = [], 0.0, []
    for n_, seed in enumerate(range(1000, 1000 + nseeds)):
        x = frames[n_]
        with torch.no_grad():
            out, _ = O.dlaseg_forward(x, sd, dataset)
        for prec in (0, 1, "timed"):
            cands = timed[n_] if prec == "timed" else [None]
            for slot in cands:
                if slot is None:
                    plans[prec].forward(x.cuda())
                det = []
                same, err = pc.compare_topk_with_oracle(plans[prec] if slot is None else slot, out, 100, logit_tol=logit_tol, tie=tie, details=det)
                worst[prec] = max(worst[prec], err)
                if not same and seed not in diff[prec]:
                    diff[prec].append(seed)
                    events[prec].append({"seed": seed, "differences": det, "reaches_the_tracker": any(d["score"] > out_thresh for d in det),
                                         # a detection only ONE side reports, above the threshold: the tracker would see another detection set
                                         "another_detection_reaches_the_tracker": any(d["score"] > out_thresh and d["only_in"] != "order" for d in det)})
    rep = {"dataset": dataset, "H": H, "W": W, "frames": nseeds, "K": 100,
           "frames_with_tie_level_index_differences": {"prec0_fp32_mfma": len(diff[0]), "prec1_split": len(diff[1]),
                                                       "timed_plans_2x16_frames_2_streams": len(diff["timed"])},
           "seeds": {"prec0": diff[0], "prec1": diff[1], "timed": diff["timed"]},
           "max_abs_logit_error": {"prec0": worst[0], "prec1": worst[1], "timed": worst["timed"]},
           "every_difference_is_a_tie_below_logit": tie if tie is not None else "2 x the frame's max |logit error|",
           # does a tie-level difference ever concern a detection the tracker would keep?
           "out_thresh": out_thresh, "events": {"prec0": events[0], "prec1": events[1], "timed": events["timed"]},
           "frames_whose_difference_reaches_the_tracker": {"prec0": sum(e["reaches_the_tracker"] for e in events[0]),
                                                           "prec1": sum(e["reaches_the_tracker"] for e in events[1]),
                                                           "timed": sum(e["reaches_the_tracker"] for e in events["timed"])},
           "frames_where_another_detection_reaches_the_tracker": {"prec0": sum(e["another_detection_reaches_the_tracker"] for e in events[0]),
                                                                  "prec1": sum(e["another_detection_reaches_the_tracker"] for e in events[1]),
                                                                  "timed": sum(e["another_detection_reaches_the_tracker"] for e in events["timed"])},
           "max_score_of_a_differing_detection": max([d["score"] for p_ in (0, 1, "timed") for e in events[p_] for d in e["differences"]] + [0.0])}
    print(json.dumps(rep))
    try:
        os.makedirs(os.path.join(ROOT, "gpurun_out"), exist_ok=True)
        json.dump(rep, open(os.path.join(ROOT, "gpurun_out", "topk_sweep_%s.json" % dataset), "w"), indent=1)
    except OSError:
        pass
    # the default arithmetic is not worse than the fp32 MFMA (binomial counting noise allowed: the events are rare and independent)
    assert len(diff[1]) <= len(diff[0]) + max(2, len(diff[0]) // 2), rep
    assert worst[1] <= logit_tol and worst[0] <= logit_tol and worst[1] <= 2.5 * worst[0] + 1e-5
    assert worst["timed"] <= logit_tol and len(diff["timed"]) <= len(diff[0]) + max(2, len(diff[0]) // 2), rep


@pytest.mark.parametrize("prec", [0, 1])
def test_peaked_heatmap_ordered_topk(gpu_lib, prec):
    """A heat map shaped like a trained detector's (sparse Gaussian blobs on the -4.6 prior, base_model.py:91-92) through the
    real hm head + NMS + top-K at config B's map size: ordered index equality with the oracle must hold OUTRIGHT."""
    from deft_amd import engine
    saved, engine.PREC = engine.PREC, prec
    try:
        pc.check_peaked_heatmap(gpu_lib, "cuda", 608, 1088, K=100, nblobs=140)
    finally:
        engine.PREC = saved


@pytest.mark.parametrize("dataset,H,W", [("kitti_tracking", 384, 1280), ("nuscenes", 448, 800), ("mot", 512, 512)])
def test_full_size_other_configs(gpu_lib, dataset, H, W):
    """BASELINE configs D (KITTI 1280x384), E (nuScenes 800x448, one camera) and A (512x512) at full size against
    the oracle: top-K indices ordered-equal, floats within 1e-3, embeddings within 1e-4 relative,
    plus the batched LSTM step the configs name."""
    from deft_amd import engine
    sd = O.synth_state_dict(dataset)
    seed, x, out, maps, od = pc.stable_frame(sd, dataset, H, W, K=100, seed0=3)      # chosen from the oracle alone
    plan = engine.DlaSegPlan(sd, 1, H, W, dataset, K=100, device="cuda", lib=gpu_lib)
    plan.forward(x.cuda())
    assert torch.equal(plan.inds[0].cpu().long(), od["inds"][0]) and torch.equal(plan.clses[0].cpu().float(), od["clses"][0])
    d = plan.dets()
    for k in ["scores", "bboxes", "tracking"] + [k for k in ("rot", "dim", "amodel_offset") if k in od]:
        assert pc.maxabs(d[k].cpu(), od[k]) <= pc.TOL, k
    afe = engine.AfePlan(sd, 100, "cuda", gpu_lib)
    cen = torch.rand(1, 30, 2, generator=torch.Generator().manual_seed(5)) * 2 - 1
    emb = afe.extract(plan.fmaps, cen).cpu()
    ref = O.afe_extract(maps, cen.view(1, 30, 1, 1, 2), sd)
    assert pc.maxabs(emb, ref) <= 1e-4 * max(1.0, float(ref.abs().max()))
    hist = [emb[0, :30] for _ in range(2)]
    aff, starts = afe.affinity(hist, emb[0, 10:])
    ref_a = torch.from_numpy(O.afe_affinity(emb[:, :30], emb[:, 10:], sd, 100))
    assert pc.maxabs(aff[starts[0]:starts[1]], ref_a) <= 1e-4
    pc.check_lstm(gpu_lib, "cuda", "mot" if dataset == "kitti_tracking" else "nuscenes")


def test_seam_dcn_module(gpu_lib):
    pc.check_seam_dcn(gpu_lib, "cuda")


def test_seam_lstm(gpu_lib):
    pc.check_seam_lstm(gpu_lib, "cuda", "mot")
    pc.check_seam_lstm(gpu_lib, "cuda", "nuscenes")


@pytest.mark.parametrize("dataset", ["mot", "nuscenes"])
def test_seam_model_afe_decode(gpu_lib, dataset):
    pc.check_seam_model(gpu_lib, "cuda", dataset, 96, 128)


def test_frame_pipeline_matches_per_frame_affinity(gpu_lib):
    """The product pipeline (HipCompute on 2 HIP streams + FramePipeline: batched detect/embed, ring
    affinity, cross-step overlap) against the plain per-frame calls on the same embeddings, and the
    embeddings against the oracle."""
    from deft_amd import engine
    from deft_amd.pipeline import FramePipeline, HipCompute
    sd = O.synth_state_dict("mot")
    H, W, B, K, HIST = 96, 160, 4, 12, 2
    comp = HipCompute(sd, B, H, W, "mot", K=K, device="cuda", lib=gpu_lib, streams=2)
    pipe = FramePipeline(comp, B, K, comp.D, history=HIST, device="cuda")
    afe = engine.AfePlan(sd, 100, "cuda", gpu_lib)
    g = torch.Generator().manual_seed(77)
    embs = []
    for step in range(3):
        x = torch.randn(B, 3, H, W, generator=g)
        outs = pipe.step(x.cuda())
        torch.cuda.synchronize()
        emb = comp.emb.clone()                      # this step's embeddings [B,K,D]
        if step == 0:                               # embeddings vs the oracle at the plan's own detection centres
            with torch.no_grad():
                _, maps = O.dlaseg_forward(x[:1], sd, "mot")
            ref = O.afe_extract(maps, comp.plans[0].centers[0:1].cpu().view(1, K, 1, 1, 2), sd)
            assert pc.maxabs(emb[0:1].cpu(), ref) <= 1e-4 * max(1.0, float(ref.abs().max()))
        for b in range(B):
            embs.append(emb[b])
            gidx = len(embs) - 1
            hist = embs[max(0, gidx - HIST):gidx]
            if not hist:
                assert outs[b] is None
                continue
            want, _ = afe.affinity(hist, embs[gidx])
            assert tuple(outs[b].shape) == tuple(want.shape) and pc.maxabs(outs[b], want) <= 1e-5, (step, b)


def test_detector_mirror_loads_reference_checkpoint(gpu_lib, tmp_path):
    """deft_amd.detector.Detector(opt): reads a checkpoint in the reference's format (model.py:40-53:
    {"epoch", "state_dict"} with DataParallel's "module." prefix), keeps the reference's process()
    signature, returns generic_decode's dict as numpy with ONE device->host copy."""
    from types import SimpleNamespace
    from deft_amd.detector import Detector
    sd = O.synth_state_dict("mot")
    ck = tmp_path / "model_last.pth"
    torch.save({"epoch": 7, "state_dict": {"module." + k: v for k, v in sd.items()}}, ck)
    opt = SimpleNamespace(dataset="mot", K=20, max_object=100, gpus=[0], load_model=str(ck))
    det = Detector(opt)
    x = torch.randn(1, 3, 128, 160, generator=torch.Generator().manual_seed(0))
    output, dets, fmaps = det.process(x)
    with torch.no_grad():
        out, maps = O.dlaseg_forward(x, sd, "mot")
    od = O.generic_decode(O.sigmoid_output(out), K=20)
    assert isinstance(dets["scores"], __import__("numpy").ndarray) and len(fmaps) == 13
    assert (dets["inds"][0] == od["inds"][0].numpy()).all()
    for k in ("scores", "bboxes", "tracking"):
        assert pc.maxabs(torch.from_numpy(dets[k]), od[k]) <= pc.TOL, k
    # frames 2 and 3 of the same shape replay the captured hipGraph: same bits as the eager first frame, and a
    # different image gives that image's detections
    for _ in range(2):
        _, again, _ = det.process(x)
        for k in dets:
            assert (again[k] == dets[k]).all(), k
    assert det._graphs[(1, 128, 160)] is not None
    x2 = torch.randn(1, 3, 128, 160, generator=torch.Generator().manual_seed(1))
    _, d2, _ = det.process(x2)
    with torch.no_grad():
        out2, _ = O.dlaseg_forward(x2, sd, "mot")
    assert (d2["inds"][0] == O.generic_decode(O.sigmoid_output(out2), K=20)["inds"][0].numpy()).all()
    det.reset_tracking(opt)


@pytest.mark.parametrize("kw", [
    dict(bm=64, bn=64, S=4),
    dict(bm=64, bn=64, S=3, k=3, Ci=32),                      # S does not divide the 9 chunks evenly
    dict(bm=128, bn=64, S=2, two_stage=True),                  # LDS-DMA loop form
    dict(bm=32, bn=32, S=4, Co=27),                            # intra-workgroup (4 waves) + cross-workgroup split
    dict(bm=64, bn=32, S=2, Co=20, two_stage=True),
    dict(bm=64, bn=64, S=4, k=1, Ci=320),                      # 1x1: the cursor is the flat k
    dict(bm=64, bn=64, S=5, korder=1),                         # (channel block, tap) K order
    dict(bm=128, bn=128, S=2, k=3, Ci=16),                     # Cin < 32: per-lane taps
])
def test_conv_splitk(gpu_lib, kw):
    pc.check_conv_splitk(gpu_lib, "cuda", **kw)


def test_splitk_auto(gpu_lib):
    pc.check_splitk_auto(gpu_lib, "cuda")


def test_conv_dcn_random_shapes(gpu_lib):
    """The seeded geometry sweeps of tests/test_emu_kernels.py on the real kernels."""
    import random
    rnd = random.Random(20260926)
    tiles = [pc.T(128, 128), pc.T(128, 64), pc.T(128, 32), pc.T(64, 64), pc.T(64, 128), pc.T(64, 32), pc.T(32, 32), 0]
    for case in range(14):
        k = rnd.choice([1, 3, 3, 5])
        Ci = rnd.choice([4, 8, 16, 32, 64, 128]) if k > 1 else rnd.choice([4, 12, 36, 64, 100, 256])
        Co = rnd.choice([1, 5, 16, 27, 33, 64, 96, 130])
        stride = rnd.choice([1, 1, 2])
        pad = rnd.choice([0, k // 2])
        H = rnd.randint(max(k, 3), 13); W = rnd.randint(max(k, 3), 15)
        N = rnd.randint(1, 3)
        tile = rnd.choice(tiles)
        if tile and rnd.random() < 0.4:
            tile |= 1 << 29
        if Ci < 32 and k == 5 and ((Ci * 25 + 31) // 32 * 32) // Ci > 64:
            continue
        pc.check_conv(gpu_lib, "cuda", N, H, W, Ci, Co, k, stride, pad, tile, res=bool(case & 1), relu=bool(case & 2), seed=case)
    rnd = random.Random(7)
    for case in range(8):
        Ci = rnd.choice([32, 64, 128])
        Co = rnd.choice([8, 27, 40, 64, 100, 130])
        N, H, W = rnd.randint(1, 2), rnd.randint(2, 9), rnd.randint(2, 11)
        tile = rnd.choice([0, pc.T(64, 64), pc.T(64, 128), pc.T(128, 64), pc.T(64, 64) | (1 << 29)])
        pc.check_dcn(gpu_lib, "cuda", N, H, W, Ci, Co, tile=tile, seed=case, big_offsets=bool(case & 1))


def test_embed_align_corners_switch(gpu_lib):
    """grid_sample(align_corners=True): the torch 1.2 behaviour of the authors' environment."""
    pc.check_embed_map(gpu_lib, "cuda", 64, 48, align_corners=True)
    pc.check_embed_fused(gpu_lib, "cuda", align_corners=True)


@pytest.mark.parametrize("prec", [0, 1])
def test_both_contraction_arithmetics(gpu_lib, prec):
    """DeftGemmDesc.prec: 0 = fp32 MFMA (k-ordered fmaf chain), 1 = six bf16 MFMA products per fp32 product with fp32
    accumulation (the default).  The same conv / DCN / pair-MLP checks against the oracle with either."""
    from deft_amd import engine
    saved, engine.PREC = engine.PREC, prec
    try:
        pc.check_conv(gpu_lib, "cuda", 1, 10, 12, 64, 64, 3, 1, 1, pc.T(128, 64), res=True)
        pc.check_conv(gpu_lib, "cuda", 2, 6, 10, 448, 128, 1, 1, 0, pc.T(128, 128))
        pc.check_conv(gpu_lib, "cuda", 1, 9, 7, 16, 40, 3, 2, 1, pc.T(64, 64))          # Cin < 32: per-lane taps
        pc.check_conv_splitk(gpu_lib, "cuda", bm=64, bn=64, S=4)
        pc.check_dcn(gpu_lib, "cuda", 1, 9, 11, 64, 64)
        pc.check_dcn(gpu_lib, "cuda", 2, 5, 6, 128, 130, tile=pc.T(64, 128), big_offsets=True)
        pc.check_affinity(gpu_lib, "cuda", O.synth_state_dict("mot"))
    finally:
        engine.PREC = saved


@pytest.mark.parametrize("args", [
    (1, 9, 11, 64, 64, 128, 3, 1, pc.T(128, 64), pc.T(128, 128)),
    (2, 10, 12, 32, 64, 64, 3, 2, pc.T(64, 64), pc.T(256, 64)),
    (1, 7, 9, 96, 128, 64, 1, 1, pc.T(256, 128), pc.T(128, 64) | (1 << 29)),
    (1, 7, 9, 64, 128, 256, 3, 1, pc.T(128, 128) | (1 << 29), pc.T(128, 256)),
    (3, 38, 68, 256, 256, 256, 3, 1, pc.T(256, 128), pc.T(128, 128)),         # many tiles, long K: every stage of the ring in use
    (2, 76, 136, 128, 128, 128, 3, 2, 0, pc.T(128, 128) | (1 << 29)),
    (1, 152, 272, 64, 64, 256, 3, 1, pc.T(256, 64), pc.T(128, 256)),
    (1, 19, 34, 512, 512, 512, 1, 1, pc.T(64, 64), pc.T(64, 64) | (1 << 29)),
    (2, 76, 136, 128, 128, 128, 3, 1, pc.T(128, 128) | (1 << 30), pc.T(128, 64) | (1 << 30)),      # one LDS stage, 3-4 workgroups per CU
    (2, 38, 68, 256, 256, 64, 3, 2, pc.T(64, 128) | (1 << 30), pc.T(64, 64) | (1 << 30)),
])
def test_conv_presplit(gpu_lib, args):
    """DeftGemmDesc.x3 (igemm3.hip: operands pre-split into bf16 pieces, LDS-DMA pipeline) is BIT-identical to the
    in-loop split of igemm.hip on the hardware, for every tile and both ring depths."""
    pc.check_conv_p3(gpu_lib, "cuda", *args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("args", [
    (1, 8, 32, 32, 64, 3, 1, 1, 0), (2, 9, 37, 64, 128, 3, 1, 1, 0), (1, 5, 70, 64, 64, 3, 1, 1, pc.T(4, 64)),
    (1, 6, 33, 32, 32, 3, 1, 1, pc.T(4, 32)), (1, 10, 40, 64, 128, 3, 1, 1, pc.T(8, 128)), (1, 9, 31, 128, 64, 3, 1, 1, pc.T(8, 64)),
    (1, 4, 20, 64, 200, 3, 1, 1, pc.T(4, 128)), (2, 7, 40, 64, 32, 3, 1, 1, pc.T(4, 32) | (1 << 29)),
    (1, 9, 24, 64, 128, 3, 1, 1, pc.T(8, 128) | (1 << 28)), (2, 16, 16, 32, 64, 3, 1, 1, pc.T(8, 64) | (1 << 28)), (1, 11, 37, 64, 32, 3, 1, 1, pc.T(8, 32) | (1 << 28)),
    (3, 76, 136, 128, 128, 3, 1, 1, pc.T(8, 128) | (1 << 28)), (2, 152, 272, 64, 32, 3, 1, 1, pc.T(8, 32) | (1 << 28)),      # 8 x 16 pixel tiles
    (3, 76, 136, 128, 128, 3, 1, 1, 0), (2, 152, 272, 64, 64, 3, 1, 1, 0), (2, 152, 272, 64, 256, 3, 1, 1, pc.T(8, 128)), (4, 38, 68, 256, 32, 3, 1, 1, 0),
])
def test_conv_halo(gpu_lib, args):
    """Halo-tile form of the 3x3 / stride 1 convs (DeftGemmDesc.p3_kernel = 1) against torch conv2d: ragged edges, all tile
    shapes, and full-size maps (every LDS stage and both workgroups of a CU in flight)."""
    pc.check_conv(gpu_lib, "cuda", *args, res=True, relu=True, p3="halo")
    torch.cuda.synchronize()


@pytest.mark.parametrize("prec", [0, 1])
def test_autotune_keeps_every_bit(gpu_lib, prec):
    """_Plan.autotune() may only pick among result-identical kernels -- outputs before and after tuning are
    bit-identical for both contraction arithmetics."""
    from deft_amd import engine
    saved, engine.PREC = engine.PREC, prec
    try:
        sd = O.synth_state_dict("mot")
        plan = engine.DlaSegPlan(sd, 2, 128, 160, "mot", K=20, device="cuda", lib=gpu_lib)
        x = torch.randn(2, 3, 128, 160, generator=torch.Generator().manual_seed(3)).cuda()
        plan.forward(x); torch.cuda.synchronize()
        before = [fm.to_nchw().clone() for fm in plan.fmaps] + [plan.dense["hm"].to_nchw().clone(), plan.bboxes.clone()]
        tiles0 = [d.tile for _, _, d in plan._gemms]
        plan.autotune(reps=1)
        plan.forward(x); torch.cuda.synchronize()
        after = [fm.to_nchw() for fm in plan.fmaps] + [plan.dense["hm"].to_nchw(), plan.bboxes]
        assert tiles0 != [d.tile for _, _, d in plan._gemms], "autotune changed nothing: the test would be vacuous"
        for a, b in zip(before, after):
            assert torch.equal(a, b)
    finally:
        engine.PREC = saved


@pytest.mark.parametrize("tag", ["mot", "mot_lstm"])
def test_composed_dropin_replays_reference_trace(gpu_lib, tag):
    """the COMPOSED drop-in on the hardware.  tests/golden/detector_trace_*.npz is a trace of the reference's own
    `Detector.run` (its pre-processed branch, post-processing and Tracker; written by oracle/make_golden.py where /root/reference
    exists): every call it made into the seams this repository replaces, with inputs and outputs.  Replayed here on cuda:0 in
    the same order -- fused Detector.process with hipGraph replay, embeddings at the reference's centres, recorder blocks,
    device-side similarity medians, batched LSTM motion update -- each against the reference's value at that point."""
    worst = pc.check_detector_trace(gpu_lib, "cuda", tag)
    torch.cuda.synchronize()
    print(worst)


def test_nuscenes_run_replays_reference_trace(gpu_lib):
    """BASELINE configs[4] on the hardware: tests/golden/detector_trace_nuscenes.npz (the reference's own nuScenes `Detector.run`, traced)
    replayed on cuda:0 -- process(), the vectorised post-processing + class thresholds + quaternion / Box chain + per-class NMS against the
    arguments of every per-class `Tracker.update` call, every embedding call, and the batched 3-D LSTM motion update."""
    worst = pc.check_detector_trace_nuscenes(gpu_lib, "cuda")
    torch.cuda.synchronize()
    print(worst)


def test_preprocess_u8(gpu_lib):
    """uint8 frame -> warp + normalise + NHWC on the device, exact against the numpy restatement."""
    pc.check_preprocess_u8(gpu_lib, "cuda")
    pc.check_preprocess_u8(gpu_lib, "cuda", N=1, sh=1080, sw=1920, H=608, W=1088, seed=1)      # MOT17 frame into config B's input
    torch.cuda.synchronize()


@pytest.mark.parametrize("dataset", ["mot", "kitti_tracking"])
def test_device_detect_record(gpu_lib, dataset):
    pc.check_device_detect(gpu_lib, "cuda", dataset, H=128, W=160, K=100, first_n=30)


@pytest.mark.parametrize("mode", ["fix_res", "fix_short", "keep_res"])
def test_fused_detector_run_on_uint8_frames(gpu_lib, mode):
    pc.check_fused_run_u8(gpu_lib, "cuda", sh=270, sw=480, H=128, W=160, K=50, mode=mode)


def test_fused_run_with_lookahead(gpu_lib):
    """Detector.run(frame, prefetch=next): two plan buffer sets, frame k+1's hipGraph beside frame k's tracker -- identical to the serial order."""
    pc.check_fused_run_prefetch(gpu_lib, "cuda")
    pc.check_fused_run_prefetch(gpu_lib, "cuda", sh=270, sw=480, H=160, W=288, K=50, T=8)
    pc.check_fused_run_prefetch(gpu_lib, "cuda", sh=270, sw=480, H=160, W=288, K=50, T=8, hook=True)
    pc.check_fused_run_prefetch(gpu_lib, "cuda", sh=270, sw=480, H=160, W=288, K=50, T=9, hook=True, pairs=True)
    pc.check_fused_run_prefetch(gpu_lib, "cuda", sh=270, sw=480, H=160, W=288, K=50, T=8, pairs=True)
    pc.check_fused_run_prefetch(gpu_lib, "cuda", sh=270, sw=480, H=160, W=288, K=50, T=11, hook=True, pairs=4)


def test_frame_feeder_with_side_streams(gpu_lib):
    """FrameFeeder (pinned double buffer, copy stream) feeding the multi-stream HipCompute: every step's frames are different, and the
    side streams must see THIS step's H2D copy (the round-2 advisor's race: they waited only on the previous step's event).  Two
    streams against one stream, frame for frame."""
    from deft_amd import pipeline, preprocess
    sd = O.synth_state_dict("mot")
    H, W, sh, sw, B = 64, 96, 45, 80, 4
    outs = {}
    for streams in (1, 2):
        comp = pipeline.HipCompute(sd, B, H, W, "mot", K=20, device="cuda", lib=gpu_lib, streams=streams)
        comp.use_u8(sh, sw)
        feeder = preprocess.FrameFeeder(B, sh, sw, "cuda")
        g = torch.Generator().manual_seed(5)
        res = []
        frames = [torch.randint(0, 256, (B, sh, sw, 3), dtype=torch.uint8, generator=g) for _ in range(5)]
        k = feeder.push(frames[0])
        for i in range(5):
            dev = feeder.take(k)
            kn = feeder.push(frames[i + 1]) if i + 1 < 5 else None           # next step's copy flies while this one computes
            emb = comp.detect_embed(dev)
            res.append(emb.clone())
            comp.release_emb()
            feeder.release(k)
            k = kn
        torch.cuda.synchronize()
        outs[streams] = torch.stack(res).cpu()
    assert torch.equal(outs[1], outs[2])
    assert not torch.equal(outs[1][0], outs[1][1])              # (the steps really saw different frames)


def test_sharded_stream_over_rccl(gpu_lib):
    """the `nccl` (RCCL) branch of the sharded tracker stream on the 1-GPU box -- run_stream.py with a
    1-rank process group: both collectives run on device buffers, and the gathered records / affinity blocks must equal the
    collective-free path bit for bit.  (The 2-rank logic, with the reference's Tracker on rank 0, is tests/test_stream_dist.py.)"""
    import json
    import subprocess
    import sys
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29547", HSA_ENABLE_IPC_MODE_LEGACY="0")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "run_stream.py"), "--frames", "5", "--size", "128x160", "--dets", "12", "--force-dist", "--check"],
                       capture_output=True, text=True, timeout=600, env=env)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    rep = json.loads([ln for ln in r.stdout.strip().splitlines() if ln.startswith("{")][-1])
    assert rep["check"] == "ok" and rep["collectives"] and rep["backend"] == "nccl" and rep["bytes_gathered_per_step"] > 0


def test_frame_pipeline_over_rccl(gpu_lib):
    """The throughput pipeline's all-gather through a 1-rank RCCL group (DEFT_FORCE_DIST=1): bench.py must complete and report."""
    import json
    import subprocess
    import sys
    env = dict(os.environ, DEFT_FORCE_DIST="1", MASTER_ADDR="127.0.0.1", MASTER_PORT="29549", HSA_ENABLE_IPC_MODE_LEGACY="0")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--config", "A", "--batch", "4", "--streams", "1", "--steps", "4", "--warmup", "2",
                        "--no-cpu-baseline", "--no-extras"], capture_output=True, text=True, timeout=600, env=env)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    rep = json.loads([ln for ln in r.stdout.strip().splitlines() if ln.startswith("{")][-1])
    assert rep["value"] > 0 and rep["n_gpus"] == 1


@pytest.mark.parametrize("kw", [{}, {"k": 1, "stride": 1, "Ci": 96, "Cm": 128, "Co": 64}, {"Cm": 256, "Ci": 64, "H": 9, "W": 11}, {"N": 4, "H": 152, "W": 272, "Ci": 64, "Cm": 128, "Co": 128}])
def test_conv_inloop_piece_output(gpu_lib, kw):
    pc.check_conv_inloop_y3(gpu_lib, "cuda", **kw)


def test_weight_dma_identical(gpu_lib):
    pc.check_weight_dma_identical(gpu_lib, "cuda")
    torch.cuda.synchronize()


def test_conv_presplit_splitk(gpu_lib):
    pc.check_conv_p3(gpu_lib, "cuda", 1, 19, 34, 512, 512, 256, 3, 1, pc.T(128, 128), pc.T(256, 128), splitk=4)
    pc.check_conv_p3(gpu_lib, "cuda", 1, 7, 9, 128, 128, 64, 3, 1, pc.T(256, 128), pc.T(64, 64) | (1 << 29), splitk=4)
    torch.cuda.synchronize()


def test_split_is_exact_identity_conv(gpu_lib):
    """prec = 1: the operand pieces carry fp32 values through the matrix cores -- exactly (three bf16 pieces) or to half an fp32 ulp inside
    the fp16 range and loudly beyond it (two fp16 pieces).  See parity_checks.check_split_identity."""
    from deft_amd import engine
    assert engine.PREC == 1
    pc.check_split_identity(gpu_lib, "cuda")


@pytest.mark.parametrize("N,H,W", [(1, 608, 1088), (2, 96, 160)])
def test_dataflow_schedule_bit_identical(gpu_lib, N, H, W):
    """The launch list spread over several HIP streams along its data dependencies (engine._Plan.build_schedule), eagerly and as a
    hipGraph with parallel branches, against the same list on one stream: identical bits, replay after replay."""
    from deft_amd import engine, synth
    sd = synth.synth_state_dict("mot")
    g = torch.Generator().manual_seed(11)
    xs = [torch.randn(N, 3, H, W, generator=g).cuda() for _ in range(3)]
    plan = engine.DlaSegPlan(sd, N, H, W, "mot", K=100, device="cuda", lib=gpu_lib)
    outs = lambda: [t.clone() for t in (plan.scores, plan.inds, plan.bboxes, plan.head_vals)] + [fm.buf.clone() for fm in plan.fmaps]
    ref = []
    for x in xs:
        plan.forward(x); torch.cuda.synchronize()
        ref.append(outs())
    S = 2                                                          # what the product captures (engine.tune_schedule holds captures to two streams)
    model = plan.tune_schedule(S)
    assert model is not None and plan.sched["n"] == S and any(plan.sched["where"]) and model[1] < model[0]
    print("ops per stream:", [plan.sched["where"].count(c) for c in range(S)], "cross-stream waits:", sum(len(w) for w in plan.sched["waits"]))
    for _ in range(2):
        for x, r in zip(xs, ref):
            plan.forward(x); torch.cuda.synchronize()          # eager, several streams
            assert all(torch.equal(a, b) for a, b in zip(r, outs()))
    graph = plan.capture_graph()
    for _ in range(3):
        for x, r in zip(xs, ref):
            plan.image.copy_(x)
            graph.replay(); torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(r, outs()))


def test_bench_parity_gate_on_the_timed_plans(gpu_lib):
    """The parity gate of BASELINE.md section 3 runs inside the bench command, on the plans the timed loop runs (64 frames per step as two
    32-frame sub-batch plans on two HIP streams -- halo / patch / pre-split kernels, not the one-frame plan of the other full-size tests), and its
    verdict is DECIDABLE: the raw frames 0, 31, 32, 63 (floats; index differences only inside the oracle's own tie class), the
    mined well-conditioned frames in the same slots (ordered top-K equality demanded), the trained-shaped heat-map stream (ordered equality on all 64
    frames) -- `pass` must be true, the strict verdict on the raw frames is reported beside it."""
    import json
    import subprocess
    import sys
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--steps", "3", "--warmup", "1", "--no-extras", "--no-cpu-baseline"],
                       capture_output=True, text=True, timeout=900, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-3000:]
    out = json.loads([ln for ln in r.stdout.splitlines() if ln.startswith("{")][-1])
    par = out["parity"]
    rawf = [f for f in par["frames"] if f["stream"] == "raw"]
    assert [f["frame"] for f in rawf] == [0, 31, 32, 63] and rawf[0]["affinity_block"] == [500, 101]
    cp = out["config"]["parity"]                     # the compact verdict where the driver keeps it
    assert cp["frames"] == [0, 31, 32, 63] and cp["pass_up_to_roundoff_ties"] is True and cp["pass"] == par["pass"] and cp["error"] is None
    assert set(cp["max_err"]) == {"score", "bbox", "embedding", "affinity", "hm_logit"} and max(cp["max_err"].values()) <= 1e-3
    assert par["floats_within_tol"] and par["pass_up_to_roundoff_ties"], par
    assert par["max_err"]["affinity"] <= 1e-3 and par["max_err"]["embedding"] <= 1e-3 and par["max_err"]["bbox"] <= 1e-3
    assert par["max_err"]["hm_logit"] <= 2.5e-4
    for f in par["frames"]:
        assert f["common_detections"] >= 97 and f["embedding_rows_compared"] >= 97
    dec = par["decidable"]
    assert dec["pass"] and dec["topk_ordered_equal"] and dec["every_plan_has_a_decidable_frame"] and len(dec["decidable_here"]) >= 2, dec
    assert par["peaked"]["pass"] and par["peaked"]["frames"] == 64 and par["peaked"]["topk_ordered_equal"], par["peaked"]
    assert par["pass"] is True and cp["raw"]["pass"] in (True, False) and cp["decidable"]["pass"] and cp["peaked"]["pass"]
    assert out["dtype"].startswith("f32 via ")
    assert out["n_gpus"] == 1 and out["config"]["frames_per_step_per_gpu"] == 64 and out["config"]["hip_streams"] == 2


def test_graph_replay_survives_tracker_teardown(gpu_lib):
    """parity_checks.check_graph_replay_survives_tracker_teardown: captured hipGraphs and queued lookahead passes against tracker close / reset /
    garbage collection / allocator flushes between frames."""
    assert pc.check_graph_replay_survives_tracker_teardown(gpu_lib, "cuda") == 6


def test_captured_graphs_have_no_parallel_branch_by_default(gpu_lib):
    """With ROCm 7.2 the replay of a graph WITH parallel branches has ended in a host segmentation fault after certain process histories
    (profiles/r6_graph_replay_segfault.md).  The package therefore captures its launch lists on ONE stream unless DEFT_DATAFLOW=2 asks for the two-branch
    schedule: a serial Detector.run loop captures a plan without a schedule, and its results are what the eager launch list gives."""
    from types import SimpleNamespace
    from deft_amd import engine
    from deft_amd.detector import Detector
    import numpy as np
    assert engine.DATAFLOW == 1 and not engine.REPLAY_STREAM
    sd = O.synth_state_dict("mot")
    g = np.random.RandomState(2)
    frames = [g.randint(0, 256, (120, 170, 3), dtype=np.uint8) for _ in range(4)]
    out = {}
    for graphs in (True, False):
        opt = SimpleNamespace(dataset="mot", K=20, max_object=100, gpus=[0], hip_graphs=graphs, depth_scale=1.0, input_h=96, input_w=128, out_thresh=-1.0,
                              test_scales=[1.0], flip_test=False, public_det=False)
        det = Detector(opt, sd)
        out[graphs] = [[(float(r["score"]), tuple(float(v) for v in r["bbox"])) for r in det.run(f)] for f in frames]
        plans = list(det._plans.values())
        assert len(plans) == 1 and plans[0].sched is None                    # no multi-stream schedule: the capture is one chain of kernel nodes
        assert (sum(v is not None for v in det._graphs.values()) == 1) == graphs
    assert out[True] == out[False]


def test_pair_mlp_fused(gpu_lib):
    """deft_pair_mlp on the hardware: small shapes, the config sizes (5 x (100 x 100), 4 x (32 x 32)), the ring form, both arithmetics."""
    pc.check_pair_mlp(gpu_lib, "cuda", shapes=((5, 12, 1, 9), (100, 100, 100, 100, 100), (32, 32, 32, 32)), Q=(7, 100, 32))
    pc.check_pair_mlp(gpu_lib.twin(), "cuda", shapes=((100, 100, 100, 100, 100),), Q=(100,))


def test_out_of_range_frame_is_rerun_on_the_range_free_arithmetic(gpu_lib):
    """VERDICT r5 #3 on the hardware: both arithmetics live in the ONE libdeft_hip.so; a frame that overflows the two-fp16-piece range comes back
    correct from the `_p3` entry points (parity_checks.check_out_of_range_fallback), graphs and all."""
    pc.check_out_of_range_fallback(gpu_lib, 0)


def test_twin_arithmetic_forward_matches_oracle(gpu_lib):
    """The three-bf16-piece twins of the same library (DeftGemmDesc consumers `deft_*_p3`) on a whole small frame against the golden fixtures."""
    t = gpu_lib.twin()
    assert t is not None and t.pieces == 3
    plan, rep, _ = pc.check_forward(t, "cuda", "mot", 128, 160, golden_tag="mot_128x160", sd=O.synth_state_dict("mot"))
    assert plan.np == 3


def test_float_errors_over_seeds_on_the_timed_plans(gpu_lib):
    """the FLOAT errors (embedding, bbox, score, heat-map logit, affinity) of the device path against the oracle over input
    seeds, on the timed plans' configuration (32 frames per step, 2 x 16 on two HIP streams), for BOTH arithmetics of the library on one oracle
    pass (tools/probe/float_sweep.py; the 64 / 16 / 16 / 16-seed runs are profiles/r6_float_sweep_*.json).  Bars: the north-star 1e-3 on every
    float, the gate's heat-map bound, and no index difference outside the oracle's tie class.  (The maxima over 64 seeds are 9.3e-4 / 1.4e-4:
    the distance is fp32 summation order -- both arithmetics sit at the same level -- so the bar here is the stated one, not a tighter one.)"""
    import json
    import subprocess
    import sys
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "probe", "float_sweep.py"), "A", "8"], capture_output=True, text=True, timeout=900, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    rep = json.loads([ln for ln in r.stdout.splitlines() if ln.startswith("{")][-1])
    for arith in ("fp16x2", "bf16x3"):
        mx = rep[arith]["max"]
        assert mx["embedding"] <= 1e-3 and mx["bbox"] <= 1e-3 and mx["score"] <= 1e-3 and mx["affinity"] <= 1e-3, (arith, mx)
        assert mx["hm_logit"] <= 2.5e-4 and rep[arith]["frames_outside_tie_class"] == 0, (arith, mx)
    assert rep["fp16x2"]["max"]["embedding"] <= 2.0 * rep["bf16x3"]["max"]["embedding"] + 1e-4          # the two arithmetics sit at the same level


def test_launches_bit_exact_beside_another_kernel(gpu_lib):
    """Round 4 finding: a launch must not change its bits when another stream's kernel shares the compute units (the timed plans run on two
    HIP streams).  See parity_checks.check_co_residency."""
    pc.check_co_residency(gpu_lib)


def test_afe_and_lstm_launches_bit_exact_beside_another_kernel(gpu_lib):
    """the co-residency check of the launches the product overlaps OUTSIDE DlaSegPlan -- the embedding head, both
    forms of the affinity chain, the LSTM step and the fused motion step -- each beside a foreign matrix-core launch, bit for bit."""
    n, names = pc.check_co_residency_afe_lstm(gpu_lib)
    print("co-residency, AFE / LSTM chain: %d launches beside a foreign kernel, bit-exact; entries %s" % (n, names))


def test_fp16_split_sequences_equal_the_cpp_expression(gpu_lib):
    """csrc/common.h deft_split2_pair / deft_split2_pair_scaled: the two-fp16-piece split as v_cvt_pk_f16_f32 + v_fma_mix{lo,hi}_f16 (3 - 4 VALU
    per pair of values) must give the bits of `h = (_Float16)y; m = (_Float16)(y - (float)h)` -- the emulator runs the C++ expression, so only
    the hardware can check the instruction sequences: tools/probe/f16_split_asm.hip (built by __graft_entry__.build()), 1024 values over
    several binades incl. fp16-subnormal residuals, with and without the power-of-two scale."""
    import subprocess
    exe = os.path.join(ROOT, "tools", "probe", "f16_split_asm.bin")
    if gpu_lib.pieces != 2:
        pytest.skip("the library under test uses three bf16 pieces")
    if not os.path.exists(exe):                      # normally built by __graft_entry__.build(); the GPU box has hipcc too
        b = subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O2", exe[:-4] + ".hip", "-o", exe],
                           capture_output=True, text=True, timeout=300)
        if b.returncode != 0 or not os.path.exists(exe):
            pytest.skip("tools/probe/f16_split_asm.bin is not built and cannot be built here: " + b.stderr[-200:])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 mismatches" in r.stdout, r.stdout + r.stderr


def test_motion_bank_shared_by_two_callers(gpu_lib):
    """several trackers share one MotionBank (model.motion: the seven per-class nuScenes trackers, two 2-D trackers on one model) and
    each reads its asynchronous step a frame later.  With ONE pinned (in, out) pair per bank the second caller's copies landed in the first
    caller's buffers before it had read them; every call in flight owns its pair now.  Two interleaved callers against the blocking step()."""
    import numpy as np
    from deft_amd import engine, tracker as DT
    lsd = O.synth_lstm_state_dict("mot")
    shared = DT.MotionBank(engine.LstmPlan(lsd, "cuda", gpu_lib))
    ref = DT.MotionBank(engine.LstmPlan(lsd, "cuda", gpu_lib))
    sa, sb = [shared.alloc() for _ in range(40)], [shared.alloc() for _ in range(70)]
    ra, rb = [ref.alloc() for _ in range(40)], [ref.alloc() for _ in range(70)]
    g = np.random.RandomState(3)
    pend = None
    for fid in range(1, 6):
        ba, bb = g.rand(40, 4) * 80 + 5, g.rand(70, 4) * 80 + 5
        wa = shared.step_async(sa, ba, fid)
        wb = shared.step_async(sb, bb, fid)               # the second caller steps before the first has read its result ...
        ea, eb = ref.step(ra, ba, fid)[1], ref.step(rb, bb, fid)[1]
        if pend is not None:                              # ... and results are read a frame later, like ArrayTracker._resolve does
            (pa, xa), (pb, xb) = pend
            assert np.array_equal(pa(), xa) and np.array_equal(pb(), xb)
            assert np.array_equal(pa(), xa)               # (a second read returns the same array)
        pend = ((wa, ea), (wb, eb))
    (pa, xa), (pb, xb) = pend
    assert np.array_equal(pb(), xb) and np.array_equal(pa(), xa)


@pytest.mark.parametrize("tag", ["mot", "mot_lstm", "nuscenes"])
def test_tracks_against_reference_trace_on_device(gpu_lib, tag):
    """Detector.run -> ArrayTracker on the MI355X against the tracks of the reference's own Detector.run + Tracker
    (ids exact, boxes / scores / 3-D boxes 1e-3)."""
    pc.check_tracks_against_reference_trace(gpu_lib, "cuda", tag)


@pytest.mark.parametrize("dataset,lstm", [("kitti_tracking", True), ("nuscenes", True)])
def test_fused_run_array_tracker_on_device(gpu_lib, dataset, lstm):
    pc.check_fused_run_array_tracker(gpu_lib, "cuda", dataset, lstm, sh=270, sw=480, H=128, W=160, K=40, T=5, pairs=True)
