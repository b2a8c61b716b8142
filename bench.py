#!/usr/bin/env python
"""Contract benchmark: ray-samples/sec of one optimisation step of the Spurfies hot path
(kNN + SDF + render, forward + backward + Adam) on synthetic DTU-scan24-shaped batches.

    python bench.py --gpus N --steps K --warmup W
    python -m torch.distributed.run --nnodes=1 --nproc-per-node N --master-addr 127.0.0.1 \
        --master-port P bench.py --gpus N --steps K --warmup W

One JSON line on rank 0.  A "step" = `TrainStep` (spurfies_amd/train.py) on 1024 rays per GPU:
sampler pass (128 samples/ray through kNN + SDF), main pass (98 samples/ray: kNN, SDF + Jacobian,
colour MLPs, compositing), pseudo-point loss, TV, backward, grad all-reduce (N > 1), clip, Adam.
value = 226 * rays_total * K / seconds (SURVEY.md §8(d) counting convention).
"""
from __future__ import annotations

import argparse
import json
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

SAMPLES_PER_RAY = 128 + 98          # sampler + main pass
F_FWD = 2.0 * (35 * 256 + 3 * 256 * 256 + 256)      # F_geometry (4 layers; the 5th folds into T) + T, per pair
F_JAC = 2.0 * (3 * 256 * 256 + 256 * 35)            # input-Jacobian sweep, per pair
PEAK_F32_MFMA_TFLOPS = 157.3                        # MI355X_MICROARCH.md: v_mfma_f32_32x32x2_f32 dense peak
PEAK_BF16_MFMA_TFLOPS = 2516.6                      # dense bf16 MFMA: 256 CUs x 4 SIMDs x 1024 FLOP/clk x 2.4 GHz
# The dominant kernel forms every fp32 product from 6 exact bf16 piece products (fp32-class accuracy): its matrix-pipe ceiling in
# ALGORITHMIC (fp32) FLOP/s is the bf16 peak / 6.
PEAK_SPLIT_TFLOPS = PEAK_BF16_MFMA_TFLOPS / 6.0
PEAK_H2_TFLOPS = PEAK_BF16_MFMA_TFLOPS / 3.0          # H2: three fp16 piece products per fp32 product (the fp16 and bf16 dense MFMA peaks are equal)


def geo_peak(engine):
    """Ceiling of the geometry kernel's algorithmic fp32 FLOP/s for an engine name (ops.geo_mode())."""
    return PEAK_H2_TFLOPS if engine == "h2" else PEAK_SPLIT_TFLOPS


def family_peak(kernel):
    """(ceiling, piece form) of a kernel of the 'split' family — 'color_fwd' | 'color_bwd' | 'wgrad' | 'rhead_fwd' | 'rhead_bwd' — as this process runs it."""
    from spurfies_amd import ops

    fam = "color" if kernel.startswith("color") else ("rhead" if kernel.startswith("rhead") else "wgrad")
    if ops._arith_of(ops._ARITH[fam], kernel) == 3:
        return PEAK_H2_TFLOPS, "H2: three fp16 piece products per fp32 product; ceiling = dense fp16 MFMA peak / 3"
    return PEAK_SPLIT_TFLOPS, "six bf16 piece products per fp32 product; ceiling = dense bf16 MFMA peak / 6"
PEAK_HBM_GBS = 8000.0                               # MI355X_MICROARCH.md: HBM3E ~8 TB/s
F_COLOR_FWD = 2.0 * (103 * 256 + 2 * 256 * 256)     # F_color's three activated layers, per pair (the linear fourth runs per point)
F_COLOR_BWD = 2.0 * (2 * 256 * 256 + 256 * 64)      # data-gradient chain of the same, per pair (weight gradients: spf_wgrad)


def parse():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--rays", type=int, default=1024, help="rays per step (config/ours.yaml:14 num_pixels).  N > 1: ONE batch of this many rays, rank r renders "
                    "rays r::N of it (strong scaling of BASELINE.json configs[1] — the default); with --weak: rays PER GPU")
    ap.add_argument("--global-rays", type=int, default=0, help="strong scaling with this many rays per step instead of --rays (kept for older command lines)")
    ap.add_argument("--weak", action="store_true", help="weak scaling: --rays rays per GPU, the batch grows with N (no BASELINE config has such batches; "
                    "reported as an `extra` record of the default run at N > 1)")
    ap.add_argument("--extras", choices=["auto", "on", "off"], default="auto", help="extra records in the same JSON line (`extra`), measured AFTER the contract "
                    "region under a timer.  N = 1 (auto / on): the DTU recipe's real step (feature-consistency term on every batch -> ms_per_step_with_local) "
                    "and one evaluation-render chunk (fast = -1, realised sampler iterations).  N > 1 (auto / on), N = 1 (on): BASELINE.json configs[4] "
                    "strong-scaled (2e5 points, 4096 rays per step) and the weak-scaling figure (1024 rays per GPU)")
    ap.add_argument("--c4-points", type=int, default=200000, help="neural points of the configs[4] extra record (tests shrink it)")
    ap.add_argument("--c4-rays", type=int, default=4096, help="rays per step of the configs[4] extra record")
    ap.add_argument("--local", action="store_true", help="also time the DTU recipe's real step: synthetic local_data on every batch (find_surface_points + "
                    "feature-consistency loss, local_weight 0.5) -> extra record + ms_per_step_with_local")
    ap.add_argument("--gc", choices=["off", "on"], default="off", help="Python's cyclic garbage collector during the timed regions (off: collected once before them)")
    ap.add_argument("--settle", type=float, default=2.0, help="seconds of the same step run UNTIMED behind the --warmup steps, before the timed region, so that "
                    "the chip's clock has settled under load (the 20-step region read 6.7 %% faster than the sustained one without it)")
    ap.add_argument("--points", type=int, default=10000, help="neural points (DTU-like cloud)")
    ap.add_argument("--spacing", type=float, default=0.025, help="nearest-neighbour spacing of the synthetic cloud (0.0125 = dense stress cloud)")
    ap.add_argument("--prior", choices=["fitted", "kaiming"], default="fitted", help="fitted: F_geometry/T + latents reproduce the signed distance to the "
                    "analytic surface (realistic sampler convergence / pair counts, SURVEY.md section 8(d)); kaiming: random prior (round-1 scene)")
    ap.add_argument("--scenes", type=int, default=1, help="BASELINE.json configs[3]: this many scenes optimised concurrently on the same ray-sharded "
                    "group (round-robin, no cross-scene collective); a step = one round over all scenes")
    ap.add_argument("--exact-draws", action="store_true", help="N > 1: every rank draws the sampler's CPU random numbers for the WHOLE batch and keeps its "
                    "rays' rows (bit-equal to a single-GPU run of the batch; N times the host-side draws). Default at N > 1: per-rank generator "
                    "streams, each rank draws for its own rays only")
    ap.add_argument("--sustained", type=int, default=200, help="extra steps timed after the contract region (sustained clocks); 0 = skip")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--sync", action="store_true", help="default (reference-shaped) step with one host read-back per step")
    ap.add_argument("--graph", action="store_true", help="replay forward + loss + backward as one hipGraph (measured no faster than the eager sync-free "
                    "step on MI355X: ~3 us of dependency handling per graph node; the eager launches run ahead of the GPU)")
    ap.add_argument("--no-graph", action="store_true", help="eager launches even at <= 256 rays per GPU (where the graph replay is the default: the eager step is host-bound there)")
    ap.add_argument("--fork", action="store_true", help="graph-replayed steps with independent passes as forked branches of the graph (TrainStep(fork=True); measured "
                    "within +-1 %% of the single-stream graph on ROCm 7.2, default off)")
    ap.add_argument("--no-fork", action="store_true", help="(kept for older command lines: the default)")
    ap.add_argument("--off", default="", help="comma list of round-5 launch fusions to switch OFF for same-box A/B runs: fused_sampler, defer_loss, merge_head")
    ap.add_argument("--cpu-rays", type=int, default=1024)
    ap.add_argument("--mode", choices=["train", "eval"], default="train", help="train (the contract line): one optimisation step per step; eval: one evaluation-render chunk per "
                    "step (PointVolSDF.forward(fast=-1) under no_grad: the full error-bounded sampler, kNN, SDF + normals, colour, compositing — SURVEY.md "
                    "section 8(d): reported separately, with the realised sampler iterations), followed by the reference-sized get_sdf_eval grid sweep")
    ap.add_argument("--image", type=int, nargs=2, default=[576, 768], metavar=("H", "W"), help="eval mode: also render ONE full image of this size as a stream of "
                    "--rays-pixel chunks (eval_graph.ImageRenderer: train.py:399-433 / eval_spurfies.py:276-292 without per-chunk host work) and report images/s; 0 0 = skip")
    ap.add_argument("--eval-outputs", choices=["render", "reference"], default="render", help="eval mode: render = the outputs the reference's evaluation loops read "
                    "(rgb_values, depth_values, normal_map: train.py:419-424, eval_spurfies.py:282-287; PointVolSDF.eval_keys), reference = every key of the reference's "
                    "forward (adds the pseudo-point pass, the TV term and the per-slot plot maps)")
    ap.add_argument("--sweep-resolution", type=int, default=512, help="eval mode: samples along the shortest axis of the mesh-extraction grid (the reference: 512); 0 = skip")
    ap.add_argument("--geo-engine", choices=["auto", "split", "split_w", "h2"], default="h2", help="arithmetic / MFMA shape of the dominant kernel: six bf16 piece "
                    "products per fp32 product on 16x16x32 (split) or 32x32x16 tiles (split_w); three fp16 piece products on 32x32x16 tiles (h2: two fp16 pieces per "
                    "operand, 22 mantissa bits, same measured error against float64 as the fp32-MFMA kernel: tools/engine_accuracy.py — the DEFAULT since round 6); auto = "
                    "time the two bf16 shapes on this box before the warm-up steps (TrainStep.autotune_geo_engine) and keep the faster of THOSE")
    ap.add_argument("--ab-reps", type=int, default=10, help="forward+backward passes per leg of the A B B A engine comparison after the timed region (0 = skip)")
    return ap.parse_args()


def self_launch(args) -> int:
    """`python bench.py --gpus N` with no launcher around it (WORLD_SIZE unset): start the N ranks as FRESH child processes through
    torch.distributed.run — before anything in this process has touched the GPU (it never does: importing torch and counting devices do not
    initialise HIP) — relay rank 0's single JSON line to stdout, everything else to stderr, and return the launcher's exit code (non-zero if
    any rank failed).  Never an exec: a process that has initialised the GPU must not be replaced on this pool."""
    import socket
    import subprocess

    backend = os.environ.get("SPF_DIST_BACKEND", "nccl")
    n_dev = torch.cuda.device_count()
    if backend == "nccl" and n_dev < args.gpus:
        sys.stderr.write(f"[bench] --gpus {args.gpus} over RCCL needs {args.gpus} visible GPUs, this node shows {n_dev} "
                         "(SPF_DIST_BACKEND=gloo runs the ranks on the GPUs there are: plumbing check only)\n")
        return 2
    with socket.socket() as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={args.gpus}", "--master-addr", "127.0.0.1",
           "--master-port", str(port), os.path.abspath(__file__), *sys.argv[1:]]
    env = dict(os.environ, SPF_BENCH_LAUNCHER="self", HSA_ENABLE_IPC_MODE_LEGACY=os.environ.get("HSA_ENABLE_IPC_MODE_LEGACY", "0"))
    env.setdefault("OMP_NUM_THREADS", "1")
    sys.stderr.write("[bench] starting %d ranks: %s\n" % (args.gpus, " ".join(cmd)))
    sys.stderr.flush()
    proc = subprocess.Popen(cmd, stdout=subprocess.PIPE, env=env, text=True, bufsize=1)
    line_out = None
    for line in proc.stdout:
        if line.startswith('{"metric"'):
            line_out = line.rstrip("\n")
        else:
            sys.stderr.write(line)
    rc = proc.wait()
    if rc == 0 and line_out is None:
        sys.stderr.write("[bench] the ranks exited cleanly but rank 0 printed no result line\n")
        rc = 1
    if rc == 0:
        print(line_out, flush=True)
    else:
        sys.stderr.write(f"[bench] multi-process run failed (launcher exit code {rc})\n")
    return rc


def init_ranks(args):
    """RANK / LOCAL_RANK / WORLD_SIZE from the launcher's environment -> (world, rank, device, dist_info).  N > 1: the process group over RCCL
    ("nccl" IS RCCL on ROCm; SPF_DIST_BACKEND=gloo for plumbing checks on a single-GPU box) and one all-reduce through it, under a watchdog —
    an RCCL bring-up that hangs (xGMI / IPC misconfiguration) ends the rank with a message and a non-zero code after SPF_DIST_INIT_TIMEOUT
    seconds (default 120: the slowest rank may still be paging in torch when the first one arrives) instead of sitting in the driver's clock."""
    import datetime
    import threading

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    n_dev = max(torch.cuda.device_count(), 1)
    local_rank = int(os.environ.get("LOCAL_RANK", "0")) % n_dev
    torch.cuda.set_device(local_rank)
    device = torch.device("cuda", local_rank)
    if world == 1:
        return world, rank, device, None
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    backend = os.environ.get("SPF_DIST_BACKEND", "nccl")   # "nccl" is RCCL on ROCm; gloo only for single-GPU plumbing tests
    limit = float(os.environ.get("SPF_DIST_INIT_TIMEOUT", "120"))

    def bail():
        sys.stderr.write(f"[bench] rank {rank}/{world} on {device}: process-group bring-up over '{backend}' (init + first all-reduce) did not "
                         f"complete within {limit:.0f} s - giving up (exit 86)\n")
        sys.stderr.flush()
        os._exit(86)

    dog = threading.Timer(limit, bail)
    dog.daemon = True
    dog.start()
    t0 = time.perf_counter()
    kw = {"device_id": device} if backend == "nccl" else {}
    torch.distributed.init_process_group(backend, rank=rank, world_size=world, timeout=datetime.timedelta(seconds=max(2 * limit, 120.0)), **kw)
    probe = torch.full((1,), float(rank + 1), device=device)
    torch.distributed.all_reduce(probe)
    torch.cuda.synchronize()
    dog.cancel()
    if float(probe.item()) != world * (world + 1) / 2.0:
        raise SystemExit(f"[bench] rank {rank}: first all-reduce over '{backend}' returned {float(probe.item())}, expected {world * (world + 1) / 2.0}")
    mine = {"rank": rank, "device": str(device), "name": torch.cuda.get_device_name(device), "pid": os.getpid()}
    devs = [None] * world
    torch.distributed.all_gather_object(devs, mine)
    info = {"backend": torch.distributed.get_backend(), "library": "RCCL (torch.distributed 'nccl' backend on ROCm)" if backend == "nccl" else backend,
            "world_size": torch.distributed.get_world_size(), "ranks": devs, "visible_gpus": torch.cuda.device_count(),
            "bring_up_s": time.perf_counter() - t0, "launcher": "bench.py (self-started torch.distributed.run)" if os.environ.get("SPF_BENCH_LAUNCHER") == "self"
            else "external (torch.distributed.run)"}
    return world, rank, device, info


def make_batches(scene, n_steps, rays_total, rank, world, device, seed=12345, local=False):
    """Seeded synthetic batches of `rays_total` rays, resident on the device before the timed region; rank r keeps rays r::world.
    local: every batch carries its view's synthetic `local_data` (feature maps + MVS camera packs of the shapes datasets/dtu.py:268-291
    provides; resident on the device, one dict per view)."""
    from spurfies_amd import synthetic as syn

    g = torch.Generator().manual_seed(seed)
    K = torch.from_numpy(scene["intrinsics"])[None].to(device)
    out = []
    views = None
    if local:
        views = [{k: (torch.from_numpy(np.asarray(v)).to(device) if isinstance(v, (np.ndarray, np.floating)) else v)
                  for k, v in syn.make_local_data(scene, v_, channels=32, seed=0).items()} for v_ in range(len(scene["poses"]))]      # 32 channels: VisMVSNet's FeatExt (feat_utils.py:347-349)
    for s in range(n_steps):
        uv = torch.from_numpy(syn.make_pixels(rays_total, g))
        rgb = torch.rand((rays_total, 3), generator=g)
        mask = (torch.rand((rays_total,), generator=g) > 0.1).float()
        sel = torch.arange(rank, rays_total, world)
        pose = torch.from_numpy(scene["poses"][s % len(scene["poses"])])[None].to(device)
        out.append(({"intrinsics": K, "uv": uv[sel][None].to(device), "pose": pose, "local_data": None if views is None else views[s % len(views)]},
                    {"rgb": rgb[sel][None].to(device), "mask": mask[sel][None, :, None].repeat(1, 1, 3).to(device)}))
    return out


def cpu_baseline(scene, n_rays):
    """The oracle (CPU restatement of the reference's PyTorch path, pinned to the reference through tests/golden) timed on this box's
    host cores on a bounded sample of the same workload: full optimisation steps (forward, loss, backward, clip, Adam — train.py:330-363)
    with (i) one thread, as the reference itself pins (train.py:24), and (ii) the host's cores."""
    from oracle import path as P
    from spurfies_amd import synthetic as syn

    cfg = P.PathConfig(ranges=tuple(scene["ranges"]))
    g = torch.Generator().manual_seed(999)

    def run(threads, rays, n_steps):
        torch.set_num_threads(threads)
        st = P.load_state(scene["state"])
        grid = P.make_grid(cfg, st["neural_pts"])
        opt, sched = P.make_optimizer(st)
        uv = torch.from_numpy(syn.make_pixels(rays, g))[None]
        inp = {"intrinsics": torch.from_numpy(scene["intrinsics"])[None], "uv": uv, "pose": torch.from_numpy(scene["poses"][0])[None]}
        rgb, mask = torch.rand((rays, 3), generator=g), torch.ones(rays)
        t0 = time.time()
        for _ in range(n_steps):
            P.train_step_grads(inp, rgb, mask, st, cfg, grid=grid)
            P.optimizer_step(st, opt, sched)
        dt = time.time() - t0
        return SAMPLES_PER_RAY * rays * n_steps / dt, dt

    cores = min(os.cpu_count() or 1, 8)   # more intra-op threads only slow these small CPU ops down
    v_all, t_all = run(cores, n_rays, 2)
    r1 = n_rays          # the SAME batch size on one thread (no extrapolation from a quarter batch)
    v_one, t_one = run(1, r1, 1)
    torch.set_num_threads(cores)
    return {"value": v_all, "unit": "ray-samples/s", "cores": cores, "kind": "port",
            "sample": f"2 optimisation steps (fwd+loss+bwd+clip+Adam) of {n_rays} rays on the same scene, {t_all:.1f} s on {cores} threads",
            "single_thread": {"value": v_one, "unit": "ray-samples/s", "cores": 1,
                              "sample": f"1 optimisation step of {r1} rays, {t_one:.1f} s (the reference pins torch.set_num_threads(1), train.py:24)"}}


def build_scene_step(args, seed, device, world, use_graph):
    from spurfies_amd import synthetic as syn
    from spurfies_amd.conf import default_model_conf
    from spurfies_amd.model.pointneus_disent import PointVolSDF
    from spurfies_amd.train import TrainStep

    scene = syn.make_scene(args.points, seed=seed, spacing=args.spacing, prior=args.prior)
    st = scene["state"]
    conf = default_model_conf(near=0.5, grid_ranges=list(scene["ranges"]))
    model = PointVolSDF(conf, 24, "dtu", neural_points={"pts": st["neural_pts"], "colors": scene["colors"]}, device=device)
    model.load_state_dict({k: torch.as_tensor(np.asarray(v)) for k, v in st.items()}, strict=False)
    return scene, model, TrainStep(model, sync_free=not args.sync, use_graph=use_graph, draws="batch" if (args.exact_draws or world == 1) else "local",
                                   fork=bool(args.fork) and not args.no_fork)


def eval_cpu_baseline(scene, n_rays):
    """The oracle's evaluation render (forward, fast=-1, no_grad) on a bounded ray sample, host cores of this box."""
    from oracle import path as P
    from spurfies_amd import synthetic as syn

    cfg = P.PathConfig(ranges=tuple(scene["ranges"]))
    st = P.load_state(scene["state"], requires_grad=False)
    grid = P.make_grid(cfg, st["neural_pts"])
    g = torch.Generator().manual_seed(999)
    cores = min(os.cpu_count() or 1, 8)
    torch.set_num_threads(cores)
    inp = {"intrinsics": torch.from_numpy(scene["intrinsics"])[None], "uv": torch.from_numpy(syn.make_pixels(n_rays, g))[None],
           "pose": torch.from_numpy(scene["poses"][0])[None]}
    stages = {}
    t0 = time.time()
    with torch.enable_grad():          # the oracle forms the normals through autograd, as the reference does (pointneus_disent.py:315-323)
        P.forward(inp, st, cfg, grid=grid, training=False, fast=-1, stages=stages)
    dt = time.time() - t0
    iters = (stages.get("trace") or {}).get("iters")
    return {"value": n_rays / dt, "unit": "rays/s", "cores": cores, "kind": "port",
            "sample": f"one evaluation render of {n_rays} rays (fast=-1) on the same scene, {dt:.1f} s on {cores} threads", "sampler_iterations": iters}


def ops_geo_is_split_w():
    from spurfies_amd import ops

    return ops.geo_mode() == "split_w"


def eval_chunk_record(args, device, scene, steps=20, warmup=5):
    """`extra` record of the default N = 1 line: the evaluation render (PointVolSDF.forward(fast=-1) under no_grad: the full error-bounded
    sampler + main pass with normals + colour + compositing; train.py:399-433 / eval_spurfies.py:276-292 chunks) of --rays-pixel chunks on the
    main record's scene, replayed as one hipGraph per chunk with the outputs those loops read (eval_graph.GraphedRenderer(keys=...))."""
    from spurfies_amd import synthetic as syn
    from spurfies_amd.conf import default_model_conf
    from spurfies_amd.eval_graph import GraphedRenderer
    from spurfies_amd.model.pointneus_disent import PointVolSDF

    st = scene["state"]
    model = PointVolSDF(default_model_conf(near=0.5, grid_ranges=list(scene["ranges"])), 24, "dtu",
                        neural_points={"pts": st["neural_pts"], "colors": scene["colors"]}, device=device)
    model.load_state_dict({k: torch.as_tensor(np.asarray(v)) for k, v in st.items()}, strict=False)
    model.eval()
    g = torch.Generator().manual_seed(777)
    K = torch.from_numpy(scene["intrinsics"])[None].to(device)
    batches = [{"intrinsics": K, "uv": torch.from_numpy(syn.make_pixels(args.rays, g))[None].to(device),
                "pose": torch.from_numpy(scene["poses"][i % len(scene["poses"])])[None].to(device)} for i in range(8)]
    render = GraphedRenderer(model, args.rays, keys=("rgb_values", "depth_values", "normal_map"))
    iters = []
    with torch.no_grad():
        for i in range(warmup):
            render(batches[i % len(batches)])
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for i in range(steps):
            render(batches[i % len(batches)])
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        for i in range(3):                       # realised sampler iterations: read back outside the timed region (one small copy per chunk)
            render(batches[i % len(batches)])
            iters.append(model.ray_sampler.last_iters)
    # opt-in variant, reported beside the default: the sampler's SDF-only passes with reduced products (SPF_ARITH_LITE; main pass unchanged)
    lite = None
    if ops_geo_is_split_w():
        model.sampler_lite = True
        r2 = GraphedRenderer(model, args.rays, keys=("rgb_values", "depth_values", "normal_map"))
        with torch.no_grad():
            for i in range(warmup):
                r2(batches[i % len(batches)])
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            for i in range(steps):
                r2(batches[i % len(batches)])
            torch.cuda.synchronize()
            lite = {"ms_per_step": (time.perf_counter() - t0) / steps * 1e3, "sampler_iterations": int(model.ray_sampler.last_iters),
                    "what": "PointVolSDF.sampler_lite = True (OFF by default): the evaluation sampler's SDF-only passes with two bf16 pieces per operand; the "
                            "main pass, normals and colours keep the fp32-class products (tolerance study: tests/test_gpu_sampler.py::test_reduced_product_...)"}
        model.sampler_lite = False
    samples = args.rays * (128 * float(np.mean(iters)) + 98)
    return {"reduced_product_sampler_passes": lite, "record": "evaluation render: one hipGraph replay per chunk, outputs rgb_values / depth_values / normal_map (what train.py:419-424 and eval_spurfies.py:282-287 read)",
            "metric": "ray-samples/sec (kNN+SDF+render, evaluation render fast=-1)", "value": samples * steps / dt, "unit": "ray-samples/s", "n_gpus": 1, "steps": steps,
            "warmup": warmup, "ms_per_step": dt / steps * 1e3, "scaling": "weak",
            "config": {"workload": f"evaluation render of {args.rays}-ray chunks on the main record's scene ({args.points} neural points): full error-bounded sampler "
                                   "(up to 5 iterations of 128 samples per ray) + 98 main samples per ray, SDF + normals + colour + compositing, no_grad",
                       "mode": "eval", "rays_per_gpu": args.rays, "sampler_iterations_realised": {"mean": float(np.mean(iters)), "min": int(min(iters)), "max": int(max(iters))},
                       "rays_per_s": args.rays * steps / dt}}


def main_eval(args):
    """--mode eval: a step = one evaluation-render chunk of --rays rays per GPU; no collective (chunks of an image are independent)."""
    from spurfies_amd import ops
    from spurfies_amd import synthetic as syn
    from spurfies_amd.conf import default_model_conf
    from spurfies_amd.model.pointneus_disent import PointVolSDF
    from spurfies_amd.utils import surface

    world, rank, device, dist_info = init_ranks(args)
    scene = syn.make_scene(args.points, seed=0, spacing=args.spacing, prior=args.prior)
    st = scene["state"]
    model = PointVolSDF(default_model_conf(near=0.5, grid_ranges=list(scene["ranges"])), 24, "dtu",
                        neural_points={"pts": st["neural_pts"], "colors": scene["colors"]}, device=device)
    model.load_state_dict({k: torch.as_tensor(np.asarray(v)) for k, v in st.items()}, strict=False)
    model.eval()
    g = torch.Generator().manual_seed(777 + rank)
    K = torch.from_numpy(scene["intrinsics"])[None].to(device)
    n = args.warmup + args.steps
    batches = [{"intrinsics": K, "uv": torch.from_numpy(syn.make_pixels(args.rays, g))[None].to(device),
                "pose": torch.from_numpy(scene["poses"][i % len(scene["poses"])])[None].to(device), "local_data": None} for i in range(min(n, 64))]

    def sync():
        if world > 1:
            torch.distributed.barrier()
        torch.cuda.synchronize()

    torch.set_num_threads(1)
    ops.geo_clock_enable(True)                    # this process is the one measuring caller of the library's held-clock counters
    iters = []
    tune = None
    keys = ("rgb_values", "depth_values", "normal_map") if args.eval_outputs == "render" else None
    model.eval_keys = keys
    render = lambda b: model(dict(b), fast=-1)
    with torch.no_grad():
        if args.geo_engine == "auto":          # MFMA shape of the geometry kernels: both timed on one chunk on THIS box (untimed), the faster kept
            tune = {}
            for mode in ("split", "split_w", "split_w", "split"):
                ops.set_geo_mode(mode)
                model(dict(batches[0]), fast=-1)
                ops.profile_start(tags=("geo",))
                model(dict(batches[0]), fast=-1)
                tune[mode] = tune.get(mode, 0.0) + sum(p["ms"] for p in ops.profile_stop())
            ops.set_geo_mode(min(tune, key=tune.get))
            tune = {**{k: v / 2 for k, v in tune.items()}, "selected": ops.geo_mode(), "what": "geometry-kernel ms per chunk (all passes)"}
        else:
            ops.set_geo_mode(args.geo_engine)
        if args.graph:                             # one hipGraph replay per chunk (spurfies_amd/eval_graph.py)
            from spurfies_amd.eval_graph import GraphedRenderer

            render = GraphedRenderer(model, args.rays, keys=keys)
        for i in range(args.warmup):
            render(batches[i % len(batches)])
        ops.geo_clock(reset=True)
        if not args.graph:
            ops.profile_start(tags=("geo", "knn", "color_fwd", "render_fwd"))
        sync()
        t0 = time.perf_counter()
        for i in range(args.warmup, n):
            out = render(batches[i % len(batches)])
            iters.append(model.ray_sampler.last_iters)
        sync()
        dt = time.perf_counter() - t0
        clk = ops.geo_clock(reset=True)
        if args.graph:                             # events cannot sit inside a replay: per-kernel timing over eager passes of the same chunks afterwards
            ops.profile_start(tags=("geo", "knn", "color_fwd", "render_fwd"))
            for i in range(args.warmup, n):
                model(dict(batches[i % len(batches)]), fast=-1)
            sync()
        prof = ops.profile_stop()
    tmax = torch.tensor([dt], device=device, dtype=torch.float64)
    if world > 1:
        torch.distributed.all_reduce(tmax, op=torch.distributed.ReduceOp.MAX)
    dt = float(tmax.item())
    samples = sum(args.rays * (128 * t + 98) for t in iters) * world         # every sampler iteration evaluates 128 new samples per ray, the main pass 98
    # ---- roofline: the forward-only geometry kernel (sampler passes; 411 648 FLOP per pair) and the with-Jacobian launch of the main pass ----
    fwd = [p for p in prof if p["tag"] == "geo" and not p["with_grad"] and p["pairs"] > 0]
    jac = [p for p in prof if p["tag"] == "geo" and p["with_grad"] and p["pairs"] > 0]
    engine = ops.geo_mode()
    roof = None
    if fwd:
        ms, pairs = sum(p["ms"] for p in fwd), sum(p["pairs"] for p in fwd)
        ach = pairs * F_FWD / (ms * 1e-3) / 1e12
        ck = clk.get(("split_w" if engine == "h2" else engine, False))
        gpk = geo_peak(engine)
        cpk, cform = family_peak("color_fwd")
        roof = {"bound": "mfma", "achieved": ach, "peak": gpk, "unit": "TFLOP/s", "frac": ach / gpk,
                "kernel": ("geo_pairs_x3_kernel<false>" if engine == "split" else ("geo_pairs_x3w_kernel<false, 2, true>" if engine == "h2" else "geo_pairs_x3w_kernel<false, 3, false>")) + " (sampler passes: SDF only)",
                "launches": len(fwd), "avg_ms": ms / len(fwd), "pairs_per_launch": pairs / len(fwd), "flop_per_pair": F_FWD, "total_ms_per_step": ms / args.steps,
                "held_clock": held_clock(ach, ck, gpk), "traffic": None, "timing": "HIP events over the timed region",
                "engine": {"selected": engine, "autotune_ms": tune},
                "peak_basis": ("algorithmic fp32 FLOP/s against the dense fp16 MFMA peak / 3 (H2: three exact fp16 piece products per fp32 product)" if engine == "h2" else
                               "algorithmic fp32 FLOP/s against the dense bf16 MFMA peak / 6 (six exact bf16 piece products per fp32 product)")}
        sec = []
        if jac:
            ms2, pairs2 = sum(p["ms"] for p in jac), sum(p["pairs"] for p in jac)
            a2 = pairs2 * (F_FWD + F_JAC) / (ms2 * 1e-3) / 1e12
            sec.append({"kernel": "geometry kernel with the Jacobian sweep (main pass: SDF + normals)", "bound": "mfma", "achieved": a2, "peak": gpk,
                        "unit": "TFLOP/s", "frac": a2 / gpk, "avg_ms": ms2 / len(jac), "pairs_per_launch": pairs2 / len(jac), "total_ms_per_step": ms2 / args.steps})
        col = [p for p in prof if p["tag"] == "color_fwd" and p["pairs"] > 0]
        if col:
            ms3, pairs3 = sum(p["ms"] for p in col), sum(p["pairs"] for p in col)
            a3 = pairs3 * F_COLOR_FWD / (ms3 * 1e-3) / 1e12
            sec.append({"kernel": "color_forward_x3_kernel<false>", "bound": "mfma", "achieved": a3, "peak": cpk, "peak_basis": cform, "unit": "TFLOP/s",
                        "frac": a3 / cpk, "avg_ms": ms3 / len(col), "pairs_per_launch": pairs3 / len(col), "total_ms_per_step": ms3 / args.steps})
        knn = [p for p in prof if p["tag"] == "knn"]
        if knn:
            sec.append({"kernel": "spf_grid_query (all passes)", "bound": "hbm", "total_ms_per_step": sum(p["ms"] for p in knn) / args.steps, "launches_per_step": len(knn) / args.steps})
        roof["secondary"] = sec
    res = {"metric": "ray-samples/sec (kNN+SDF+render, evaluation render fast=-1)", "value": samples / dt, "unit": "ray-samples/s", "n_gpus": world,
           "steps": args.steps, "warmup": args.warmup, "ms_per_step": dt / args.steps * 1e3, "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
           "dtype": "f32", "data": "synthetic",
           "config": {"workload": f"evaluation render (train.py:399-472 / eval_spurfies.py:276-292 chunks): {args.points} neural points, {args.rays} rays per chunk and GPU, "
                                  f"full error-bounded sampler (up to 5 iterations of 128 samples/ray) + 98 main samples/ray, SDF + normals + colour + compositing, no_grad; prior = {args.prior}",
                      "mode": "eval", "outputs": args.eval_outputs, "launch": "one hipGraph replay per chunk" if args.graph else "eager launches", "rays_per_gpu": args.rays, "neural_points": args.points, "prior": args.prior, "parallelism": f"chunk-sharded dp{world}",
                      "sampler_iterations_realised": {"mean": float(np.mean(iters)), "min": int(min(iters)), "max": int(max(iters))},
                      "rays_per_s": args.rays * world * args.steps / dt,
                      "host_syncs_per_step": "none inside the forward (device-side loop control of the sampler, worst-case buffers + device counts); this bench reads the realised iteration count back once per chunk"},
           "roofline": roof, "dist": dist_info}
    if rank == 0:
        sweep = None
        if args.sweep_resolution > 0:       # the mesh-extraction entry (plots.py:188-287): get_sdf_eval over the reference-sized grid, chunks back to back
            b = scene["base_radius"] * 1.25
            grid = surface.get_grid(None, args.sweep_resolution, input_min=np.asarray([-b] * 3), input_max=np.asarray([b] * 3), eps=0.0)
            with torch.no_grad():
                model.get_sdf_eval(grid["grid_points"][:100000].to(device))          # warm-up chunk (allocator pools)
                torch.cuda.synchronize()
                ops.profile_start(tags=("geo",))
                t0 = time.perf_counter()
                vol_d = model.sdf_eval_grid(*grid["xyz"])          # what surface.sdf_volume(model.get_sdf_eval, grid) runs
                torch.cuda.synchronize()
                td = time.perf_counter() - t0
                vol = vol_d.cpu().numpy()
                ts = time.perf_counter() - t0
                gp = [p for p in ops.profile_stop() if p["pairs"] > 0]
            sweep = {"grid_points": int(vol.size), "resolution": args.sweep_resolution, "seconds": td, "value": vol.size / td, "unit": "points/s",
                     "seconds_incl_d2h": ts, "d2h_gb_per_s": vol.size * 4 / max(ts - td, 1e-9) / 1e9, "defined_fraction": float((vol != 1000.0).mean()),
                     "note": "PointVolSDF.sdf_eval_grid (the path surface.sdf_volume takes for the product model): grid points generated on the device from the "
                             "three axes, occupancy pre-filter (spf_grid_sweep_hits), 4 M-point chunks of the compacted hits; `seconds` = volume resident "
                             "in HBM, `seconds_incl_d2h` = with the one pageable copy of the float32 volume to the host (PCIe-inclusive)"}
            if gp:
                ms, pairs = sum(p["ms"] for p in gp), sum(p["pairs"] for p in gp)
                sweep["geo_kernel"] = {"achieved": pairs * F_FWD / (ms * 1e-3) / 1e12, "frac": pairs * F_FWD / (ms * 1e-3) / 1e12 / geo_peak(ops.geo_mode()), "unit": "TFLOP/s",
                                       "pairs": pairs, "kernel_ms_total": ms}
        res["sdf_eval_sweep"] = sweep
        image = None
        if args.image[0] > 0 and args.image[1] > 0:       # the full-image evaluation loop (864 chunks of 512 pixels at 576 x 768) as a stream
            from spurfies_amd.eval_graph import ImageRenderer

            H, W = args.image
            ys, xs = torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij")
            uv_all = torch.stack([xs, ys], -1).reshape(1, -1, 2).float().to(device)              # datasets/dtu.py:100-103 pixel order, uv = (x, y)
            r = ImageRenderer(model, args.rays, fast=-1, graph=args.graph)
            view = {"uv": uv_all, "pose": torch.from_numpy(scene["poses"][0])[None].to(device), "intrinsics": K}
            r(dict(view, uv=uv_all[:, : 4 * args.rays]), 4 * args.rays)                           # warm-up (capture, allocator pools) on four chunks
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            img = r(view, H * W)
            torch.cuda.synchronize()
            ti = time.perf_counter() - t0
            acc = img["depth_values"]
            image = {"height": H, "width": W, "pixels": H * W, "chunks": (H * W + args.rays - 1) // args.rays, "rays_per_chunk": args.rays, "seconds": ti,
                     "images_per_s": 1.0 / ti, "rays_per_s": H * W / ti, "ms_per_chunk": ti / ((H * W + args.rays - 1) // args.rays) * 1e3,
                     "launch": "one hipGraph launch per chunk (cursor + uv gather + forward + scatter into the merged image)" if args.graph else "eager launches per chunk",
                     "finite": bool(torch.isfinite(img["rgb_values"]).all().item()), "mean_depth": float(acc.mean().item()),
                     "note": "pixel coordinates resident on the device, outputs written into pre-allocated [H*W, ...] tensors by the chunk itself; no per-chunk host copy / list / cat"}
        res["image_render"] = image
        res["cpu_baseline"] = None if (args.no_cpu_baseline or world > 1) else eval_cpu_baseline(scene, min(args.cpu_rays, 128))
        print(json.dumps(res), flush=True)
    if world > 1:
        torch.distributed.barrier()
        torch.distributed.destroy_process_group()


# sources of operators that the measured steps do not run (training operators with 8-bit saved activations; last section of the header)
OTHER_SOURCES = ("act8.hip", "norm.hip", "saved8.h", "wgrad8.hip")
OTHER_SECTION = " * Training operators of normalised MLP layers"


def csrc_digest():
    """sha256 over the sources of the measured steps' kernels (spurfies_amd/csrc/*, include/spurfies_hip.h, both without OTHER_SOURCES) and the compiler flags: the
    identity of the KERNEL code behind this bench's figures.  The counter / power collections under profiles/ record it (tools/pmc_traffic.py,
    tools/power_probe.py); a collection whose digest differs from the running tree's is stale evidence and is not quoted."""
    import hashlib

    h = hashlib.sha256()
    folder = os.path.join(ROOT, "spurfies_amd", "csrc")
    for name in sorted(os.listdir(folder)):
        if name not in OTHER_SOURCES:
            h.update(name.encode())
            h.update(open(os.path.join(folder, name), "rb").read())
    h.update(b"spurfies_hip.h")
    h.update(open(os.path.join(ROOT, "include", "spurfies_hip.h"), "rb").read().split(OTHER_SECTION.encode())[0])
    from spurfies_amd import build as _build

    h.update(" ".join(_build.FLAGS).encode())          # the compiler flags are part of the kernels' identity (-amdgpu-mfma-vgpr-form and the like)
    return h.hexdigest()


def committed_evidence(kind):
    """Newest profiles/r*_{kind}.json whose recorded `csrc_sha256` is the running tree's -> (record, file name), else (None, reason)."""
    want = csrc_digest()
    pdir = os.path.join(ROOT, "profiles")
    names = sorted((n for n in os.listdir(pdir) if n.endswith(kind + ".json")), reverse=True) if os.path.isdir(pdir) else []
    stale = []
    for name in names:
        try:
            rec = json.load(open(os.path.join(pdir, name)))
        except Exception:
            continue
        if rec.get("csrc_sha256") == want:
            return rec, name
        stale.append(name)
    return None, (f"no profiles/*{kind}.json was collected on this tree's kernel sources (csrc sha256 {want[:12]}...; "
                  f"{len(stale)} older collection(s) ignored as stale)")


def workload_name(points, scenes):
    if scenes > 1:
        return f"BASELINE.json configs[3] shape: {scenes} scenes optimised concurrently (round-robin, one ray-sharded group), each "
    if points >= 100000:
        return "BASELINE.json configs[4] shape (dense cloud, large ray batches) on a synthetic scene: "
    if points >= 40000:
        return "BASELINE.json configs[2] shape (garden-like cloud in the +-2 grid) on a synthetic scene: "
    return "BASELINE.json configs[1] shape (DTU scan24 3-view optimisation, 1024-ray batches) on a synthetic scene: "


def measure_train(args, ctx, w):
    """One workload `w` = {points, spacing, rays_total, scenes, steps, warmup, sustained, light, strong, local} on the ranks of `ctx`
    -> the contract's result dict.  light: an `extra` record — no MFMA-shape autotune (the main record's choice stands), no A/B, no secondary
    rooflines, no CPU baseline."""
    from spurfies_amd import ops
    from spurfies_amd.train import MultiSceneTrainer

    world, rank, device, dist_info = ctx["world"], ctx["rank"], ctx["device"], ctx["dist"]
    a = argparse.Namespace(**vars(args))
    a.points, a.spacing, a.scenes = w["points"], w["spacing"], w["scenes"]
    strong, light = w["strong"], w["light"]
    steps, warmup, n_sust = w["steps"], w["warmup"], w["sustained"]
    rays_total = w["rays_total"]
    if rays_total % world:
        raise SystemExit(f"{rays_total} rays per step must be a multiple of the {world} ranks")
    rays_local = rays_total // world
    # strong scaling = ONE batch shared by the ranks: the ranks then draw the sampler's CPU random numbers batch-wide and keep their rows, so the
    # N-GPU run is the same optimisation as the 1-GPU run of that batch (cheap there: the batch does not grow with N).  Weak scaling grows the
    # batch with N; batch-wide draws would cost every rank N times the host-side random numbers (5 ms at 8 x 1024 rays): per-rank streams.
    a.exact_draws = bool(args.exact_draws or strong)
    torch.manual_seed(0)
    # small per-rank batches are host-bound in eager mode (the host needs ~2 ms to enqueue the ~40 launches of a step the GPU runs in ~1 ms
    # at 128 rays: profiles/r04_strong_proxy.json): forward + loss + backward replay as hipGraphs there unless --no-graph
    use_graph = (args.graph or (rays_local <= 256 and not args.no_graph)) and not args.sync
    scenes = [build_scene_step(a, seed, device, world, use_graph) for seed in range(a.scenes)]
    scene, model, step = scenes[0]
    n_batches = warmup + steps + max(n_sust, 0)
    batches = [make_batches(sc, min(n_batches, 64), rays_total, rank, world, device, seed=12345 + i, local=w["local"]) for i, (sc, _, _) in enumerate(scenes)]
    multi = MultiSceneTrainer([st for _, _, st in scenes], n_streams=2, device=device) if a.scenes > 1 else None

    def run_step(i):
        if multi is not None:
            return multi.step([b[i % len(b)] for b in batches])[0], None
        return step(*batches[0][i % len(batches[0])])

    def sync():
        if world > 1:
            torch.distributed.barrier()
        torch.cuda.synchronize()

    # host side of the step = a few hundred tiny torch ops: with the intra-op pool enabled a strided slice of the draws costs tens of
    # milliseconds (thread wake-ups); the reference pins one thread as well (train.py:24).  cpu_baseline sets its own thread counts.
    torch.set_num_threads(1)
    # MFMA shape of the dominant kernel: chosen on THIS box on a warm chip — a few untimed steps first (the clock each shape holds differs
    # between a cold and a loaded chip), then both shapes timed A B B A twice (TrainStep.autotune_geo_engine); all before the W warm-up steps
    tune = None
    if args.geo_engine == "auto" and not light:
        for i in range(40):                        # forward + backward passes only: no optimiser step, nothing captured yet in --graph mode
            step._forward_backward(dict(batches[0][i % len(batches[0])][0]), batches[0][i % len(batches[0])][1])
        tune = step.autotune_geo_engine(*batches[0][0])
    elif args.geo_engine != "auto":
        ops.set_geo_mode(args.geo_engine)
    engine = ops.geo_mode()
    torch.manual_seed(1 if (a.exact_draws or world == 1) else 1 + rank)
    t_w = time.perf_counter()
    for i in range(warmup):
        run_step(i)
    # ---- settle: the chip's clock under a continuous load is lower than in the first tenths of a second (power-averaging window); a 20-step
    # region right behind a short warm-up read 6.7 % faster than the 200-step region behind it (BENCH_r04).  So the same step runs UNTIMED
    # for >= args.settle seconds more (extra warm-up, whatever --warmup says) before the contract region; both figures stay in the line.
    sync()
    # Python's cyclic collector is kept out of the timed regions (a generation-2 pass over this process's ~10^6 objects takes ~0.1 s: one of
    # them inside a 40-step region doubled its reading); collected once HERE — in front of the settle phase, not between it and the timed region:
    # 0.1 - 0.3 s of idle GPU there let the chip drop its clock state, and the first steps of a 20-step region paid for the ramp (+2 - 3 %)
    import gc

    gc_was = gc.isenabled()
    if args.gc == "off":
        gc.collect()
        gc.disable()
    settle = 0
    if args.settle > 0:
        # The NUMBER of settle steps must be the same on every rank (each step holds collectives at world > 1: a rank that ran one step more than
        # its peers would wait for them forever — an earlier time-bounded loop did exactly that on two ranks): ten probe steps are timed, every rank
        # derives a count from its own clock and the ranks agree on the largest.
        probe = 10
        t_s = time.perf_counter()
        for _ in range(probe):
            run_step(warmup + settle)
            settle += 1
        sync()
        per = max((time.perf_counter() - t_s) / probe, 1e-5)
        more = torch.tensor([max(0, int((args.settle - per * probe) / per) + 1)], device=device, dtype=torch.int64)
        if world > 1:
            torch.distributed.all_reduce(more, op=torch.distributed.ReduceOp.MAX)
        for _ in range(min(int(more.item()), 100000)):
            run_step(warmup + settle)
            settle += 1
        sync()
    first = warmup + settle
    ops.geo_clock(reset=True)                     # in-kernel clock counters of the dominant kernel: zeroed before the timed region
    if not use_graph:
        ops.profile_start(tags=("geo",))          # HIP events around the dominant kernel's launches of the timed region
    for _, _, st_ in scenes:
        if st_.buckets is not None:
            st_.buckets.timing = []               # an event pair around every finish(): the exposed part of the gradient exchange
    sync()
    host_max = 0.0
    t0 = time.perf_counter()
    for i in range(first, first + steps):
        th = time.perf_counter()
        losses, out = run_step(i)
        host_max = max(host_max, time.perf_counter() - th)
    sync()
    dt = time.perf_counter() - t0
    dinfo = None
    if dist_info is not None:
        dinfo = dict(dist_info)
        exposed = [ms for _, _, st_ in scenes if st_.buckets is not None for ms in st_.buckets.exposed_ms()]
        for _, _, st_ in scenes:
            if st_.buckets is not None:
                st_.buckets.timing = None
        nbytes = 4 * step.flat.buffer.numel()
        dinfo.update({
            "allreduce_bytes_per_step": (nbytes + 16) * a.scenes,
            "allreduce_what": f"one flat fp32 gradient buffer of {nbytes} B per scene step (" +
                              ("ONE dense all-reduce behind the two graph replays" if use_graph else "4 buckets, reduced asynchronously as the backward completes them") +
                              ") + 16 B of loss normalisers between forward and loss",
            "buckets_bytes": step.buckets.bytes_per_step() if step.buckets is not None else None,
            "bucket_order_last_step": list(step.buckets.log) if (step.buckets is not None and not use_graph) else None,
            "finish_ms_per_step": (sum(exposed) / steps) if exposed else None,
            "finish_what": "HIP events on rank 0's compute stream around BucketedAllReduce.finish() (launch of the last bucket + wait for all): "
                           "the part of the exchange not hidden behind the backward"})
    loss_last = float(losses["loss"].item())
    clk = ops.geo_clock(reset=True).get(("split_w" if engine == "h2" else engine, True))       # the clock the chip held under the dominant kernel DURING the timed region (h2 = the 32x32x16 kernel: its counter slot)
    if use_graph and a.scenes == 1:
        # events cannot be placed inside a hipGraph replay: time the dominant kernel over eager forward+backward passes of
        # the SAME batches right after the timed region (same kernels, same inputs; no optimiser step)
        ops.profile_start(tags=("geo",))
        nb = len(batches[0])
        for i in range(first, first + steps):
            step._forward_backward(dict(batches[0][i % nb][0]), batches[0][i % nb][1])
        sync()
    prof = ops.profile_stop()
    tmax = torch.tensor([dt], device=device, dtype=torch.float64)
    if world > 1:
        torch.distributed.all_reduce(tmax, op=torch.distributed.ReduceOp.MAX)
    dt = float(tmax.item())
    sustained = None
    if n_sust > 0:        # the same step over a >= 1 s region, reported beside the contract region
        if not use_graph:
            ops.profile_start(tags=("geo",))      # the SAME instrumentation as the contract region (its events cost ~1 % of a step): the two
        sync()                                    # figures then differ by settling only; this region's events are discarded
        t1 = time.perf_counter()
        for i in range(first + steps, first + steps + n_sust):
            run_step(i)
        sync()
        ts = torch.tensor([time.perf_counter() - t1], device=device, dtype=torch.float64)
        if not use_graph:
            ops.profile_stop()
        if world > 1:
            torch.distributed.all_reduce(ts, op=torch.distributed.ReduceOp.MAX)
        sustained = float(ts.item()) / n_sust * 1e3
    if gc_was:
        gc.enable()

    if not use_graph and a.scenes == 1 and not light:          # the other regimes' kernels, timed over separate steps (outside both timed regions)
        ops.profile_start(tags=("color_fwd", "color_bwd", "wgrad", "knn", "render_fwd", "render_bwd"))
        for i in range(first, first + min(steps, 10)):
            run_step(i)
        prof += ops.profile_stop()

    # ---- roofline: dominant kernel = geo_pairs_x3_kernel<true> of the main pass (the largest with-Jacobian launch per step) ----
    geo = [p for p in prof if p["tag"] == "geo"]
    main_ = [p for p in geo if p["with_grad"] and p["rows"] >= rays_local * 2]
    roof = None
    # HBM bytes per launch need a rocprofv3 --pmc pass around the process: they cannot be collected from inside this run.  The figure below
    # is a committed collection (tools/pmc_traffic.py) — quoted ONLY when it was collected on this tree's kernel sources (csrc digest), on
    # the same workload; otherwise null, with the reason.
    traffic, traffic_src = None, None
    if not light:
        rec, name = committed_evidence("pmc_traffic")
        if rec is None:
            traffic_src = name
        elif not (rec["config"].get("points") == a.points and rec["config"].get("rays") == rays_local and rec["config"].get("prior", "kaiming") == a.prior):
            traffic_src = f"profiles/{name} is of this code but of another workload ({rec['config']}): not quoted"
        else:
            want = "geo_pairs_x3_kernel<true>" if ops.geo_mode() == "split" else ("geo_pairs_x3w_kernel<true, 2, true>" if ops.geo_mode() == "h2" else "geo_pairs_x3w_kernel<true, 3, false>")
            hit = [v for k, v in rec["kernels"].items() if want in k] or [v for k, v in rec["kernels"].items() if "geo_pairs_x3" in k and "<true>" in k]
            if hit:
                traffic = hit[0]["hbm_bytes_max_corrected"]
                traffic_src = (f"profiles/{name}: rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE (separate passes, gfx950 corrections) of the same workload on THIS "
                               "tree's kernel sources (csrc sha256 matches), collected on another box and committed — not measured in this run")
    if main_:
        ms = sum(p["ms"] for p in main_)
        pairs = sum(p["pairs"] for p in main_)
        ach = pairs * (F_FWD + F_JAC) / (ms * 1e-3) / 1e12
        kname = "geo_pairs_x3_kernel<true>" if engine == "split" else ("geo_pairs_x3w_kernel<true, 2, true>" if engine == "h2" else "geo_pairs_x3w_kernel<true, 3, false>")
        shape = "v_mfma_f32_16x16x32_bf16" if engine == "split" else ("v_mfma_f32_32x32x16_f16" if engine == "h2" else "v_mfma_f32_32x32x16_bf16")
        peak = geo_peak(engine)
        roof = {"bound": "mfma", "achieved": ach, "peak": peak, "unit": "TFLOP/s", "frac": ach / peak,
                "peak_basis": (f"algorithmic fp32 FLOP/s; each fp32 product = 3 exact fp16 piece products (two fp16 pieces per operand, main + cross accumulators) on the "
                               f"matrix pipe (this run: {shape}), so the ceiling is the dense fp16 MFMA peak (2516.6 TFLOP/s) / 3; for scale, the fp32-MFMA peak is 157.3 TFLOP/s"
                               if engine == "h2" else
                               f"algorithmic fp32 FLOP/s; each fp32 product = 6 exact bf16 piece products on the bf16 matrix pipe (this run: {shape}), so the "
                               "ceiling is the dense bf16 MFMA peak (2516.6 TFLOP/s) / 6; for scale, the fp32-MFMA peak is 157.3 TFLOP/s"),
                "achieved_over_fp32_mfma_peak": ach / PEAK_F32_MFMA_TFLOPS,
                "achieved_over_bf16x3_ceiling": ach / PEAK_SPLIT_TFLOPS,          # rounds 1 - 5 priced `frac` against this (bf16 peak / 6 = 419.4): comparable across rounds
                "sustainable": None if light else sustainable_ceiling(ach, engine),
                "held_clock": held_clock(ach, clk, peak),
                "engine": {"selected": engine, "mfma": shape, "how": ("timed both shapes on this box after 40 untimed passes, before the warm-up steps (main-pass launch; the shape alternates every pass, A B B A x 10)" if tune else ("the main record's choice" if light else "--geo-engine")),
                           "autotune_ms": tune},
                "traffic": traffic, "traffic_source": traffic_src, "kernel": kname + " (+ geo_point_reduce_kernel, < 1 % of the launch)",
                "timing": ("HIP events over eager passes of the timed batches, right after the timed region (events cannot sit inside a "
                           "hipGraph replay)") if use_graph else "HIP events over the timed region", "launches": len(main_), "avg_ms": ms / len(main_),
                "pairs_per_launch": pairs / len(main_), "flop_per_pair": F_FWD + F_JAC}
        if not light:
            roof["secondary"] = secondary_rooflines(prof, rays_local)
            if args.ab_reps > 0 and a.scenes == 1:
                roof["ab"] = engine_ab(step, batches[0], first, args.ab_reps, rays_local, sync)
    spr = SAMPLES_PER_RAY * rays_total * a.scenes
    counts = model.stats.get("counts")
    if use_graph:
        launch = ("hipGraph replay (fwd+loss+bwd) + 2 eager launches (clip + non-finite guard + Adam)" if world == 1 else
                  "two hipGraph replays ([forward + counts] | 16-byte count all-reduce | [loss + backward]), dense gradient all-reduce, 2 eager launches (clip + guard + Adam)")
    else:
        launch = "eager, reference-shaped (one host read-back)" if args.sync else "eager launches, no host synchronisation (one host-to-device copy of the sampler's CPU random draws per step)"
    res = {
        "metric": "ray-samples/sec (kNN+SDF+render, train step)", "value": spr * steps / dt,
        "unit": "ray-samples/s", "n_gpus": world, "steps": steps, "warmup": warmup, "ms_per_step": dt / steps * 1e3,
        "higher_is_better": True, "scaling": "strong" if strong else "weak", "vs_baseline": None, "dtype": "f32", "data": "synthetic",
        "config": {"workload": workload_name(a.points, a.scenes) +
                               f"{a.points} neural points, {rays_total} rays/step over {world} GPU(s) x (128 sampler + 98 main) samples, fast=1 optimisation step "
                               f"(fwd+bwd+clip+Adam)" + (" incl. find_surface_points + the multi-view feature-consistency loss on synthetic local_data (the DTU recipe's local_weight 0.5)" if w["local"] else "") +
                               f"; prior = {a.prior}",
                   "rays_per_gpu": rays_local, "rays_per_step": rays_total, "scenes": a.scenes, "neural_points": a.points, "k": 8, "max_shading_pts": 80,
                   "prior": a.prior, "parallelism": f"ray-sharded dp{world}", "local_data": bool(w["local"]),
                   "valid_points_last_step": model.stats.get("valid_points", int(counts[0].item()) if counts is not None else None),
                   "pairs_last_step": model.stats.get("pairs", int(counts[1].item()) if counts is not None else None),
                   "host_syncs_per_step": 1 if args.sync else 0,
                   "settle_steps_untimed": settle, "settle_seconds": args.settle,
                   "sampler_draws": "CPU generator, reference call order" + ("" if world == 1 else ("; batch-wide per rank, own rows kept (--exact-draws)" if a.exact_draws
                                                                                                   else "; per-rank streams, own rays only")),
                   "arithmetic": arithmetic_text(engine),
                   "launch": launch},
        "roofline": roof, "dist": dinfo,
        "sustained_ms_per_step": sustained, "sustained_steps": n_sust if sustained is not None else 0,
        "loss_last": loss_last, "host_enqueue_ms_max": host_max * 1e3,
    }
    del scenes, batches, multi, step, model
    torch.cuda.empty_cache()
    return res, scene


def main():
    args = parse()
    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:      # the driver's command shape: `python bench.py --gpus N` — start the ranks ourselves
        raise SystemExit(self_launch(args))
    if args.mode == "eval":
        return main_eval(args)
    world, rank, device, dist_info = init_ranks(args)
    if world != args.gpus:
        raise SystemExit(f"--gpus {args.gpus} but the launcher started {world} ranks")

    from spurfies_amd import ops

    ops.geo_clock_enable(True)                    # this process is the one measuring caller of the library's held-clock counters
    off = {t.strip() for t in args.off.split(",") if t.strip()}
    if off - {"fused_sampler", "defer_loss", "merge_head"}:
        raise SystemExit(f"--off: unknown switches {sorted(off)}")
    ops.set_fused_sampler("fused_sampler" not in off)
    ops.set_loss_finalize_deferred("defer_loss" not in off)
    ops.set_head_wgrad_merged("merge_head" not in off)
    ctx = {"world": world, "rank": rank, "device": device, "dist": dist_info}
    # ---- what N GPUs measure: by default the SAME workload as N = 1 — BASELINE.json configs[1], one 1024-ray batch per step, rank r renders
    # rays r::N of it (strong scaling) — so that the driver's N = 1, 2, 4, 8 lines are one scaling curve of a
    # BASELINE config.  --weak: --rays rays PER GPU (the batch grows with N).
    strong = not args.weak
    rays_total = (args.global_rays or args.rays) if strong else args.rays * world
    main_w = {"points": args.points, "spacing": args.spacing, "scenes": args.scenes, "rays_total": rays_total, "steps": args.steps, "warmup": args.warmup,
              "sustained": args.sustained, "light": False, "strong": strong, "local": False}
    res, scene = measure_train(args, ctx, main_w)
    extras = []
    want_extras = args.extras == "on" or (args.extras == "auto" and world > 1)
    want_local = args.local or (args.extras != "off" and world == 1 and args.mode == "train")
    if want_extras and args.scenes == 1:
        es, ew = max(5, args.steps // 2), 2
        # the dense cloud with 4096-ray batches, strong-scaled over the same ranks
        extras.append({"points": args.c4_points, "spacing": 0.0125, "scenes": 1, "rays_total": args.c4_rays, "steps": es, "warmup": ew, "sustained": 0, "light": True,
                       "strong": True, "local": False, "record": "BASELINE.json configs[4], strong-scaled over the same ranks"})
        # the weak-scaling figure of the main workload (1024 rays PER GPU)
        extras.append({"points": args.points, "spacing": args.spacing, "scenes": 1, "rays_total": args.rays * world, "steps": es, "warmup": ew, "sustained": 0,
                       "light": True, "strong": False, "local": False, "record": "weak scaling of the main workload (--rays rays PER GPU; no BASELINE config has such batches)"})
    if want_local and args.scenes == 1:
        # the DTU recipe's real step (pointneus_disent.py:727-763, feat_utils.py:377-451; config/ours.yaml local_weight 0.5): find_surface_points + the
        # feature-consistency loss on synthetic per-view feature maps, every step
        extras.insert(0, {"points": args.points, "spacing": args.spacing, "scenes": 1, "rays_total": rays_total, "steps": args.steps, "warmup": args.warmup,
                          "sustained": 0, "light": True, "strong": strong, "local": True,
                          "record": "the main workload with the DTU recipe's feature-consistency loss (local_weight 0.5) on every step: find_surface_points + "
                                    "get_local_loss as one HIP launch inside the step (32-channel synthetic feature maps of 3 views at half resolution)"})
    res["extra"] = []
    # The extra records must never cost the contract line: a rank that fails or hangs inside one of them (a collective its peers never reach)
    # would leave rank 0 without anything to print.  Every rank arms the same timer; when it fires, rank 0 prints the main record with what
    # the extras have produced so far and all ranks leave (os._exit: no second program is started, nothing waits for the stuck collective).
    import threading

    line_lock, line_done = threading.Lock(), [False]     # the JSON line is printed exactly once, by the main thread or by the timer thread

    def abandon(code=0):
        """code: 0 when the timer fired (the contract line is complete: the run counts), 3 from the rank whose own extra record raised."""
        with line_lock:
            if not line_done[0] and rank == 0:
                line_done[0] = True
                out = dict(res, extra=list(res["extra"]) + [{"record": "extras abandoned", "error": f"an extra record failed or did not finish within {limit:.0f} s "
                                                                                                     "(SPF_EXTRAS_TIMEOUT); the main record above is complete"}])
                out.setdefault("cpu_baseline", None)
                print(json.dumps(out), flush=True)
            os._exit(code)

    limit = float(os.environ.get("SPF_EXTRAS_TIMEOUT", "300"))
    timer = threading.Timer(limit, abandon) if ((extras or want_local) and limit > 0) else None
    if timer is not None:
        timer.daemon = True
        timer.start()
    for w in extras:
        try:
            r, _ = measure_train(args, ctx, w)
        except Exception as e:  # noqa: BLE001 — recorded in the line; at world > 1 the peers' timer ends the run if they wait for this rank
            import traceback

            print(f"[bench] rank {rank}: extra record {w['record']!r} failed:\n{traceback.format_exc()}", file=sys.stderr, flush=True)
            res["extra"].append({"record": w["record"], "error": repr(e)[:400]})
            if world > 1:
                abandon(3)             # the peers are inside collectives this rank will not join: leave now (non-zero: this rank failed), their timers end them
            continue
        keep = {"record": w["record"], **{k: r[k] for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "scaling", "config", "dist", "loss_last")}}
        keep["roofline"] = None if r["roofline"] is None else {k: r["roofline"][k] for k in ("bound", "achieved", "peak", "unit", "frac", "avg_ms", "pairs_per_launch", "kernel")}
        res["extra"].append(keep)
        if w["local"]:
            res["ms_per_step_with_local"] = r["ms_per_step"]
    if want_local and args.scenes == 1 and world == 1:      # (same switch: the N = 1 line's second short record)
        try:
            res["extra"].append(eval_chunk_record(args, device, scene))
        except Exception as e:  # noqa: BLE001
            import traceback

            print(f"[bench] the evaluation-chunk record failed:\n{traceback.format_exc()}", file=sys.stderr, flush=True)
            res["extra"].append({"record": "evaluation render", "error": repr(e)[:400]})
    if timer is not None:
        timer.cancel()
    if rank == 0:
        res["cpu_baseline"] = None if (args.no_cpu_baseline or world > 1) else cpu_baseline(scene, args.cpu_rays)     # N = 1 only
        with line_lock:
            if not line_done[0]:
                line_done[0] = True
                print(json.dumps(res), flush=True)
    if world > 1:
        torch.distributed.barrier()
        torch.distributed.destroy_process_group()


def arithmetic_text(engine):
    """config.arithmetic of the contract line: which piece form every dense kernel of THIS process computes in (ops._H2 / ops._ARITH as they stand)."""
    from spurfies_amd import ops

    h2 = [k for k in ("color_fwd", "color_bwd", "wgrad", "rhead_fwd", "rhead_bwd")
          if ops._arith_of(ops._ARITH["color" if k.startswith("color") else ("rhead" if k.startswith("rhead") else "wgrad")], k) == 3]
    names = {"color_fwd": "colour trunk forward", "color_bwd": "colour trunk backward", "wgrad": "weight-gradient GEMMs", "rhead_fwd": "per-point head forward",
             "rhead_bwd": "per-point head backward"}
    b3 = [names[k] for k in names if k not in h2]
    h2 = [names[k] for k in h2] + (["geometry kernel (engine h2)"] if engine == "h2" else [])
    if engine != "h2":
        b3.append(f"geometry kernel (engine {engine})")
    txt = "fp32 storage and accumulation throughout; every fp32 product of a dense kernel is formed exactly from 16-bit pieces on the matrix pipe. "
    if h2:
        txt += ("H2 — two fp16 pieces per operand (22 mantissa bits), 3 exact fp16 piece products per fp32 product, fp32 accumulators (MLP tiles: main + 2^-11 x cross, "
                "combined once per layer; gradient rows / weight-gradient operands block-scaled by powers of two): " + ", ".join(h2) + ". Measured error against float64 "
                "equal to the fp32-MFMA twins' (tools/engine_accuracy.py, tools/color_accuracy.py, tests/test_gpu_wgrad.py). ")
    if b3:
        txt += "bf16 x 3 — three bf16 pieces per operand, 6 exact bf16 piece products (<= 2 ulp per product): " + ", ".join(b3) + "."
    return txt


def sustainable_ceiling(achieved_tflops, engine="split_w"):
    """`frac` is priced against the 2.4 GHz data-sheet peak.  What the chip SUSTAINS on this instruction mix was measured with socket power beside
    it (tools/power_probe.py -> profiles/r*_power.json; another box, labelled): every dense kernel of the step runs near the 1.40 kW cap with
    the clock pulled down to ~2.0 GHz (power-limited); the library's own GEMM loop run alone peaks at ~75 % matrix-pipe duty / full clock with
    the lightest epilogue and loses clock faster than it gains duty when made denser.  Quoted only from a collection made on THIS tree's kernel
    sources (csrc digest); otherwise {'peak': None, 'why': ...}."""
    rec, name = committed_evidence("power")
    if rec is None:
        return {"peak": None, "frac": None, "why": name}
    loads = rec.get("loads", {})
    pre = "h2_loop_" if engine == "h2" else "x3_loop_"          # the GEMM loop in the run's own piece form
    best = max((v.get("tflops_fp32_equiv", 0.0) for k, v in loads.items() if k.startswith(pre)), default=0.0)
    if best <= 0.0:
        return {"peak": None, "frac": None, "why": f"profiles/{name} holds no {pre}* load"}
    geo = loads.get("geo_h2" if engine == "h2" else "geo_split_w", {})
    return {"peak": best, "unit": "TFLOP/s", "frac": achieved_tflops / best,
            "what": f"highest algorithmic fp32 rate the library's {'H2 (three fp16 piece products)' if engine == 'h2' else 'bf16-piece'} GEMM loop sustained when run ALONE (tools/micro/x3_loop_rate.hip, three epilogue "
                    "variants), with socket power sampled beside it",
            "power_cap_w": rec.get("power_cap_w"), "geo_kernel_power_w": geo.get("power_w_mean"), "geo_kernel_ghz": geo.get("ghz_in_kernel"),
            "loop_variants": {k: {kk: v.get(kk) for kk in ("what", "tflops_fp32_equiv", "mfma_duty", "ghz", "power_w_mean")} for k, v in loads.items() if k.startswith(pre)},
            "source": f"profiles/{name} — collected on ANOTHER box (hwmon power1_input of the HIP device's PCI card, 100 Hz) on this tree's kernel sources "
                      "(csrc sha256 matches), committed; not measured in this run"}


def held_clock(achieved_tflops, clk, peak=None):
    """The shader clock the dominant kernel HELD inside the timed region, measured by the kernel itself (s_memtime / s_memrealtime stamps
    of every workgroup, spf_geo_clock_read) in this run, and the roofline fraction at that clock."""
    if not clk:
        return None
    ghz = clk["ghz"]
    peak = peak or PEAK_SPLIT_TFLOPS
    return {"ghz": ghz, "nominal_ghz": 2.4, "peak_at_held_clock": peak * ghz / 2.4, "frac_at_held_clock": achieved_tflops / (peak * ghz / 2.4),
            "workgroups": clk["workgroups"], "mean_us_per_workgroup": clk["mean_us_per_workgroup"],
            "source": "measured in this run: in-kernel s_memtime / s_memrealtime stamps of every workgroup of the dominant kernel's launches in the timed region "
                      "(spf_geo_clock_read); `frac` above stays priced at 2.4 GHz"}


def engine_ab(step, batches, first, reps, rays_local, sync):
    """Two arithmetic modes of the dominant kernel on the SAME batches in this process, after the timed regions — the run's own (h2: three fp16 piece
    products per fp32 product) against the six-product bf16 kernel on the same 32x32x16 tiles, or, for a bf16 run, the two bf16 MFMA shapes: legs A B B A of
    `reps` forward + backward passes each (no optimiser step: every leg sees the same parameters and pair counts), main-pass launch timed with HIP events,
    clock read from the kernels' own counters."""
    from spurfies_amd import ops

    prev = ops.geo_mode()
    A, B = ("h2", "split_w") if prev == "h2" else ("split", "split_w")
    acc = {A: {"ms": 0.0, "pairs": 0.0, "n": 0, "cyc": 0.0, "ticks": 0.0}, B: {"ms": 0.0, "pairs": 0.0, "n": 0, "cyc": 0.0, "ticks": 0.0}}
    try:
        for mode in (A, B, B, A):
            ops.set_geo_mode(mode)
            step._forward_backward(dict(batches[first % len(batches)][0]), batches[first % len(batches)][1])
            ops.geo_clock(reset=True)
            ops.profile_start(tags=("geo",))
            for i in range(reps):
                b = batches[(first + i) % len(batches)]
                step._forward_backward(dict(b[0]), b[1])
            sync()
            rows = [p for p in ops.profile_stop() if p["with_grad"] and p["rows"] >= 2 * rays_local]
            c = ops.geo_clock(reset=True).get(("split_w" if mode == "h2" else mode, True))
            a = acc[mode]
            a["ms"] += sum(p["ms"] for p in rows)
            a["pairs"] += sum(p["pairs"] for p in rows)
            a["n"] += len(rows)
            if c:
                a["cyc"] += c["ghz"] * c["workgroups"] * c["mean_us_per_workgroup"]
                a["ticks"] += c["workgroups"] * c["mean_us_per_workgroup"]
    finally:
        ops.set_geo_mode(prev)
    out = {"order": "A B B A, %d forward+backward passes per leg on the timed batches, after the timed regions" % reps}
    shapes = {"split": ("v_mfma_f32_16x16x32_bf16", 6.0), "split_w": ("v_mfma_f32_32x32x16_bf16", 6.0), "h2": ("v_mfma_f32_32x32x16_f16", 3.0)}
    for mode in (A, B):
        a = acc[mode]
        if a["n"]:
            ach = a["pairs"] * (F_FWD + F_JAC) / (a["ms"] * 1e-3) / 1e12
            out[mode] = {"mfma": shapes[mode][0], "piece_products_per_fp32_product": int(shapes[mode][1]), "avg_ms": a["ms"] / a["n"], "pairs_per_launch": a["pairs"] / a["n"],
                         "achieved": ach, "frac": ach / (PEAK_BF16_MFMA_TFLOPS / shapes[mode][1]), "held_ghz": (a["cyc"] / a["ticks"]) if a["ticks"] else None, "launches": a["n"]}
    if A in out and B in out:
        out["faster"] = min((A, B), key=lambda m: out[m]["avg_ms"])
    return out


def secondary_rooflines(prof, rays_local):
    """The other regimes of the step, same HIP events: the colour-trunk kernels against the same MFMA ceiling, the kNN and
    compositing kernels against HBM (algorithmic bytes / time / 8 TB/s)."""
    out = []

    def mean(rows, key):
        return sum(r[key] for r in rows) / len(rows)

    for tag, flop, name in (("color_fwd", F_COLOR_FWD, "color_forward_x3_kernel<true>"), ("color_bwd", F_COLOR_BWD, "color_backward_x3_kernel")):
        rows = [p for p in prof if p["tag"] == tag and p["pairs"] > 0]
        if rows:
            ach = sum(p["pairs"] for p in rows) * flop / (sum(p["ms"] for p in rows) * 1e-3) / 1e12
            pk, form = family_peak(tag)
            out.append({"kernel": name, "bound": "mfma", "achieved": ach, "peak": pk, "peak_basis": form, "unit": "TFLOP/s", "frac": ach / pk,
                        "avg_ms": mean(rows, "ms"), "pairs_per_launch": mean(rows, "pairs"), "flop_per_pair": flop})
    wg = [p for p in prof if p["tag"] == "wgrad" and p.get("rows_x_c", 0) > 0 and p.get("problems", 0) >= 3]        # the colour trunk's + head's problems in one launch pair
    if wg:
        # dW[256, C] += G[:rows]^T A[:rows, :C] per problem: 512 rows C FLOP, and both operands are read ONCE from HBM (4 (256 + C) bytes per row) —
        # the kernel is priced against both ceilings and bound by the nearer one
        sec_ = sum(p["ms"] for p in wg) * 1e-3
        tf, gbs = sum(p["rows_x_c"] for p in wg) * 512.0 / sec_ / 1e12, sum(p["operand_floats"] for p in wg) * 4.0 / sec_ / 1e9
        pk, form = family_peak("wgrad")
        hbm_nearer = gbs / PEAK_HBM_GBS >= tf / pk
        out.append({"kernel": "wgrad_split8_batched_kernel (+ its slab reduce launch)", "bound": "hbm" if hbm_nearer else "mfma",
                    "achieved": gbs if hbm_nearer else tf, "peak": PEAK_HBM_GBS if hbm_nearer else pk, "unit": "GB/s" if hbm_nearer else "TFLOP/s",
                    "frac": max(gbs / PEAK_HBM_GBS, tf / pk), "avg_ms": mean(wg, "ms"), "problems_per_launch": mean(wg, "problems"),
                    "hbm": {"achieved": gbs, "peak": PEAK_HBM_GBS, "unit": "GB/s", "frac": gbs / PEAK_HBM_GBS, "bytes_per_launch": sum(p["operand_floats"] for p in wg) * 4.0 / len(wg),
                            "what": "operand bytes (G and A rows, fp32, each read once) / launch time"},
                    "mfma": {"achieved": tf, "peak": pk, "unit": "TFLOP/s", "frac": tf / pk, "peak_basis": form}})
    knn = [p for p in prof if p["tag"] == "knn" and p["slots"] > 1 and p["rays"] == rays_local]        # the main pass (98 samples/ray, SR = 80)
    if knn:
        # 12 B position in + 1 B mask out per sample; per hit slot 4 k B of indices + 16 B (location, sample id) out
        byts = [p["rays"] * p["samples_per_ray"] * 13.0 + p["hit_slots"] * (4.0 * p["k"] + 16.0) for p in knn]
        ach = sum(byts) / (sum(p["ms"] for p in knn) * 1e-3) / 1e9
        out.append({"kernel": "spf_grid_query, main pass (point_slots + hit_slots + knn + ray_valid kernels)", "bound": "hbm", "achieved": ach,
                    "peak": PEAK_HBM_GBS, "unit": "GB/s", "frac": ach / PEAK_HBM_GBS, "avg_ms": mean(knn, "ms"), "hit_slots_per_launch": mean(knn, "hit_slots"),
                    "note": "latency-bound at this size (1e5 samples): ~100 candidate reads per hit slot are L2 hits, not HBM traffic"})
    for tag, bps, name in (("render_fwd", 29.0, "render_forward_kernel"), ("render_bwd", 45.0, "render_backward_kernel")):
        rows = [p for p in prof if p["tag"] == tag]
        if rows:
            ach = sum(p["rays"] * p["slots"] * bps for p in rows) / (sum(p["ms"] for p in rows) * 1e-3) / 1e9
            out.append({"kernel": name, "bound": "hbm", "achieved": ach, "peak": PEAK_HBM_GBS, "unit": "GB/s", "frac": ach / PEAK_HBM_GBS,
                        "avg_ms": mean(rows, "ms"), "bytes_per_slot": bps, "note": "launch-latency-bound: 1024 rays x 80 slots is ~3 MB"})
    return out


if __name__ == "__main__":
    main()
