"""Optimisation step with the reference's recipe (spurfies/train.py:117-189, 330-397, 548-564):
frozen F_geometry/T, Adam over the remaining parameters (lr 5e-4; the reference's first param group
is empty), CosineAnnealingLR(T_max=100000, eta_min=3e-4), grad-norm clip 1.0, NaN/Inf gradient guard.

`TrainStep` is the part of `VolOpt.train_step` that touches the GPU; dataset / checkpoint / logging
plumbing around it is host code outside the hot path.  With `world_size > 1` rays are sharded
across ranks and gradients are summed with one all-reduce of a flat buffer (spurfies_amd/dist.py).
"""
from __future__ import annotations

import numpy as np
import torch

from . import dist as sdist
from . import ops
from .model.loss import VolSDFLoss
from .optim import FlatAdam


def default_loss() -> VolSDFLoss:
    """Weights of config/ours.yaml:15-20."""
    return VolSDFLoss("torch.nn.L1Loss", local_weight=0.5, pseudo_weight=0.5, eikonal_weight=0.001, rgb_weight=1.0, tv_weight=0.01)


class TrainStep:
    N_STAGING = 4            # pinned staging buffers for the CPU-generator draws (sync-free steps run ahead of the GPU)

    def __init__(self, model, loss=None, lr=5.0e-4, grad_clip=True, process_group=None, sync_free=False, use_graph=False, draws="batch", keep_grads=False,
                 fork=None, force_collectives=False):
        """sync_free: static shapes and device-side counts everywhere — no host synchronisation inside the step (the
        default path reads [P, n_pairs] back once per step to size the colour buffers exactly).
        use_graph (implies sync_free): forward + loss + backward (~50 kernel launches) are captured once into a hipGraph
        and replayed; the gradient all-reduce, clipping and Adam stay eager.  Ray-sharded (world > 1): two graphs around the eager
        16-byte count all-reduce, then ONE dense all-reduce of the flat gradient buffer — the mode for small per-rank batches, where
        the host cannot enqueue ~50 launches as fast as the GPU runs them (strong scaling).
        fork (default off): independent passes of the step are issued on side streams (ops.branch) and become parallel branches of the
        captured graph — the pseudo-point pass beside the colour stage (split compositing), the geometry passes' latent scatters beside the
        colour backward; same kernels, same sums.  Measured on MI355X / ROCm 7.2 (profiles/r05_fork_*.txt): the graph executor
        serialises child branches onto a few queues in capture order and every cross-queue edge costs 5 - 10 us, so at 128 rays the forked
        graph is within +-1 % of the single-stream one (0.965 vs 0.957 ms) and LOSES when several scenes' graphs already share the chip
        (11 scenes: 9.4 vs 8.3 ms per round) — what did pay was folding the independent small launches into launches that exist anyway."""
        self.model = model
        # force_collectives (tests / bench on a one-GPU box): with an initialised process group of ONE rank the step still issues everything a
        # ray-sharded step issues — the 16-byte count all-reduce, the bucketed async all-reduces + finish() (eager) or the two-graph form with
        # the dense all-reduce (use_graph) — so that the step's stream semantics run on RCCL itself; the sums over one rank change nothing.
        self.force_collectives = bool(force_collectives)
        self.fork = bool(fork) if fork is not None else False
        sync_free = sync_free or use_graph
        self.sync_free = sync_free
        self.use_graph = use_graph
        self._graph = None
        self._one = None
        self._graph_key = None
        model.sync_free = sync_free
        self._draws = None
        self.loss = loss or default_loss()
        model.freeze_prior()                                    # train.py:151-154
        self.params = [p for p in model.parameters() if p.requires_grad]
        self.flat = sdist.FlatGrads(self.params)                # .grad of every trainable tensor is a view of one buffer
        ops.set_grad_sinks(self.params, on=sync_free)           # sync-free: backward kernels add straight into those views
        self.optimizer = FlatAdam([{"params": [], "lr": 1e-2}, {"params": self.params, "lr": lr}], flat_grads=self.flat)
        self.scheduler = torch.optim.lr_scheduler.CosineAnnealingLR(self.optimizer, T_max=100_000, eta_min=3e-4, last_epoch=-1)
        self.grad_clip = grad_clip
        self.group = process_group
        self.world = sdist.world_size(process_group)
        self.rank = sdist.rank(process_group)
        # ray-sharded batches, draws="batch" (default): every rank issues the reference's CPU-generator calls for the WHOLE batch (same seed,
        # same order) and keeps the rows of its own rays (rank::world, dist.shard_rays), so N ranks over a batch consume exactly the draws
        # one GPU would — at the price of N times the host-side random numbers per rank (5 ms per step at 8 x 1024 rays: more than the GPU
        # step).  draws="local": a rank draws only for its own rays from ITS OWN generator stream (seed the ranks differently): the same
        # distribution, not the same numbers as a single-GPU run — what a throughput run wants.
        if draws not in ("batch", "local"):
            raise ValueError(draws)
        self.draw_world = self.world if draws == "batch" else 1
        model.ray_sampler.shard = (self.rank, self.world) if self.draw_world > 1 else None
        self.buckets = None
        self.collective = self.world > 1 or self.force_collectives
        if self.collective:
            # the all-reduce sums gradients only: replicas must START identical (latents and MLPs are drawn from the local
            # generators in the constructors).  Rank 0's parameters, frozen prior and cloud win.
            sdist.broadcast_model(model, self.optimizer, process_group)
            if sync_free:      # gradients go straight into the flat buffer: bucket by bucket, each all-reduced as soon as it is final
                names = [n for n, p in model.named_parameters() if p.requires_grad]
                self.buckets = sdist.BucketedAllReduce(self.flat, names, process_group, force=self.force_collectives)
        self.iter_step = 0
        self.skipped = 0
        # sync-free steps: the Adam sweep clears the flat gradient buffer behind itself (the next step's optimizer.zero_grad(), train.py:357,
        # without its fill launch); keep_grads=True leaves the clipped gradient readable after a step (tests, debugging)
        self.zero_in_adam = sync_free and not keep_grads
        self._grads_clean = False

    def __call__(self, model_input, ground_truth):
        """model_input: {'intrinsics','uv','pose','local_data'} for THIS rank's rays; returns (loss dict, model outputs)."""
        with ops.scratch_owner(self):      # this step's workspaces are its own, whatever stream (or graph) its launches run in
            return self._step(model_input, ground_truth)

    def _step(self, model_input, ground_truth):
        self.model.train()
        if self.use_graph:
            losses, out = self._graphed_forward_backward(model_input, ground_truth)
        else:
            losses, out = self._forward_backward(model_input, ground_truth, reduce_buckets=True)
        if self.collective:
            if self.buckets is not None and self.buckets.armed:
                # the backward that just ran had the bucket hooks (eager sync-free step): reduce the buckets nobody announced (geometry
                # latents: last), then wait for all of them — never a second, dense reduce on top (that summed three buckets twice:
                # round-3 advisor finding)
                self.buckets.finish()
            else:
                sdist.all_reduce_sum(self.flat.buffer, self.group, self.force_collectives)
        # train.py:359-363, 548-564 — clip_grad_norm_(1.0), skip the update when a gradient is not finite, Adam: one fused
        # device-side sequence (spurfies_amd/optim.py), no sync
        self.optimizer.step(max_norm=1.0 if self.grad_clip else 0.0, zero_grads=self.zero_in_adam)
        self._grads_clean = self.zero_in_adam and self.optimizer._flat is not None
        self.scheduler.step()
        self.iter_step += 1
        return losses, out

    def _forward_backward(self, model_input, ground_truth, reduce_buckets=False, collectives=True):
        """reduce_buckets: announce finished gradient buckets to the asynchronous all-reduce (only the optimisation step itself does; timing
        passes that call this directly leave the gradients local).  collectives=False: not even the 16-byte count all-reduce is issued (the
        loss is normalised by this rank's own counts): graph warm-up passes, whose results are discarded — a rank that (re)captures on its
        own must not issue collectives its peers do not."""
        with ops.scratch_owner(self):
            return self._forward_backward_impl(model_input, ground_truth, reduce_buckets, collectives)

    def _forward_backward_impl(self, model_input, ground_truth, reduce_buckets, collectives):
        prev_fork = ops.set_fork(self.fork)
        try:
            return self._forward_backward_body(model_input, ground_truth, reduce_buckets, collectives)
        finally:
            ops.set_fork(prev_fork)

    def _forward_backward_body(self, model_input, ground_truth, reduce_buckets, collectives):
        model_input = dict(model_input)
        model_input["iter_step"] = self.iter_step
        ops.drop_pending_wgrad()                 # (left behind only by a backward that was abandoned half way)
        if self.sync_free:
            self._refresh_draws(model_input["uv"].shape[1], model_input["uv"].device)
        out = self.model(model_input, fast=1)
        if self.collective:
            losses = sdist.sharded_loss(self.loss, out, ground_truth, self.group, reduce=collectives, force=self.force_collectives)
        else:
            losses = self.loss(out, ground_truth)
        if not self._grads_clean:                                               # else: cleared by the previous step's Adam sweep
            self.flat.zero_()
        self._grads_clean = False
        if self.buckets is not None:
            self.buckets.begin(armed=reduce_buckets)
            if reduce_buckets:
                ops.set_bucket_hook(self.buckets.ready)
        try:
            losses["loss"].backward(gradient=self._root_grad(losses["loss"]))   # a cached 1 (autograd would launch a fill for its own)
            ops.flush_pending_wgrad()                                           # (no-op: the colour trunk's launch took the head's GEMMs along)
            ops.join(losses["loss"].device)                                     # forked step: the backward's side branches (no-op otherwise)
        finally:
            ops.set_bucket_hook(None)
        return losses, out

    # ------------------------------------------------------------------ MFMA-shape selection of the dominant kernel
    def autotune_geo_engine(self, model_input, ground_truth, reps=10):
        """The geometry kernel exists on two MFMA shapes with the same arithmetic (ops.set_geo_mode: 'split' = 16x16x32, 'split_w' =
        32x32x16).  Which one is faster is decided by the clock the chip holds under each, and that differs from box to box by as much
        as the two differ: time the main-pass launch of both inside `reps` forward + backward passes of this batch
        (no optimiser step, the CPU generator is restored) and keep the faster.  The shape alternates EVERY pass in the order A B B A (4 x reps
        timed passes after four untimed ones), so that the slow clock drift of a chip that is still warming up — larger than the difference
        between the shapes — cancels; call it on a loaded chip (after a few steps): the cold ranking was the opposite of the steady-state one on
        two boxes of eleven.  -> {'split': ms, 'split_w': ms, 'selected': name}."""
        from . import _prof

        rng = torch.get_rng_state()
        prev = ops.geo_mode()
        R = model_input["uv"].shape[1]
        ms = {"split": [], "split_w": []}
        try:
            order = ("split", "split_w", "split_w", "split")
            for i in range(4 * (int(reps) + 1)):
                mode = order[i % 4]
                ops.set_geo_mode(mode)
                if i >= 4:
                    _prof.start(("geo",))
                self._forward_backward(model_input, ground_truth)
                if i >= 4:
                    ms[mode] += [p["ms"] for p in _prof.stop() if p["with_grad"] and p["rows"] >= 2 * R]
        finally:
            ops.set_geo_mode(prev)
            torch.set_rng_state(rng)
        res = {m: sum(v) / max(len(v), 1) for m, v in ms.items()}
        res["selected"] = min(("split", "split_w"), key=lambda m: res[m])
        ops.set_geo_mode(res["selected"])
        return res

    # ------------------------------------------------------------------ hipGraph path
    def _graphed_forward_backward(self, model_input, ground_truth):
        prev_fork = ops.set_fork(self.fork)
        try:
            return self._graphed_forward_backward_body(model_input, ground_truth)
        finally:
            ops.set_fork(prev_fork)

    def _graphed_forward_backward_body(self, model_input, ground_truth):
        from . import feat_utils

        dev = model_input["uv"].device
        keys_in = ("intrinsics", "uv", "pose")
        # the DTU recipe's feature-consistency term (local_data, local_weight 0.5) is part of the captured step: its kernels read the view's
        # feature-map addresses, cameras and sizes from a DESCRIPTOR in device memory (feat_utils.LocalDesc), and each replay is preceded by a
        # copy of the current view's descriptor into the graph's static one — one graph for all training views
        local = model_input.get("local_data")
        desc = None if local is None else feat_utils.local_desc(local, dev)
        key = (self.model.cache_key(), desc is not None)
        if self._graph is None or self._static_in["uv"].shape != model_input["uv"].shape or key != self._graph_key:
            self._graph_key = key
            self._static_in = {k: model_input[k].clone() for k in keys_in}
            self._static_desc = None if desc is None else feat_utils.LocalDesc(desc.buf.clone(), desc.n_src)
            static_local = self._static_desc
            self._static_gt = {k: ground_truth[k].to(dev).clone() for k in ("rgb", "mask")}
            # warm-up on a side stream (builds the cell table, TV graph, workspaces, allocator pools) without touching the
            # training trajectory: parameters are restored afterwards and no optimiser step is taken
            rng = torch.get_rng_state()
            side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                for _ in range(2):       # no collective in the warm-up: ranks may (re)capture independently of each other
                    self._forward_backward(dict(self._static_in, local_data=static_local), self._static_gt, collectives=False)
            torch.cuda.current_stream(dev).wait_stream(side)
            torch.set_rng_state(rng)
            self._refresh_draws(model_input["uv"].shape[1], dev)      # allocates the persistent draw buffers
            torch.set_rng_state(rng)
            self._graph = torch.cuda.CUDAGraph()
            self._graph_tail, self._counts = None, None
            if not self.collective:
                ops.drop_pending_wgrad()
                with ops.capture_guard(), torch.cuda.graph(self._graph):
                    out = self.model(dict(self._static_in, local_data=static_local, iter_step=0), fast=1)
                    losses = self.loss(out, self._static_gt)
                    if not self.zero_in_adam:      # else the previous step's Adam sweep left the gradient buffer zero: no fill node in the graph
                        self.flat.zero_()
                    losses["loss"].backward(gradient=self._root_grad(losses["loss"]))
                    ops.flush_pending_wgrad()
                    ops.join(dev)                  # the backward's forked branches end inside the capture
            else:
                # ray-sharded: the step has one exchange INSIDE forward + backward — the 16 bytes of loss normalisers between the forward and
                # the loss kernels (dist.sharded_loss).  No collective is captured (a mis-captured one hangs every rank): the step is TWO
                # graphs over one memory pool, [forward + this rank's counts] and [loss + backward], with the count all-reduce issued eagerly
                # between the replays and the gradient all-reduce after them.  The autograd graph spans both captures; its saved tensors
                # live in the shared pool.  Nothing executes during capture and NO collective is issued around it (nor in the warm-up above):
                # whether and when a rank (re)captures — first step, a new batch shape, parameters re-pointed by load_state_dict — is then
                # invisible to its peers, whose collective sequences stay aligned (a lone re-capture used to issue
                # three extra all-reduces and hang the group).
                # Captured per thread: RCCL's watchdog asks events of earlier eager collectives from its own thread whenever it likes, and a capture
                # that forbids such calls to every thread ends the process when they meet.
                pool = torch.cuda.graph_pool_handle()
                with ops.capture_guard(), torch.cuda.graph(self._graph, pool=pool, capture_error_mode="thread_local"):
                    out = self.model(dict(self._static_in, local_data=static_local, iter_step=0), fast=1)
                    self._counts = sdist.fused_counts(out)
                self._graph_tail = torch.cuda.CUDAGraph()
                with ops.capture_guard(), torch.cuda.graph(self._graph_tail, pool=pool, capture_error_mode="thread_local"):
                    losses = self.loss.fused_forward(out, self._static_gt, denom=self._counts, world=self.world)
                    if not self.zero_in_adam:
                        self.flat.zero_()
                    losses["loss"].backward(gradient=self._root_grad(losses["loss"]))
                    ops.flush_pending_wgrad()
                    ops.join(dev)
            self._static_out = (losses, out)
            self._grads_clean = False              # the warm-up passes left gradients behind (nothing ran during the capture)
        # the batch -> the graph's static input buffers: ONE multi-tensor copy launch (five D2D copies were 24 us of a 1 ms step at 128 rays)
        src = [model_input[k] for k in keys_in] + [ground_truth[k] for k in ("rgb", "mask")]
        dst = [self._static_in[k] for k in keys_in] + [self._static_gt[k] for k in ("rgb", "mask")]
        if desc is not None:
            src.append(desc.buf)
            dst.append(self._static_desc.buf)
            self._static_desc.keep = desc.keep       # the maps the replay reads
        if all(a.is_cuda and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(src, dst)):
            torch._foreach_copy_(dst, src)
        else:
            for a, b in zip(src, dst):
                b.copy_(a, non_blocking=True)
        self._refresh_draws(model_input["uv"].shape[1], dev)
        if self.zero_in_adam and not self._grads_clean:        # only behind passes that ran without an optimiser step (warm-up, timing passes)
            self.flat.zero_()
        self._grads_clean = False
        self._graph.replay()
        if self._graph_tail is not None:
            sdist.all_reduce_sum(self._counts, self.group, self.force_collectives)
            self._graph_tail.replay()
        return self._static_out

    def skipped_updates(self) -> int:
        """Updates the device-side clip + Adam sequence SKIPPED because a gradient was not finite (the reference skips them too: train.py:548-564 —
        but there a skipped step is visible in the loop; here nothing reads the device).  One 16-byte read: call it where the host waits anyway
        (checkpoints, logging).  A count that keeps growing means the run is no longer learning (round 6's soak found an overflowing row factor
        this way)."""
        f = getattr(self.optimizer, "_flat", None)
        return int(self.skipped) if f is None else int(f["state"][1].item())

    # ---- whole-step state: what a run needs to CONTINUE as if it had not stopped ---------------------------------------------------
    def state_dict(self):
        """Model, optimiser moments, learning-rate schedule, step counter and the CPU generator the reference draws its per-step random
        numbers from (ray_sampler.py:55,514,550,562).  The reference's own checkpoints (train.py:221-241: model + optimiser, written by
        VolOpt.save_checkpoints in the same layout) restart the schedule and the generator; with this blob a resumed run takes the same
        steps the uninterrupted one would have — bit for bit under ops.set_scatter_mode("fixed") (tools/soak.py, tests/test_gpu_model.py)."""
        return {"model_state_dict": self.model.state_dict(), "optimizer_state_dict": self.optimizer.state_dict(),
                "scheduler_state_dict": self.scheduler.state_dict(), "iter_step": self.iter_step, "cpu_rng_state": torch.get_rng_state(),
                "loss_iter_step": int(self.loss.iter_step), "skipped": int(self.skipped)}

    def load_state_dict(self, blob):
        self.model.load_state_dict(blob["model_state_dict"])
        self.optimizer.load_state_dict(blob["optimizer_state_dict"])
        self.scheduler.load_state_dict(blob["scheduler_state_dict"])
        self.iter_step = int(blob["iter_step"])
        self.loss.iter_step = int(blob.get("loss_iter_step", blob["iter_step"]))
        self.skipped = int(blob.get("skipped", 0))
        self._draws = None                                      # staged draws of the abandoned trajectory are not reused
        rng = blob["cpu_rng_state"].cpu()                       # torch.load(map_location=device) moves it
        if self.world > 1:
            # replicas must continue with ONE generator stream and one step count: rank 0's blob wins; a rank that loaded a different one is told
            import torch.distributed as tdist

            head = torch.tensor([self.iter_step, self.loss.iter_step], dtype=torch.int64)
            mine = torch.cat([head, rng.to(torch.int64)])
            ref = mine.clone().to(self.flat.buffer.device if tdist.get_backend(self.group) == "nccl" else "cpu")
            tdist.broadcast(ref, src=0, group=self.group)
            if not torch.equal(ref.cpu(), mine):
                import warnings

                warnings.warn(f"TrainStep.load_state_dict: rank {self.rank} loaded a different step count / generator state than rank 0 — continuing with rank 0's")
                self.iter_step, self.loss.iter_step = int(ref[0]), int(ref[1])
                rng = ref.cpu()[2:].to(torch.uint8)
        torch.set_rng_state(rng)
        self.flat.zero_()                  # re-attach the flat gradient views
        self._grads_clean = False

    def _root_grad(self, loss):
        if self._one is None or self._one.device != loss.device:
            self._one = torch.ones((), dtype=loss.dtype, device=loss.device)
        return self._one

    def _refresh_draws(self, R, dev):
        """The reference draws its random numbers from the CPU generator and moves them (ray_sampler.py:55,514,550,562); in
        sync-free mode the same calls are issued here, in the same order, into persistent device buffers the sampler reads."""
        s = self.model.ray_sampler
        n0, N, Ne, M = s.N_samples_eval, s.N_samples, s.N_samples_extra, s.N_samples + 2 + s.N_samples_extra
        if self._draws is None or self._draws["t_rand"].shape[0] != R:
            # one flat staging buffer on each side (the int32 selection rides as raw bits): one host-to-device copy per step
            a, b = R * n0, R * n0 + R * N

            def views(flat):
                return {"t_rand": flat[:a].view(R, n0), "u": flat[a:b].view(R, N), "sel": flat[b:].view(torch.int32)}

            self._draws_flat = torch.empty((b + Ne,), dtype=torch.float32, device=dev)
            self._draws = views(self._draws_flat)
            # The host runs several steps ahead of the GPU in this mode, so ONE pinned buffer would be rewritten while an earlier
            # step's copy is still queued: a ring of pinned buffers, each guarded by an event recorded behind its copy.
            self._pinned_ring = []
            for _ in range(self.N_STAGING):
                flat = torch.empty((b + Ne,), dtype=torch.float32).pin_memory()
                self._pinned_ring.append((flat, views(flat), torch.cuda.Event()))
            self._pinned_next = 0
            self._pinned_used = [False] * self.N_STAGING
        slot = self._pinned_next
        self._pinned_next = (slot + 1) % self.N_STAGING
        pinned_flat, pinned, ev = self._pinned_ring[slot]
        if self._pinned_used[slot]:
            ev.synchronize()                         # the copy that last read this buffer has completed (normally long ago)
        if self.draw_world > 1:                      # batch-wide draws, this rank's rows
            pinned["t_rand"].copy_(torch.rand((R * self.world, n0))[self.rank::self.world])
            pinned["u"].copy_(torch.rand((R * self.world, N))[self.rank::self.world])
        else:
            torch.rand((R, n0), out=pinned["t_rand"])
            torch.rand((R, N), out=pinned["u"])
        pinned["sel"].copy_(torch.randperm(n0)[:Ne])
        torch.randint(M, (R * self.draw_world,))     # the unused eikonal index (:562) — keeps the generator in step
        self._draws_flat.copy_(pinned_flat, non_blocking=True)
        ev.record(torch.cuda.current_stream(dev))
        self._pinned_used[slot] = True
        s.draws = self._draws


class MultiSceneTrainer:
    """several scenes optimised concurrently on ONE ray-sharded process group — S independent
    (model, TrainStep) pairs, stepped round-robin; no collective ever mixes scenes (each step's flat-gradient all-reduce belongs to
    its own scene).  Scenes alternate between `n_streams` HIP streams, so one scene's gradient all-reduce overlaps the next
    scene's kernels; a scene always runs on the same stream, which keeps its own steps ordered."""

    def __init__(self, steps, n_streams=2, device=None):
        self.steps = list(steps)
        self.device = device
        cuda = device is not None and torch.device(device).type == "cuda"
        self.streams = [torch.cuda.Stream(device=device) for _ in range(max(1, n_streams))] if cuda else [None]
        self.order = []                                  # (round, scene) log of the last call, for tests

    def __len__(self):
        return len(self.steps)

    def step(self, batches):
        """batches[s] = (model_input, ground_truth) of scene s for this round -> [loss dict per scene]."""
        if len(batches) != len(self.steps):
            raise ValueError(f"{len(batches)} batches for {len(self.steps)} scenes")
        out, self.order = [], []
        cur = torch.cuda.current_stream(self.device) if self.streams[0] is not None else None
        for s, (step, batch) in enumerate(zip(self.steps, batches)):
            st = self.streams[s % len(self.streams)]
            self.order.append(s)
            if st is None:
                out.append(step(*batch)[0])
                continue
            st.wait_stream(cur)                          # inputs prepared on the caller's stream
            with torch.cuda.stream(st):
                out.append(step(*batch)[0])
        if cur is not None:
            for st in self.streams:
                cur.wait_stream(st)
        return out


# ---------------------------------------------------------------------------------------------------------------
# VolOpt: the reference's trainer object (spurfies/train.py:20-564) around TrainStep — "next" row N1 of SURVEY.md §8(f)
# ---------------------------------------------------------------------------------------------------------------
import os
from datetime import datetime

from .conf import Conf, default_model_conf
from .utils import general as utils
from .utils import rend_util


def rename_prior_state_dict(prior: dict) -> dict:
    """ckpt/local_prior.pt's `model_state_dict` -> this model's frozen-prior keys, exactly as the reference renames it
    (spurfies/train.py:125-140): drop `sdf_features`; the i-th entry whose key contains `local_sdf_field` becomes
    `F_geometry.{2 * (i // 2)}.<tail after the 4th dot>` (i counts ALL remaining entries, the MLP's ten tensors come first);
    `density_branch.weight / .bias` become `T.0.weight / .bias`."""
    prior = {k: v for k, v in prior.items() if k != "sdf_features"}
    cnt = [0, 0, 2, 2, 4, 4, 6, 6, 8, 8]
    out = {}
    for i, (k, v) in enumerate(prior.items()):
        if "local_sdf_field" in k:
            if i >= len(cnt):
                raise ValueError(f"prior checkpoint: unexpected position {i} of {k!r} (the reference expects the ten MLP tensors first)")
            out[f"F_geometry.{cnt[i]}." + ".".join(k.split(".")[4:])] = v
        if "density_branch.weight" in k:
            out["T.0.weight"] = v
        if "density_branch.bias" in k:
            out["T.0.bias"] = v
    return out


class SyntheticDataset(torch.utils.data.Dataset):
    """Stand-in for spurfies/datasets/dtu.py:DTUDataset (images / cameras come from an unavailable download): same item layout
    `(idx, sample, ground_truth)`, `collate_fn`, `change_sampling_idx`, `total_pixels`, `img_res`."""

    def __init__(self, scene, img_res=(576, 768), n_views=3, seed=0, local=False):
        """local=True: every item carries a synthetic `local_data` dict (synthetic.make_local_data: feature maps + MVS camera packs of the
        shapes datasets/dtu.py:268-291 provides), so the feature-consistency loss (local_weight 0.5) takes part in the optimisation."""
        from . import synthetic as syn

        self.img_res = list(img_res)
        self.total_pixels = img_res[0] * img_res[1]
        self.scale_factor = 1.0
        self.n_images = n_views
        self.intrinsics = torch.from_numpy(scene["intrinsics"])
        self.poses = torch.from_numpy(scene["poses"][:n_views])
        g = torch.Generator().manual_seed(seed)
        ys, xs = torch.meshgrid(torch.arange(img_res[0]), torch.arange(img_res[1]), indexing="ij")
        self.uv = torch.stack([xs, ys], -1).reshape(-1, 2).float()
        base = torch.stack([xs / img_res[1], ys / img_res[0], 0.5 + 0 * xs], -1).reshape(-1, 3).float()
        self.rgb = [(base * (0.6 + 0.4 * torch.rand(3, generator=g))).clamp(0, 1) for _ in range(n_views)]
        cx, cy = syn.CX, syn.CY
        self.mask = [(((self.uv[:, 0] - cx) ** 2 + (self.uv[:, 1] - cy) ** 2) < (0.45 * img_res[0]) ** 2).float() for _ in range(n_views)]
        self.sampling_idx = None
        self.local = None
        if local:
            self.local = [{k: (torch.from_numpy(np.asarray(v)) if isinstance(v, (np.ndarray, np.floating)) else v)
                           for k, v in syn.make_local_data(scene, v_, seed=seed).items()} for v_ in range(n_views)]

    def __len__(self):
        return self.n_images

    def change_sampling_idx(self, sampling_size):
        """datasets/dtu.py:360-364."""
        self.sampling_idx = None if sampling_size == -1 else torch.randperm(self.total_pixels)[:sampling_size]

    def __getitem__(self, idx):
        sample = {"uv": self.uv, "intrinsics": self.intrinsics, "pose": self.poses[idx], "local_data": None if self.local is None else self.local[idx]}
        if self.sampling_idx is not None:            # select first, widen the mask to three channels afterwards
            sample["uv"] = self.uv[self.sampling_idx]
            gt = {"rgb": self.rgb[idx][self.sampling_idx], "mask": self.mask[idx][self.sampling_idx][:, None].repeat(1, 3)}
        else:
            gt = {"rgb": self.rgb[idx], "mask": self.mask[idx][:, None].repeat(1, 3)}
        return idx, sample, gt

    @staticmethod
    def collate_fn(batch):
        idx, samples, gts = zip(*batch)
        # datasets/dtu.py:339-356: `local_data` is passed through from the first item, everything else is stacked
        stack = lambda ds: {k: (ds[0][k] if (k == "local_data" or ds[0][k] is None) else torch.stack([d[k] for d in ds])) for k in ds[0]}
        return torch.as_tensor(idx), stack(samples), stack(gts)


class VolOpt:
    """Trainer with the reference's surface (spurfies/train.py): `VolOpt(args=..., batch_size=1, is_continue=False,
    timestamp='latest', checkpoint='latest', scan='scan24')`, `.gen_dataset(stg)`, `.stg`, `.run(opt_stepN) -> epoch`,
    `.train_step(batch)`, `.render_step(batch)`, `.save_checkpoints(epoch)`, `.load_from_dir(dir, checkpoint)`, and the same
    checkpoint files (`checkpoints/ModelParameters/{latest,<epoch>}.pth` = {epoch, model_state_dict, iter_step},
    `checkpoints/OptimizerParameters/*.pth` = {epoch, optimizer_state_dict}).  Dataset and cloud are injectable because the
    reference's data is a separate download; hydra / OmegaConf / TensorBoard are not required."""

    def __init__(self, **kwargs):
        torch.set_default_dtype(torch.float32)
        # train.py:23-24 — and not a detail here: with the intra-op pool enabled the per-step host work of the loop (randperm over the
        # image's pixels, three small gathers) costs 25 + 14 ms on the GPU box instead of 5 + 0.1 ms, ten times the GPU step
        torch.set_num_threads(kwargs.get("num_threads", 1))
        args = kwargs.get("args") or Conf()
        self.hparams = args
        self.conf = Conf(args.get("vol", {})) if isinstance(args, dict) else Conf()
        self.batch_size = kwargs.get("batch_size", 1)
        self.exps_folder_name = args.get("exps_folder", "exps_vsdf") if isinstance(args, dict) else "exps_vsdf"
        scan = kwargs.get("scan", "scan24")
        self.data_dir = self.conf.get_string("dataset.data_dir", "dtu")
        self.scan_id = int(scan[4:]) if (self.data_dir == "dtu" and str(scan).startswith("scan")) else scan
        self.expname = self.conf.get_string("train.expname", "ours") + f"_{self.scan_id}"
        root = kwargs.get("root", "./")
        self.expdir = os.path.join(root, self.exps_folder_name, self.expname)
        is_continue, timestamp = kwargs.get("is_continue", False), kwargs.get("timestamp", "latest")
        if is_continue and timestamp == "latest":
            stamps = sorted(os.listdir(self.expdir)) if os.path.exists(self.expdir) else []
            is_continue, timestamp = (True, stamps[-1]) if stamps else (False, None)
        self.timestamp = "{:%Y_%m_%d_%H_%M_%S}".format(datetime.now())
        self.plots_dir = os.path.join(self.expdir, self.timestamp, "plots")
        self.checkpoints_path = os.path.join(self.expdir, self.timestamp, "checkpoints")
        self.model_params_subdir, self.optimizer_params_subdir = "ModelParameters", "OptimizerParameters"
        for d in (self.plots_dir, os.path.join(self.checkpoints_path, self.model_params_subdir),
                  os.path.join(self.checkpoints_path, self.optimizer_params_subdir)):
            os.makedirs(d, exist_ok=True)

        device = kwargs.get("device", "cuda")
        self.scene = kwargs.get("scene")
        self.train_dataset = kwargs.get("dataset")
        model_conf = self.conf.get_config("model") or default_model_conf()
        model_cls = utils.get_class(self.conf.get_string("train.model_class", "spurfies_amd.model.pointneus_disent.PointVolSDF"))
        self.model = model_cls(conf=model_conf if isinstance(model_conf, Conf) else Conf(model_conf), scan_id=self.scan_id,
                               dataset=self.data_dir, neural_points=kwargs.get("neural_points"), device=device)
        prior = kwargs.get("prior_state_dict")            # already in F_geometry.* / T.0.* form, or:
        prior_path = kwargs.get("prior_path", "ckpt/local_prior.pt")     # the reference's file (train.py:125-140), if present
        if prior is None and prior_path and os.path.exists(prior_path):
            prior = rename_prior_state_dict(torch.load(prior_path, map_location="cpu")["model_state_dict"])
        if prior is not None:
            self.model.load_state_dict(prior, strict=False)
        init = kwargs.get("init_state_dict")               # e.g. fitted geometry latents: start values, applied BEFORE a checkpoint is restored
        if init is not None:
            self.model.load_state_dict(init, strict=False)
        self.num_pixels = self.conf.get_int("train.num_pixels", 1024)
        self.checkpoint_freq = self.conf.get_int("train.checkpoint_freq", 100)
        self.render_freq = self.conf.get_int("train.render_freq", 500)
        self.split_n_pixels = self.conf.get_int("train.split_n_pixels", 500)
        lw = self.conf.get_config("loss") or {}
        loss = VolSDFLoss(lw.get("rgb_loss", "torch.nn.L1Loss"), local_weight=lw.get("local_weight", 0.5), pseudo_weight=lw.get("pseudo_weight", 0.5),
                          eikonal_weight=lw.get("eikonal_weight", 0.001), rgb_weight=lw.get("rgb_weight", 1.0), tv_weight=lw.get("tv_weight", 0.01))
        self.lr = self.conf.get_float("train.learning_rate", 5.0e-4)
        grad_clip = args.get("grad_clip", True) if isinstance(args, dict) else True
        # default execution mode = the one bench.py times: on a GPU the sync-free step (static shapes, device-side counts, fused
        # loss kernels, gradients added straight into the flat buffer); sync_free=False keeps the reference-shaped step with its per-step outputs
        # (`grad_theta [P,3]`, one host read-back) — what a caller that inspects those outputs wants, and the only mode without a GPU
        sync_free = kwargs.get("sync_free")
        if sync_free is None:
            sync_free = torch.device(device).type == "cuda"
        self.step = TrainStep(self.model, loss=loss, lr=self.lr, grad_clip=grad_clip, sync_free=bool(sync_free), use_graph=kwargs.get("use_graph", False))
        self.loss, self.optimizer, self.scheduler = self.step.loss, self.step.optimizer, self.step.scheduler
        self.start_epoch, self.iter_step, self.total_step = 0, 0, 0
        self.stg = 2
        if is_continue:
            self.load_from_dir(dir=os.path.join(self.expdir, timestamp), checkpoint=kwargs.get("checkpoint", "latest"))
        self.model.hparams = self.hparams
        self.last_losses = None
        self.last_psnr = None
        self.psnr_every = int(kwargs.get("psnr_every", 50))
        # H2 arithmetic (the default of the large kernels) has fp16's exponent range where the reference's fp32 has 2^127: a value beyond it turns the
        # step's gradient non-finite, and the device-side guard (train.py:548-564's, on the device) skips the update — silently, unless somebody reads
        # the counter.  Every `arith_guard` steps this trainer does (one 16-byte read), and when updates were skipped since the last look it moves the
        # process to the bf16 x 3 kernels (fp32's range, same results to fp32 accuracy, ~1.3x the step time) — once, with a warning.  0 = never look.
        self.arith_guard = int(kwargs.get("arith_guard", 500))
        self._skipped_guard, self._arith_fallback = 0, False
        self._local_cache = {}

    # ---- data -----------------------------------------------------------------------------------------------
    def gen_dataset(self, stg):
        self.stg = stg
        self._local_cache = {}           # device copies of the views' feature maps belong to the dataset that is being replaced
        if self.train_dataset is None:
            if self.scene is None:
                raise RuntimeError("no dataset: pass dataset=... or scene=... (the reference's DTU / MipNeRF-360 loaders need its data download)")
            self.train_dataset = SyntheticDataset(self.scene)
        ds = self.train_dataset
        self.train_dataloader = torch.utils.data.DataLoader(ds, batch_size=self.batch_size, shuffle=True, collate_fn=ds.collate_fn)
        self.eval_dataloader = torch.utils.data.DataLoader(ds, batch_size=1, shuffle=False, collate_fn=ds.collate_fn)
        self.total_pixels, self.img_res, self.n_batches = ds.total_pixels, ds.img_res, len(self.train_dataloader)
        self.ds_len = len(ds)

    # ---- checkpoints (train.py:221-241, 293-328) -----------------------------------------------------------------
    def save_checkpoints(self, epoch, latest_only=False):
        skipped = self.step.skipped_updates()               # (the host is about to wait for the device anyway)
        if skipped > getattr(self, "_skipped_seen", 0):
            import warnings

            warnings.warn(f"{skipped - getattr(self, '_skipped_seen', 0)} optimisation steps since the last checkpoint had a non-finite gradient and were "
                          f"skipped ({skipped} of {self.iter_step} in total): ops.set_h2(color_fwd=False, color_bwd=False, wgrad=False) and "
                          "ops.set_geo_mode('split_w') select the six-product bf16 arithmetic, 'f32' the fp32-MFMA twins", RuntimeWarning)
            self._skipped_seen = skipped
        model_blob = {"epoch": epoch, "model_state_dict": self.model.state_dict(), "iter_step": self.iter_step}
        opt_blob = {"epoch": epoch, "optimizer_state_dict": self.optimizer.state_dict()}
        names = ["latest"] if latest_only else ["latest", str(epoch)]
        for n in names:
            torch.save(model_blob, os.path.join(self.checkpoints_path, self.model_params_subdir, n + ".pth"))
            torch.save(opt_blob, os.path.join(self.checkpoints_path, self.optimizer_params_subdir, n + ".pth"))

    def load_from_dir(self, dir, checkpoint="latest"):
        ck = os.path.join(dir, "checkpoints")
        saved = torch.load(os.path.join(ck, "ModelParameters", str(checkpoint) + ".pth"), map_location=self.model.neural_pts.device)
        self.model.load_state_dict(saved["model_state_dict"])
        self.start_epoch, self.iter_step = saved["epoch"], saved["iter_step"]
        self.step.iter_step = self.iter_step
        data = torch.load(os.path.join(ck, "OptimizerParameters", str(checkpoint) + ".pth"), map_location=self.model.neural_pts.device)
        self.optimizer.load_state_dict(data["optimizer_state_dict"])
        self.step.flat.zero_()     # re-attach the flat gradient views (the reference does not save the scheduler either)

    # ---- steps ---------------------------------------------------------------------------------------------------
    def train_step(self, batch, use_mvs=False, use_depth_reg=True):
        """train.py:330-397."""
        indices, model_input, ground_truth = batch
        dev = self.model.neural_pts.device
        model_input = {k: (v.to(dev, non_blocking=True) if torch.is_tensor(v) else v) for k, v in model_input.items()}
        local = model_input.get("local_data")
        if local is not None:          # train.py:339-343 moves the view's feature maps (tens of MB) every step; they never change: once per view
            model_input["local_data"] = self._local_to_device(local, indices, dev)
        ground_truth = {k: v.to(dev, non_blocking=True) for k, v in ground_truth.items()}
        self.step.iter_step = self.iter_step
        losses, out = self.step(model_input, ground_truth)
        self.last_losses = losses
        if self.iter_step % self.psnr_every == 0:      # the reference logs it every 50 steps (train.py:370-392)
            self.last_psnr = rend_util.get_psnr(out["rgb_values"].detach(), ground_truth["rgb"].reshape(-1, 3))
        self.train_dataset.change_sampling_idx(self.num_pixels)
        self.iter_step += 1
        self.total_step += 1
        if self.arith_guard > 0 and self.total_step % self.arith_guard == 0:
            self._guard_arithmetic()
        return losses

    def _guard_arithmetic(self):
        """See `arith_guard` in __init__.  -> True when this call switched the arithmetic."""
        skipped = self.step.skipped_updates()
        grew, self._skipped_guard = skipped > self._skipped_guard, skipped
        if not grew or self._arith_fallback:
            return False
        from . import ops

        if ops.geo_mode() != "h2" and not any(ops._H2.values()):
            return False                                  # already on fp32-range arithmetic: the non-finite gradients are the run's own
        import warnings

        warnings.warn(f"{skipped} optimisation steps of {self.total_step} had a non-finite gradient and were skipped; switching the geometry / colour / "
                      "weight-gradient kernels of this process from H2 (fp16 pieces: |value| < 65504) to bf16 x 3 (fp32's range) — "
                      "ops.set_geo_mode('split_w'), ops.set_h2(color_fwd=False, color_bwd=False, wgrad=False)", RuntimeWarning)
        ops.set_geo_mode("split_w")
        ops.set_h2(color_fwd=False, color_bwd=False, wgrad=False, rhead_fwd=False, rhead_bwd=False)
        self.step._graph = None                           # a captured step holds the old kernels: re-captured by the next call
        self._arith_fallback = True
        return True

    def _local_to_device(self, local, indices, dev):
        """Device copy of a view's `local_data`, cached per VIEW INDEX (the reference's DTUDataset builds a fresh dict and freshly indexed
        tensors on every __getitem__, datasets/dtu.py:268-291, so object identity is no key) in an LRU bounded by the number of views; an entry
        is reused only while the host tensors have the shapes it was made from."""
        idx = int(indices.reshape(-1)[0]) if torch.is_tensor(indices) else int(indices if not isinstance(indices, (list, tuple)) else indices[0])
        # identity of the dataset object rides in the signature: the same view index of ANOTHER dataset (new scene / stage, same
        # resolution) must not hit the old view's maps
        sig = (id(self.train_dataset),) + tuple((k, tuple(v.shape), str(v.dtype)) for k, v in sorted(local.items()) if torch.is_tensor(v))
        hit = self._local_cache.get(idx)
        if hit is not None and hit[0] == sig:
            self._local_cache[idx] = self._local_cache.pop(idx)          # most recently used last
            return hit[1]
        moved = {k: (v.to(dev) if torch.is_tensor(v) else v) for k, v in local.items()}
        self._local_cache.pop(idx, None)
        self._local_cache[idx] = (sig, moved)
        n_views = getattr(self, "ds_len", 0) or (len(self.train_dataset) if self.train_dataset is not None else 0)
        cap = max(1, int(n_views))
        while len(self._local_cache) > cap:
            self._local_cache.pop(next(iter(self._local_cache)))
        return moved

    def render_step(self, batch, epoch=0, dataset=None, fast=-1, graph=False):
        """train.py:399-472 without the image files / TensorBoard: full-image render in `split_n_pixels` chunks, streamed
        (spurfies_amd/eval_graph.py:ImageRenderer): pixel coordinates resident on the device, every chunk's outputs written straight into
        their rows of pre-allocated [H*W, ...] tensors — no per-chunk list / clone / cat (`utils.split_input` + `utils.merge_output` remain
        available under their reference names).  graph=True: one hipGraph launch per chunk."""
        from .eval_graph import ImageRenderer

        self.model.eval()
        indices, model_input, ground_truth = batch
        dev = self.model.neural_pts.device
        model_input = {k: (v.to(dev) if torch.is_tensor(v) else v) for k, v in model_input.items()}
        total = model_input["uv"].shape[1]
        use_graph = bool(graph) and torch.device(dev).type == "cuda" and fast != 1
        r = getattr(self, "_renderer", None)
        if r is None or r.n_rays != self.split_n_pixels or r.fast != fast or r.use_graph != use_graph:
            r = self._renderer = ImageRenderer(self.model, self.split_n_pixels, fast=fast, graph=use_graph)
        merged = {k: v.clone() for k, v in r(model_input, total).items()}      # once per IMAGE: the renderer's buffers are reused by the next one
        merged["psnr"] = rend_util.get_psnr(merged["rgb_values"], ground_truth["rgb"].to(dev).reshape(-1, 3))
        return merged

    def run(self, opt_stepN):
        """train.py:496-546: epochs over the image loader until `opt_stepN` steps; returns the epoch reached."""
        import gc

        epoch = self.start_epoch
        self.train_dataset.change_sampling_idx(self.num_pixels)
        # everything built so far (model, dataset, torch's module tables: ~10^6 objects) moves to the collector's permanent generation: a
        # full collection inside the loop then walks the loop's own garbage only, instead of stalling the host for ~0.1 s (measured in bench.py:
        # 78 - 142 ms, i.e. 15 - 30 steps of GPU work that the launch queue may or may not cover)
        gc.collect()
        gc.freeze()
        while self.iter_step < opt_stepN:
            if self.checkpoint_freq > 0 and epoch % self.checkpoint_freq == 0 and epoch > self.start_epoch:
                self.save_checkpoints(epoch)
            for batch in self.train_dataloader:
                if self.iter_step >= opt_stepN:
                    break
                self.train_step(batch)
            epoch += 1
        self.save_checkpoints(epoch)
        return epoch
