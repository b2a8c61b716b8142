"""The captured ray-sharded step beside RCCL's watchdog, which asks events of earlier collectives from its own thread at any time: a capture that forbids such
calls to every thread ends the process when they meet, so the step captures per thread."""
import os

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from tests.test_gpu_dist import R_TOTAL, _free_port

pytestmark = pytest.mark.gpu


def _worker(port, q):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    try:
        from spurfies_amd import synthetic as syn
        from spurfies_amd.conf import default_model_conf
        from spurfies_amd.model.pointneus_disent import PointVolSDF
        from spurfies_amd.train import TrainStep

        torch.cuda.set_device(0)
        torch.distributed.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0))
        scene = syn.make_scene(3000, seed=4, prior="fitted")
        st = scene["state"]
        g = torch.Generator().manual_seed(8)
        uv = torch.from_numpy(syn.make_pixels(R_TOTAL, g))[None].cuda()
        batch = ({"intrinsics": torch.from_numpy(scene["intrinsics"])[None].cuda(), "uv": uv, "pose": torch.from_numpy(scene["poses"][0])[None].cuda(), "local_data": None},
                 {"rgb": torch.rand((R_TOTAL, 3), generator=g)[None].cuda(), "mask": torch.ones(R_TOTAL)[None, :, None].repeat(1, 1, 3).cuda()})
        model = PointVolSDF(default_model_conf(near=0.5, grid_ranges=list(scene["ranges"])), 24, "dtu", neural_points={"pts": st["neural_pts"], "colors": scene["colors"]})
        model.load_state_dict({k: torch.as_tensor(np.asarray(v)) for k, v in st.items()}, strict=False)
        step = TrainStep(model, use_graph=True, force_collectives=True)
        modes, original = [], torch.cuda.graph

        class Spy(original):
            def __init__(self, *args, **kw):
                modes.append(kw.get("capture_error_mode", "global"))
                super().__init__(*args, **kw)

        torch.cuda.graph = Spy
        torch.manual_seed(21)
        losses = [float(step(*batch)[0]["loss"].item()) for _ in range(3)]
        torch.cuda.graph = original
        q.put(("ok", modes, losses))
        torch.distributed.destroy_process_group()
    except Exception:  # noqa: BLE001
        import traceback

        q.put(("error", traceback.format_exc()[-1500:], None))


def test_ray_sharded_captures_forbid_calls_to_their_own_thread_only():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_worker, args=(_free_port(), q))
    p.start()
    try:
        status, modes, losses = q.get(timeout=100)
    finally:
        p.join(timeout=10)
        if p.is_alive():
            p.terminate()
    assert status == "ok", modes
    assert modes == ["thread_local", "thread_local"] and all(np.isfinite(losses))
