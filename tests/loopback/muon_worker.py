"""One rank of a several-ranks-on-one-GPU run with the optimizer of configs/nerf/muon.json (tests/test_muon_ranks_gpu.py starts `world` of these; the collectives are those of
librccl_loopback.so, as in dp_worker.py).  Writes the first steps' weights and gradients to <out>/rank<r>.npz, and a snapshot.

usage: muon_worker.py <rank> <world> <key> <out_dir>
"""
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
sys.path[:0] = [ROOT, os.path.join(ROOT, "blender-ngp_amd"), os.path.join(ROOT, "tests")]


def main():
    rank, world, key, out_dir = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3], sys.argv[4]
    import torch
    import scene
    ds = scene.make_dataset(n_train=8, n_test=1, res=64, device=torch.device("cuda:0"))
    tb = scene.build_testbed(ds, os.path.join(ROOT, "blender-ngp_amd", "configs", "nerf", "muon.json"))
    tb.network_pass = "fused"
    tb.training_batch_size = 256 * world * ((1 << 18) // (256 * world))   # split evenly
    tb.init_data_parallel(rank, world, key, True)
    assert tb.dp_comm_size == world and tb.dp_sharded_optimizer      # the default: Muon steps are replicated whatever it says
    res = {"params_0": tb.debug_params("training")}
    n = tb.n_params()

    class Gradients:
        __cuda_array_interface__ = {"shape": (n,), "typestr": "<f2", "data": (tb.gradients_ptr(), False), "version": 3}

    for step in (1, 2, 3):
        scene.train(tb, step)
        tb.sync()
        res["params_%d" % step] = tb.debug_params("training")
        res["gradients_%d" % step] = torch.as_tensor(Gradients(), device="cuda").cpu().numpy()
    scene.train(tb, 12)
    res["params"], res["inference"], res["loss"] = tb.debug_params("training"), tb.debug_params("inference"), np.float64(tb.loss)   # inference: whole on every rank, so not refused
    res["stale"] = np.array([tb.dp_state_stale, tb.dp_inference_stale])
    tb.dp_gather_optimizer_state()                            # a collective where state is sharded: nothing to do here
    tb.save_snapshot(os.path.join(out_dir, "rank%d.msgpack" % rank), True)
    tb.shutdown_data_parallel()
    tb.set_distributed(0, 1)
    scene.train(tb, 14)
    res["loss_after"] = np.float64(tb.loss)
    np.savez(os.path.join(out_dir, "rank%d.npz" % rank), **res)
    print("rank %d of %d done" % (rank, world), flush=True)


if __name__ == "__main__":
    main()
