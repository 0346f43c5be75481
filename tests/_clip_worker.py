"""Worker of the clipped view steps in tests/test_multirank_gpu.py: one rank of a job whose ranks
share one GPU and exchange over gloo."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main():
    out_path = sys.argv[1]
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo")
    from vings_mono_amd import _lib, harness, parallel, synth
    dev = torch.device("cuda:0")
    W, H, n, steps = 160, 96, 5000, 2
    raw = synth.make_splats(n, W, H, n_views=world * steps, seed=33)
    intr = synth.intrinsic_for(W, H)
    c2w = synth.window_poses(world * steps)
    gtp = {k: v.to(dev) for k, v in synth.perturb_splats(raw).items()}
    reducer = lambda: parallel.GradReducer(n, dev, world, compact=False)

    def view(s):
        k = s * world + rank
        w2c = torch.linalg.inv(c2w[k]).to(dev)
        with torch.no_grad():
            pr = harness.render(gtp, w2c, intr)
        gt = {"rgb": pr["rgb"].clone(), "depth": pr["depth"].clone(), "depth_cov": torch.ones_like(pr["depth"])}
        return k, w2c, gt

    def fused(m, red, s):
        k, w2c, gt = view(s)
        m.fused_view(harness.view_settings(w2c, intr), intr, gt, w2c[:3, :3].cpu(), k, red)

    def autograd(m, red, s):
        k, w2c, gt = view(s)
        m.finish_view(*m.backward_view(w2c, intr, gt), k, red)

    def state(m):
        st = m.optimizer.state
        return {"norm": m.last_grad_norm.cpu().clone(),
                "params": {k: m.params[k].detach().cpu().clone() for k in m.NAMES},
                "m": {k: st[m.params[k]]["exp_avg"].cpu().clone() for k in m.NAMES},
                "v": {k: st[m.params[k]]["exp_avg_sq"].cpu().clone() for k in m.NAMES}}

    loose = harness.SurfelMapper(raw, dev, max_grad_norm=1e9)
    fused(loose, reducer(), 0)
    full = float(loose.last_grad_norm)
    result = {"full": full, "loose": state(loose)}
    for name, step in (("fused", fused), ("autograd", autograd)):
        m, red = harness.SurfelMapper(raw, dev, max_grad_norm=full / 8), reducer()
        for s in range(steps):
            step(m, red, s)
            result[f"{name}{s}"] = state(m)
    try:
        fused(harness.SurfelMapper(raw, dev, max_grad_norm=1.0), parallel.GradReducer(n, dev, world), 0)
        result["refused"] = False
    except _lib.VingsError:
        result["refused"] = True
    torch.cuda.synchronize()
    torch.save(result, out_path + f".rank{rank}.pt")
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
