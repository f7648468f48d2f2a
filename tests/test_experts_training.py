"""Networks with experts through the trainer, on the CPU: which pipeline a stage takes, and the two-stage schedule with the
expert kernels on the SIMT emulation."""
import types

import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd.deform import TimeNet
from dimo_amd.trainer import TrainConfig, Trainer
from tests import expert_emulation


def _decided(stage, experts):
    """What Trainer._decide_direct chooses on a GPU (no kernel runs: the model is a stand-in of the shapes it looks at)."""
    g = types.SimpleNamespace(_r=torch.zeros(1, 1) if stage == "s1" else torch.empty(0), _c_xyz=torch.zeros(64, 3),
                              _timenet=TimeNet(D=2, W=8, skips=(), experts=experts, top_k=1))
    tr = Trainer.__new__(Trainer)
    tr.cfg, tr.stage, tr.device, tr._direct_wanted = TrainConfig(), stage, torch.device("cuda"), None
    tr.renderer = types.SimpleNamespace(gaussians=g, _rasterizer_factory=None, capacity=object())
    tr._decide_direct()
    return tr.direct


def test_pipeline_of_networks_with_experts():
    """Stage s1's direct pipeline needs the fused TimeNet; a network with experts takes the autograd one there."""
    assert _decided("s1", 0) and _decided("s2", 0)
    assert not _decided("s1", 2)
    assert _decided("s2", 2)


def test_two_stages_with_experts(monkeypatch):
    """Stage s1, the hand-over and stage s2: the block's parameters move in both."""
    from tests.cpu_backend import OracleRasterizer, dist2_cpu, fps_cpu, knn_cpu, ssim_ref
    from tests.test_train_step_cpu import small_cfg
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    expert_emulation.use(monkeypatch, ex)
    cfg = small_cfg(stage="s1", num_pts=40, num_cpts=16, num_pts_per_cpt=3, motions_per_step=1, views_per_step=1,
                    frames_per_step=1, resolution=32, FPS_iter=10, density_end_iter=0)
    rd = Renderer(sh_degree=cfg.sh_degree, num_latent_code=cfg.num_motions, latent_code_dim=cfg.latent_code_dim,
                  add_normal=cfg.add_normal, device="cpu", rasterizer_factory=OracleRasterizer, dist2_fn=dist2_cpu,
                  timenet_experts=3, timenet_top_k=2)
    init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=cfg.seed, regime="trained", num_latent=cfg.num_motions)
    g = rd.gaussians
    g._r = torch.nn.Parameter(g._scaling.detach().mean() * torch.ones(1, 1))
    tr = Trainer(cfg, rd, ssim_fn=ssim_ref, knn_fn=knn_cpu, fps_fn=fps_cpu)
    seen = [{n: p.detach().clone() for n, p in g._timenet.experts.named_parameters()}]

    def note(t):
        if (t.stage, t.step) in (("s1", 3), ("s2", 2)):
            seen.append({n: p.detach().clone() for n, p in t.renderer.gaussians._timenet.experts.named_parameters()})
    tr.train_dynamic(3, 2, on_step=note)
    assert tr.stage == "s2" and torch.isfinite(tr.last_loss) and len(seen) == 3
    for a, b in zip(seen, seen[1:]):
        for n in a:
            assert not torch.equal(a[n], b[n]), n
