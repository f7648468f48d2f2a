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


def test_the_ranks_gradients_sum_to_the_single_ones(monkeypatch):
    """Data parallelism with experts: the block's gradients are in the bucket that is summed over the ranks."""
    from tests.cpu_backend import OracleRasterizer, dist2_cpu, fps_cpu, knn_cpu, ssim_ref
    from tests.test_train_step_cpu import small_cfg
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    expert_emulation.use(monkeypatch, ex)
    cfg = small_cfg(motions_per_step=2, views_per_step=1, frames_per_step=2, resolution=32, num_pts=80, num_cpts=12)

    def grads(rank, world, triples=None):
        rd = Renderer(sh_degree=cfg.sh_degree, num_latent_code=cfg.num_motions, latent_code_dim=cfg.latent_code_dim,
                      add_normal=cfg.add_normal, device="cpu", rasterizer_factory=OracleRasterizer, dist2_fn=dist2_cpu,
                      timenet_experts=3, timenet_top_k=2)
        init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=cfg.seed, regime="trained", num_latent=cfg.num_motions)
        g = rd.gaussians
        with torch.no_grad():
            g._timenet.experts.w2.copy_(torch.randn(g._timenet.experts.w2.shape, generator=torch.Generator().manual_seed(0)) / 16)
        tr = Trainer(cfg, rd, rank=rank, world_size=world, ssim_fn=ssim_ref, knn_fn=knn_cpu, fps_fn=fps_cpu)
        tr.all_reduce_grads = tr.optimizer.step = g.zero_grad = lambda *a, **k: None
        tr.step = 300
        triples = tr.sample() if triples is None else triples
        tr.train_step(triples)
        return triples, g.flat_grads.clone(), [p.grad.clone() for p in g._timenet.experts.parameters()]
    triples, whole, block = grads(0, 1)
    parts = [grads(r, 2, triples) for r in range(2)]
    assert all(float(b.abs().sum()) > 0 for b in block)
    total = sum(p[1] for p in parts)
    assert (total - whole).abs().sum() / whole.abs().sum() < 1e-5
    for i, b in enumerate(block):
        assert (sum(p[2][i] for p in parts) - b).abs().sum() / b.abs().sum() < 1e-4
