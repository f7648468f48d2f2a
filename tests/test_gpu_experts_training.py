"""Networks with experts through the trainer on the GPU, on its default path."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_two_stages_with_experts():
    """Renderer(timenet_experts=...) through Trainer.train_dynamic with the default pipeline: the block's parameters move in
    stage s1 (autograd) and in stage s2 (direct)."""
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    from dimo_amd.trainer import TrainConfig, Trainer
    cfg = TrainConfig(num_pts=300, num_cpts=48, num_pts_per_cpt=10, num_motions=3, num_frames=4, num_views=4,
                      motions_per_step=2, views_per_step=1, frames_per_step=2, resolution=64, stage="s1", FPS_iter=10 ** 6,
                      density_end_iter=0, position_lr_max_steps=500)
    rd = Renderer(sh_degree=0, num_latent_code=cfg.num_motions, add_normal=True, device="cuda", timenet_experts=4, timenet_top_k=2)
    init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=0, num_latent=cfg.num_motions)
    g = rd.gaussians
    g._r = torch.nn.Parameter(g._scaling.detach().mean() * torch.ones(1, 1, device="cuda"))
    tr = Trainer(cfg, rd)
    assert not tr.direct
    values = lambda: {n: p.detach().clone() for n, p in g._timenet.experts.named_parameters()}
    seen = [values()]

    def note(t):
        if (t.stage, t.step) in (("s1", 3), ("s2", 2)):
            seen.append(values())
    tr.train_dynamic(3, 2, on_step=note)
    torch.cuda.synchronize()
    assert tr.stage == "s2" and tr.direct and torch.isfinite(g.flat_params).all() and len(seen) == 3
    for a, b in zip(seen, seen[1:]):
        for n in a:
            assert not torch.equal(a[n], b[n]), n


def test_renders_through_quantized_experts():
    """Render-only use: a model with experts, quantized, through Renderer.render -- the image is the one of its quantized
    network's deformation, handed to render as it is."""
    from dimo_amd.experts import QuantizedExpertMLP
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    from dimo_amd.trainer import TrainConfig, Trainer
    cfg = TrainConfig(num_pts=2000, num_cpts=64, num_motions=2, resolution=96, motions_per_step=1, views_per_step=1, frames_per_step=1)
    rd = Renderer(sh_degree=0, num_latent_code=2, add_normal=True, device="cuda", timenet_experts=4, timenet_top_k=2)
    init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=0, num_latent=2)
    g = rd.gaussians
    tr = Trainer(cfg, rd, direct=False)
    tr.find_knn(k=4)
    with torch.no_grad():
        g._timenet.experts.w2.copy_(torch.randn(g._timenet.experts.w2.shape, device="cuda",
                                                generator=torch.Generator(device="cuda").manual_seed(0)) / 16)
    cam = tr.cams.get(0.0, 40.0, cfg.radius, 96, 96)
    with torch.no_grad():
        full = rd.render(cam, time=0.5, stage="s2", latent_index=1)["image"] + 0
        g.quantize_experts()
        assert isinstance(g._timenet.experts, QuantizedExpertMLP)
        dx, dq = g._timenet(g._c_xyz, 0.5, g.latent_code(1))
        image = rd.render(cam, time=0.5, stage="s2", latent_index=1)["image"] + 0
        want = rd.render(cam, time=0.5, stage="s2", latent_index=1, deform=(dx, dq))["image"] + 0
    assert torch.isfinite(image).all() and float((image - want).abs().max()) <= 1e-5  # (as batched and immediate renders agree)
    assert float((image - full).abs().max()) > 1e-5  # (the block's products count, in the one form as in the other)
    with pytest.raises(RuntimeError, match="no_grad"):
        rd.render(cam, time=0.5, stage="s2", latent_index=1)


def test_direct_pipeline_equals_autograd_pipeline_with_experts():
    """Stage s2: the direct pipeline around the module's autograd gives the loss and the gradients -- the block's and the
    router's among them -- of the reference-shaped autograd path."""
    from dimo_amd.rasterizer import CapacityPolicy
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    from dimo_amd.trainer import TrainConfig, Trainer
    cfg = TrainConfig(num_pts=3000, num_cpts=48, num_motions=3, num_frames=5, num_views=4, motions_per_step=2, views_per_step=2,
                      frames_per_step=2, resolution=128)
    res = []
    for direct in (False, True):
        rd = Renderer(sh_degree=0, num_latent_code=cfg.num_motions, add_normal=True, device="cuda",
                      capacity=CapacityPolicy(initial=1 << 19) if direct else None, timenet_experts=4, timenet_top_k=2)
        init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=0, num_latent=cfg.num_motions)
        g = rd.gaussians
        with torch.no_grad():
            g._timenet.experts.w2.copy_(torch.randn(g._timenet.experts.w2.shape, device="cuda",
                                                    generator=torch.Generator(device="cuda").manual_seed(0)) / 16)
        tr = Trainer(cfg, rd, direct=direct)
        assert tr.direct == direct
        tr.optimizer.step = lambda *a, **k: None
        g.zero_grad = lambda: None
        tr.step = 298
        tr.train_step(tr.sample())
        torch.cuda.synchronize()
        res.append((tr.last_loss.item(), g.flat_grads.clone(), {n: p.grad.clone() for n, p in g._timenet.experts.named_parameters()}))
    (la, ga, ba), (lb, gb, bb) = res
    assert abs(la - lb) <= 1e-5 * abs(la), (la, lb)
    assert (ga - gb).abs().sum() / ga.abs().sum() < 1e-4
    for n in ba:
        assert float(ba[n].abs().sum()) > 0 and (ba[n] - bb[n]).abs().sum() / ba[n].abs().sum() < 1e-3, n
