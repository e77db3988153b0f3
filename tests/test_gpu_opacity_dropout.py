"""The training step's opacity dropout, against the autograd front end with
dropout.dropout between the activation and the renderer."""

import numpy as np
import pytest
import torch

import draws
from dp_helpers import RATES, initial_values

pytestmark = pytest.mark.gpu


def _scene(n, cuda):
    values = initial_values(n, seed=5)
    values["xyz"] = values["xyz"] * 0.6
    values["scaling"] = torch.rand(n, 3, generator=torch.Generator().manual_seed(6)) * 2 - 5
    return {k: v.to(cuda) for k, v in values.items()}


@pytest.mark.parametrize("sh_exchange", ["grads", "seeds"])
def test_step_draws_and_differentiates(cuda, sh_exchange):
    import dropout
    import rasterizer
    from data_parallel import DataParallelTrainer, orbit_camera

    n, W, H, p, seed = 3001, 96, 64, 0.4, 77
    cam = orbit_camera(1, 8, width=W, height=H, device=cuda)
    target = torch.rand(3, H, W, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    trainer = DataParallelTrainer(_scene(n, cuda), RATES, device=cuda, sh_exchange=sh_exchange,
                                  opacity_dropout=p, dropout_seed=seed)
    a = trainer.adam
    settings = rasterizer.GaussianRasterizationSettings(
        image_height=H, image_width=W, tanfovx=cam.tan_x, tanfovy=cam.tan_y,
        bg=torch.zeros(3, device=cuda), scale_modifier=1.0, viewmatrix=cam.view,
        projmatrix=cam.proj, sh_degree=3, campos=cam.campos, prefiltered=False, debug=False)
    seen = []
    for step in range(2):
        trainer.backward(cam, target)
        # The same activations through the front end: the images agree bit for bit.
        opacity = a.saved["opacity"][:n].clone().requires_grad_(True)
        xyz = a.params["xyz"][:n].clone()
        image, _, _ = rasterizer.GaussianRasterizer(settings)(
            means3D=xyz, means2D=torch.zeros_like(xyz),
            opacities=dropout.dropout(opacity, p, seed, step),
            shs=a.params["sh"][:n].clone().view(n, 16, 3), scales=a.saved["scaling"][:n].clone(),
            rotations=a.saved["rotation"][:n].clone())
        assert torch.equal(image.detach(), trainer.image)
        (want,) = torch.autograd.grad((image - target).abs().mean(), opacity)
        got = a.grads["opacity"][:n]
        kept = torch.from_numpy(draws.keep(np.arange(n), p, seed, step)).to(cuda).view(n, 1)
        assert not got[~kept].any() and (got[kept] != 0).sum() > 300
        # Float atomics add a Gaussian's pixels in any order.
        assert ((got - want).abs() <= 1e-4 * want.abs() + 1e-5 * want.abs().max()).all()
        seen.append(kept)
        before = a.params["opacity"][:n].clone()
        trainer.step(cam, target) if sh_exchange == "grads" else a.step()
        assert (a.params["opacity"][:n] != before).any()
    assert not torch.equal(*seen)
    trainer.close()


def test_without_dropout_nothing_changes(cuda):
    from data_parallel import DataParallelTrainer, orbit_camera

    cam = orbit_camera(1, 8, width=96, height=64, device=cuda)
    target = torch.rand(3, 64, 96, device=cuda)
    images = []
    for more in ({}, dict(opacity_dropout=0.0, dropout_seed=5)):
        trainer = DataParallelTrainer(_scene(500, cuda), RATES, device=cuda, **more)
        assert trainer._dropped is None
        trainer.step(cam, target)
        images.append(trainer.image.clone())
        trainer.close()
    assert torch.equal(*images)


@pytest.mark.parametrize("more", [dict(opacity_dropout=1.0), dict(opacity_dropout=-0.1),
                                  dict(opacity_dropout=float("nan")), dict(dropout_seed=-1),
                                  dict(dropout_seed=0.5), dict(dropout_seed=2 ** 64)])
def test_refusals(cuda, more):
    from data_parallel import DataParallelTrainer

    with pytest.raises(ValueError):
        DataParallelTrainer(_scene(10, cuda), RATES, device=cuda, **more)


def _image(trainer, opacity, cam, W, H, xyz=None):
    """The front end's image of a trainer's Gaussians under another opacity."""
    import rasterizer

    a, n = trainer.adam, opacity.shape[0]
    settings = rasterizer.GaussianRasterizationSettings(
        image_height=H, image_width=W, tanfovx=cam.tan_x, tanfovy=cam.tan_y,
        bg=torch.zeros(3, device=opacity.device), scale_modifier=1.0, viewmatrix=cam.view,
        projmatrix=cam.proj, sh_degree=3, campos=cam.campos, prefiltered=False, debug=False)
    xyz = a.params["xyz"][:n].clone()
    return rasterizer.GaussianRasterizer(settings)(
        means3D=xyz, means2D=torch.zeros_like(xyz), opacities=opacity,
        shs=a.params["sh"][:n].clone().view(n, 16, 3), scales=a.saved["scaling"][:n].clone(),
        rotations=a.saved["rotation"][:n].clone())[0]


@pytest.mark.parametrize("sh_exchange", ["grads", "seeds"])
def test_no_dropout_renders_the_undropped_opacity(cuda, sh_exchange):
    from data_parallel import DataParallelTrainer, orbit_camera

    n, W, H = 2001, 96, 64
    cam = orbit_camera(1, 8, width=W, height=H, device=cuda)
    target = torch.rand(3, H, W, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    trainer = DataParallelTrainer(_scene(n, cuda), RATES, device=cuda, sh_exchange=sh_exchange)
    trainer.backward(cam, target)
    opacity = trainer.adam.saved["opacity"][:n].clone().requires_grad_(True)
    image = _image(trainer, opacity, cam, W, H)
    assert torch.equal(image.detach(), trainer.image)
    (want,) = torch.autograd.grad((image - target).abs().mean(), opacity)
    got = trainer.adam.grads["opacity"][:n]
    assert ((got - want).abs() <= 1e-4 * want.abs() + 1e-5 * want.abs().max()).all()
    trainer.close()


def test_colour_form_draws_and_differentiates(cuda):
    """The colour form under the dropout: the same draws as the front end's, and
    the SH gradients of dropped Gaussians are nothing (their coefficients' first
    moments stay zero)."""
    import dropout
    from data_parallel import DataParallelTrainer, orbit_camera

    n, W, H, p, seed = 3001, 96, 64, 0.4, 77
    cams = [orbit_camera(k, 8, width=W, height=H, device=cuda) for k in (1, 2, 3)]
    target = torch.rand(3, H, W, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    trainer = DataParallelTrainer(_scene(n, cuda), RATES, device=cuda, sh_exchange="colours",
                                  opacity_dropout=p, dropout_seed=seed)
    a = trainer.adam
    for step in range(2):
        kept = torch.from_numpy(draws.keep(np.arange(n), p, seed, step)).to(cuda).view(n, 1)
        image = {}
        made = a.activate
        def activate():
            act = made()
            opacity = a.saved["opacity"][:n].clone().requires_grad_(True)
            image["opacity"] = opacity
            image["out"] = _image(trainer, dropout.dropout(opacity, p, seed, step), cams[step], W, H)
            return act
        a.activate = activate
        trainer.step(cams[step], target, cams[step + 1])
        a.activate = made
        assert torch.equal(image["out"].detach(), trainer.image)
        (want,) = torch.autograd.grad((image["out"] - target).abs().mean(), image["opacity"])
        got = a.grads["opacity"][:n]
        assert not got[~kept].any() and (got[kept] != 0).sum() > 300
        # Float atomics add a Gaussian's pixels in any order.
        assert ((got - want).abs() <= 1e-4 * want.abs() + 1e-5 * want.abs().max()).all()
        if step == 0:
            moved = a.first["sh"][:n].ne(0).any(1, keepdim=True)
            assert not moved[~kept].any() and moved[kept].sum() > 300
    trainer.close()
