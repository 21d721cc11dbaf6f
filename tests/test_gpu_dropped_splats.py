"""Dropped splats in the training-step companions: the densification statistics and the whole step with its optimizer."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from conftest import scene_tensors  # noqa: E402
from ds_splat_b200 import scenes  # noqa: E402
from ds_splat_b200.dp import (CameraTensors, DensifyStats, GradientBuffer, ParameterBuffer, ShardedAdam, SplatDropout,  # noqa: E402
                              ViewRenderer, training_step)


def setup(n=8_000):
    sc = scenes.headline(n=n, seed=31, W=256, H=160, focal=180.0, views=3, ring=True)
    return sc, scene_tensors(sc), [CameraTensors.from_view(v, "cuda") for v in sc.views], \
        [torch.from_numpy(sc.image_grad(i)).cuda() for i in range(3)]


def test_statistics_count_a_dropped_splat_with_a_gradient_of_zero():
    sc, t, cams, vimgs = setup()
    renderer = ViewRenderer(t["means"], t["shs"], t["opacities"], t["scales"], t["rotations"])
    plain, none, some = (DensifyStats(sc.n, "cuda") for _ in range(3))
    renderer.render_views(cams, vimgs, GradientBuffer(sc.n, "cuda"), stats=plain)
    renderer.render_views(cams, vimgs, GradientBuffer(sc.n, "cuda"), stats=none, dropout=SplatDropout(1.0, 5))
    renderer.render_views(cams, vimgs, GradientBuffer(sc.n, "cuda"), stats=some, dropout=SplatDropout(0.4, 5))
    for stats in (none, some):
        assert torch.equal(stats.visible_count, plain.visible_count) and torch.equal(stats.max_radius, plain.max_radius)
    assert not none.grad_norm_sum.any()
    seen = plain.visible_count > 0
    # a splat whose choice was to go has no gradient; 0.4 of 8000 is 3200 +- 5 standard deviations of 44
    still = (some.grad_norm_sum[seen] == 0).float().mean() - (plain.grad_norm_sum[seen] == 0).float().mean()
    assert 0.2 < float(still) < 0.5


def test_the_whole_step_with_dropped_splats():
    """training_step hands the argument on: without a splat nothing moves, and each step drops splats of its own."""
    sc, t, cams, vimgs = setup()
    lrs = dict(means3d=1e-4, shs=1e-3, opacities=1e-2, scales=1e-4, rotations=1e-4)
    names = dict(means3d=t["means"], shs=t["shs"], opacities=t["opacities"], scales=t["scales"], rotations=t["rotations"])
    params = ParameterBuffer.from_tensors(names)
    renderer = ViewRenderer(*(params.views[k] for k in ("means3d", "shs", "opacities", "scales", "rotations")))
    grads, optimizer, stats = GradientBuffer(sc.n, "cuda"), ShardedAdam(params, lrs), DensifyStats(sc.n, "cuda")
    before = params.views["opacities"].clone()
    training_step(renderer, cams, vimgs, grads, optimizer, stats=stats, dropout=SplatDropout(1.0, 3, 0))
    # every splat dropped: no gradient anywhere, so Adam moves nothing
    assert torch.equal(params.views["opacities"], before) and not grads.flat.any() and bool(stats.visible_count.any())
    training_step(renderer, cams, vimgs, grads, optimizer, dropout=SplatDropout(0.3, 3, 1))
    moved = (params.views["opacities"] != before).view(-1)
    share = grads.views["opacities"].view(-1) != 0
    assert bool(moved.any()) and bool((moved <= share).all())      # nothing moves without a gradient
    gone = ~share
    training_step(renderer, cams, vimgs, grads, optimizer, dropout=SplatDropout(0.3, 3, 2))
    assert bool((grads.views["opacities"].view(-1)[gone] != 0).any())    # another step drops others
