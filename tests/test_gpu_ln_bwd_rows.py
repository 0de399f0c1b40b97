"""LayerNorm backward at the width of the base models (its own kernel, two rows a wave): every row of dz, and of the branch's gradient, against the formula."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [16, 2048, 16384])
@pytest.mark.parametrize("rep", range(3))
def test_every_row_of_the_wide_kernel(dev, M, rep):
    """dz = rstd (dy gamma - mean(dy gamma) - xhat mean(dy gamma xhat)): fp32 sums of 768 terms rounded once to bf16: half a step, 2^-8 of the value, and the sums'
    own error, 768 * 2^-24 of the terms' size (|dz| of some units here), 1e-3"""
    from spokennlp_amd import ops
    g = torch.Generator(device=dev).manual_seed(M + rep)
    H = 768
    y, r, dy = (torch.randn(M, H, generator=g, device=dev).bfloat16() for _ in range(3))
    ga, be = torch.randn(H, generator=g, device=dev), torch.randn(H, generator=g, device=dev)
    z = y.clone()
    _, mean, rstd = ops.add_ln_fwd(z, r, ga, be, 1e-12)
    grads = [torch.zeros(H, device=dev) for _ in range(3)]
    dz = ops.ln_bwd(dy, z, mean, rstd, ga, dgamma=grads[0], dbeta=grads[1], dbias=grads[2])[0].double()
    x = (z.double() - z.double().mean(1, keepdim=True)) * rstd.double()[:, None]
    gg = dy.double() * ga.double()
    want = rstd.double()[:, None] * (gg - gg.mean(1, keepdim=True) - x * (gg * x).mean(1, keepdim=True))
    bad = (dz - want).abs() > 2.0 ** -8 * want.abs() + 1e-3
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
