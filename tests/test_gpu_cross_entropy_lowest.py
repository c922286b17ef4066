"""The cross entropy with biases of the type's lowest finite value."""
import math

import pytest
import torch

from test_gpu_ops import bound_of, entropy_case, plain_cross_entropy, rel

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('everywhere', [True, False])
def test_cross_entropy_of_the_lowest_bias(dt, everywhere):
    """Everywhere: f32 and bf16 (3.4e38) absorb the products, in 32 bits as in 64, and the softmax is uniform.  f16 (65504): a logit in 32 bits is
    off by half a step there, 2^-9; a loss is the difference of two such numbers, 2^-8, and probabilities are off by e^(2^-8) - 1
    relative, which goes into the gradients' bound.  On all but a few entries: those cannot be chosen."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, 70, 300, 64, seed=9, ignored=0.1)
    with torch.no_grad():
        if everywhere:
            b.fill_(torch.finfo(dt).min)
        else:
            b[5:290] = torch.finfo(dt).min
            target = torch.where(target == -100, target, target % 5)
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    up = torch.rand(70, generator=torch.Generator().manual_seed(1)) + 0.5
    got = torch.autograd.grad(rows, [h, w, b], up.to(DEV))
    want, *grads = plain_cross_entropy(h, w, b, target, -100, up)
    off = 2.0 ** -8 if dt == torch.float16 and everywhere else 0.0
    assert float((rows.detach().cpu().double() - want).abs().max()) <= off + 1e-5 * float(want.abs().max())
    for a, e in zip(got, grads):
        assert rel(a, e) < bound_of(dt, e) + math.expm1(off)
    if everywhere and dt != torch.float16:
        used = target != -100
        assert float((rows.detach()[used] - math.log(300)).abs().max()) <= 1e-5
    if not everywhere:
        assert float(got[1][5:290].abs().sum()) == 0.0 and float(got[2][5:290].abs().sum()) == 0.0
