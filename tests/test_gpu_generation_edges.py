"""
Calls at the edges of what nn_ops' packed and paged attention, its beam step and the searches built on them document.
"""
import pytest
import torch

from tests import attention_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"


def cu_of(lens, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=dtype, device=DEV)


def randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


@gpu
@pytest.mark.parametrize("group", [3, 5])
def test_gradients_of_rows_far_apart(group):
    """rows almost 8 MB apart, 600 of them, in groups that leave rows of a tile empty; what lies between is NaN"""
    n, d, pitch = 600, 32, (1 << 22) - 8 * 1021  # elements of 2 bytes
    wide = torch.full((n, pitch), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, :group * d] = randn(n, group * d, dtype=torch.bfloat16, seed=1)
    leaf = wide[:, :group * d].view(n, group, d).detach().requires_grad_()
    assert leaf.stride(0) == pitch
    k, v = (randn(n, 1, d, dtype=torch.bfloat16, seed=i).requires_grad_() for i in (2, 3))
    g = randn(n, group, d, dtype=torch.bfloat16, seed=4)
    from aps_amd import nn_ops
    for causal in (True, False):
        out = nn_ops.attention_packed(leaf, k, v, cu_of([n]), causal=causal)
        grads = torch.autograd.grad(out, (leaf, k, v), g)
        vals, bounds = ref.packed(leaf, k, v, [n], causal, g=g)
        for name, got, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
            ref.check(got, want, bound, f"{name} causal={causal}")
