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


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 40, 90])
def test_positions_behind_the_table(kind, new):
    """more positions than the table has pages for: such tokens are not written and see what is cached; the others
    keep their places"""
    from aps_amd import nn_ops
    hq, hkv, d, page, width = 4, 2, 64, 8, 9
    most = page * width
    kv_lens = [most + 3, most + new, most + 2000, most - 1, (1 << 31) - 1]
    n = len(kv_lens)
    cache = [randn(n * width + 1, page, hkv, d, dtype=TYPES[kind], seed=i) for i in (1, 2)]
    table = (torch.randperm(n * width, generator=torch.Generator().manual_seed(3)).view(n, width) + 1).int()
    q, k, v = (randn(n * new, h, d, dtype=TYPES[kind], seed=i) for i, h in ((4, hq), (5, hkv), (6, hkv)))
    want = [c.clone() for c in cache]
    for i, kv in enumerate(kv_lens):
        for j in range(new):
            p = kv - new + j
            if 0 <= p < most:
                want[0][table[i, p // page], p % page] = k[i * new + j]
                want[1][table[i, p // page], p % page] = v[i * new + j]
    args = (*cache, table.to(DEV), cu_of([new] * n), torch.tensor(kv_lens, device=DEV))
    nn_ops.paged_append(k, v, *args)
    assert torch.equal(cache[0], want[0]) and torch.equal(cache[1], want[1])
    out = nn_ops.attention_paged(q, *args)
    for i, kv in enumerate(kv_lens):
        ks, vs = (c[table[i].long()].reshape(most, hkv, d).double().cpu() for c in cache)
        for h in range(hq):
            rows = q[i * new:(i + 1) * new, h].double().cpu()
            off = min(kv - new, most)  # (a position behind the table sees all of it)
            val, bound = ref.attend(rows, ks[:, h // 2], vs[:, h // 2], off, True, d**-0.5, TYPES[kind])
            ref.check(out[i * new:(i + 1) * new, h], val, bound, f"sequence {i} head {h}")


@gpu
def test_tables_of_one_row_or_one_column():
    """a table whose only row or column has the stride of what it was cut from"""
    from aps_amd import nn_ops
    hkv, d, page = 2, 64, 16
    pages = torch.tensor([5, 0, 3, 2], dtype=torch.int32, device=DEV)
    for table, kv in ((pages.view(4, 1).t(), [60]),               # 1 x 4, strides (1, 1)
                      (pages.view(1, 4)[:, :3], [40]),
                      (pages.view(1, 4).t(), [16, 3, 9, 1]),      # 4 x 1, strides (1, 4)
                      (pages.repeat(3, 1).t()[:, 1:2], [4, 16, 2, 7]),
                      (pages[:1].expand(1, 1), [12]),
                      (torch.stack([pages, pages.flip(0)]).t()[::2].t(), [30, 2])):
        n = len(kv)
        plain = table.contiguous().clone()
        q, k, v = (randn(n, h, d, seed=i) for i, h in enumerate((4, hkv, hkv)))
        got = []
        for t in (plain, table if table.stride(1) == 1 or table.shape[1] == 1 else plain):
            cache = [randn(6, page, hkv, d, seed=i) for i in (7, 8)]
            args = (*cache, t, cu_of([1] * n), torch.tensor(kv, device=DEV))
            nn_ops.paged_append(k, v, *args)
            got.append([nn_ops.attention_paged(q, *args), *cache])
        assert all(torch.equal(a, b) for a, b in zip(*got))


@gpu
def test_reordered_states_that_are_lazy_views():
    """conjugated complex states and the imaginary part of one: their values, not their memory"""
    from aps_amd import nn_ops
    z = torch.randn(6, 5, dtype=torch.complex64, generator=torch.Generator().manual_seed(1)).to(DEV)
    parent = torch.tensor([[2, 0, 0], [1, 1, 2]], device=DEV)
    rows = (parent + 3 * torch.arange(2, device=DEV)[:, None]).reshape(-1)
    states = [z, z.conj(), z.conj().imag, z.conj().t()]
    out = nn_ops.beam_reorder(states, parent, dims=[0, 0, 0, 1])
    for x, s, d in zip(out, states, (0, 0, 0, 1)):
        assert torch.equal(x, s.index_select(d, rows)), s
