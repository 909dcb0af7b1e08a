"""
f16 gradients of nn_ops.attention_packed over upstream gradients from 1e-4 to 1e4, as loss scaling makes them: what is
rounded to f16 between the products keeps its 11 bits, whatever the size.

Elementwise bounds, as in attention_reference.py (u = 2^-24, t = 2^-11 half a step of f16) but without its allowance of an
unscaled f16 number per visible pair.  In its place:
  * P of dv is rounded after a factor 2^14: off by t of itself or, below f16's normal numbers, by 2^-25 2^-14 = 2^-39.
  * dS is rounded after a factor of at least 2^13 / x, x >= |do_r| |v_j| for every row (dq) or for the rows that see
    the key (dk; from the first row of a block of up to 64 tokens and 32 rows that begins at or before the key): off by
    t of itself or by 2^-25 x 2^-13 = 2^-38 x.
  * the forward weights, taken against a reference no larger than the row's maximum: 2^-25 over the sum of exp(s - max).
The result itself is rounded to f16: t of itself or z = 2^-25.
"""
import pytest
import torch

from tests import attention_reference as ref

gpu = pytest.mark.gpu
DEV = "cuda:0"
U, T16, Z = 2.0**-24, 2.0**-11, 2.0**-25


def one_head(q, k, v, g, causal, scale, value_norm, row_norms):
    """64-bit gradients of one query head and their bounds; value_norm: largest |v_j|, row_norms: largest |do_r| of the
    group's heads by token"""
    n, d = q.shape
    w, rel, see = ref.weights(q, k, 0, causal, scale)
    see = see.double()
    s = (q @ k.T * scale).masked_fill(see == 0, float("-inf"))
    total = torch.exp(s - s.max(-1, keepdim=True)[0]).sum(-1, keepdim=True)
    out = w @ v
    gp = g @ v.T
    e_gp = (d + 2) * U * (g.abs() @ v.abs().T)
    delta = (g * out).sum(-1, keepdim=True)
    e_whole = 1.01 * ((rel + T16) * (w @ v.abs()) + Z / total * (see @ v.abs()) + (T16 * T16 + 2 * U) * out.abs() + Z)
    e_delta = (g.abs() * e_whole).sum(-1, keepdim=True) + (d + 2) * U * (g * out).abs().sum(-1, keepdim=True)
    gs = w * (gp - delta)
    e_gs = w * (e_gp + e_delta + 2 * U * (gp.abs() + delta.abs())) + (rel + T16) * gs.abs()
    zq = 2.0**-38 * g.norm(dim=1, keepdim=True) * value_norm * see
    first = (torch.arange(n) // 64 * 64 - 64).clamp_min(0) if causal else torch.zeros(n, dtype=torch.long)
    seen_by = torch.flip(torch.cummax(torch.flip(row_norms, [0]), 0)[0], [0])[first]
    zk = 2.0**-38 * value_norm * seen_by[None, :] * see
    gv = w.T @ g
    e_gv = ((rel + T16 + n * U) * w + 2.0**-39 * see).T @ g.abs() + T16 * gv.abs() + Z
    gq = gs @ k * scale
    e_gq = ((e_gs + zq) @ k.abs() + n * U * (gs.abs() @ k.abs())) * scale + (T16 + 3 * U) * gq.abs() + Z
    gk = gs.T @ q * scale
    e_gk = ((e_gs + zk).T @ q.abs() + n * U * (gs.abs().T @ q.abs())) * scale + (T16 + 3 * U) * gk.abs() + Z
    return [gq, gk, gv], [1.01 * e + 1e-30 for e in (e_gq, e_gk, e_gv)]


def check(q, k, v, g, lens, causal):
    from aps_amd import nn_ops
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device=DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(nn_ops.attention_packed(*leaves, cu, causal=causal), leaves, g.to(DEV))
    q, k, v, g = (t.double() for t in (q, k, v, g))
    want = [torch.zeros_like(t) for t in (q, k, v)]
    bound = [torch.zeros_like(t) for t in (q, k, v)]
    a = 0
    for n in lens:
        at = slice(a, a + n)
        for h in range(hq if n else 0):
            c = h * hkv // hq
            rows = g[at, c * (hq // hkv):(c + 1) * (hq // hkv)].norm(dim=2).max(1)[0]
            x, e = one_head(q[at, h], k[at, c], v[at, c], g[at, h], causal, d**-0.5, v[at, c].norm(dim=1).max(), rows)
            for i, to in enumerate((h, c, c)):
                want[i][at, to] += x[i]
                bound[i][at, to] += e[i]
        a += n
    for name, x, w, e in zip(("gq", "gk", "gv"), got, want, bound):
        ref.check(x, w, e, name)


def half(*shape, seed, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).half()


@gpu
@pytest.mark.parametrize("std", [1e-4, 1e-3, 1.0, 300.0])
@pytest.mark.parametrize("hq,hkv,d,lens,causal", [(2, 2, 64, [400, 33, 1], True), (3, 1, 32, [200, 0, 129], False),
                                                  (4, 2, 128, [130, 500], True), (1, 1, 64, [2500], True)])
def test_gradients_of_any_size(std, hq, hkv, d, lens, causal):
    t = sum(lens)
    q, k, v = (half(t, h, d, seed=i) for i, h in enumerate((hq, hkv, hkv)))
    check(q, k, v, half(t, hq, d, seed=8, std=std), lens, causal)


@gpu
def test_gradients_near_the_largest():
    """gradients of 1e4: the weights times do . v pass 65 504 ahead of the scale, the results do not"""
    q, k, v = (half(128, 2, 128, seed=i) for i in range(3))
    check(q, k, v, half(128, 2, 128, seed=3, std=9e3).clamp(-3e4, 3e4), [64, 64], True)


@gpu
def test_values_of_any_size_and_rows_of_different_sizes():
    """small and large values; sequences and rows of one sequence whose gradients differ by 1e6"""
    lens = [300, 150, 77]
    t = sum(lens)
    for std in (1e-3, 100.0):
        q, k = (half(t, 2, 64, seed=i) for i in range(2))
        check(q, k, half(t, 2, 64, seed=2, std=std), half(t, 2, 64, seed=4, std=0.1), lens, True)
    q, k, v = (half(t, 2, 64, seed=i) for i in range(3))
    sizes = torch.full((t, 1, 1), 100.0)
    sizes[300:450] = 1e-4
    sizes[377:] = 1e-2
    falling = 10.0**torch.linspace(2, -4, 77)[:, None, None]
    sizes[450:] = falling
    check(q, k, v, (torch.randn(t, 2, 64, generator=torch.Generator().manual_seed(5)) * sizes).half(), lens, True)


@gpu
def test_gradients_of_zero_and_of_one_row():
    q, k, v = (half(70, 2, 64, seed=i) for i in range(3))
    g = torch.zeros(70, 2, 64).half()
    check(q, k, v, g, [70], True)
    g[69, 1] = half(64, seed=3, std=1e-4)
    check(q, k, v, g, [70], True)
    check(q, k, torch.zeros_like(v), half(70, 2, 64, seed=4), [40, 30], False)


@gpu
def test_captured_gradients_of_a_fused_projection():
    """slices of one projection in f16, forward and gradients captured: replays with gradients of other sizes equal the
    eager pass and stay within the bounds"""
    from aps_amd import nn_ops
    lens, h, d = [90, 41], 2, 64
    t = sum(lens)
    leaf = half(t, 3 * h * d, seed=1).to(DEV).requires_grad_()
    g = half(t, h, d, seed=2).to(DEV)
    cu = torch.tensor([0, 90, 131], device=DEV)

    def step():
        q, k, v = leaf.view(t, 3, h, d).unbind(1)
        return torch.autograd.grad(nn_ops.attention_packed(q, k, v, cu), leaf, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, std in enumerate((1e-4, 1e4, 1.0)):
        with torch.no_grad():
            leaf.copy_(half(t, 3 * h * d, seed=10 + i, std=0.3))
            g.copy_(half(t, h, d, seed=20 + i, std=std))
        graph.replay()
        torch.cuda.synchronize()
        first = held.clone()
        assert torch.equal(first, step())
        q, k, v = leaf.detach().cpu().view(t, 3, h, d).unbind(1)
        check(q, k, v, g.cpu(), lens, True)


@gpu
@pytest.mark.parametrize("causal", [True, False])
def test_values_whose_size_changes_within_a_sequence(causal):
    """keys with small values beside keys with large ones: do . o, which all of a row's values are in, is in every dS"""
    lens = [600, 300]
    t = sum(lens)
    at = torch.cat([torch.arange(n) for n in lens])
    q, k = (half(t, 2, 64, seed=i) for i in range(2))
    for size in (10.0**(3 - at / 100), 10.0**(at / 100 - 3), torch.where(at < 200, 1000.0, 1e-3), torch.where(at < 256, 0.0, 500.0),
                 torch.where(at < 256, 500.0, 0.0)):
        v = (torch.randn(t, 2, 64, generator=torch.Generator().manual_seed(2)) * size[:, None, None]).clamp(-6e4, 6e4).half()
        check(q, k, v, half(t, 2, 64, seed=4, std=0.2), lens, causal)
